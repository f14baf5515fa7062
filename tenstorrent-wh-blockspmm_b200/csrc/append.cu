// Appending keys and values to the paged 8-bit cache, the keys rotated on the
// way.
//
// Work is cut by (page, head): a page's scale belongs to all its tokens, so the
// team of warps that writes new tokens of a page also finds their largest
// magnitude, joins it with the page's scale and, where that grew, rounds the
// page's earlier codes again.
//
// A job is one head of the keys, the values or the queries of a chunk (the new
// tokens of one sequence on one page); a team does several of a chunk's jobs.  It
// has one warp per 16 tokens of its chunk, so a long prompt and many single tokens
// go together (90 tokens with one each of 63 other sequences: 13.3 us, 37 us with
// one warp a team).  Memory-bound, so the loads of the next job are
// always in flight: asynchronous copies bring its 16-bit values to shared
// memory (each lane its own, two buffers), while (cos, sin) of the warp's 16
// tokens stay in registers for all its jobs.  Keys are rotated twice, for their
// maximum and for their codes: cheaper than keeping them in 32 bits (fp32 between
// the passes spilled: 140 us against 91 then).
//
// 14278 tokens, 32 + 2 x 8 heads of 128, pages of 16: 66 us, 5400 GB/s, 83 % of a
// plain copy's rate (58 % of the issue slots, 23 % of the warps: registers allow
// two blocks an SM).  A token each of 64 sequences: 5.0 us, latency.
#include <cuda_fp8.h>

#include "bsp_ptx.cuh"
#include "rope.cuh"

namespace bsp {
using namespace dev;

namespace {

constexpr int kApWarps = 8;
// Tokens of one head that a warp takes at once: side by side (a head of 128 is 8
// lanes, of 64 4) and one after the other, 16 in all where sequences bring many.
constexpr int kApTokens = 16;
constexpr int ap_across(int d) { return 512 / d; }

// New tokens [t0, t0 + n) of one sequence, at slots [slot, slot + n) of page.
struct Chunk {
  int32_t page, slot, n;
  int32_t warps;  // of a team, a power of two
  int64_t t0, pos0;
};

// Chunk c of the launch: sequence s owns the chunks from starts[s] / page + 2 s
// on (it touches at most (starts[s + 1] - starts[s]) / page + 2 pages), or from
// starts[s] on where that is fewer in all (it touches at most a page a token: a
// token each of 64 sequences takes 4.9 us that way, 6.0 us with twice as many
// blocks, half of them without a chunk).  So the sequence is found by a search in
// steps of 32 and no host copy of the lengths is needed.
__device__ __forceinline__ int64_t first_chunk(const AppendParams& p, int s) {
  const int64_t start = p.starts[s];
  return p.by_token ? start : (start >> p.page_shift) + 2 * static_cast<int64_t>(s);
}
__device__ __forceinline__ bool find_chunk(const AppendParams& p, int64_t c, int lane, Chunk& out) {
  const int page = p.cache.page;
  int lo = 0, n_left = p.n_seqs;  // the last s in [lo, lo + n_left) with first_chunk(s) <= c
  while (n_left > 1) {
    const int step = (n_left + 31) / 32, s = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, lane * step < n_left && first_chunk(p, s) <= c);
    const int k = below ? 31 - __clz(below) : 0;
    lo += k * step;
    n_left = min(step, n_left - k * step);
  }
  const int64_t t0 = p.starts[lo], n = p.starts[lo + 1] - t0, b = p.before[lo];
  if (t0 < 0 || n < 0 || t0 + n > p.tokens || b < 0) {
    if (lane == 0) atomicOr(p.status, ST_BAD_INDEX);
    return false;
  }
  const int64_t local = c - (p.by_token ? t0 : (t0 >> p.page_shift) + 2 * static_cast<int64_t>(lo));
  const int64_t off = b & (page - 1);
  if (local < 0 || n == 0 || local >= (off + n + page - 1) >> p.page_shift) return false;
  const int64_t index = (b >> p.page_shift) + local;
  out.slot = local == 0 ? static_cast<int32_t>(off) : 0;
  out.t0 = t0 + local * page + out.slot - off;
  out.pos0 = b + (out.t0 - t0);
  const int64_t left = t0 + n - out.t0;
  out.n = static_cast<int32_t>(left < page - out.slot ? left : page - out.slot);
  out.page = index < p.table_width ? p.page_table[lo * p.table_stride + index] : -1;
  if (p.table && out.pos0 + out.n > p.n_pos) {
    if (lane == 0) atomicOr(p.status, ST_BAD_INDEX);
    return false;
  }
  return true;
}

// Smallest e in [-100, 119] with amax <= 448 * 2^e (448 = 1.75 * 2^8, the
// largest e4m3 value), from the bits of amax; 0 when amax is 0.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  if (b == 0) return 0;
  const int e = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return min(max(e, -100), 119);
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ __forceinline__ float finite_or_nan(float x) {
  return fabsf(x) <= 3.402823466e38f ? x : __uint_as_float(0x7FC00000u);
}
__device__ __forceinline__ uint32_t codes4(const float* v, float f) {
  const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(finite_or_nan(v[0]) * f, finite_or_nan(v[1]) * f),
                                              __NV_SATFINITE, __NV_E4M3);
  const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(finite_or_nan(v[2]) * f, finite_or_nan(v[3]) * f),
                                              __NV_SATFINITE, __NV_E4M3);
  return a | (b << 16);
}

__device__ __forceinline__ float code_value(uint32_t c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(c), __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

__device__ __forceinline__ void team_sync(int team, int team_warps) {
  if (team_warps == 1) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(32 * team_warps) : "memory");
}

__device__ __forceinline__ bool bad_page(const AppendParams& p, const Chunk& ck, int lane) {
  if (ck.page >= 0 && ck.page < p.cache.n_pages) return false;
  if (lane == 0) atomicOr(p.status, ST_BAD_INDEX);
  return true;
}

// Largest finite magnitude.
__device__ __forceinline__ float magnitude(const float (&lo)[8], const float (&hi)[8], float m) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = fabsf(lo[j]), b = fabsf(hi[j]);
    m = fmaxf(m, a <= 3.402823466e38f ? a : 0.f);
    m = fmaxf(m, b <= 3.402823466e38f ? b : 0.f);
  }
  return m;
}

// Where a team's keys or values of one head go.
struct Target {
  uint8_t* codes;  // of the chunk's first token
  float scale;     // 2^-e
};

// The warp looks whether `bytes` codes (a multiple of 16) are all zeros.
__device__ __forceinline__ bool only_zeros(const uint8_t* codes, int bytes, int lane) {
  uint32_t some = 0;
  for (int i = lane; i < bytes / 16; i += 32) {
    const uint4 c = reinterpret_cast<const uint4*>(codes)[i];
    some |= c.x | c.y | c.z | c.w;
  }
  return !__any_sync(0xFFFFFFFFu, (some & 0x7F7F7F7Fu) != 0);
}

// The page's exponent from the lanes' maxima and what the page holds; earlier
// codes are rounded again where it grew.
template <int kD>
__device__ __forceinline__ Target settle(const AppendParams& p, const Chunk& ck, bool is_v, int h, int team, int in_team,
                                        int lane, float* s_max, float m) {
  uint8_t* codes = static_cast<uint8_t*>(is_v ? p.cache.v : p.cache.k) + ck.page * p.cache.page_stride +
                   h * p.cache.head_stride;
  float* sp = (is_v ? p.cache.v_scale : p.cache.k_scale) + static_cast<int64_t>(ck.page) * p.cache.kv_heads + h;
  const uint32_t old_bits = ck.slot > 0 ? __float_as_uint(*sp) : 0;
  for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, k));
  if (ck.warps > 1) {
    team_sync(team, ck.warps);  // the last job's maxima have been read
    if (lane == 0) s_max[team * ck.warps + in_team] = m;
    team_sync(team, ck.warps);
    for (int k = 0; k < ck.warps; ++k) m = fmaxf(m, s_max[team * ck.warps + k]);
  } else {
    __syncwarp();
  }
  int e = scale_exponent(m);
  if (ck.slot > 0) {
    int was = min(max(static_cast<int>((old_bits >> 23) & 0xFFu) - 127, -100), 119);
    // Zeros have no size: a page that holds nothing else has scale 1, which smaller
    // values behind them would be rounded away with.  Any scale is theirs.
    if (was == 0 && e < 0 && only_zeros(codes, ck.slot * kD, lane)) was = e;
    if (was >= e) {
      e = was;
    } else {
      const float f = two_to(max(was - e, -126));
      uint32_t* w = reinterpret_cast<uint32_t*>(codes);
      for (int i = 32 * in_team + lane; i < ck.slot * (kD / 4); i += 32 * ck.warps) {
        const uint32_t c = w[i];
        const float v[4] = {code_value(c & 0xFF), code_value((c >> 8) & 0xFF), code_value((c >> 16) & 0xFF),
                            code_value(c >> 24)};
        w[i] = codes4(v, f);
      }
    }
  }
  // every thread of the team has its copy of the old scale by now
  if (in_team == 0 && lane == 0) *sp = two_to(e);
  return {codes + static_cast<int64_t>(ck.slot) * kD, two_to(-e)};
}

__device__ __forceinline__ void put_codes(uint8_t* c, const RopeUnit<8>& un, const float (&lo)[8], const float (&hi)[8],
                                         float scale) {
  *reinterpret_cast<uint2*>(c + un.lo) = make_uint2(codes4(lo, scale), codes4(lo + 4, scale));
  *reinterpret_cast<uint2*>(c + un.hi) = make_uint2(codes4(hi, scale), codes4(hi + 4, scale));
}

// A job of a chunk: input, 16-bit output (may be null) and what becomes of it.
struct Job {
  const uint16_t* x;
  uint16_t* y;
  int64_t x_token, y_token;
  int h;
  bool is_q, is_v;
};
__device__ __forceinline__ Job job_of(const AppendParams& p, const Chunk& ck, int job) {
  const int hk = p.cache.kv_heads;
  Job j;
  j.is_q = job >= 2 * hk;
  j.is_v = !j.is_q && job >= hk;
  j.h = j.is_q ? job - 2 * hk : j.is_v ? job - hk : job;
  const HeadsView& in = j.is_q ? p.q : j.is_v ? p.v : p.k;
  const HeadsOut& out = j.is_q ? p.q_out : p.k_out;
  j.x_token = in.token;
  j.y_token = out.token;
  j.x = static_cast<const uint16_t*>(in.p) + ck.t0 * in.token + j.h * in.head;
  j.y = !j.is_v && out.p ? static_cast<uint16_t*>(out.p) + ck.t0 * out.token + j.h * out.head : nullptr;
  return j;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// More tokens on the page than the team's warps hold at once (a long prompt
// among many single tokens): straight from memory, twice for keys and values.
template <int kUnits, bool kInterleaved>
__device__ __noinline__ void append_long(const AppendParams& p, const Chunk& ck, int job, int team, int in_team,
                                         int lane, float* s_max) {
  constexpr int kAcross = 32 / kUnits, kD = 16 * kUnits;
  const Job j = job_of(p, ck, job);
  const int u = lane % kUnits;
  const RopeUnit<8> un(u, p.table && !j.is_v ? p.rot : 0, kD);
  float m = 0.f;
  Target to{nullptr, 1.f};
  for (int pass = j.is_q ? 1 : 0; pass < 2; ++pass) {
    for (int t = in_team * kAcross + lane / kUnits; t < ck.n; t += kAcross * ck.warps) {
      float lo[8], hi[8];
      load_vec(j.x + t * j.x_token + un.lo, lo);
      load_vec(j.x + t * j.x_token + un.hi, hi);
      if (un.turns) {
        float2 cs[8];
        load_turns<8>(p.table + (ck.pos0 + t) * (p.rot / 2), u, p.rot, kInterleaved, cs);
        turn_unit<8>(lo, hi, cs, kInterleaved, 1.f);
      }
      if (pass == 0) {
        m = magnitude(lo, hi, m);
      } else {
        if (!j.is_q) put_codes(to.codes + t * kD, un, lo, hi, to.scale);
        if (j.y) {
          store_vec(j.y + t * j.y_token + un.lo, lo);
          store_vec(j.y + t * j.y_token + un.hi, hi);
        }
      }
    }
    if (pass == 0) to = settle<kD>(p, ck, j.is_v, j.h, team, in_team, lane, s_max, m);
  }
}

// kUnits: units of two vectors of 8 values in a head (d / 16); kDeep: tokens one
// after the other.  With one, a block needs half the registers, and twice as many
// are on an SM.
template <int kUnits, bool kInterleaved, int kDeep>
__global__ void __launch_bounds__(32 * kApWarps, kDeep == 1 ? 4 : 2) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kAcross = 32 / kUnits;        // tokens side by side in a warp
  constexpr int kTokens = kAcross * kDeep;
  constexpr int kD = 16 * kUnits;
  __shared__ float s_max[kApWarps];
  extern __shared__ uint4 s_raw[];            // per warp 2 x [kDeep][2][32]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int jobs = 2 * p.cache.kv_heads + (p.q.p ? p.heads : 0);
  stream_release();
  stream_wait();
  Chunk ck;
  if (!find_chunk(p, blockIdx.x, lane, ck)) return;
  // log2 of the team's warps: kTokens << shift holds the chunk, or it is the block
  const int shift = min(32 - __clz((ck.n - 1) / kTokens), 31 - __clz(kApWarps));
  ck.warps = 1 << shift;
  const int team = warp >> shift, in_team = warp & (ck.warps - 1), teams = kApWarps >> shift;
  const int first = blockIdx.y * teams + team, step = gridDim.y * teams;
  if (ck.n > kTokens * ck.warps) {
    const bool bad = bad_page(p, ck, lane);
    for (int job = first; job < jobs && !bad; job += step)
      append_long<kUnits, kInterleaved>(p, ck, job, team, in_team, lane, s_max);
    return;
  }
  const int u = lane % kUnits, t0 = in_team * kTokens + lane / kUnits;  // this lane's tokens: t0 + kAcross k
  const RopeUnit<8> turned(u, p.table ? p.rot : 0, kD), plain(u, 0, kD);
  uint4* raw = s_raw + warp * (2 * kDeep * 2 * 32) + lane;
  auto fetch = [&](int job, int buf) {
    if (job < jobs) {
      const Job j = job_of(p, ck, job);
      const int lo = j.is_v ? plain.lo : turned.lo, hi = j.is_v ? plain.hi : turned.hi;
#pragma unroll
      for (int k = 0; k < kDeep; ++k) {
        const int t = t0 + kAcross * k;
        if (t < ck.n) {
          copy16(smem_u32(raw + ((buf * kDeep + k) * 2 + 0) * 32), j.x + t * j.x_token + lo);
          copy16(smem_u32(raw + ((buf * kDeep + k) * 2 + 1) * 32), j.x + t * j.x_token + hi);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(first, 0);
  float2 cs[kDeep][8];
  if (turned.turns) {
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
      if (t0 + kAcross * k < ck.n)
        load_turns<8>(p.table + (ck.pos0 + t0 + kAcross * k) * (p.rot / 2), u, p.rot, kInterleaved, cs[k]);
  }
  if (bad_page(p, ck, lane)) {  // (looked at behind the first copies, which do not wait for the page)
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    return;
  }
  int buf = 0;
  for (int job = first; job < jobs; job += step, buf ^= 1) {
    fetch(job + step, buf ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    const Job j = job_of(p, ck, job);
    const RopeUnit<8>& un = j.is_v ? plain : turned;
    float lo[8], hi[8];
    auto take = [&](int k) {  // token t0 + kAcross k, rotated
      unpack8(raw[((buf * kDeep + k) * 2 + 0) * 32], lo);
      unpack8(raw[((buf * kDeep + k) * 2 + 1) * 32], hi);
      if (un.turns) turn_unit<8>(lo, hi, cs[k], kInterleaved, 1.f);
    };
    Target to{nullptr, 1.f};
    if (!j.is_q) {
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < kDeep; ++k)
        if (t0 + kAcross * k < ck.n) {
          take(k);
          m = magnitude(lo, hi, m);
        }
      to = settle<kD>(p, ck, j.is_v, j.h, team, in_team, lane, s_max, m);
    }
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int t = t0 + kAcross * k;
      if (t < ck.n) {
        take(k);
        if (!j.is_q) put_codes(to.codes + t * kD, un, lo, hi, to.scale);
        if (j.y) {
          store_vec(j.y + t * j.y_token + un.lo, lo);
          store_vec(j.y + t * j.y_token + un.hi, hi);
        }
      }
    }
  }
}

using AppendKernel = void (*)(AppendParams);
template <int kUnits, bool kInterleaved>
AppendKernel pick(bool few) {
  return few ? append_kernel<kUnits, kInterleaved, 1> : append_kernel<kUnits, kInterleaved, kApTokens * kUnits / 32>;
}
AppendKernel pick(int d, bool interleaved, bool few) {
  return d == 64 ? (interleaved ? pick<4, true>(few) : pick<4, false>(few))
                 : (interleaved ? pick<8, true>(few) : pick<8, false>(few));
}
constexpr int raw_bytes(int d, bool few) { return kApWarps * 2 * (few ? ap_across(d) : kApTokens) * d * 2; }

}  // namespace

bsp_status launch_append(AppendParams& p, bsp_device* dev, cudaStream_t stream) {
  if (!dev->append_ready) {
    for (int d : {64, 128})
      for (bool i : {false, true}) {
        const bsp_status s = cuda_check(
            cudaFuncSetAttribute(pick(d, i, false), cudaFuncAttributeMaxDynamicSharedMemorySize, raw_bytes(d, false)),
            "cudaFuncSetAttribute(append)");
        if (s != BSP_OK) return s;
      }
    dev->append_ready = true;
  }
  const int page = p.cache.page;
  p.page_shift = __builtin_ctz(static_cast<unsigned>(page));
  const int64_t per_seq = p.tokens / p.n_seqs;
  // A step of decoding (no more tokens than sequences) whose chunks do not fit the
  // GPU's blocks at once: a warp takes fewer tokens, so that twice as many blocks do
  // (a token each of 512 sequences 13.4 us, 17.0 us with 16 tokens a warp; of 64
  // sequences 5.0 us either way).
  const bool few = p.tokens <= p.n_seqs && p.n_seqs > 2 * dev->sm_count;
  const int64_t by_page = p.tokens / page + 2 * static_cast<int64_t>(p.n_seqs);
  p.by_token = p.tokens < by_page;
  const int64_t chunks = std::min(p.tokens, by_page);
  if (chunks > 0x7FFFFFFF) return set_error(BSP_ERR_UNSUPPORTED, "too many sequences");
  const int jobs = 2 * p.cache.kv_heads + (p.q.p ? p.heads : 0);
  int64_t teams = kApWarps;  // that a block has for a chunk of average length
  while (teams > 1 && kApTokens * kApWarps <= teams * std::min<int64_t>(per_seq, page) / 2) teams /= 2;
  // A job to a team while that does not need more blocks than the GPU holds at
  // once (two an SM), else several: 14278 tokens in pages of 16 take 68 us with
  // one block to a chunk (of 904), 74 us with three and 96 us with six; a token
  // each of 64 sequences 4.9 us with four blocks to a chunk, 5.1 us with six.
  const int64_t most = (jobs + teams - 1) / teams;
  const int64_t enough = std::max<int64_t>((few ? 4 : 2) * static_cast<int64_t>(dev->sm_count) / (p.tokens / page + p.n_seqs), 1);
  const dim3 grid(static_cast<unsigned>(chunks), static_cast<unsigned>(std::min(most, enough)));
  return launch_overlapped(pick(p.cache.d, p.interleaved, few), grid, 32 * kApWarps, raw_bytes(p.cache.d, few), stream, p,
                           "cache append launch");
}

}  // namespace bsp
