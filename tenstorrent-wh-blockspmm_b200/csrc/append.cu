// Appending keys and values to the paged 8-bit cache, the keys rotated on the
// way.
//
// Work is cut by (page, head): a page's scale belongs to all its tokens, so the
// team of warps that writes new tokens of a page also finds their largest
// magnitude, joins it with the page's scale and, where that grew, rounds the
// page's earlier codes again.  Memory-bound: 16 tokens of a head stay in the
// registers of a warp between the search for the maximum and the store, so each
// value is read once.
//
// Jobs of a chunk (the new tokens of one sequence on one page): keys of a head,
// values of a head, and queries of four heads, for which each (cos, sin) is
// loaded once.  A team has one warp per 16 tokens of the page when sequences
// bring pages of tokens, and a single warp when they bring one token each: a
// warp with nothing to do still costs its start.  Finding the chunk is a chain
// of dependent loads, so a team does several jobs of its chunk once there are
// enough warps to fill the GPU, and the page number is not waited for before
// the data are on their way.
#include <cuda_fp8.h>

#include "rope.cuh"

namespace bsp {
using namespace dev;

namespace {

constexpr int kApWarps = 8;
constexpr int kApTokens = 16;  // of one head in a warp's registers
constexpr int kApQHeads = 4;   // query heads of a job

// New tokens [t0, t0 + n) of one sequence, at slots [slot, slot + n) of page.
struct Chunk {
  int32_t page, slot, n;
  int64_t t0, pos0;
};

// Chunk c of the launch: sequence s owns the chunks from starts[s] / page + 2 s
// on (it touches at most (starts[s + 1] - starts[s]) / page + 2 pages), so the
// sequence is found by a search in steps of 32 and no host copy of the lengths
// is needed.
__device__ __forceinline__ int64_t first_chunk(const AppendParams& p, int s) {
  return (static_cast<int64_t>(__ldg(p.starts + s)) >> p.page_shift) + 2 * static_cast<int64_t>(s);
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
  const int64_t t0 = __ldg(p.starts + lo), n = __ldg(p.starts + lo + 1) - t0, b = __ldg(p.before + lo);
  if (t0 < 0 || n < 0 || t0 + n > p.tokens || b < 0) {
    if (lane == 0) atomicOr(p.status, ST_BAD_INDEX);
    return false;
  }
  const int64_t local = c - ((t0 >> p.page_shift) + 2 * static_cast<int64_t>(lo));
  const int64_t off = b & (page - 1);
  if (local < 0 || n == 0 || local >= (off + n + page - 1) >> p.page_shift) return false;
  const int64_t index = (b >> p.page_shift) + local;
  out.slot = local == 0 ? static_cast<int32_t>(off) : 0;
  out.t0 = t0 + local * page + out.slot - off;
  out.pos0 = b + (out.t0 - t0);
  const int64_t left = t0 + n - out.t0;
  out.n = static_cast<int32_t>(left < page - out.slot ? left : page - out.slot);
  out.page = index < p.table_width ? __ldg(p.page_table + lo * p.table_stride + index) : -1;
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

// Queries of up to four heads of a chunk, from h0 on.
template <int kUnits, bool kInterleaved>
__device__ __forceinline__ void append_queries(const AppendParams& p, const Chunk& ck, int h0, int in_team, int lane) {
  constexpr int kAcross = 32 / kUnits, kD = 16 * kUnits;
  const int u = lane % kUnits, nh = min(kApQHeads, p.heads - h0);
  const RopeUnit<8> un(u, p.rot, kD);
  const float2* turns = p.table + ck.pos0 * (p.rot / 2);
  for (int t = in_team * kAcross + lane / kUnits; t < ck.n; t += kAcross * p.team_warps) {
    const uint16_t* x = static_cast<const uint16_t*>(p.q.p) + (ck.t0 + t) * p.q.token + h0 * p.q.head;
    uint16_t* y = static_cast<uint16_t*>(p.q_out.p) + (ck.t0 + t) * p.q_out.token + h0 * p.q_out.head;
    uint4 raw[kApQHeads][2];
#pragma unroll
    for (int h = 0; h < kApQHeads; ++h)
      if (h < nh) {
        raw[h][0] = *reinterpret_cast<const uint4*>(x + h * p.q.head + un.lo);
        raw[h][1] = *reinterpret_cast<const uint4*>(x + h * p.q.head + un.hi);
      }
    float2 cs[8];
    if (un.turns) load_turns<8>(turns + static_cast<int64_t>(t) * (p.rot / 2), u, p.rot, kInterleaved, cs);
#pragma unroll
    for (int h = 0; h < kApQHeads; ++h)
      if (h < nh) {
        float lo[8], hi[8];
        unpack8(raw[h][0], lo);
        unpack8(raw[h][1], hi);
        if (un.turns) turn_unit<8>(lo, hi, cs, kInterleaved, 1.f);
        store_vec(y + h * p.q_out.head + un.lo, lo);
        store_vec(y + h * p.q_out.head + un.hi, hi);
      }
  }
}

// Keys or values of one head of a chunk.  What stays in registers between the
// two passes are the 16-bit values as they came: the rotation is done in both.
template <int kUnits, bool kInterleaved>
__device__ __forceinline__ void append_codes(const AppendParams& p, const Chunk& ck, bool is_v, int h, int team,
                                             int in_team, int lane, float* s_max) {
  constexpr int kAcross = 32 / kUnits;           // tokens side by side in a warp
  constexpr int kDeep = kApTokens / kAcross;     // and one after the other
  constexpr int kD = 16 * kUnits;
  const int u = lane % kUnits, at = lane / kUnits;
  const int stride = kApTokens * p.team_warps;
  const RopeUnit<8> un(u, p.table && !is_v ? p.rot : 0, kD);
  const float2* turns = p.table + ck.pos0 * (p.rot / 2);
  const HeadsView& in = is_v ? p.v : p.k;
  const uint16_t* x = static_cast<const uint16_t*>(in.p) + ck.t0 * in.token + h * in.head;
  uint4 raw[kDeep][2];
  auto load = [&](int base) {
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int t = base + k * kAcross + at;
      raw[k][0] = raw[k][1] = make_uint4(0, 0, 0, 0);
      if (t < ck.n) {
        raw[k][0] = *reinterpret_cast<const uint4*>(x + t * in.token + un.lo);
        raw[k][1] = *reinterpret_cast<const uint4*>(x + t * in.token + un.hi);
      }
    }
  };
  float lo[8], hi[8];
  auto values = [&](const uint4 (&r)[2], int t) {
    unpack8(r[0], lo);
    unpack8(r[1], hi);
    if (un.turns && t < ck.n) {
      float2 cs[8];
      load_turns<8>(turns + static_cast<int64_t>(t) * (p.rot / 2), u, p.rot, kInterleaved, cs);
      turn_unit<8>(lo, hi, cs, kInterleaved, 1.f);
    }
  };
  float m = 0.f;
  for (int base = in_team * kApTokens; base < ck.n; base += stride) {
    load(base);
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      values(raw[k], base + k * kAcross + at);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = fabsf(lo[j]), b = fabsf(hi[j]);
        m = fmaxf(m, a <= 3.402823466e38f ? a : 0.f);
        m = fmaxf(m, b <= 3.402823466e38f ? b : 0.f);
      }
    }
  }
  if (ck.page < 0 || ck.page >= p.cache.n_pages) {  // the whole team leaves
    if (lane == 0) atomicOr(p.status, ST_BAD_INDEX);
    return;
  }
  uint8_t* codes = static_cast<uint8_t*>(is_v ? p.cache.v : p.cache.k) + ck.page * p.cache.page_stride +
                   h * p.cache.head_stride;
  float* sp = (is_v ? p.cache.v_scale : p.cache.k_scale) +
              static_cast<int64_t>(ck.page) * p.cache.kv_heads + h;
  const uint32_t old_bits = ck.slot > 0 ? __float_as_uint(*sp) : 0;
  for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, k));
  if (p.team_warps > 1) {
    team_sync(team, p.team_warps);  // the last job's maxima have been read
    if (lane == 0) s_max[team * p.team_warps + in_team] = m;
    team_sync(team, p.team_warps);
    for (int k = 0; k < p.team_warps; ++k) m = fmaxf(m, s_max[team * p.team_warps + k]);
  } else {
    __syncwarp();
  }
  int e = scale_exponent(m);
  if (ck.slot > 0) {
    const int was = min(max(static_cast<int>((old_bits >> 23) & 0xFFu) - 127, -100), 119);
    if (was >= e) {
      e = was;
    } else {
      const float f = two_to(max(was - e, -126));
      uint32_t* w = reinterpret_cast<uint32_t*>(codes);
      for (int i = 32 * in_team + lane; i < ck.slot * (kD / 4); i += 32 * p.team_warps) {
        const uint32_t c = w[i];
        const float v[4] = {code_value(c & 0xFF), code_value((c >> 8) & 0xFF), code_value((c >> 16) & 0xFF),
                            code_value(c >> 24)};
        w[i] = codes4(v, f);
      }
    }
  }
  // every thread of the team has its copy of the old scale by now
  if (in_team == 0 && lane == 0) *sp = two_to(e);
  const float scale = two_to(-e);
  codes += static_cast<int64_t>(ck.slot) * kD;
  uint16_t* y = !is_v && p.k_out.p
                    ? static_cast<uint16_t*>(p.k_out.p) + ck.t0 * p.k_out.token + h * p.k_out.head : nullptr;
  const bool again = ck.n > stride;  // more tokens than the team's registers hold
  for (int base = in_team * kApTokens; base < ck.n; base += stride) {
    if (again) load(base);
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int t = base + k * kAcross + at;
      if (t < ck.n) {
        values(raw[k], t);
        uint8_t* c = codes + t * kD;
        *reinterpret_cast<uint2*>(c + un.lo) = make_uint2(codes4(lo, scale), codes4(lo + 4, scale));
        *reinterpret_cast<uint2*>(c + un.hi) = make_uint2(codes4(hi, scale), codes4(hi + 4, scale));
        if (y) {
          store_vec(y + t * p.k_out.token + un.lo, lo);
          store_vec(y + t * p.k_out.token + un.hi, hi);
        }
      }
    }
  }
}

// kUnits: units of two vectors of 8 values in a head (d / 16).
template <int kUnits, bool kInterleaved>
__global__ void __launch_bounds__(32 * kApWarps, 2) append_kernel(const AppendParams p) {
  __shared__ float s_max[kApWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int team = warp / p.team_warps, in_team = warp % p.team_warps;
  const int teams = kApWarps / p.team_warps, hk = p.cache.kv_heads;
  const int jobs = 2 * hk + (p.q.p ? (p.heads + kApQHeads - 1) / kApQHeads : 0);
  Chunk ck;
  if (!find_chunk(p, blockIdx.x, lane, ck)) return;
  for (int job = blockIdx.y * teams + team; job < jobs; job += gridDim.y * teams) {
    if (job < 2 * hk)
      append_codes<kUnits, kInterleaved>(p, ck, job >= hk, job >= hk ? job - hk : job, team, in_team, lane, s_max);
    else
      append_queries<kUnits, kInterleaved>(p, ck, (job - 2 * hk) * kApQHeads, in_team, lane);
  }
}

}  // namespace

bsp_status launch_append(AppendParams& p, int sm_count, cudaStream_t stream) {
  const int page = p.cache.page;
  p.page_shift = __builtin_ctz(static_cast<unsigned>(page));
  const int64_t per_seq = p.tokens / p.n_seqs;
  p.team_warps = 1;
  while (p.team_warps * 2 * kApTokens <= std::min<int64_t>(per_seq, page)) p.team_warps *= 2;
  const int64_t chunks = p.tokens / page + 2 * static_cast<int64_t>(p.n_seqs);
  if (chunks > 0x7FFFFFFF) return set_error(BSP_ERR_UNSUPPORTED, "too many sequences");
  const int jobs = 2 * p.cache.kv_heads + (p.q.p ? (p.heads + kApQHeads - 1) / kApQHeads : 0);
  const int teams = kApWarps / p.team_warps;
  // as many blocks to a chunk as its jobs fill, or fewer once four rounds of
  // blocks of all chunks fill the GPU (two of them fit an SM)
  const int64_t most = (jobs + teams - 1) / teams, enough = 8 * static_cast<int64_t>(sm_count) / (p.tokens / page + 1) + 1;
  const dim3 grid(static_cast<unsigned>(chunks), static_cast<unsigned>(std::min(most, enough)));
  const auto kernel = p.cache.d == 64 ? (p.interleaved ? append_kernel<4, true> : append_kernel<4, false>)
                                      : (p.interleaved ? append_kernel<8, true> : append_kernel<8, false>);
  kernel<<<grid, 32 * kApWarps, 0, stream>>>(p);
  return cuda_check(cudaGetLastError(), "cache append launch");
}

}  // namespace bsp
