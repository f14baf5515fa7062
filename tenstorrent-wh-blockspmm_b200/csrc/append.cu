// Appending keys and values to the paged 8-bit cache, the keys rotated on the
// way.
//
// Work is cut by (page, head): a page's scale belongs to all its tokens, so the
// block that writes new tokens of a page also finds their largest magnitude,
// joins it with the page's scale and, where that grew, rounds the page's
// earlier codes again.
#include <cuda_fp8.h>

#include "rope.cuh"

namespace bsp {
using namespace dev;

namespace {

constexpr int kApThreads = 128;

// New tokens [t0, t0 + n) of one sequence, at slots [slot, slot + n) of page.
struct Chunk {
  int32_t page, slot, n;
  int64_t t0, pos0;
};

// Chunk c of the launch: sequence s owns the chunks from starts[s] / page + 2 s
// on (it touches at most (starts[s + 1] - starts[s]) / page + 2 pages), so the
// sequence is found by bisection and no host copy of the lengths is needed.
__device__ bool find_chunk(const AppendParams& p, int64_t c, Chunk& out) {
  const int page = p.cache.page;
  int lo = 0, hi = p.n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (static_cast<int64_t>(__ldg(p.starts + mid)) / page + 2 * static_cast<int64_t>(mid) <= c) lo = mid;
    else hi = mid - 1;
  }
  const int64_t t0 = __ldg(p.starts + lo), n = __ldg(p.starts + lo + 1) - t0, b = __ldg(p.before + lo);
  if (t0 < 0 || n < 0 || t0 + n > p.tokens || b < 0) {
    if (threadIdx.x == 0) atomicOr(p.status, ST_BAD_INDEX);
    return false;
  }
  const int64_t local = c - (t0 / page + 2 * static_cast<int64_t>(lo));
  const int64_t off = b % page;
  if (local < 0 || n == 0 || local >= (off + n + page - 1) / page) return false;
  const int64_t index = b / page + local;
  out.slot = local == 0 ? static_cast<int32_t>(off) : 0;
  out.t0 = t0 + local * page + out.slot - off;
  out.pos0 = b + (out.t0 - t0);
  const int64_t left = t0 + n - out.t0;
  out.n = static_cast<int32_t>(left < page - out.slot ? left : page - out.slot);
  out.page = index < p.table_width ? __ldg(p.page_table + lo * p.table_stride + index) : -1;
  if (out.page < 0 || out.page >= p.cache.n_pages || (p.table && out.pos0 + out.n > p.n_pos)) {
    if (threadIdx.x == 0) atomicOr(p.status, ST_BAD_INDEX);
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

__global__ void __launch_bounds__(kApThreads) append_kernel(const AppendParams p) {
  Chunk ck;
  if (!find_chunk(p, blockIdx.x, ck)) return;
  const int d = p.cache.d, units = d / 16, hk = p.cache.kv_heads;
  const int job = blockIdx.y;  // K of a head, V of a head, then the query heads
  const bool is_k = job < hk, is_v = !is_k && job < 2 * hk;
  const int h = is_k ? job : is_v ? job - hk : job - 2 * hk;
  const HeadsView& in = is_k ? p.k : is_v ? p.v : p.q;
  const uint16_t* x = static_cast<const uint16_t*>(in.p) + ck.t0 * in.token + h * in.head;
  const bool rotate = p.table != nullptr && !is_v;
  const HeadsOut& o16 = is_k ? p.k_out : p.q_out;
  const bool keep16 = !is_v && o16.p != nullptr;
  auto unit = [&](int i, float (&lo)[8], float (&hi)[8], int& t, int& u) {
    t = i / units;
    u = i - t * units;
    const RopeUnit un(u, rotate ? p.rot : 0, p.interleaved);
    load8(x + t * in.token + un.lo, lo);
    load8(x + t * in.token + un.hi, hi);
    if (un.turns) {
      float2 cs[8];
      load_turns(p.table + (ck.pos0 + t) * (p.rot / 2), u, cs);
      turn16(lo, hi, cs, p.interleaved, 1.f);
    }
    return un;
  };
  const int n_units = ck.n * units;
  float lo[8], hi[8];
  int t, u;
  float scale = 1.f;
  __shared__ float s_max[kApThreads / 32];
  if (is_k || is_v) {
    float m = 0.f;
    for (int i = threadIdx.x; i < n_units; i += kApThreads) {
      unit(i, lo, hi, t, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = fabsf(lo[j]), b = fabsf(hi[j]);
        m = fmaxf(m, a <= 3.402823466e38f ? a : 0.f);
        m = fmaxf(m, b <= 3.402823466e38f ? b : 0.f);
      }
    }
    for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, k));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    int e = scale_exponent(m);
    uint8_t* codes = static_cast<uint8_t*>(is_k ? p.cache.k : p.cache.v) + ck.page * p.cache.page_stride +
                     h * p.cache.head_stride;
    float* sp = (is_k ? p.cache.k_scale : p.cache.v_scale) + static_cast<int64_t>(ck.page) * hk + h;
    if (ck.slot > 0) {
      const int was = min(max(static_cast<int>((__float_as_uint(*sp) >> 23) & 0xFFu) - 127, -100), 119);
      if (was >= e) {
        e = was;
      } else {
        const float f = two_to(max(was - e, -126));
        for (int i = threadIdx.x; i < ck.slot * d / 4; i += kApThreads) {
          const uint32_t w = reinterpret_cast<uint32_t*>(codes)[i];
          const float v[4] = {code_value(w & 0xFF), code_value((w >> 8) & 0xFF), code_value((w >> 16) & 0xFF),
                              code_value(w >> 24)};
          reinterpret_cast<uint32_t*>(codes)[i] = codes4(v, f);
        }
      }
    }
    __syncthreads();  // every thread has read the old scale
    if (threadIdx.x == 0) *sp = two_to(e);
    scale = two_to(-e);
    codes += static_cast<int64_t>(ck.slot) * d;
    for (int i = threadIdx.x; i < n_units; i += kApThreads) {
      const RopeUnit un = unit(i, lo, hi, t, u);
      uint8_t* c = codes + t * d;
      *reinterpret_cast<uint2*>(c + un.lo) = make_uint2(codes4(lo, scale), codes4(lo + 4, scale));
      *reinterpret_cast<uint2*>(c + un.hi) = make_uint2(codes4(hi, scale), codes4(hi + 4, scale));
      if (keep16) {
        uint16_t* y = static_cast<uint16_t*>(o16.p) + (ck.t0 + t) * o16.token + h * o16.head;
        store8(y + un.lo, lo);
        store8(y + un.hi, hi);
      }
    }
  } else {
    for (int i = threadIdx.x; i < n_units; i += kApThreads) {
      const RopeUnit un = unit(i, lo, hi, t, u);
      uint16_t* y = static_cast<uint16_t*>(o16.p) + (ck.t0 + t) * o16.token + h * o16.head;
      store8(y + un.lo, lo);
      store8(y + un.hi, hi);
    }
  }
}

}  // namespace

bsp_status launch_append(const AppendParams& p, cudaStream_t stream) {
  const int64_t chunks = p.tokens / p.cache.page + 2 * static_cast<int64_t>(p.n_seqs);
  const dim3 grid(static_cast<unsigned>(chunks), 2 * p.cache.kv_heads + (p.q.p ? p.heads : 0));
  append_kernel<<<grid, kApThreads, 0, stream>>>(p);
  return cuda_check(cudaGetLastError(), "cache append launch");
}

}  // namespace bsp
