// Attention of one token of each sequence over the paged 8-bit cache:
//   o = sum_t softmax_t(scale q k_t) v_t,  k_t = code * page scale.
// A block takes one (sequence, query head); each warp walks every fourth token
// with a running maximum and sum, and the warps' results are joined at the end.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "decoder.h"

namespace bsp {
namespace {

__device__ __forceinline__ float code_value(uint32_t c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(c), __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

template <int kD>
__global__ void __launch_bounds__(128) decode_kernel(const DecodeParams p) {
  constexpr int kPer = kD / 32;
  const int seq = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = p.cache.kv_heads, kh = head / (p.heads / hk), page = p.cache.page;
  int64_t len = __ldg(p.lens + seq);
  if (len < 0 || len > p.table_width * page) {
    if (threadIdx.x == 0) atomicOr(p.status, ST_BAD_INDEX);
    len = 0;
  }
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q.p) + seq * p.q.token + head * p.q.head;
  float qr[kPer], acc[kPer], m = -INFINITY, l = 0.f;
  for (int i = 0; i < kPer; ++i) qr[i] = __bfloat162float(q[lane * kPer + i]), acc[i] = 0.f;
  for (int64_t t = warp; t < len; t += 4) {
    const int32_t id = __ldg(p.page_table + seq * p.table_stride + t / page);
    if (id < 0 || id >= p.cache.n_pages) {
      if (lane == 0) atomicOr(p.status, ST_BAD_INDEX);
      continue;
    }
    const int64_t at = id * p.cache.page_stride + kh * p.cache.head_stride + (t % page) * kD + lane * kPer;
    const float ks = p.cache.k_scale[static_cast<int64_t>(id) * hk + kh];
    const float vs = p.cache.v_scale[static_cast<int64_t>(id) * hk + kh];
    float s = 0.f;
    for (int i = 0; i < kPer; ++i) s += qr[i] * code_value(static_cast<const uint8_t*>(p.cache.k)[at + i]);
    for (int k = 16; k; k >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, k);
    s *= ks * p.scale;
    const float mn = fmaxf(m, s), c = m == mn ? 1.f : expf(m - mn), w = expf(s - mn);
    l = l * c + w;
    for (int i = 0; i < kPer; ++i)
      acc[i] = acc[i] * c + w * vs * code_value(static_cast<const uint8_t*>(p.cache.v)[at + i]);
    m = mn;
  }
  __shared__ float sm[4], sl[4], so[4][kD];
  for (int i = 0; i < kPer; ++i) so[warp][lane * kPer + i] = acc[i];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  __syncthreads();
  const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float L = 0.f, w[4];
  for (int k = 0; k < 4; ++k) {
    w[k] = sl[k] == 0.f ? 0.f : expf(sm[k] - M);
    L += w[k] * sl[k];
  }
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.o.p) + seq * p.o.token + head * p.o.head;
  if (threadIdx.x < kD) {
    float v = 0.f;
    for (int k = 0; k < 4; ++k) v += w[k] * so[k][threadIdx.x];
    o[threadIdx.x] = __float2bfloat16(L == 0.f ? 0.f : v / L);
  }
  if (threadIdx.x == 0 && p.lse) p.lse[static_cast<int64_t>(seq) * p.heads + head] = M + logf(L);
}

}  // namespace

bsp_status launch_decode(const bsp_decode_plan* plan, const DecodeParams& p, cudaStream_t stream) {
  const dim3 grid(p.n_seqs, p.heads);
  if (plan->d == 64) decode_kernel<64><<<grid, 128, 0, stream>>>(p);
  else decode_kernel<128><<<grid, 128, 0, stream>>>(p);
  return cuda_check(cudaGetLastError(), "decode attention launch");
}

}  // namespace bsp
