// Attention over whole prompts, packed sequences of different lengths:
//   O_i = sum_j softmax_j(scale q_i k_j) v_j,  j <= i + (kv_len - q_len).
// A warp takes one (query, head) and walks its keys with a running maximum and
// sum.
#include <cuda_bf16.h>

#include "decoder.h"

namespace bsp {
namespace {

template <int kD>
__global__ void __launch_bounds__(128) prompt_kernel(const PromptParams p) {
  constexpr int kPer = kD / 32;
  const int token = blockIdx.x * 4 + (threadIdx.x >> 5), head = blockIdx.y, lane = threadIdx.x & 31;
  if (token >= p.tokens) return;
  int s = 0;
  while (s + 1 < p.n_seqs && p.seqs[s + 1].q0 <= token) ++s;
  const PromptSeq sq = p.seqs[s];
  const int kh = head / (p.heads / p.kv_heads);
  const int n = p.causal ? min(sq.kv_len, max(0, token - sq.q0 + sq.kv_len - sq.q_len + 1)) : sq.kv_len;
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q.p) + token * p.q.token + head * p.q.head;
  const __nv_bfloat16* kp = static_cast<const __nv_bfloat16*>(p.k.p) + sq.kv0 * p.k.token + kh * p.k.head;
  const __nv_bfloat16* vp = static_cast<const __nv_bfloat16*>(p.v.p) + sq.kv0 * p.v.token + kh * p.v.head;
  float qr[kPer], acc[kPer], m = -INFINITY, l = 0.f;
  for (int i = 0; i < kPer; ++i) qr[i] = __bfloat162float(q[lane * kPer + i]), acc[i] = 0.f;
  for (int j = 0; j < n; ++j) {
    float x = 0.f;
    for (int i = 0; i < kPer; ++i) x += qr[i] * __bfloat162float(kp[j * p.k.token + lane * kPer + i]);
    for (int k = 16; k; k >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, k);
    x *= p.scale;
    const float mn = fmaxf(m, x), c = m == mn ? 1.f : expf(m - mn), w = expf(x - mn);
    l = l * c + w;
    for (int i = 0; i < kPer; ++i) acc[i] = acc[i] * c + w * __bfloat162float(vp[j * p.v.token + lane * kPer + i]);
    m = mn;
  }
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.o.p) + token * p.o.token + head * p.o.head;
  for (int i = 0; i < kPer; ++i) o[lane * kPer + i] = __float2bfloat16(n == 0 ? 0.f : acc[i] / l);
  if (lane == 0 && p.lse) p.lse[static_cast<int64_t>(token) * p.heads + head] = m + logf(l);
}

}  // namespace

bsp_status launch_prompt(const bsp_prompt_plan* plan, const PromptParams& p, cudaStream_t stream) {
  const dim3 grid((p.tokens + 3) / 4, p.heads);
  if (plan->d == 64) prompt_kernel<64><<<grid, 128, 0, stream>>>(p);
  else prompt_kernel<128><<<grid, 128, 0, stream>>>(p);
  return cuda_check(cudaGetLastError(), "prompt attention launch");
}

}  // namespace bsp
