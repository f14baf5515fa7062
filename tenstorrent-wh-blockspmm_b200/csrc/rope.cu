// Rotary positions: the table of (cos, sin) and the rotation of queries, keys
// or their gradients.
#include <math.h>

#include "rope.cuh"

namespace bsp {
using namespace dev;

namespace {

// The angle position * f_i is formed in 64 bits and goes to sincos() in 64
// bits: at position 10^6 a 32-bit product alone would be 0.03 rad off.
__global__ void rope_table_kernel(float2* table, int64_t n_pos, int half, double base, bsp_rope_scaling sc) {
  const int64_t n = n_pos * half;
  for (int64_t k = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; k < n;
       k += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t pos = k / half;
    const int i = static_cast<int>(k - pos * half);
    double f = pow(base, -static_cast<double>(i) / half);
    if (sc.kind == BSP_ROPE_LINEAR) {
      f /= sc.factor;
    } else if (sc.kind == BSP_ROPE_BASE) {
      f = pow(base * pow(sc.factor, half / (half - 1.0)), -static_cast<double>(i) / half);
    } else if (sc.kind == BSP_ROPE_PARTS) {
      const double turns = sc.context * f / (2.0 * M_PI);
      const double keep = fmin(fmax((turns - sc.slow) / (sc.fast - sc.slow), 0.0), 1.0);
      f = f * keep + f / sc.factor * (1.0 - keep);
    }
    double s, c;
    sincos(static_cast<double>(pos) * f, &s, &c);
    table[k] = make_float2(static_cast<float>(c * sc.magnitude), static_cast<float>(s * sc.magnitude));
  }
}

// A thread turns unit u of one head of one token.
template <typename T>
__global__ void __launch_bounds__(256) rope_kernel(const RopeParams p, int units, int items_per_block) {
  const int u = threadIdx.x % units, y = threadIdx.x / units;
  const uint32_t item = blockIdx.x * static_cast<uint32_t>(items_per_block) + y;
  const uint32_t token = item / p.heads, head = item - token * p.heads;
  if (y >= items_per_block || token >= p.tokens) return;
  const RopeUnit un(u, p.rot, p.interleaved);
  const T* x = static_cast<const T*>(p.x.p) + token * p.x.token + head * p.x.head;
  T* out = static_cast<T*>(p.y.p) + token * p.y.token + head * p.y.head;
  const int32_t pos = __ldg(p.positions + token);
  if (pos < 0 || pos >= p.n_pos) {
    if (u == 0) atomicOr(p.status, ST_BAD_INDEX);
    return;
  }
  float lo[8], hi[8];
  load8(x + un.lo, lo);
  load8(x + un.hi, hi);
  if (un.turns) {
    float2 cs[8];
    load_turns(p.table + static_cast<int64_t>(pos) * (p.rot / 2), u, cs);
    turn16(lo, hi, cs, p.interleaved, p.sign);
  }
  store8(out + un.lo, lo);
  store8(out + un.hi, hi);
}

}  // namespace

bsp_status launch_rope_table(bsp_device* dev, int64_t n_pos, int32_t rot, double base, const bsp_rope_scaling& sc,
                             float* table, cudaStream_t stream) {
  const int64_t n = n_pos * (rot / 2);
  const int64_t blocks = std::min<int64_t>((n + 255) / 256, 8 * static_cast<int64_t>(dev->sm_count));
  rope_table_kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(reinterpret_cast<float2*>(table), n_pos,
                                                                      rot / 2, base, sc);
  return cuda_check(cudaGetLastError(), "rotary table launch");
}

bsp_status launch_rope(const RopeParams& p, bsp_dtype type, cudaStream_t stream) {
  const int units = p.d / 16;
  const int per_block = 256 / units;
  const int64_t items = p.tokens * p.heads;
  const unsigned blocks = static_cast<unsigned>((items + per_block - 1) / per_block);
  if (type == BSP_BF16)
    rope_kernel<uint16_t><<<blocks, 256, 0, stream>>>(p, units, per_block);
  else
    rope_kernel<float><<<blocks, 256, 0, stream>>>(p, units, per_block);
  return cuda_check(cudaGetLastError(), "rotary kernel launch");
}

}  // namespace bsp
