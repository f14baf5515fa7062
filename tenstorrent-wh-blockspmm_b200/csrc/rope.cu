// Rotary positions: the table of (cos, sin) and the rotation of queries, keys
// or their gradients.
#include <math.h>

#include "bsp_ptx.cuh"
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

// A thread turns unit u of kHeads heads of one token: (cos, sin) are loaded
// once for them, and 2 kHeads loads are in flight.  Memory-bound: 8191 tokens of
// 32 heads of 128 in f32 take 41.7 us, 6490 GB/s, a plain copy's rate.  16 tokens
// take 1.8 us on the device, their launch more than that.
template <typename T, int kHeads>
__global__ void __launch_bounds__(256) rope_kernel(const RopeParams p) {
  const int units = p.units, items_per_block = p.items_per_block, groups = p.groups;
  stream_release();
  stream_wait();
  constexpr int kN = Vec<T>::kN;
  const int u = threadIdx.x % units, y = threadIdx.x / units;
  const uint32_t item = blockIdx.x * static_cast<uint32_t>(items_per_block) + y;
  const uint32_t token = item / groups, head0 = (item - token * groups) * kHeads;
  if (y >= items_per_block || token >= p.tokens) return;
  const RopeUnit<kN> un(u, p.rot, p.d);
  const T* x = static_cast<const T*>(p.x.p) + token * p.x.token + head0 * p.x.head;
  T* out = static_cast<T*>(p.y.p) + token * p.y.token + head0 * p.y.head;
  const int32_t pos = p.positions[token];
  float lo[kHeads][kN], hi[kHeads][kN];
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
    if (head0 + h < p.heads) {
      load_vec(x + h * p.x.head + un.lo, lo[h]);
      load_vec(x + h * p.x.head + un.hi, hi[h]);
    }
  if (pos < 0 || pos >= p.n_pos) {
    if (u == 0) atomicOr(p.status, ST_BAD_INDEX);
    return;
  }
  float2 cs[kN];
  if (un.turns) load_turns<kN>(p.table + static_cast<int64_t>(pos) * (p.rot / 2), u, p.rot, p.interleaved, cs);
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
    if (head0 + h < p.heads) {
      if (un.turns) turn_unit<kN>(lo[h], hi[h], cs, p.interleaved, p.sign);
      store_vec(out + h * p.y.head + un.lo, lo[h]);
      store_vec(out + h * p.y.head + un.hi, hi[h]);
    }
}

template <typename T, int kHeads>
bsp_status run_rope(RopeParams& p, cudaStream_t stream) {
  p.units = p.d / (2 * Vec<T>::kN);
  p.items_per_block = 256 / p.units;
  p.groups = (p.heads + kHeads - 1) / kHeads;
  const int64_t items = p.tokens * p.groups;
  const unsigned blocks = static_cast<unsigned>((items + p.items_per_block - 1) / p.items_per_block);
  return launch_overlapped(rope_kernel<T, kHeads>, dim3(blocks), 256, 0, stream, p, "rotary kernel launch");
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

bsp_status launch_rope(RopeParams& p, bsp_dtype type, int sm_count, cudaStream_t stream) {
  // One head a thread for up to about 512 threads an SM, two above: 16 tokens of
  // 32 heads of 128 in bf16 take 1.8 and 2.2 us, 300 tokens 3.0 either way, 1000
  // 4.5 and 4.2, 3000 10.1 and 8.7 (four heads: 3.1, 3.5, 3.8 and 9.1).  In f32
  // four: 2000 tokens 6.9 us (two 7.1), 8191 half rotated 41.7 (two 42.4).
  const bool few = p.tokens * p.heads * (p.d / 16) < static_cast<int64_t>(sm_count) * 512;
  if (type == BSP_BF16) return few ? run_rope<uint16_t, 1>(p, stream) : run_rope<uint16_t, 2>(p, stream);
  return few ? run_rope<float, 1>(p, stream) : run_rope<float, 4>(p, stream);
}

}  // namespace bsp
