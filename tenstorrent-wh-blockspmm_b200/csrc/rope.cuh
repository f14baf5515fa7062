// Rotation of 16 values of a head, the unit of rope.cu and append.cu.
#pragma once
#include <cuda_bf16.h>

#include "decoder.h"

namespace bsp {
namespace dev {

__device__ __forceinline__ void load8(const uint16_t* p, float (&v)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(r[i] << 16);
    v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]),
                                            bf16_pair(v[6], v[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// Unit u of a head (d / 16 units): its two groups of 8 values.  Units below
// rot / 16 hold the pairs 8 u .. 8 u + 7, the others are not rotated.
struct RopeUnit {
  int lo, hi;
  bool turns;
  __device__ __forceinline__ RopeUnit(int u, int rot, bool interleaved) {
    turns = 16 * u < rot;
    lo = turns && !interleaved ? 8 * u : 16 * u;
    hi = turns && !interleaved ? 8 * u + rot / 2 : 16 * u + 8;
  }
};

// y_a = x_a c - x_b s, y_b = x_b c + x_a s.  The products are rounded before
// the sum (no fused multiply-add): the result then has the same bits wherever
// it is computed, also where it is rounded to 8 bits afterwards.
__device__ __forceinline__ void turn(float& a, float& b, float2 cs, float sign) {
  const float s = cs.y * sign;
  const float ya = __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, s));
  const float yb = __fadd_rn(__fmul_rn(b, cs.x), __fmul_rn(a, s));
  a = ya;
  b = yb;
}
__device__ __forceinline__ void turn16(float (&lo)[8], float (&hi)[8], const float2 (&cs)[8], bool interleaved,
                                       float sign) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      turn(lo[2 * i], lo[2 * i + 1], cs[i], sign);
      turn(hi[2 * i], hi[2 * i + 1], cs[4 + i], sign);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn(lo[i], hi[i], cs[i], sign);
  }
}
__device__ __forceinline__ void load_turns(const float2* row, int u, float2 (&cs)[8]) {
  const float4* t = reinterpret_cast<const float4*>(row + 8 * u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 w = __ldg(t + i);
    cs[2 * i] = make_float2(w.x, w.y);
    cs[2 * i + 1] = make_float2(w.z, w.w);
  }
}

}  // namespace dev
}  // namespace bsp
