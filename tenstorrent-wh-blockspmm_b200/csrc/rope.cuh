// Rotation of two 16-byte vectors of a head, the unit of rope.cu and append.cu.
#pragma once
#include <cuda_bf16.h>

#include "decoder.h"

namespace bsp {
namespace dev {

// Values of a 16-byte vector.
template <typename T> struct Vec;
template <> struct Vec<uint16_t> { static constexpr int kN = 8; };
template <> struct Vec<float> { static constexpr int kN = 4; };

__device__ __forceinline__ void unpack8(const uint4& w, float (&v)[8]) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(r[i] << 16);
    v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void load_vec(const uint16_t* p, float (&v)[8]) {
  unpack8(*reinterpret_cast<const uint4*>(p), v);
}
__device__ __forceinline__ void load_vec(const float* p, float (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
}
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store_vec(uint16_t* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]),
                                            bf16_pair(v[6], v[7]));
}
__device__ __forceinline__ void store_vec(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// Unit u of a head of d values, the first rot of them rotated: vector u of the
// first half of the rotated values and vector u of their second half (then the
// same of the values behind them, which are not rotated).  Neighbouring
// threads take neighbouring vectors, so accesses are whole sectors, and both
// layouts find the two values of a pair in one thread: half in the two
// vectors, interleaved in one.
template <int kN>
struct RopeUnit {
  int lo, hi;
  bool turns;
  __device__ __forceinline__ RopeUnit(int u, int rot, int d) {
    turns = 2 * kN * u < rot;
    const int first = turns ? 0 : rot;
    lo = first + kN * (u - first / (2 * kN));
    hi = lo + (turns ? rot : d - rot) / 2;
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
template <int kN>
__device__ __forceinline__ void turn_unit(float (&lo)[kN], float (&hi)[kN], const float2 (&cs)[kN], bool interleaved,
                                          float sign) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      turn(lo[2 * i], lo[2 * i + 1], cs[i], sign);
      turn(hi[2 * i], hi[2 * i + 1], cs[kN / 2 + i], sign);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) turn(lo[i], hi[i], cs[i], sign);
  }
}
// A load that stays where it is written: the compiler would keep the values of
// two passes over the same positions in registers between them.
__device__ __forceinline__ float4 load_once(const float2* p) {
  float4 v;
  asm volatile("ld.global.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}
// (cos, sin) of unit u's pairs from a position's row of the table.
template <int kN>
__device__ __forceinline__ void load_turns(const float2* row, int u, int rot, bool interleaved, float2 (&cs)[kN]) {
  // interleaved: pairs kN/2 u ... of the first half, then of the second
  const float2* a = row + (interleaved ? kN / 2 * u : kN * u);
  const float2* b = interleaved ? a + rot / 4 : a + kN / 2;
#pragma unroll
  for (int i = 0; i < kN / 4; ++i) {
    const float4 w = load_once(a + 2 * i), x = load_once(b + 2 * i);
    cs[2 * i] = make_float2(w.x, w.y);
    cs[2 * i + 1] = make_float2(w.z, w.w);
    cs[kN / 2 + 2 * i] = make_float2(x.x, x.y);
    cs[kN / 2 + 2 * i + 1] = make_float2(x.z, x.w);
  }
}

}  // namespace dev
}  // namespace bsp
