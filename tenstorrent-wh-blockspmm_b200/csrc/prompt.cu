// Attention over whole prompts on the tcgen05 tensor cores, packed sequences
// of different lengths, several query heads to a key/value head:
//   O_i = sum_j softmax_j(scale q_i k_j) v_j,  j <= i + (kv_len - q_len).
//
// Rows.  A tile is 128 rows = 128 / P queries x P query heads of one key/value
// head (P: the largest power of two up to 32 that divides heads / kv_heads), so
// that a short sequence still fills a tile and a causal tile wastes little on its
// diagonal.  One TMA box {64 values, P heads, 128 / P queries} brings it in
// that order.  A unit is one or two such tiles of consecutive queries; both
// read the same keys.
//
// Steps.  128 keys a step.  Per tile and step
//   S = Q K^T            128 x 128 x d    fp32 in TMEM
//   P = exp2(S c - m)    one thread a row; c = scale log2 e; m follows the
//                        running maximum when it is 2^8 behind, and only then
//                        O and the row sum l are rescaled; P goes back to TMEM
//                        as bf16 pairs, over S
//   O += P V             128 x d x 128, A = P read from TMEM
// and at the end O / l, m ln 2 + ln l.  With two tiles the tensor cores work on
// one while the softmax of the other runs: the MMA warp issues
//   S_a(0) S_b(0) | O_a(0) S_a(1) | O_b(0) S_b(1) | O_a(1) S_a(2) | ...
// S_t(j + 1) is issued behind O_t(j), so P(j) has been read when S(j + 1)
// overwrites it, and a thread that sees S_t(j) complete knows O_t(j - 1) to be
// complete and may rescale it.
//
// TMEM (512 columns): S_a 0, S_b 128 (P in their first 64), O_a 256, O_b 384.
// Shared memory: Q of both tiles, then a ring of K and V slots in the order
// K0 V0 K1 V1 ...
//
// Warps (320 threads, one CTA per SM): 0-3 softmax of tile a, 4-7 of tile b
// (TMEM lane quarter = warp & 3), 8 MMA, 9 TMA.  Every wait is bounded.
//
// What bounds it: the tensor cores with their hand-overs, and power.  At 16384
// tokens, 8 heads of 128, one step of both tiles takes 3000 cycles, of which the
// products need 2048 (64 for each MMA of 128 x 128 x 16); without any softmax
// work the same waits and products take 83 % of the time, without its arithmetic
// 87 %.  The MMAs are 62 % of the cycles, the exponential unit 47 %.  The SMs run
// at 1.62 GHz in a burst and at 1.35 GHz once the power limit holds: 442 us (1240
// TFLOP/s) and 512 us for 0.55 TFLOP.  Heads of 64 do half the products on the
// same softmax and hand-overs: 16 heads, 6025 tokens 57 us (500 TFLOP/s).
//
// What shortens a step: the softmax does not wait for its own maximum (weights
// are formed with the maximum of the steps before, the step's own is found
// beside them and only moves m for the next step, or at once if it is 2^20
// above); a quarter of the exponentials is computed in the FMA pipe (exp2_pair);
// scaling and sums are packed two to an instruction; P is handed over in two
// parts of 64 keys, so that O += P V begins while the second part is worked on.
// What did not: steps of 64 keys with two S buffers (545 us against 442), two
// threads a row (471), an MMA warp for each tile (566), P of d = 64 in columns of
// its own so that S comes a step ahead (416 against 392), the next unit's first
// scores behind the unit's last products (457).
//
// Few rows of many keys: the planner cuts a block's keys into parts.  A part
// leaves O unnormalised in fp32 with m and l; prompt_join puts them together.
// (Joined by the part that ends last, inside this kernel, 16 tokens behind 32768
// keys took 61 us; with a kernel of its own 39 us.)
#include <cuda_bf16.h>

#include "bsp_ptx.cuh"
#include "decoder.h"

namespace bsp {
using namespace dev;

namespace {

constexpr int kPrThreads = 320;
constexpr int kPrMmaWarp = 8, kPrTmaWarp = 9;
constexpr uint32_t kPrAtom = 128 * 128;  // 128 rows x 128 bytes (64 values)
constexpr float kPrRescale = 8.f;        // log2 of the growth that forces a rescale
constexpr float kPrLate = 20.f;          // and of the one that cannot wait for the next step
constexpr int kPrMaxSlots = 8;
constexpr int kPrByFma = 2;                // of each 8 pairs of exponentials, those in the FMA pipe

__host__ __device__ constexpr uint32_t pr_tile(int d) { return 128u * 2u * static_cast<uint32_t>(d); }
__host__ __device__ constexpr int pr_slots(int d) { return d == 128 ? 5 : 8; }

struct PrHeader {
  uint64_t q_full, q_empty;
  uint64_t kv_full[kPrMaxSlots], kv_empty[kPrMaxSlots];
  uint64_t s_full[2], p_full[2][2], h_full[2], o_full[2], o_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
};
constexpr uint32_t kPrHeader = 1024;
static_assert(sizeof(PrHeader) <= kPrHeader, "header must fit its slot");

__device__ __forceinline__ uint32_t baddr(const uint64_t* b) { return smem_u32(b); }

__device__ __forceinline__ bool wait_all(const uint64_t* bar, uint32_t parity, const WaitCtl& ctl, uint32_t what) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(baddr(bar), parity, ctl, what));
}

// A wait for copies or MMAs in flight that does not give up when another role
// did: shared memory and TMEM may not be left while they are written.
__device__ __noinline__ bool drain_wait(uint32_t bar, uint32_t parity, const WaitCtl& ctl) {
  int zero = 0;
  WaitCtl c2{&zero, ctl.status, ctl.timeout_ns};
  return mbar_wait_bounded(bar, parity, c2, ST_TIMEOUT_DRAIN);
}

__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if one is
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two fp32 values in a register pair: one instruction for both.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^x of two values without the exponential unit: x = n + f with n the nearest
// whole number (adding 1.5 * 2^23 leaves it in the low bits), 2^f by a
// polynomial of degree 4 on [-1/2, 1/2] with p(0) = 1, fitted for the least
// relative error (2.9e-6), and n added to the exponent.  x <= 127; from -127
// down (a masked score) the result is 0: p(0) = 1, and its exponent less 127 is an
// empty field.  (So a hidden key weighs nothing, whatever its value.  Between -127
// and -126 the result is somewhere below 2^-126.)
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  const uint64_t magic = pair_of(12582912.f, 12582912.f), back = pair_of(-12582912.f, -12582912.f);
  float a, b;
  unpair(x, a, b);
  x = pair_of(fmaxf(a, -127.f), fmaxf(b, -127.f));
  const uint64_t t = add2(x, magic);
  const uint64_t f = fma2(add2(t, back), pair_of(-1.f, -1.f), x);
  uint64_t p = fma2(f, pair_of(0.009582852944731712f, 0.009582852944731712f),
                    pair_of(0.055906426161527634f, 0.055906426161527634f));
  p = fma2(p, f, pair_of(0.24024099111557007f, 0.24024099111557007f));
  p = fma2(p, f, pair_of(0.6931241750717163f, 0.6931241750717163f));
  p = fma2(p, f, pair_of(1.f, 1.f));
  float ta, tb;
  unpair(t, ta, tb);
  unpair(p, a, b);
  return pair_of(__uint_as_float(__float_as_uint(a) + (__float_as_uint(ta) << 23)),
                 __uint_as_float(__float_as_uint(b) + (__float_as_uint(tb) << 23)));
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int kD>
__device__ __forceinline__ void pr_tma(const PromptParams& p, PrHeader* hdr, uint32_t q_smem, uint32_t ring, int u0,
                                      int u1, const WaitCtl& ctl, int lane) {
  constexpr int kHalves = kD / 64, kSlots = pr_slots(kD);
  constexpr uint32_t kTile = pr_tile(kD);
  int64_t slot_n = 0;
  int units = 0;
  uint32_t armed = 0, armed_parity = 0;
  bool q_armed = false, ok = true;
  auto load = [&](const CUtensorMap* tm, int kvh, int token) -> bool {
    const int sl = static_cast<int>(slot_n % kSlots);
    const uint32_t ph = static_cast<uint32_t>((slot_n / kSlots) & 1);
    ++slot_n;
    if (!wait_all(&hdr->kv_empty[sl], ph ^ 1u, ctl, ST_TIMEOUT_PRODUCER)) return false;
    const uint32_t bar = baddr(&hdr->kv_full[sl]);
    mbar_arrive_expect_tx_pred(bar, kTile, lane == 0);
    tma_load_3d_pred(ring + sl * kTile + lane * kPrAtom, tm, 64 * lane, kvh, token, bar, lane < kHalves);
    armed |= 1u << sl;
    armed_parity = (armed_parity & ~(1u << sl)) | (ph << sl);
    return true;
  };
#pragma unroll 1
  for (int u = u0; u < u1 && ok; ++u) {
    const PromptUnit un = p.units[u];
    const int n = max(un.n[0], un.n[1]);
    if (n == 0) continue;
    ok = wait_all(&hdr->q_empty, (units & 1) ^ 1u, ctl, ST_TIMEOUT_PRODUCER);
    if (!ok) break;
    ++units;
    q_armed = true;
    const int tiles = un.n[1] > 0 ? 2 : 1;
    mbar_arrive_expect_tx_pred(baddr(&hdr->q_full), tiles * kTile, lane == 0);
    tma_load_3d_pred(q_smem + lane * kPrAtom, &p.tm_q, 64 * (lane % kHalves), un.head0,
                     un.q0 + (lane / kHalves) * p.tile_tokens, baddr(&hdr->q_full), lane < tiles * kHalves);
    const int kvh = un.head0 / p.group;
#pragma unroll 1
    for (int j = 0; j < n && ok; ++j) {
      ok = load(&p.tm_k, kvh, un.kv0 + 128 * j);
      if (ok) ok = load(&p.tm_v, kvh, un.kv0 + 128 * j);
    }
  }
  if (lane == 0) {
    if (q_armed) drain_wait(baddr(&hdr->q_full), (units - 1) & 1, ctl);
    for (int s = 0; s < kSlots; ++s)
      if (armed & (1u << s)) drain_wait(baddr(&hdr->kv_full[s]), (armed_parity >> s) & 1u, ctl);
  }
  __syncwarp();
}

// The warp waits as one; each batch of MMAs and their commits sits in one
// branch of a single elected thread.  (An MMA that every lane passes under a
// predicate costs about 54 cycles of issue; in such a branch 33 or less, and
// the warp shares its scheduler with four softmax warps.)
template <int kD>
__device__ __forceinline__ void pr_mma(const PromptParams& p, PrHeader* hdr, uint32_t q_smem, uint32_t ring,
                                      uint32_t tmem, int u0, int u1, const WaitCtl& ctl, int lane) {
  constexpr int kSlots = pr_slots(kD);
  constexpr uint32_t kTile = pr_tile(kD), kAtom16 = kPrAtom >> 4;
  const uint32_t idesc_s = idesc_bf16_f32(128, 128, 0, 0), idesc_o = idesc_bf16_f32(128, kD, 0, 1);
  const uint64_t qd = smem_desc(q_smem, 16u, 1024u, 2u);
  const uint64_t kd = smem_desc(ring, 16u, 1024u, 2u);
  const uint64_t vd = smem_desc(ring, kPrAtom, 1024u, 2u);  // MN-major: LBO = next 64 columns of d
  int slot = 0;          // ring slot of the next K or V
  uint32_t phase = 0;    // and its parity
  uint32_t units = 0, steps[2] = {0, 0}, outs[2] = {0, 0};
  bool ok = true;
  auto full = [&]() { return wait_all(&hdr->kv_full[slot], phase, ctl, ST_TIMEOUT_MMA); };
  auto next_slot = [&]() {
    if (++slot == kSlots) slot = 0, phase ^= 1u;
  };
  auto scores = [&](int t, int at) {  // in an elected branch
    const uint64_t a = qd + t * (kTile >> 4), b = kd + at * (kTile >> 4);
#pragma unroll
    for (int i = 0; i < kD / 16; ++i)
      mma_bf16(tmem + 128u * t, a + (i >> 2) * kAtom16 + (i & 3) * 2u, b + (i >> 2) * kAtom16 + (i & 3) * 2u, idesc_s,
               i > 0);
    mma_commit(baddr(&hdr->s_full[t]));
  };
#pragma unroll 1
  for (int u = u0; u < u1 && ok; ++u) {
    const PromptUnit un = p.units[u];
    const int n = max(un.n[0], un.n[1]);
    if (n == 0) continue;
    ok = wait_all(&hdr->q_full, units & 1, ctl, ST_TIMEOUT_MMA) && full();
    if (!ok) break;
    ++units;
    tc_fence_after();
    if (elect_one()) {
      for (int t = 0; t < 2; ++t)
        if (un.n[t] > 0) scores(t, slot);
      mma_commit(baddr(&hdr->kv_empty[slot]));
      if (n == 1) mma_commit(baddr(&hdr->q_empty));
    }
    __syncwarp();
    next_slot();
#pragma unroll 1
    for (int j = 0; j < n && ok; ++j) {
      ok = full();
      const int v_slot = slot;
      next_slot();
      const int k_slot = slot;
      if (ok && j + 1 < n) {
        ok = full();
        next_slot();
      }
      const int last = j < un.n[1] ? 1 : 0;           // last tile that uses V of this step
      const int last_next = j + 1 < un.n[1] ? 1 : 0;  // and K of the next
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!ok || j >= un.n[t]) continue;
        if (j == 0) {
          ok = wait_all(&hdr->o_empty[t], (outs[t] & 1) ^ 1u, ctl, ST_TIMEOUT_MMA);
          ++outs[t];
        }
        const uint64_t b = vd + v_slot * (kTile >> 4);
        const bool more = j + 1 < un.n[t];
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          ok = ok && wait_all(&hdr->p_full[t][part], steps[t] & 1, ctl, ST_TIMEOUT_MMA);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int i = 4 * part; i < 4 * part + 4; ++i)
              mma_bf16_ts(tmem + 256u + 128u * t, tmem + 128u * t + 8u * i, b + i * 128u, idesc_o, i > 0 || j > 0);
            if (part == 0) {
              mma_commit(baddr(&hdr->h_full[t]));
            } else {
              if (!more) mma_commit(baddr(&hdr->o_full[t]));
              if (t == last) mma_commit(baddr(&hdr->kv_empty[v_slot]));
              if (more) {
                scores(t, k_slot);
                if (t == last_next) {
                  mma_commit(baddr(&hdr->kv_empty[k_slot]));
                  if (j + 2 == n) mma_commit(baddr(&hdr->q_empty));
                }
              }
            }
          }
          __syncwarp();
        }
        ++steps[t];
      }
    }
  }
  if (elect_one()) {
    mma_commit(baddr(&hdr->drain));
    drain_wait(baddr(&hdr->drain), 0, ctl);
  }
  __syncwarp();
}

// Store 32 bytes of a row; keep: all bits, or none (zeros).
__device__ __forceinline__ void store32(uint16_t* dst, const uint32_t (&o)[32], int at, float f, uint32_t keep) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    w[i] = pack2(__uint_as_float(o[at + 2 * i]) * f, __uint_as_float(o[at + 2 * i + 1]) * f) & keep;
  *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(dst + 8) = make_uint4(w[4], w[5], w[6], w[7]);
}

// Largest of 64 scores, NaN if one is.
__device__ __forceinline__ float row_max(const uint32_t (&a)[32], const uint32_t (&b)[32]) {
  float x[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t* y = (k < 2 ? a : b) + 16 * (k & 1);
    x[k] = max3(__uint_as_float(y[0]), __uint_as_float(y[1]), __uint_as_float(y[2]));
#pragma unroll
    for (int i = 3; i < 15; i += 2) x[k] = max3(x[k], __uint_as_float(y[i]), __uint_as_float(y[i + 1]));
    x[k] = max3(x[k], __uint_as_float(y[15]), __uint_as_float(y[15]));
  }
  return max3(max3(x[0], x[1], x[2]), x[3], x[3]);
}

// w = exp2(s c - m) of 64 scores as bf16 pairs; their sum.
__device__ __forceinline__ float pr_weights(uint32_t (&a)[32], uint32_t (&b)[32], float c, float m, uint32_t (&w)[32]) {
  float mm = m == -INFINITY ? 0.f : m;
  // The exponent is one fused step.  For |m| above 2^24 the rounding of m itself
  // would show in it: there the product is rounded like m first.
  if (__any_sync(0xffffffffu, fabsf(mm) > 16777216.f)) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      a[i] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(a[i]), c), mm));
      b[i] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(b[i]), c), mm));
    }
    c = 1.f;
    mm = 0.f;
  }
  const uint64_t c2 = pair_of(c, c), m2 = pair_of(-mm, -mm);
  uint64_t l0 = 0, l1 = 0;  // (0, 0)
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint32_t* y = i < 16 ? a + 2 * i : b + 2 * (i - 16);
    const uint64_t e = fma2(pair_of(__uint_as_float(y[0]), __uint_as_float(y[1])), c2, m2);
    float p, q;
    if (i % 8 < kPrByFma) {
      unpair(exp2_pair(e), p, q);
    } else {
      unpair(e, p, q);
      p = ex2(p);
      q = ex2(q);
    }
    if (i & 1) l1 = add2(l1, pair_of(p, q));
    else l0 = add2(l0, pair_of(p, q));
    w[i] = pack2(p, q);
  }
  float p, q;
  unpair(add2(l0, l1), p, q);
  return p + q;
}

// What a row's sums are multiplied with: 1 / l; 0 where the row saw no key (l is
// 0 then).  A NaN or infinite score makes m NaN or infinite, and the row NaN.
__device__ __forceinline__ float share_of(float m, float& l) {
  if (!(m < INFINITY)) l = __uint_as_float(0x7FC00000u);
  return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // a NaN sum stays one
}
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
}

template <int kD>
__device__ __forceinline__ void pr_softmax(const PromptParams& p, PrHeader* hdr, uint8_t* ring_ptr, uint32_t tmem,
                                          int u0, int u1, const WaitCtl& ctl, int warp, int lane) {
  const int t = warp >> 2, row = 32 * (warp & 3) + lane;
  const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
  const uint32_t t_s = lanes + 128u * t, t_o = lanes + 256u + 128u * t;
  const int dt = t * p.tile_tokens + row / p.packed, dh = row % p.packed;
  int64_t slot_n = 0;  // ring position of K0 of the unit
  uint32_t steps = 0, outs = 0;
  auto scale_o = [&](float alpha) {
#pragma unroll 1
    for (int c = 0; c < kD / 16; ++c) {
      uint32_t o[16];
      tmem_ld_32x32b_x16(t_o + 16u * c, o);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
      tmem_st_32x32b_x16(t_o + 16u * c, o);
    }
  };
  auto weights = [&](uint32_t (&a)[32], uint32_t (&b)[32], float m, uint32_t (&w)[32]) {
    return pr_weights(a, b, p.scale_log2, m, w);
  };
#pragma unroll 1
  for (int u = u0; u < u1; ++u) {
    const PromptUnit un = p.units[u];
    const int n = un.n[t];
    const int64_t token = static_cast<int64_t>(un.q0) + dt;
    const bool valid = token < un.q_end && (t == 0 || un.two);
    uint16_t* orow = static_cast<uint16_t*>(p.o.p) + token * p.o.token + (un.head0 + dh) * p.o.head;
    float* lrow = p.lse ? p.lse + token * p.heads + un.head0 + dh : nullptr;
    float* work = p.work + (static_cast<int64_t>(un.first) + 2 * un.part + t) * prompt_slot_floats(kD);
    if (n == 0) {
      slot_n += 2 * max(un.n[0], un.n[1]);
      if (valid && un.parts > 1) {
        work[128 * kD + row] = -INFINITY;
        work[128 * kD + 128 + row] = 0.f;
      } else if (valid) {
        for (int c = 0; c < kD / 8; ++c) reinterpret_cast<uint4*>(orow)[c] = make_uint4(0, 0, 0, 0);
        if (lrow) *lrow = -INFINITY;
      }
      continue;
    }
    const int sees = p.causal ? min(un.kv_len, un.sees + dt) : un.kv_len;  // keys this row attends to
    float m = -INFINITY, l = 0.f;  // reference of the exponents, sum of the weights
    float seen = -INFINITY;        // largest score so far; m follows when it is 2^8 behind
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      if (!wait_all(&hdr->s_full[t], steps & 1, ctl, ST_TIMEOUT_EPILOGUE)) return;
      ++steps;
      tc_fence_after();
      uint32_t v[2][32];
      tmem_ld_32x32b_x32(t_s, v[0]);
      tmem_ld_32x32b_x32(t_s + 32u, v[1]);
      // Rows of V behind the sequence's end belong to its neighbour; their weight
      // is 0, but 0 times an infinity or NaN there is not: clear them before P is
      // handed over.
      if (un.kv_len - 128 * j < 128) {
        const int64_t kv = slot_n + 2 * j + 1;
        if (!wait_all(&hdr->kv_full[kv % pr_slots(kD)], static_cast<uint32_t>((kv / pr_slots(kD)) & 1), ctl,
                      ST_TIMEOUT_EPILOGUE))
          return;
        uint8_t* vt = ring_ptr + (kv % pr_slots(kD)) * pr_tile(kD);
        for (int i = (un.kv_len - 128 * j) * 8 + row; i < 128 * 8; i += 128)
          for (int h = 0; h < kD / 64; ++h) *reinterpret_cast<uint4*>(vt + h * kPrAtom + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
      }
      // The maximum grew in the step before: O holds exactly the steps before
      // this one now.
      if (__any_sync(0xffffffffu, seen > m + kPrRescale)) {
        const float mn = seen > m + kPrRescale ? seen : m;
        if (j > 0) scale_o(m == -INFINITY ? 0.f : ex2(m - mn));
        l *= m == -INFINITY ? 0.f : ex2(m - mn);
        m = mn;
      }
      tmem_ld_wait_regs(v[0]);
      tmem_ld_wait_regs(v[1]);
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        if (part == 1) {
          tmem_ld_wait_regs(v[0]);
          tmem_ld_wait_regs(v[1]);
        }
        uint32_t(&a)[32] = v[0];
        uint32_t(&b)[32] = v[1];
        const int limit = sees - 128 * j - 64 * part;
        auto mask = [&]() {
          if (__any_sync(0xffffffffu, limit < 64)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (i >= limit) a[i] = 0xFF800000u;
              if (32 + i >= limit) b[i] = 0xFF800000u;
            }
          }
        };
        mask();
        if (part == 0 && j == 0) m = row_max(a, b) * p.scale_log2;
        // Weights with the maximum known so far; this part's own is found on the way.
        uint32_t w[32];
        const float mx = row_max(a, b) * p.scale_log2;
        float sum = weights(a, b, m, w);
        if (__any_sync(0xffffffffu, !(mx <= m + kPrLate) && m == m)) {
          // It is too far above: move to it now, from the scores in TMEM.
          const float mn = max3(m, mx, mx);
          const float alpha = m == -INFINITY ? 0.f : ex2(m - mn);
          if (part == 1) {  // O holds part 0 of this step too: wait for that product
            if (!wait_all(&hdr->h_full[t], (steps - 1) & 1, ctl, ST_TIMEOUT_EPILOGUE)) return;
            tc_fence_after();
          }
          if (part == 1 || j > 0) scale_o(alpha);
          l *= alpha;
          m = mn;
          tmem_ld_32x32b_x32(t_s + 64u * part, a);
          tmem_ld_32x32b_x32(t_s + 64u * part + 32u, b);
          tmem_ld_wait_regs(a);
          tmem_ld_wait_regs(b);
          mask();
          sum = weights(a, b, m, w);
        }
        seen = fmaxf(seen, mx);
        if (part == 0) {
          tmem_ld_32x32b_x32(t_s + 64u, v[0]);
          tmem_ld_32x32b_x32(t_s + 96u, v[1]);
        }
        tmem_st_32x32b_x32(t_s + 32u * part, w);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_pred(baddr(&hdr->p_full[t][part]), lane == 0);
        l += sum;
      }
    }
    slot_n += 2 * max(un.n[0], un.n[1]);
    if (!wait_all(&hdr->o_full[t], outs & 1, ctl, ST_TIMEOUT_EPILOGUE)) return;
    ++outs;
    tc_fence_after();
    const bool whole = un.parts == 1;
    const float inv = whole ? share_of(m, l) : 1.f;
    const uint32_t keep = l == 0.f ? 0u : ~0u;  // no key: O is 0 but for a NaN or infinity in V
#pragma unroll 1
    for (int c = 0; c < kD / 32; ++c) {
      uint32_t o[32];
      tmem_ld_32x32b_x32(t_o + 32u * c, o);
      tmem_ld_wait();
      if (valid && !whole) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          reinterpret_cast<uint4*>(work)[(8 * c + i) * 128 + row] =
              make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      } else if (valid) {
        store32(orow + 32 * c, o, 0, inv, keep);
        store32(orow + 32 * c + 16, o, 16, inv, keep);
      }
    }
    if (valid && !whole) {
      work[128 * kD + row] = m;
      work[128 * kD + 128 + row] = l;
    } else if (valid && lrow) {
      *lrow = lse_of(m, l);
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(baddr(&hdr->o_empty[t]));
  }
}

template <int kD>
__global__ void __launch_bounds__(kPrThreads, 1) prompt_tcgen05(const __grid_constant__ PromptParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  PrHeader* hdr = reinterpret_cast<PrHeader*>(gbase);
  const uint32_t q_smem = base + kPrHeader, ring = q_smem + 2u * pr_tile(kD);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int u0 = p.cta_begin[blockIdx.x], u1 = p.cta_begin[blockIdx.x + 1];
  if (threadIdx.x == 0) {
    mbar_init(baddr(&hdr->q_full), 1);
    mbar_init(baddr(&hdr->q_empty), 1);
    for (int s = 0; s < pr_slots(kD); ++s) {
      mbar_init(baddr(&hdr->kv_full[s]), 1);
      mbar_init(baddr(&hdr->kv_empty[s]), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(baddr(&hdr->s_full[t]), 1);
      mbar_init(baddr(&hdr->p_full[t][0]), 4);
      mbar_init(baddr(&hdr->p_full[t][1]), 4);
      mbar_init(baddr(&hdr->h_full[t]), 1);
      mbar_init(baddr(&hdr->o_full[t]), 1);
      mbar_init(baddr(&hdr->o_empty[t]), 4);
    }
    mbar_init(baddr(&hdr->drain), 1);
    hdr->abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tm_q);
    tma_prefetch_desc(&p.tm_k);
    tma_prefetch_desc(&p.tm_v);
  }
  if (warp == kPrMmaWarp) {
    tmem_alloc(smem_u32(&hdr->tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = hdr->tmem_base;
  stream_release();
  stream_wait();
  const WaitCtl ctl{&hdr->abort_flag, p.status, p.timeout_ns};
  if (warp >= kPrMmaWarp) {
    if (warp == kPrMmaWarp)
      pr_mma<kD>(p, hdr, q_smem, ring, tmem, u0, u1, ctl, lane);
    else if (warp == kPrTmaWarp)
      pr_tma<kD>(p, hdr, q_smem, ring, u0, u1, ctl, lane);
  } else {
    pr_softmax<kD>(p, hdr, gbase + kPrHeader + 2 * pr_tile(kD), tmem, u0, u1, ctl, warp, lane);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kPrMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The parts of the blocks that are cut, joined in their order:
//   m = max m_k,  l = sum 2^(m_k - m) l_k,  O = sum 2^(m_k - m) O_k / l.
// A thread takes 16 columns of a row of tile blockIdx.x & 1.  Bound by the round
// trips to L2, one for kPrDeep parts: about 3 us behind the kernel before it.
constexpr int kPrDeep = 4;  // parts whose loads are in flight
template <int kD>
__global__ void __launch_bounds__(256) prompt_join(const __grid_constant__ PromptParams p) {
  constexpr int kGroups = kD / 16, kRows = 256 / kGroups;
  const int t = blockIdx.x & 1, row = blockIdx.y * kRows + threadIdx.x % kRows, g = threadIdx.x / kRows;
  const PromptUnit un = p.joins[blockIdx.x >> 1];
  const int token = un.q0 + t * p.tile_tokens + row / p.packed, head = un.head0 + row % p.packed;
  stream_release();
  stream_wait();
  if (token >= un.q_end || (t == 1 && !un.two)) return;
  const int64_t stride = 2 * prompt_slot_floats(kD);
  const float* work = p.work + (static_cast<int64_t>(un.first) + t) * prompt_slot_floats(kD);
  const float* ms = work + 128 * kD + row;
  const float4* src = reinterpret_cast<const float4*>(work) + 4 * g * 128 + row;
  float m = -INFINITY, l = 0.f, sum[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) sum[i] = 0.f;
  for (int k0 = 0; k0 < un.parts; k0 += kPrDeep) {
    float4 v[kPrDeep][4];
    float mk[kPrDeep], lk[kPrDeep];
#pragma unroll
    for (int k = 0; k < kPrDeep; ++k) {
      const bool have = k0 + k < un.parts;
      mk[k] = have ? __ldcg(ms + (k0 + k) * stride) : -INFINITY;
      lk[k] = have ? __ldcg(ms + (k0 + k) * stride + 128) : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[k][i] = have ? __ldcg(src + (k0 + k) * (stride / 4) + i * 128) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < kPrDeep; ++k) top = max3(top, mk[k], mk[k]);
    const float f0 = m == -INFINITY ? 0.f : ex2(m - top);
    m = top;
    l *= f0;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] *= f0;
#pragma unroll
    for (int k = 0; k < kPrDeep; ++k) {
      if (mk[k] == -INFINITY) continue;  // a part without keys has written no sums
      const float f = ex2(mk[k] - m);
      l += f * lk[k];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum[4 * i] += f * v[k][i].x, sum[4 * i + 1] += f * v[k][i].y;
        sum[4 * i + 2] += f * v[k][i].z, sum[4 * i + 3] += f * v[k][i].w;
      }
    }
  }
  const float inv = share_of(m, l);
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack2(sum[2 * i] * inv, sum[2 * i + 1] * inv);
  uint16_t* dst = static_cast<uint16_t*>(p.o.p) + token * p.o.token + head * p.o.head + 16 * g;
  *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(dst + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  if (g == 0 && p.lse) p.lse[static_cast<int64_t>(token) * p.heads + head] = lse_of(m, l);
}

// Tensor map of a [tokens][heads][d] operand, box {64, box_heads, box_tokens}.
// A dimension of one entry is never stepped over: its stride is any valid one.
bsp_status encode_heads(bsp_device* dev, CUtensorMap* tm, const HeadsView& x, int64_t tokens, int heads, int d,
                        uint32_t box_heads, uint32_t box_tokens) {
  const uint64_t dims[3] = {static_cast<uint64_t>(d), static_cast<uint64_t>(heads), static_cast<uint64_t>(tokens)};
  const uint64_t strides[2] = {static_cast<uint64_t>(heads > 1 ? x.head : d) * 2,
                               static_cast<uint64_t>(tokens > 1 ? x.token : static_cast<int64_t>(heads) * d) * 2};
  const uint32_t box[3] = {64, box_heads, box_tokens};
  return encode_nd(dev, tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, x.p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

using PromptKernel = void (*)(PromptParams);
PromptKernel pick(int d) { return d == 64 ? prompt_tcgen05<64> : prompt_tcgen05<128>; }

}  // namespace

int prompt_smem_bytes(int d) { return static_cast<int>(1024u + kPrHeader + (2u + pr_slots(d)) * pr_tile(d)); }

bsp_status prepare_prompt(const bsp_prompt_plan* plan) {
  return cuda_check(cudaFuncSetAttribute(pick(plan->d), cudaFuncAttributeMaxDynamicSharedMemorySize, plan->smem_bytes),
                    "cudaFuncSetAttribute(prompt)");
}

bsp_status launch_prompt(const bsp_prompt_plan* plan, PromptParams& p, cudaStream_t stream) {
  bsp_device* dev = plan->dev;
  bsp_status st = encode_heads(dev, &p.tm_q, p.q, plan->q_tokens, plan->heads, plan->d, plan->packed,
                               plan->tile_tokens);
  p.tm_k = p.tm_v = p.tm_q;  // without any key nothing loads through these
  if (st == BSP_OK && plan->kv_tokens > 0) {
    st = encode_heads(dev, &p.tm_k, p.k, plan->kv_tokens, plan->kv_heads, plan->d, 1, 128);
    if (st == BSP_OK) st = encode_heads(dev, &p.tm_v, p.v, plan->kv_tokens, plan->kv_heads, plan->d, 1, 128);
  }
  if (st != BSP_OK) return st;
  st = launch_overlapped(pick(plan->d), dim3(plan->grid), kPrThreads, plan->smem_bytes, stream, p,
                         "prompt attention launch");
  if (st != BSP_OK || plan->h_joins.empty()) return st;
  return launch_overlapped(plan->d == 64 ? prompt_join<64> : prompt_join<128>,
                           dim3(2 * static_cast<unsigned>(plan->h_joins.size()), plan->d / 32), 256, 0, stream, p,
                           "prompt join launch");
}

}  // namespace bsp
