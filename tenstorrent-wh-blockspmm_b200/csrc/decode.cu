// Attention of one token of each sequence over the paged 8-bit cache:
//   o = sum_t softmax_t(scale q k_t) v_t,  k_t = code * 2^a, v_t = code * 2^b
// with a and b of the token's page.
//
// Memory-bound: 2 d bytes of codes per token and key/value head are read once,
// for all the query heads that share it.
//
// Work.  A row is one sequence x one key/value head x up to 16 of its query
// heads; a tile is 128 tokens of a row.  The tiles of all rows form one list,
// and each CTA takes an equal stretch of it, whatever the lengths (read from
// the device).  A row that crosses a stretch's end is cut: its parts leave
// (m, l, O) in the workspace, and the CTA that finishes last joins them, in
// the order of the parts (the result does not depend on who is last).
//
// Tile.  K and V codes of 128 tokens come by TMA, one box per page (or 128
// tokens of it) and operand, swizzled so that ldmatrix reads without bank
// conflicts.  Each of four warps takes 32 tokens with its own running maximum:
//   S^T [16 tokens x 8 heads]  = K Q^T    m16n8k16, A = K, B = Q
//   P'  = 2^(S c - m + 7 + b - r)         c = scale log2 e 2^a; m follows the
//                                         largest S c; l sums P' 2^(r - b - 7)
//   O^T [d x 8 heads]         += V^T P'   A = V (ldmatrix.trans), B = P'
// V enters the product as its codes, so O is in units of 2^(r - 7), r the warp's
// reference: b <= r <= b + 7 for the pages at hand, moved (and O with it, in
// fp32) only when a page's b leaves that span.
// e4m3 codes are exact in fp16.  Q is scaled to [1, 2) by a power of two per
// head before it is rounded to fp16: bf16's 8 bits fit down to 2^-17 of the head's
// largest value, below that a value is off by up to 2^-25 of the largest.
// P' <= 2^15 is rounded to fp16: 2^-11 of a weight, or, far below, 2^-25 of the
// largest weight (2^-32 where the pages' scales are alike).  Were b part of m, one
// page of large scale would take all other pages' weights below what fp16 holds,
// whether its values count or not (a page of zeros has scale 1).  Sums are in fp32.
//
// Warps (192 threads): 0-3 as above, 4 issues the copies of K, 5 those of V;
// they hold the page numbers and scales of the next tiles in their lanes, so
// that those loads are off the path.  Every wait is bounded; a CTA that gave up
// still counts its parts, so the counters stay right for the next launch.
//
// Measured: two contexts of 100003 and 131072 tokens, 8 key/value heads of 128
// for 40 query heads, 85 us (5580 GB/s, 85 % of a plain copy's rate); 64 of 500
// to 8000 tokens 65 us (5180 GB/s).  Its steady state runs at the copy's rate (a
// copy of the kernel that only loads takes 80 and 61 us); the rest, about 10 us,
// is the launch, the first loads of a CTA and the joining.  24 sequences in
// pages of 16, 16 heads of 64: 29 us (2890 GB/s), where a box is 1 KB.  One
// sequence of 1000 tokens: 7.2 us (taken apart when it was 7.0: 0.8 an empty
// launch, 0.7 finding the tiles, 3.4 a tile from its page number to its result and
// 2.1 the joining).  With b in the running maximum these were 85, 64, 27 and 6.9 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bsp_ptx.cuh"
#include "decoder.h"

namespace bsp {
using namespace dev;

namespace {

constexpr int kDcSlices = 2;             // of 16 tokens that a warp takes of a tile
constexpr int kDcTile = 64 * kDcSlices;  // tokens
constexpr int kDcThreads = 192;
constexpr int kDcTmaWarp = 4;  // K; the next one V
constexpr int kDcMaxSlots = 12;
constexpr int kDcJoin = 8;
constexpr float kDcRescale = 8.f;    // log2 of the growth that moves the maximum
constexpr float kDcSpan = 7.f;       // how far a page's exponent may be below the reference: 2^(8 + 7) fits fp16
constexpr float kDcNoRef = -128.f;   // below any exponent

struct DcHeader {
  uint64_t full[kDcMaxSlots], empty[kDcMaxSlots];
  int32_t base;         // first tile of sequence `seq`
  int32_t seq;
  int32_t ctas;         // CTAs that take part: CTA b has `each` tiles, one more if b < `extra`
  uint32_t each, extra;
  int32_t last;         // this CTA joins the row
  int abort_flag;
  float scales[kDcMaxSlots][kDcTile / 16];  // 2^a, or b, of each 16 tokens of a slot
};
static_assert(sizeof(DcHeader) <= 1024, "header must fit its 1 KiB slot");

// Shared memory from the 1 KiB-aligned base: header, slots (K and V of a tile
// in turn), then the warps' results: O [4][heads][d], m [4][heads], l [4][heads].
// CTAs on an SM: two; four for rows of up to 8 heads of 64, whose tiles are half
// the bytes for the same work on scores (16 heads of 64 in pages of 16, the same
// inputs again and again: 31.8 us with two, 26.8 with three, 25.6 with four).  Rows
// of 16 heads with one CTA, which leaves them more registers: 64 contexts of 4000
// tokens, 4 key/value heads of 128 72 us, with two 57; heads of 64 54 and 39.
__host__ __device__ constexpr int dc_per_sm(int d, int heads) { return heads <= 8 && d == 64 ? 4 : 2; }
// As many slots as fit the SM's 228 KB then (1 KB of each CTA is the system's).
__host__ __device__ constexpr int dc_slot_bytes(int d) { return kDcTile * d; }
__host__ __device__ constexpr int dc_result_bytes(int d, int heads) { return 16 * heads * (d + 2); }
__host__ __device__ constexpr int dc_slots(int d, int heads) {
  const int n = ((228 / dc_per_sm(d, heads) - 1) * 1024 - 2048 - dc_result_bytes(d, heads)) / dc_slot_bytes(d);
  return n < kDcMaxSlots ? n : kDcMaxSlots;
}
__host__ __device__ constexpr int dc_smem(int d, int heads) {
  return 2048 + dc_slots(d, heads) * dc_slot_bytes(d) + dc_result_bytes(d, heads);
}

__device__ __forceinline__ uint32_t baddr(const uint64_t* b) { return smem_u32(b); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// two e4m3 codes (16 bits) to two fp16, exactly
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// transpose of an 8 x 8 matrix of 16-bit values held by the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half_pair(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t bf16_two(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

__device__ __forceinline__ void tma_load_4d_pred(uint32_t smem_dst, const void* tmap, int32_t x, int32_t y, int32_t z,
                                                 int32_t w, uint32_t bar, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %7, 0;\n\t"
      "@q cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];\n\t}" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar), "r"(issue)
      : "memory");
}

// Tokens of sequence s that count: 0 where the length is not one that the page
// table holds.
__device__ __forceinline__ int dc_len(const DecodeParams& p, int s) {
  const int len = p.lens[s];
  return len < 0 || len > p.max_len ? 0 : len;
}
__device__ __forceinline__ int dc_tiles(const DecodeParams& p, int s) { return (dc_len(p, s) + kDcTile - 1) / kDcTile; }

// The CTA that has tile x of the list.
__device__ __forceinline__ int cta_of(const DcHeader* hdr, uint32_t x) {
  const uint32_t longer = hdr->extra * (hdr->each + 1);
  return static_cast<int>(x < longer ? x / (hdr->each + 1) : hdr->extra + (x - longer) / hdr->each);
}

// A CTA's way through its stretch [g, g1) of the list of tiles (under 2^31 in
// all: 2^38 tokens).
struct Walk {
  int32_t g, g1, base;
  int seq, tiles;  // of the current sequence
};
struct Piece {
  int seq, stream, tile0, n, tiles;  // tiles [tile0, tile0 + n) of the row's `tiles`
  int32_t row0;                      // the row's first tile in the list
};
__device__ __forceinline__ bool next_piece(const DecodeParams& p, Walk& w, Piece& pc) {
  if (w.g >= w.g1) return false;
  while (w.g - w.base >= w.tiles * p.streams) {
    w.base += w.tiles * p.streams;
    if (++w.seq >= p.n_seqs) return false;
    w.tiles = dc_tiles(p, w.seq);
  }
  const uint32_t rel = static_cast<uint32_t>(w.g - w.base);
  pc.seq = w.seq;
  pc.tiles = w.tiles;
  pc.stream = static_cast<int>(rel / static_cast<uint32_t>(w.tiles));
  pc.tile0 = static_cast<int>(rel) - pc.stream * w.tiles;
  pc.n = min(w.tiles - pc.tile0, w.g1 - w.g);
  pc.row0 = w.base + pc.stream * w.tiles;
  w.g += pc.n;
  return true;
}

// Copy x of a CTA (K of its first tile 0, V 1, K of the next 2, ...) goes to slot
// x % kSlots, which with an odd number of slots passes between the two warps.  A
// parity names a phase only while the others of that parity are over: before copy x
// its warp waits for the reading of copy x - kSlots, and when it gets there copy
// x - 2 - kSlots has been read (its last wait), so copy x - 2 kSlots too, since the
// consumers go in order.
template <int kD, int kSlots>
__device__ __forceinline__ void dc_produce(const DecodeParams& p, DcHeader* hdr, uint32_t ring, Walk w,
                                          const WaitCtl& ctl, int kind, int lane) {
  const int page = p.cache.page, shift = __ffs(page) - 1;  // a power of two
  const int box = min(page, kDcTile), boxes = kDcTile / box;  // per tile and operand
  const int shift_b = __ffs(boxes) - 1;
  const int at = lane >> shift_b, sub = lane & (boxes - 1);  // lane's tile of a batch, its box
  const int per_batch = 32 >> shift_b;
  const float* scale = kind ? p.cache.v_scale : p.cache.k_scale;
  const CUtensorMap* tm = kind ? &p.tm_v : &p.tm_k;
  int slot = kind;  // K of the first tile has slot 0, V slot 1, K of the next 2 ...
  uint32_t phase = 0;
  int done = 0;  // tiles
  bool ok = true;
  Piece pc;
  while (ok && next_piece(p, w, pc)) {
    const int len = dc_len(p, pc.seq), kvh = pc.stream / p.chunks;
    const int32_t* pages = p.page_table + pc.seq * p.table_stride;
    // lane's box of the batch that starts at tile b: its page and scale
    auto page_of = [&](int b) -> int32_t {
      const int64_t token = static_cast<int64_t>(pc.tile0 + b + at) * kDcTile + sub * box;
      return b + at < pc.n && token < len ? pages[token >> shift] : -2;  // -2: no box
    };
    auto checked = [&](int32_t id) -> int32_t {
      if (id == -2 || (id >= 0 && id < p.cache.n_pages)) return id;
      atomicOr(p.status, ST_BAD_INDEX);
      return -1;  // read as zeros
    };
    auto scale_of = [&](int32_t id) {
      return id >= 0 ? scale[static_cast<int64_t>(id) * p.cache.kv_heads + kvh] : 1.f;
    };
    auto held = [&](float s) {  // what the slot holds of a scale: a V slot its exponent
      return kind ? static_cast<float>(static_cast<int>((__float_as_uint(s) >> 23) & 0xFFu) - 127) : s;
    };
    int32_t id = checked(page_of(0)), id_next = page_of(per_batch);
    float sc = scale_of(id);
#pragma unroll 1
    for (int b = 0; b < pc.n && ok; b += per_batch) {
      const int32_t idn = checked(id_next);
      id_next = page_of(b + 2 * per_batch);
      const float sc_next = scale_of(idn);
      const int n = min(per_batch, pc.n - b);
#pragma unroll 1
      for (int k = 0; k < n; ++k) {
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(baddr(&hdr->empty[slot]), phase ^ 1u, ctl, ST_TIMEOUT_PRODUCER));
        if (!ok) break;
        const bool mine = at == k && id != -2;
        const uint32_t bar = baddr(&hdr->full[slot]);
        // The copies go first: their scales may still be on the way.
        tma_load_4d_pred(ring + slot * dc_slot_bytes(kD) + sub * box * kD, tm, 0, 0, kvh,
                         id >= 0 ? id : static_cast<int32_t>(p.cache.n_pages), bar, mine);
        if (at == k)
          for (int i = 0; i < box / 16; ++i) hdr->scales[slot][sub * (box / 16) + i] = held(sc);
        const uint32_t bytes = static_cast<uint32_t>(__popc(__ballot_sync(0xffffffffu, mine))) * box * kD;
        __syncwarp();  // the scales are written before lane 0 arrives
        mbar_arrive_expect_tx_pred(bar, bytes, lane == 0);
        ++done;
        slot += 2;
        if (slot >= kSlots) slot -= kSlots, phase ^= 1u;
      }
      id = idn;
      sc = sc_next;
    }
  }
  if (lane == 0) {
    // No copy may be in flight when the CTA leaves: wait for the last round of
    // slots (one that was filled again since has been consumed).
    int zero = 0;
    const WaitCtl c2{&zero, ctl.status, ctl.timeout_ns};
    for (int i = max(0, done - (kSlots + 1) / 2); i < done; ++i) {
      const int at = 2 * i + kind;
      if (at + kSlots >= 2 * done)
        mbar_wait_bounded(baddr(&hdr->full[at % kSlots]), static_cast<uint32_t>(at / kSlots) & 1u, c2, ST_TIMEOUT_DRAIN);
    }
  }
  __syncwarp();
}

// A warp's (m, l, O) to shared memory, slot of four, as what the results of warps
// and parts are joined by: O = 2^m O', sum of weights = 2^m l'.  The reference goes
// into m and l as far as 2^+-50, so that a factor 2^(m - m') never takes another's
// sum of weights below fp32's range; what is left of it into O.
template <int kD, int kNt>
__device__ __forceinline__ void put_result(float* red_o, float* red_m, float* red_l, int slot, int g, int t,
                                          float (&o)[kNt][kD / 16][4], const float (&m)[kNt][2],
                                          const float (&l)[kNt][2], float ref, int nh) {
  constexpr int kHeads = 8 * kNt;
  const float fit = fminf(fmaxf(ref, -50.f), 50.f);
  if (ref != fit) {
    const float f = ex2(ref - fit);
#pragma unroll
    for (int n = 0; n < kNt; ++n)
#pragma unroll
      for (int c = 0; c < kD / 16; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][c][i] *= f;
  }
  const float shift = fit - kDcSpan, unit = ex2(-shift);
#pragma unroll
  for (int n = 0; n < kNt; ++n) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x = l[n][h];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      const int head = 8 * n + 2 * t + h;
      if (g == 0) {
        red_m[slot * kHeads + head] = m[n][h] + shift;
        red_l[slot * kHeads + head] = x * unit;
      }
      float* dst = red_o + (slot * kHeads + head) * kD + 2 * g;
      if (head < nh)
#pragma unroll
        for (int c = 0; c < kD / 16; ++c) *reinterpret_cast<float2*>(dst + 16 * c) = make_float2(o[n][c][h], o[n][c][2 + h]);
    }
  }
}

template <int kD, int kNt>
__device__ __forceinline__ void dc_consume(const DecodeParams& p, DcHeader* hdr, uint32_t ring, float* red, Walk w,
                                          const WaitCtl& ctl, int warp, int lane) {
  constexpr int kChunks = kD / 16, kHeads = 8 * kNt, kSlots = dc_slots(kD, kHeads);
  const int g = lane >> 2, t = lane & 3;
  // ldmatrix: lane's row in a 16-token slice and its 16-byte chunk, swizzled.
  // Matrices: (tokens 0-7, 8-15) x (chunk c, c + 1); chunk c is c * 16 exclusive-or
  // this address.
  const int row = (lane & 7) + ((lane >> 3) & 1) * 8;
  const int swz = kD == 128 ? (row & 7) : ((row >> 1) & 3);
  const uint32_t first = static_cast<uint32_t>((16 * kDcSlices * warp + row) * kD + (((lane >> 4) ^ swz) << 4));
  float* red_o = red;                            // [4][kHeads][kD]
  float* red_m = red + 4 * kHeads * kD;          // [4][kHeads]
  float* red_l = red_m + 4 * kHeads;
  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;
  Piece pc;
  while (next_piece(p, w, pc)) {
    const int len = dc_len(p, pc.seq);
    const int kvh = pc.stream / p.chunks, h0 = kvh * p.group + (pc.stream % p.chunks) * 16;
    const int nh = min(16, p.group - (pc.stream % p.chunks) * 16);
    uint32_t q[kNt][kChunks][2];
    float qs[kNt][2];  // scale log2 e times the power of two taken out of q, of heads 2 t, 2 t + 1
#pragma unroll
    for (int n = 0; n < kNt; ++n) {
      float v[kChunks][4], top = 0.f;
      const bool have = 8 * n + g < nh;
      const uint16_t* src = static_cast<const uint16_t*>(p.q.p) + pc.seq * p.q.token + (h0 + 8 * n + g) * p.q.head;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const uint2 x = have ? *reinterpret_cast<const uint2*>(src + 16 * c + 4 * t) : make_uint2(0, 0);
        v[c][0] = __uint_as_float(x.x << 16);
        v[c][1] = __uint_as_float(x.x & 0xFFFF0000u);
        v[c][2] = __uint_as_float(x.y << 16);
        v[c][3] = __uint_as_float(x.y & 0xFFFF0000u);
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(v[c][i]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e with e the exponent of the largest value, kept where 2^-e is a normal number
      const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
      const float down = __uint_as_float((254u - e) << 23), up = __uint_as_float(e << 23);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        q[n][c][0] = half_pair(v[c][0] * down, v[c][1] * down);
        q[n][c][1] = half_pair(v[c][2] * down, v[c][3] * down);
      }
      // head g's factor sits in the lanes 4 g ..; this lane needs heads 2 t, 2 t + 1
      qs[n][0] = __shfl_sync(0xffffffffu, up, 8 * t) * p.scale_log2;
      qs[n][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4) * p.scale_log2;
    }
    float o[kNt][kChunks][4], m[kNt][2], l[kNt][2];
    float ref = kDcNoRef;
#pragma unroll
    for (int n = 0; n < kNt; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) o[n][c][0] = o[n][c][1] = o[n][c][2] = o[n][c][3] = 0.f;
    }
    auto wait_slot = [&]() {
      return __all_sync(0xffffffffu, mbar_wait_bounded(baddr(&hdr->full[slot]), phase, ctl, ST_TIMEOUT_EPILOGUE));
    };
    auto free_slot = [&]() {
      __syncwarp();
      mbar_arrive_pred(baddr(&hdr->empty[slot]), lane == 0);
      if (++slot == kSlots) slot = 0, phase ^= 1u;
    };
#pragma unroll 1
    for (int k = 0; k < pc.n && ok; ++k) {
      const int left = len - (pc.tile0 + k) * kDcTile - 16 * kDcSlices * warp;  // tokens of this warp
      ok = wait_slot();
      if (!ok) break;
      if (left <= 0) {
        free_slot();
        ok = wait_slot();
        if (!ok) break;
      } else {
        const uint32_t kb = ring + slot * dc_slot_bytes(kD) + first;
        const float* k_scales = hdr->scales[slot] + kDcSlices * warp;
        float s[kDcSlices][kNt][4];
        bool grow = false;
        float mx[kNt][2];
#pragma unroll
        for (int n = 0; n < kNt; ++n) mx[n][0] = mx[n][1] = -INFINITY;
#pragma unroll
        for (int sl = 0; sl < kDcSlices; ++sl) {
#pragma unroll
          for (int n = 0; n < kNt; ++n) s[sl][n][0] = s[sl][n][1] = s[sl][n][2] = s[sl][n][3] = 0.f;
#pragma unroll
          for (int c = 0; c < kChunks; c += 2) {
            uint32_t r[4];  // (tokens 0-7, chunk c), (8-15, c), (0-7, c + 1), (8-15, c + 1)
            ldmatrix4((kb ^ (c << 4)) + sl * 16 * kD, r);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t a0, a1, a2, a3;
              codes_to_half(r[2 * i], a0, a2);
              codes_to_half(r[2 * i + 1], a1, a3);
#pragma unroll
              for (int n = 0; n < kNt; ++n) mma16816(s[sl][n], a0, a1, a2, a3, q[n][c + i][0], q[n][c + i][1]);
            }
          }
          // s[sl][n]: tokens g and g + 8 (rows) of heads 2 t, 2 t + 1 (columns)
#pragma unroll
          for (int n = 0; n < kNt; ++n) {
#pragma unroll
            for (int h = 0; h < 4; ++h) s[sl][n][h] *= qs[n][h & 1] * k_scales[sl];
          }
        }
        free_slot();
        ok = wait_slot();
        if (!ok) break;
        const uint32_t vb_at = ring + slot * dc_slot_bytes(kD) + first;
        const float* v_scales = hdr->scales[slot] + kDcSlices * warp;
#pragma unroll
        for (int sl = 0; sl < kDcSlices; ++sl) {
          const bool in0 = 16 * sl + g < left, in1 = 16 * sl + g + 8 < left;
#pragma unroll
          for (int n = 0; n < kNt; ++n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              s[sl][n][h] = in0 ? s[sl][n][h] : -INFINITY;
              s[sl][n][2 + h] = in1 ? s[sl][n][2 + h] : -INFINITY;
              mx[n][h] = fmaxf(mx[n][h], fmaxf(s[sl][n][h], s[sl][n][2 + h]));
            }
          }
        }
#pragma unroll
        for (int n = 0; n < kNt; ++n) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x = mx[n][h];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            mx[n][h] = x;
            grow |= x > m[n][h] + kDcRescale;
          }
        }
        // log2 of the factor in a slice's P', and its inverse
        float up[kDcSlices], down[kDcSlices], vb[kDcSlices];
        bool move = grow;
#pragma unroll
        for (int sl = 0; sl < kDcSlices; ++sl) {
          vb[sl] = 16 * sl < left ? v_scales[sl] : vb[0];
          up[sl] = kDcSpan + vb[sl] - ref;
          down[sl] = ex2(-up[sl]);
          move |= !(fabsf(2.f * up[sl] - kDcSpan) <= kDcSpan);
        }
        // Codes behind the last token are whatever the page held: clear them
        // (0 times a NaN code would not be 0).
        const bool tail = left < 16 * kDcSlices;
        auto add_slice = [&](int sl) {
          uint32_t pb[kNt][2];
#pragma unroll
          for (int n = 0; n < kNt; ++n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float mm = (m[n][h] == -INFINITY ? 0.f : m[n][h]) - up[sl];
              s[sl][n][h] = ex2(s[sl][n][h] - mm);
              s[sl][n][2 + h] = ex2(s[sl][n][2 + h] - mm);
              l[n][h] += (s[sl][n][h] + s[sl][n][2 + h]) * down[sl];
            }
            pb[n][0] = transpose8(half_pair(s[sl][n][0], s[sl][n][1]));  // B: tokens 2 t, 2 t + 1 of head g
            pb[n][1] = transpose8(half_pair(s[sl][n][2], s[sl][n][3]));  // tokens 2 t + 8, 2 t + 9
          }
          uint32_t keep0 = ~0u, keep1 = ~0u;
          if (tail) {
            const int at = left - 16 * sl - 2 * t;
            keep0 = (0 < at ? 0xFFFFu : 0u) | (1 < at ? 0xFFFF0000u : 0u);
            keep1 = (8 < at ? 0xFFFFu : 0u) | (9 < at ? 0xFFFF0000u : 0u);
          }
#pragma unroll
          for (int c = 0; c < kChunks; c += 2) {
            uint32_t r[4];
            ldmatrix4t((vb_at ^ (c << 4)) + sl * 16 * kD, r);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              // register: codes (token 2 t, d 2 g), (2 t, 2 g + 1), (2 t + 1, 2 g), (2 t + 1, 2 g + 1)
              uint32_t a0, a1, a2, a3;  // rows 0-7 of A: even d, rows 8-15: odd d
              codes_to_half(__byte_perm(r[2 * i], 0, 0x3120), a0, a1);
              codes_to_half(__byte_perm(r[2 * i + 1], 0, 0x3120), a2, a3);
              if (tail) a0 &= keep0, a1 &= keep0, a2 &= keep1, a3 &= keep1;
#pragma unroll
              for (int n = 0; n < kNt; ++n) mma16816(o[n][c + i], a0, a1, a2, a3, pb[n][0], pb[n][1]);
            }
          }
        };
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll 1
          for (bool last = false; !last;) {
            // The reference nearest to the present one that holds both slices, or,
            // where none does, the first slice (which is added here then) and after
            // it the second.  Downwards O's numbers grow: they stay below 2^100, and
            // what a page that the reference cannot come down to would add is less
            // than 2^-60 of O's largest: it only counts in l.
            last = fabsf(vb[0] - vb[1]) <= kDcSpan;
            float to = fminf(fmaxf(ref, last ? fmaxf(vb[0], vb[1]) : vb[0]), (last ? fminf(vb[0], vb[1]) : vb[0]) + kDcSpan);
            if (to < ref) {
              float top = 0.f;
#pragma unroll
              for (int n = 0; n < kNt; ++n)
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
#pragma unroll
                  for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(o[n][c][i]));
              const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
              const int room = min(max(227 - static_cast<int>(bits >> 23), 0), 120);
              if (bits != 0) to = fmaxf(to, ref - static_cast<float>(room));
            }
            const float unit = ex2(fminf(ref - to, 120.f));
            ref = to;
#pragma unroll
            for (int n = 0; n < kNt; ++n) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float mn = fmaxf(m[n][h], mx[n][h]);
                const float f = m[n][h] == -INFINITY ? 0.f : ex2(m[n][h] - mn);
                m[n][h] = mn;
                l[n][h] *= f;
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                  o[n][c][h] *= f * unit;
                  o[n][c][2 + h] *= f * unit;
                }
              }
            }
#pragma unroll
            for (int sl = 0; sl < kDcSlices; ++sl) {
              up[sl] = kDcSpan + vb[sl] - ref;
              down[sl] = ex2(-up[sl]);
              if (up[sl] < 0.f && (sl == 0 || last)) {
#pragma unroll
                for (int n = 0; n < kNt; ++n)
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const float mm = m[n][h] == -INFINITY ? 0.f : m[n][h];
                    l[n][h] += ex2(s[sl][n][h] - mm) + ex2(s[sl][n][2 + h] - mm);
                  }
                up[sl] = -INFINITY;
                down[sl] = 0.f;
              }
            }
            if (!last) {
              add_slice(0);
#pragma unroll
              for (int n = 0; n < kNt; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[0][n][i] = -INFINITY;  // it has been added
              vb[0] = vb[1];
            }
          }
        }
#pragma unroll
        for (int sl = 0; sl < kDcSlices; ++sl) add_slice(sl);
      }
      free_slot();
    }
    // ---- the four warps' results of this piece
    consumers_sync();  // the last piece's have been read
    put_result<kD, kNt>(red_o, red_m, red_l, warp, g, t, o, m, l, ref, nh);
    consumers_sync();
    const int tid = 32 * warp + lane;
    const bool whole = pc.n == pc.tiles;
    const int64_t slot_floats = 16 * (kD + 2);
    float* ws = p.work + (2 * static_cast<int64_t>(blockIdx.x) + (pc.tile0 == 0 ? 1 : 0)) * slot_floats;
    auto put_o = [&](int head, int col, float4 a, float M, float L) {
      const float inv = 1.f / L;
      uint16_t* dst = static_cast<uint16_t*>(p.o.p) + pc.seq * p.o.token + (h0 + head) * p.o.head + 4 * col;
      *reinterpret_cast<uint2*>(dst) = make_uint2(bf16_two(a.x * inv, a.y * inv), bf16_two(a.z * inv, a.w * inv));
      if (col == 0 && p.lse)
        p.lse[static_cast<int64_t>(pc.seq) * p.heads + h0 + head] = (M + log2f(L)) * 0.6931471805599453f;
    };
    for (int i = tid; i < nh * (kD / 4); i += 128) {
      const int head = i / (kD / 4), col = i % (kD / 4);
      float M = red_m[head];
      for (int k = 1; k < 4; ++k) M = fmaxf(M, red_m[k * kHeads + head]);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      float L = 0.f;
      for (int k = 0; k < 4; ++k) {
        const float mk = red_m[k * kHeads + head];
        // a warp without tokens has m = -inf and l = 0; one that met only NaN has l = NaN
        const float f = mk == -INFINITY ? 1.f : ex2(mk - M);
        const float4 v = reinterpret_cast<const float4*>(red_o + (k * kHeads + head) * kD)[col];
        a.x += f * v.x, a.y += f * v.y, a.z += f * v.z, a.w += f * v.w;
        L += f * red_l[k * kHeads + head];
      }
      if (whole) {
        put_o(head, col, a, M, L);
      } else {
        __stcg(reinterpret_cast<float4*>(ws + head * kD) + col, a);
        if (col == 0) {
          __stcg(ws + 16 * kD + head, M);
          __stcg(ws + 16 * kD + 16 + head, L);
        }
      }
    }
    if (whole) continue;
    // ---- a part of a row: the last of its CTAs joins the parts
    const int first_cta = cta_of(hdr, pc.row0), last_cta = cta_of(hdr, pc.row0 + pc.tiles - 1);
    const int parts = last_cta - first_cta + 1;
    consumers_sync();  // all of this part is written: the release below covers it
    if (tid == 0) {
      int before;
      asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;"
                   : "=r"(before) : "l"(p.counters + first_cta) : "memory");
      hdr->last = before == parts - 1 ? 1 : 0;
    }
    consumers_sync();
    if (!hdr->last) continue;
    const float* first_ws = p.work + (2 * static_cast<int64_t>(first_cta) + 1) * slot_floats;
    for (int i = tid; i < nh * (kD / 4); i += 128) {
      const int head = i / (kD / 4), col = i % (kD / 4);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      float M = -INFINITY, L = 0.f;
      for (int k0 = 0; k0 < parts; k0 += kDcJoin) {  // kDcJoin parts a round trip to L2
        float4 v[kDcJoin];
        float mk[kDcJoin], lk[kDcJoin];
#pragma unroll
        for (int k = 0; k < kDcJoin; ++k) {
          const bool have = k0 + k < parts;
          const float* src = k0 + k == 0 ? first_ws : p.work + 2 * static_cast<int64_t>(first_cta + k0 + k) * slot_floats;
          v[k] = have ? __ldcg(reinterpret_cast<const float4*>(src + head * kD) + col) : make_float4(0.f, 0.f, 0.f, 0.f);
          mk[k] = have ? __ldcg(src + 16 * kD + head) : -INFINITY;
          lk[k] = have ? __ldcg(src + 16 * kD + 16 + head) : 0.f;
        }
        float top = M;
#pragma unroll
        for (int k = 0; k < kDcJoin; ++k) top = fmaxf(top, mk[k]);
        const float f0 = M == -INFINITY ? 1.f : ex2(M - top);
        a.x *= f0, a.y *= f0, a.z *= f0, a.w *= f0;
        L *= f0;
        M = top;
#pragma unroll
        for (int k = 0; k < kDcJoin; ++k) {
          const float f = mk[k] == -INFINITY ? 1.f : ex2(mk[k] - top);
          a.x += f * v[k].x, a.y += f * v[k].y, a.z += f * v[k].z, a.w += f * v[k].w;
          L += f * lk[k];
        }
      }
      put_o(head, col, a, M, L);
    }
    if (tid == 0) p.counters[first_cta] = 0;  // ready for the next launch
  }
}

template <int kD, int kNt>
__global__ void __launch_bounds__(kDcThreads, dc_per_sm(kD, 8 * kNt)) decode_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  DcHeader* hdr = reinterpret_cast<DcHeader*>(gbase);
  const uint32_t ring = base + 1024u;
  constexpr int kSlots = dc_slots(kD, 8 * kNt);
  float* red = reinterpret_cast<float*>(gbase + 1024 + kSlots * dc_slot_bytes(kD));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0 && lane == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(baddr(&hdr->full[s]), 1);
      mbar_init(baddr(&hdr->empty[s]), 4);
    }
    hdr->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kDcTmaWarp && lane < 2) tma_prefetch_desc(lane ? &p.tm_v : &p.tm_k);
  stream_release();
  stream_wait();
  if (warp == kDcTmaWarp) {
    // tiles of all rows, then the sequence in which this CTA's stretch begins
    const int first = lane < p.n_seqs ? dc_tiles(p, lane) : 0;
    int64_t total = first;
    int longest = first;  // tiles of the longest row
    for (int s = lane + 32; s < p.n_seqs; s += 32) {
      const int n = dc_tiles(p, s);
      total += n;
      longest = max(longest, n);
    }
    for (int k = 16; k; k >>= 1) total += __shfl_xor_sync(0xffffffffu, total, k);
    longest = __reduce_max_sync(0xffffffffu, longest);
    total *= p.streams;
    if (total > 0x7FFFFFFF) {
      if (lane == 0) atomicOr(p.status, ST_BAD_INDEX);
      total = 0;
    }
    // A tile takes a CTA 1 us, and each part of a row 0.1 us more where they are
    // joined: a row of n tiles in parts of t takes t + 0.1 n / t, least at t =
    // sqrt(0.1 n).  Fewer tiles to a CTA only lengthen the joining (131072 tokens,
    // one key/value head: this rule 29.9 us, 16 tiles a CTA 30.5, 8 31.3, 4 45, one
    // 51; 8000 tokens: 11.8 us, 16 18.1, 8 13.9, 4 11.7, one 14.8).
    const uint32_t least = max(__float2uint_rn(sqrtf(0.09f * static_cast<float>(longest))), 1u);
    const int ctas = static_cast<int>(min(gridDim.x, (static_cast<uint32_t>(total) + least - 1) / least));
    const uint32_t each = ctas > 0 ? static_cast<uint32_t>(total) / static_cast<uint32_t>(ctas) : 0u;
    const uint32_t extra = static_cast<uint32_t>(total) - each * static_cast<uint32_t>(ctas);
    const int g0 = static_cast<int>(blockIdx.x * each + min(blockIdx.x, extra));
    int at = 0, seq = 0;
    bool found = false;
    for (int s0 = 0; s0 < p.n_seqs && !found; s0 += 32) {
      const int mine = (s0 == 0 ? first : s0 + lane < p.n_seqs ? dc_tiles(p, s0 + lane) : 0) * p.streams;
      int upto = mine;
      for (int k = 1; k < 32; k <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, k);
        if (lane >= k) upto += x;
      }
      const unsigned past = __ballot_sync(0xffffffffu, at + upto > g0);
      found = past != 0;
      const int src = found ? __ffs(past) - 1 : 31;
      const int incl = __shfl_sync(0xffffffffu, upto, src), own = __shfl_sync(0xffffffffu, mine, src);
      seq = s0 + src;
      at += found ? incl - own : incl;
    }
    if (lane == 0) {
      hdr->ctas = ctas;
      hdr->each = each;
      hdr->extra = extra;
      hdr->seq = seq;
      hdr->base = at;
    }
  }
  __syncthreads();
  // sequences without a token: O = 0, lse = -inf
  for (int s = blockIdx.x; s < p.n_seqs; s += gridDim.x) {
    if (dc_len(p, s) > 0) continue;
    if (threadIdx.x == 0 && p.lens[s] != 0) atomicOr(p.status, ST_BAD_INDEX);
    for (int i = threadIdx.x; i < p.heads * (kD / 8); i += kDcThreads) {
      const int head = i / (kD / 8), col = i % (kD / 8);
      uint16_t* dst = static_cast<uint16_t*>(p.o.p) + s * p.o.token + head * p.o.head;
      reinterpret_cast<uint4*>(dst)[col] = make_uint4(0, 0, 0, 0);
      if (col == 0 && p.lse) p.lse[static_cast<int64_t>(s) * p.heads + head] = -INFINITY;
    }
  }
  if (static_cast<int>(blockIdx.x) >= hdr->ctas) return;
  Walk w;
  w.g = static_cast<int32_t>(blockIdx.x * hdr->each + min(blockIdx.x, hdr->extra));
  w.g1 = w.g + static_cast<int32_t>(hdr->each + (blockIdx.x < hdr->extra ? 1u : 0u));
  w.base = hdr->base;
  w.seq = hdr->seq;
  w.tiles = dc_tiles(p, w.seq);
  const WaitCtl ctl{&hdr->abort_flag, p.status, p.timeout_ns};
  if (warp >= kDcTmaWarp) dc_produce<kD, kSlots>(p, hdr, ring, w, ctl, warp - kDcTmaWarp, lane);
  else dc_consume<kD, kNt>(p, hdr, ring, red, w, ctl, warp, lane);
}

bsp_status encode_codes(bsp_device* dev, CUtensorMap* tm, const bsp_kv_cache& c, const void* codes) {
  const uint64_t dims[4] = {static_cast<uint64_t>(c.d), static_cast<uint64_t>(c.page),
                            static_cast<uint64_t>(c.kv_heads), static_cast<uint64_t>(c.n_pages)};
  const uint64_t strides[3] = {static_cast<uint64_t>(c.d), static_cast<uint64_t>(c.head_stride),
                               static_cast<uint64_t>(c.page_stride)};
  const uint32_t box[4] = {static_cast<uint32_t>(c.d), static_cast<uint32_t>(std::min(c.page, kDcTile)), 1, 1};
  return encode_nd(dev, tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, codes, dims, strides, box,
                   c.d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

using DecodeKernel = void (*)(const DecodeParams);
DecodeKernel pick(int d, int group) {
  if (d == 64) return group > 8 ? decode_kernel<64, 2> : decode_kernel<64, 1>;
  return group > 8 ? decode_kernel<128, 2> : decode_kernel<128, 1>;
}

}  // namespace

int64_t decode_work_floats(int32_t ctas, int32_t d) { return 2 * static_cast<int64_t>(ctas) * 16 * (d + 2); }

int32_t decode_ctas(const bsp_device* dev, int d, int group) { return dc_per_sm(d, group > 8 ? 16 : 8) * dev->sm_count; }

int decode_smem_bytes(int d, int group) { return dc_smem(d, group > 8 ? 16 : 8); }

bsp_status prepare_decode(const bsp_decode_plan* plan) {
  return cuda_check(cudaFuncSetAttribute(pick(plan->d, plan->heads / plan->kv_heads),
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, plan->smem_bytes),
                    "cudaFuncSetAttribute(decode)");
}

bsp_status launch_decode(const bsp_decode_plan* plan, DecodeParams& p, cudaStream_t stream) {
  bsp_status st = encode_codes(plan->dev, &p.tm_k, p.cache, p.cache.k);
  if (st == BSP_OK) st = encode_codes(plan->dev, &p.tm_v, p.cache, p.cache.v);
  if (st != BSP_OK) return st;
  return launch_overlapped(pick(plan->d, p.group), dim3(plan->grid), kDcThreads, plan->smem_bytes, stream, p,
                           "decode attention launch");
}

}  // namespace bsp
