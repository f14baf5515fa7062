// Types of the decoder-attention operators (rotary positions, the paged 8-bit
// key/value cache, prompt attention, single-token attention).
#pragma once
#include "bsp_internal.h"

namespace bsp {

// A [token][head][d] operand: pointer and strides in elements.
struct HeadsView {
  const void* p;
  int64_t token, head;
};
struct HeadsOut {
  void* p;
  int64_t token, head;
};

struct RopeParams {
  HeadsView x;
  HeadsOut y;
  const int32_t* positions;
  const float2* table;   // [n_pos][rot / 2] (cos, sin)
  int64_t n_pos;
  int64_t tokens;
  int32_t heads, d, rot;
  int32_t interleaved;
  float sign;            // -1: transposed rotation
  // set at the launch: units of a head, (token, head group) items of a block,
  // head groups of a token
  int32_t units, items_per_block, groups;
  unsigned int* status;
};

struct AppendParams {
  HeadsView q, k, v;
  HeadsOut q_out, k_out;      // p may be null
  bsp_kv_cache cache;
  const int32_t* starts;      // [n_seqs + 1]
  const int32_t* before;      // [n_seqs]
  const int32_t* page_table;
  int64_t table_stride, table_width;
  const float2* table;        // null: no rotation
  int64_t n_pos;
  int64_t tokens;
  int32_t n_seqs, heads, rot, interleaved;
  int32_t page_shift;
  int32_t by_token;           // blocks are counted by tokens, not by pages
  unsigned int* status;
};

struct DecodeParams {
  CUtensorMap tm_k, tm_v;     // codes: [page][head][token][d], boxes of up to 128 tokens of one page and head
  HeadsView q;
  HeadsOut o;
  float* lse;
  bsp_kv_cache cache;
  const int32_t* lens;
  const int32_t* page_table;
  int64_t table_stride;
  int32_t max_len;            // tokens that a row of the page table holds, a tile below 2^31
  int32_t n_seqs, heads;
  int32_t group;              // query heads of one key/value head
  int32_t chunks;             // rows of up to 16 query heads per key/value head
  int32_t streams;            // rows per sequence: kv_heads * chunks
  float scale_log2;
  float* work;                // two slots per CTA: O [16][d], m [16], l [16] of a row's part
  int32_t* counters;          // one per CTA: finished parts of the row that begins in it, 0 between launches
  unsigned int* status;
  uint64_t timeout_ns;
};

// A unit of prompt attention: one or two tiles (tile_tokens queries x packed
// heads each) of consecutive queries of one sequence.
struct PromptUnit {
  int32_t q0, q_end;     // first query token (packed index); end of the sequence's tokens
  int32_t kv0, kv_len;   // the sequence's keys
  int32_t sees;          // keys that query q0 attends to (causal; may be <= 0)
  int32_t head0;         // first query head
  int32_t n[2];          // steps of 128 keys of tile a and b (0: the tile sees no key)
  int32_t two;           // the unit has a tile b
  // A unit may be one part of a block's keys: kv0, kv_len and sees then count
  // from the part's first key, n its steps.
  int32_t parts, part;   // 1, 0: the whole
  int32_t first;         // first of the block's 2 x parts workspace slots (tile t of part k: 2 k + t)
};
static_assert(sizeof(PromptUnit) == 48, "unit layout");

struct PromptParams {
  CUtensorMap tm_q, tm_k, tm_v;   // [token][head][d], boxes {64, packed, tile_tokens} and {64, 1, 128}
  HeadsView q, k, v;
  HeadsOut o;
  float* lse;
  const PromptUnit* units;
  const int32_t* cta_begin;       // [grid + 1]
  float* work;                    // slots of 128 rows: O [d / 4][128][4], exponents' reference [128], sums [128]
  const PromptUnit* joins;        // the blocks that are cut, their part 0
  int32_t heads, group;           // group: query heads of one key/value head
  int32_t packed, tile_tokens;
  int32_t causal;
  float scale_log2;
  unsigned int* status;
  uint64_t timeout_ns;
};

// Launch so that the kernel may start while the one before it in the stream is
// still finishing: it sets itself up (barriers, tensor memory, its place on an
// SM) and calls stream_wait() before it touches what others wrote.
template <typename P>
inline bsp_status launch_overlapped(void (*kernel)(P), dim3 grid, int threads, int smem, cudaStream_t stream,
                                    const P& params, const char* what) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_check(cudaLaunchKernelEx(&cfg, kernel, params), what);
}

}  // namespace bsp

struct bsp_prompt_plan {
  bsp_device* dev = nullptr;
  int ordinal = 0;
  int32_t n_seqs = 0, heads = 0, kv_heads = 0, d = 0, causal = 0;
  int64_t q_tokens = 0, kv_tokens = 0;
  int32_t packed = 1, tile_tokens = 128;
  int32_t grid = 0, smem_bytes = 0;
  int64_t n_units = 0, n_tiles = 0;
  uint64_t timeout_ns = 0;
  int64_t slots = 0;       // workspace slots of the blocks that are cut
  void* d_blob = nullptr;  // units | joins | cta_begin | workspace
  size_t blob_bytes = 0;
  bsp::PromptUnit* d_units = nullptr;
  int32_t* d_cta_begin = nullptr;
  bsp::PromptUnit* d_joins = nullptr;
  float* d_work = nullptr;
  std::vector<bsp::PromptUnit> h_units, h_joins;
  std::vector<int32_t> h_cta_begin;
};

struct bsp_decode_plan {
  bsp_device* dev = nullptr;
  int ordinal = 0;
  int32_t max_seqs = 0, heads = 0, kv_heads = 0, d = 0, page = 0;
  int32_t grid = 0, smem_bytes = 0;
  uint64_t timeout_ns = 0;
  void* d_blob = nullptr;  // counters | partial results
  size_t blob_bytes = 0;
  int32_t* d_counters = nullptr;
  float* d_work = nullptr;
};

namespace bsp {
bsp_status launch_rope_table(bsp_device* dev, int64_t n_pos, int32_t rot, double base, const bsp_rope_scaling& sc,
                             float* table, cudaStream_t stream);
bsp_status launch_rope(RopeParams& p, bsp_dtype type, int sm_count, cudaStream_t stream);
bsp_status launch_append(AppendParams& p, bsp_device* dev, cudaStream_t stream);
// one-time settings of the kernel that a plan launches
bsp_status prepare_prompt(const bsp_prompt_plan* plan);
bsp_status prepare_decode(const bsp_decode_plan* plan);
bsp_status launch_decode(const bsp_decode_plan* plan, DecodeParams& p, cudaStream_t stream);
int32_t decode_ctas(const bsp_device* dev, int d, int group);
int64_t decode_work_floats(int32_t ctas, int32_t d);
int decode_smem_bytes(int d, int group);
bsp_status plan_prompt_host(bsp_prompt_plan* p, const int32_t* q_lens, const int32_t* kv_lens, int sm_count,
                            const bsp_spmm_opts* opts);
bsp_status launch_prompt(const bsp_prompt_plan* plan, PromptParams& p, cudaStream_t stream);
int prompt_smem_bytes(int d);
__host__ __device__ constexpr int64_t prompt_slot_floats(int d) { return 128 * (static_cast<int64_t>(d) + 2); }
}  // namespace bsp
