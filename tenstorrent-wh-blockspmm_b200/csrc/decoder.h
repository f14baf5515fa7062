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
  unsigned int* status;
};

struct DecodeParams {
  HeadsView q;
  HeadsOut o;
  float* lse;
  bsp_kv_cache cache;
  const int32_t* lens;
  const int32_t* page_table;
  int64_t table_stride, table_width;
  int32_t n_seqs, heads;
  float scale;
  unsigned int* status;
};

struct PromptSeq {
  int32_t q0, q_len;    // query tokens [q0, q0 + q_len)
  int32_t kv0, kv_len;
};

struct PromptParams {
  HeadsView q, k, v;
  HeadsOut o;
  float* lse;
  const PromptSeq* seqs;
  int32_t n_seqs, heads, kv_heads, d, causal;
  int32_t tokens;
  float scale;
};

}  // namespace bsp

struct bsp_prompt_plan {
  bsp_device* dev = nullptr;
  int32_t n_seqs = 0, heads = 0, kv_heads = 0, d = 0, causal = 0;
  int64_t q_tokens = 0, kv_tokens = 0;
  int32_t grid = 0;
  int64_t n_units = 0;
  void* d_blob = nullptr;
  size_t blob_bytes = 0;
  bsp::PromptSeq* d_seqs = nullptr;
  std::vector<bsp::PromptSeq> h_seqs;
};

struct bsp_decode_plan {
  bsp_device* dev = nullptr;
  int32_t max_seqs = 0, heads = 0, kv_heads = 0, d = 0, page = 0;
};

namespace bsp {
bsp_status launch_rope_table(bsp_device* dev, int64_t n_pos, int32_t rot, double base, const bsp_rope_scaling& sc,
                             float* table, cudaStream_t stream);
bsp_status launch_rope(const RopeParams& p, bsp_dtype type, cudaStream_t stream);
bsp_status launch_append(const AppendParams& p, cudaStream_t stream);
bsp_status launch_decode(const bsp_decode_plan* plan, const DecodeParams& p, cudaStream_t stream);
bsp_status launch_prompt(const bsp_prompt_plan* plan, const PromptParams& p, cudaStream_t stream);
}  // namespace bsp
