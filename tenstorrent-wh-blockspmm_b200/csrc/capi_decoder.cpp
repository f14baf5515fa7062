// C ABI of the decoder-attention operators (declared in include/bsp.h).
#include <math.h>

#include <algorithm>
#include <cstring>
#include <exception>
#include <mutex>
#include <new>

#include "bsp_testing.h"
#include "decoder.h"

using namespace bsp;

namespace {

constexpr int64_t kMaxTokens = 0x7FFFFFFF;

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// A [tokens][heads][d] operand of `size`-byte elements: 16-byte vectors are
// loaded from every head of every token.
bsp_status check_heads(const char* name, const void* p, int64_t token, int64_t head, int size) {
  if (!p) return set_error(BSP_ERR_INVALID_ARG, std::string(name) + " is null");
  if (!aligned16(p) || (token * size) % 16 || (head * size) % 16)
    return set_error(BSP_ERR_INVALID_ARG, std::string(name) + " must be 16-byte aligned with strides of 16-byte multiples");
  if (token < 0 || head < 0) return set_error(BSP_ERR_INVALID_ARG, std::string(name) + ": negative stride");
  return BSP_OK;
}

bsp_status check_cache(const bsp_kv_cache* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return set_error(BSP_ERR_INVALID_ARG, "null cache");
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128)
    return set_error(BSP_ERR_INVALID_ARG, "a cache page holds 16, 32, 64 or 128 tokens");
  if (c->d != 64 && c->d != 128) return set_error(BSP_ERR_INVALID_ARG, "head size must be 64 or 128");
  if (c->kv_heads < 1 || c->n_pages < 1 || c->n_pages > kMaxTokens)
    return set_error(BSP_ERR_INVALID_ARG, "bad cache dimensions");
  const int64_t block = static_cast<int64_t>(c->page) * c->d;
  if (c->page_stride % 16 || c->head_stride % 16 || c->page_stride < block || c->head_stride < block)
    return set_error(BSP_ERR_INVALID_ARG, "cache strides must be multiples of 16 bytes that hold a page of one head");
  if (!aligned16(c->k) || !aligned16(c->v))
    return set_error(BSP_ERR_INVALID_ARG, "cache pointers must be 16-byte aligned");
  return BSP_OK;
}

bsp_status check_rot(int32_t d, int32_t rot, int32_t layout) {
  if (rot < 16 || rot % 16 || rot > d) return set_error(BSP_ERR_INVALID_ARG, "rot must be a multiple of 16 in [16, d]");
  if (layout != BSP_ROPE_HALF && layout != BSP_ROPE_INTERLEAVED)
    return set_error(BSP_ERR_INVALID_ARG, "unknown rotary layout");
  return BSP_OK;
}

bsp_status check_attention_heads(int32_t heads, int32_t kv_heads, int32_t d) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads)
    return set_error(BSP_ERR_INVALID_ARG, "heads must be a positive multiple of kv_heads");
  if (d != 64 && d != 128) return set_error(BSP_ERR_INVALID_ARG, "head size must be 64 or 128");
  return BSP_OK;
}

// The prompt and decode plans come and go with a batch: their memory comes from
// a pool per GPU that keeps what is freed (microseconds, where cudaMalloc takes
// up to milliseconds).  It belongs to the process: plans may outlive the
// bsp_device they were made with.
constexpr int kMaxGpus = 64;
std::mutex g_pool_mutex;
cudaMemPool_t g_pools[kMaxGpus] = {};

// `bytes` of the pool, ready on every stream once the legacy stream has been
// synchronised (the callers do, behind their copies).
bsp_status plan_alloc(int ordinal, size_t bytes, void** out) {
  *out = nullptr;
  if (ordinal < 0 || ordinal >= kMaxGpus) return set_error(BSP_ERR_UNSUPPORTED, "GPU ordinal out of range");
  std::lock_guard<std::mutex> lock(g_pool_mutex);
  cudaMemPool_t& pool = g_pools[ordinal];
  if (!pool) {
    cudaMemPoolProps props{};
    props.allocType = cudaMemAllocationTypePinned;
    props.location.type = cudaMemLocationTypeDevice;
    props.location.id = ordinal;
    const bsp_status s = cuda_check(cudaMemPoolCreate(&pool, &props), "cudaMemPoolCreate");
    if (s != BSP_OK) {
      pool = nullptr;
      return s;
    }
    uint64_t keep = UINT64_MAX;
    cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep);
  }
  if (cudaMallocFromPoolAsync(out, bytes, pool, nullptr) != cudaSuccess) {
    *out = nullptr;
    cudaGetLastError();
    return set_error(BSP_ERR_ALLOC, "device memory of the plan");
  }
  return BSP_OK;
}
// Launches of the plan may be on any stream: wait for the device, as cudaFree does.
void plan_free(int ordinal, void* p) {
  if (!p) return;
  OnDevice on(ordinal);
  cudaDeviceSynchronize();
  cudaFreeAsync(p, nullptr);
}

}  // namespace

void bsp::trim_plan_pool(int ordinal) {
  std::lock_guard<std::mutex> lock(g_pool_mutex);
  if (ordinal >= 0 && ordinal < kMaxGpus && g_pools[ordinal]) cudaMemPoolTrimTo(g_pools[ordinal], 0);
}

extern "C" {

bsp_status bsp_rope_table(bsp_device* dev, int64_t n_pos, int32_t rot, double base, const bsp_rope_scaling* scaling,
                          float* table, void* stream) {
  if (!dev || !table) return set_error(BSP_ERR_INVALID_ARG, "null argument");
  if (!aligned16(table)) return set_error(BSP_ERR_INVALID_ARG, "the table must be 16-byte aligned");
  if (n_pos < 1 || n_pos > kMaxTokens) return set_error(BSP_ERR_INVALID_ARG, "n_pos out of range");
  bsp_status s = check_rot(512, rot, BSP_ROPE_HALF);
  if (s != BSP_OK) return s;
  if (!(base > 0) || !std::isfinite(base)) return set_error(BSP_ERR_INVALID_ARG, "base must be positive");
  bsp_rope_scaling sc{};
  if (scaling) sc = *scaling;
  if (sc.kind < BSP_ROPE_NONE || sc.kind > BSP_ROPE_PARTS) return set_error(BSP_ERR_INVALID_ARG, "unknown scaling kind");
  if (sc.kind != BSP_ROPE_NONE && (!(sc.factor > 0) || !std::isfinite(sc.factor)))
    return set_error(BSP_ERR_INVALID_ARG, "the scaling factor must be positive");
  if (sc.kind == BSP_ROPE_PARTS && (!(sc.context > 0) || !(sc.fast > sc.slow)))
    return set_error(BSP_ERR_INVALID_ARG, "by parts: context > 0 and fast > slow");
  if (!std::isfinite(sc.magnitude) || sc.magnitude < 0) return set_error(BSP_ERR_INVALID_ARG, "bad magnitude");
  if (sc.magnitude == 0) sc.magnitude = 1;
  OnDevice on(dev->ordinal);
  return launch_rope_table(dev, n_pos, rot, base, sc, table, static_cast<cudaStream_t>(stream));
}

bsp_status bsp_rope(bsp_device* dev, const void* x, int64_t x_token, int64_t x_head, const int32_t* positions,
                    const float* table, int64_t n_pos, int64_t tokens, int32_t heads, int32_t d, int32_t rot,
                    bsp_rope_layout layout, int32_t transpose, bsp_dtype type, void* y, int64_t y_token,
                    int64_t y_head, void* stream) {
  if (!dev) return set_error(BSP_ERR_INVALID_ARG, "null device");
  if (type != BSP_BF16 && type != BSP_F32) return set_error(BSP_ERR_INVALID_ARG, "type must be BSP_BF16 or BSP_F32");
  if (tokens < 0 || heads < 1 || tokens > kMaxTokens / heads || n_pos < 0)
    return set_error(BSP_ERR_INVALID_ARG, "bad dimensions");
  if (d < 16 || d % 16 || d > 512) return set_error(BSP_ERR_INVALID_ARG, "d must be a multiple of 16, at most 512");
  bsp_status s = check_rot(d, rot, layout);
  if (s != BSP_OK) return s;
  if (tokens == 0) return BSP_OK;
  const int size = type == BSP_F32 ? 4 : 2;
  if ((s = check_heads("x", x, x_token, x_head, size)) != BSP_OK) return s;
  if ((s = check_heads("y", y, y_token, y_head, size)) != BSP_OK) return s;
  if (!positions || !table || !aligned16(table)) return set_error(BSP_ERR_INVALID_ARG, "positions or table missing");
  RopeParams p{};
  p.x = {x, x_token, x_head};
  p.y = {y, y_token, y_head};
  p.positions = positions;
  p.table = reinterpret_cast<const float2*>(table);
  p.n_pos = n_pos;
  p.tokens = tokens;
  p.heads = heads;
  p.d = d;
  p.rot = rot;
  p.interleaved = layout == BSP_ROPE_INTERLEAVED;
  p.sign = transpose ? -1.f : 1.f;
  p.status = dev->d_status;
  OnDevice on(dev->ordinal);
  return launch_rope(p, type, dev->sm_count, static_cast<cudaStream_t>(stream));
}

bsp_status bsp_kv_append(bsp_device* dev, const bsp_kv_cache* cache, const void* k, int64_t k_token, int64_t k_head,
                         const void* v, int64_t v_token, int64_t v_head, int64_t tokens, int32_t n_seqs,
                         const int32_t* starts, const int32_t* before, const int32_t* page_table,
                         int64_t table_stride, int64_t table_width, const float* table, int64_t n_pos, int32_t rot,
                         bsp_rope_layout layout, const void* q, int64_t q_token, int64_t q_head, int32_t heads,
                         void* q_out, int64_t qo_token, int64_t qo_head, void* k_out, int64_t ko_token,
                         int64_t ko_head, void* stream) {
  if (!dev) return set_error(BSP_ERR_INVALID_ARG, "null device");
  bsp_status s = check_cache(cache);
  if (s != BSP_OK) return s;
  if (tokens < 0 || tokens > kMaxTokens || n_seqs < 0 || table_width < 0 || table_stride < 0 || n_pos < 0)
    return set_error(BSP_ERR_INVALID_ARG, "bad dimensions");
  if (table) {
    if ((s = check_rot(cache->d, rot, layout)) != BSP_OK) return s;
    if (!aligned16(table)) return set_error(BSP_ERR_INVALID_ARG, "the table must be 16-byte aligned");
  } else if (q || k_out) {
    return set_error(BSP_ERR_INVALID_ARG, "q and k_out are rotated outputs: they need a rotary table");
  }
  if (tokens == 0 || n_seqs == 0) return BSP_OK;
  if ((s = check_heads("k", k, k_token, k_head, 2)) != BSP_OK) return s;
  if ((s = check_heads("v", v, v_token, v_head, 2)) != BSP_OK) return s;
  if (q) {
    if (heads < 1) return set_error(BSP_ERR_INVALID_ARG, "bad number of query heads");
    if ((s = check_heads("q", q, q_token, q_head, 2)) != BSP_OK) return s;
    if ((s = check_heads("q_out", q_out, qo_token, qo_head, 2)) != BSP_OK) return s;
  }
  if (2 * static_cast<int64_t>(cache->kv_heads) + (q ? heads : 0) > 65000)
    return set_error(BSP_ERR_UNSUPPORTED, "too many heads");
  if (k_out && (s = check_heads("k_out", k_out, ko_token, ko_head, 2)) != BSP_OK) return s;
  if (!starts || !before || !page_table) return set_error(BSP_ERR_INVALID_ARG, "null index array");
  AppendParams p{};
  p.q = {q, q_token, q_head};
  p.k = {k, k_token, k_head};
  p.v = {v, v_token, v_head};
  p.q_out = {q_out, qo_token, qo_head};
  p.k_out = {k_out, ko_token, ko_head};
  p.cache = *cache;
  p.starts = starts;
  p.before = before;
  p.page_table = page_table;
  p.table_stride = table_stride;
  p.table_width = table_width;
  p.table = reinterpret_cast<const float2*>(table);
  p.n_pos = n_pos;
  p.tokens = tokens;
  p.n_seqs = n_seqs;
  p.heads = heads;
  p.rot = rot;
  p.interleaved = layout == BSP_ROPE_INTERLEAVED;
  p.status = dev->d_status;
  OnDevice on(dev->ordinal);
  return launch_append(p, dev, static_cast<cudaStream_t>(stream));
}

bsp_status bsp_prompt_plan_create(bsp_device* dev, int32_t n_seqs, const int32_t* q_lens, const int32_t* kv_lens,
                                  int32_t heads, int32_t kv_heads, int32_t d, int32_t causal,
                                  const bsp_spmm_opts* opts, bsp_prompt_plan** out) {
  if (!out) return set_error(BSP_ERR_INVALID_ARG, "null argument");
  *out = nullptr;
  if (!dev) return set_error(BSP_ERR_INVALID_ARG, "null device");
  if (n_seqs < 0 || (n_seqs > 0 && (!q_lens || !kv_lens))) return set_error(BSP_ERR_INVALID_ARG, "bad lengths");
  bsp_status s = check_attention_heads(heads, kv_heads, d);
  if (s != BSP_OK) return s;
  (void)opts;
  bsp_prompt_plan* p = new (std::nothrow) bsp_prompt_plan();
  if (!p) return set_error(BSP_ERR_ALLOC, "host allocation failed");
  p->dev = dev;
  p->ordinal = dev->ordinal;
  p->n_seqs = n_seqs;
  p->heads = heads;
  p->kv_heads = kv_heads;
  p->d = d;
  p->causal = causal != 0;
  try {
    s = plan_prompt_host(p, q_lens, kv_lens, dev->sm_count, opts);
  } catch (const std::exception&) {
    s = set_error(BSP_ERR_ALLOC, "host allocation failed");
  }
  p->smem_bytes = prompt_smem_bytes(d);
  if (s == BSP_OK && p->n_units > 0) {
    OnDevice on(dev->ordinal);
    const size_t ub = p->h_units.size() * sizeof(PromptUnit), jb = p->h_joins.size() * sizeof(PromptUnit);
    const size_t cb = p->h_cta_begin.size() * sizeof(int32_t), tables = (ub + jb + cb + 255) / 256 * 256;
    p->blob_bytes = tables + static_cast<size_t>(p->slots * prompt_slot_floats(d)) * sizeof(float);
    s = plan_alloc(dev->ordinal, p->blob_bytes, &p->d_blob);
    if (s == BSP_OK) {
      uint8_t* at = static_cast<uint8_t*>(p->d_blob);
      p->d_units = reinterpret_cast<PromptUnit*>(at);
      p->d_joins = reinterpret_cast<PromptUnit*>(at + ub);
      p->d_cta_begin = reinterpret_cast<int32_t*>(at + ub + jb);
      p->d_work = reinterpret_cast<float*>(at + tables);
      auto upload = [&](void* dst, const void* src, size_t bytes) {
        if (s == BSP_OK && bytes > 0)
          s = cuda_check(cudaMemcpyAsync(dst, src, bytes, cudaMemcpyHostToDevice, nullptr), "upload plan tables");
      };
      upload(p->d_units, p->h_units.data(), ub);
      upload(p->d_joins, p->h_joins.data(), jb);
      upload(p->d_cta_begin, p->h_cta_begin.data(), cb);
      if (s == BSP_OK) s = cuda_check(cudaStreamSynchronize(nullptr), "upload plan tables");
      if (s == BSP_OK) s = prepare_prompt(p);
    }
  }
  if (s != BSP_OK) {
    bsp_prompt_plan_destroy(p);
    return s;
  }
  *out = p;
  return BSP_OK;
}

bsp_status bsp_prompt_execute(const bsp_prompt_plan* plan, const void* q, int64_t q_token, int64_t q_head,
                              const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token,
                              int64_t v_head, float scale, void* o, int64_t o_token, int64_t o_head, float* lse,
                              void* stream) {
  if (!plan) return set_error(BSP_ERR_INVALID_ARG, "null plan");
  if (!(scale > 0) || !std::isfinite(scale)) return set_error(BSP_ERR_INVALID_ARG, "scale must be positive");
  if (plan->q_tokens == 0) return BSP_OK;
  bsp_status s = check_heads("q", q, q_token, q_head, 2);
  if (s == BSP_OK) s = check_heads("o", o, o_token, o_head, 2);
  if (s == BSP_OK && plan->kv_tokens > 0) {
    s = check_heads("k", k, k_token, k_head, 2);
    if (s == BSP_OK) s = check_heads("v", v, v_token, v_head, 2);
  }
  if (s != BSP_OK) return s;
  PromptParams p{};
  p.q = {q, q_token, q_head};
  p.k = {k, k_token, k_head};
  p.v = {v, v_token, v_head};
  p.o = {o, o_token, o_head};
  p.lse = lse;
  p.units = plan->d_units;
  p.cta_begin = plan->d_cta_begin;
  p.work = plan->d_work;
  p.joins = plan->d_joins;
  p.heads = plan->heads;
  p.group = plan->heads / plan->kv_heads;
  p.packed = plan->packed;
  p.tile_tokens = plan->tile_tokens;
  p.causal = plan->causal;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.status = plan->dev->d_status;
  p.timeout_ns = plan->timeout_ns;
  OnDevice on(plan->dev->ordinal);
  return launch_prompt(plan, p, static_cast<cudaStream_t>(stream));
}

bsp_status bsp_prompt_plan_destroy(bsp_prompt_plan* plan) {
  if (!plan) return BSP_OK;
  plan_free(plan->ordinal, plan->d_blob);
  delete plan;
  return BSP_OK;
}

bsp_status bsp_prompt_plan_info(const bsp_prompt_plan* p, int64_t info[16]) {
  if (!p || !info) return set_error(BSP_ERR_INVALID_ARG, "null argument");
  memset(info, 0, sizeof(int64_t) * 16);
  info[0] = p->n_units;
  info[1] = p->grid;
  info[2] = p->q_tokens;
  info[3] = p->kv_tokens;
  info[4] = p->heads;
  info[5] = p->kv_heads;
  info[6] = p->d;
  info[7] = p->n_tiles;
  info[8] = static_cast<int64_t>(p->blob_bytes);
  info[9] = p->smem_bytes;
  info[10] = 512;
  info[11] = p->packed;
  info[12] = p->slots * prompt_slot_floats(p->d) * static_cast<int64_t>(sizeof(float));
  return BSP_OK;
}

bsp_status bsp_prompt_plan_inspect(int32_t n_seqs, const int32_t* q_lens, const int32_t* kv_lens, int32_t heads,
                                   int32_t kv_heads, int32_t d, int32_t causal, const bsp_spmm_opts* opts,
                                   int32_t sm_count, int64_t info[16], int32_t* units_out, int32_t* cta_begin_out) {
  if (n_seqs < 0 || (n_seqs > 0 && (!q_lens || !kv_lens)) || !info || sm_count < 1)
    return set_error(BSP_ERR_INVALID_ARG, "bad arguments");
  bsp_status s = check_attention_heads(heads, kv_heads, d);
  if (s != BSP_OK) return s;
  bsp_prompt_plan p;
  p.n_seqs = n_seqs;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.d = d;
  p.causal = causal != 0;
  try {
    s = plan_prompt_host(&p, q_lens, kv_lens, sm_count, opts);
  } catch (const std::exception&) {
    s = set_error(BSP_ERR_ALLOC, "host allocation failed");
  }
  if (s != BSP_OK) return s;
  bsp_prompt_plan_info(&p, info);
  if (units_out && !p.h_units.empty()) memcpy(units_out, p.h_units.data(), p.h_units.size() * sizeof(PromptUnit));
  if (cta_begin_out) memcpy(cta_begin_out, p.h_cta_begin.data(), p.h_cta_begin.size() * sizeof(int32_t));
  return BSP_OK;
}

bsp_status bsp_decode_plan_create(bsp_device* dev, int32_t max_seqs, int32_t heads, int32_t kv_heads, int32_t d,
                                  int32_t page, const bsp_spmm_opts* opts, bsp_decode_plan** out) {
  if (!out) return set_error(BSP_ERR_INVALID_ARG, "null argument");
  *out = nullptr;
  if (!dev) return set_error(BSP_ERR_INVALID_ARG, "null device");
  if (max_seqs < 0) return set_error(BSP_ERR_INVALID_ARG, "bad max_seqs");
  bsp_status s = check_attention_heads(heads, kv_heads, d);
  if (s != BSP_OK) return s;
  if (page != 16 && page != 32 && page != 64 && page != 128)
    return set_error(BSP_ERR_INVALID_ARG, "a cache page holds 16, 32, 64 or 128 tokens");
  bsp_decode_plan* p = new (std::nothrow) bsp_decode_plan();
  if (!p) return set_error(BSP_ERR_ALLOC, "host allocation failed");
  p->dev = dev;
  p->ordinal = dev->ordinal;
  p->max_seqs = max_seqs;
  p->heads = heads;
  p->kv_heads = kv_heads;
  p->d = d;
  p->page = page;
  p->grid = decode_ctas(dev, d, heads / kv_heads);
  if (opts && opts->max_ctas > 0) p->grid = std::min(p->grid, opts->max_ctas);
  p->smem_bytes = decode_smem_bytes(d, heads / kv_heads);
  p->timeout_ns = static_cast<uint64_t>(opts && opts->timeout_ms > 0 ? opts->timeout_ms : 2000) * 1000000ull;
  OnDevice on(dev->ordinal);
  const size_t counters = (sizeof(int32_t) * p->grid + 255) / 256 * 256;
  p->blob_bytes = counters + sizeof(float) * decode_work_floats(p->grid, d);
  s = plan_alloc(dev->ordinal, p->blob_bytes, &p->d_blob);
  if (s != BSP_OK) {
    delete p;
    return s;
  }
  p->d_counters = static_cast<int32_t*>(p->d_blob);
  p->d_work = reinterpret_cast<float*>(static_cast<uint8_t*>(p->d_blob) + counters);
  s = cuda_check(cudaMemsetAsync(p->d_counters, 0, counters, nullptr), "clear the decode counters");
  if (s == BSP_OK) s = prepare_decode(p);
  // the clearing ran on the legacy stream: executes may come on any other
  if (s == BSP_OK) s = cuda_check(cudaStreamSynchronize(nullptr), "clear the decode counters");
  if (s != BSP_OK) {
    bsp_decode_plan_destroy(p);
    return s;
  }
  *out = p;
  return BSP_OK;
}

bsp_status bsp_decode_execute(const bsp_decode_plan* plan, const bsp_kv_cache* cache, const void* q, int64_t q_token,
                              int64_t q_head, int32_t n_seqs, const int32_t* lens, const int32_t* page_table,
                              int64_t table_stride, int64_t table_width, float scale, void* o, int64_t o_token,
                              int64_t o_head, float* lse, void* stream) {
  if (!plan) return set_error(BSP_ERR_INVALID_ARG, "null plan");
  bsp_status s = check_cache(cache);
  if (s != BSP_OK) return s;
  if (cache->kv_heads != plan->kv_heads || cache->d != plan->d || cache->page != plan->page)
    return set_error(BSP_ERR_INVALID_ARG, "the cache differs from the plan's heads, head size or page");
  if (n_seqs < 0 || n_seqs > plan->max_seqs) return set_error(BSP_ERR_INVALID_ARG, "more sequences than the plan holds");
  if (!(scale > 0) || !std::isfinite(scale)) return set_error(BSP_ERR_INVALID_ARG, "scale must be positive");
  if (table_width < 0 || table_width > kMaxTokens || table_stride < 0)
    return set_error(BSP_ERR_INVALID_ARG, "bad page table");
  if (n_seqs == 0) return BSP_OK;
  if ((s = check_heads("q", q, q_token, q_head, 2)) != BSP_OK) return s;
  if ((s = check_heads("o", o, o_token, o_head, 2)) != BSP_OK) return s;
  if (!lens || !page_table) return set_error(BSP_ERR_INVALID_ARG, "null index array");
  DecodeParams p{};
  p.q = {q, q_token, q_head};
  p.o = {o, o_token, o_head};
  p.lse = lse;
  p.cache = *cache;
  p.lens = lens;
  p.page_table = page_table;
  p.table_stride = table_stride;
  p.max_len = static_cast<int32_t>(std::min<int64_t>(table_width * plan->page, 0x7FFFFF00));
  p.n_seqs = n_seqs;
  p.heads = plan->heads;
  p.group = plan->heads / plan->kv_heads;
  p.chunks = (p.group + 15) / 16;
  p.streams = plan->kv_heads * p.chunks;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.work = plan->d_work;
  p.counters = plan->d_counters;
  p.status = plan->dev->d_status;
  p.timeout_ns = plan->timeout_ns;
  OnDevice on(plan->dev->ordinal);
  return launch_decode(plan, p, static_cast<cudaStream_t>(stream));
}

bsp_status bsp_decode_plan_destroy(bsp_decode_plan* plan) {
  if (!plan) return BSP_OK;
  plan_free(plan->ordinal, plan->d_blob);
  delete plan;
  return BSP_OK;
}

bsp_status bsp_decode_plan_info(const bsp_decode_plan* p, int64_t info[16]) {
  if (!p || !info) return set_error(BSP_ERR_INVALID_ARG, "null argument");
  memset(info, 0, sizeof(int64_t) * 16);
  info[0] = p->max_seqs;
  info[1] = p->grid;
  info[2] = p->heads;
  info[3] = p->kv_heads;
  info[4] = p->d;
  info[5] = p->page;
  info[8] = static_cast<int64_t>(p->blob_bytes);
  info[9] = p->smem_bytes;
  return BSP_OK;
}

}  // extern "C"
