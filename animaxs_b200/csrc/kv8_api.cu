// kv8_api.cu -- C ABI of the 8-bit K/V cache (declared in include/animaxs_attn.h):
// argument checks, workspaces and launches of kv8_cache.cu, kv8_rows_sm100.cu
// and kv8_attn_sm100.cu.
#include <cuda_runtime.h>

#include <cmath>
#include <initializer_list>

#include "../../include/animaxs_attn.h"
#include "api_internal.h"
#include "kernels.h"

namespace {

struct DeviceScope {
  int prev = 0, dev = 0;
  explicit DeviceScope(int d) : dev(d) {
    cudaGetDevice(&prev);
    if (prev != dev) cudaSetDevice(dev);
  }
  ~DeviceScope() {
    if (prev != dev) cudaSetDevice(prev);
  }
};

// Positions are numbered in 32 bits up to the end of the last block.
constexpr int kMaxCapacity = 0x7fffffff - ax::kKv8Block;

bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

int check_cache(animaxs_attn_ctx* ctx, const animaxs_kv8_cache* c) {
  if (c == nullptr) return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "null K/V cache");
  if (c->batch <= 0 || c->capacity <= 0 || c->kv_heads <= 0)
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "8-bit K/V cache sizes must be positive");
  if (c->head_dim != 64 && c->head_dim != 128)
    return ax_set_error(ctx, ANIMAXS_ERR_UNSUPPORTED, "8-bit K/V cache requires headDim 64 or 128 (got %d)",
                        c->head_dim);
  if (c->format != ANIMAXS_KV8_INT8 && c->format != ANIMAXS_KV8_E4M3)
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "unknown 8-bit K/V cache format %d", c->format);
  if (c->capacity > kMaxCapacity || static_cast<int64_t>(c->batch) * c->kv_heads > 0x7fffffffLL ||
      static_cast<__int128>(c->batch) * c->kv_heads * c->capacity * c->head_dim > (static_cast<__int128>(1) << 46))
    return ax_set_error(ctx, ANIMAXS_ERR_OVERFLOW, "attention byte size overflow");
  if (c->k_codes == nullptr || c->v_codes == nullptr || c->k_scale == nullptr || c->v_scale == nullptr)
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "8-bit K/V cache buffers must not be null");
  if (misaligned(c->k_codes) || misaligned(c->v_codes) || reinterpret_cast<uintptr_t>(c->k_scale) % 4 ||
      reinterpret_cast<uintptr_t>(c->v_scale) % 4)
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG,
                        "8-bit K/V cache codes must be 16-byte aligned and scales 4-byte aligned");
  return ANIMAXS_OK;
}

// Optional DEVICE int32 arrays, one value per sequence.
int check_ints(animaxs_attn_ctx* ctx, std::initializer_list<const int32_t*> arrays) {
  for (const int32_t* a : arrays)
    if (reinterpret_cast<uintptr_t>(a) % 4 != 0)
      return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "lengths, starts and counts must be 4-byte aligned");
  return ANIMAXS_OK;
}

// Strides of an fp16 [batch][tokens][heads][dim] view.
int check_strides(animaxs_attn_ctx* ctx, std::initializer_list<int64_t> strides) {
  for (int64_t s : strides) {
    if (s < 0 || s % 8 != 0)
      return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "8-bit K/V cache requires strides that are multiples of 8");
    if (s >= (static_cast<int64_t>(1) << 39))
      return ax_set_error(ctx, ANIMAXS_ERR_OVERFLOW, "attention byte size overflow");
  }
  return ANIMAXS_OK;
}

int check_write(animaxs_attn_ctx* ctx, const animaxs_kv8_cache* c, const animaxs_kv8_write_desc* d, const void* k,
                const void* v) {
  int rc = check_cache(ctx, c);
  if (rc != ANIMAXS_OK) return rc;
  if (d == nullptr || k == nullptr || v == nullptr)
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "8-bit K/V cache write needs a descriptor, k and v");
  if (misaligned(k) || misaligned(v))
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "8-bit K/V cache write requires 16-byte-aligned k and v");
  rc = check_ints(ctx, {d->starts, d->counts});
  if (rc != ANIMAXS_OK) return rc;
  if (d->tokens <= 0) return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "tokens must be positive");
  if (d->starts == nullptr &&
      (d->start < 0 || static_cast<int64_t>(d->start) + (d->counts == nullptr ? d->tokens : 0) > c->capacity))
    return ax_set_error(ctx, ANIMAXS_ERR_OOB, "positions [%d, %lld) outside the cache's capacity %d", d->start,
                        static_cast<long long>(d->start) + d->tokens, c->capacity);
  rc = check_strides(ctx, {d->k_tok_stride, d->k_head_stride, d->k_batch_stride, d->v_tok_stride, d->v_head_stride,
                           d->v_batch_stride});
  if (rc != ANIMAXS_OK) return rc;
  if ((d->tokens > 1 && (d->k_tok_stride == 0 || d->v_tok_stride == 0)) ||
      (c->kv_heads > 1 && (d->k_head_stride == 0 || d->v_head_stride == 0)))
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "token and head strides must not be 0");
  // A CTA for K and one for V of every (sequence, head, block).
  if (2LL * c->batch * c->kv_heads > 0x7fffffffLL / ax::kv8_write_window(d->tokens, c->capacity))
    return ax_set_error(ctx, ANIMAXS_ERR_OVERFLOW, "8-bit K/V cache write of too many blocks for one call");
  return ANIMAXS_OK;
}

int check_attn(animaxs_attn_ctx* ctx, const animaxs_kv8_cache* c, const animaxs_attn_desc* d, const void* q,
               const void* o) {
  int rc = check_cache(ctx, c);
  if (rc != ANIMAXS_OK) return rc;
  if (d == nullptr || q == nullptr || o == nullptr)
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "attention buffers must not be null");
  if (d->batch != c->batch || d->kv_heads != c->kv_heads || d->head_dim != c->head_dim)
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG,
                        "batch, kv heads and headDim (%d, %d, %d) must be the cache's (%d, %d, %d)", d->batch,
                        d->kv_heads, d->head_dim, c->batch, c->kv_heads, c->head_dim);
  if (d->kv_len > c->capacity)
    return ax_set_error(ctx, ANIMAXS_ERR_OOB, "kv_len %d exceeds the cache's capacity %d", d->kv_len, c->capacity);
  if (d->qk_norm == ANIMAXS_QK_RMS_ROPE)
    return ax_set_error(ctx, ANIMAXS_ERR_UNSUPPORTED,
                        "attention over an 8-bit K/V cache rotates nothing: rotate q and k where they are projected");
  if (d->qk_norm == ANIMAXS_QK_RMS && d->qk_norm_targets != ANIMAXS_QK_NORM_Q_ONLY)
    return ax_set_error(ctx, ANIMAXS_ERR_UNSUPPORTED,
                        "attention over an 8-bit K/V cache normalises q only (K is normalised before it is written)");
  if (d->numerics == ANIMAXS_NUMERICS_FP32_SCORES_AND_SOFTMAX)
    return ax_set_error(ctx, ANIMAXS_ERR_UNSUPPORTED, "attention over an 8-bit K/V cache has LEGACY numerics only");
  rc = check_ints(ctx, {d->kv_valid_lens});
  if (rc != ANIMAXS_OK) return rc;
  if (ctx != nullptr && ctx->score_probe != nullptr)
    return ax_set_error(ctx, ANIMAXS_ERR_UNSUPPORTED, "the score probe does not read an 8-bit K/V cache");
  if (d->batch > 1 && d->o_batch_stride == 0)
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "invalid attention shape, offset, or causal dimensions");
  // The rest as animaxs_attn_forward checks it, with the cache in place of k
  // and v, and any q_len beside any kv_len.
  animaxs_attn_desc r = *d;
  r.causal = 0;
  r.k_tok_stride = r.v_tok_stride = d->head_dim;
  r.k_head_stride = r.v_head_stride = static_cast<int64_t>(c->capacity) * d->head_dim;
  r.k_batch_stride = r.v_batch_stride = 0;
  r.k_bytes = r.v_bytes = 0;
  rc = ax_validate(ctx, &r, q, c->k_codes, c->v_codes, o);
  if (rc != ANIMAXS_OK) return rc;
  // A kv head's query rows are numbered in 32 bits, up to the end of their last pair of tiles.
  if (static_cast<int64_t>(d->heads) * d->q_len > 0x7fffffffLL - 2 * ax::kTileM)
    return ax_set_error(ctx, ANIMAXS_ERR_OVERFLOW, "attention byte size overflow");
  return ANIMAXS_OK;
}

// Workspaces of split attention.  Launches have one CTA per SM at most, which
// bounds both: 2.5 MB for few rows, 39 MB for many.
int ensure_rows_workspace(animaxs_attn_ctx* ctx) {
  if (ctx->kv8_count != nullptr) return ANIMAXS_OK;
  const size_t counts = ctx->num_sms * sizeof(unsigned int);
  unsigned int* count = nullptr;
  cudaError_t e = cudaSuccess;
  if (ctx->kv8_rows_part == nullptr) {
    e = cudaMalloc(&ctx->kv8_rows_part, ax::kv8_rows_part_floats(128, ctx->num_sms) * sizeof(float));
    if (e != cudaSuccess) ctx->kv8_rows_part = nullptr;
  }
  if (e == cudaSuccess) e = cudaMalloc(&count, counts);
  if (e == cudaSuccess) e = cudaMemset(count, 0, counts);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();  // before work on a non-blocking stream counts
  if (e != cudaSuccess) {
    if (count != nullptr) cudaFree(count);
    return ax_cuda_fail(ctx, e, "8-bit K/V cache attention workspace");
  }
  ctx->kv8_count = count;
  return ANIMAXS_OK;
}
int ensure_tile_workspace(animaxs_attn_ctx* ctx) {
  if (ctx->kv8_tile_part != nullptr) return ANIMAXS_OK;
  const cudaError_t e =
      cudaMalloc(&ctx->kv8_tile_part, ax::kv8_attn_part_floats(128, ctx->num_sms) * sizeof(float));
  if (e == cudaSuccess) return ANIMAXS_OK;
  ctx->kv8_tile_part = nullptr;
  return ax_cuda_fail(ctx, e, "8-bit K/V cache attention workspace");
}

}  // namespace

extern "C" int animaxs_kv8_cache_bytes(int batch, int capacity, int kv_heads, int head_dim, int64_t* code_bytes,
                                       int64_t* scale_bytes) {
  if (code_bytes == nullptr || scale_bytes == nullptr || batch <= 0 || capacity <= 0 || kv_heads <= 0)
    return ANIMAXS_ERR_INVALID_ARG;
  if (head_dim != 64 && head_dim != 128) return ANIMAXS_ERR_UNSUPPORTED;
  const __int128 heads = static_cast<__int128>(batch) * kv_heads;
  if (capacity > kMaxCapacity || heads * capacity * head_dim > (static_cast<__int128>(1) << 46))
    return ANIMAXS_ERR_OVERFLOW;
  *code_bytes = static_cast<int64_t>(heads * capacity * head_dim);
  *scale_bytes = static_cast<int64_t>(heads * ((static_cast<int64_t>(capacity) + ax::kKv8Block - 1) / ax::kKv8Block) * 4);
  return ANIMAXS_OK;
}

extern "C" int animaxs_kv8_write_validate(animaxs_attn_ctx* ctx, const animaxs_kv8_cache* cache,
                                          const animaxs_kv8_write_desc* desc, const void* k, const void* v) {
  const int rc = check_write(ctx, cache, desc, k, v);
  if (rc == ANIMAXS_OK && ctx != nullptr) ctx->last_error.clear();
  return rc;
}

extern "C" int animaxs_kv8_write(animaxs_attn_ctx* ctx, const animaxs_kv8_cache* cache,
                                 const animaxs_kv8_write_desc* d, const void* k, const void* v, void* stream) {
  AxRange range("animaxs_kv8_write");
  if (ctx == nullptr) return ANIMAXS_ERR_INVALID_ARG;
  const int rc = check_write(ctx, cache, d, k, v);
  if (rc != ANIMAXS_OK) return rc;
  DeviceScope scope(ctx->device);
  ax::Kv8WriteParams p{};
  p.format = cache->format;
  p.head_dim = cache->head_dim;
  p.batch = cache->batch;
  p.kv_heads = cache->kv_heads;
  p.capacity = cache->capacity;
  p.tokens = d->tokens;
  p.start = d->start;
  p.starts = d->starts;
  p.counts = d->counts;
  p.src[0] = static_cast<const __half*>(k);
  p.src[1] = static_cast<const __half*>(v);
  p.tok[0] = d->k_tok_stride;
  p.tok[1] = d->v_tok_stride;
  p.head[0] = d->k_head_stride;
  p.head[1] = d->v_head_stride;
  p.bat[0] = d->k_batch_stride;
  p.bat[1] = d->v_batch_stride;
  p.codes[0] = static_cast<uint8_t*>(cache->k_codes);
  p.codes[1] = static_cast<uint8_t*>(cache->v_codes);
  p.scale[0] = cache->k_scale;
  p.scale[1] = cache->v_scale;
  const cudaError_t e = ax::launch_kv8_write(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return ax_cuda_fail(ctx, e, "8-bit K/V cache write");
  ctx->last_error.clear();
  return ANIMAXS_OK;
}

extern "C" int animaxs_kv8_read(animaxs_attn_ctx* ctx, const animaxs_kv8_cache* cache, int start, int tokens,
                                const int32_t* lens, void* k_out, void* v_out, int64_t tok_stride,
                                int64_t head_stride, int64_t batch_stride, void* stream) {
  AxRange range("animaxs_kv8_read");
  if (ctx == nullptr) return ANIMAXS_ERR_INVALID_ARG;
  int rc = check_cache(ctx, cache);
  if (rc != ANIMAXS_OK) return rc;
  rc = check_ints(ctx, {lens});
  if (rc != ANIMAXS_OK) return rc;
  if (k_out == nullptr || v_out == nullptr || misaligned(k_out) || misaligned(v_out))
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "8-bit K/V cache read requires 16-byte-aligned outputs");
  if (tokens <= 0) return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "tokens must be positive");
  if (start < 0 || static_cast<int64_t>(start) + tokens > cache->capacity)
    return ax_set_error(ctx, ANIMAXS_ERR_OOB, "positions [%d, %lld) outside the cache's capacity %d", start,
                        static_cast<long long>(start) + tokens, cache->capacity);
  rc = check_strides(ctx, {tok_stride, head_stride, batch_stride});
  if (rc != ANIMAXS_OK) return rc;
  if ((tokens > 1 && tok_stride == 0) || (cache->kv_heads > 1 && head_stride == 0) ||
      (cache->batch > 1 && batch_stride == 0))
    return ax_set_error(ctx, ANIMAXS_ERR_INVALID_ARG, "output strides must not be 0");
  if (2LL * cache->batch * cache->kv_heads > 0x7fffffffLL / ((tokens + ax::kKv8Block - 1LL) / ax::kKv8Block))
    return ax_set_error(ctx, ANIMAXS_ERR_OVERFLOW, "8-bit K/V cache read of too many blocks for one call");
  DeviceScope scope(ctx->device);
  ax::Kv8ReadParams p{};
  p.format = cache->format;
  p.head_dim = cache->head_dim;
  p.batch = cache->batch;
  p.kv_heads = cache->kv_heads;
  p.capacity = cache->capacity;
  p.start = start;
  p.tokens = tokens;
  p.lens = lens;
  p.codes[0] = static_cast<const uint8_t*>(cache->k_codes);
  p.codes[1] = static_cast<const uint8_t*>(cache->v_codes);
  p.scale[0] = cache->k_scale;
  p.scale[1] = cache->v_scale;
  p.out[0] = static_cast<__half*>(k_out);
  p.out[1] = static_cast<__half*>(v_out);
  p.tok = tok_stride;
  p.head = head_stride;
  p.bat = batch_stride;
  const cudaError_t e = ax::launch_kv8_read(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return ax_cuda_fail(ctx, e, "8-bit K/V cache read");
  ctx->last_error.clear();
  return ANIMAXS_OK;
}

extern "C" int animaxs_kv8_attn_validate(animaxs_attn_ctx* ctx, const animaxs_kv8_cache* cache,
                                         const animaxs_attn_desc* desc, const void* q, const void* o) {
  const int rc = check_attn(ctx, cache, desc, q, o);
  if (rc == ANIMAXS_OK && ctx != nullptr) ctx->last_error.clear();
  return rc;
}

extern "C" int animaxs_kv8_attn_forward(animaxs_attn_ctx* ctx, const animaxs_kv8_cache* cache,
                                        const animaxs_attn_desc* d, const void* q, void* o, void* stream) {
  AxRange range("animaxs_kv8_attn_forward");
  if (ctx == nullptr) return ANIMAXS_ERR_INVALID_ARG;
  int rc = check_attn(ctx, cache, d, q, o);
  if (rc != ANIMAXS_OK) return rc;
  DeviceScope scope(ctx->device);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t D = d->head_dim;
  ax::Kv8AttnParams p{};
  p.format = cache->format;
  p.head_dim = d->head_dim;
  p.batch = d->batch;
  p.kv_heads = d->kv_heads;
  p.group = d->heads / d->kv_heads;
  p.q_len = d->q_len;
  p.kv_len = d->kv_len;
  p.capacity = cache->capacity;
  p.n_blocks = (cache->capacity + ax::kKv8Block - 1) / ax::kKv8Block;
  p.kv_valid = d->kv_valid_len > 0 ? d->kv_valid_len : d->kv_len;
  p.lens = d->kv_valid_lens;
  p.causal = d->causal ? 1 : 0;
  const float scale = d->scale > 0.f ? d->scale : 1.0f / std::sqrt(static_cast<float>(D));
  p.scale_log2 = scale * 1.4426950408889634f;
  p.q = static_cast<const __half*>(q);
  p.q_tok = d->q_tok_stride;
  p.q_head = d->q_head_stride;
  p.q_batch = d->q_batch_stride;
  p.o = static_cast<__half*>(o);
  p.o_tok = d->o_tok_stride;
  p.o_head = d->o_head_stride;
  p.o_batch = d->o_batch_stride;
  p.k_scale = cache->k_scale;
  p.v_scale = cache->v_scale;
  p.status = ctx->d_status;
  p.rows = p.group * p.q_len;
  if (d->qk_norm == ANIMAXS_QK_RMS) {
    // q normalised into context scratch, by the kernel that normalises for animaxs_attn_forward.
    rc = ax_ensure_scratch(ctx, static_cast<size_t>(d->batch) * d->q_len * d->heads * D * 2, s);
    if (rc != ANIMAXS_OK) return rc;
    ax::NormParams np{};
    np.head_dim = d->head_dim;
    np.eps = d->eps > 0.f ? d->eps : 1e-6f;
    np.njobs = 1;
    np.status = ctx->d_status;
    ax::NormJob& j = np.job[0];
    j.in = p.q;
    j.out = static_cast<__half*>(ctx->scratch.ptr);
    j.in_tok = p.q_tok;
    j.in_head = p.q_head;
    j.in_batch = p.q_batch;
    j.out_tok = static_cast<int64_t>(d->heads) * D;
    j.out_head = D;
    j.out_batch = static_cast<int64_t>(d->q_len) * d->heads * D;
    j.tokens = d->q_len;
    j.heads = d->heads;
    j.batch = d->batch;
    j.weight = static_cast<const __half*>(d->q_norm_weight);
    j.rows = static_cast<int64_t>(d->batch) * d->q_len * d->heads;
    const cudaError_t e = ax::launch_qk_norm(np, s);
    if (e != cudaSuccess) return ax_cuda_fail(ctx, e, "qk_norm launch");
    p.q = j.out;
    p.q_tok = j.out_tok;
    p.q_head = j.out_head;
    p.q_batch = j.out_batch;
  }
  // Up to 16 rows of a kv head fit the row kernel's one tile, which streams the
  // cache once; more rows are bound by the products and go to 128-row tiles.  Both
  // at 16 rows (8 kv heads of 128): 300 keys 7.2 and 8.5 us, 4096 keys 10.6 and
  // 12.9, batch 16 x 4096 keys 34 and 66; at 2 rows batch 32 x 4096 50 and 129.
  const bool few = p.rows <= 16;
  CUtensorMap tq, tk, tv, to;
  const int64_t heads = static_cast<int64_t>(cache->batch) * cache->kv_heads;
  const int box = few ? ax::kv8_rows_tile() : ax::kKv8Block;
  rc = ax_make_tmap_codes(ctx, &tk, cache->k_codes, D, cache->capacity, heads, box);
  if (rc == ANIMAXS_OK) rc = ax_make_tmap_codes(ctx, &tv, cache->v_codes, D, cache->capacity, heads, box);
  if (rc != ANIMAXS_OK) return rc;
  cudaError_t e;
  cudaEvent_t ev_stop = nullptr;
  if (few) {
    const int grid = ax::kv8_rows_plan(&p, ctx->num_sms);
    rc = ensure_rows_workspace(ctx);
    if (rc != ANIMAXS_OK) return rc;
    p.part = ctx->kv8_rows_part;
    p.count = ctx->kv8_count;
    rc = ax_timing_begin(ctx, s, &ev_stop);
    if (rc != ANIMAXS_OK) return rc;
    e = ax::launch_kv8_rows(tk, tv, p, grid, ctx->device, s);
  } else {
    if (!ax::kv8_attn_plan(&p, ctx->num_sms))
      return ax_set_error(ctx, ANIMAXS_ERR_OVERFLOW, "attention byte size overflow");
    if (p.split) rc = ensure_tile_workspace(ctx);
    if (rc != ANIMAXS_OK) return rc;
    p.part = ctx->kv8_tile_part;
    rc = ax_make_tmap_rows(ctx, &tq, p.q, D, p.pack, p.q_len, p.lines, p.batch, p.q_tok, p.q_head, p.q_batch,
                           ax::kTileM);
    if (rc == ANIMAXS_OK)
      rc = ax_make_tmap_rows(ctx, &to, p.o, D, p.pack, p.q_len, p.lines, p.batch, p.o_tok, p.o_head, p.o_batch, 32);
    if (rc == ANIMAXS_OK) rc = ax_timing_begin(ctx, s, &ev_stop);
    if (rc != ANIMAXS_OK) return rc;
    e = ax::launch_kv8_attn(tq, tk, tv, to, p, ctx->device, s);
  }
  if (e != cudaSuccess) return ax_cuda_fail(ctx, e, "attention launch");
  ax_timing_end(ctx, s, ev_stop);
  ctx->query_tiles += static_cast<int64_t>(d->heads) * d->batch * ((d->q_len + ax::kTileM - 1LL) / ax::kTileM);
  ctx->last_error.clear();
  return ANIMAXS_OK;
}
