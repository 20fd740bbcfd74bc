// extern "C" entry points of libxpu_cuda (declared in include/xpu_cuda.h).
// Each validates its arguments on the host, launches on the caller's stream
// and converts every failure into a status code plus a thread-local message.
#include <cmath>
#include <exception>
#include <string>

#include "serving.h"
#include "xpu_internal.h"

namespace xpu {

namespace {
thread_local std::string g_last_error;
}

void set_error(const std::string &message) { g_last_error = message; }

int fail(int status, const std::string &message) {
  g_last_error = message;
  return status;
}

int cuda_status(cudaError_t error, const char *what) {
  if (error == cudaSuccess) return XPU_OK;
  return fail(XPU_ERR_CUDA, std::string(what) + ": " + cudaGetErrorName(error) + " (" +
                                cudaGetErrorString(error) + ")");
}

}  // namespace xpu

using namespace xpu;

static inline cudaStream_t as_stream(void *stream) { return static_cast<cudaStream_t>(stream); }

#define XPU_REQUIRE(cond, msg) \
  do {                         \
    if (!(cond)) return fail(XPU_ERR_INVALID, msg); \
  } while (0)

// Wraps a body so that no C++ exception crosses the C boundary.
#define XPU_GUARD(...)                                                \
  try {                                                               \
    __VA_ARGS__                                                       \
  } catch (const std::exception &e) {                                 \
    return fail(XPU_ERR_INVALID, std::string("exception: ") + e.what()); \
  } catch (...) {                                                     \
    return fail(XPU_ERR_INVALID, "unknown exception");                \
  }

// Checks of a serving cache that every operator makes; XPU_OK if it is usable.
static int check_cache(const xpu_kv_cache_t *c, const char *who) {
  const std::string at = std::string(who) + ": ";
  XPU_REQUIRE(c, at + "null cache");
  XPU_REQUIRE(c->k && c->v && c->tables && c->lens && c->refs && c->status && c->workspace, at + "null pointer in the cache");
  XPU_REQUIRE(aligned16(c->k) && aligned16(c->v) && aligned16(c->workspace), at + "pools and workspace must be 16-byte aligned");
  XPU_REQUIRE(c->dtype == XPU_BF16 || c->dtype == XPU_FP16, at + "dtype must be XPU_BF16 or XPU_FP16");
  XPU_REQUIRE(c->layers && c->pages && c->kv_heads && c->sequences && c->table_width, at + "empty cache");
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return fail(XPU_ERR_UNSUPPORTED, at + "page_size must be 16, 32, 64 or 128");
  if (c->head_dim != 64 && c->head_dim != 128) return fail(XPU_ERR_UNSUPPORTED, at + "head_dim must be 64 or 128");
  XPU_REQUIRE(c->sequences <= XPU_KV_MAX_SEQUENCES, at + "too many sequences");
  XPU_REQUIRE(static_cast<uint64_t>(c->pages) * c->kv_heads * c->page_size < (1ull << 31) &&
                  static_cast<uint64_t>(c->table_width) * c->page_size < (1ull << 31),
              at + "pool too large");
  return XPU_OK;
}

static int check_list(const void *a, const void *b, uint32_t count, const char *who) {
  XPU_REQUIRE((a && b) || count == 0, std::string(who) + ": null pointer");
  XPU_REQUIRE(count <= XPU_KV_MAX_REQUESTS, std::string(who) + ": more than 1024 sequences in one call");
  return XPU_OK;
}

static int check_rows(const xpu_kv_cache_t &c, const void *k, const void *v, uint32_t held, uint64_t layer_stride,
                      uint64_t row_stride, uint32_t layer, uint32_t layers, const char *who) {
  const std::string at = std::string(who) + ": ";
  XPU_REQUIRE(k && v, at + "null pointer");
  XPU_REQUIRE(aligned16(k) && aligned16(v) && layer_stride % 8 == 0 && row_stride % 8 == 0,
              at + "k and v must be 16-byte aligned with strides in multiples of 8 elements");
  XPU_REQUIRE(row_stride >= static_cast<uint64_t>(c.kv_heads) * c.head_dim, at + "row stride shorter than a row");
  XPU_REQUIRE(held < (1u << 31), at + "too many rows");
  XPU_REQUIRE(layers > 0 && layer < c.layers && layers <= c.layers - layer, at + "layer out of range");
  return XPU_OK;
}

static int check_attention(int dtype, const AttnTensors &t, const char *who) {
  const std::string at = std::string(who) + ": ";
  XPU_REQUIRE(t.q && t.k && t.v && t.out, at + "null pointer");
  XPU_REQUIRE(aligned16(t.q) && aligned16(t.k) && aligned16(t.v) && aligned16(t.out),
              at + "q, k, v and out must be 16-byte aligned");
  XPU_REQUIRE(dtype == XPU_BF16 || dtype == XPU_FP16, at + "dtype must be XPU_BF16 or XPU_FP16");
  if (t.head_dim != 64 && t.head_dim != 128) return fail(XPU_ERR_UNSUPPORTED, at + "head_dim must be 64 or 128");
  XPU_REQUIRE(t.kv_heads > 0 && t.q_heads >= t.kv_heads && t.q_heads % t.kv_heads == 0,
              at + "q_heads must be a positive multiple of kv_heads");
  if (t.q_heads / t.kv_heads > 64) return fail(XPU_ERR_UNSUPPORTED, at + "more than 64 query heads per kv head");
  XPU_REQUIRE(t.tokens < (1u << 31), at + "too many tokens");
  XPU_REQUIRE(t.q_stride % 8 == 0 && t.kv_stride % 8 == 0 && t.out_stride % 8 == 0,
              at + "row strides must be multiples of 8 elements");
  const uint64_t q = static_cast<uint64_t>(t.q_heads) * t.head_dim, kv = static_cast<uint64_t>(t.kv_heads) * t.head_dim;
  XPU_REQUIRE(t.q_stride >= q && t.out_stride >= q && t.kv_stride >= kv, at + "row stride shorter than a row");
  XPU_REQUIRE(t.scale > 0.f && t.scale < INFINITY, at + "scale must be positive and finite");
  XPU_REQUIRE(t.q_stride < (1ull << 38) && t.kv_stride < (1ull << 38), at + "row stride too long");
  return XPU_OK;
}

#define XPU_CHECKED(expr)                  \
  do {                                     \
    const int status_ = (expr);            \
    if (status_ != XPU_OK) return status_; \
  } while (0)

extern "C" {

const char *xpu_last_error(void) { return g_last_error.c_str(); }

int xpu_abi_version(void) { return 1; }

int xpu_gemv(int dtype, const void *matrix, const void *vector, void *output, uint32_t m,
             uint32_t k, void *stream) {
  XPU_GUARD({
    XPU_REQUIRE(matrix && vector && output, "xpu_gemv: null pointer");
    XPU_REQUIRE(m > 0 && k > 0, "xpu_gemv: m and k must be positive");
    cudaError_t e;
    if (dtype == XPU_BF16)
      e = gemv_launch(static_cast<const __nv_bfloat16 *>(matrix),
                      static_cast<const __nv_bfloat16 *>(vector),
                      static_cast<__nv_bfloat16 *>(output), m, k, as_stream(stream));
    else if (dtype == XPU_FP16)
      e = gemv_launch(static_cast<const __half *>(matrix), static_cast<const __half *>(vector),
                      static_cast<__half *>(output), m, k, as_stream(stream));
    else
      return fail(XPU_ERR_INVALID, "xpu_gemv: dtype must be XPU_BF16 or XPU_FP16");
    return cuda_status(e, "xpu_gemv");
  })
}

int xpu_gemm(int dtype, const void *a, const void *b, void *c, uint32_t m, uint32_t n, uint32_t k,
             void *stream) {
  XPU_GUARD({
    XPU_REQUIRE(a && b && c, "xpu_gemm: null pointer");
    XPU_REQUIRE(m > 0 && n > 0 && k > 0, "xpu_gemm: m, n and k must be positive");
    if (dtype != XPU_BF16 && dtype != XPU_FP16)
      return fail(XPU_ERR_INVALID, "xpu_gemm: dtype must be XPU_BF16 or XPU_FP16");
    return cuda_status(gemm_launch(dtype == XPU_FP16, a, b, c, m, n, k, as_stream(stream)), "xpu_gemm");
  })
}

int xpu_gemm_bt(int dtype, const void *a, const void *w, void *c, uint32_t m, uint32_t n, uint32_t k, void *stream) {
  XPU_GUARD({
    XPU_REQUIRE(a && w && c, "xpu_gemm_bt: null pointer");
    XPU_REQUIRE(m > 0 && n > 0 && k > 0, "xpu_gemm_bt: m, n and k must be positive");
    XPU_REQUIRE(n % 8 == 0 && k % 8 == 0, "xpu_gemm_bt: n and k must be multiples of 8");
    XPU_REQUIRE(aligned16(a) && aligned16(w) && aligned16(c), "xpu_gemm_bt: operands must be 16-byte aligned");
    if (dtype != XPU_BF16 && dtype != XPU_FP16)
      return fail(XPU_ERR_INVALID, "xpu_gemm_bt: dtype must be XPU_BF16 or XPU_FP16");
    return cuda_status(gemm_launch_ex(dtype == XPU_FP16, true, a, w, c, m, n, k, as_stream(stream)), "xpu_gemm_bt");
  })
}

int xpu_device_status(uint32_t *flags) {
  XPU_GUARD({
    XPU_REQUIRE(flags, "xpu_device_status: null pointer");
    cudaError_t e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return cuda_status(e, "xpu_device_status");
    *flags = take_device_error() | take_peak_error() | take_attention_error();
    return XPU_OK;
  })
}

int xpu_qwen_embedding(const uint16_t *table, uint16_t *output, uint32_t token, uint32_t width,
                       void *stream) {
  XPU_GUARD({
    XPU_REQUIRE(table && output, "xpu_qwen_embedding: null pointer");
    if (width == 0) return XPU_OK;
    return cuda_status(qwen_embedding_launch(table, output, token, width, as_stream(stream)),
                       "xpu_qwen_embedding");
  })
}

int xpu_qwen_rms_norm(const uint16_t *input, const uint16_t *weight, uint16_t *output,
                      uint32_t width, float epsilon, void *stream) {
  XPU_GUARD({
    XPU_REQUIRE(input && weight && output, "xpu_qwen_rms_norm: null pointer");
    XPU_REQUIRE(width > 0, "xpu_qwen_rms_norm: width must be positive");
    return cuda_status(qwen_rms_norm_launch(input, weight, output, width, epsilon,
                                            as_stream(stream)),
                       "xpu_qwen_rms_norm");
  })
}

int xpu_qwen_gemv(const uint16_t *matrix, const uint16_t *vector, uint16_t *output,
                  uint32_t rows, uint32_t columns, void *stream) {
  return xpu_gemv(XPU_BF16, matrix, vector, output, rows, columns, stream);
}

int xpu_qwen_qkv_rope_cache(uint16_t *query, uint16_t *key, const uint16_t *value,
                            const uint16_t *query_norm, const uint16_t *key_norm,
                            const uint16_t *rope_cos, const uint16_t *rope_sin,
                            uint16_t *key_cache, uint16_t *value_cache, uint32_t position,
                            uint32_t maximum_sequence, uint32_t query_heads,
                            uint32_t key_value_heads, void *stream) {
  XPU_GUARD({
    XPU_REQUIRE(query && key && value && query_norm && key_norm && rope_cos && rope_sin &&
                    key_cache && value_cache,
                "xpu_qwen_qkv_rope_cache: null pointer");
    XPU_REQUIRE(key_value_heads > 0 && query_heads >= key_value_heads &&
                    query_heads % key_value_heads == 0,
                "xpu_qwen_qkv_rope_cache: query_heads must be a positive multiple of "
                "key_value_heads");
    return cuda_status(
        qwen_qkv_rope_cache_launch(query, key, value, query_norm, key_norm, rope_cos, rope_sin,
                                   key_cache, value_cache, position, maximum_sequence,
                                   query_heads, key_value_heads, as_stream(stream)),
        "xpu_qwen_qkv_rope_cache");
  })
}

size_t xpu_qwen_attention_workspace_size(uint32_t query_heads, uint32_t maximum_positions) {
  return qwen_attention_workspace(query_heads, maximum_positions);
}

int xpu_qwen_attention(const uint16_t *query, const uint16_t *key_cache,
                       const uint16_t *value_cache, uint16_t *output, uint32_t position,
                       uint32_t query_heads, uint32_t key_value_heads, void *workspace,
                       size_t workspace_bytes, void *stream) {
  XPU_GUARD({
    XPU_REQUIRE(query && key_cache && value_cache && output && workspace,
                "xpu_qwen_attention: null pointer");
    XPU_REQUIRE(aligned16(workspace), "xpu_qwen_attention: workspace must be 16-byte aligned");
    XPU_REQUIRE(key_value_heads > 0 && query_heads % key_value_heads == 0,
                "xpu_qwen_attention: query_heads must be a multiple of key_value_heads");
    const uint32_t group = query_heads / key_value_heads;
    if (group != 1 && group != 2 && group != 4 && group != 8)
      return fail(XPU_ERR_UNSUPPORTED, "xpu_qwen_attention: query_heads / key_value_heads must "
                                       "be 1, 2, 4 or 8");
    XPU_REQUIRE(position != UINT32_MAX, "xpu_qwen_attention: position out of range");
    const size_t need = qwen_attention_workspace(query_heads, position + 1);
    if (workspace_bytes < need)
      return fail(XPU_ERR_INVALID, "xpu_qwen_attention: workspace holds " +
                                       std::to_string(workspace_bytes) + " bytes, needs " +
                                       std::to_string(need));
    return cuda_status(qwen_attention_launch(query, key_cache, value_cache, output, position,
                                             query_heads, key_value_heads,
                                             static_cast<float *>(workspace), as_stream(stream)),
                       "xpu_qwen_attention");
  })
}

int xpu_qwen_add(uint16_t *left, const uint16_t *right, uint32_t width, void *stream) {
  XPU_GUARD({
    XPU_REQUIRE(left && right, "xpu_qwen_add: null pointer");
    if (width == 0) return XPU_OK;
    return cuda_status(qwen_add_launch(left, right, width, as_stream(stream)), "xpu_qwen_add");
  })
}

int xpu_qwen_silu_multiply(uint16_t *gate, const uint16_t *up, uint32_t width, void *stream) {
  XPU_GUARD({
    XPU_REQUIRE(gate && up, "xpu_qwen_silu_multiply: null pointer");
    if (width == 0) return XPU_OK;
    return cuda_status(qwen_silu_multiply_launch(gate, up, width, as_stream(stream)),
                       "xpu_qwen_silu_multiply");
  })
}

int xpu_qwen_argmax(const uint16_t *values, uint32_t *token, uint32_t width, void *stream) {
  XPU_GUARD({
    XPU_REQUIRE(values && token, "xpu_qwen_argmax: null pointer");
    return cuda_status(qwen_argmax_launch(values, token, width, as_stream(stream)),
                       "xpu_qwen_argmax");
  })
}

size_t xpu_kv_workspace_size(uint32_t pages) { return kv_workspace_bytes(pages); }

int xpu_kv_extend(const xpu_kv_cache_t *cache, const int32_t *sequences, const int32_t *starts, uint32_t count,
                  void *stream) {
  XPU_GUARD({
    XPU_CHECKED(check_cache(cache, "xpu_kv_extend"));
    XPU_CHECKED(check_list(sequences, starts, count, "xpu_kv_extend"));
    if (count == 0) return XPU_OK;
    return cuda_status(kv_extend_launch(*cache, sequences, starts, count, as_stream(stream)), "xpu_kv_extend");
  })
}

int xpu_kv_write(const xpu_kv_cache_t *cache, const int32_t *sequences, const int32_t *starts, uint32_t count,
                 uint32_t tokens, const int32_t *rows, const void *k, const void *v, uint32_t held,
                 uint64_t layer_stride, uint64_t row_stride, uint32_t layer, uint32_t layers, void *stream) {
  XPU_GUARD({
    XPU_CHECKED(check_cache(cache, "xpu_kv_write"));
    XPU_CHECKED(check_list(sequences, starts, count, "xpu_kv_write"));
    if (count == 0 || tokens == 0) return XPU_OK;
    XPU_CHECKED(check_rows(*cache, k, v, held, layer_stride, row_stride, layer, layers, "xpu_kv_write"));
    return cuda_status(kv_write_launch(*cache, sequences, starts, count, tokens, rows, k, v, held, layer_stride, row_stride,
                                       layer, layers, false, as_stream(stream)),
                       "xpu_kv_write");
  })
}

int xpu_kv_append(const xpu_kv_cache_t *cache, const int32_t *sequences, const int32_t *starts, uint32_t count,
                  uint32_t tokens, const int32_t *rows, const void *k, const void *v, uint32_t held,
                  uint64_t layer_stride, uint64_t row_stride, void *stream) {
  XPU_GUARD({
    XPU_CHECKED(check_cache(cache, "xpu_kv_append"));
    XPU_CHECKED(check_list(sequences, starts, count, "xpu_kv_append"));
    if (count == 0 || tokens == 0) return XPU_OK;
    XPU_CHECKED(check_rows(*cache, k, v, held, layer_stride, row_stride, 0, cache->layers, "xpu_kv_append"));
    return cuda_status(kv_write_launch(*cache, sequences, starts, count, tokens, rows, k, v, held, layer_stride, row_stride,
                                       0, cache->layers, true, as_stream(stream)),
                       "xpu_kv_append");
  })
}

int xpu_kv_trim(const xpu_kv_cache_t *cache, const int32_t *sequences, const int32_t *new_lens, uint32_t count,
                void *stream) {
  XPU_GUARD({
    XPU_CHECKED(check_cache(cache, "xpu_kv_trim"));
    XPU_CHECKED(check_list(sequences, new_lens, count, "xpu_kv_trim"));
    if (count == 0) return XPU_OK;
    return cuda_status(kv_trim_launch(*cache, sequences, new_lens, count, as_stream(stream)), "xpu_kv_trim");
  })
}

int xpu_kv_fork(const xpu_kv_cache_t *cache, const int32_t *parents, const int32_t *children, uint32_t count,
                void *stream) {
  XPU_GUARD({
    XPU_CHECKED(check_cache(cache, "xpu_kv_fork"));
    XPU_CHECKED(check_list(parents, children, count, "xpu_kv_fork"));
    if (count == 0) return XPU_OK;
    return cuda_status(kv_fork_launch(*cache, parents, children, count, as_stream(stream)), "xpu_kv_fork");
  })
}

int xpu_kv_compact(const xpu_kv_cache_t *cache, void *stream) {
  XPU_GUARD({
    XPU_CHECKED(check_cache(cache, "xpu_kv_compact"));
    return cuda_status(kv_compact_launch(*cache, as_stream(stream)), "xpu_kv_compact");
  })
}

int xpu_prompt_plan(const uint32_t *lens, uint32_t count, uint32_t q_heads, uint32_t kv_heads, int32_t *plan,
                    size_t capacity, size_t *used) {
  XPU_GUARD({
    XPU_REQUIRE((lens || count == 0) && (plan || capacity == 0) && used, "xpu_prompt_plan: null pointer");
    XPU_REQUIRE(kv_heads > 0 && q_heads >= kv_heads && q_heads % kv_heads == 0,
                "xpu_prompt_plan: q_heads must be a positive multiple of kv_heads");
    if (q_heads / kv_heads > 64) return fail(XPU_ERR_UNSUPPORTED, "xpu_prompt_plan: more than 64 query heads per kv head");
    uint64_t tokens = 0;
    for (uint32_t i = 0; i < count; ++i) tokens += lens[i];
    XPU_REQUIRE(tokens < (1ull << 31), "xpu_prompt_plan: too many tokens");
    *used = prompt_plan(lens, count, q_heads, kv_heads, sm_count(), plan, capacity);
    if (*used > capacity)
      return fail(XPU_ERR_INVALID, "xpu_prompt_plan: the plan needs " + std::to_string(*used) + " ints");
    return XPU_OK;
  })
}

int xpu_prompt_attention(int dtype, const int32_t *plan, uint32_t plan_blocks, const void *q, const void *k, const void *v,
                         void *out, float *lse, uint32_t tokens, uint32_t q_heads, uint32_t kv_heads,
                         uint32_t head_dim, uint64_t q_stride, uint64_t kv_stride, uint64_t out_stride, float scale,
                         void *stream) {
  XPU_GUARD({
    const AttnTensors t{q, k, v, out, lse, tokens, q_heads, kv_heads, head_dim, q_stride, kv_stride, out_stride, scale};
    if (tokens == 0) return XPU_OK;
    XPU_REQUIRE(plan_blocks > 0, "xpu_prompt_attention: the plan has no tiles for these tokens");
    XPU_REQUIRE(plan && aligned16(plan), "xpu_prompt_attention: the plan must be a 16-byte aligned device pointer");
    XPU_CHECKED(check_attention(dtype, t, "xpu_prompt_attention"));
    return cuda_status(prompt_attention_launch(dtype == XPU_FP16, plan, plan_blocks, t, as_stream(stream)),
                       "xpu_prompt_attention");
  })
}

size_t xpu_tree_attention_workspace_size(uint32_t count, uint32_t nodes, uint32_t q_heads, uint32_t kv_heads,
                                         uint32_t head_dim) {
  if (kv_heads == 0 || q_heads < kv_heads) return 0;
  return tree_workspace_bytes(count, nodes, q_heads, kv_heads, head_dim);
}

int xpu_tree_attention(const xpu_kv_cache_t *cache, uint32_t layer, const int32_t *sequences, const int32_t *starts,
                       const uint64_t *ancestors, uint32_t count, uint32_t nodes, const void *q, const void *k,
                       const void *v, void *out, float *lse, uint32_t q_heads, uint64_t q_stride, uint64_t kv_stride,
                       uint64_t out_stride, float scale, void *workspace, size_t workspace_bytes, void *stream) {
  XPU_GUARD({
    XPU_CHECKED(check_cache(cache, "xpu_tree_attention"));
    XPU_CHECKED(check_list(sequences, starts, count, "xpu_tree_attention"));
    XPU_REQUIRE(layer < cache->layers, "xpu_tree_attention: layer out of range");
    if (count == 0 || nodes == 0) return XPU_OK;
    XPU_REQUIRE(ancestors && workspace, "xpu_tree_attention: null pointer");
    XPU_REQUIRE(aligned16(workspace), "xpu_tree_attention: workspace must be 16-byte aligned");
    const AttnTensors t{q, k, v, out, lse, nodes, q_heads, cache->kv_heads, cache->head_dim, q_stride, kv_stride, out_stride,
                        scale};
    XPU_CHECKED(check_attention(cache->dtype, t, "xpu_tree_attention"));
    // the work is counted in key tiles of 128, in 32 bits
    const uint64_t tiles = (static_cast<uint64_t>(cache->table_width) * cache->page_size + 127) / 128 + 4;
    const uint64_t blocks = (static_cast<uint64_t>(q_heads / cache->kv_heads) * XPU_TREE_MAX_NODES + 127) / 128 + 1;
    if (tiles * blocks * cache->kv_heads * count >= (1ull << 32))
      return fail(XPU_ERR_UNSUPPORTED, "xpu_tree_attention: too many sequences of such length in one call");
    const size_t need = tree_workspace_bytes(count, nodes, q_heads, cache->kv_heads, cache->head_dim);
    if (workspace_bytes < need)
      return fail(XPU_ERR_INVALID, "xpu_tree_attention: workspace holds " + std::to_string(workspace_bytes) +
                                       " bytes, needs " + std::to_string(need));
    return cuda_status(tree_attention_launch(*cache, layer, sequences, starts, ancestors, count, t, workspace,
                                             as_stream(stream)),
                       "xpu_tree_attention");
  })
}

}  // extern "C"
