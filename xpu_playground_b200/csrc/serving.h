// Launchers of the serving operators (attention over packed prompts and over
// the paged cache, and the cache's page operators), shared between their
// kernels and the C entry points.
#pragma once

#include "xpu_internal.h"

namespace xpu {

// Launch that may begin under the tail of the kernel before it (programmatic
// dependent launch): every serving kernel sets itself up, then waits for that
// kernel's end before its first access to global memory. Saves about a
// microsecond of launch latency a kernel.
template <typename... Params, typename... Given>
cudaError_t launch_after(void (*kernel)(Params...), uint32_t blocks, uint32_t threads, size_t smem, cudaStream_t stream,
                         const Given &...given) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(given)...);
}

// SMs of the current device (a B200's where there is none).
uint32_t sm_count();

// ---- paged cache (kv_cache.cu) ----
size_t kv_workspace_bytes(uint32_t pages);
cudaError_t kv_extend_launch(const xpu_kv_cache_t &c, const int32_t *sequences, const int32_t *starts, uint32_t count,
                             cudaStream_t s);
// Writes rows into the positions that the last extension added, or (extend) extends first.
cudaError_t kv_write_launch(const xpu_kv_cache_t &c, const int32_t *sequences, const int32_t *starts, uint32_t count,
                            uint32_t tokens, const int32_t *rows, const void *k, const void *v, uint32_t held,
                            uint64_t layer_stride, uint64_t row_stride, uint32_t layer, uint32_t layers, bool extend,
                            cudaStream_t s);
cudaError_t kv_trim_launch(const xpu_kv_cache_t &c, const int32_t *sequences, const int32_t *new_lens, uint32_t count,
                           cudaStream_t s);
cudaError_t kv_fork_launch(const xpu_kv_cache_t &c, const int32_t *parents, const int32_t *children, uint32_t count,
                           cudaStream_t s);
cudaError_t kv_compact_launch(const xpu_kv_cache_t &c, cudaStream_t s);

// ---- attention (serving_attention.cu) ----
// Rows of one head group's tile: row r is position (or node) r / group, head
// r % group of the group, so a tile of 128 rows holds 128 / group of them.
constexpr uint32_t kTileRows = 128;
__host__ __device__ constexpr uint32_t tile_positions(uint32_t group) { return kTileRows / group; }

// Host plan of a packed batch: {blocks, tokens, items, group}, blocks + 1
// offsets into the items, padding to 4 ints, then per item {first token of
// the prompt, its length, first position of the item, kv head}: two tiles of
// positions each.
constexpr uint32_t kPlanHeader = 4;
__host__ __device__ constexpr uint32_t plan_items_at(uint32_t blocks) { return (kPlanHeader + blocks + 1 + 3) / 4 * 4; }
size_t prompt_plan(const uint32_t *lens, uint32_t count, uint32_t q_heads, uint32_t kv_heads, uint32_t sms, int32_t *plan,
                   size_t capacity);

struct AttnTensors {
  const void *q, *k, *v;
  void *out;
  float *lse;
  uint32_t tokens, q_heads, kv_heads, head_dim;
  uint64_t q_stride, kv_stride, out_stride;
  float scale;
};
cudaError_t prompt_attention_launch(bool fp16, const int32_t *plan, uint32_t blocks, const AttnTensors &t,
                                    cudaStream_t s);
size_t tree_workspace_bytes(uint32_t count, uint32_t nodes, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim);
cudaError_t tree_attention_launch(const xpu_kv_cache_t &c, uint32_t layer, const int32_t *sequences,
                                  const int32_t *starts, const uint64_t *ancestors, uint32_t count,
                                  const AttnTensors &t, void *workspace, cudaStream_t s);

}  // namespace xpu
