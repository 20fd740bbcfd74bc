// Attention of the serving path: causal over packed prompts, and of drafted
// token trees over the paged cache (xpu_prompt_attention and
// xpu_tree_attention in include/xpu_cuda.h).
//
// One warp per (row, head): for each allowed key j, s = scale (q . k_j), and
// the running form of the softmax
//   m' = max(m, s), l' = l e^(m - m') + e^(s - m'), o' = o e^(m - m') + e^(s - m') v_j
// in FP32; out = o / l rounded once, lse = m + log l. Masked keys are never
// read, so what stands in them cannot matter.
#include <algorithm>
#include <numeric>
#include <queue>
#include <vector>

#include "common.cuh"
#include "serving.h"

namespace xpu {
namespace {

template <typename T, int D>
struct Row {
  static constexpr int N = D / 32;
  float q[N], o[N], m = -INFINITY, l = 0.f;

  __device__ void begin(const T *row) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      q[i] = Elem<T>::to_float(row[(threadIdx.x & 31) + 32 * i]);
      o[i] = 0.f;
    }
  }
  __device__ void key(const T *k, const T *v, float scale) {
    const int lane = threadIdx.x & 31;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(q[i], Elem<T>::to_float(k[lane + 32 * i]), s);
    s = warp_sum(s) * scale;
    const float top = fmaxf(m, s), keep = m == -INFINITY ? 0.f : expf(m - top), p = top == -INFINITY ? 0.f : expf(s - top);
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * keep + p * Elem<T>::to_float(v[lane + 32 * i]);
    m = top;
  }
  __device__ void end(T *row, float *lse) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < N; ++i) row[lane + 32 * i] = Elem<T>::from_float(l == 0.f ? 0.f : o[i] / l);
    if (lse && lane == 0) *lse = l == 0.f ? -INFINITY : m + logf(l);
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(256) k_prompt(const int32_t *plan, const __grid_constant__ AttnTensors t) {
  const uint32_t group = t.q_heads / t.kv_heads, warp = threadIdx.x / 32;
  const int4 *items = reinterpret_cast<const int4 *>(plan + plan_items_at(plan[0]));
  for (int32_t i = plan[kPlanHeader + blockIdx.x]; i < plan[kPlanHeader + blockIdx.x + 1]; ++i) {
    const int4 it = items[i];
    const uint32_t first = it.x, len = it.y, pos0 = it.z, head = it.w;
    const uint32_t rows = min(2 * tile_positions(group), len - pos0) * group;
    for (uint32_t r = warp; r < rows; r += 8) {
      const uint32_t pos = pos0 + r / group, h = head * group + r % group;
      const size_t token = static_cast<size_t>(first) + pos;
      if (token >= t.tokens) continue;
      Row<T, D> row;
      row.begin(static_cast<const T *>(t.q) + token * t.q_stride + h * D);
      for (uint32_t j = 0; j <= pos; ++j) {
        const size_t at = (static_cast<size_t>(first) + j) * t.kv_stride + head * D;
        row.key(static_cast<const T *>(t.k) + at, static_cast<const T *>(t.v) + at, t.scale);
      }
      row.end(static_cast<T *>(t.out) + token * t.out_stride + h * D,
              t.lse ? t.lse + token * t.q_heads + h : nullptr);
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) k_tree(const __grid_constant__ xpu_kv_cache_t c, uint32_t layer,
                                              const int32_t *sequences, const int32_t *starts,
                                              const uint64_t *ancestors, uint32_t count,
                                              const __grid_constant__ AttnTensors t) {
  const uint32_t group = t.q_heads / t.kv_heads;
  const uint64_t w = blockIdx.x * 8ull + threadIdx.x / 32;
  if (w >= static_cast<uint64_t>(t.tokens) * t.q_heads) return;
  const uint32_t node = static_cast<uint32_t>(w / t.q_heads), h = static_cast<uint32_t>(w % t.q_heads), head = h / group;
  uint32_t lo = 0, hi = count;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (starts[mid] <= static_cast<int32_t>(node)) lo = mid;
    else hi = mid;
  }
  const int32_t begin = starts[lo], end = starts[lo + 1], s = sequences[lo];
  const int32_t nodes = end - begin;
  if (static_cast<int32_t>(node) < begin || static_cast<int32_t>(node) >= end) return;
  uint32_t len = 0;
  bool bad = s < 0 || static_cast<uint32_t>(s) >= c.sequences || nodes > static_cast<int32_t>(XPU_TREE_MAX_NODES);
  if (!bad) {
    const int32_t n = c.lens[s];
    bad = n < 0 || static_cast<uint32_t>(n) > c.table_width * c.page_size;
    len = bad ? 0 : n;
  }
  Row<T, D> row;
  row.begin(static_cast<const T *>(t.q) + node * t.q_stride + h * D);
  for (uint32_t j = 0; j < len; ++j) {
    const int32_t page = c.tables[static_cast<size_t>(s) * c.table_width + j / c.page_size];
    if (page < 0 || static_cast<uint32_t>(page) >= c.pages) {
      bad = true;
      continue;
    }
    const size_t at = (((static_cast<size_t>(layer) * c.pages + page) * c.kv_heads + head) * c.page_size + j % c.page_size) * D;
    row.key(static_cast<const T *>(c.k) + at, static_cast<const T *>(c.v) + at, t.scale);
  }
  const uint64_t set = ancestors[node];
  for (int32_t j = 0; j < min(nodes, static_cast<int32_t>(XPU_TREE_MAX_NODES)); ++j) {
    if (!(set >> j & 1u)) continue;
    const size_t at = static_cast<size_t>(begin + j) * t.kv_stride + head * D;
    row.key(static_cast<const T *>(t.k) + at, static_cast<const T *>(t.v) + at, t.scale);
  }
  row.end(static_cast<T *>(t.out) + node * t.out_stride + h * D,
          t.lse ? t.lse + static_cast<size_t>(node) * t.q_heads + h : nullptr);
  if (bad && (threadIdx.x & 31) == 0) atomicOr(c.status, XPU_KV_BAD_INDEX);
}

}  // namespace

size_t prompt_plan(const uint32_t *lens, uint32_t count, uint32_t q_heads, uint32_t kv_heads, uint32_t sms, int32_t *plan,
                   size_t capacity) {
  const uint32_t group = q_heads / kv_heads, span = 2 * tile_positions(group);
  struct Item {
    int32_t token, len, pos, head;
    uint32_t cost;
  };
  std::vector<Item> items;
  uint64_t tokens = 0;
  for (uint32_t i = 0; i < count; ++i) {
    for (uint32_t pos = 0; pos < lens[i]; pos += span)
      for (uint32_t h = 0; h < kv_heads; ++h)
        items.push_back({static_cast<int32_t>(tokens), static_cast<int32_t>(lens[i]), static_cast<int32_t>(pos),
                         static_cast<int32_t>(h), (std::min(pos + span, lens[i]) + 127) / 128 + 1});
    tokens += lens[i];
  }
  const uint32_t blocks = static_cast<uint32_t>(std::min<size_t>(items.size(), sms));
  const size_t used = plan_items_at(blocks) + 4 * items.size();
  if (used > capacity) return used;
  // longest first, each to the block with the least work
  std::stable_sort(items.begin(), items.end(), [](const Item &a, const Item &b) { return a.cost > b.cost; });
  std::vector<std::vector<const Item *>> per(blocks);
  using Load = std::pair<uint64_t, uint32_t>;
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> loads;
  for (uint32_t b = 0; b < blocks; ++b) loads.push({0, b});
  for (const Item &it : items) {
    const Load least = loads.top();
    loads.pop();
    per[least.second].push_back(&it);
    loads.push({least.first + it.cost, least.second});
  }
  plan[0] = static_cast<int32_t>(blocks);
  plan[1] = static_cast<int32_t>(tokens);
  plan[2] = static_cast<int32_t>(items.size());
  plan[3] = static_cast<int32_t>(group);
  std::fill(plan + kPlanHeader, plan + plan_items_at(blocks), 0);
  int32_t at = 0, *out = plan + plan_items_at(blocks);
  for (uint32_t b = 0; b < blocks; ++b) {
    plan[kPlanHeader + b] = at;
    for (const Item *it : per[b]) {
      const int32_t v[4] = {it->token, it->len, it->pos, it->head};
      std::copy(v, v + 4, out + 4 * at++);
    }
  }
  plan[kPlanHeader + blocks] = at;
  return used;
}

cudaError_t prompt_attention_launch(bool fp16, const int32_t *plan, uint32_t blocks, const AttnTensors &t,
                                    cudaStream_t s) {
  auto kernel = fp16 ? (t.head_dim == 128 ? k_prompt<__half, 128> : k_prompt<__half, 64>)
                     : (t.head_dim == 128 ? k_prompt<__nv_bfloat16, 128> : k_prompt<__nv_bfloat16, 64>);
  kernel<<<blocks, 256, 0, s>>>(plan, t);
  return cudaGetLastError();
}

size_t tree_workspace_bytes(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return 16; }

cudaError_t tree_attention_launch(const xpu_kv_cache_t &c, uint32_t layer, const int32_t *sequences,
                                  const int32_t *starts, const uint64_t *ancestors, uint32_t count,
                                  const AttnTensors &t, void *, cudaStream_t s) {
  auto kernel = c.dtype == XPU_FP16 ? (t.head_dim == 128 ? k_tree<__half, 128> : k_tree<__half, 64>)
                                    : (t.head_dim == 128 ? k_tree<__nv_bfloat16, 128> : k_tree<__nv_bfloat16, 64>);
  const uint64_t warps = static_cast<uint64_t>(t.tokens) * t.q_heads;
  kernel<<<static_cast<uint32_t>((warps + 7) / 8), 256, 0, s>>>(c, layer, sequences, starts, ancestors, count, t);
  return cudaGetLastError();
}

}  // namespace xpu
