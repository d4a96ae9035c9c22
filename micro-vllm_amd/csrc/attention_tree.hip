// Attention for trees of drafted tokens over the paged cache.
//
// Request r holds C cached tokens and T drafted nodes, whose rows lie behind
// them at cache positions C .. C + T - 1. Node i sees the cached positions
// [start(i), C) and the nodes j whose bit j is set in its mask:
//   out_i = sum_p softmax_p(q_i . k_p * scale) v_p
// over those positions, scores, maxima and sums in fp32.
#include <cmath>

#include "attention_tree.h"
#include "worklists.h"

namespace mvllm {
namespace {

// Largest i in [0, R] with qsl[i] <= t (qsl is non-decreasing).
__device__ __forceinline__ int64_t owner_of(const TreeArgs& a, int64_t t) {
  int64_t lo = 0, hi = a.num_requests;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (a.qsl[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// ---- any shape ------------------------------------------------------------------
//
// One workgroup of four waves per (node, query head): each wave takes every
// fourth block of 64 keys, a lane scores one key, then the lanes hold the
// output's dims. Only visible keys are read, so nothing that a masked row
// holds can reach the output. Bound by its loads: a lane reads its key's row one
// element at a time, and neither nodes nor heads share what they read. 4 requests
// of 24 nodes over 2,000 keys, 32/8 heads, bf16: 1,139 us at head_dim 80, 1,630 at
// 128 in blocks of 8 (the tile kernel takes 26 in blocks of 16).
constexpr int kAnyWaves = 4;

template <typename T, int DPL>
__global__ __launch_bounds__(64 * kAnyWaves) void tree_any_kernel(TreeArgs a) {
  const int64_t t = blockIdx.x;
  const int hq = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int D = a.head_dim;
  T* const out = static_cast<T*>(a.out) + t * a.o_s0 + static_cast<int64_t>(hq) * a.o_s1;
  const int64_t r = owner_of(a, t);
  if (r >= a.num_requests || a.qsl[r] > t || t >= a.qsl[r + 1]) {
    for (int d = threadIdx.x; d < D; d += 64 * kAnyWaves) Elem<T>::store(out + d * a.o_s2, 0.f);
    return;
  }
  __shared__ float qs[64 * DPL];
  __shared__ float part[kAnyWaves][64 * DPL];
  __shared__ float part_m[kAnyWaves], part_l[kAnyWaves];
  const T* const q = static_cast<const T*>(a.q) + t * a.q_s0 + static_cast<int64_t>(hq) * a.q_s1;
  for (int d = threadIdx.x; d < D; d += 64 * kAnyWaves) qs[d] = Elem<T>::load(q + d * a.q_s2) * a.scale_log2;
  __syncthreads();

  const TreeSpan span = tree_span(a, r);
  int64_t start = a.starts[t];
  if (start < 0) start = 0;
  const int64_t first = start < span.prefix ? start : (span.prefix > 0 ? span.prefix : 0);
  const T* const cache = static_cast<const T*>(a.cache) + static_cast<int64_t>(hq / a.group) * a.c_s[3];
  float acc[DPL];
#pragma unroll
  for (int j = 0; j < DPL; ++j) acc[j] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int64_t base = first + 64 * wave; base < span.end; base += 64 * kAnyWaves) {
    const int64_t p = base + lane;
    int64_t row = -1;  // element offset of this lane's key row
    if (p < span.end && (p < span.prefix ? p >= start : tree_bit(a, t, p - span.prefix))) {
      const int64_t b = a.table[r * a.t_s0 + (p / a.block_size) * a.t_s1];
      if (b >= 0 && b < a.num_blocks) row = b * a.c_s[1] + (p % a.block_size) * a.c_s[2];
    }
    uint64_t seen = __ballot(row >= 0);
    if (!seen) continue;
    float s = -INFINITY;
    if (row >= 0) {
      // Four sums, so that a lane keeps several loads of its row in flight.
      float part4[4] = {0.f, 0.f, 0.f, 0.f};
      int d = 0;
      for (; d + 4 <= D; d += 4)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          part4[e] = __builtin_fmaf(qs[d + e], Elem<T>::load(cache + row + (d + e) * a.c_s[4]), part4[e]);
      for (; d < D; ++d) part4[0] = __builtin_fmaf(qs[d], Elem<T>::load(cache + row + d * a.c_s[4]), part4[0]);
      s = (part4[0] + part4[1]) + (part4[2] + part4[3]);
    }
    float top = s;
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    const float mn = fmaxf(m, top);
    const float base_m = mn == -INFINITY ? 0.f : mn;  // all scores -inf: their weights are zero, not NaN
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - base_m);
    const float w = row >= 0 ? exp2f(s - base_m) : 0.f;
    float sum = w;
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) sum += __shfl_xor(sum, x, 64);
    l = l * alpha + sum;
    m = mn;
#pragma unroll
    for (int j = 0; j < DPL; ++j) acc[j] *= alpha;
    for (; seen; seen &= seen - 1) {
      const int k = __builtin_ctzll(seen);
      const int64_t vrow = __shfl(row, k, 64);
      const float wk = __shfl(w, k, 64);
#pragma unroll
      for (int j = 0; j < DPL; ++j)
        if (lane + 64 * j < D)
          acc[j] = __builtin_fmaf(wk, Elem<T>::load(cache + a.c_s[0] + vrow + (lane + 64 * j) * a.c_s[4]), acc[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < DPL; ++j) part[wave][lane + 64 * j] = acc[j];
  if (lane == 0) {
    part_m[wave] = m;
    part_l[wave] = l;
  }
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kAnyWaves; ++w) top = fmaxf(top, part_m[w]);
  float total = 0.f, scale[kAnyWaves];
#pragma unroll
  for (int w = 0; w < kAnyWaves; ++w) {
    scale[w] = part_m[w] == -INFINITY ? (part_l[w] == 0.f ? 0.f : 1.f) : exp2f(part_m[w] - top);
    total += part_l[w] * scale[w];
  }
  // Nothing visible: 0 / 0, NaN.
  for (int d = threadIdx.x; d < D; d += 64 * kAnyWaves) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kAnyWaves; ++w)
      if (scale[w] != 0.f) v = __builtin_fmaf(part[w][d], scale[w], v);
    Elem<T>::store(out + d * a.o_s2, v / total);
  }
}

template <typename T>
int launch_any(const TreeArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.num_tokens), static_cast<unsigned>(a.num_q_heads));
  const int dpl = (a.head_dim + 63) / 64;
  if (dpl <= 1) hipLaunchKernelGGL((tree_any_kernel<T, 1>), grid, dim3(64 * kAnyWaves), 0, s, a);
  else if (dpl <= 2) hipLaunchKernelGGL((tree_any_kernel<T, 2>), grid, dim3(64 * kAnyWaves), 0, s, a);
  else if (dpl <= 4) hipLaunchKernelGGL((tree_any_kernel<T, 4>), grid, dim3(64 * kAnyWaves), 0, s, a);
  else hipLaunchKernelGGL((tree_any_kernel<T, 8>), grid, dim3(64 * kAnyWaves), 0, s, a);
  MVLLM_LAUNCH_CHECK("tree_any_kernel");
  return MVLLM_OK;
}

int check_tree_tensor(const mvllm_tensor3* t, const char* name, int32_t dtype, int64_t n, int64_t heads, int64_t dim) {
  if (!t) return fail(MVLLM_ERR_INVALID, "%s descriptor is null", name);
  if (t->dtype != dtype)
    return fail(MVLLM_ERR_INVALID, "%s dtype %s differs from the cache's %s", name, dtype_name(t->dtype),
                dtype_name(dtype));
  if (t->size[0] != n || t->size[1] != heads || t->size[2] != dim)
    return fail(MVLLM_ERR_INVALID, "%s shape [%lld, %lld, %lld] does not match [%lld, %lld, %lld]", name,
                (long long)t->size[0], (long long)t->size[1], (long long)t->size[2], (long long)n, (long long)heads,
                (long long)dim);
  for (int i = 0; i < 3; ++i)
    if (t->stride[i] < 0) return fail(MVLLM_ERR_INVALID, "%s has a negative stride", name);
  if (n > 0 && heads > 0 && dim > 0 && !t->data) return fail(MVLLM_ERR_INVALID, "%s data pointer is null", name);
  return MVLLM_OK;
}

}  // namespace
}  // namespace mvllm

using namespace mvllm;

namespace mvllm {
namespace {

// What the kernels need of the cache and the batch (query and output aside).
void fill_tree_args(TreeArgs& a, const mvllm_batch* batch, const mvllm_kv_cache* cache, int64_t Hq) {
  a.cache = cache->data;
  for (int i = 0; i < 5; ++i) a.c_s[i] = cache->stride[i];
  a.starts = batch->query_context_start_positions;
  a.qsl = batch->query_start_locations;
  a.lengths = batch->context_lengths;
  a.table = batch->block_table;
  a.t_s0 = batch->block_table_stride[0];
  a.t_s1 = batch->block_table_stride[1];
  a.width = batch->block_table_width;
  a.num_tokens = batch->num_tokens;
  a.num_requests = batch->num_requests;
  a.num_blocks = cache->num_blocks;
  a.block_size = cache->block_size;
  a.num_q_heads = static_cast<int32_t>(Hq);
  a.num_kv_heads = static_cast<int32_t>(cache->num_kv_heads);
  a.group = static_cast<int32_t>(Hq / cache->num_kv_heads);
  a.head_dim = static_cast<int32_t>(cache->head_dim);
  a.esize = static_cast<int32_t>(dtype_bytes(cache->dtype));
}

// [tokens, heads, dim] rows that can be read 16 bytes at a time.
bool rows_aligned(const mvllm_tensor3* t) {
  const int64_t es = dtype_bytes(t->dtype);
  return t->stride[2] == 1 && t->stride[0] * es % 16 == 0 && t->stride[1] * es % 16 == 0 && aligned16(t->data);
}

int64_t tree_bytes(TreeArgs& a, int32_t dtype, int64_t max_nodes, void* workspace) {
  return dtype == MVLLM_DTYPE_F32 ? tree_f32_layout(a, workspace) : tree_tiles_layout(a, max_nodes, workspace);
}

// Sizes, for calls that the workspace question and the attention both take.
int check_tree_sizes(const mvllm_batch* batch, const mvllm_kv_cache* cache, int64_t Hq) {
  if (dtype_bytes(cache->dtype) == 0) return fail(MVLLM_ERR_UNSUPPORTED, "cache has unsupported dtype");
  if (cache->num_blocks < 1 || cache->block_size < 1 || cache->num_kv_heads < 1 || cache->head_dim < 1)
    return fail(MVLLM_ERR_INVALID, "cache has an empty dimension");
  for (int i = 0; i < 5; ++i)
    if (cache->stride[i] < 0) return fail(MVLLM_ERR_INVALID, "negative cache stride");
  const int64_t N = batch->num_tokens, R = batch->num_requests;
  if (N < 0 || R < 0 || batch->block_table_width < 0) return fail(MVLLM_ERR_INVALID, "negative batch size");
  if (batch->block_size != cache->block_size)
    return fail(MVLLM_ERR_INVALID, "metadata block_size %lld != cache block_size %lld", (long long)batch->block_size,
                (long long)cache->block_size);
  if (Hq < 1 || Hq % cache->num_kv_heads != 0)
    return fail(MVLLM_ERR_INVALID, "query heads %lld not a multiple of KV heads %lld", (long long)Hq,
                (long long)cache->num_kv_heads);
  if (N > INT32_MAX / 4 || R > INT32_MAX / 4 || Hq > 65535)
    return fail(MVLLM_ERR_INVALID, "too many tokens, requests or heads");
  if (cache->head_dim > 512) return fail(MVLLM_ERR_UNSUPPORTED, "head_dim %lld is above 512", (long long)cache->head_dim);
  if (batch->block_table_width > (int64_t{1} << 30) || batch->block_size > (int64_t{1} << 30) ||
      batch->block_table_width * batch->block_size >= (int64_t{1} << 30))
    return fail(MVLLM_ERR_UNSUPPORTED, "positions beyond 2^30 are not supported");
  return MVLLM_OK;
}

}  // namespace
}  // namespace mvllm

extern "C" int64_t mvllm_tree_attention_workspace_bytes(const mvllm_batch* batch, int64_t num_q_heads,
                                                        const mvllm_kv_cache* cache) {
  clear_error();
  if (!batch || !cache || batch->num_tokens <= 0 || batch->num_requests <= 0) return 0;
  if (check_tree_sizes(batch, cache, num_q_heads)) return 0;
  TreeArgs a = {};
  fill_tree_args(a, batch, cache, num_q_heads);
  return tree_bytes(a, cache->dtype, batch->max_query_len, nullptr);
}

extern "C" int mvllm_tree_attention(const mvllm_tensor3* query, const mvllm_tensor3* key, const mvllm_tensor3* value,
                                    const mvllm_kv_cache* cache, const mvllm_batch* batch, const int64_t* tree_mask,
                                    int64_t mask_stride, int64_t mask_words, const mvllm_tensor3* out, float scale,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (!query || !cache || !batch || !out) return fail(MVLLM_ERR_INVALID, "query, cache, batch or out is null");
  if (!cache->data) return fail(MVLLM_ERR_INVALID, "cache is null");
  const int64_t N = batch->num_tokens, R = batch->num_requests;
  const int64_t Hq = query->size[1], Hkv = cache->num_kv_heads, D = cache->head_dim;
  if (int rc = check_tree_sizes(batch, cache, Hq)) return rc;
  if (int rc = check_tree_tensor(query, "query", cache->dtype, N, Hq, D)) return rc;
  if (int rc = check_tree_tensor(out, "out", cache->dtype, N, Hq, D)) return rc;
  if ((key == nullptr) != (value == nullptr)) return fail(MVLLM_ERR_INVALID, "key and value come together");
  if (N == 0) return MVLLM_OK;
  if (!batch->query_start_locations || !batch->query_context_start_positions)
    return fail(MVLLM_ERR_INVALID, "query_start_locations or context starts are null");
  if (R > 0 && (!batch->context_lengths || (batch->block_table_width > 0 && !batch->block_table)))
    return fail(MVLLM_ERR_INVALID, "context_lengths/block_table are null");
  if (!(scale > 0.f) || std::isinf(scale)) return fail(MVLLM_ERR_INVALID, "scale must be positive and finite");
  if (mask_words < 1 || mask_stride < mask_words || !tree_mask)
    return fail(MVLLM_ERR_INVALID, "tree_mask needs at least one word per token");
  if (batch->max_query_len > 64 * mask_words)
    return fail(MVLLM_ERR_INVALID, "trees of %lld nodes need %lld mask words, got %lld",
                (long long)batch->max_query_len, (long long)ceil_div(batch->max_query_len, 64), (long long)mask_words);
  KvRowArgs rows = {};
  bool fused = false;
  if (key) {
    if (!batch->slot_mapping) return fail(MVLLM_ERR_INVALID, "slot_mapping is null");
    if (int rc = check_tree_tensor(key, "key", cache->dtype, N, Hkv, D)) return rc;
    if (int rc = check_tree_tensor(value, "value", cache->dtype, N, Hkv, D)) return rc;
    if (int rc = kv_write_prepare(key, value, cache, batch->slot_mapping, N, &rows, &fused)) return rc;
  }

  TreeArgs a = {};
  fill_tree_args(a, batch, cache, Hq);
  a.q = query->data;
  a.q_s0 = query->stride[0]; a.q_s1 = query->stride[1]; a.q_s2 = query->stride[2];
  a.out = out->data;
  a.o_s0 = out->stride[0]; a.o_s1 = out->stride[1]; a.o_s2 = out->stride[2];
  a.mask = reinterpret_cast<const uint32_t*>(tree_mask);
  a.mask_stride = 2 * mask_stride;
  a.mask_bits = static_cast<int32_t>(mask_words > (1 << 20) ? (1 << 26) : 64 * mask_words);
  a.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  bool tiles = cache->dtype == MVLLM_DTYPE_F32 ? tree_f32_supported(a) : tree_tiles_supported(a, cache->dtype);
  if (tiles) {
    const int64_t need = tree_bytes(a, cache->dtype, batch->max_query_len, workspace);
    tiles = tree_grid_fits(a);
    if (tiles && need > 0 && (!workspace || workspace_bytes < need))
      return fail(MVLLM_ERR_WORKSPACE, "workspace of %lld bytes is smaller than the %lld required",
                  (long long)(workspace ? workspace_bytes : 0), (long long)need);
    if (tiles && !aligned16(workspace)) return fail(MVLLM_ERR_INVALID, "workspace must be 16-byte aligned");
  }
  // The rows in the same launch, where they can be copied 16 bytes at a time.
  const bool with_rows = key && tiles && (a.self_planned ? rows_aligned(key) && rows_aligned(value) : fused);
  if (key && !with_rows)
    if (int rc = mvllm_kv_write(key, value, cache, batch->slot_mapping, N, stream)) return rc;
  if (with_rows && a.self_planned) {
    a.key = key->data;
    a.value = value->data;
    a.k_s0 = key->stride[0]; a.k_s1 = key->stride[1];
    a.v_s0 = value->stride[0]; a.v_s1 = value->stride[1];
    a.slot_mapping = batch->slot_mapping;
  }
  if (tiles)
    return cache->dtype == MVLLM_DTYPE_F32 ? launch_tree_f32(a, with_rows ? &rows : nullptr, s)
                                           : launch_tree_tiles(a, cache->dtype, with_rows ? &rows : nullptr, s);
  switch (cache->dtype) {
    case MVLLM_DTYPE_F32: return launch_any<float>(a, s);
    case MVLLM_DTYPE_F16: return launch_any<f16_t>(a, s);
    default: return launch_any<bf16_t>(a, s);
  }
}
