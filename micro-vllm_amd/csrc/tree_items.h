// The work items of the tree attention kernels: which rows and keys a workgroup
// takes, who writes the nodes' K/V rows, and the merge of split keys. The same
// for the 16-bit (attention_tree_tiles.hip) and the fp32 kernel
// (attention_tree_f32.hip).
#pragma once

#include <climits>
#include <cmath>
#include <type_traits>

#include "attention_tree.h"
#include "worklists.h"

namespace mvllm {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kBuckets = 32;
constexpr int32_t kFar = 1 << 30;  // no position reaches it

// ---- plan ------------------------------------------------------------------------

// First key of request r's splits, a guess from its first node: the others may
// see earlier keys, which split 0 adds.
__device__ __forceinline__ int64_t first_key(const TreeArgs& a, const TreeSpan& s) {
  int64_t k = a.starts[s.qs];
  if (k > s.prefix) k = s.prefix;
  return k < 0 ? 0 : k & ~int64_t{15};
}

struct TreeReq {
  int32_t first, keys, blocks;  // first key of the splits, keys behind it, row blocks
  int32_t qs, nodes, prefix;
};

__device__ __forceinline__ TreeReq tree_request(const TreeArgs& a, int64_t r) {
  TreeReq q = {0, 0, 0, 0, 0, 0};
  if (r >= a.num_requests) return q;
  const TreeSpan s = tree_span(a, r);
  if (s.qe == s.qs) return q;
  const int64_t first = first_key(a, s);
  q.first = static_cast<int32_t>(first < kFar ? first : kFar);
  q.keys = static_cast<int32_t>(s.end > first ? s.end - first : 0);
  q.qs = static_cast<int32_t>(s.qs);
  q.nodes = static_cast<int32_t>(s.qe - s.qs);
  q.blocks = static_cast<int32_t>((static_cast<int64_t>(q.nodes) * a.group + a.rows - 1) / a.rows);
  q.prefix = static_cast<int32_t>(s.prefix < kFar ? s.prefix : kFar);
  return q;
}

__host__ __device__ __forceinline__ int64_t tree_load(const TreeReq& q) {
  return static_cast<int64_t>(q.blocks) * (q.keys > 0 ? q.keys : 1);
}

__host__ __device__ __forceinline__ int32_t tree_splits(const TreeArgs& a, const TreeReq& q, int32_t split) {
  return a.merge_capacity > 0 && q.keys > split ? (q.keys + split - 1) / split : 1;
}

// Keys of each of a request's `ns` splits but the last: even shares, at most the
// split length that gave ns, so that the last one has keys as well.
__host__ __device__ __forceinline__ int32_t tree_share(const TreeReq& q, int32_t ns) {
  return ns > 1 ? ((q.keys + ns - 1) / ns + 63) & ~63 : q.keys;
}

__device__ __forceinline__ TreeItem tree_item(const TreeReq& q, int32_t r, int32_t k, int32_t rb, int32_t ns,
                                              int32_t share, int32_t slot) {
  const int32_t begin = q.first + k * share;
  return TreeItem{r, rb, begin, k + 1 < ns ? begin + share : q.first + q.keys, k, ns, slot + k * q.blocks + rb, q.qs,
                  q.nodes, q.prefix, 0, 0};
}

// Whether a place exists. Query starts that do not ascend may count the same
// tokens so often that places wrap around.
__device__ __forceinline__ bool in_list(int32_t place, int32_t places) {
  return static_cast<uint32_t>(place) < static_cast<uint32_t>(places);
}

// Inclusive sums over a wave's lanes, by row shifts and row broadcasts (a step is
// one instruction; through LDS it is a round trip).
__device__ __forceinline__ int32_t wave_scan(int32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // lane 15 of a row to the next one
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31 to the upper half
  return v;
}

__device__ __forceinline__ int32_t wave_sum(int32_t v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

__device__ __forceinline__ float wave_sum(float v) {
  auto step = [&](auto ctrl, auto rows) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
  };
  using All = std::integral_constant<int, 0xF>;
  step(std::integral_constant<int, 0x111>{}, All{});
  step(std::integral_constant<int, 0x112>{}, All{});
  step(std::integral_constant<int, 0x114>{}, All{});
  step(std::integral_constant<int, 0x118>{}, All{});
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// 1 / x to a unit in the last place.
__host__ __device__ __forceinline__ float reciprocal(float x) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_rcpf(x);
#else
  return 1.0f / x;
#endif
}

// Split lengths to choose from, for `total` keys over all row blocks: attempt c
// shares them among (16 - c) / 16 of the workgroups that run at once, the last
// one among half. Keys are summed in fp32 and divided by reciprocals: each length
// is longer by more than their rounding (2^-14 relative to a few times 2^-22).
constexpr int kAttempts = 8;
__host__ __device__ __forceinline__ float split_share(const TreeArgs& a, float total) {
  return total * reciprocal(static_cast<float>(a.target)) * (16.0f + 0.001f);
}
__host__ __device__ __forceinline__ int32_t split_length(const TreeArgs& a, float share, int c) {
  const float x = fmaxf(share * reciprocal(static_cast<float>(16 - c)) + 1.0f, static_cast<float>(a.shortest));
  return x < static_cast<float>(kFar) ? (static_cast<int32_t>(x) + 63) & ~63 : kFar;
}

// Items of `blocks` row blocks of `keys` keys in splits of `length`, at least
// (1 / length is rounded up: a quotient just below an integer counts as that).
__host__ __device__ __forceinline__ int32_t split_count(int32_t blocks, int32_t keys, int32_t length) {
  const float q = static_cast<float>(keys - 1) * (reciprocal(static_cast<float>(length)) * (1.0f + 0x1p-20f));
  const int32_t n = static_cast<int32_t>(q) + 1;
  return blocks * (n > 1 ? n : 1);
}

// Whether the shortest split leaves no more items than run at once.
__host__ __device__ __forceinline__ bool all_shortest(const TreeArgs& a, float total, float blocks) {
  const float shortest = static_cast<float>(a.shortest);
  return total + blocks * shortest <= static_cast<float>(a.target) * shortest;
}

// The batch's split length, the same in all W waves of the workgroup: the
// shortest of the attempts, no shorter than `shortest`, that leaves no more items
// than workgroups run at once (a second round of a few costs a whole round),
// else twice the even share; the lists and the partials were sized by the same
// rule. Thread t holds request t, nth(r) is any. Thread (c, i) of 8 x 8 W counts
// the items of attempt c over requests i, i + 8 W, ...: code that is short, since
// a launch fetches it anew. Uses W * kPlanBytes of LDS.
constexpr int kPlanBytes = 8 * 64 + 4 * kAttempts;
template <int W, typename Nth>
__device__ __forceinline__ int32_t plan_split(const TreeArgs& a, const Nth& nth, uint8_t* lds) {
  int2* const work = reinterpret_cast<int2*>(lds);                            // [64 W] (row blocks, keys)
  int32_t* const sums = reinterpret_cast<int32_t*>(lds + 8 * 64 * W);         // [W][kAttempts]
  float2* const totals = reinterpret_cast<float2*>(sums);                     // [W]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t R = a.num_requests;
  float total = 0.f, blocks = 0.f;
  for (int64_t r = tid; r < R; r += 64 * W) {
    const TreeReq q = nth(r);
    total += static_cast<float>(tree_load(q));
    blocks += static_cast<float>(q.blocks);
  }
  total = wave_sum(total);
  blocks = wave_sum(blocks);
  if (lane == 0) totals[wave] = float2{total, blocks};
  __syncthreads();
  total = blocks = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) total += totals[w].x, blocks += totals[w].y;
  if (all_shortest(a, total, blocks)) return a.shortest;
  const int c = lane & (kAttempts - 1);
  const float share = split_share(a, total);
  const int32_t twice = split_length(a, share, kAttempts);
  if (blocks >= static_cast<float>(a.target)) return __builtin_amdgcn_readfirstlane(twice);
  const int32_t mine = split_length(a, share, c);
  int32_t count = 0;
  for (int64_t at = 0; at < R; at += 64 * W) {
    __syncthreads();
    const TreeReq q = nth(at + tid);
    work[tid] = int2{q.blocks, q.keys};
    __syncthreads();
    const int here = R - at < 64 * W ? static_cast<int>(R - at) : 64 * W;
    for (int i = tid / kAttempts; i < here; i += 64 * W / kAttempts)
      count += split_count(work[i].x, work[i].y, mine);
  }
#pragma unroll
  for (int x = 32; x >= kAttempts; x >>= 1) count += __shfl_xor(count, x, 64);
  if (lane < kAttempts) sums[kAttempts * wave + lane] = count;
  __syncthreads();
  count = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) count += sums[kAttempts * w + c];
  const uint32_t fits = static_cast<uint32_t>(__ballot(count <= a.target)) & ((1u << kAttempts) - 1);
  return fits ? __builtin_amdgcn_readlane(mine, __builtin_ctz(fits)) : __builtin_amdgcn_readfirstlane(twice);
}

// The same for up to 64 requests, which a wave finds by itself: lane r holds
// request r.
__device__ __forceinline__ int32_t plan_split64(const TreeArgs& a, const TreeReq& q) {
  const float total = wave_sum(static_cast<float>(tree_load(q))), blocks = wave_sum(static_cast<float>(q.blocks));
  if (all_shortest(a, total, blocks)) return a.shortest;
  const float share = split_share(a, total);
  if (blocks < static_cast<float>(a.target))
    for (int c = 0; c < kAttempts; ++c) {
      const int32_t length = split_length(a, share, c);
      if (wave_sum(split_count(q.blocks, q.keys, length)) <= a.target) return length;
    }
  return split_length(a, share, kAttempts);
}

// Item `slot` of the batch in order of request, split and row block, and with
// `lists` the merge list: for up to 64 requests, by each wave by itself (no
// barrier and no LDS: 5,600 cycles of a launch over 16 requests instead of 8,500).
__device__ TreeItem find_item64(const TreeArgs& a, int32_t slot, bool lists) {
  const int lane = threadIdx.x & 63;
  const TreeReq q = tree_request(a, lane);
  const int32_t split = __builtin_amdgcn_readfirstlane(plan_split64(a, q));
  const int32_t ns = tree_splits(a, q, split), items = q.blocks * ns;
  const int32_t at = wave_scan(items) - items, slot_at = wave_scan(ns > 1 ? items : 0) - (ns > 1 ? items : 0);
  if (lists && threadIdx.x < 64) {
    const int32_t blocks = ns > 1 ? q.blocks : 0, merge_end = wave_scan(blocks), merge_at = merge_end - blocks;
    for (int32_t rb = 0; rb < blocks && in_list(merge_at + rb, a.merge_capacity); ++rb)
      a.merges[merge_at + rb] = TreeMerge{q.qs, q.nodes, rb, ns, slot_at + rb, q.blocks, 0, 0};
    for (int32_t i = max(__builtin_amdgcn_readlane(merge_end, 63), 0) + lane; i < a.merge_capacity; i += 64) a.merges[i].ns = 0;
  }
  const uint64_t mine = __ballot(slot >= at && slot < at + items);
  if (!mine) return TreeItem{-1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  const int r = __builtin_ctzll(mine);
  const auto of = [&](int32_t x) { return __builtin_amdgcn_readlane(x, r); };
  const TreeReq found = {of(q.first), of(q.keys), of(q.blocks), of(q.qs), of(q.nodes), of(q.prefix)};
  const int32_t n = of(ns), i = slot - of(at), k = __builtin_amdgcn_readfirstlane(i / found.blocks);
  return tree_item(found, r, k, i - k * found.blocks, n, __builtin_amdgcn_readfirstlane(tree_share(found, n)), of(slot_at));
}

// The same for any number of requests, by one workgroup of W waves (r = -1:
// there is none). For grids whose workgroups all run at once: their order does
// not matter then, and a list of a launch of its own would cost more than to
// find it. Uses the first bytes of LDS.
template <int W>
__device__ TreeItem find_item(const TreeArgs& a, int32_t slot, bool lists, uint8_t* lds) {
  if (a.num_requests <= 64) return find_item64(a, slot, lists);
  constexpr int kWaves = W, kThreads = 64 * kWaves;
  static_assert(12 * kWaves <= 256, "the sums lie before the item");
  int32_t* const sums = reinterpret_cast<int32_t*>(lds);  // [kWaves][3]
  TreeItem* const found = reinterpret_cast<TreeItem*>(lds + 256);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t R = a.num_requests;
  const TreeReq own = tree_request(a, tid);  // all there is, up to 64 W requests
  auto nth = [&](int64_t r) { return r < kThreads ? own : tree_request(a, r); };
  if (tid == 0) found->r = -1;
  const int32_t split = plan_split<W>(a, nth, lds + 512);
  int32_t carry[3] = {0, 0, 0};  // items, partial slots, merge places
  for (int64_t base = 0; base < R; base += kThreads) {
    const int32_t r = static_cast<int32_t>(base) + tid;
    const TreeReq q = nth(r);
    const int32_t ns = tree_splits(a, q, split), items = q.blocks * ns;
    const int32_t mine[3] = {items, ns > 1 ? items : 0, ns > 1 ? q.blocks : 0};
    int32_t at[3] = {mine[0], mine[1], mine[2]};
#pragma unroll
    for (int i = 0; i < 3; ++i) at[i] = wave_scan(at[i]);
    if (lane == 63)
#pragma unroll
      for (int i = 0; i < 3; ++i) sums[3 * wave + i] = at[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      at[i] += carry[i] - mine[i];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        if (w < wave) at[i] += sums[3 * w + i];
        carry[i] += sums[3 * w + i];
      }
    }
    if (slot >= at[0] && slot < at[0] + items) {
      const int32_t k = (slot - at[0]) / q.blocks;
      *found = tree_item(q, r, k, slot - at[0] - k * q.blocks, ns, tree_share(q, ns), at[1]);
    }
    if (lists && ns > 1)
      for (int32_t rb = 0; rb < q.blocks && in_list(at[2] + rb, a.merge_capacity); ++rb)
        a.merges[at[2] + rb] = TreeMerge{q.qs, q.nodes, rb, ns, at[1] + rb, q.blocks, 0, 0};
    __syncthreads();
  }
  if (lists)
    for (int32_t i = max(carry[2], 0) + tid; i < a.merge_capacity; i += kThreads) a.merges[i].ns = 0;
  const auto one = [](int32_t x) { return __builtin_amdgcn_readfirstlane(x); };
  return TreeItem{one(found->r),    one(found->rb), one(found->begin), one(found->end),   one(found->split), one(found->ns),
                  one(found->slot), one(found->qs), one(found->nodes), one(found->prefix), 0, 0};
}

// The item list, heaviest first, and the merge list, written by one workgroup.
__device__ void plan_items(const TreeArgs& a) {
  __shared__ alignas(8) uint8_t plan[kPlanThreads / 64 * kPlanBytes];
  __shared__ int32_t sums[kPlanThreads / 64][3];
  __shared__ int32_t bucket[kBuckets], cursor[kBuckets + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t R = a.num_requests;
  const TreeReq own = tree_request(a, tid);  // all there is, up to 1,024 requests
  auto nth = [&](int64_t r) { return r < kPlanThreads ? own : tree_request(a, r); };
  if (tid < kBuckets) bucket[tid] = 0;
  const int32_t split = plan_split<kPlanThreads / 64>(a, nth, plan);
  auto bucket_of = [&](int32_t keys) {
    const int32_t b = static_cast<int32_t>(static_cast<float>(keys) * kBuckets / static_cast<float>(split));
    return kBuckets - 1 - (b < kBuckets - 1 ? b : kBuckets - 1);
  };
  for (int64_t r = tid; r < R; r += kPlanThreads) {
    const TreeReq q = nth(r);
    if (q.blocks == 0) continue;
    const int32_t ns = tree_splits(a, q, split);
    const int32_t share = tree_share(q, ns);
    if (ns > 1) atomicAdd(&bucket[bucket_of(share)], (ns - 1) * q.blocks);
    atomicAdd(&bucket[bucket_of(q.keys - (ns - 1) * share)], q.blocks);
  }
  __syncthreads();
  if (tid < 64) {
    const int32_t mine = tid < kBuckets ? bucket[tid] : 0;
    int32_t inc = mine;
#pragma unroll
    for (int x = 1; x < kBuckets; x <<= 1) {
      const int32_t y = __shfl_up(inc, x, 64);
      if (lane >= x) inc += y;
    }
    if (tid < kBuckets) cursor[tid] = inc - mine;
    if (tid == kBuckets - 1) cursor[kBuckets] = inc;
  }
  __syncthreads();
  for (int64_t i = max(cursor[kBuckets], 0) + tid; i < a.capacity; i += kPlanThreads) a.items[i].r = -1;
  int32_t carry[3] = {0, 0, 0};  // partial slots, merge places
  for (int64_t base = 0; base < R; base += kPlanThreads) {
    const int32_t r = static_cast<int32_t>(base) + tid;
    const TreeReq q = nth(r);
    const int32_t ns = tree_splits(a, q, split);
    // Partial slots and merge places in order of the requests.
    const int32_t mine[3] = {ns > 1 ? ns * q.blocks : 0, ns > 1 ? q.blocks : 0, 0};
    int32_t at[3] = {mine[0], mine[1], 0};
#pragma unroll
    for (int i = 0; i < 3; ++i) at[i] = wave_scan(at[i]);
    if (lane == 63)
#pragma unroll
      for (int i = 0; i < 2; ++i) sums[wave][i] = at[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      at[i] += carry[i] - mine[i];
#pragma unroll
      for (int w = 0; w < kPlanThreads / 64; ++w) {
        if (w < wave) at[i] += sums[w][i];
        carry[i] += sums[w][i];
      }
    }
    __syncthreads();
    if (q.blocks == 0) continue;
    const int32_t share = tree_share(q, ns);
    for (int32_t k = 0; k < ns; ++k) {
      const int32_t keys = k + 1 < ns ? share : q.keys - k * share;
      const int32_t to = atomicAdd(&cursor[bucket_of(keys)], q.blocks);
      for (int32_t rb = 0; rb < q.blocks && in_list(to + rb, a.capacity); ++rb)
        a.items[to + rb] = tree_item(q, r, k, rb, ns, share, at[0]);
    }
    if (ns > 1)
      for (int32_t rb = 0; rb < q.blocks && in_list(at[1] + rb, a.merge_capacity); ++rb)
        a.merges[at[1] + rb] = TreeMerge{q.qs, q.nodes, rb, ns, at[0] + rb, q.blocks, 0, 0};
  }
  for (int32_t i = max(carry[1], 0) + tid; i < a.merge_capacity; i += kPlanThreads) a.merges[i].ns = 0;
}

// Workgroup 0 plans; the others copy the K/V rows of `per_wg` tokens each into
// the cache (kv.key may be null) and zero the rows of tokens outside every
// request.
__global__ __launch_bounds__(kPlanThreads) void tree_prologue_kernel(TreeArgs a, KvRowArgs kv, int32_t per_wg) {
  if (blockIdx.x == 0) {
    plan_items(a);
    return;
  }
  const int span = kPlanThreads / per_wg;
  const int64_t t = (static_cast<int64_t>(blockIdx.x) - 1) * per_wg + threadIdx.x / span;
  const int first = threadIdx.x % span;
  if (t >= a.num_tokens) return;
  if (kv.key) copy_kv_row(kv, t, first, span);
  if (t >= a.qsl[0] && t < a.qsl[a.num_requests]) return;
  char* const out = static_cast<char*>(a.out) + t * a.o_s0 * a.esize;
  const int chunks = a.head_dim * a.esize / 16;
  for (int i = first; i < a.num_q_heads * chunks; i += span)
    *reinterpret_cast<uint4*>(out + (i / chunks) * a.o_s1 * a.esize + 16 * (i % chunks)) = uint4{0, 0, 0, 0};
}

// The K/V rows of KV head h that the item's keys include, into the cache: every
// item writes what it reads, so that nobody waits for another workgroup. (Items
// that share keys write the same bytes.) The first split takes the nodes before
// its keys too, the last one those behind, so that all are written. The rows are
// 2 kChunks pieces of 16 bytes each; each thread's first piece is loaded ahead,
// beside the other loads that only the item is needed for. E: bytes of an
// element, W: waves of the workgroup.
struct OwnPiece {
  uint4 data;
  int64_t slot;
};

__device__ __forceinline__ int32_t own_begin(const TreeItem& item) {
  return item.split == 0 ? 0 : max(item.begin - item.prefix, 0);
}

__device__ __forceinline__ int32_t own_end(const TreeItem& item) {
  return item.split + 1 == item.ns ? item.nodes : min(item.end - item.prefix, item.nodes);
}

template <int D, int E>
__device__ __forceinline__ OwnPiece own_piece(const TreeArgs& a, const TreeItem& item, int h, int32_t x) {
  constexpr int kChunks = D * E / 16;
  const int32_t j = own_begin(item) + x / (2 * kChunks), c = x % (2 * kChunks);
  if (j >= own_end(item)) return OwnPiece{uint4{0, 0, 0, 0}, -1};
  const int64_t t = item.qs + j;
  const char* const row = c >= kChunks ? static_cast<const char*>(a.value) + E * (t * a.v_s0 + h * a.v_s1)
                                       : static_cast<const char*>(a.key) + E * (t * a.k_s0 + h * a.k_s1);
  return OwnPiece{*reinterpret_cast<const uint4*>(row + 16 * (c % kChunks)), a.slot_mapping[t]};
}

template <int D, int E, int W>
__device__ __forceinline__ void own_rows(const TreeArgs& a, const TreeItem& item, int h, OwnPiece p) {
  constexpr int kChunks = D * E / 16;
  const int32_t pieces = (own_end(item) - own_begin(item)) * 2 * kChunks;
  const int64_t slots = a.num_blocks * a.block_size;
  for (int32_t x = static_cast<int32_t>(threadIdx.x); x < pieces;) {
    const int32_t c = x % (2 * kChunks);
    if (p.slot >= 0 && p.slot < slots) {
      const int64_t block = slots <= UINT32_MAX ? static_cast<uint32_t>(p.slot) / static_cast<uint32_t>(a.block_size) : p.slot / a.block_size;
      char* const dst = const_cast<char*>(static_cast<const char*>(a.cache)) +
                        E * ((c >= kChunks ? a.c_s[0] : 0) + block * a.c_s[1] + (p.slot - block * a.block_size) * a.c_s[2] +
                             h * a.c_s[3]);
      *reinterpret_cast<uint4*>(dst + 16 * (c % kChunks)) = p.data;
    }
    x += 64 * W;
    if (x < pieces) p = own_piece<D, E>(a, item, h, x);
  }
  // In L2, where the loads behind the next barrier find them.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// Tokens outside every request, kOutside per workgroup of the grid's last rows:
// zeros, and their K/V rows into the cache as those of any token.
constexpr int kOutside = 64;

inline int64_t outside_wgs(const TreeArgs& a) {
  return ceil_div(a.num_tokens, static_cast<int64_t>(kOutside) * a.num_kv_heads);
}

__device__ __forceinline__ void outside_rows(const TreeArgs& a) {
  const int64_t wg = (static_cast<int64_t>(blockIdx.y) - a.capacity) * gridDim.x + blockIdx.x;
  const int64_t first = a.qsl[0], last = a.qsl[a.num_requests];
  const int64_t t0 = wg * kOutside, t1 = t0 + kOutside < a.num_tokens ? t0 + kOutside : a.num_tokens;
  if (t0 >= first && t1 <= last) return;
  const int E = a.esize, chunks = a.head_dim * E / 16;
  const int64_t slots = a.num_blocks * a.block_size;
  for (int64_t t = t0; t < t1; ++t) {
    if (t >= first && t < last) continue;
    char* const out = static_cast<char*>(a.out) + E * t * a.o_s0;
    for (int i = threadIdx.x; i < a.num_q_heads * chunks; i += blockDim.x)
      *reinterpret_cast<uint4*>(out + E * (i / chunks) * a.o_s1 + 16 * (i % chunks)) = uint4{0, 0, 0, 0};
    const int64_t slot = a.key ? a.slot_mapping[t] : -1;
    if (slot < 0 || slot >= slots) continue;
    char* const dst = const_cast<char*>(static_cast<const char*>(a.cache)) +
                      E * (slot / a.block_size * a.c_s[1] + slot % a.block_size * a.c_s[2]);
    for (int i = threadIdx.x; i < 2 * a.num_kv_heads * chunks; i += blockDim.x) {
      const bool is_value = i >= a.num_kv_heads * chunks;
      const int x = is_value ? i - a.num_kv_heads * chunks : i, h = x / chunks, c = x % chunks;
      const char* const row = is_value ? static_cast<const char*>(a.value) + E * (t * a.v_s0 + h * a.v_s1)
                                       : static_cast<const char*>(a.key) + E * (t * a.k_s0 + h * a.k_s1);
      *reinterpret_cast<uint4*>(dst + E * ((is_value ? a.c_s[0] : 0) + h * a.c_s[3]) + 16 * c) =
          *reinterpret_cast<const uint4*>(row + 16 * c);
    }
  }
}

// ---- merge of the splits --------------------------------------------------------------

// Rows of a row block that was split, P times 32 lanes each: every part takes
// splits of its own, scaled to the row's common maximum, and the parts add up in
// LDS. P = 4 where rows have many splits (a request alone: 60 of 30,000 keys took
// 12 us one after the other), else 1, which keeps four times as many rows in
// flight (72 row blocks in two splits each: 4 us, 12 with P = 4).
constexpr int kMergeGroups = 8;

template <typename T, int D, int P>
__global__ __launch_bounds__(32 * kMergeGroups) void tree_merge_kernel(TreeArgs a) {
  constexpr int E = D / 32;  // dims per lane
  constexpr int kFlight = 8;
  constexpr int kMergeRows = kMergeGroups / P;
  struct Dims {
    float v[E];
  };
  __shared__ float sum[P > 1 ? kMergeRows : 1][P][P > 1 ? D : 1];
  __shared__ float weight[P > 1 ? kMergeRows : 1][P];
  const int lane = threadIdx.x & 31, h = static_cast<int>(blockIdx.x), G = a.group;
  const int group = threadIdx.x >> 5, part = group % P, mine = group / P;
  const TreeMerge q = a.merges[blockIdx.y];
  if (q.ns < 2 || q.qs < 0 || q.rb < 0 || q.qs + q.nodes > a.num_tokens || q.slot < 0 || q.step < 1 ||
      q.slot + static_cast<int64_t>(q.ns - 1) * q.step >= a.slots)
    return;
  const int32_t row = static_cast<int32_t>(blockIdx.z) * kMergeRows + mine;
  const int32_t f = q.rb * a.rows + row;
  const bool live = f < q.nodes * G;
  const int64_t first = (static_cast<int64_t>(q.slot) * a.num_kv_heads + h) * a.rows + row;
  const int64_t step = static_cast<int64_t>(q.step) * a.num_kv_heads * a.rows;
  const int32_t s0 = static_cast<int32_t>(static_cast<int64_t>(q.ns) * part / P);
  const int32_t s1 = static_cast<int32_t>(static_cast<int64_t>(q.ns) * (part + 1) / P);
  float total = 0.f;
  Dims acc = {};
  if (live) {
    float top = -INFINITY;
    for (int32_t s = lane; s < q.ns; s += 32) top = fmaxf(top, a.ml[first + s * step].x);
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 32));
    for (int32_t base = s0; base < s1; base += kFlight) {
      Dims v[kFlight];
      float2 ml[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const int64_t at = first + (base + u < s1 ? base + u : s1 - 1) * step;
        v[u] = *reinterpret_cast<const Dims*>(a.acc + at * D + E * lane);
        ml[u] = a.ml[at];
      }
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        if (base + u >= s1) break;
        const float w = ml[u].x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml[u].x - top);
        total = __builtin_fmaf(ml[u].y, w, total);
#pragma unroll
        for (int e = 0; e < E; ++e) acc.v[e] = __builtin_fmaf(v[u].v[e], w, acc.v[e]);
      }
    }
  }
  if constexpr (P > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) sum[mine][part][E * lane + e] = acc.v[e];
    if (lane == 0) weight[mine][part] = total;
    __syncthreads();
    if (part != 0) return;
    total = 0.f;
    acc = {};
#pragma unroll
    for (int p = 0; p < P; ++p) {
      total += weight[mine][p];
#pragma unroll
      for (int e = 0; e < E; ++e) acc.v[e] += sum[mine][p][E * lane + e];
    }
  }
  if (!live) return;
  const int32_t node = f / G;
  T* const out = static_cast<T*>(a.out) + static_cast<int64_t>(q.qs + node) * a.o_s0 +
                 static_cast<int64_t>(h * G + f - node * G) * a.o_s1 + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) Elem<T>::store(out + e, acc.v[e] / total);
}

template <typename T, int D>
int launch_tree_merge(const TreeArgs& a, hipStream_t s) {
  if (a.merge_capacity == 0) return MVLLM_OK;
  const unsigned heads = static_cast<unsigned>(a.num_kv_heads), places = static_cast<unsigned>(a.merge_capacity);
  const unsigned groups = kMergeGroups, rows = static_cast<unsigned>(a.rows);
  if (a.many_splits)
    hipLaunchKernelGGL((tree_merge_kernel<T, D, 4>), dim3(heads, places, 4 * rows / groups), dim3(32 * groups), 0, s, a);
  else
    hipLaunchKernelGGL((tree_merge_kernel<T, D, 1>), dim3(heads, places, rows / groups), dim3(32 * groups), 0, s, a);
  MVLLM_LAUNCH_CHECK("tree_merge_kernel");
  return MVLLM_OK;
}

// Sizes of the plan and the partials for items of `rows` rows, no splits shorter
// than `shortest` (a multiple of 64), on a chip that runs `residents` of their
// workgroups per CU; bound to `workspace` (may be null). Returns the bytes.
inline int64_t tree_layout(TreeArgs& a, int32_t rows, int32_t shortest, int64_t residents, void* workspace) {
  const int64_t R = a.num_requests, N = a.num_tokens, reach = a.width * a.block_size;
  a.rows = rows;
  const int64_t blocks = N * a.group / a.rows + R;  // row blocks, at most
  const int64_t slots = residents * device_cu_count() / a.num_kv_heads;
  const int64_t target = slots > 1 ? slots : 1;
  a.target = static_cast<int32_t>(target);
  a.shortest = shortest;
  const bool splits = reach > shortest;
  // Where the split lengths come to fewer items than target, there are no more;
  // else to half of target and one more of each row block at most, and never
  // more than the reach holds. A row block that is split has at least two
  // items, and a whole share of target for each but one.
  int64_t capacity = blocks;
  if (splits) {
    const int64_t most = blocks + target / 2 > target ? blocks + target / 2 : target, per_block = ceil_div(reach, int64_t{shortest});
    capacity = blocks > 0 && per_block < most / blocks + 1 && per_block * blocks < most ? per_block * blocks : most;
  }
  a.capacity = static_cast<int32_t>(capacity < INT32_MAX ? capacity : INT32_MAX);  // (a grid's rows bound it: tree_grid_fits)
  a.slots = static_cast<int32_t>(!splits ? 0 : (capacity < 2 * target ? capacity : 2 * target));
  a.merge_capacity = static_cast<int32_t>(!splits ? 0 : (blocks < target ? blocks : target));
  a.many_splits = target >= 8 * blocks ? 1 : 0;
  // All items at once on the chip (two rounds at most, the second of short ones):
  // their order does not matter.
  a.self_planned = a.capacity <= 2 * slots && R <= 1024 ? 1 : 0;
  int64_t at = 0;
  char* const w = static_cast<char*>(workspace);
  auto take = [&](int64_t bytes) {
    char* const p = w ? w + at : nullptr;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  const int64_t slot_rows = static_cast<int64_t>(a.slots) * a.num_kv_heads * a.rows;
  if (!a.self_planned) a.items = reinterpret_cast<TreeItem*>(take(a.capacity * static_cast<int64_t>(sizeof(TreeItem))));
  a.merges = reinterpret_cast<TreeMerge*>(take(a.merge_capacity * static_cast<int64_t>(sizeof(TreeMerge))));
  a.ml = reinterpret_cast<float2*>(take(slot_rows * 8));
  a.acc = reinterpret_cast<float*>(take(slot_rows * a.head_dim * 4));
  return at;
}

// The prologue, where the items need one.
inline int launch_tree_prologue(const TreeArgs& a, const KvRowArgs* kv, hipStream_t s) {
  if (a.self_planned) return MVLLM_OK;
  KvRowArgs rows = {};
  int per_wg = 8;
  if (kv) {
    rows = *kv;
    per_wg = 1;
    while (per_wg < 64 && 2 * per_wg * 2 * static_cast<int64_t>(kv->chunks) <= kPlanThreads) per_wg *= 2;
  }
  const int64_t wgs = 1 + ceil_div(a.num_tokens, per_wg);
  hipLaunchKernelGGL(tree_prologue_kernel, dim3(static_cast<unsigned>(wgs)), dim3(kPlanThreads), 0, s, a, rows, per_wg);
  MVLLM_LAUNCH_CHECK("tree_prologue_kernel");
  return MVLLM_OK;
}

}  // namespace
}  // namespace mvllm
