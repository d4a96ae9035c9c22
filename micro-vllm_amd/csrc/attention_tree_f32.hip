// Tree attention in fp32 on the fp32 matrix cores: head_dim 64, 96 or 128, any
// block size.
//
// An item's rows are 16 (node, query head) pairs of a KV head; eight waves take
// every eighth tile of 16 keys each, straight from HBM into registers: V of the
// next tile beside this one's, K once its scores are done, the table entry two
// tiles ahead. S^T = K . Q^T and O^T += V^T . P^T on v_mfma_f32_16x16x4_f32: lane
// (col, grp) holds row col's scores of keys 4 grp .. 4 grp + 3, which are the
// second product's B operand as they stand, so no weight is rounded. Items,
// splits and their merge are those of the 16-bit kernel (tree_items.h).
//
// Small batches are bound by latency: a wave has a handful of tiles of ~1 us (64
// products of 32 cycles, the softmax, and the next tile's loads). 4 requests of
// 128 nodes over 1,024 keys, 32/8 heads, take 155 us, the matrix cores 40% busy
// (five vector instructions between two products) and the L2 at 7.8 TB/s, since
// each block of 16 rows reads its KV head's K/V for itself (38 MB as 1.2 GB); with
// 32 rows per item, which need all 256 registers, 184 us.
#include "tree_items.h"

namespace mvllm {
namespace {

constexpr int kF32Waves = 8;
constexpr int kF32Rows = 16;

// Each wave's accumulators and (maximum, sum).
template <int D>
constexpr size_t kF32Lds = kF32Waves * kF32Rows * (D + 4) * 4 + kF32Waves * kF32Rows * 8;

template <int D>
__global__ __launch_bounds__(64 * kF32Waves) void tree_f32_kernel(TreeArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int kStride = D + 4;
  constexpr int kSteps = D / 16;
  constexpr int VW = D % 64 == 0 ? 4 : 2;  // dims per V load of a lane
  constexpr int J = D / (16 * VW);
  typedef float vec_t __attribute__((ext_vector_type(VW)));
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int Hkv = a.num_kv_heads, G = a.group;
  const int h = static_cast<int>(blockIdx.x);
  if (a.self_planned && static_cast<int32_t>(blockIdx.y) >= a.capacity) {
    outside_rows(a);
    return;
  }
  const TreeItem item = a.self_planned
                            ? find_item<kF32Waves>(a, static_cast<int32_t>(blockIdx.y), blockIdx.x + blockIdx.y == 0, smem)
                            : a.items[blockIdx.y];
  const int32_t rows = item.nodes * G;
  // A list made from tokens that do not ascend may hold anything.
  if (item.r < 0 || item.r >= a.num_requests || item.qs < 0 || item.nodes < 1 || item.qs + item.nodes > a.num_tokens ||
      item.rb < 0 || item.rb >= (rows + kF32Rows - 1) / kF32Rows || (item.ns > 1 && (item.slot < 0 || item.slot >= a.slots)))
    return;
  const int64_t r = item.r;
  const int32_t prefix = item.prefix;
  const int64_t reach = a.width * a.block_size;
  const int32_t kend = item.end < reach ? item.end : static_cast<int32_t>(reach);

  OwnPiece own = {uint4{0, 0, 0, 0}, -1};
  if (a.self_planned && a.key) own = own_piece<D, 4>(a, item, h, static_cast<int32_t>(threadIdx.x));

  // ---- this lane's row
  const int32_t f = item.rb * kF32Rows + col;
  const bool row_ok = f < rows;
  const int32_t node = row_ok ? f / G : 0;
  const int hq = h * G + (row_ok ? f - node * G : 0);
  const int64_t tok = item.qs + node;
  float4_t qf[kSteps];
  {
    const float* const qp = static_cast<const float*>(a.q) + tok * a.q_s0 + static_cast<int64_t>(hq) * a.q_s1 + 4 * grp;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) qf[i] = *reinterpret_cast<const float4_t*>(qp + 16 * i);
  }
  int32_t start = kFar;
  if (row_ok) {
    const int64_t s = a.starts[tok];
    start = static_cast<int32_t>(s < 0 ? 0 : (s < kFar ? s : kFar - 1));
    if (start > prefix) start = prefix < 0 ? 0 : prefix;
  }
  const uint32_t* const mask_row = a.mask + tok * a.mask_stride;
  const int32_t mask_words = a.mask_bits >> 5;
  int32_t klo = item.begin;
  if (item.split == 0) klo = min(klo, wave_reduce_i(start, [](int32_t x, int32_t y) { return x < y ? x : y; }));
  if (klo < 0) klo = 0;
  klo = __builtin_amdgcn_readfirstlane(klo);
  const int32_t base = klo & ~15;
  const int32_t ntiles = kend > base ? (kend - base + 15) / 16 : 0;
  if (a.self_planned && a.key) own_rows<D, 4, kF32Waves>(a, item, h, own);
  __syncthreads();

  const float* const cache = static_cast<const float*>(a.cache) + static_cast<int64_t>(h) * a.c_s[3];
  const uint32_t bs = static_cast<uint32_t>(a.block_size);
  // A wave's tile: K of key `col` and V of keys 4 grp + s in registers. V of two
  // tiles is held in turn. Keys that do not exist read block 0.
  struct Key {
    int64_t block;  // -1: no key
    uint32_t row;   // in its block
  };
  auto look_up = [&](int32_t tile) {
    const int32_t pos = base + 16 * tile + col;
    Key k = {-1, 0};
    if (pos >= klo && pos < kend) {
      const uint32_t blk = static_cast<uint32_t>(pos) / bs;
      k.row = static_cast<uint32_t>(pos) - blk * bs;
      k.block = a.table[r * a.t_s0 + static_cast<int64_t>(blk) * a.t_s1];
    }
    return k;
  };
  auto offset = [&](const Key& k) {
    return k.block >= 0 && k.block < a.num_blocks ? k.block * a.c_s[1] + static_cast<int64_t>(k.row) * a.c_s[2] : int64_t{-1};
  };
  float4_t kt[kSteps];
  vec_t vt[2][4][J];
  auto load_k = [&](int64_t off) {
    const float* const kp = cache + (off >= 0 ? off : 0) + 4 * grp;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) kt[i] = *reinterpret_cast<const float4_t*>(kp + 16 * i);
  };
  auto load_v = [&](int64_t off, vec_t (&vt)[4][J]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int64_t voff = __shfl(off, 4 * grp + s, 64);
      const float* const vp = cache + a.c_s[0] + (voff >= 0 ? voff : 0) + VW * col;
#pragma unroll
      for (int j = 0; j < J; ++j) vt[s][j] = *reinterpret_cast<const vec_t*>(vp + 16 * VW * j);
    }
  };
  // Bit kk: this row sees key k0 + kk (of 16).
  auto visible = [&](int32_t k0) -> uint32_t {
    auto below = [](int32_t x) -> uint32_t { return x <= 0 ? 0u : (x >= 32 ? ~0u : (1u << x) - 1u); };
    uint32_t v = below(prefix - k0) & ~below(start - k0);
    const int32_t j0 = k0 - prefix;
    if (j0 > -16 && row_ok) {
      if (j0 < 0) {
        v |= mask_row[0] << -j0;
      } else {
        const int32_t w = j0 >> 5;
        const uint32_t lo = w < mask_words ? mask_row[w] : 0u, hi = w + 1 < mask_words ? mask_row[w + 1] : 0u;
        v |= __builtin_amdgcn_alignbit(hi, lo, j0 & 31);
      }
    }
    return v;
  };

  float4_t acc[J][VW];  // dims 16 VW j + VW m + c of row col, m = 4 grp + e
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int c = 0; c < VW; ++c) acc[j][c] = float4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  uint32_t mapped = 0;  // keys of this tile that exist
  int64_t next = -1;    // this lane's key of the next tile
  Key later = {-1, 0};  // and of the one after
  if (wave < ntiles) {
    const Key k0 = look_up(wave), k1 = look_up(wave + kF32Waves);
    later = look_up(wave + 2 * kF32Waves);
    const int64_t off = offset(k0);
    next = offset(k1);
    mapped = static_cast<uint32_t>(__ballot(off >= 0)) & 0xFFFFu;
    load_k(off);
    load_v(off, vt[0]);
  }
  auto step = [&](int32_t tile, vec_t (&vt)[4][J], vec_t (&vn)[4][J]) {
    load_v(next, vn);
    // Four chains, added pairwise: shorter ones round less than one of D terms.
    float4_t part[4] = {};
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        part[i & 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(kt[i][s], qf[i][s], part[i & 3], 0, 0, 0);
    const float4_t score = (part[0] + part[1]) + (part[2] + part[3]);
    load_k(next);
    const int32_t k0 = base + 16 * tile;
    const uint32_t vis = visible(k0) & mapped;
    float s[4], p[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = (vis >> (4 * grp + e)) & 1u ? score[e] * a.scale_log2 : -INFINITY;
    float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    top = max_xor32_f(max_xor16_f(top));
    const float mn = fmaxf(m, top);
    const float off = mn == -INFINITY ? 0.f : mn;
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = (vis >> (4 * grp + e)) & 1u ? exp2f(s[e] - off) : 0.f;
    const float sum = (p[0] + p[1]) + (p[2] + p[3]);
    // Where no maximum grew, what was summed stays as it is.
    if (__ballot(mn > m)) {
      const float alpha = m == -INFINITY ? 0.f : exp2f(m - off);
      l = m == -INFINITY ? l : l * alpha;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int c = 0; c < VW; ++c) acc[j][c] = m == -INFINITY ? acc[j][c] : acc[j][c] * alpha;
      m = mn;
    }
    l += sum;
    // Rows of V that are no keys hold anything: zeros. One that is not finite
    // must reach only the rows that see it: its tile is multiplied row by row.
    if (mapped != 0xFFFFu)
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const bool exists = (mapped >> (4 * grp + st)) & 1u;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int c = 0; c < VW; ++c) vt[st][j][c] = exists ? vt[st][j][c] : 0.f;
      }
    float finite = 0.f;
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int c = 0; c < VW; ++c) finite = __builtin_fmaf(vt[st][j][c], 0.f, finite);
    if (!__ballot(finite != finite)) {
#pragma unroll
      for (int st = 0; st < 4; ++st)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int c = 0; c < VW; ++c)
            acc[j][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(vt[st][j][c], p[st], acc[j][c], 0, 0, 0);
    } else {
      for (int x = 0; x < 16; ++x) {
        const uint32_t theirs = __shfl(vis, x, 64);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int c = 0; c < VW; ++c) {
            float4_t sums = acc[j][c];
#pragma unroll
            for (int st = 0; st < 4; ++st) {
              const bool sees = (theirs >> (4 * grp + st)) & 1u;
              sums = __builtin_amdgcn_mfma_f32_16x16x4f32(sees ? vt[st][j][c] : 0.f, p[st], sums, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][c][e] = col == x ? sums[e] : acc[j][c][e];
          }
      }
    }
    mapped = static_cast<uint32_t>(__ballot(next >= 0)) & 0xFFFFu;
    next = offset(later);
    later = look_up(tile + 3 * kF32Waves);
  };
  for (int32_t tile = wave; tile < ntiles; tile += 2 * kF32Waves) {
    step(tile, vt[0], vt[1]);
    if (tile + kF32Waves < ntiles) step(tile + kF32Waves, vt[1], vt[0]);
  }
  // ---- the waves' states
  float* const buf = reinterpret_cast<float*>(smem);  // [wave][row][kStride]
  float2* const ml = reinterpret_cast<float2*>(smem + kF32Waves * kF32Rows * kStride * 4);
  l = sum_xor32_f(sum_xor16_f(l));
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      vec_t v;
#pragma unroll
      for (int c = 0; c < VW; ++c) v[c] = acc[j][c][e];
      *reinterpret_cast<vec_t*>(buf + (wave * kF32Rows + col) * kStride + 16 * VW * j + VW * (4 * grp + e)) = v;
    }
  if (grp == 0) ml[wave * kF32Rows + col] = float2{m, l};
  __syncthreads();
  for (int i = tid; i < kF32Rows * D / 4; i += 64 * kF32Waves) {
    const int x = i / (D / 4), d = 4 * (i % (D / 4));
    const int32_t fx = item.rb * kF32Rows + x;
    if (fx >= rows) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kF32Waves; ++w) top = fmaxf(top, ml[w * kF32Rows + x].x);
    float total = 0.f;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kF32Waves; ++w) {
      const float2 theirs = ml[w * kF32Rows + x];
      const float weight = theirs.x == -INFINITY ? 1.f : exp2f(theirs.x - top);
      total = __builtin_fmaf(theirs.y, weight, total);
      const float4_t v = *reinterpret_cast<const float4_t*>(buf + (w * kF32Rows + x) * kStride + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(v[e], weight, o[e]);
    }
    if (item.ns > 1) {
      const int64_t row = (static_cast<int64_t>(item.slot) * Hkv + h) * kF32Rows + x;
      *reinterpret_cast<float4_t*>(a.acc + row * D + d) = o;
      if (d == 0) a.ml[row] = float2{top, total};
      continue;
    }
    const int32_t nx = fx / G;
    float* const out = static_cast<float*>(a.out) + static_cast<int64_t>(item.qs + nx) * a.o_s0 +
                       static_cast<int64_t>(h * G + fx - nx * G) * a.o_s1 + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] / total;  // nothing visible: 0 / 0, NaN
    *reinterpret_cast<float4_t*>(out) = o;
  }
}

template <int D>
int launch_f32(const TreeArgs& a, hipStream_t s) {
  static bool raised = false;  // per instantiation; the attribute is process-wide
  if (!raised) {
    MVLLM_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(tree_f32_kernel<D>),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kF32Lds<D>)));
    raised = true;
  }
  const int64_t wgs = a.capacity + (a.self_planned ? outside_wgs(a) : 0);
  hipLaunchKernelGGL(tree_f32_kernel<D>, dim3(static_cast<unsigned>(a.num_kv_heads), static_cast<unsigned>(wgs)),
                     dim3(64 * kF32Waves), kF32Lds<D>, s, a);
  MVLLM_LAUNCH_CHECK("tree_f32_kernel");
  return launch_tree_merge<float, D>(a, s);
}

}  // namespace

bool tree_f32_supported(const TreeArgs& a) {
  if (a.head_dim != 64 && a.head_dim != 96 && a.head_dim != 128) return false;
  if (a.num_requests < 1 || a.num_tokens * a.group >= (int64_t{1} << 30) || a.num_blocks >= INT32_MAX) return false;
  const int64_t strides[] = {a.q_s0, a.q_s1, a.o_s0, a.o_s1, a.c_s[0], a.c_s[1], a.c_s[2], a.c_s[3]};
  for (int64_t s : strides)
    if (s % 4 != 0) return false;
  return a.q_s2 == 1 && a.o_s2 == 1 && a.c_s[4] == 1 && aligned16(a.q) && aligned16(a.out) && aligned16(a.cache);
}

// Splits of 128 keys or more, with the merge that they need: 3 requests of 5 to
// 17 nodes over at most 272 keys take 16.0 us so and 18.5 with 384. One workgroup
// of 8 waves fits a CU's registers.
int64_t tree_f32_layout(TreeArgs& a, void* workspace) { return tree_layout(a, kF32Rows, 128, 1, workspace); }

int launch_tree_f32(const TreeArgs& a, const KvRowArgs* kv, hipStream_t s) {
  if (int rc = launch_tree_prologue(a, kv, s)) return rc;
  if (a.head_dim == 64) return launch_f32<64>(a, s);
  if (a.head_dim == 96) return launch_f32<96>(a, s);
  return launch_f32<128>(a, s);
}

}  // namespace mvllm
