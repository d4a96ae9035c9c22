// Tree attention on the matrix cores: bf16 / fp16, head_dim 64, 96 or 128,
// block sizes that are multiples of 16.
//
// The rows of a KV head are (node, query head of its group) pairs, row f ->
// node f / G, head f % G, so all G heads of all nodes read a K/V tile once. A
// wave owns 32 rows. A workgroup of four waves covers 32 RW rows with RW = 1, 2
// or 4 row waves; its 4 / RW key groups take the tiles of the item's keys in
// turn and are merged through LDS at its end. An item is (request, row block,
// split of the keys); the splits are chosen on the device from the lengths
// (plan_split) and merged by tree_merge_kernel.
//
// S^T = K . Q^T and O^T += V^T . P^T on v_mfma_f32_32x32x16: a lane holds 16 of
// 32 keys' scores of one row, so maxima and sums are in-lane plus one
// v_permlane32_swap, and P^T is the B operand of the second product as it
// stands. K and V pages of 16 keys go HBM -> LDS directly, a tile and a half
// ahead. Online softmax in the exp2 domain; the accumulators are rescaled only
// when a maximum has grown much. Scores, maxima, sums and the output stay fp32.
// The weights enter P.V as two values of the input type, the rounded weight and
// what it lacks: 16 bits in bf16, 22 in fp16 (lifted by 2^7, so that the second
// value's subnormals, 2^-24, are 2^-31 of the row's largest weight), as many as
// the paged decode kernel's pair, whatever else is in the batch. Rounded weights
// alone left 1.4 times the error of fp32 ones; the pair costs nothing in items of
// 32 or 64 rows (one request of 8 nodes 12.5 us, 16 of 24-32 48.4, both ways) and
// a second P.V product where the matrix cores are the bound: 64 requests of 64
// nodes over 1k-8k keys 377 -> 480 us, 24 of 40-90 in a window 37.6 -> 44.5, 4 of
// 20-27 over 16k-33k 96 -> 97-109.
//
// Which keys a row sees is a 32-bit word per 32 keys: cached positions from its
// start on, then its mask bits shifted to the tile. Tiles wholly among the
// cached keys that every row sees skip it.
#include <climits>
#include <cmath>

#include "mfma_tiles.h"
#include "tree_items.h"

namespace mvllm {
namespace {

constexpr int kTreeWaves = 4;

template <int RW> constexpr int kTreeTile = RW == 4 ? 64 : 32;  // keys of a tile
template <int D, int RW> constexpr int kTreeTileBytes = kTreeTile<RW> * 2 * D;
template <int D, int RW> constexpr size_t kTreeLds = size_t{4} * (kTreeWaves / RW) * kTreeTileBytes<D, RW>;  // two K, two V tiles per group

// Workgroups that share a CU: by LDS, and by the registers of head_dim's
// accumulators (168 at head_dim 64, else up to 256).
constexpr int tree_residents(int d, int rw) {
  const int by_lds = static_cast<int>((160 * 1024 - 64) / (4 * (kTreeWaves / rw) * (rw == 4 ? 64 : 32) * 2 * d));
  const int by_registers = d == 64 ? 3 : 2;
  return by_lds < by_registers ? by_lds : by_registers;
}
// Behind the tiles: a word of each wave (its first key, later the rows whose
// result is not finite), and with key groups its lanes' (maximum, sum).
template <int RW> constexpr size_t kRedBytes = 4 * kTreeWaves + (RW < kTreeWaves ? 8 * 64 * kTreeWaves : 0);

// ---- one row over its visible keys ------------------------------------------------

// Answered by one wave over [begin, end), with fp32 scores and weights: a lane
// scores one key of 64, then holds dims lane and lane + 64. For rows whose tiles
// gave something that is not finite, so its time does not count: a value of V
// that is not finite must reach only the rows that see it, and in the tiles it
// meets every row as 0 * inf.
template <typename T, int D>
__device__ __forceinline__ void tree_row(const TreeArgs& a, int64_t r, int64_t tok, int hq, int h, int64_t prefix,
                                         int32_t begin, int32_t end, float (&acc)[(D + 63) / 64], float& m, float& l) {
  constexpr int J = (D + 63) / 64;
  const int lane = threadIdx.x & 63;
  const uint16_t* const q = static_cast<const uint16_t*>(a.q) + tok * a.q_s0 + static_cast<int64_t>(hq) * a.q_s1;
  const uint16_t* const cache = static_cast<const uint16_t*>(a.cache) + static_cast<int64_t>(h) * a.c_s[3];
  const int64_t start = a.starts[tok];
#pragma unroll
  for (int j = 0; j < J; ++j) acc[j] = 0.f;
  m = -INFINITY;
  l = 0.f;
  for (int32_t base = begin; base < end; base += 64) {
    const int32_t p = base + lane;
    int64_t row = -1;
    if (p < end && (p < prefix ? p >= start : tree_bit(a, tok, p - prefix))) {
      const int64_t b = a.table[r * a.t_s0 + (p / a.block_size) * a.t_s1];
      if (b >= 0 && b < a.num_blocks) row = b * a.c_s[1] + (p % a.block_size) * a.c_s[2];
    }
    uint64_t seen = __ballot(row >= 0);
    if (!seen) continue;
    float s = -INFINITY;
    if (row >= 0) {
      float part[4] = {0.f, 0.f, 0.f, 0.f};
      for (int d = 0; d < D; d += 4)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          part[e] = __builtin_fmaf(Elem<T>::from_bits(q[d + e]) * a.scale_log2, Elem<T>::from_bits(cache[row + d + e]), part[e]);
      s = (part[0] + part[1]) + (part[2] + part[3]);
    }
    float top = s;
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    const float mn = fmaxf(m, top);
    const float off = mn == -INFINITY ? 0.f : mn;
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - off);
    const float w = row >= 0 ? exp2f(s - off) : 0.f;
    float sum = w;
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) sum += __shfl_xor(sum, x, 64);
    l = m == -INFINITY ? l + sum : l * alpha + sum;
#pragma unroll
    for (int j = 0; j < J; ++j) acc[j] = m == -INFINITY ? acc[j] : acc[j] * alpha;
    for (; seen; seen &= seen - 1) {
      const int k = __builtin_ctzll(seen);
      const int64_t vrow = __shfl(row, k, 64);
      const float wk = __shfl(w, k, 64);
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (lane + 64 * j < D)
          acc[j] = __builtin_fmaf(wk, Elem<T>::from_bits(cache[a.c_s[0] + vrow + lane + 64 * j]), acc[j]);
    }
    m = mn;
  }
}

// The kernel's arguments again, read from memory where they are used: what the
// tile loop does not need must not hold scalar registers throughout it.
__device__ __forceinline__ const TreeArgs& cold_args() {
  auto p = reinterpret_cast<const __attribute__((address_space(4))) TreeArgs*>(
      reinterpret_cast<uintptr_t>(__builtin_amdgcn_kernarg_segment_ptr()));
  asm volatile("" : "+s"(p));
  return *(const TreeArgs*)p;
}

// A value that the compiler cannot compute ahead of its place: what follows from
// it on the loop's rare paths would hold vector registers throughout the loop.
__device__ __forceinline__ int32_t here(int32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// ---- the tile kernel ----------------------------------------------------------------

template <typename T, int D, int RW>
__global__ __launch_bounds__(64 * kTreeWaves, tree_residents(D, RW)) void tree_tile_kernel(TreeArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int KG = kTreeWaves / RW;
  constexpr int TK = kTreeTile<RW>;
  constexpr int kTileBytes = kTreeTileBytes<D, RW>;
  constexpr int kPageBytes = 32 * D;    // 16 rows
  constexpr int PT = TK / 16;           // pages of a tile
  constexpr int PW = PT / RW;           // of which this wave loads
  constexpr int kSteps = D / 16;
  constexpr int kBlocks = D / 32;
  constexpr float kLift = std::is_same_v<T, f16_t> ? 7.f : 0.f;
  int32_t* const red = reinterpret_cast<int32_t*>(smem + kTreeLds<D, RW>);

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave / RW, rw = wave % RW;
  const int n = lane & 31, hh = lane >> 5;
  const int Hkv = a.num_kv_heads, G = a.group;
  const int h = static_cast<int>(blockIdx.x);
  if (a.self_planned && static_cast<int32_t>(blockIdx.y) >= a.capacity) {
    outside_rows(a);
    return;
  }
  const TreeItem item = a.self_planned ? find_item<kTreeWaves>(a, static_cast<int32_t>(blockIdx.y), blockIdx.x + blockIdx.y == 0, smem)
                                       : a.items[blockIdx.y];
  // A list made from tokens that do not ascend may hold anything.
  const int32_t rows = item.nodes * G;
  if (item.r < 0 || item.r >= a.num_requests || item.qs < 0 || item.nodes < 1 || item.qs + item.nodes > a.num_tokens ||
      item.rb < 0 || item.rb >= (rows + 32 * RW - 1) / (32 * RW) ||
      (item.ns > 1 && (item.slot < 0 || item.slot >= a.slots)))
    return;
  const int64_t r = item.r;
  const int32_t prefix = item.prefix;
  const int64_t reach = a.width * a.block_size;
  const int32_t kend = item.end < reach ? item.end : static_cast<int32_t>(reach);

  // Position of key group `grp`'s page `i` (of its own sequence of tiles).
  auto page_pos = [&](int32_t from, int32_t i) { return from + TK * (grp + KG * (i / PT)) + 16 * (i % PT); };
  struct Entry {
    int64_t block;
    int32_t group;  // -1: behind the item's keys
  };
  auto entry = [&](int32_t from, int32_t first) {
    const TreeArgs& c = cold_args();
    const int32_t pos = page_pos(from, first + here(lane));
    Entry e = {0, -1};
    if (pos < kend) {
      const uint32_t p16 = static_cast<uint32_t>(pos) >> 4, pages_per_block = static_cast<uint32_t>(c.block_size) >> 4;
      const uint32_t blk = p16 / pages_per_block;
      e.group = static_cast<int32_t>(p16 - blk * pages_per_block);
      e.block = c.table[r * c.t_s0 + static_cast<int64_t>(blk) * c.t_s1];
    }
    return e;
  };
  // What only the item is needed for is loaded at once: its own rows, the first
  // pages' entries (of the keys that its rows see if no start lies before its
  // own, which is rare) and below the starts and Q.
  const int32_t likely = (item.begin > 0 ? item.begin : 0) & ~15;
  OwnPiece own = {uint4{0, 0, 0, 0}, -1};
  if (a.self_planned && a.key) own = own_piece<D, 2>(a, item, h, tid);
  Entry e0 = entry(likely, 0), e1 = entry(likely, 64);

  // ---- this lane's row
  const int32_t f = (item.rb * RW + rw) * 32 + n;
  const bool row_ok = f < rows;
  const int32_t node = row_ok ? f / G : 0;
  const int hq = h * G + (row_ok ? f - node * G : 0);
  const int64_t tok = item.qs + node;
  int32_t start = kFar;
  if (row_ok) {
    const int64_t s = a.starts[tok];
    start = static_cast<int32_t>(s < 0 ? 0 : (s < kFar ? s : kFar - 1));
    if (start > prefix) start = prefix < 0 ? 0 : prefix;  // below kFar: the mark of a row that is none
  }
  const int32_t lo_min = __builtin_amdgcn_readfirstlane(wave_reduce_i(start, [](int32_t x, int32_t y) { return x < y ? x : y; }));
  const int32_t lo_max = __builtin_amdgcn_readfirstlane(
      wave_reduce_i(row_ok ? start : -1, [](int32_t x, int32_t y) { return x > y ? x : y; }));
  if (lane == 0) red[wave] = lo_min;

  // Q^T as B operands: lane (n, hh) holds row n, dims 16 st + 8 hh .. +7.
  short8_t qv[kSteps];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + tok * a.q_s0 + static_cast<int64_t>(hq) * a.q_s1 + 8 * hh;
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
      qv[st] = row_ok ? *reinterpret_cast<const short8_t*>(qp + 16 * st) : short8_t{0, 0, 0, 0, 0, 0, 0, 0};
  }
  __syncthreads();
  int32_t klo = item.begin;
  if (item.split == 0) {
#pragma unroll
    for (int w = 0; w < RW; ++w) klo = min(klo, red[w]);
  }
  if (klo < 0) klo = 0;
  klo = __builtin_amdgcn_readfirstlane(klo);
  const int32_t base = klo & ~15;
  const int32_t ntiles = kend > base ? (kend - base + TK - 1) / TK : 0;
  const int32_t trips = (ntiles + KG - 1) / KG;

  float16v oacc[kBlocks];
#pragma unroll
  for (int c = 0; c < kBlocks; ++c) oacc[c] = float16v{};
  float m = -INFINITY;  // the row's offset in the exp2 domain
  float l = 0.f;        // this lane's share of the row's sum

  const uint32_t lds0 = __builtin_amdgcn_groupstaticsize() + grp * 4 * kTileBytes;
  const uint32_t kaddr = lds0, vaddr = lds0 + 2 * kTileBytes;
  uint8_t* const vbuf = smem + grp * 4 * kTileBytes + 2 * kTileBytes;
  uint32_t klane[kSteps], vlane[kSteps];
#pragma unroll
  for (int st = 0; st < kSteps; ++st) klane[st] = kaddr + tile_off<D>(n, 2 * st + hh);
  {
    const int g4 = lane >> 4, jj = lane & 15;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < kBlocks; ++c) {
        const int row = 8 * u + 4 * (g4 >> 1) + (jj >> 2);
        const int dim = 32 * c + 16 * (g4 & 1) + 4 * (jj & 3);
        vlane[kBlocks * u + c] = vaddr + tile_off<D>(row, dim >> 3) + 2 * (dim & 7);
      }
  }
#pragma unroll
  for (int x = 0; x < kSteps; ++x) asm volatile("" : "+v"(klane[x]), "+v"(vlane[x]));
  // Load i of a page covers its 16-byte chunks 64 i .. 64 i + 63; lane l lands
  // at chunk 64 i + l and fetches what the permutation puts there.
  auto page_row = [&](int i) { return (64 * i + lane) / (D / 8); };
  uint32_t dma_off[kBlocks];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) {
    const int rip = page_row(i);
    dma_off[i] = static_cast<uint32_t>(2 * (rip * a.c_s[2] + 8 * row_logical<D>(rip, (64 * i + lane) % (D / 8))));
  }
  const char* const cache_head = static_cast<const char*>(a.cache) + 2 * static_cast<int64_t>(h) * a.c_s[3];
  const uint32_t blk_bytes = static_cast<uint32_t>(2 * a.c_s[1]);
  const uint32_t grp_bytes = static_cast<uint32_t>(32 * a.c_s[2]);
  const int64_t plane_bytes = 2 * a.c_s[0];

  // 128 pages' entries at a time, two per lane: (block << 4) | 16-row group, or
  // -1 for one that is not mapped or lies behind the item's keys.
  int32_t ids[2] = {-1, -1};
  uint64_t mapped[2] = {0, 0};
  int32_t looked_up = 0;  // trips that look-ups have covered
  auto look_up = [&](const Entry& e0, const Entry& e1) {
    const int64_t blocks = cold_args().num_blocks;
    ids[0] = e0.group >= 0 && e0.block >= 0 && e0.block < blocks ? static_cast<int32_t>((e0.block << 4) | e0.group) : -1;
    ids[1] = e1.group >= 0 && e1.block >= 0 && e1.block < blocks ? static_cast<int32_t>((e1.block << 4) | e1.group) : -1;
    mapped[0] = __ballot(ids[0] >= 0);
    mapped[1] = __ballot(ids[1] >= 0);
  };
  constexpr int kTrips = 128 / PT;  // trips whose pages one look-up covers

  // Where one trip's pages lie, and which of all its tile's pages are mapped.
  // Load x of kHalfLoads moves 1 KiB of this wave's K (or V) pages.
  constexpr int kHalfLoads = PW * kBlocks;
  struct Pages {
    const char* k[PW];
    uint32_t bits;
  };
  auto pages_of = [&](int32_t trip) {
    const int32_t at = trip % kTrips * PT;
    if (trip >= looked_up) {
      look_up(entry(base, trip * PT), entry(base, trip * PT + 64));
      looked_up += kTrips;
    }
    Pages p;
    p.bits = static_cast<uint32_t>((at < 64 ? mapped[0] : mapped[1]) >> (at & 63));
#pragma unroll
    for (int j = 0; j < PW; ++j) {
      // A page that is not mapped reads block 0, so that every trip has as many
      // loads: its scores are masked, its values zeroed when they have landed.
      const int32_t lane_at = (at & 63) + rw * PW + j;
      const int32_t id0 = __builtin_amdgcn_readlane(ids[0], lane_at), id1 = __builtin_amdgcn_readlane(ids[1], lane_at);
      const int32_t id = at < 64 ? id0 : id1;
      const uint32_t u = id >= 0 ? static_cast<uint32_t>(id) : 0u;
      // (64 bits: one group fits 32, fifteen need not.)
      p.k[j] = cache_head + static_cast<uint64_t>(u >> 4) * blk_bytes + static_cast<uint64_t>(u & 15u) * grp_bytes;
    }
    return p;
  };
  auto load_k = [&](const Pages& p, int stage, int x) {
    const int j = x / kBlocks, i = x % kBlocks;
    lds_dma_load16_sbase(p.k[j], dma_off[i], kaddr + stage * kTileBytes + (rw * PW + j) * kPageBytes + i * 1024);
  };
  auto load_v = [&](const Pages& p, int stage, int x) {
    const int j = x / kBlocks, i = x % kBlocks;
    lds_dma_load16_sbase(p.k[j] + plane_bytes, dma_off[i], vaddr + stage * kTileBytes + (rw * PW + j) * kPageBytes + i * 1024);
  };
  // The key group's waves at one point, their LDS reads and writes done.
  auto group_sync = [&] {
    if constexpr (RW > 1) {
      __syncthreads();
    } else {
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      wave_lds_sync();
    }
  };
  // Rows of this wave's pages outside [klo, kend) or not mapped hold anything:
  // zeros.
  auto fix_v = [&](int32_t trip, int stage, uint32_t page_bits) {
#pragma unroll
    for (int j = 0; j < PW; ++j) {
      const int page = rw * PW + j;
      const int32_t pos = base + TK * (grp + KG * trip) + 16 * page;
      const bool gone = !((page_bits >> page) & 1u);
      if (pos >= klo && pos + 16 <= kend && !gone) continue;
      uint8_t* const v = vbuf + stage * kTileBytes + page * kPageBytes;
      const int lane_ = here(lane);
      const uint32_t zero = static_cast<uint32_t>(here(0));
      for (int i = 0; i < kBlocks; ++i) {
        const int32_t p = pos + (64 * i + lane_) / (D / 8);
        if (gone || p < klo || p >= kend) *reinterpret_cast<uint4*>(v + i * 1024 + 16 * lane_) = uint4{zero, zero, zero, zero};
      }
    }
  };
  // Bit kk: this row sees key k0 + kk.
  auto visible = [&](int32_t k0, uint32_t page_bits) -> uint32_t {
    auto below = [](int32_t x) -> uint32_t { return x <= 0 ? 0u : (x >= 32 ? ~0u : (1u << x) - 1u); };
    uint32_t v = below(prefix - k0) & ~below(start - k0);
    const int32_t j0 = k0 - prefix;
    if (j0 > -32) {
      const TreeArgs& c = cold_args();
      const uint32_t* const mask_row = c.mask + static_cast<int64_t>(here(static_cast<int32_t>(tok))) * c.mask_stride;
      const int32_t mask_words = c.mask_bits >> 5;
      uint32_t tree = 0;
      if (start < kFar) {
        if (j0 < 0) {
          tree = mask_row[0] << -j0;
        } else {
          const int32_t w = j0 >> 5, sh = j0 & 31;
          const uint32_t lo = w < mask_words ? mask_row[w] : 0u, hi = w + 1 < mask_words ? mask_row[w + 1] : 0u;
          tree = __builtin_amdgcn_alignbit(hi, lo, sh);
        }
      }
      v |= tree;
    }
    v &= below(kend - k0);
    v &= ~below(klo - k0);
    if (!(page_bits & 1u)) v &= 0xFFFF0000u;
    if (!(page_bits & 2u)) v &= 0x0000FFFFu;
    return v;
  };

  // P^T of 32 keys as MFMA B operands: the rounded weights, and what they lack.
  struct Weights {
    short8_t part[2][2];
  };
  auto read_k = [&](int hb, int stage, short8_t (&kf)[kSteps]) {
#pragma unroll
    for (int st = 0; st < kSteps; ++st) kf[st] = lds_read_b128_at(klane[st] + stage * kTileBytes + 2 * kPageBytes * hb);
  };
  auto read_v = [&](int hb, int q, int stage, short4v (&vq)[kSteps]) {
#pragma unroll
    for (int x = 0; x < kSteps; ++x)
      vq[x] = lds_read_tr16_at(vlane[x] + stage * kTileBytes + 2 * kPageBytes * hb + kPageBytes * q);
  };
  // S^T of half hb, in the first half with the V loads of the next trip between
  // its products: issued in a burst they would stall the wave.
  auto scores = [&](const short8_t (&kf)[kSteps], int hb, const Pages& p, int stage) {
    float16v s = float16v{};
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      s = Mma32<T>::mma(kf[st], qv[st], s);
      const int x0 = hb == 0 ? kHalfLoads * st / kSteps : 0, x1 = hb == 0 ? kHalfLoads * (st + 1) / kSteps : 0;
      if (x1 > x0) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = x0; x < x1; ++x) load_v(p, stage, x);
      if (x1 > x0) __builtin_amdgcn_sched_barrier(0);
    }
    return s;
  };
  auto hide = [&](float16v& s, uint32_t vis) {
    const uint32_t mine = vis >> (4 * here(hh));
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = (mine >> (8 * (i >> 2) + (i & 3))) & 1u ? s[i] : -INFINITY;
  };
  // O^T += V^T . P^T of 32 keys; `between(i)` follows pair i of 2 kBlocks products.
  auto accumulate = [&](const short4v (&vf)[2][kSteps], const Weights& p, auto&& between) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int c = 0; c < kBlocks; ++c) {
        const short4v lo4 = vf[q][c], hi4 = vf[q][kBlocks + c];
        const short8_t av = {lo4[0], lo4[1], lo4[2], lo4[3], hi4[0], hi4[1], hi4[2], hi4[3]};
        oacc[c] = Mma32<T>::mma(av, p.part[0][q], oacc[c]);
        oacc[c] = Mma32<T>::mma(av, p.part[1][q], oacc[c]);
        between(q * kBlocks + c);
      }
  };
  // Weights against the offset `off`; returns this lane's sum.
  auto weigh = [&](const float16v& s, float off, Weights& p) {
    float sum = 0.f;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t w[2][4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * q + 2 * x], a.scale_log2, -off));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * q + 2 * x + 1], a.scale_log2, -off));
        sum += p0 + p1;
        w[0][x] = Mma32<T>::pack2(p0, p1);
        const float2v rest = Mma32<T>::less(p0, p1, w[0][x]);
        w[1][x] = Mma32<T>::pack2(rest[0], rest[1]);
      }
#pragma unroll
      for (int y = 0; y < 2; ++y)
        p.part[y][q] = __builtin_bit_cast(short8_t, uint4{w[y][0], w[y][1], w[y][2], w[y][3]});
    }
    return sum;
  };
  // A new offset where a maximum grew by more than 2^8 over the current one,
  // then the weights against it.
  auto weigh_anew = [&](const float16v& s, Weights& p) {
    float mx = fmaxf(s[0], s[1]);
#pragma unroll
    for (int i = 2; i < 16; ++i) mx = fmaxf(mx, s[i]);
    mx = max_with_partner(mx) * a.scale_log2;
    const bool grow = mx > m + (8.f + kLift);
    const float m_new = grow ? mx - kLift : m;
    const float alpha = grow ? __builtin_amdgcn_exp2f(m - m_new) : 1.f;
    l *= alpha;
#pragma unroll
    for (int c = 0; c < kBlocks; ++c) oacc[c] *= alpha;
    m = m_new;
    return weigh(s, m == -INFINITY ? 0.f : m, p);
  };
  // The weights are first taken against the current offset, without a maximum,
  // and taken again if a row has no offset yet or they sum too high (or to no
  // number): below that sum none overflows 16 bits or the fp32 sums.
  constexpr float kMostSum = kLift > 0.f ? 32768.f : 4096.f;
  auto softmax = [&](const float16v& s, Weights& p, auto&& work) {
    work();  // matrix instructions that do not need the weights, in one block with them
    float sum = weigh(s, m, p);
    if (__ballot(m == -INFINITY || !(sum <= kMostSum))) sum = weigh_anew(s, p);
    l += sum;
  };
  // One trip. Its K has landed when it starts, its V when the weights need it;
  // the V of the next trip is loaded into the stage that the last trip's P.V has
  // left, the K of the one after it into the stage that this trip's scores leave.
  // So each load has a trip and a half to land and three of the four tiles in
  // LDS are in flight: with all of the next trip's loads issued at its start, one
  // trip ahead, the loads alone reached 4.4 TB/s. Nothing skips a tile, whatever
  // its rows see: a path around it would make the compiler copy the accumulators.
  // Behind the last trip its pages are read again (from L2), into stages that
  // nobody reads.
  Pages ahead1 = {}, ahead2 = {};  // pages of the next trip and the one after
  uint32_t page_bits = 0, next_bits = 0;  // of this trip and the next
  auto trip_body = [&](int32_t trip, auto stage_c) {
    constexpr int stage = decltype(stage_c)::value;
    constexpr int H = TK / 32;
    const int32_t k0 = base + TK * (grp + KG * trip);
    bool edge[H];
#pragma unroll
    for (int hb = 0; hb < H; ++hb) {
      const int32_t k = k0 + 32 * hb;
      edge[hb] = k < lo_max || k < klo || k + 32 > prefix || k + 32 > kend || ((page_bits >> (2 * hb)) & 3u) != 3u;
    }
    auto masked = [&](float16v& s, int hb) {
      if (!edge[hb]) return;
      asm volatile("");  // interior tiles skip the masking
      hide(s, visible(k0 + 32 * hb, (page_bits >> (2 * hb)) & 3u));
    };
    auto scored = [&](int hb) {
      short8_t kf[kSteps];
      read_k(hb, stage, kf);
      __builtin_amdgcn_sched_barrier(0);
      return scores(kf, hb, ahead1, stage ^ 1);
    };
    auto v_landed = [&] {
      compiler_fence();
      wait_vmcnt<2 * kHalfLoads>();
      compiler_fence();
      fix_v(trip, stage, page_bits);
      group_sync();
      ahead2 = pages_of(trip + 2 < trips ? trip + 2 : trips - 1);
    };
    auto next_k = [&](int i) {
#pragma unroll
      for (int x = kHalfLoads * i / (2 * kBlocks); x < kHalfLoads * (i + 1) / (2 * kBlocks); ++x) load_k(ahead2, stage, x);
    };
    compiler_fence();
    wait_vmcnt<2 * kHalfLoads>();
    compiler_fence();
    group_sync();
    short4v vf[2][kSteps];
    Weights p0;
    float16v s0 = scored(0);
    if constexpr (H == 1) {
      __builtin_amdgcn_sched_barrier(0);
      masked(s0, 0);
      softmax(s0, p0, [] {});
      __builtin_amdgcn_sched_barrier(0);
      v_landed();
      read_v(0, 0, stage, vf[0]);
      read_v(0, 1, stage, vf[1]);
      accumulate(vf, p0, next_k);
    } else {
      // The first half's softmax beside the second one's scores, the second
      // half's beside the first one's P.V: blocks that the compiler interleaves.
      short8_t kf[kSteps];
      read_k(1, stage, kf);
      __builtin_amdgcn_sched_barrier(0);
      masked(s0, 0);
      float16v s1;
      softmax(s0, p0, [&] { s1 = scores(kf, 1, ahead1, stage ^ 1); });
      __builtin_amdgcn_sched_barrier(0);
      v_landed();
      Weights p1;
      read_v(0, 0, stage, vf[0]);
      read_v(0, 1, stage, vf[1]);
      __builtin_amdgcn_sched_barrier(0);
      masked(s1, 1);
      softmax(s1, p1, [&] { accumulate(vf, p0, next_k); });
      __builtin_amdgcn_sched_barrier(0);
      read_v(1, 0, stage, vf[0]);
      read_v(1, 1, stage, vf[1]);
      __builtin_amdgcn_sched_barrier(0);
      accumulate(vf, p1, [](int) {});
    }
    ahead1 = ahead2;
    page_bits = next_bits;
    next_bits = ahead2.bits;
  };
  if (trips > 0) {
    if (base != likely) e0 = entry(base, 0), e1 = entry(base, 64);
    // All waves' rows are written before a page is read.
    if (a.self_planned && a.key) {
      own_rows<D, 2, kTreeWaves>(a, item, h, own);
      __syncthreads();
    }
    look_up(e0, e1);
    looked_up = kTrips;
    const Pages first = pages_of(0);
    ahead1 = pages_of(trips > 1 ? 1 : 0);
    page_bits = first.bits;
    next_bits = ahead1.bits;
#pragma unroll
    for (int x = 0; x < kHalfLoads; ++x) load_k(first, 0, x);
#pragma unroll
    for (int x = 0; x < kHalfLoads; ++x) load_v(first, 0, x);
#pragma unroll
    for (int x = 0; x < kHalfLoads; ++x) load_k(ahead1, 1, x);
  } else if (a.self_planned && a.key) {
    own_rows<D, 2, kTreeWaves>(a, item, h, own);
  }
  int32_t trip = 0;
  for (; trip + 1 < trips; trip += 2) {
    trip_body(trip, std::integral_constant<int, 0>{});
    trip_body(trip + 1, std::integral_constant<int, 1>{});
  }
  if (trip < trips) trip_body(trip, std::integral_constant<int, 0>{});
  l = sum_with_partner(l);
  wait_vmcnt<0>();  // no load may land in LDS that others use next
  compiler_fence();

  // ---- key groups: the waves of the same rows add up PB of the output's blocks
  // of 32 dims each (one wave alone took 3,400 cycles
  // for four groups and 3,500 for its rows: one request of 8 nodes 11.7 us, 10.7 so)
  constexpr int PB = (kBlocks + KG - 1) / KG;
  const int first_block = KG > 1 ? grp * PB : 0;
  auto mine = [&](int i) { return kBlocks % KG == 0 || first_block + i < kBlocks; };
  float16v merged[PB];
  auto& out = [&]() -> auto& {
    if constexpr (KG > 1) return merged;
    else return oacc;
  }();
  if constexpr (KG > 1) {
    constexpr int kWaveBytes = 64 * 16 * kBlocks * 4;
    static_assert(kWaveBytes * kTreeWaves <= static_cast<int>(kTreeLds<D, RW>), "merge fits the tiles");
    float2* const ml = reinterpret_cast<float2*>(smem + kTreeLds<D, RW> + 4 * kTreeWaves);
    __syncthreads();  // every wave is done with its tiles
    float4* const to = reinterpret_cast<float4*>(smem + wave * kWaveBytes);
#pragma unroll
    for (int c = 0; c < kBlocks; ++c)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        to[(4 * c + q) * 64 + lane] = float4{oacc[c][4 * q], oacc[c][4 * q + 1], oacc[c][4 * q + 2], oacc[c][4 * q + 3]};
    ml[wave * 64 + lane] = float2{m, l};
    __syncthreads();
    float2 state[KG];
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      state[g] = ml[(g * RW + rw) * 64 + lane];
      top = fmaxf(top, state[g].x);
    }
    l = 0.f;
#pragma unroll
    for (int i = 0; i < PB; ++i) out[i] = float16v{};
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      const float w = state[g].x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(state[g].x - top);
      l = __builtin_fmaf(state[g].y, w, l);
      const float4* const theirs = reinterpret_cast<const float4*>(smem + (g * RW + rw) * kWaveBytes);
#pragma unroll
      for (int i = 0; i < PB; ++i) {
        if (!mine(i)) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 v = theirs[(4 * (first_block + i) + q) * 64 + lane];
          out[i][4 * q] = __builtin_fmaf(v.x, w, out[i][4 * q]);
          out[i][4 * q + 1] = __builtin_fmaf(v.y, w, out[i][4 * q + 1]);
          out[i][4 * q + 2] = __builtin_fmaf(v.z, w, out[i][4 * q + 2]);
          out[i][4 * q + 3] = __builtin_fmaf(v.w, w, out[i][4 * q + 3]);
        }
      }
    }
    m = top;
  }

  // ---- rows with something that is not finite
  const TreeArgs& c_ = cold_args();
  const int32_t f_ = (item.rb * RW + rw) * 32 + here(n);
  const bool ok = f_ < rows;
  const int32_t node_ = ok ? f_ / G : 0;
  float zero = 0.f;
#pragma unroll
  for (int i = 0; i < PB; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) zero = __builtin_fmaf(out[i][e], 0.f, zero);
  const uint64_t bad = __ballot(zero != zero && ok);
  uint32_t redo = static_cast<uint32_t>(bad) | static_cast<uint32_t>(bad >> 32);
  if constexpr (KG > 1) {
    if (lane == 0) red[wave] = static_cast<int32_t>(redo);
    __syncthreads();
#pragma unroll
    for (int g = 0; g < KG; ++g) redo |= static_cast<uint32_t>(red[g * RW + rw]);
    redo = __builtin_amdgcn_readfirstlane(redo);
  }
  const bool store_row = ok && !((redo >> n) & 1u);
  constexpr int J = (D + 63) / 64;
  if (item.ns > 1) {
    const int64_t first_row = (static_cast<int64_t>(item.slot) * Hkv + h) * (32 * RW) + rw * 32;
    if (store_row) {
      float* const to = c_.acc + (first_row + n) * D;
#pragma unroll
      for (int i = 0; i < PB; ++i) {
        if (!mine(i)) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float4*>(to + 32 * (first_block + i) + 8 * q + 4 * hh) =
              float4{out[i][4 * q], out[i][4 * q + 1], out[i][4 * q + 2], out[i][4 * q + 3]};
      }
      if (hh == 0 && grp == 0) c_.ml[first_row + n] = float2{m, l};
    }
    for (; redo; redo &= redo - 1) {
      const int x = __builtin_ctz(redo);
      if (x % KG != grp) continue;
      const int32_t fx = (item.rb * RW + rw) * 32 + x;
      float acc[J], mr, lr;
      tree_row<T, D>(c_, r, item.qs + fx / G, h * G + fx % G, h, prefix, klo, kend, acc, mr, lr);
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (lane + 64 * j < D) c_.acc[(first_row + x) * D + lane + 64 * j] = acc[j];
      if (lane == 0) c_.ml[first_row + x] = float2{mr, lr};
    }
    return;
  }
  const float inv = 1.f / l;  // nothing visible: 0 * inf, NaN
  uint16_t* const op = static_cast<uint16_t*>(c_.out) + static_cast<int64_t>(item.qs + node_) * c_.o_s0 +
                       static_cast<int64_t>(h * G + f_ - node_ * G) * c_.o_s1;
#pragma unroll
  for (int i = 0; i < PB; ++i) {
    if (!mine(i)) continue;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      // Lanes n and n + 32 hold the halves of each group of 8 dims; one swap
      // per word gives lane hh the whole group 2 p + hh.
      uint32_t w[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int q = 2 * p + u;
        w[u][0] = Mma32<T>::pack2(out[i][4 * q] * inv, out[i][4 * q + 1] * inv);
        w[u][1] = Mma32<T>::pack2(out[i][4 * q + 2] * inv, out[i][4 * q + 3] * inv);
      }
      uint32_t got[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t send = hh ? w[0][k] : w[1][k];
        const auto r2 = __builtin_amdgcn_permlane32_swap(send, send, false, false);
        got[k] = hh ? r2[0] : r2[1];
      }
      const uint4 piece = hh ? uint4{got[0], got[1], w[1][0], w[1][1]} : uint4{w[0][0], w[0][1], got[0], got[1]};
      if (store_row) *reinterpret_cast<uint4*>(op + 32 * (first_block + i) + 8 * (2 * p + hh)) = piece;
    }
  }
  for (; redo; redo &= redo - 1) {
    const int x = __builtin_ctz(redo);
    if (x % KG != grp) continue;
    const int32_t fx = (item.rb * RW + rw) * 32 + x;
    const int64_t t = item.qs + fx / G;
    float acc[J], mr, lr;
    tree_row<T, D>(c_, r, t, h * G + fx % G, h, prefix, klo, kend, acc, mr, lr);
    uint16_t* const row = static_cast<uint16_t*>(c_.out) + t * c_.o_s0 + static_cast<int64_t>(h * G + fx % G) * c_.o_s1;
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (lane + 64 * j < D) row[lane + 64 * j] = static_cast<uint16_t>(Elem<T>::to_bits(acc[j] / lr));
  }
}

template <typename T, int D, int RW>
int launch_tiles(const TreeArgs& a, hipStream_t s) {
  constexpr size_t kLds = kTreeLds<D, RW> + kRedBytes<RW>;
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
  static bool raised = false;  // per instantiation; the attribute is process-wide
  if (!raised) {
    MVLLM_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(tree_tile_kernel<T, D, RW>),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kLds)));
    raised = true;
  }
  const unsigned heads = static_cast<unsigned>(a.num_kv_heads);
  const int64_t wgs = a.capacity + (a.self_planned ? outside_wgs(a) : 0);
  hipLaunchKernelGGL((tree_tile_kernel<T, D, RW>), dim3(heads, static_cast<unsigned>(wgs)),
                     dim3(64 * kTreeWaves), kLds, s, a);
  MVLLM_LAUNCH_CHECK("tree_tile_kernel");
  return launch_tree_merge<T, D>(a, s);
}

template <typename T, int D>
int launch_rows(const TreeArgs& a, hipStream_t s) {
  switch (a.rows) {
    case 32: return launch_tiles<T, D, 1>(a, s);
    case 64: return launch_tiles<T, D, 2>(a, s);
    default: return launch_tiles<T, D, 4>(a, s);
  }
}

template <typename T>
int launch_dims(const TreeArgs& a, hipStream_t s) {
  if (a.head_dim == 64) return launch_rows<T, 64>(a, s);
  if (a.head_dim == 96) return launch_rows<T, 96>(a, s);
  return launch_rows<T, 128>(a, s);
}

}  // namespace

bool tree_tiles_supported(const TreeArgs& a, int32_t dtype) {
  if (dtype != MVLLM_DTYPE_BF16 && dtype != MVLLM_DTYPE_F16) return false;
  if ((a.head_dim != 64 && a.head_dim != 96 && a.head_dim != 128) || a.block_size % 16 != 0 || a.block_size > 256)
    return false;
  // Page entries pack (block id, 16-row group); strides within 32-bit offsets.
  if (a.num_blocks >= (int64_t{1} << 27) || 2 * a.c_s[1] >= (int64_t{1} << 32) || 32 * a.c_s[2] >= (int64_t{1} << 32))
    return false;
  if (a.num_requests < 1 || a.num_tokens * a.group >= (int64_t{1} << 30)) return false;
  const int64_t strides[] = {a.q_s0, a.q_s1, a.o_s0, a.o_s1, a.c_s[0], a.c_s[1], a.c_s[2], a.c_s[3]};
  for (int64_t s : strides)
    if (s % 8 != 0) return false;
  return a.q_s2 == 1 && a.o_s2 == 1 && a.c_s[4] == 1 && aligned16(a.q) && aligned16(a.out) && aligned16(a.cache);
}

int64_t tree_tiles_layout(TreeArgs& a, int64_t max_nodes, void* workspace) {
  // Rows of an item by the largest tree, if the caller knows it, else by the
  // average one.
  const int64_t most = (max_nodes > 0 ? max_nodes : ceil_div(a.num_tokens, a.num_requests)) * a.group;
  const int rw = most <= 32 ? 1 : (most <= 64 ? 2 : 4);
  // Splits of 384 keys or more: 32 nodes of one request over 2,000 keys take 20.5
  // us so, 25.6 with 512 and 20.3 with 128, but a table that holds no more than
  // 384 keys needs no merge (12.3 us for 8 nodes over 320 instead of 13.4; a wider
  // table has its merge launched whatever the lengths, which the host does not know).
  return tree_layout(a, 32 * rw, 384, tree_residents(a.head_dim, rw), workspace);
}

int launch_tree_tiles(const TreeArgs& a, int32_t dtype, const KvRowArgs* kv, hipStream_t s) {
  if (int rc = launch_tree_prologue(a, kv, s)) return rc;
  return dtype == MVLLM_DTYPE_BF16 ? launch_dims<bf16_t>(a, s) : launch_dims<f16_t>(a, s);
}

}  // namespace mvllm
