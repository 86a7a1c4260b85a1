// Attention over a paged cache held in 8 bits with one scale per block and head,
// for few rows per sequence (decoding, checking drafted tokens).
//
// Mathematics.  With codes k, v and scales a, b per (block, head):
//   S[t] = scale * a(t) * (q . k[t]),   o = sum_t 2^(S'[t] - m) b(t) v[t] / sum_t 2^(S'[t] - m)
// with S' = S * log2(e).  The 8-bit tensor cores see the codes as they lie in the cache, so no
// code is ever converted: what multiplies them is split into three 8-bit terms instead, and
// there is little of that (a handful of rows of q, and their weights).
//   E4M3: x = x1 + x2 / 16 + x3 / 256 ... with x1 = e4m3(x), x2 = e4m3(16 (x - x1)), ...: each term
//     rounds off 2^-4 of what it is given, three leave 2^-12 of a value, or 2^-18 in all.
//     A row of q is scaled to a maximum in [2^7, 2^8) (three terms), weights to at most 2^8 (four).
//   int8: x = x1 2^16 + x2 2^8 + x3, a whole number in balanced base 256: q to a maximum in
//     [2^21, 2^22), weights to 127 * 2^24 (four digits).  The products are summed exactly in s32.
// So a value of q (bf16: 8 bits, f16: 11) goes in exactly, or to 2^-22 (int8) or 2^-26 (E4M3) of its row's
// largest where it is that much smaller, and a weight is good to 2^-12 of itself or 2^-30 of its tile's largest.  The fourth term is free:
// 8 rows with three terms would be 24 columns, and the tensor cores want a multiple of 16.
// Each step of one or two 128-token tiles has its own maximum, largest V scale and product with V;
// steps are joined in 32-bit registers, so the tensor cores' accumulators never need rescaling.
//
// Layout.  Tokens are the M axis of the scores (A = K, MN-major: tokens contiguous) and head_dim
// the M axis of the products (A = V, K-major: tokens contiguous again); the rows of q (heads that
// share a cache head, times the rows of a sequence), term by term, are N.  A block of the
// cache is a [head_dim][block_size] byte tile, which for block_size 16 is exactly the tensor
// core's unswizzled operand layout (one contiguous bulk copy) and for 32 to 128 its 32- to
// 128-byte swizzled one (one TMA box).
//
// Work.  All (sequence, head, row group) units laid end to end as 128-token tiles are cut into
// equal runs, one per thread block, whatever the lengths; a block finds its run from the lengths
// alone.  A unit cut by that leaves partial sums (maximum, sum, accumulators) and the last block
// to arrive joins them.  Roles: warps 0-3 softmax (a thread per token, then per head_dim row),
// warp 4 copies, warp 5 issues the tensor cores; two steps are in flight between them.
//
// Numbers that are none.  What a row does not see reaches none of its sums, whatever it holds: masked scores are set
// apart, V scales that are infinite or NaN count as 0 in the products, and so do E4M3 codes that are NaN where not every
// row sees their tokens.  The rows that do see them get NaN at the unit's end (odd_rows).  That code is kept out of the
// loop: inside it 64 sequences took 1.5 % longer, 16-row groups 5 %.
//
// Measured (a copy runs at 6.47 TB/s).  4 sequences of 100000 to 131072 tokens, 8 cache heads of 128 with 8 query
// heads each, E4M3, blocks of 64: 156 to 169 us on several GPUs, 5.4 to 5.9 TB/s, bound by HBM.  64 sequences of 256 to
// 4096, 4 query heads each, blocks of 16: 61 to 62 us, 4.7 TB/s: a block gets two or three units, and between units the
// copies wait for some 10000 cycles (masks of the last step, the next rows of q, the sums), as what they run ahead by is
// two tiles of K and four of V, all that shared memory holds.  Of 8.3 cycles between two instructions of a warp 2.8 go
// to loads, 1.6 to waits of fixed length, 0.7 to instructions that come late; with groups of 8 rows, twice the code, 1.5
// of 6: less code is faster code.  Taking the next unit's rows and first scores before the last step ends: 65 us, as the
// loop grows; three blocks per SM with fewer tiles each: 65 us.  16 sequences of 300 to 4500, 16 heads of 64 on one
// cache head, 1 to 8 rows: 25 to 28 us, either kernel.  One sequence of 777 tokens: 9 to 10 us, a chain of latencies
// (lengths, block ids, K, scores, weights, sums).
#include "block_attn.cuh"
#include "tcgen05.cuh"

namespace mak {
namespace {

constexpr int kTile = 128;  // tokens per step
constexpr int kThreads = 192;
constexpr int kSoft = 128;  // threads of the softmax warps
constexpr int kMaxGrid = 148 * 4;  // blocks of the largest grid; the workspace has two partial sums for each
constexpr int kMaxRows = 16;
constexpr int kMaxDim = 256;
// Tiles per block that are worth another block.  One sequence of 777 tokens with 1, 2, 4, 8: 10.8, 10.8, 13.2, 16.6 us.
constexpr int kMinChunk = 2;
// A unit's beginning and end (its rows of q, its result) take a block about as long as this many tiles.  64 sequences
// of 256 to 4096 tokens with 2, 3, 4: 62.2, 61.7, 62.8 us; in groups of 8 rows with 1, 2, 3, 4, 6: 86.7, 80.7, 76.8,
// 77.0, 77.4 us.
constexpr int kUnitCost = 3;

template <int HD, int ROWS>
struct Cfg {
  static constexpr int kN = 4 * ROWS;              // columns of the products
  static constexpr int kParts = HD == 256 ? 2 : 1; // 128-row parts of head_dim
  // Tiles of one softmax step.  Two halve the barriers for each tile, which pays for 8 rows; for 4 rows the shorter
  // code of one does (62.8 against 64.0 us for 64 sequences of 256 to 4096 tokens), for 16 two need more registers
  // than there are.
  static constexpr int kStep = ROWS == 8 ? 2 : 1;
  // Tiles of K and V in shared memory.  Scores are taken as soon as K is there; V waits for the
  // weights, a step of it held and a step on its way.
  static constexpr int kKs = HD == 64 ? 4 : 2;
  static constexpr int kVs = HD == 64 ? 6 : ROWS <= 8 ? 4 : 3;
  static constexpr int kTileBytes = HD * kTile;
  static constexpr int kScores = 0, kOut = 2 * kStep * kN;  // TMEM columns: two steps' scores, one product
  static constexpr int kCols = kOut + kParts * kN;
  static constexpr int kTmem = kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
};

template <int HD, int ROWS>
struct Smem {
  using C = Cfg<HD, ROWS>;
  // V first: with head_dim 64 the products read 128 rows from it, the last 64 past a tile's end
  alignas(1024) uint8_t v[C::kVs][C::kTileBytes];
  alignas(1024) uint8_t k[C::kKs][C::kTileBytes];
  alignas(1024) uint8_t p[C::kN * kTile * C::kStep];
  // The products read four terms of q, of which there are three: what follows makes columns nobody reads.  Columns
  // lie in groups of 8.
  uint8_t q[2][(3 * ROWS + 7) / 8 * 8 * HD];  // of this unit and the next
  alignas(16) float ks[16][8], vs[16][8];  // scales per 16 tokens, tile number mod 16
  uint32_t have[16];                       // bit c: 16-token piece c has a block
  int page[16][8], head[16];               // for the copies of V, which follow those of K
  alignas(16) float wmax[2][4][ROWS];
  alignas(16) float row_scale[2][ROWS];
  int row_lo[2][ROWS], row_hi[2][ROWS];
  alignas(8) int64_t row_out[2][ROWS], row_lse[2][ROWS];  // places of the results
  int unit_seq[2], unit_head[2], unit_lo[2], unit_hi[2];  // tokens [lo, hi) of this block's tiles; lo on a tile's border
  float lsum[4][ROWS];
  alignas(8) uint64_t k_full[C::kKs], k_empty[C::kKs], v_full[C::kVs], v_empty[C::kVs];
  uint64_t q_full, s_full[2], p_full, o_full, spare;
  uint32_t tmem;
  int gave_up, last;
  int odd;  // this block met a V scale that is infinite or NaN, or an E4M3 NaN
};

// Tiles of a unit of sequence v (at least one, so that empty rows are written).
__device__ __forceinline__ int unit_tiles(const SeqView& v) {
  const int t0 = v.lo / kTile, t1 = (v.hi + kTile - 1) / kTile;
  return t1 > t0 ? t1 - t0 : 1;
}

template <int ROWS>
__device__ __forceinline__ int row_groups(const BlockAttnParams& p, const SeqView& v) {
  return (v.rows * p.group + ROWS - 1) / ROWS;
}
template <int ROWS>
__device__ __forceinline__ int64_t seq_work(const BlockAttnParams& p, const SeqView& v) {
  return static_cast<int64_t>(row_groups<ROWS>(p, v)) * p.nh * (unit_tiles(v) + kUnitCost);
}

// A block's run [w, w_end) of work, unit by unit; every warp walks it for itself.  A unit of n
// tiles is kUnitCost + n steps long, its tiles being the last ones.
struct Walk {
  SeqView v;
  int seq, head, group, groups, tiles;  // the unit that begins at w0
  int64_t w, w_end, w0;
};
struct Unit {
  int seq;
  int head, row0, live;               // rows row0 .. row0 + live (row i * group + j: row i, query head j)
  int tiles, ta, tb;                  // of the unit's tiles this block has [ta, tb)
  int t_first, t_last;                // absolute tiles of those that some row sees
  int any_lo, any_hi, all_lo, all_hi; // tokens that some / all rows see
  int64_t w_tiles;                    // where the unit's tiles begin
  SeqView v;
};

template <int ROWS>
__device__ __forceinline__ void begin_walk(const BlockAttnParams& p, Walk& k, int seq, int64_t base) {
  k.seq = seq;
  k.v = seq_view(p, seq);
  k.tiles = unit_tiles(k.v);
  k.groups = row_groups<ROWS>(p, k.v);
  const int64_t rel = k.w - base;
  const uint32_t len = k.tiles + kUnitCost;
  const int64_t unit = (rel >> 32) == 0 ? static_cast<uint32_t>(rel) / len : rel / len;
  k.w0 = base + unit * len;
  k.head = static_cast<int>(static_cast<uint32_t>(unit) / static_cast<uint32_t>(k.groups));
  k.group = static_cast<int>(unit - static_cast<int64_t>(k.head) * k.groups);
}

// The next unit of which this block has any tiles.
template <int ROWS>
__device__ __forceinline__ bool next_unit(const BlockAttnParams& p, Walk& k, Unit& u) {
  for (;;) {
    if (k.w >= k.w_end) return false;
    u.ta = static_cast<int>(max(k.w - k.w0 - kUnitCost, static_cast<int64_t>(0)));
    u.tb = static_cast<int>(min(k.w_end - k.w0 - kUnitCost, static_cast<int64_t>(k.tiles)));
    u.seq = k.seq;
    u.v = k.v;
    u.tiles = k.tiles;
    u.head = k.head;
    u.row0 = k.group * ROWS;
    u.w_tiles = k.w0 + kUnitCost;
    k.w0 += kUnitCost + k.tiles;
    k.w = k.w0;
    if (k.w < k.w_end && ++k.group == k.groups) {
      k.group = 0;
      if (++k.head == p.nh) {
        k.head = 0;
        do {
          k.v = seq_view(p, ++k.seq);
        } while (k.v.rows == 0);
        k.tiles = unit_tiles(k.v);
        k.groups = row_groups<ROWS>(p, k.v);
      }
    }
    if (u.tb > u.ta) break;
  }
  const SeqView& v = u.v;
  u.live = min(ROWS, v.rows * p.group - u.row0);
  row_range(p, v, u.row0 / p.group, &u.any_lo, &u.all_hi);
  row_range(p, v, (u.row0 + u.live - 1) / p.group, &u.all_lo, &u.any_hi);
  const int tile0 = v.hi > v.lo ? v.lo / kTile : 0;
  u.t_first = u.t_last = 0;
  if (u.any_hi > u.any_lo) {
    u.t_first = max(tile0 + u.ta, u.any_lo / kTile);
    u.t_last = max(u.t_first, min(tile0 + u.tb, (u.any_hi + kTile - 1) / kTile));
  }
  return true;
}

__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Two values (E4M3: at most 448) to their terms, low byte of t[i] the first value's.
template <int TERMS>
__device__ __forceinline__ void split_e4m3(float x, float y, uint32_t (&t)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    uint16_t b;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(y), "f"(x));
    t[i] = b;
    if (i + 1 < TERMS) {
      uint32_t h;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(b));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      x = (x - f.x) * 16.f;
      y = (y - f.y) * 16.f;
    }
  }
}
// Whole number below 127.4 * 2^24 to its balanced base-256 digits, highest in byte 3.
__device__ __forceinline__ uint32_t split_int8(float x) {
  return (static_cast<uint32_t>(__float2int_rn(x)) + 0x808080u) ^ 0x808080u;
}

// The terms' products to their sum in units of the first: a digit is worth 1 / 256 of the one before it, an E4M3 term
// 1 / 16.
template <int CODE, int TERMS>
__device__ __forceinline__ float join_terms(const uint32_t (&t)[TERMS]) {
  float x = 0.f;
  if constexpr (CODE == MAK_CODE_INT8) {
#pragma unroll
    for (int i = 0; i < TERMS; ++i) x = fmaf(static_cast<float>(static_cast<int>(t[i])), 1.f / (1u << (8 * i)), x);
  } else {
#pragma unroll
    for (int i = TERMS - 1; i >= 0; --i) x = fmaf(x, 1.f / 16.f, __uint_as_float(t[i]));
  }
  return x;
}

// E4M3 values of the tile at token tk: in its 16-token pieces `part`, codes that no row sees and NaN become 0.
template <int HD>
__device__ __forceinline__ void clean_tile(uint8_t* tile, int tk, uint32_t part, uint32_t have, int any_lo, int any_hi, int bs_log2,
                                        volatile int* odd) {
  const int bs = 1 << bs_log2, per_line = bs >> 4;  // 16-byte pieces of a line
  for (uint32_t left = part & 0xffu; left != 0; left &= left - 1) {
    const int c = __ffs(left) - 1;
    const int from = have >> c & 1 ? any_lo - tk - 16 * c : 16, to = any_hi - tk - 16 * c;  // of its tokens, what some row sees
    uint32_t mask[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      mask[b] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * b + e >= from && 4 * b + e < to) mask[b] |= 0xffu << (8 * e);
    }
    for (int d = threadIdx.x; d < HD; d += kSoft) {
      const int swz = bs_log2 == 7 ? d & 7 : bs_log2 == 6 ? (d >> 1) & 3 : bs_log2 == 5 ? (d >> 2) & 1 : 0;
      uint4* at = reinterpret_cast<uint4*>(tile + (c / per_line) * (HD * bs) + d * bs + (((c % per_line) ^ swz) << 4));
      uint4 v = *at;
      uint32_t bad = 0;
      auto clean = [&](uint32_t w, uint32_t m) {
        const uint32_t nan = nan_codes(w & m);
        bad |= nan;
        return w & m & ~((nan >> 7) * 0xffu);
      };
      v = make_uint4(clean(v.x, mask[0]), clean(v.y, mask[1]), clean(v.z, mask[2]), clean(v.w, mask[3]));
      if (bad != 0) *odd = 1;
      *at = v;
    }
  }
}

// Results that are no numbers: the rows, one bit each, of the unit whose rows lie in `buf` that see a block whose V scale
// is infinite or NaN, and in E4M3 those whose dimension d is NaN at a token that they see.  Both were 0 in the products,
// where a weight of 0 would have brought them to every row.  Called once this block has met any; by whole warps.
template <int HD, int ROWS, int CODE>
__device__ __noinline__ uint32_t odd_rows(const BlockAttnParams& p, const Smem<HD, ROWS>& sm, int buf, int d) {
  auto rows_seeing = [&](int t0, int t1) {
    uint32_t rows = 0;
    for (int z = 0; z < ROWS; ++z)
      if (max(sm.row_lo[buf][z], t0) < min(sm.row_hi[buf][z], t1)) rows |= 1u << z;
    return rows;
  };
  const int begin = sm.unit_lo[buf], end = sm.unit_hi[buf], bs = 1 << p.bs_log2;
  const int64_t head = sm.unit_head[buf];
  const int32_t* table = p.tables + sm.unit_seq[buf] * p.table_stride;
  auto page_of = [&](int tk) {
    const int page = __ldg(table + (tk >> p.bs_log2));
    return page < p.num_blocks ? page : -1;
  };
  uint32_t rows = 0;
  for (int tk = begin + (threadIdx.x & 31) * 16; tk < end; tk += 512) {
    const int page = page_of(tk);
    if (page >= 0 && !(fabsf(__ldg(p.value_scale + page * p.vs_sb + head * p.vs_sh)) < INFINITY)) rows |= rows_seeing(tk, tk + 16);
  }
  rows = __reduce_or_sync(0xffffffffu, rows);
  if (CODE == MAK_CODE_E4M3 && d < HD) {
    for (int tk = begin; tk < end; tk += 16) {
      const int page = page_of(tk);
      if (page < 0) continue;
      const uint8_t* codes = p.value + page * p.v_sb + head * p.v_sh + static_cast<int64_t>(d) * bs + (tk & (bs - 1));
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(codes));
      if ((nan_codes(v.x) | nan_codes(v.y) | nan_codes(v.z) | nan_codes(v.w)) == 0) continue;
      for (int t = 0; t < 16; ++t)
        if (nan_codes(__ldg(codes + t)) != 0) rows |= rows_seeing(tk + t, tk + t + 1);
    }
  }
  return rows;
}

template <int HD, int ROWS, int CODE>
__global__ void __launch_bounds__(kThreads, HD == 256 ? 1 : 2)
    block_attn_rows_kernel(const __grid_constant__ BlockAttnParams p, const __grid_constant__ CUtensorMap kmap,
                           const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<HD, ROWS>;
  constexpr int kKs = C::kKs, kVs = C::kVs;
  extern __shared__ __align__(1024) uint8_t raw[];
  Smem<HD, ROWS>& sm = *reinterpret_cast<Smem<HD, ROWS>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_trigger();

  // ---- the run of this block: every warp finds it for itself --------------------
  Walk walk;
  int64_t chunk;
  {
    const int per = (p.num_seqs + 31) / 32;
    const int s0 = min(lane * per, p.num_seqs), s1 = min(s0 + per, p.num_seqs);
    int64_t mine = 0;
    for (int s = s0; s < s1; ++s) mine += seq_work<ROWS>(p, seq_view(p, s));
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const int64_t total = __shfl_sync(0xffffffffu, incl, 31);
    chunk = (total >> 31) == 0 ? (static_cast<uint32_t>(total) + gridDim.x - 1) / gridDim.x : (total + gridDim.x - 1) / gridDim.x;
    if (chunk < kMinChunk) chunk = kMinChunk;
    walk.w = blockIdx.x * chunk;
    walk.w_end = min(walk.w + chunk, total);
    if (walk.w >= walk.w_end) return;
    const bool here = incl - mine <= walk.w && walk.w < incl;
    int seq = 0;
    int64_t base = incl - mine;
    if (here) {
      for (seq = s0;; ++seq) {
        const int64_t w = seq_work<ROWS>(p, seq_view(p, seq));  // zero for a sequence without rows
        if (walk.w < base + w) break;
        base += w;
      }
    }
    const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    begin_walk<ROWS>(p, walk, __shfl_sync(0xffffffffu, seq, from), __shfl_sync(0xffffffffu, base, from));
  }
  const int64_t w_begin = walk.w;
  if (tid == kSoft) {
    sm.gave_up = 0;
    sm.odd = 0;
    for (int i = 0; i < kKs; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.k_empty[i], 1);
    }
    for (int i = 0; i < kVs; ++i) {
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.v_empty[i], 1);
    }
    mbar_init(&sm.q_full, 4);
    mbar_init(&sm.s_full[0], 1);
    mbar_init(&sm.s_full[1], 1);
    mbar_init(&sm.p_full, 4);
    mbar_init(&sm.o_full, 1);
    mbar_init(&sm.spare, 1);
    mbar_init_fence();
  }
  if (warp == 5) tmem_alloc<C::kTmem>(&sm.tmem);
  // Ends the set-up: what a role can load before, it does.
  auto ready = [&]() {
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };
  volatile int *gave_up = &sm.gave_up, *odd = &sm.odd;
  const int bs = 1 << p.bs_log2;
  Unit u;
  auto block_of = [&](int64_t w) {
    return (w >> 32) == 0 && (chunk >> 32) == 0 ? static_cast<uint32_t>(w) / static_cast<uint32_t>(chunk) : w / chunk;
  };

  if (warp < 4) {
    // ---- softmax ----------------------------------------------------------------
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const int piece = tid >> 4;  // 16-token piece of this thread's token
    uint32_t it = 0, tiles_done = 0;  // steps and tiles before this unit
    bool ok = true;
    // Rows of a unit: their places, and q as three 8-bit terms.  A row's threads are neighbours.
    constexpr int kPer = HD * ROWS / kSoft < 4 ? 4 : HD * ROWS / kSoft;  // values of a thread
    constexpr int kRowThreads = HD / kPer;
    const int r = tid / kRowThreads, d0 = tid % kRowThreads * kPer;
    uint32_t w[kPer / 2];
    auto fetch = [&](const Unit& u) {
#pragma unroll
      for (int e = 0; e < kPer / 2; ++e) w[e] = 0;
      if (r < u.live) {
        const int i = (u.row0 + r) / p.group, j = u.head * p.group + (u.row0 + r) - i * p.group;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) + (u.v.first + i) * p.q_sr + j * p.q_sh + d0;
#pragma unroll
        for (int e = 0; e < kPer / 4; ++e) {
          const uint2 x = __ldg(reinterpret_cast<const uint2*>(src) + e);
          w[2 * e] = x.x, w[2 * e + 1] = x.y;
        }
      }
    };
    auto stage = [&](const Unit& u, int buf) {
      if (tid == 0) {
        sm.unit_seq[buf] = u.seq;
        sm.unit_head[buf] = u.head;
        sm.unit_lo[buf] = u.t_first * kTile;
        sm.unit_hi[buf] = min(u.t_last * kTile, u.any_hi);
      }
      if (r < ROWS && d0 == 0) {
        const int i = (u.row0 + r) / p.group, j = u.head * p.group + (u.row0 + r) - i * p.group;
        int lo = 0, hi = 0;
        if (r < u.live) row_range(p, u.v, i, &lo, &hi);
        sm.row_lo[buf][r] = lo;
        sm.row_hi[buf][r] = hi;
        sm.row_out[buf][r] = (u.v.first + i) * p.o_sr + j * p.o_sh;
        sm.row_lse[buf][r] = static_cast<int64_t>(u.v.first + i) * p.nh * p.group + j;
      }
      if (u.t_last > u.t_first) {
        float x[kPer], top = 0.f;
#pragma unroll
        for (int e = 0; e < kPer / 2; ++e) {
          if (p.q_bf16) {
            x[2 * e] = __uint_as_float(w[e] << 16);
            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
          } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
            x[2 * e] = f.x;
            x[2 * e + 1] = f.y;
          }
          top = fmaxf(top, fmaxf(fabsf(x[2 * e]), fabsf(x[2 * e + 1])));
          if (x[2 * e] != x[2 * e] || x[2 * e + 1] != x[2 * e + 1]) top = INFINITY;
        }
#pragma unroll
        for (int o = kRowThreads / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        constexpr int kTop = CODE == MAK_CODE_INT8 ? 21 : 7;
        const int up = top > 0.f && top < INFINITY ? kTop - ilogbf(top) : 0;
        const int up1 = up / 2, up2 = up - up1;  // two steps: 2^up itself may leave the exponent range
        const float f1 = __uint_as_float(static_cast<uint32_t>(127 + up1) << 23);
        const float f2 = __uint_as_float(static_cast<uint32_t>(127 + up2) << 23);
#pragma unroll
        for (int e = 0; e < kPer; e += 4) {
          float y[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) y[b] = x[e + b] * f1 * f2;
          uint32_t t[3];
          if constexpr (CODE == MAK_CODE_INT8) {
            uint32_t v[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) v[b] = split_int8(y[b]);
#pragma unroll
            for (int z = 0; z < 3; ++z) {
              const uint32_t pick = (2 - z) | ((6 - z) << 4);  // byte 2 - z of both
              t[z] = __byte_perm(__byte_perm(v[0], v[1], pick), __byte_perm(v[2], v[3], pick), 0x5410);
            }
          } else {
            uint32_t a[3], b[3];
            split_e4m3(y[0], y[1], a);
            split_e4m3(y[2], y[3], b);
#pragma unroll
            for (int z = 0; z < 3; ++z) t[z] = a[z] | (b[z] << 16);
          }
#pragma unroll
          for (int z = 0; z < 3; ++z) {
            const int col = z * ROWS + r, d = d0 + e;
            if (r < ROWS) *reinterpret_cast<uint32_t*>(sm.q[buf] + (col >> 3) * (HD * 8) + (d >> 4) * 128 + (col & 7) * 16 + (d & 15)) = t[z];
          }
        }
        constexpr int kFirst = CODE == MAK_CODE_INT8 ? 16 : 0;  // 2^kFirst: a unit of the first term
        if (r < ROWS && d0 == 0) sm.row_scale[buf][r] = top < INFINITY ? ldexpf(p.scale_log2, kFirst - up) : __uint_as_float(0x7fffffffu);
        fence_async_shared();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full);
      }
    };
    auto put = [&](int buf, int z, int d, float y) {
      const int64_t at = sm.row_out[buf][z] + d;
      if (p.q_bf16)
        reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
      else
        reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(y);
    };
    auto put_lse = [&](int buf, int z, float mx, float sum) {
      if (p.lse != nullptr)
        p.lse[sm.row_lse[buf][z]] = sum > 0.f || sum != sum ? (mx + log2f(sum)) * 0.69314718055994531f : -INFINITY;
    };
    constexpr int kFloats = ROWS * (HD + 2);  // of one partial sum
    // A unit whose partial sum was left: the last of its blocks to get here joins them.  Whether this one
    // is the last is asked for at once and looked at a unit later.
    struct {
      int first, last, slot, live, buf;
      int64_t w_tiles;
      int ticket;
    } open;
    open.first = -1;
    auto close = [&]() {
      if (open.first < 0) return;
      if (tid == 0) sm.last = open.ticket == open.last - open.first;
      soft_sync();
      if (sm.last) {
        for (int idx = tid; idx < open.live * (HD / 4); idx += kSoft) {
          const int z = idx / (HD / 4), d = idx % (HD / 4) * 4;
          float mx = -INFINITY, sum = 0.f;
          float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
          for (int b = open.first; b <= open.last; ++b) {
            const float* src = p.partial + (2 * static_cast<int64_t>(b) + (open.w_tiles > b * chunk ? 1 : 0)) * kFloats;
            const float pm = __ldcg(src + ROWS * HD + z), pl = __ldcg(src + ROWS * HD + ROWS + z);
            const float4 po = __ldcg(reinterpret_cast<const float4*>(src + z * HD + d));
            const float mn = fmaxf(mx, pm);
            const float ms = mn == -INFINITY ? 0.f : mn;
            const float k0 = exp2_fast(mx - ms), k1 = exp2_fast(pm - ms);
            o[0] = o[0] * k0 + po.x * k1;
            o[1] = o[1] * k0 + po.y * k1;
            o[2] = o[2] * k0 + po.z * k1;
            o[3] = o[3] * k0 + po.w * k1;
            sum = sum * k0 + pl * k1;
            mx = mn;
          }
          const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) put(open.buf, z, d + e, o[e] * inv);
          if (d == 0) put_lse(open.buf, z, mx, sum);
        }
        if (tid == 0) p.counters[open.slot] = 0;
      }
      open.first = -1;
      soft_sync();
    };

    int buf = 0;
    bool more = next_unit<ROWS>(p, walk, u);
    if (more) fetch(u);
    ready();
    const uint32_t tmem = sm.tmem;
    if (more) stage(u, 0);
    soft_sync();
    while (more) {
      const int n = u.t_last - u.t_first;
      const int steps = (n + C::kStep - 1) / C::kStep;
      float acc[C::kParts][ROWS], m[ROWS], l[ROWS], gain[ROWS];
#pragma unroll
      for (int z = 0; z < ROWS; ++z) {
#pragma unroll
        for (int h = 0; h < C::kParts; ++h) acc[h][z] = 0.f;
        m[z] = -INFINITY;
        l[z] = 0.f;
        gain[z] = 0.f;
      }
      // the product with V of step x joins the sums
      auto collect = [&](uint32_t x) {
        if (!mbar_wait_warp(&sm.o_full, x & 1, gave_up)) return false;
        if (HD == 64 && warp >= 2) return true;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < C::kParts; ++h) {
          uint32_t o[4][ROWS];
          const uint32_t at = tmem + lanes + C::kOut + h * C::kN;
#pragma unroll
          for (int z = 0; z < 4; ++z) tmem_ld(at + z * ROWS, o[z]);
#pragma unroll
          for (int z = 0; z < 4; ++z) tmem_wait(o[z]);
#pragma unroll
          for (int z = 0; z < ROWS; ++z) {
            const uint32_t t[4] = {o[0][z], o[1][z], o[2][z], o[3][z]};
            acc[h][z] += join_terms<CODE>(t) * gain[z];
          }
        }
        return true;
      };
      // A warp that gave up goes through the same barriers as the others, without waiting for anything else.
      for (int t = 0; t < steps; ++t) {
        const uint32_t x = it + t, tile = tiles_done + t * C::kStep;
        const int count = min(C::kStep, n - t * C::kStep);  // tiles of this step
        ok = ok && mbar_wait_warp(&sm.s_full[x & 1], (x >> 1) & 1, gave_up);
        tc_fence_after();
        float s[C::kStep][ROWS];
        float top[ROWS], vtop = 0.f, vs[C::kStep];
        const int tok0 = (u.t_first + t * C::kStep) * kTile;
        uint32_t o[C::kStep][3][ROWS];
#pragma unroll
        for (int y = 0; y < C::kStep; ++y)
#pragma unroll
          for (int z = 0; z < 3; ++z) tmem_ld(tmem + lanes + C::kScores + ((x & 1) * C::kStep + y) * C::kN + z * ROWS, o[y][z]);
#pragma unroll
        for (int y = 0; y < C::kStep; ++y)
#pragma unroll
          for (int z = 0; z < 3; ++z) tmem_wait(o[y][z]);
#pragma unroll
        for (int y = 0; y < C::kStep; ++y) {
          const uint32_t k = (tile + y) & 15;
          const float ks = sm.ks[k][piece];
#pragma unroll
          for (int z = 0; z < ROWS; ++z) {
            const uint32_t t3[3] = {o[y][0][z], o[y][1][z], o[y][2][z]};
            s[y][z] = join_terms<CODE>(t3) * (sm.row_scale[buf][z] * ks);
          }
          vs[y] = sm.vs[k][piece];
          const int tk = tok0 + y * kTile;
          const uint32_t have = y < count ? sm.have[k] : 0u;
          if (tk < u.all_lo || tk + kTile > u.all_hi || have != 0xffu) {
            const bool there = (have >> piece) & 1;
            if (!there) vs[y] = 0.f;
#pragma unroll
            for (int z = 0; z < ROWS; ++z)
              if (!there || tk + tid < sm.row_lo[buf][z] || tk + tid >= sm.row_hi[buf][z]) s[y][z] = -INFINITY;
          }
          if (y < count) {
#pragma unroll
            for (int c = 0; c < 8; ++c) vtop = fmaxf(vtop, fabsf(sm.vs[k][c]));
          }
        }
#pragma unroll
        for (int z = 0; z < ROWS; ++z) top[z] = warp_max(C::kStep == 2 ? fmaxf(s[0][z], s[C::kStep - 1][z]) : s[0][z]);
        if (lane == 0) {
#pragma unroll
          for (int z = 0; z < ROWS; z += 4)
            *reinterpret_cast<float4*>(&sm.wmax[x & 1][warp][z]) = make_float4(top[z], top[z + 1], top[z + 2], top[z + 3]);
        }
        soft_sync();
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int z = 0; z < ROWS; z += 4) {
            const float4 o = *reinterpret_cast<const float4*>(&sm.wmax[x & 1][w][z]);
            top[z] = fmaxf(top[z], o.x);
            top[z + 1] = fmaxf(top[z + 1], o.y);
            top[z + 2] = fmaxf(top[z + 2], o.z);
            top[z + 3] = fmaxf(top[z + 3], o.w);
          }
        // The largest weight, in units of its last digit (int8) and of its first term.  By the reciprocal first: kFull
        // over a scale of 2^-109 leaves 32 bits.  Scales that have no reciprocal, below 2^-126, count as 0.
        constexpr float kFull = CODE == MAK_CODE_INT8 ? 127.f * 16777216.f : 256.f, kLead = CODE == MAK_CODE_INT8 ? 127.f : 256.f;
        const float inv = vtop >= 0x1p-126f ? 1.f / vtop : 0.f;
#pragma unroll
        for (int y = 0; y < C::kStep; ++y) vs[y] = vs[y] * inv * kFull;
        float fade[ROWS], next_gain[ROWS];
        uint32_t words[C::kStep][4][ROWS / 4];  // weights of this thread's tokens: term, four rows
#pragma unroll
        for (int z0 = 0; z0 < ROWS; z0 += 4) {
          float w[C::kStep][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int z = z0 + e;
            const float mt = top[z], mn = fmaxf(m[z], mt);
            const float ms = mn == -INFINITY ? 0.f : mn, mz = mt == -INFINITY ? 0.f : mt;
            const float old = exp2_fast(m[z] - ms), add = exp2_fast(mt - ms);
            float sum = 0.f;
#pragma unroll
            for (int y = 0; y < C::kStep; ++y) {
              w[y][e] = exp2_fast(s[y][z] - mz);
              sum += w[y][e];
              w[y][e] *= vs[y];
            }
            l[z] = l[z] * old + sum * add;
            fade[z] = old;
            next_gain[z] = add * vtop * (1.f / kLead);
            m[z] = mn;
          }
#pragma unroll
          for (int y = 0; y < C::kStep; ++y) {
            if constexpr (CODE == MAK_CODE_INT8) {
              uint32_t v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = split_int8(w[y][e]);
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const uint32_t pick = (3 - c) | ((7 - c) << 4);  // byte 3 - c of both
                words[y][c][z0 / 4] = __byte_perm(__byte_perm(v[0], v[1], pick), __byte_perm(v[2], v[3], pick), 0x5410);
              }
            } else {
              uint32_t a[4], b[4];
              split_e4m3(w[y][0], w[y][1], a);
              split_e4m3(w[y][2], w[y][3], b);
#pragma unroll
              for (int c = 0; c < 4; ++c) words[y][c][z0 / 4] = a[c] | (b[c] << 16);
            }
          }
        }
        // The step before: its product is the last reader of the weights' place, and has had until now.
        if (t > 0) ok = ok && collect(x - 1);
#pragma unroll
        for (int z = 0; z < ROWS; ++z) {
#pragma unroll
          for (int h = 0; h < C::kParts; ++h) acc[h][z] *= fade[z];
          gain[z] = next_gain[z];
        }
        // 16 columns of a token are 16 bytes, the next 16 a step's tokens further on
#pragma unroll
        for (int y = 0; y < C::kStep; ++y) {
          const uint32_t* x4 = &words[y][0][0];
#pragma unroll
          for (int c = 0; c < ROWS / 4; ++c)
            *reinterpret_cast<uint4*>(sm.p + (c * C::kStep * kTile + y * kTile + tid) * 16) =
                make_uint4(x4[4 * c], x4[4 * c + 1], x4[4 * c + 2], x4[4 * c + 3]);
        }
        // E4M3: codes may be NaN, which a weight of zero does not cancel.  They become 0 in the pieces that not every row
        // sees whole, as does what no row sees; the rows that do see one get NaN with their results.
        if (CODE == MAK_CODE_E4M3) {
          for (int y = 0; y < count; ++y) {
            const int tk = tok0 + y * kTile;
            const uint32_t have = sm.have[(tile + y) & 15];
            if (tk >= u.all_lo && tk + kTile <= u.all_hi && have == 0xffu) continue;
            const uint32_t slot = (tile + y) % kVs;
            ok = ok && mbar_wait_warp(&sm.v_full[slot], ((tile + y) / kVs) & 1, gave_up);
            uint32_t part = ~have & 0xffu;
            if (tk < u.all_lo) part |= (2u << min((u.all_lo - tk) >> 4, 7)) - 1;
            if (tk + kTile > u.all_hi) part |= 0xffu << (max(u.all_hi - tk, 0) >> 4);
            clean_tile<HD>(sm.v[slot], tk, part, have, u.any_lo, u.any_hi, p.bs_log2, odd);
          }
        }
        fence_async_shared();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full);
      }
      if (__any_sync(0xffffffffu, *odd)) {  // the last product has yet to join the sums: NaN stays NaN
#pragma unroll
        for (int h = 0; h < C::kParts; ++h) {
          const uint32_t rows = odd_rows<HD, ROWS, CODE>(p, sm, buf, h * 128 + tid);
#pragma unroll
          for (int z = 0; z < ROWS; ++z)
            if (rows >> z & 1) acc[h][z] = __uint_as_float(0x7fffffffu);
        }
      }
      // The next unit's rows, so that the tensor cores begin on it while this one ends.
      close();
      const Unit done = u;
      more = next_unit<ROWS>(p, walk, u);
      if (more) {
        fetch(u);
        stage(u, buf ^ 1);
      }
      if (ok && n > 0) ok = collect(it + steps - 1);
      it += steps;
      tiles_done += n;

      // ---- this block's share of the unit -----------------------------------------
      {
        // the rows' sums over the threads, through the weights' place
        float* sums = reinterpret_cast<float*>(sm.p);
#pragma unroll
        for (int z = 0; z < ROWS; z += 4)
          *reinterpret_cast<float4*>(sums + tid * ROWS + z) = make_float4(l[z], l[z + 1], l[z + 2], l[z + 3]);
        soft_sync();
        const int z = tid % ROWS, part = tid / ROWS;
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < ROWS; ++k) sum += sums[(part * ROWS + k) * ROWS + z];
#pragma unroll
        for (int o = ROWS; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane < ROWS) sm.lsum[warp][z] = ok ? sum : __uint_as_float(0x7fffffffu);  // a block that gave up leaves NaN
      }
      soft_sync();
#pragma unroll
      for (int z = 0; z < ROWS; ++z) l[z] = sm.lsum[0][z] + sm.lsum[1][z] + sm.lsum[2][z] + sm.lsum[3][z];
      if (done.ta == 0 && done.tb == done.tiles) {
#pragma unroll
        for (int z = 0; z < ROWS; ++z) {
          if (z < done.live) {
            const float inv = l[z] > 0.f || l[z] != l[z] ? 1.f / l[z] : 0.f;
#pragma unroll
            for (int h = 0; h < C::kParts; ++h)
              if (HD >= 128 || tid < HD) put(buf, z, h * 128 + tid, acc[h][z] * inv);
            if (tid == z) put_lse(buf, z, m[z], l[z]);
          }
        }
        soft_sync();  // the rows' places and sums are read
      } else {
        float* part = p.partial + (2 * static_cast<int64_t>(blockIdx.x) + (done.w_tiles > w_begin ? 1 : 0)) * kFloats;
#pragma unroll
        for (int z = 0; z < ROWS; ++z) {
#pragma unroll
          for (int h = 0; h < C::kParts; ++h)
            if (HD >= 128 || tid < HD) part[z * HD + h * 128 + tid] = acc[h][z];
          if (tid == z) {
            part[ROWS * HD + z] = m[z];
            part[ROWS * HD + ROWS + z] = l[z];
          }
        }
        open.first = static_cast<int>(block_of(done.w_tiles));
        open.last = static_cast<int>(block_of(done.w_tiles + done.tiles - 1));
        open.slot = 2 * open.first + (done.w_tiles > open.first * chunk ? 1 : 0);
        open.live = done.live;
        open.buf = buf;
        open.w_tiles = done.w_tiles;
        soft_sync();
        if (tid == 0)  // releases what the barrier has gathered
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(open.ticket) : "l"(p.counters + open.slot) : "memory");
      }
      buf ^= 1;
    }
    close();
  } else if (warp == 4) {
    // ---- copies: block ids and scales for four tiles at a time, a lane per 16 tokens ---------
    const int mine = lane >> 3, piece = lane & 7;
    const uint32_t per_line = bs >> 4, bytes = HD * bs;
    const bool leads = piece % per_line == 0;  // issues its block's copies
    const uint32_t k_to = smem_addr(sm.k) + piece * (HD * 16), v_to = smem_addr(sm.v) + piece * (HD * 16);
    struct Batch {
      int count, head, page;
      float ks, vs;
    } next;
    int gt = 0;
    u.t_last = 0;
    // the next batch of at most four tiles of one unit; none at the end
    auto look_ahead = [&]() {
      next.count = 0;
      while (gt >= u.t_last) {
        if (!next_unit<ROWS>(p, walk, u)) return;
        gt = u.t_first;
      }
      next.count = min(4, u.t_last - gt);
      next.head = u.head;
      const int tok = ((gt + mine) * kTile + 16 * piece) & ~(bs - 1);  // the block's first token
      next.page = -1;
      if (mine < next.count && tok < u.any_hi && tok + bs > u.any_lo)
        next.page = __ldg(p.tables + u.seq * p.table_stride + (tok >> p.bs_log2));
      if (next.page >= p.num_blocks) next.page = -1;
      next.ks = next.vs = 0.f;
      if (next.page >= 0) {
        next.ks = __ldg(p.key_scale + next.page * p.ks_sb + next.head * p.ks_sh);
        next.vs = __ldg(p.value_scale + next.page * p.vs_sb + next.head * p.vs_sh);
      }
      if (!(fabsf(next.vs) < INFINITY)) {  // counts as 0 until the results: an integer weight cannot say so
        next.vs = 0.f;
        *odd = 1;
      }
      gt += next.count;
    };
    look_ahead();
    ready();
    Batch b = next;
    next.count = 0;
    bool looked = false;
    uint32_t k_sent = 0, v_sent = 0, k_slot = 0, k_parity = 1, v_slot = 0, v_parity = 1, idle = 0;
    int j = 0;
    // K of tile k_sent and V of tile v_sent, whichever has room; V's blocks are read back from shared memory
    while (b.count > 0 || v_sent < k_sent) {
      bool did = false;
      if (b.count > 0 && k_sent - v_sent < 12 && __all_sync(0xffffffffu, mbar_try(&sm.k_empty[k_slot], k_parity))) {
        const uint32_t ring = k_sent & 15;
        const bool on = mine == j && b.page >= 0;
        const uint32_t there = __ballot_sync(0xffffffffu, on), led = __ballot_sync(0xffffffffu, on && leads);
        if (on && leads) {
          if (p.bs_log2 == 4)
            bulk_load(k_to + k_slot * C::kTileBytes, p.key + b.page * p.k_sb + b.head * p.k_sh, bytes, &sm.k_full[k_slot]);
          else
            tensor_load(k_to + k_slot * C::kTileBytes, &kmap, b.head, b.page, &sm.k_full[k_slot]);
        }
        if (mine == j) {
          sm.ks[ring][piece] = b.ks;
          sm.vs[ring][piece] = b.vs;
          sm.page[ring][piece] = b.page;
          if (piece == 0) {
            sm.have[ring] = there >> (8 * j);
            sm.head[ring] = b.head;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect(&sm.k_full[k_slot], __popc(led) * bytes);
        ++k_sent;
        if (++k_slot == kKs) k_slot = 0, k_parity ^= 1;
        if (!looked) {
          look_ahead();
          looked = true;
        }
        if (++j == b.count) {
          b = next;
          j = 0;
          looked = false;
        }
        did = true;
      }
      if (v_sent < k_sent && __all_sync(0xffffffffu, mbar_try(&sm.v_empty[v_slot], v_parity))) {
        const uint32_t ring = v_sent & 15;
        const int page = lane < 8 && leads ? sm.page[ring][piece] : -1, head = sm.head[ring];
        const uint32_t led = __ballot_sync(0xffffffffu, page >= 0);
        if (page >= 0) {
          if (p.bs_log2 == 4)
            bulk_load(v_to + v_slot * C::kTileBytes, p.value + page * p.v_sb + head * p.v_sh, bytes, &sm.v_full[v_slot]);
          else
            tensor_load(v_to + v_slot * C::kTileBytes, &vmap, head, page, &sm.v_full[v_slot]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect(&sm.v_full[v_slot], __popc(led) * bytes);
        ++v_sent;
        if (++v_slot == kVs) v_slot = 0, v_parity ^= 1;
        did = true;
      }
      if (did) {
        idle = 0;
      } else if (++idle >= kWaitLimit || __any_sync(0xffffffffu, (idle & 255) == 255 && *gave_up)) {
        *gave_up = 1;
        break;
      }
    }
    // copies in flight end before the block does
    for (uint32_t i = k_sent > kKs ? k_sent - kKs : 0; i < k_sent; ++i)
      for (uint32_t z = 0; z < kWaitLimit && !mbar_try(&sm.k_full[i % kKs], (i / kKs) & 1); ++z) {
      }
    for (uint32_t i = v_sent > kVs ? v_sent - kVs : 0; i < v_sent; ++i)
      for (uint32_t z = 0; z < kWaitLimit && !mbar_try(&sm.v_full[i % kVs], (i / kVs) & 1); ++z) {
      }
  } else {
    ready();
    const uint32_t tmem = sm.tmem;
    if (lane == 0) {
    // ---- the tensor cores ---------------------------------------------------------
    constexpr int kFmt = CODE == MAK_CODE_INT8 ? 1 : 0, kAcc = CODE == MAK_CODE_INT8 ? 2 : 1;
    constexpr uint32_t kQk = instr_desc(C::kN, kAcc, kFmt, true, false), kPv = instr_desc(C::kN, kAcc, kFmt, false, true);
    const int line = p.bs_log2;
    // K: lines of 8 head_dim rows, then blocks; V: the same lines as rows of M
    const uint32_t k_lbo = line == 4 ? 128 : HD * bs, k_sbo = line == 4 ? HD * 16 : 8 * bs;
    const uint32_t v_lbo = line == 4 ? HD * 16 : 16, v_sbo = 8 * bs;
    auto mma = [&](uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
      if constexpr (CODE == MAK_CODE_INT8)
        mma_ss_i8(d, a, b, idesc, add);
      else
        mma_ss_f8(d, a, b, idesc, add);
    };
    // Descriptors differ in their addresses alone, in units of 16 bytes: no carry leaves that field.
    const uint64_t k_desc = smem_desc(smem_addr(sm.k), k_lbo, k_sbo, line);
    uint64_t q_desc = 0;
    const uint64_t v_desc = smem_desc(smem_addr(sm.v), v_lbo, v_sbo, line);
    const uint64_t p_desc = smem_desc(smem_addr(sm.p), 128, kTile * 16 * C::kStep, 0);
    constexpr uint32_t kTileStep = C::kTileBytes / 16;
    uint32_t v_step[kTile / 32];  // 32 tokens of V each
#pragma unroll
    for (int i = 0; i < kTile / 32; ++i) v_step[i] = (((32 * i) >> line) * (HD * bs) + ((32 * i) & (bs - 1))) >> 4;
    uint32_t it = 0, units = 0;
    int buf = 1;  // of q: unit by unit
    uint32_t k_slot = 0, k_parity = 0, v_slot = 0, v_parity = 0;
    bool ok = true;
    // scores of step x, `count` tiles
    auto scores = [&](uint32_t x, int count) {
      for (int y = 0; y < count; ++y) {
        if (!mbar_wait(&sm.k_full[k_slot], k_parity, gave_up)) return false;
        tc_fence_after();
        const uint64_t kd = k_desc + k_slot * kTileStep;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i)
          mma(tmem + C::kScores + ((x & 1) * C::kStep + y) * C::kN, kd + i * 2 * bs, q_desc + i * 16, kQk, i > 0);
        tc_commit(&sm.k_empty[k_slot]);
        if (++k_slot == kKs) k_slot = 0, k_parity ^= 1;
      }
      tc_commit(&sm.s_full[x & 1]);
      return true;
    };
    while (ok && next_unit<ROWS>(p, walk, u)) {
      const int n = u.t_last - u.t_first;
      buf ^= 1;
      if (n == 0) continue;
      const int steps = (n + C::kStep - 1) / C::kStep;
      ok = mbar_wait(&sm.q_full, units & 1, gave_up);
      ++units;
      q_desc = smem_desc(smem_addr(sm.q[buf]), 128, HD * 8, 0);
      for (int t = 0; t < 2 && t < steps && ok; ++t) ok = scores(it + t, min(C::kStep, n - t * C::kStep));
      for (int t = 0; t < steps && ok; ++t) {
        const uint32_t x = it + t;
        const int count = min(C::kStep, n - t * C::kStep);
        for (int y = 0; y < count && ok; ++y) {
          ok = mbar_wait(&sm.v_full[v_slot], v_parity, gave_up);
          if (y == 0) ok = ok && mbar_wait(&sm.p_full, x & 1, gave_up);
          if (!ok) break;
          tc_fence_after();
          const uint64_t vd = v_desc + v_slot * kTileStep, pd = p_desc + y * kTile;
#pragma unroll
          for (int h = 0; h < C::kParts; ++h)
#pragma unroll
            for (int i = 0; i < kTile / 32; ++i)
              mma(tmem + C::kOut + h * C::kN, vd + h * 8 * bs + v_step[i], pd + i * 32, kPv, y > 0 || i > 0);
          tc_commit(&sm.v_empty[v_slot]);
          if (++v_slot == kVs) v_slot = 0, v_parity ^= 1;
        }
        if (!ok) break;
        tc_commit(&sm.o_full);
        if (t + 2 < steps) ok = scores(x + 2, min(C::kStep, n - (t + 2) * C::kStep));
      }
      it += steps;
    }
    if (!ok) {  // let what was issued end before the TMEM is given back
      tc_commit(&sm.spare);
      for (uint32_t i = 0; i < kWaitLimit && !mbar_try(&sm.spare, 0); ++i) {
      }
    }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    __syncwarp();
    tc_fence_after();
    tmem_free<C::kTmem>(sm.tmem);
  }
}

template <int HD, int ROWS, int CODE>
int launch_rows(const BlockAttnParams& p, cudaStream_t st) {
  const auto kernel = block_attn_rows_kernel<HD, ROWS, CODE>;
  constexpr int kBytes = sizeof(Smem<HD, ROWS>);
  static_assert(kBytes <= (HD == 256 ? 227 : 113) * 1024, "blocks per SM");  // 228 KB less 1 KB per block
  // The occupancy query answers 1 for these kernels; two blocks do run where their shared memory, registers and
  // TMEM columns fit twice (11.7 of 12 warps active on average).  TMEM has 512 columns, and a block whose allocation
  // has to wait for another's end gains nothing.
  constexpr int kPerSm = HD == 256 || 2 * Cfg<HD, ROWS>::kTmem > 512 ? 1 : 2;
  static bool ready[kMaxDevices] = {};
  if (int rc = prepare_kernel(kernel, kBytes, ready)) return rc;
  CUtensorMap maps[2] = {};
  if (p.bs_log2 > 4 && p.num_blocks > 0) {
    if (int rc = cache_map(&maps[0], p.key, p.k_sb, p.k_sh, p.num_blocks, p.nh, HD, 1 << p.bs_log2)) return rc;
    if (int rc = cache_map(&maps[1], p.value, p.v_sb, p.v_sh, p.num_blocks, p.nh, HD, 1 << p.bs_log2)) return rc;
  }
  int64_t grid = kPerSm * sm_count();
  if (grid > kMaxGrid) grid = kMaxGrid;
  // no more blocks than there can be work for
  const int64_t seq_tiles = ((static_cast<int64_t>(p.max_blocks) << p.bs_log2) + kTile - 1) / kTile + 1 + kUnitCost;
  const int64_t groups = static_cast<int64_t>(p.num_rows) * p.group / ROWS + p.num_seqs;
  const int64_t most = (groups * p.nh * seq_tiles + kMinChunk - 1) / kMinChunk;
  if (most < grid) grid = most;
  return launch_pdl("mak_block_attention", kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), kBytes, st, p, maps[0], maps[1]);
}

template <int HD, int ROWS>
int launch_rows_code(const BlockAttnParams& p, int code, cudaStream_t st) {
  return code == MAK_CODE_INT8 ? launch_rows<HD, ROWS, MAK_CODE_INT8>(p, st) : launch_rows<HD, ROWS, MAK_CODE_E4M3>(p, st);
}

constexpr int64_t kCounterBytes = (2 * kMaxGrid * 4 + 255) / 256 * 256;

}  // namespace

int cache_map(CUtensorMap* map, const uint8_t* base, int64_t sb, int64_t sh, int64_t num_blocks, int nh, int hd, int bs) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  if (encode == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess || fn == nullptr) {
      (void)cudaGetLastError();
      return fail(MAK_E_CUDA, "mak_block_attention: no cuTensorMapEncodeTiled in this driver");
    }
    encode = reinterpret_cast<Encode>(fn);
  }
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(bs), static_cast<cuuint64_t>(hd), static_cast<cuuint64_t>(nh),
                              static_cast<cuuint64_t>(num_blocks)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(bs), static_cast<cuuint64_t>(sh), static_cast<cuuint64_t>(sb)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(bs), static_cast<cuuint32_t>(hd), 1, 1}, steps[4] = {1, 1, 1, 1};
  const CUtensorMapSwizzle swizzle =
      bs == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : bs == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
  const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t*>(base), dims, strides, box, steps,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(MAK_E_INVALID, "mak_block_attention: the cache's strides make no tensor map (%d)", static_cast<int>(rc));
  return MAK_OK;
}

int64_t block_attn_tc_partial_bytes();
int64_t block_attn_tc_plan_bytes();
bool block_attn_tc_fits(const BlockAttnParams& p);
int launch_block_attn_tc(const BlockAttnParams& p, int head_dim, int code, void* plan, cudaStream_t st);

int check_block_cache(const mak_block_cache_desc& c, const char* name) {
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
    return fail(MAK_E_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256, got %d", name, c.head_dim);
  if (c.block_size != 16 && c.block_size != 32 && c.block_size != 64 && c.block_size != 128)
    return fail(MAK_E_UNSUPPORTED, "%s: block_size must be 16, 32, 64 or 128, got %d", name, c.block_size);
  if (c.code_type != MAK_CODE_INT8 && c.code_type != MAK_CODE_E4M3)
    return fail(MAK_E_INVALID, "%s: unknown code type %d", name, c.code_type);
  if (c.num_seqs < 0 || c.num_blocks < 0 || c.max_blocks < 0 || c.num_rows < 0 || c.num_heads <= 0)
    return fail(MAK_E_INVALID, "%s: negative size", name);
  if (c.num_seqs > 0x7fffffff || c.num_blocks > 0x7fffffff || c.num_rows > 0x7fffffff ||
      c.max_blocks > 0x7fffffff / c.block_size)
    return fail(MAK_E_UNSUPPORTED, "%s: sequences, blocks, rows and tokens of a sequence are 32-bit counts", name);
  if (c.num_seqs > 0 && (c.context_lens == nullptr || (c.max_blocks > 0 && c.block_tables == nullptr)))
    return fail(MAK_E_INVALID, "%s: null block_tables or context_lens", name);
  if (c.num_blocks > 0 && (c.key == nullptr || c.value == nullptr || c.key_scale == nullptr || c.value_scale == nullptr))
    return fail(MAK_E_INVALID, "%s: null cache", name);
  const uint64_t bits = reinterpret_cast<uintptr_t>(c.key) | reinterpret_cast<uintptr_t>(c.value) |
                        static_cast<uint64_t>(c.key_stride_block | c.key_stride_head | c.value_stride_block | c.value_stride_head);
  if (bits & 15) return fail(MAK_E_INVALID, "%s: caches need 16-byte aligned addresses and block / head strides", name);
  return MAK_OK;
}

}  // namespace mak

using namespace mak;

// counters, the plan of the many-row kernel, partial sums of either kernel
static int64_t plan_bytes() { return (block_attn_tc_plan_bytes() + 255) / 256 * 256; }

extern "C" int64_t mak_block_attention_workspace_bytes(void) {
  const int64_t few = static_cast<int64_t>(2 * kMaxGrid) * kMaxRows * (kMaxDim + 2) * 4, many = block_attn_tc_partial_bytes();
  return kCounterBytes + plan_bytes() + (few > many ? few : many);
}

extern "C" int mak_block_attention(const mak_block_attn_desc* d, void* stream) {
  const char* name = "mak_block_attention";
  if (d == nullptr) return fail(MAK_E_INVALID, "%s: null descriptor", name);
  const mak_block_cache_desc& c = d->cache;
  if (int rc = check_block_cache(c, name)) return rc;
  if (d->q_dtype != MAK_DT_F16 && d->q_dtype != MAK_DT_BF16)
    return fail(MAK_E_UNSUPPORTED, "%s: q must be float16 or bfloat16", name);
  if (d->num_q_heads <= 0 || d->num_q_heads % c.num_heads)
    return fail(MAK_E_INVALID, "%s: %d query heads over %d cache heads", name, d->num_q_heads, c.num_heads);
  if (d->window < 0 || (d->window > 0 && !d->causal))
    return fail(MAK_E_INVALID, "%s: a window needs causal attention", name);
  if (c.num_seqs == 0 || c.num_rows == 0) return MAK_OK;
  if (d->q == nullptr || d->out == nullptr) return fail(MAK_E_INVALID, "%s: null q or out", name);
  if ((reinterpret_cast<uintptr_t>(d->q) & 15) || ((d->q_stride_row | d->q_stride_head) & 7))
    return fail(MAK_E_INVALID, "%s: q needs 16-byte aligned rows", name);
  if (d->workspace == nullptr || d->workspace_bytes < mak_block_attention_workspace_bytes())
    return fail(MAK_E_WORKSPACE, "%s: workspace missing or too small", name);
  // partial sums are read from it 16 bytes at a time
  if (reinterpret_cast<uintptr_t>(d->workspace) & 15) return fail(MAK_E_WORKSPACE, "%s: the workspace must begin on 16 bytes", name);
  BlockAttnParams p = {};
  p.key = static_cast<const uint8_t*>(c.key);
  p.value = static_cast<const uint8_t*>(c.value);
  p.key_scale = c.key_scale;
  p.value_scale = c.value_scale;
  p.k_sb = c.key_stride_block, p.k_sh = c.key_stride_head;
  p.v_sb = c.value_stride_block, p.v_sh = c.value_stride_head;
  p.ks_sb = c.key_scale_stride_block, p.ks_sh = c.key_scale_stride_head;
  p.vs_sb = c.value_scale_stride_block, p.vs_sh = c.value_scale_stride_head;
  p.tables = c.block_tables;
  p.ctx_lens = c.context_lens;
  p.starts = c.cu_seqlens;
  p.table_stride = c.table_stride;
  p.num_blocks = c.num_blocks;
  p.q = d->q, p.out = d->out, p.lse = d->lse;
  p.q_sr = d->q_stride_row, p.q_sh = d->q_stride_head, p.o_sr = d->out_stride_row, p.o_sh = d->out_stride_head;
  p.num_seqs = static_cast<int32_t>(c.num_seqs);
  p.max_blocks = static_cast<int32_t>(c.max_blocks);
  p.num_rows = static_cast<int32_t>(c.num_rows);
  p.nh = c.num_heads;
  p.group = d->num_q_heads / c.num_heads;
  p.bs_log2 = c.block_size == 16 ? 4 : c.block_size == 32 ? 5 : c.block_size == 64 ? 6 : 7;
  p.q_bf16 = d->q_dtype == MAK_DT_BF16;
  p.causal = d->causal != 0;
  p.window = d->window;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.counters = static_cast<int32_t*>(d->workspace);
  p.partial = reinterpret_cast<float*>(static_cast<char*>(d->workspace) + kCounterBytes + plan_bytes());
  cudaStream_t st = as_stream(stream);
  // Rows that share a cache head, on average.  Above 32 the many-row kernel costs less whatever the lengths:
  // 16 sequences of 4096 tokens, 8 cache heads of 128: 32 rows 81.6 us here and 83.9 there, 40 rows 117 and 84, 64 rows
  // 154 and 85; heads of 64: 32 rows 74 and 70, 64 rows 137 and 71; one sequence of 2000: 64 rows 23.3 and 25.3, 128 rows
  // 26.6 and 28.0, of 16000: 64 rows 46 and 43, 128 rows 73 and 55.
  const int64_t rows = c.num_rows * p.group / c.num_seqs;
  if (rows > 32 && c.head_dim <= 128 && block_attn_tc_fits(p))
    return launch_block_attn_tc(p, c.head_dim, c.code_type, static_cast<char*>(d->workspace) + kCounterBytes, st);
  // Groups of 16 rows instead of 8, but where three of 8 hold them: the same cache, heads of 128, groups of 8 and of 16:
  // 8 rows 36 and 50 us, 12 rows 52.2 and 51.7, 16 rows 52.8 and 52.8, 24 rows 73 and 81, 32 rows 94 and 81; heads of 64:
  // 12 rows 50 and 45, 24 rows 67 and 73, 32 rows 87 and 74.  Heads of 256 leave shared memory for groups of 8 alone.
  const bool wide = c.head_dim < 256 && rows > 8 && (rows <= 16 || rows > 24);
  // Groups of 4, groups of 8: one row, 4 query heads on each of 8 cache heads, 16 x 4096, 64 x 512, 1 x 777 tokens: heads
  // of 64: 28.9 and 31.1, 23.9 and 29.9, 10.2 and 11.4 us; of 128: 33.3 and 36.1, 24.4 and 30.8, 10.9 and 11.6; of 256:
  // 56 and 60, 39 and 49, 11.7 and 12.9.
  if (rows <= 4)
    return c.head_dim == 64    ? launch_rows_code<64, 4>(p, c.code_type, st)
           : c.head_dim == 128 ? launch_rows_code<128, 4>(p, c.code_type, st)
                               : launch_rows_code<256, 4>(p, c.code_type, st);
  if (c.head_dim == 64) return wide ? launch_rows_code<64, 16>(p, c.code_type, st) : launch_rows_code<64, 8>(p, c.code_type, st);
  if (c.head_dim == 128) return wide ? launch_rows_code<128, 16>(p, c.code_type, st) : launch_rows_code<128, 8>(p, c.code_type, st);
  return launch_rows_code<256, 8>(p, c.code_type, st);
}
