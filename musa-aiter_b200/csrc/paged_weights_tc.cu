// The attention weights that cached tokens gather, for many rows per sequence: the scores on the tcgen05 tensor cores.
//
// S^T = K Q^T of 128 tokens and 128 rows at a time (the heads of a group next to one another), in tensor memory: a thread
// has a token, its sum runs over the columns and stays in a register, so no thread waits for another's maximum or sum.
// A weight is 2^(s scale log2 e - lse log2 e): one rounding of the difference and that of lse log2 e, 2^-24 of 2^4 or so.
//
// Bound by the exponentials: 16 a cycle and SM take 1024 cycles for a chunk of 128 x 128, the products 512.  Sixteen warps
// take them, so that loads from tensor memory and waits hide behind one another's exponentials.  Measured, calls in a graph,
// 8 cache heads of 128 for 32 query heads: two prompts of 1500 to 2048 rows on 4000 to 6000 tokens 216 us; 16 sequences of
// 4096 tokens with 8 rows 80 us, a unit's beginning and end for the most part.  Eight warps: 227 and 104 us, 220 with three
// of eight pairs of exponentials by polynomial, which gains nothing with sixteen.
//
// A unit is a tile of 128 tokens of one cache head, its work the chunks of rows that see it; K of a unit is loaded once, the
// rows stream by TMA.  All units laid end to end are cut into equal runs, one per block; a unit cut by that leaves partial
// sums, and the last block to arrive adds them in order of position, so results do not depend on timing.  Roles:
//   warps 0-15  exponentials: 32 columns of a chunk each, a thread per token (TMEM lane)
//   warp 16     TMA loads of K and rows
//   warp 17     one thread issues all tcgen05.mma
//   warp 18     lse of the rows
#include "paged_weights.cuh"
#include "tcgen05.cuh"

namespace mak {
namespace {

constexpr int kTile = 128;     // tokens of a unit
constexpr int kMath = 16;      // warps of the exponentials
constexpr int kSides = kMath / 4, kCols = kTile / kSides;  // columns of a warp
constexpr int kThreads = 32 * (kMath + 4);
constexpr int kMaxGrid = 148;
constexpr int kUnitCost = 2;   // a unit's beginning and end, in chunks
constexpr int kMinRun = 4;     // chunks that are worth another block
constexpr int kPlaces = 4;     // for scores in tensor memory
constexpr int kQ = 4, kK = 2;  // chunks of rows and tiles of K in shared memory
static_assert(kCols == 32, "one word of columns");
static_assert(kMaxGrid * 4 <= kPagedCounterBytes, "a counter per block");
constexpr int kHave = 16;      // units whose pages are remembered
constexpr float kLog2e = 1.4426950408889634f;

// Tiles of a sequence: those that some row sees, or, where sums begin, all places of its row of sums.
struct Seq {
  PagedSeq v;
  Span s;
  int tiles;
};
__device__ __forceinline__ Seq seq_of(const WeightParams& w, int s) {
  Seq x;
  x.v = paged_seq(w.a, s);
  x.s = Span{};
  if (x.v.rows > 0) x.s = span_of<kTile>(w.a, x.v, 0, x.v.rows - 1);
  x.tiles = sum_row(w, s) < 0 ? 0 : w.add ? x.s.tiles : (w.max_tokens + kTile - 1) / kTile;
  return x;
}
__device__ __forceinline__ int tile_at(const WeightParams& w, const Seq& x, int j) { return w.add ? tile_token<kTile>(x.s, j) : j * kTile; }

// Chunks [c0, c1) of rows that see a token of the tile at tok; a chunk is `per` rows of the sequence.
__device__ __forceinline__ void chunks_of(const WeightParams& w, const Seq& x, int tok, int per, int* c0, int* c1) {
  *c0 = *c1 = 0;
  const PagedParams& p = w.a;
  if (x.v.rows == 0 || tok >= x.s.any_hi || (tok + kTile <= x.s.any_lo && tok >= p.sinks)) return;
  const int base = x.v.ctx - x.v.rows;  // position of row 0
  const int i0 = max(tok - base, 0);
  int i1 = x.v.rows - 1;
  if (p.window > 0 && tok >= p.sinks) {
    const int64_t last = static_cast<int64_t>(tok) + kTile - 1 - base + p.window - 1;
    if (last < i1) i1 = static_cast<int>(last);
  }
  if (i0 > i1) return;
  *c0 = i0 / per;
  *c1 = i1 / per + 1;
}

__global__ void __launch_bounds__(256) weights_plan_kernel(const __grid_constant__ WeightParams w, int64_t* work, int per) {
  __shared__ int64_t sums[8];
  pdl_wait();
  pdl_trigger();
  const Seq x = seq_of(w, blockIdx.x);
  int64_t mine = 0;
  for (int j = threadIdx.x; j < x.tiles; j += 256) {
    int c0, c1;
    chunks_of(w, x, tile_at(w, x, j), per, &c0, &c1);
    mine += kUnitCost + max(c1 - c0, 1);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) mine += sums[i];
    work[blockIdx.x] = mine * w.a.nh;
  }
}

struct Walk {
  int64_t at, end, w0;  // w0: where the current unit begins
  int seq, tile, head;
};
struct Unit {
  PagedSeq v;
  int seq, head, tok, any_lo, any_hi;
  int c0, n;       // this block has n chunks from c0 on
  int ta, tb, len; // of the unit's len, at least 1
  int64_t wt;      // where the unit's chunks begin in all work
};
__device__ __forceinline__ bool next_unit(const WeightParams& w, Walk& k, Unit& u, int per) {
  while (k.at < k.end) {
    const Seq x = seq_of(w, k.seq);
    if (k.tile >= x.tiles) {
      k.tile = k.head = 0;
      ++k.seq;
      continue;
    }
    const int tok = tile_at(w, x, k.tile);
    int c0, c1;
    chunks_of(w, x, tok, per, &c0, &c1);
    const int len = max(c1 - c0, 1);
    u.ta = static_cast<int>(max(k.at - k.w0 - kUnitCost, static_cast<int64_t>(0)));
    u.tb = static_cast<int>(min(k.end - k.w0 - kUnitCost, static_cast<int64_t>(len)));
    u.len = len, u.wt = k.w0 + kUnitCost;
    u.v = x.v, u.seq = k.seq, u.head = k.head, u.tok = tok;
    u.any_lo = x.s.any_lo, u.any_hi = x.s.any_hi;
    u.c0 = c0 + u.ta;
    u.n = c1 > c0 ? u.tb - u.ta : 0;
    k.w0 += kUnitCost + len;
    k.at = k.w0;
    if (++k.head == w.a.nh) k.head = 0, ++k.tile;
    if (u.tb > u.ta) return true;
  }
  return false;
}

__device__ __forceinline__ void math_sync() { asm volatile("bar.sync 1, 512;" ::: "memory"); }
__device__ __forceinline__ void box3(uint32_t to, const void* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}

template <int HD>
struct TcSmem {
  static constexpr int kBytes = kTile * HD * 2;
  alignas(1024) uint8_t q[kQ][kBytes];  // pieces of [128][64], lines of 128 bytes swizzled
  alignas(1024) uint8_t k[kK][kBytes];
  alignas(16) float lse[kQ][kTile];     // negated, times log2 e
  alignas(8) uint64_t q_full[kQ], q_empty[kQ], k_full[kK], k_empty[kK], s_full[kPlaces], s_empty[kPlaces], spare;
  int64_t before[kThreads + 1];
  int64_t sums[kThreads / 32];
  float side[kSides][kTile];
  uint32_t have[kHave];  // bit c: 16 tokens c of a unit's tile have a page
  uint32_t tmem;
  int gave_up, last;
};

template <int HD, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    weights_tc_kernel(const __grid_constant__ WeightParams w, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap q_map,
                      const int64_t* work, int per) {
  using Sm = TcSmem<HD>;
  constexpr int kBytes = Sm::kBytes, kPieces = HD / 64;
  extern __shared__ __align__(1024) uint8_t raw[];
  Sm& sm = *reinterpret_cast<Sm*>(raw);
  const PagedParams& p = w.a;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  pdl_wait();
  pdl_trigger();

  // ---- the run of this block ----------------------------------------------------
  const int share = (p.num_seqs + kThreads - 1) / kThreads;
  {
    const int s0 = min(tid * share, p.num_seqs), s1 = min(s0 + share, p.num_seqs);
    int64_t mine = 0;
    for (int s = s0; s < s1; ++s) mine += work[s];
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) sm.sums[warp] = incl;
    if (tid == 0) {
      sm.gave_up = 0;
      mbar_init(&sm.spare, 1);
      for (int i = 0; i < kQ; ++i) mbar_init(&sm.q_full[i], 2), mbar_init(&sm.q_empty[i], 1 + kMath);
      for (int i = 0; i < kK; ++i) mbar_init(&sm.k_full[i], 1), mbar_init(&sm.k_empty[i], 1);
      for (int i = 0; i < kPlaces; ++i) mbar_init(&sm.s_full[i], 1), mbar_init(&sm.s_empty[i], kMath);
      mbar_init_fence();
    }
    if (warp == kMath + 1) tmem_alloc<512>(&sm.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    int64_t at = incl - mine;
    for (int i = 0; i < warp; ++i) at += sm.sums[i];
    sm.before[tid] = at;
    if (tid == kThreads - 1) sm.before[kThreads] = at + mine;
    __syncthreads();
  }
  const uint32_t tmem = sm.tmem;
  volatile int* gave_up = &sm.gave_up;
  const int64_t total = sm.before[kThreads];
  int64_t run = (total + gridDim.x - 1) / gridDim.x;
  if (run < kMinRun) run = kMinRun;
  Walk walk;
  walk.at = blockIdx.x * run;
  walk.end = min(walk.at + run, total);
  const int64_t begin = walk.at;
  const bool busy = walk.at < walk.end;
  if (busy) {
    int lo = 0, n = kThreads;  // the last thread whose sequences begin at or before the run
    while (n > 1) {
      const int step = (n + 31) >> 5, at = lo + lane * step;
      const uint32_t votes = __ballot_sync(0xffffffffu, at < lo + n && sm.before[min(at, kThreads)] <= begin);
      const int k = 31 - __clz(votes), last = lo + n;
      lo += k * step;
      n = min(step, last - lo);
    }
    int64_t at = sm.before[lo];
    walk.seq = lo * share;
    for (; begin >= at + work[walk.seq]; ++walk.seq) at += work[walk.seq];
    // tiles of the sequence, 32 at a time
    const Seq x = seq_of(w, walk.seq);
    walk.tile = 0;
    for (;; walk.tile += 32) {
      int c0 = 0, c1 = 0, len = 0;
      if (walk.tile + lane < x.tiles) {
        chunks_of(w, x, tile_at(w, x, walk.tile + lane), per, &c0, &c1);
        len = kUnitCost + max(c1 - c0, 1);
      }
      int64_t incl = static_cast<int64_t>(len) * p.nh;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, at + incl > begin);
      if (past == 0) {
        at += __shfl_sync(0xffffffffu, incl, 31);
        continue;
      }
      const int first = __ffs(past) - 1;
      len = __shfl_sync(0xffffffffu, len, first);
      at += __shfl_sync(0xffffffffu, incl, first) - static_cast<int64_t>(len) * p.nh;
      walk.tile += first;
      walk.head = static_cast<int>((begin - at) / len);
      walk.w0 = at + static_cast<int64_t>(len) * walk.head;
      break;
    }
  }

  Unit u;
  bool ok = true;
  if (warp < kMath) {
    // ---- exponentials ----------------------------------------------------------------
    const int side = warp >> 2, r = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t g = 0, units = 0;  // chunks so far
    while (busy && next_unit(w, walk, u, per)) {
      const int t = u.tok + r;
      const int64_t base = static_cast<int64_t>(u.v.ctx) - u.v.rows;
      float2 sum[2] = {both(0.f), both(0.f)};
      bool there = false;
      // this thread adds the unit's sum of token t to what the row holds
      float* dst = w.sums + sum_row(w, u.seq) * w.sum_sr + u.head * w.sum_sh + t;
      const bool mine = side == 0 && t < w.max_tokens && (!w.add || (t < u.any_hi && (t >= u.any_lo || t < p.sinks)));
      for (int i = 0; i < u.n; ++i, ++g) {
        const uint32_t st = g % kPlaces, qs = g % kQ;
        static_assert(kQ == kPlaces, "one count for both");
        ok = ok && wait_warp(&sm.s_full[st], (g / kPlaces) & 1, gave_up);
        tc_fence_after();
        if (i == 0) there = sm.have[units % kHave] >> (r >> 4) & 1;
        uint32_t x[kCols];
        tmem_ld(tmem + lanes + st * 128 + side * kCols, x);
        tmem_wait(x);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.s_empty[st]);
        // Columns [from, to) are rows that see token t: those from its own position on, until their window has left it.
        const int64_t i0 = static_cast<int64_t>(u.c0 + i) * per;  // the chunk's first row
        const int64_t live = min(u.v.rows - i0, static_cast<int64_t>(per));
        int64_t a = (t - base - i0) * p.group, b = live * p.group;
        if (p.window > 0 && t >= p.sinks) b = min(b, (t - base - i0 + p.window) * p.group);
        if (!there || t >= u.v.room) b = 0;
        const int from = static_cast<int>(min(max(a - side * kCols, static_cast<int64_t>(0)), static_cast<int64_t>(kCols)));
        const int to = static_cast<int>(min(max(b - side * kCols, static_cast<int64_t>(0)), static_cast<int64_t>(kCols)));
        ok = ok && wait_warp(&sm.q_full[qs], (g / kQ) & 1, gave_up);  // has been: for what the last warp wrote
        const float4* lse = reinterpret_cast<const float4*>(sm.lse[qs] + side * kCols);
        const bool whole = __all_sync(0xffffffffu, from == 0 && to == kCols), none = __all_sync(0xffffffffu, to <= from);
        if (whole) {
#pragma unroll
          for (int e = 0; e < kCols / 4; ++e) {
            const float4 f = lse[e];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const int c = e * 4 + z * 2;
              float2 y = fma2(make_float2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), both(p.scale_log2), z ? make_float2(f.z, f.w) : make_float2(f.x, f.y));
              y.x = exp2_near(y.x);
              y.y = exp2_near(y.y);
              sum[z] = add2(sum[z], y);
            }
          }
        } else if (!none) {
          auto below = [](int k) { return k >= 32 ? 0xffffffffu : (1u << k) - 1u; };
          const uint32_t bits = below(to) & ~below(from);
#pragma unroll
          for (int e = 0; e < kCols / 4; ++e) {
            const float4 f = lse[e];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const int c = e * 4 + z * 2;
              const float2 y = fma2(make_float2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), both(p.scale_log2), z ? make_float2(f.z, f.w) : make_float2(f.x, f.y));
              sum[z].x += bits >> c & 1 ? exp2_near(y.x) : 0.f;
              sum[z].y += bits >> (c + 1) & 1 ? exp2_near(y.y) : 0.f;
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_empty[qs]);  // lse is read
      }
      sum[0] = add2(sum[0], sum[1]);
      float got = sum[0].x + sum[0].y;
      if (!ok) got = __uint_as_float(0x7fffffffu);  // a block that gave up leaves NaN
      if (u.n > 0) ++units;
      if (side > 0) sm.side[side][r] = got;
      math_sync();
      const bool cut = u.ta > 0 || u.tb < u.len;
      const int64_t first_block = cut ? u.wt / run : 0, last_block = cut ? (u.wt + u.len - 1) / run : 0;
      auto piece = [&](int64_t block) { return p.partial + (2 * block + (u.wt > block * run ? 1 : 0)) * kTile + r; };
      if (side == 0) {
#pragma unroll
        for (int z = 1; z < kSides; ++z) got += sm.side[z][r];
        if (cut) *piece(blockIdx.x) = got;
      }
      if (cut) {
        math_sync();
        if (tid == 0) {  // releases what the barrier has gathered
          int ticket;
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(ticket) : "l"(p.counters + first_block) : "memory");
          sm.last = ticket == last_block - first_block;
          if (sm.last) p.counters[first_block] = 0;
        }
        math_sync();
        if (sm.last && side == 0) {
          got = 0.f;
          for (int64_t b = first_block; b <= last_block; ++b) got += __ldcg(piece(b));
        }
      }
      if (mine && (!cut || sm.last)) *dst = (w.add ? *dst : 0.f) + got;
      math_sync();  // side and last are read
    }
  } else if (warp == kMath) {
    // ---- loads --------------------------------------------------------------------------
    const int bs = 1 << p.bs_log2, box = min(bs, kTile), pages = kTile / box, cols = per * p.group;
    uint32_t g = 0, units = 0;
    while (ok && busy && next_unit(w, walk, u, per)) {
      if (u.n == 0) continue;
      const int32_t* table = p.tables + u.seq * p.table_stride;
      int page = -1;
      const int tok = u.tok + lane * box;
      if (lane < pages && tok < u.v.room) page = page_of(p, table, tok);
      const uint32_t votes = __ballot_sync(0xffffffffu, page >= 0);
      int id[kTile / 16];
#pragma unroll
      for (int i = 0; i < kTile / 16; ++i) id[i] = __shfl_sync(0xffffffffu, page, i);
      const uint32_t ks = units % kK;
      ok = wait_warp(&sm.k_empty[ks], ((units / kK) & 1) ^ 1, gave_up);
      if (!ok) break;
      uint32_t have = 0;
      for (int c = 0; c < kTile / 16; ++c) have |= (votes >> (c * 16 / box) & 1) << c;
      if (lane == 0) sm.have[units % kHave] = have;
      __syncwarp();
      const int head = __shfl_sync(0xffffffffu, u.head, 0), n = __shfl_sync(0xffffffffu, u.n, 0);
      if (elect_one()) {
        mbar_arrive_expect(&sm.k_full[ks], kBytes);
#pragma unroll
        for (int i = 0; i < kTile / 16; ++i) {
          if (i >= pages) break;
          // a block that there is not: the load fills zeros
#pragma unroll
          for (int c = 0; c < kPieces; ++c) box_load(smem_addr(sm.k[ks]) + c * 16384 + i * box * 128, &k_map, c * 64, head, 0, id[i], &sm.k_full[ks]);
        }
      }
      ++units;
      const int64_t row0 = static_cast<int64_t>(u.v.first) + static_cast<int64_t>(u.c0) * per;
      for (int i = 0; i < n; ++i, ++g) {
        const uint32_t qs = g % kQ;
        ok = wait_warp(&sm.q_empty[qs], ((g / kQ) & 1) ^ 1, gave_up);
        if (!ok) break;
        if (elect_one()) {
          mbar_arrive_expect(&sm.q_full[qs], cols * HD * 2);
#pragma unroll
          for (int c = 0; c < kPieces; ++c)
            box3(smem_addr(sm.q[qs]) + c * 16384, &q_map, c * 64, head * p.group, static_cast<int>(row0 + static_cast<int64_t>(i) * per), &sm.q_full[qs]);
        }
      }
    }
    if (!ok) {  // the copies in flight end before the block does
      for (uint32_t t = g > kQ ? g - kQ : 0; t < g; ++t)
        for (uint32_t i = 0; i < kWaitLimit && !mbar_try(&sm.q_full[t % kQ], (t / kQ) & 1); ++i) {
        }
      for (uint32_t t = units > kK ? units - kK : 0; t < units; ++t)
        for (uint32_t i = 0; i < kWaitLimit && !mbar_try(&sm.k_full[t % kK], (t / kK) & 1); ++i) {
        }
    }
  } else if (warp == kMath + 1) {
    // ---- the tensor cores -------------------------------------------------------
    constexpr uint32_t kIdesc = instr_desc(kTile, 1, BF16 ? 1 : 0, false, false);
    const uint64_t q_desc = smem_desc(smem_addr(sm.q), 16, 1024, 7), k_desc = smem_desc(smem_addr(sm.k), 16, 1024, 7);
    constexpr uint32_t kBuffer = kBytes / 16;
    uint32_t g = 0, units = 0;
    while (ok && busy && next_unit(w, walk, u, per)) {
      const int n = __shfl_sync(0xffffffffu, u.n, 0);
      if (n == 0) continue;
      const uint32_t ks = units % kK;
      ok = wait_warp(&sm.k_full[ks], (units / kK) & 1, gave_up);
      for (int i = 0; i < n && ok; ++i, ++g) {
        const uint32_t st = g % kPlaces;
        ok = wait_warp(&sm.q_full[st], (g / kQ) & 1, gave_up) && wait_warp(&sm.s_empty[st], ((g / kPlaces) & 1) ^ 1, gave_up);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t kd = k_desc + ks * kBuffer, qd = q_desc + st * kBuffer;
          steps<HD / 16>([&](auto z) {
            constexpr int s = decltype(z)::value, at = (s >> 2) * 1024 + (s & 3) * 2;
            mma_ss_f16<at, at>(tmem + st * 128, kd, qd, kIdesc, s > 0);
          });
          tc_commit(&sm.s_full[st]);
          tc_commit(&sm.q_empty[st]);
          if (i + 1 == n) tc_commit(&sm.k_empty[ks]);
        }
      }
      ++units;
    }
    if (!ok) {  // let what was issued end before the TMEM is given back
      if (elect_one()) tc_commit(&sm.spare);
      __syncwarp();
      for (uint32_t i = 0; i < kWaitLimit && !mbar_try(&sm.spare, 0); ++i) {
      }
    }
  } else if (warp == kMath + 2) {
    // ---- lse ---------------------------------------------------------------------
    const int cols = per * p.group;
    uint32_t g = 0;
    while (ok && busy && next_unit(w, walk, u, per)) {
      auto fetch = [&](int i, float(&x)[4]) {  // of chunk i, columns 4 lane .. 4 lane + 3
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = lane * 4 + e;
          const int64_t row = static_cast<int64_t>(u.c0 + i) * per + c / p.group;
          x[e] = i < u.n && c < cols && row < u.v.rows
                     ? __ldg(w.lse + (u.v.first + row) * w.lse_sr + u.head * p.group + c % p.group)
                     : 0.f;
        }
      };
      float next[4];
      fetch(0, next);
      for (int i = 0; i < u.n; ++i, ++g) {
        const uint32_t qs = g % kQ;
        const float4 f = make_float4(next[0] * -kLog2e, next[1] * -kLog2e, next[2] * -kLog2e, next[3] * -kLog2e);
        fetch(i + 1, next);
        ok = wait_warp(&sm.q_empty[qs], ((g / kQ) & 1) ^ 1, gave_up);
        if (!ok) break;
        reinterpret_cast<float4*>(sm.lse[qs])[lane] = f;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full[qs]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMath + 1) {
    __syncwarp();
    tc_fence_after();
    tmem_free<512>(tmem);
  }
}

template <int HD, bool BF16>
int launch(const WeightParams& w, const char* name, const CUtensorMap& k, const CUtensorMap& q, int64_t* work, int per, cudaStream_t st) {
  constexpr int kBytes = sizeof(TcSmem<HD>);
  static_assert(kBytes <= 227 * 1024, "shared memory of a block");
  const auto kernel = weights_tc_kernel<HD, BF16>;
  static bool ready[kPagedDevices] = {};
  if (int rc = paged_prepare(name, kernel, kBytes, ready)) return rc;
  if (int rc = launch_pdl(name, weights_plan_kernel, dim3(static_cast<unsigned>(w.a.num_seqs)), dim3(256), 0, st, w, work, per)) return rc;
  const int sms = sm_count();
  return launch_pdl(name, kernel, dim3(sms < kMaxGrid ? sms : kMaxGrid), dim3(kThreads), kBytes, st, w, k, q, static_cast<const int64_t*>(work), per);
}

}  // namespace

// Rows of q as boxes of the `group` heads of a cache head times `per` rows, 64 columns of them, lines of 128 bytes swizzled.
static bool rows_map(CUtensorMap* map, const uint16_t* base, int64_t sr, int64_t sh, int64_t rows, int heads, int hd, bool bf16, int group, int per) {
  const int64_t dims[4] = {hd, heads, rows, 1}, strides[3] = {sh * 2, sr * 2, 0};
  const uint32_t box[4] = {64, static_cast<uint32_t>(group), static_cast<uint32_t>(per), 1};
  return paged_encode(map, base, 3, dims, strides, box, bf16);
}

bool weights_tc_fits(const WeightParams& w) { return w.a.group <= kTile && w.a.num_rows > 0; }

int launch_weights_tc(const WeightParams& w, int head_dim, bool bf16, const char* name, const CUtensorMap& k, int64_t* work, cudaStream_t st) {
  const PagedParams& p = w.a;
  const int per = kTile / p.group;
  CUtensorMap q;
  if (!rows_map(&q, p.q, p.q_sr, p.q_sh, p.num_rows, p.nh * p.group, head_dim, bf16, p.group, per))
    return fail(MAK_E_INVALID, "%s: the strides of q make no tensor map", name);
  if (head_dim == 64) return bf16 ? launch<64, true>(w, name, k, q, work, per, st) : launch<64, false>(w, name, k, q, work, per, st);
  return bf16 ? launch<128, true>(w, name, k, q, work, per, st) : launch<128, false>(w, name, k, q, work, per, st);
}

}  // namespace mak
