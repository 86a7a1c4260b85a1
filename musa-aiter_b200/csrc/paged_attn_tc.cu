// Attention over a paged 16-bit cache for many rows per sequence (prompts, trees): the products on the tcgen05 tensor
// cores, K and V brought in by TMA as they lie in their pages.
//
// S = q K^T and O = P V with S, P and O in tensor memory: of each row of 64 scores the largest is found, weights
// 2^(S c - m') are written over the scores in 16 bits and multiply V.  Sums, maxima and accumulators are 32-bit; a weight is
// rounded once to the cache's type, which the tensor cores take next to V (wider weights at half the rate): its error, half
// a step of itself, is what rounding a result adds too.  The running maximum is only moved where it grew by more than
// 2^kLazy, so accumulators are rarely rescaled; the result is the same.
//
// A block takes 256 rows of one cache head (heads of the group next to one another, so a K / V tile serves all of them) as
// two halves of 128 and walks the tokens in tiles of 64, with two places for each half's scores: while those of one tile
// are exponentiated the tensor cores make the next ones and multiply the last weights.  Of a unit with 128 rows or fewer
// each half takes every other tile instead, and the two are joined.  Roles:
//   warps 0-3, 4-7   softmax of half 0 / 1, a thread per row (TMEM lane)
//   warps 8, 9       page ids and TMA loads of K / V
//   warps 10, 11     a thread issues all tcgen05.mma of half 0 / 1: while one waits the other's products run
//   warps 12-15      values in tiles that not every row sees whole: infinite and NaN ones become 0 there
//
// What a row does not see reaches none of its sums: its weights there are 0, and 0 times a value that is no number is
// kept out by warps 12-15; the rows that do see such a value get it with their results (odd_sum).  Tiles that all rows see
// whole are left as they are.  There a weight too light for 16 bits makes NaN of an infinite value, so a NaN in the result of a
// row whose scores are all numbers is looked into at the unit's end: what it sees of values that are no numbers is its result.
//
// Work.  All (row tile, head) units laid end to end, each as long as the tiles it sees, are cut into equal runs, one per
// block; a small launch before this one adds up the lengths.  A unit cut by that leaves partial sums, and the last block to
// arrive joins them in order of position, so results do not depend on timing.
//
// Bound by the chain of scores, softmax and products within a half, and by the tensor cores' reading of shared memory: a
// 128 x 64 x 16 product reads its operands in 48 cycles and multiplies in 32, so a pair of tiles needs 1280 cycles of the
// tensor cores where the softmax needs some 1000.  Measured, calls in a graph, 8 cache heads of 128 in bfloat16 for 32 query
// heads: two prompts of 1500 to 2048 rows on 5000 to 8192 tokens, window of 4096, 257 us, 919 TFLOP/s of the 1692 that a plain
// matrix product has (270 to 290 under lasting load); the beginnings and ends of units are a ninth of that.
// 16 trees of 8 to 32 tokens on 300 to 4500 tokens 71 us, beginnings, ends and joins for the most part (K and V alone: 22).
// Light weights of infinite values are looked for at a unit's end alone; weights kept above 0 in every tile took the prompts 4 %,
// a look at every value on its way 2.3 %.
// What was tried for the prompts: one thread that issues all products 531 us, one warp 314, a warp per half 263 (kept);
// two threads to a row 347; tiles of 128 with one place for scores 302; scores fetched a tile ahead 356; some exponentials
// by polynomial 265 to 270; weights against the old maximum without looking for the new one 291.
#include "paged_attn.cuh"
#include "paged_attn_tc.cuh"
#include "tcgen05.cuh"

namespace mak {
namespace {

constexpr int kTile = 64;       // tokens per step
constexpr int kHalf = 128;      // rows of a half
constexpr int kUnitRows = 256;  // rows of a unit
constexpr int kThreads = 512;
constexpr float kLazy = 8.f;    // log2 growth of a row's maximum that is tolerated
constexpr int kUnitCost = 8;    // a unit's beginning and end, in tiles
constexpr int kMinChunk = 8;    // steps of work that are worth another block
constexpr int kMaxGrid = 148;
static_assert(4 * kMaxGrid * 4 <= kPagedCounterBytes, "a counter for each half of the two units that a block may share");
constexpr int kMaxItems = 1 << 16;
constexpr int kHave = 16;       // tiles whose pages are remembered

// What the planning launch leaves: unit lengths added up over the row tiles, and whose they are.
struct Plan {
  int64_t base[kMaxItems + 1];  // work before row tile i, over all heads
  int32_t seq[kMaxItems];
  int32_t tile[kMaxItems];
};

// Rows of row tile `tile` of a sequence (numbers below the first sequence's come as negative ones) and what they see.
__device__ __forceinline__ int live_rows(const PagedParams& p, const PagedSeq& v, int tile) {
  return tile < 0 ? 0 : max(min(v.rows * p.group - tile * kUnitRows, kUnitRows), 0);
}
__device__ __forceinline__ Span span_of_rows(const PagedParams& p, const PagedSeq& v, int tile, int row_a, int row_b) {
  const int row0 = tile * kUnitRows;
  return span_of<kTile>(p, v, (row0 + row_a) / p.group, (row0 + row_b) / p.group);
}
__device__ __forceinline__ int unit_len(const PagedParams& p, const PagedSeq& v, int tile) {
  const int live = live_rows(p, v, tile);
  return live == 0 ? 0 : kUnitCost + max(span_of_rows(p, v, tile, 0, live - 1).tiles, 1);
}

// Row tiles of sequence s take the numbers floor(starts[s] * group / 256) + s and up, at least as many as it has; numbers
// before the first sequence's are nobody's.
__device__ __forceinline__ int64_t first_item(const PagedParams& p, int s) {
  const int64_t row = p.starts != nullptr ? max(__ldg(p.starts + s), 0) : s;
  return row * p.group / kUnitRows + s;
}

__global__ void __launch_bounds__(1024) paged_plan_kernel(const __grid_constant__ PagedParams p, Plan* plan, int items) {
  __shared__ int64_t sums[32];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (items + 1023) / 1024;
  const int i0 = min(tid * per, items), i1 = min(i0 + per, items);
  int seq = 0;
  if (i0 < i1) {
    int hi = p.num_seqs;  // the last sequence whose first number is at most i0
    while (hi - seq > 1) {
      const int mid = (seq + hi) >> 1;
      if (first_item(p, mid) <= i0)
        seq = mid;
      else
        hi = mid;
    }
  }
  int64_t mine = 0;
  for (int i = i0; i < i1; ++i) {
    while (seq + 1 < p.num_seqs && first_item(p, seq + 1) <= i) ++seq;
    const int tile = static_cast<int>(i - first_item(p, seq));
    plan->seq[i] = seq;
    plan->tile[i] = tile;
    mine += unit_len(p, paged_seq(p, seq), tile);
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int64_t v = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    sums[lane] = v;
  }
  __syncthreads();
  int64_t at = (warp ? sums[warp - 1] : 0) + incl - mine;
  for (int i = i0; i < i1; ++i) {
    plan->base[i] = at * p.nh;
    at += unit_len(p, paged_seq(p, plan->seq[i]), plan->tile[i]);
  }
  if (tid == 1023) plan->base[items] = sums[31] * p.nh;
}

// The run of a block, one (row tile, head) unit after another; every role walks it for itself.
struct Walk {
  int64_t w, w_end, w0;  // w0: where the current unit begins
  int item, head, seq, tile, live;
  PagedSeq v;
  Span s;
};
struct Unit {
  PagedSeq v;
  Span s;
  int seq, head, tile, live;
  int ta, tb, len;  // this block has tiles [ta, tb) of len, at least 1
  int n;            // of these, real ones
  int64_t wt;       // where the unit's tiles begin in all work
  bool solo;        // each half takes every other tile
};

__device__ __forceinline__ void look_up(const PagedParams& p, const Plan* plan, Walk& k) {
  k.seq = plan->seq[k.item];
  k.tile = plan->tile[k.item];
  k.v = paged_seq(p, k.seq);
  k.live = live_rows(p, k.v, k.tile);
  if (k.live > 0) k.s = span_of_rows(p, k.v, k.tile, 0, k.live - 1);
}

__device__ __forceinline__ bool next_unit(const PagedParams& p, const Plan* plan, Walk& k, Unit& u) {
  for (;;) {
    if (k.w >= k.w_end) return false;
    const int len = max(k.s.tiles, 1);
    u.ta = static_cast<int>(max(k.w - k.w0 - kUnitCost, static_cast<int64_t>(0)));
    u.tb = static_cast<int>(min(k.w_end - k.w0 - kUnitCost, static_cast<int64_t>(len)));
    u.len = len;
    u.seq = k.seq, u.head = k.head, u.tile = k.tile, u.live = k.live, u.v = k.v, u.s = k.s;
    u.wt = k.w0 + kUnitCost;
    u.n = k.s.tiles > 0 ? u.tb - u.ta : 0;
    u.solo = k.live <= kHalf;
    k.w0 += kUnitCost + len;
    k.w = k.w0;
    if (k.w < k.w_end && ++k.head == p.nh) {
      k.head = 0;
      do {
        ++k.item;
        look_up(p, plan, k);
      } while (k.live == 0);
    }
    if (u.tb > u.ta) return true;
  }
}

__device__ __forceinline__ void both_sync() { asm volatile("bar.sync 3, 256;" ::: "memory"); }
__device__ __forceinline__ void half_sync(int half) { asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory"); }

// The larger of the three, NaN where one is NaN.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <int HD>
struct TcSmem {
  static constexpr int kBytes = kTile * HD * 2;      // of a tile of K or V: HD / 64 pieces of [64][64], lines of 128 bytes swizzled
  static constexpr int kK = HD == 64 ? 8 : 5, kV = HD == 64 ? 8 : 5;  // tiles of K and of V
  alignas(1024) uint8_t q[2][kHalf * HD * 2];  // pieces of [128][64]
  alignas(1024) uint8_t k[kK][kBytes];
  alignas(1024) uint8_t v[kV][kBytes];
  alignas(8) uint64_t q_full[2], k_full[kK], k_empty[kK], v_full[kV], v_clean[kV], v_empty[kV], s_full[2][2], p_full[2][2], o_full[2][2], spare[2];
  Walk walk[10];  // of the halves' softmax, the loads, the cleaning warps, the issuing ones
  Unit unit[10];
  int more[10];
  uint32_t have[kHave];  // bit c: 16 tokens c of a tile have a page
  uint32_t tmem;
  int gave_up, last[2];
  int odd_seen;  // values that are no numbers were replaced
};

// Of dimensions d .. d + 16, those of `wanted`: the sum of the values that are no numbers over the tokens that row i of the
// unit sees, in this half's tiles, all of them or those where they were replaced.
template <bool BF16>
__device__ __noinline__ void odd_sum(const PagedParams& p, const Unit& u, int i, int d, int first, int step, bool all, uint32_t wanted, float* sum) {
  const RowView r = row_view(p, u.v, i);
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[e] = 0.f;
  for (int j = u.ta + first; j < u.ta + u.n && wanted != 0; j += step) {
    const int tok = tile_token<kTile>(u.s, j);
    if (!all && tile_whole<kTile>(u.s, tok)) continue;
    uint32_t bits = 0;  // of 32 tokens of a tree
    for (int t = tok; t < tok + kTile; ++t) {
      if (p.parents != nullptr && (t & 31) == 0) bits = tree_bits(p, u.v, i, t);
      const bool seen = p.parents != nullptr ? bits >> (t & 31) & 1 : t < r.hi && (t >= r.lo || t < p.sinks);
      if (!seen) continue;
      const int page = page_of(p, p.tables + u.seq * p.table_stride, t);
      if (page < 0) continue;
      const uint16_t* v = p.value + page * p.v_sb + (t & ((1 << p.bs_log2) - 1)) * p.v_st + u.head * p.v_sh + d;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (!(wanted >> e & 1)) continue;
        const float x = to_float<BF16>(v[e]);
        if (!(fabsf(x) < INFINITY)) sum[e] += x;
        if (sum[e] != sum[e]) wanted &= ~(1u << e);  // and stays so
      }
    }
  }
}

// A row whose scores are all numbers and whose results, in part [HD][128] where there is one, else in dst, have NaN among them:
// those are the sums of the values that are no numbers.
template <int HD, bool BF16>
__device__ __noinline__ void look_again(const PagedParams& p, const Unit& u, int i, int first, int step, float* part, uint16_t* dst) {
  for (int d = 0; d < HD; d += 16) {
    uint32_t none = 0;
    float sum[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float x = part != nullptr ? part[(d + e) * kHalf] : to_float<BF16>(dst[d + e]);
      none |= x != x ? 1u << e : 0u;
    }
    odd_sum<BF16>(p, u, i, d, first, step, true, none, sum);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if (!(none >> e & 1) || sum[e] == 0.f) continue;
      if (part != nullptr)
        part[(d + e) * kHalf] = sum[e];
      else
        dst[d + e] = static_cast<uint16_t>(pack_two<BF16>(sum[e], 0.f));
    }
  }
}

template <int HD, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    paged_tc_kernel(const __grid_constant__ PagedParams p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                    const Plan* plan, int items) {
  using Sm = TcSmem<HD>;
  constexpr float kLift = BF16 ? 0.f : 6.f;  // log2 factor that weights carry: those of float16 stay below 2^15
  constexpr int kBytes = Sm::kBytes, kK = Sm::kK, kV = Sm::kV;
  extern __shared__ __align__(1024) uint8_t raw[];
  Sm& sm = *reinterpret_cast<Sm*>(raw);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // the same for all lanes, as the compiler sees it
  pdl_wait();
  pdl_trigger();

  // ---- the run of this block ----------------------------------------------------
  Walk walk;
  const int64_t total = plan->base[items];
  int64_t chunk = (total + gridDim.x - 1) / gridDim.x;
  if (chunk < kMinChunk) chunk = kMinChunk;
  walk.w = blockIdx.x * chunk;
  walk.w_end = min(walk.w + chunk, total);
  if (walk.w >= walk.w_end) return;
  {
    int lo = 0, n = items;  // the last row tile that begins at or before w
    while (n > 1) {
      const int step = (n + 31) >> 5;
      const int at = lo + lane * step;
      const uint32_t votes = __ballot_sync(0xffffffffu, at < lo + n && plan->base[at] <= walk.w);
      const int k = 31 - __clz(votes);
      const int end = lo + n;
      lo += k * step;
      n = min(step, end - lo);
    }
    walk.item = lo;
    look_up(p, plan, walk);
    const int len = kUnitCost + max(walk.s.tiles, 1);
    const int64_t rel = walk.w - plan->base[lo];
    walk.head = static_cast<int>(rel / len);
    walk.w0 = plan->base[lo] + static_cast<int64_t>(walk.head) * len;
  }
  if (tid == 0) {
    sm.gave_up = 0;
    sm.odd_seen = 0;
    for (int i = 0; i < kK; ++i) mbar_init(&sm.k_full[i], 1), mbar_init(&sm.k_empty[i], 2);
    for (int i = 0; i < kV; ++i) mbar_init(&sm.v_full[i], 1), mbar_init(&sm.v_clean[i], 4), mbar_init(&sm.v_empty[i], 2);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.q_full[i], 4);
      mbar_init(&sm.spare[i], 1);
      for (int b = 0; b < 2; ++b) mbar_init(&sm.s_full[i][b], 1), mbar_init(&sm.p_full[i][b], 4), mbar_init(&sm.o_full[i][b], 1);
    }
    mbar_init_fence();
  }
  if (warp == 10) tmem_alloc<512>(&sm.tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  volatile int* gave_up = &sm.gave_up;

  if (warp < 8) {
    regs_up<184>();  // with 72 below: what the block was launched with
    // ---- softmax ----------------------------------------------------------------
    const int half = warp >> 2;
    const int r = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + half * 128;
    const uint32_t o_at = tmem + lanes + 256 + half * HD;
    const float scale = fmaxf(fabsf(p.scale_log2), 1e-37f);  // not 0: masked scores are -inf
    const uint32_t sign = p.scale_log2 < 0.f ? 0x80008000u : 0u;
    uint32_t before = 0, mine = 0, ends = 0, ends2 = 0;  // tiles of all units and of this half, units with one and with two of these
    bool ok = true;
    if (r == 0) sm.walk[half] = walk;
    const Unit& u = sm.unit[half];
    for (;;) {
      if (r == 0) sm.more[half] = next_unit(p, plan, sm.walk[half], sm.unit[half]);
      half_sync(half);
      if (!sm.more[half]) break;
      const bool solo = u.solo;
      const int row_in = solo ? r : half * kHalf + r;  // of the unit
      const bool active = solo || half * kHalf < u.live;
      const bool on = row_in < u.live;
      const int row = u.tile * kUnitRows + (on ? row_in : 0);
      const int who = row / p.group, head = u.head * p.group + row - who * p.group;
      const int first = solo ? half : 0, step = solo ? 2 : 1;
      const int n = active && u.n > first ? (u.n - first + step - 1) / step : 0;  // tiles of this half
      float m = -INFINITY, l = 0.f;
      if (n > 0) {
        {  // this row of q
          const uint4* src = reinterpret_cast<const uint4*>(p.q + (static_cast<int64_t>(u.v.first) + who) * p.q_sr + head * p.q_sh);
          uint4 x[HD / 8];
#pragma unroll
          for (int e = 0; e < HD / 8; ++e) x[e] = on ? __ldg(src + e) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < HD / 8; ++e)
            *reinterpret_cast<uint4*>(sm.q[half] + (e >> 3) * 16384 + r * 128 + (((e & 7) ^ (r & 7)) << 4)) =
                make_uint4(x[e].x ^ sign, x[e].y ^ sign, x[e].z ^ sign, x[e].w ^ sign);
          fence_async_shared();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.q_full[half]);
        }
        const int last_row = solo ? u.live - 1 : min(u.live, half * kHalf + kHalf) - 1;
        const Span s = span_of_rows(p, u.v, u.tile, solo ? 0 : half * kHalf, last_row);  // of this half's rows
        const RowView see = row_view(p, u.v, who);
        for (int t = 0; t < n; ++t, ++mine) {
          const uint32_t place_at = s_at + (mine & 1) * 64;  // of the scores, and of the weights over them
          ok = ok && wait_warp(&sm.s_full[half][mine & 1], (mine >> 1) & 1, gave_up);
          tc_fence_after();
          const int j = first + t * step;
          const int tok = tile_token<kTile>(u.s, u.ta + j);
          const uint32_t have = sm.have[(before + j) % kHave];
          const bool whole = tile_whole<kTile>(s, tok) && have == 0xfu;
          uint32_t x[2][32];
          tmem_ld(place_at, x[0]);
          tmem_ld(place_at + 32, x[1]);
          tmem_wait(x[0]);
          tmem_wait(x[1]);
          if (!whole) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int t0 = tok + c * 32;
              uint32_t bits;
              if (p.parents != nullptr) {
                bits = tree_bits(p, u.v, who, t0);
              } else {
                auto below = [](int k) { return k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1u; };
                bits = below(see.hi - t0) & (~below(see.lo - t0) | below(p.sinks - t0));
              }
              bits &= ((have >> (2 * c)) & 1 ? 0x0000ffffu : 0u) | ((have >> (2 * c + 1)) & 1 ? 0xffff0000u : 0u);
#pragma unroll
              for (int e = 0; e < 32; ++e) x[c][e] = bits >> e & 1 ? x[c][e] : 0xff800000u;
            }
          }
          float tops[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t* at = &x[c >> 1][(c & 1) * 16];
            tops[c] = max3(__uint_as_float(at[0]), __uint_as_float(at[1]), __uint_as_float(at[15]));
#pragma unroll
            for (int e = 2; e < 14; e += 2) tops[c] = max3(tops[c], __uint_as_float(at[e]), __uint_as_float(at[e + 1]));
            tops[c] = max3(tops[c], __uint_as_float(at[14]), __uint_as_float(at[14]));
          }
          const float top = max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[3]) * scale;
          if (!(top < INFINITY)) l = __uint_as_float(0x7fffffffu);  // a score that is no number, or infinite
          const bool grow = top > m + kLazy || (m == -INFINITY && top > m);
          if (__any_sync(0xffffffffu, grow)) {
            const float mn = fmaxf(m, top);
            const float keep = mn == m ? 1.f : shrink(m - mn);
            m = mn;
            l *= keep;
            if (t > 0) {
              // The last weights' product: the next scores come after it.
              ok = ok && (t + 1 < n ? wait_warp(&sm.s_full[half][(mine + 1) & 1], ((mine + 1) >> 1) & 1, gave_up)
                                    : wait_warp(&sm.o_full[half][1], ends2 & 1, gave_up));
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < HD / 16; ++c) {
                uint32_t o[16];
                tmem_ld(o_at + c * 16, o);
                tmem_wait(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                tmem_st(o_at + c * 16, o);
              }
            }
          }
          const float ref = m > -INFINITY && m < INFINITY ? m - kLift : 0.f;
          float2 sum[2] = {both(0.f), both(0.f)};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t y[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float2 w = fma2(make_float2(__uint_as_float(x[c][2 * e]), __uint_as_float(x[c][2 * e + 1])), both(scale), both(-ref));
              w.x = exp2_near(w.x);
              w.y = exp2_near(w.y);
              sum[e & 1] = add2(sum[e & 1], w);
              y[e] = pack_two<BF16>(w.x, w.y);
            }
            tmem_st(place_at + c * 16, y);
          }
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_full[half][mine & 1]);
          sum[0] = add2(sum[0], sum[1]);
          l += sum[0].x + sum[0].y;
        }
        ok = ok && wait_warp(&sm.o_full[half][0], ends & 1, gave_up);
        tc_fence_after();
        ++ends;
        if (n > 1) ++ends2;
      }
      before += u.n;
      if (!ok) l = __uint_as_float(0x7fffffffu);  // a block that gave up leaves NaN, not stale memory

      // ---- this half's share of the unit -------------------------------------------
      auto place = [&](int row, uint16_t*& dst, float*& lse) {  // of a row's result
        const int64_t i = u.v.first + row / p.group, h = static_cast<int64_t>(u.head) * p.group + row % p.group;
        dst = static_cast<uint16_t*>(p.out) + i * p.o_sr + h * p.o_sh;
        lse = p.lse == nullptr ? nullptr : p.lse + i * p.nh * p.group + h;
      };
      auto put = [&](uint16_t* dst, const float(&o)[16], float inv) {
        uint32_t y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = pack_two<BF16>(o[2 * e] * inv, o[2 * e + 1] * inv);
        if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
          reinterpret_cast<uint4*>(dst)[0] = make_uint4(y[0], y[1], y[2], y[3]);
          reinterpret_cast<uint4*>(dst)[1] = make_uint4(y[4], y[5], y[6], y[7]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            dst[2 * e] = static_cast<uint16_t>(y[e]);
            dst[2 * e + 1] = static_cast<uint16_t>(y[e] >> 16);
          }
        }
      };
      auto put_lse = [&](float* lse, float mx, float sum) {
        if (lse != nullptr) *lse = sum > 0.f || sum != sum ? (mx - kLift + log2f(sum)) * 0.69314718055994531f : -INFINITY;
      };
      const bool cut = u.ta > 0 || u.tb < u.len, split = cut || solo;
      constexpr int kFloats = kHalf * (HD + 2);  // of one partial sum: [HD][128], maxima, sums
      auto piece = [&](int64_t block, int which) {
        return p.partial + ((2 * block + (u.wt > block * chunk ? 1 : 0)) * 2 + which) * kFloats;
      };
      float* part = piece(blockIdx.x, half);
      if (active) {
        uint16_t* dst = nullptr;
        float* lse = nullptr;
        if (on) place(row, dst, lse);
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        const bool odd_seen = n > 0 && *static_cast<volatile int*>(&sm.odd_seen);
        float most = 0.f;  // NaN where a result is none
#pragma unroll 1
        for (int d = 0; d < HD; d += 16) {
          float o[16];
          if (n > 0) {
            uint32_t x[16];
            tmem_ld(o_at + d, x);
            tmem_wait(x);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __uint_as_float(x[e]);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0.f;
          }
          if (odd_seen && on) {
            float bad[16];
            odd_sum<BF16>(p, u, who, d, first, step, false, 0xffffu, bad);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] += bad[e];
          }
          if (split) {
            if (on) {
#pragma unroll
              for (int e = 0; e < 16; ++e) part[(d + e) * kHalf + r] = o[e];
            }
          } else if (on) {
            put(dst + d, o, inv);
          }
          const float a = max3(o[0], o[1], o[2]), b = max3(o[3], o[4], o[5]), c = max3(o[6], o[7], o[8]), e = max3(o[9], o[10], o[11]);
          most = max3(max3(a, b, c), max3(e, o[12], o[13]), max3(most, o[14], o[15]));
        }
        // infinite values too light for 16 bits
        if (on && most != most && l == l) look_again<HD, BF16>(p, u, who, first, step, split ? part + r : nullptr, dst);
        if (on) {
          if (split) {
            part[HD * kHalf + r] = m;
            part[HD * kHalf + kHalf + r] = l;
          } else {
            put_lse(lse, m, l);
          }
        }
      }
      tc_fence_before();
      if (split && active) {
        const int64_t first_block = u.wt / chunk, last_block = (u.wt + u.len - 1) / chunk;
        const int64_t slot0 = (2 * first_block + (u.wt > first_block * chunk ? 1 : 0)) * 2 + (solo ? 0 : half);
        // A solo unit is both halves': the first of them joins it when both have written, and no half writes its next
        // piece, which may have the same place, before that is done.
        if (solo)
          both_sync();
        else
          half_sync(half);
        if (r == 0) {  // releases what the barrier has gathered
          bool last = !solo || half == 0;
          if (last && cut) {
            int ticket;
            asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(ticket) : "l"(p.counters + slot0) : "memory");
            last = ticket == last_block - first_block;
            if (last) p.counters[slot0] = 0;
          }
          sm.last[half] = last;
        }
        half_sync(half);
        if (sm.last[half]) {
          // Few rows leave several threads for each, which share its columns.  Four pieces' loads at a time.
          const int rows = solo ? u.live : min(u.live - half * kHalf, kHalf);
          const int span = rows > 64 ? 128 : rows > 32 ? 64 : 32, mine_row = r & (span - 1), cols = HD * span / kHalf;
          const int pieces = static_cast<int>(last_block - first_block + 1) * (solo ? 2 : 1);
          if (mine_row < rows) {
            auto from = [&](int i) {
              return (solo ? piece(first_block + (i >> 1), i & 1) : piece(first_block + i, half)) + mine_row;
            };
            float mx = -INFINITY, sum = 0.f;
#pragma unroll 4
            for (int i = 0; i < pieces; ++i) {
              const float pm = __ldcg(from(i) + HD * kHalf), pl = __ldcg(from(i) + HD * kHalf + kHalf);
              const float mn = fmaxf(mx, pm), ms = mn == -INFINITY ? 0.f : mn;
              sum = sum * exp2_near(mx - ms) + pl * exp2_near(pm - ms);
              mx = mn;
            }
            const float ms = mx == -INFINITY ? 0.f : mx, inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
            uint16_t* dst;
            float* lse;
            place(u.tile * kUnitRows + (solo ? 0 : half * kHalf) + mine_row, dst, lse);
#pragma unroll 1
            for (int d = r / span * cols, end = d + cols; d < end; d += 16) {
              float o[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = 0.f;
#pragma unroll 1
              for (int i = 0; i < pieces; i += 4) {
                float x[4][16], k[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                  const float* src = from(min(i + z, pieces - 1));
                  k[z] = __ldcg(src + HD * kHalf);
#pragma unroll
                  for (int e = 0; e < 16; ++e) x[z][e] = __ldcg(src + (d + e) * kHalf);
                }
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                  k[z] = shrink(k[z] - ms);
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[e] = i + z < pieces ? fmaf(x[z][e], k[z], o[e]) : o[e];
                }
              }
              put(dst + d, o, inv);
            }
            if (r < span) put_lse(lse, mx, sum);
          }
        }
        if (solo) both_sync();
      }
      half_sync(half);  // the unit is read
    }
  } else {
    regs_down<72>();
    if (warp < 10) {
      // ---- loads ----------------------------------------------------------------------
      constexpr int kPieces = HD / 64, kStages = kK;
      static_assert(kK == kV, "one loop for both");
      const bool is_v = warp == 9;
      const int role = warp - 6;
      const int bs = 1 << p.bs_log2, box = min(bs, kTile), pages = kTile / box;
      uint64_t *const full = is_v ? sm.v_full : sm.k_full, *const empty = is_v ? sm.v_empty : sm.k_empty;
      const uint32_t ring = smem_addr(is_v ? sm.v : sm.k);
      const void* map = is_v ? &v_map : &k_map;
      uint32_t g = 0, stage = 0, phase = 1;  // tiles so far
      bool ok = true;
      if (lane == 0) sm.walk[role] = walk;
      const Unit& u = sm.unit[role];
      while (ok) {
        __syncwarp();
        if (lane == 0) sm.more[role] = next_unit(p, plan, sm.walk[role], sm.unit[role]);
        __syncwarp();
        if (!__shfl_sync(0xffffffffu, sm.more[role], 0)) break;
        const int n = __shfl_sync(0xffffffffu, u.n, 0), head = __shfl_sync(0xffffffffu, u.head, 0);
        const int ta = u.ta, room = u.v.room;
        const Span s = u.s;
        const int32_t* table = p.tables + u.seq * p.table_stride;
        auto find = [&](int j) {  // id of page `lane` of tile j; looked at when it is needed, a tile later
          const int tok = tile_token<kTile>(s, ta + j) + lane * box;
          return j < n && lane < pages && tok < room ? __ldg(table + (tok >> p.bs_log2)) : -1;
        };
        int next = find(0);
        for (int j = 0; j < n; ++j, ++g) {
          const int page = next >= 0 && next < p.num_blocks ? next : -1;
          next = find(j + 1);
          ok = wait_warp(&empty[stage], phase, gave_up);
          if (!ok) break;
          if (!is_v) {
            const uint32_t votes = __ballot_sync(0xffffffffu, page >= 0);
            uint32_t have = 0;  // in sixteens of tokens
            for (int c = 0; c < kTile / 16; ++c) have |= (votes >> (c * 16 / box) & 1) << c;
            if (lane == 0) sm.have[g % kHave] = have;
            __syncwarp();
          }
          int id[kTile / 16];
#pragma unroll
          for (int i = 0; i < kTile / 16; ++i) id[i] = __shfl_sync(0xffffffffu, page, i);
          const int inside = tile_token<kTile>(s, ta + j) & (bs - 1);  // of a page that holds several tiles
          if (elect_one()) {
            mbar_arrive_expect(&full[stage], kBytes);
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i) {
              if (i >= pages) break;
              // a block that there is not: the load fills zeros
#pragma unroll
              for (int c = 0; c < kPieces; ++c)
                box_load(ring + stage * kBytes + c * (kTile * 128) + i * box * 128, map, c * 64, head, inside, id[i], &full[stage]);
            }
          }
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
      }
      if (!ok) {  // the copies in flight end before the block does
        for (uint32_t t = g > kStages ? g - kStages : 0; t < g; ++t)
          for (uint32_t i = 0; i < kWaitLimit && !mbar_try(&full[t % kStages], (t / kStages) & 1); ++i) {
          }
      }
    } else if (warp >= 12) {
      // ---- values that are no numbers ---------------------------------------------------
      const int mine = warp - 12, role = warp - 8;
      uint32_t g = 0;
      bool ok = true;
      if (lane == 0) sm.walk[role] = walk;
      const Unit& u = sm.unit[role];
      while (ok) {
        __syncwarp();
        if (lane == 0) sm.more[role] = next_unit(p, plan, sm.walk[role], sm.unit[role]);
        __syncwarp();
        if (!sm.more[role]) break;
        const int n = u.n;
        for (int j = 0; j < n; ++j, ++g) {
          const uint32_t vs = g % kV;
          ok = wait_warp(&sm.v_full[vs], (g / kV) & 1, gave_up);
          if (!ok) break;
          if (!tile_whole<kTile>(u.s, tile_token<kTile>(u.s, u.ta + j))) {
            uint4* v = reinterpret_cast<uint4*>(sm.v[vs]) + mine * (kBytes / 64);
            bool odd = false;
#pragma unroll 4
            for (int i = lane; i < kBytes / 64; i += 32) {
              uint4 w = v[i];
              if (odd_two<BF16>(w.x) || odd_two<BF16>(w.y) || odd_two<BF16>(w.z) || odd_two<BF16>(w.w)) {
                odd = true;
                auto fine = [](uint32_t a) {
                  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
                  return a & (((a & e) == e ? 0u : 0xffffu) | ((a & (e << 16)) == (e << 16) ? 0u : 0xffff0000u));
                };
                v[i] = make_uint4(fine(w.x), fine(w.y), fine(w.z), fine(w.w));
              }
            }
            if (odd) *static_cast<volatile int*>(&sm.odd_seen) = 1;
          }
          fence_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.v_clean[vs]);
        }
      }
    } else {
      // ---- the tensor cores -------------------------------------------------------
      // The whole warp walks, so that all addresses are known to be the same for its lanes; one of them issues.
      constexpr int kFormat = BF16 ? 1 : 0;
      constexpr uint32_t kQk = instr_desc(kTile, 1, kFormat, false, false), kPv = instr_desc(HD, 1, kFormat, false, true);
      constexpr uint32_t kBuffer = kBytes / 16, kRows = kHalf * HD * 2 / 16;
      const int half = warp - 10, role = 8 + half;
      // Descriptors differ in their addresses alone, in units of 16 bytes: no carry leaves that field.
      const uint64_t q_desc = smem_desc(smem_addr(sm.q), 16, 1024, 7) + half * kRows, k_desc = smem_desc(smem_addr(sm.k), 16, 1024, 7);
      const uint64_t v_desc = smem_desc(smem_addr(sm.v), kTile * 128, 1024, 7);
      const uint32_t s_at = tmem + half * 128, o_at = tmem + 256 + half * HD;
      uint64_t *const s_full = sm.s_full[half], *const p_full = sm.p_full[half], *const o_full = sm.o_full[half];
      struct Ring {
        uint64_t *full, *empty;
        uint32_t at, phase;
      } kr = {sm.k_full, sm.k_empty, 0, 0}, vr = {sm.v_clean, sm.v_empty, 0, 0};
      uint32_t made = 0, done = 0, begins = 0;  // scores made and weights used so far, units
      bool ok = true;
      if (lane == 0) sm.walk[role] = walk;
      static_assert(kK == kV, "one size for both");
      auto move = [](Ring& r) {
        if (++r.at == kK) r.at = 0, r.phase ^= 1;
      };
      auto there = [&](const Ring& r) { return wait_warp(&r.full[r.at], r.phase, gave_up); };
      // A tile of the other half's alone: both halves wait for every tile and both give every place back.  One that
      // skipped a wait could take an older phase for the one it wants.
      auto pass = [&](Ring& r) {
        ok = ok && there(r);
        if (ok && lane == 0) mbar_arrive(&r.empty[r.at]);
        move(r);
      };
      for (;;) {
        __syncwarp();
        if (lane == 0) sm.more[role] = next_unit(p, plan, sm.walk[role], sm.unit[role]);
        __syncwarp();
        if (!__shfl_sync(0xffffffffu, sm.more[role], 0)) break;
        const int all = __shfl_sync(0xffffffffu, sm.unit[role].n, 0);
        const bool solo = __shfl_sync(0xffffffffu, static_cast<int>(sm.unit[role].solo), 0);
        const int n = !solo ? all : (all + 1 - half) / 2;  // tiles of this half, every other one of a solo unit
        const int rounds = solo ? (all + 1) / 2 : all;
        if (n > 0) {
          ok = wait_warp(&sm.q_full[half], begins++ & 1, gave_up);
          tc_fence_after();
        }
        // The scores of two tiles, then always the values of one and the scores of the next but one.
        for (int t = 0; t < (rounds > 0 ? rounds + 2 : 0) && ok; ++t) {
          if (t >= 2) {
            if (solo && half == 1) pass(vr);
            if (t - 2 < n) {
              const uint32_t at = done & 1;
              ok = ok && there(vr) && wait_warp(&p_full[at], (done >> 1) & 1, gave_up);
              if (!ok) break;
              tc_fence_after();
              if (elect_one()) {
                const uint64_t vd = v_desc + vr.at * kBuffer;
                steps<kTile / 16>([&](auto i) {
                  constexpr int ks = decltype(i)::value;
                  mma_ts_f16<ks * 8, ks * 128>(o_at, s_at + at * 64, vd, kPv, t > 2 || ks > 0);
                });
                if (t >= n) tc_commit(&o_full[t == n ? 1 : 0]);  // of the last two tiles
                tc_commit(&vr.empty[vr.at]);
              }
              ++done;
              move(vr);
            }
            if (solo && half == 0 && 2 * (t - 2) + 1 < all) pass(vr);
          }
          if (t < rounds) {
            if (solo && half == 1) pass(kr);
            if (t < n) {
              const uint32_t at = made & 1;
              ok = ok && there(kr);
              if (!ok) break;
              if (elect_one()) {
                const uint64_t kd = k_desc + kr.at * kBuffer;
                steps<HD / 16>([&](auto i) {
                  constexpr int ks = decltype(i)::value;
                  mma_ss_f16<(ks >> 2) * (kHalf * 8) + (ks & 3) * 2, (ks >> 2) * (kTile * 8) + (ks & 3) * 2>(s_at + at * 64, q_desc, kd, kQk, ks > 0);
                });
                tc_commit(&s_full[at]);
                tc_commit(&kr.empty[kr.at]);
              }
              ++made;
              move(kr);
            }
            if (solo && half == 0 && 2 * t + 1 < all) pass(kr);
          }
        }
        if (!ok) break;
      }
      if (!ok) {  // let what was issued end before the TMEM is given back
        if (elect_one()) tc_commit(&sm.spare[half]);
        __syncwarp();
        for (uint32_t i = 0; i < kWaitLimit && !mbar_try(&sm.spare[half], 0); ++i) {
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 10) {
    __syncwarp();
    tc_fence_after();
    tmem_free<512>(tmem);
  }
}

// Row tiles of all sequences, at most.
int64_t row_tiles(const PagedParams& p) { return static_cast<int64_t>(p.num_rows) * p.group / kUnitRows + p.num_seqs; }

template <int HD, bool BF16>
int launch(const PagedParams& p, const char* name, const CUtensorMap& k, const CUtensorMap& v, Plan* plan, cudaStream_t st) {
  constexpr int kBytes = sizeof(TcSmem<HD>);
  static_assert(kBytes <= 227 * 1024, "shared memory of a block");
  const auto kernel = paged_tc_kernel<HD, BF16>;
  static bool ready[kPagedDevices] = {};
  if (int rc = paged_prepare(name, kernel, kBytes, ready)) return rc;
  const int items = static_cast<int>(row_tiles(p));
  if (int rc = launch_pdl(name, paged_plan_kernel, dim3(1), dim3(1024), 0, st, p, plan, items)) return rc;
  const int sms = sm_count();
  return launch_pdl(name, kernel, dim3(sms < kMaxGrid ? sms : kMaxGrid), dim3(kThreads), kBytes, st, p, k, v, static_cast<const Plan*>(plan), items);
}

}  // namespace

int64_t paged_tc_partial_bytes() { return static_cast<int64_t>(4 * kMaxGrid) * kHalf * (128 + 2) * 4; }
int64_t paged_tc_plan_bytes() { return sizeof(Plan); }
bool paged_tc_fits(const PagedParams& p) { return row_tiles(p) <= kMaxItems; }

bool paged_encode(CUtensorMap* map, const void* base, int rank, const int64_t* dims, const int64_t* strides, const uint32_t* box, bool bf16) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  if (encode == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess || fn == nullptr) {
      (void)cudaGetLastError();
      return false;
    }
    encode = reinterpret_cast<Encode>(fn);
  }
  cuuint64_t size[4], step[3];
  cuuint32_t part[4], each[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) size[i] = static_cast<cuuint64_t>(dims[i]), part[i] = box[i];
  for (int i = 0; i + 1 < rank; ++i) step[i] = static_cast<cuuint64_t>(strides[i]);
  const CUresult rc = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, static_cast<cuuint32_t>(rank),
                             const_cast<void*>(base), size, step, part, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS;
}

bool paged_map(CUtensorMap* map, const uint16_t* base, int64_t sb, int64_t st, int64_t sh, int64_t num_blocks, int nh, int hd, int bs, bool bf16,
               int tokens, const void* none) {
  // a pool without pages is never loaded from, but a map needs a size and an address
  const int64_t dims[4] = {hd, nh, bs, num_blocks > 0 ? num_blocks : 1}, strides[3] = {sh * 2, st * 2, sb * 2};
  const uint32_t box[4] = {64, 1, static_cast<uint32_t>(tokens), 1};
  return paged_encode(map, num_blocks > 0 ? static_cast<const void*>(base) : none, 4, dims, strides, box, bf16);
}

int paged_tc_box(int bs) { return bs < kTile ? bs : kTile; }

int launch_paged_tc(const PagedParams& p, int head_dim, bool bf16, const char* name, const CUtensorMap& k, const CUtensorMap& v, void* plan,
                    cudaStream_t st) {
  Plan* at = static_cast<Plan*>(plan);
  if (head_dim == 64) return bf16 ? launch<64, true>(p, name, k, v, at, st) : launch<64, false>(p, name, k, v, at, st);
  return bf16 ? launch<128, true>(p, name, k, v, at, st) : launch<128, false>(p, name, k, v, at, st);
}

}  // namespace mak
