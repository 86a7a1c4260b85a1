// Attention over a block-scaled 8-bit cache for many rows per sequence (prompts):
// the products on the tcgen05 tensor cores, everything else hidden behind them.
//
// Mathematics as in block_attn.cu: S = q . codes, here with q and codes in f16 (codes exactly, a bf16
// row of q by a power of two).  The V scale b of a token goes into its exponent: with m' the running
// maximum of S' + log2 b, the weight 2^(S' + log2 b - m') multiplies the code and, times 1 / b, joins the
// sum, which is taken in 32 bits before the weight is rounded once to f16: the tensor cores take 16-bit
// weights next to f16 codes, and wider ones at half the rate or less.  A weight is off by 2^-12 of
// itself at most: an f16 result's error grows by a fifth to a third (2.1e-4 to 2.5e-4 of its norm), a bf16
// result's rounding hides it.  The maximum is only moved when it grew by more than 2^8 or so: weights then
// stay below 2^15 (they carry a factor 2^6), the result is the same, and the accumulators in TMEM are
// rarely rescaled.
//
// Numbers that are none.  What a row does not see reaches none of its sums, whatever it holds: its weights
// there are 0, and E4M3 codes of V that are NaN become 0 where not every row of a unit sees their tokens;
// the rows that do see them get NaN with their results (nan_dims).  In E4M3 that costs 0.7 % of a prompt
// chunk's time, 2.6 % with a window of 512, nothing in int8.
//
// A block takes 256 rows of one cache head (heads of the group next to one another, so a K / V tile
// serves all of them) as two tiles of 128, and walks the cache in tiles of 128 tokens.  Roles:
//   warps 0-3, 4-7     softmax of row tile 0 / 1, a thread per row (TMEM lane)
//   warps 8-11, 12-15  load codes of K / V, convert to f16, store to shared memory
//   warp 16            one thread issues all tcgen05.mma
// While one row tile's scores are exponentiated the tensor cores work for the other.
//
// Work.  All (row tile, head) units laid end to end, each as long as the tiles it sees, are cut into
// equal runs, one per block, so causal masks and ragged lengths leave no block idle; a small launch
// before this one adds up the lengths.  A unit cut by that leaves partial sums, and the last block to
// arrive joins them.
//
// Layout.  The cache tile is [head_dim][tokens], tokens contiguous.  Converted to f16 it is stored as
// it is, in 128-byte swizzled lines of 64 tokens: K is read from there as an MN-major operand and V as
// a K-major one, so no element is ever transposed.  Scores and weights share TMEM columns: the product
// with V of a tile is issued before the next scores of the same rows overwrite them.
//
// Measured.  Two prompts' chunks of 1500 to 2048 rows against 5000 to 8192 tokens, 32 query heads on 8 cache heads of
// 128, int8, bf16 q: 442 to 461 us on several GPUs, 803 to 838 TFLOP/s of the 1678 that a bf16 matrix product reaches;
// in E4M3 438 us where int8 takes 448; heads of 64 (f16 q, blocks of 64) 384 us, in E4M3 373.  What bounds it is the chain from scores to scores of a row tile: some 3900 cycles
// of softmax, 1100 of its two products, 350 of handing over, against 2050 that the tensor cores need for both row
// tiles.  Four instructions for each score and 2.3 for each pair of codes converted keep the issue slots 0.44 busy, the
// exponential unit 0.39, and 128 rows take that long because each warp waits for itself; without any softmax or
// conversion the kernel would take 359 us.  Tried and slower at the time: 16 softmax warps (573 against 547 us), scores
// of 64 tokens at a time in two places (775 against 481), an issuing thread for each row tile (554 against 481), codes
// staged by bulk copies (563 against 547), the maximum looked for before the weights (481 against 453).
#include <utility>

#include "block_attn.cuh"
#include "tcgen05.cuh"

namespace mak {
namespace {

constexpr int kTile = 128;      // tokens per step
constexpr int kUnitRows = 256;  // rows of a unit
constexpr int kThreads = 640;
constexpr float kLazy = 8.f;    // log2 growth of a row's maximum that is tolerated
constexpr float kLift = 6.f;    // log2 factor that weights carry
// The sum of the weights carries 2^(kLift - kSpare): divided by the smallest scales, 2^-109 as the writer makes them, its
// terms come to 2^114 and more.  Smaller scales count as kLeast in the maximum.
constexpr int kSpare = 12;
constexpr float kLeast = -110.f;  // log2
constexpr float kSumLimit = 32768.f;  // of 16 weights, below which none of them is near f16's largest
// A unit's beginning and end, in tiles.  The prompts below with 2, 3, 4, 5: 448, 444, 439, 440 us.
constexpr int kUnitCost = 4;
// Steps of work that are worth another block.  With 2, 4, 6, 8: one prompt of 64 rows on 4096 tokens, one cache head:
// 54, 43, 48, 52 us; three of 60 rows on 400, 8 cache heads: 35, 34, 45, 48 us.
constexpr int kMinChunk = 4;
constexpr int kMaxGrid = 148;
constexpr int kMaxItems = 1 << 16;

// What the planning launch leaves: unit lengths added up over the row tiles, and whose they are.
struct Plan {
  int64_t base[kMaxItems + 1];  // work before row tile i, over all heads
  int32_t seq[kMaxItems];
  int32_t tile[kMaxItems];
};

// Tiles of row tile `tile` of a sequence (0: there is no such row tile) and the tokens they lie in.  Numbers below the
// first sequence's, whose rows need not begin at 0, come as negative ones.
struct Span {
  int live, any_lo, any_hi, all_lo, all_hi, t0, tiles;  // tokens that some / all rows see
};
__device__ __forceinline__ Span span_of(const BlockAttnParams& p, const SeqView& v, int tile) {
  Span s;
  const int64_t left = static_cast<int64_t>(v.rows) * p.group - static_cast<int64_t>(tile) * kUnitRows;
  s.live = tile < 0 || left <= 0 ? 0 : left < kUnitRows ? static_cast<int>(left) : kUnitRows;
  s.any_lo = s.any_hi = s.all_lo = s.all_hi = s.t0 = s.tiles = 0;
  if (s.live == 0) return s;
  const int64_t row0 = static_cast<int64_t>(tile) * kUnitRows;
  row_range(p, v, static_cast<int>(row0 / p.group), &s.any_lo, &s.all_hi);
  row_range(p, v, static_cast<int>((row0 + s.live - 1) / p.group), &s.all_lo, &s.any_hi);
  if (s.any_hi > s.any_lo) {
    s.t0 = s.any_lo / kTile;
    s.tiles = (s.any_hi + kTile - 1) / kTile - s.t0;
  }
  return s;
}
__device__ __forceinline__ int unit_len(const Span& s) { return s.live == 0 ? 0 : kUnitCost + (s.tiles > 0 ? s.tiles : 1); }

// Row tiles of sequence s take the numbers floor(starts[s] * group / 256) + s and up, at least as many
// as it has; numbers before the first sequence's are nobody's.
__device__ __forceinline__ int64_t first_item(const BlockAttnParams& p, int s) {
  const int64_t row = p.starts != nullptr ? max(__ldg(p.starts + s), 0) : s;
  return row * p.group / kUnitRows + s;
}

__global__ void __launch_bounds__(1024) block_attn_plan_kernel(const __grid_constant__ BlockAttnParams p, Plan* plan, int items) {
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
  const int seq0 = seq;
  int64_t mine = 0;
  for (int i = i0; i < i1; ++i) {
    while (seq + 1 < p.num_seqs && first_item(p, seq + 1) <= i) ++seq;
    const int tile = static_cast<int>(i - first_item(p, seq));
    plan->seq[i] = seq;
    plan->tile[i] = tile;
    mine += unit_len(span_of(p, seq_view(p, seq), tile));
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
  seq = seq0;
  for (int i = i0; i < i1; ++i) {
    plan->base[i] = at * p.nh;
    at += unit_len(span_of(p, seq_view(p, plan->seq[i]), plan->tile[i]));
  }
  if (tid == 1023) plan->base[items] = sums[31] * p.nh;
}

// The runs of a block, one (row tile, head) unit after another; every warp walks them for itself.
struct Walk {
  int64_t w, w_end, w0;  // w0: where the current unit begins
  int item, head, seq, tile;
  SeqView v;
  Span span;
};
struct Unit {
  int seq, head, tile, live, ta, tb, any_lo, any_hi, all_lo, all_hi, t_first, n;  // this block has tiles [ta, tb), n of them real, from t_first on
  int64_t w_tiles;
  int len;  // tiles of the whole unit, at least 1
  SeqView v;
};

template <int HD>
struct TcSmem {
  alignas(1024) uint8_t q[2][HD * 256];  // 128 rows: HD / 64 pieces of [128][64]
  alignas(1024) uint8_t k[2][HD * 256];  // 128 tokens: 2 pieces of [HD][64]
  alignas(1024) uint8_t v[2][HD * 256];
  alignas(16) float kfac[4][8], vfac[4][8];  // per 16 tokens of a tile: the scales,
  alignas(16) float vlog[4][8], vinv[4][8];  // log2 of V's and 2^-kSpare over V's
  uint32_t have[4], plain[4];                // bit c: piece c has a block; its scales are positive, finite and not below 2^kLeast.  0-3 in byte 0, 4-7 in byte 1
  alignas(8) uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], spare;
  // Walks and units of the softmax warps, the eight loading warps and the issuing thread: here, since their
  // registers are needed for scores and codes.
  Walk walk[10];
  Unit unit[10];
  int more[10];
  uint32_t tmem;
  int gave_up, last;
  int nan_seen;  // E4M3: this block replaced a NaN
};

// E4M3: the dimensions d .. d + 16, one bit each, whose values are NaN at a token that row i of the unit sees, in the
// pieces where the loading warps replaced NaN: those that not every row of the unit sees whole.
__device__ __forceinline__ uint32_t nan_dims(const BlockAttnParams& p, const Unit& u, uint32_t i, int d) {
  int lo, hi;
  row_range(p, u.v, i, &lo, &hi);
  lo = max(lo, u.t_first * kTile);
  hi = min(hi, (u.t_first + u.n) * kTile);
  const int bs = 1 << p.bs_log2;
  uint32_t bad = 0;
#pragma unroll 1
  for (int kt = lo & ~15; kt < hi; kt += 16) {
    if (kt >= u.all_lo && kt + 16 <= u.all_hi) continue;
    const int page = __ldg(p.tables + u.seq * p.table_stride + (kt >> p.bs_log2));
    if (page < 0 || page >= p.num_blocks) continue;
    const uint8_t* codes = p.value + page * p.v_sb + u.head * p.v_sh + static_cast<int64_t>(d) * bs + (kt & (bs - 1));
#pragma unroll 1
    for (int e = 0; e < 16; ++e, codes += bs)
#pragma unroll 1
      for (int t = max(lo - kt, 0); t < min(hi - kt, 16); ++t)
        if ((__ldg(codes + t) & 0x7f) == 0x7f) bad |= 1u << e;
  }
  return bad;
}

__device__ __forceinline__ void look_up(const BlockAttnParams& p, const Plan* plan, Walk& k) {
  k.seq = plan->seq[k.item];
  k.tile = plan->tile[k.item];
  k.v = seq_view(p, k.seq);
  k.span = span_of(p, k.v, k.tile);
}

__device__ __forceinline__ bool next_unit(const BlockAttnParams& p, const Plan* plan, Walk& k, Unit& u) {
  for (;;) {
    if (k.w >= k.w_end) return false;
    const int len = k.span.tiles > 0 ? k.span.tiles : 1;
    u.ta = static_cast<int>(max(k.w - k.w0 - kUnitCost, static_cast<int64_t>(0)));
    u.tb = static_cast<int>(min(k.w_end - k.w0 - kUnitCost, static_cast<int64_t>(len)));
    u.len = len;
    u.seq = k.seq, u.head = k.head, u.tile = k.tile, u.live = k.span.live, u.v = k.v;
    u.any_lo = k.span.any_lo, u.any_hi = k.span.any_hi, u.all_lo = k.span.all_lo, u.all_hi = k.span.all_hi;
    u.w_tiles = k.w0 + kUnitCost;
    u.t_first = k.span.t0 + u.ta;
    u.n = k.span.tiles > 0 ? u.tb - u.ta : 0;
    k.w0 += kUnitCost + len;
    k.w = k.w0;
    if (k.w < k.w_end && ++k.head == p.nh) {
      k.head = 0;
      do {
        ++k.item;
        look_up(p, plan, k);
      } while (k.span.live == 0);
    }
    if (u.tb > u.ta) return true;
  }
}

// f(0), f(1) ... f(N - 1) with the number as a constant.
template <int N, typename F, int... I>
__device__ __forceinline__ void steps_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void steps(F f) {
  steps_of<N>(f, std::make_integer_sequence<int, N>());
}

__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int HD, int CODE>
__global__ void __launch_bounds__(kThreads, 1)
    block_attn_tc_kernel(const __grid_constant__ BlockAttnParams p, const Plan* plan, int items) {
  extern __shared__ __align__(1024) uint8_t raw[];
  TcSmem<HD>& sm = *reinterpret_cast<TcSmem<HD>*>(raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
  const int64_t w_begin = walk.w;
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
    const int len = unit_len(walk.span);
    const int64_t rel = walk.w - plan->base[lo];
    walk.head = static_cast<int>(rel / len);
    walk.w0 = plan->base[lo] + static_cast<int64_t>(walk.head) * len;
  }
  if (tid == 0) {
    sm.gave_up = 0;
    sm.nan_seen = 0;
    mbar_init(&sm.spare, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.q_full[i], 4);
      mbar_init(&sm.k_full[i], 4);
      mbar_init(&sm.v_full[i], 4);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_empty[i], 1);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], 4);
      mbar_init(&sm.o_full[i], 1);
    }
    mbar_init_fence();
  }
  if (warp == 16) tmem_alloc<512>(&sm.tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const int bs = 1 << p.bs_log2;
  volatile int* gave_up = &sm.gave_up;

  if (warp < 8) {
    regs_up<128>();  // with 80 and 64 below: what the block was launched with
    // ---- softmax ----------------------------------------------------------------
    const int half = warp >> 2;
    const int r = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + half * 128;
    const uint32_t o_at = tmem + lanes + 256 + half * HD;
    uint32_t before = 0, mine = 0, ends = 0;  // tiles of all units so far, of those with this half, and how many of these had tiles
    bool ok = true;
    if (tid == 0) sm.walk[0] = walk;
    const Unit& u = sm.unit[0];
    for (;;) {
      if (tid == 0) sm.more[0] = next_unit(p, plan, sm.walk[0], sm.unit[0]);
      soft_sync();
      if (!sm.more[0]) break;
      const bool active = half * 128 < u.live;
      const bool on = half * 128 + r < u.live;
      const uint32_t row = u.tile * kUnitRows + half * 128 + r;  // below 2^24: see kMaxItems
      float qs = 0.f, m = -INFINITY, l = 0.f;
      float ref = -1e30f;  // weights are 2^(score - ref): m - kLift, or so low that any score but -inf shows
      if (active && u.n > 0) {
        int lo = 0, hi = 0;
        {  // this row of q to f16
          const int i = on ? row / p.group : 0, j = on ? row % p.group : 0;
          if (on) row_range(p, u.v, i, &lo, &hi);
          const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + (u.v.first + i) * p.q_sr +
                                                            (u.head * p.group + j) * p.q_sh);
          uint4 x[HD / 8];
#pragma unroll
          for (int e = 0; e < HD / 8; ++e) x[e] = on ? __ldg(src + e) : make_uint4(0, 0, 0, 0);
          int up = 0;
          if (p.q_bf16) {
            __nv_bfloat162 tops = __float2bfloat162_rn(0.f);
#pragma unroll
            for (int e = 0; e < HD / 2; ++e) tops = __hmax2(tops, __habs2(reinterpret_cast<const __nv_bfloat162*>(x)[e]));
            const float top = fmaxf(__low2float(tops), __high2float(tops));
            // the largest comes to 2^14 or, if it is below 2^-113, less
            if (top > 0.f && top < __uint_as_float(0x7f800000u)) up = min(14 - ilogbf(top), 127);
            const float factor = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
#pragma unroll
            for (int e = 0; e < HD / 2; ++e) {
              uint32_t& b = reinterpret_cast<uint32_t*>(x)[e];
              const float2 w = mul2(make_float2(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u)), make_float2(factor, factor));
              b = pack_f16(w.x, w.y);
            }
          }
#pragma unroll
          for (int e = 0; e < HD / 8; ++e)
            *reinterpret_cast<uint4*>(sm.q[half] + (e >> 3) * 16384 + r * 128 + (((e & 7) ^ (r & 7)) << 4)) = x[e];
          qs = ldexpf(p.scale_log2, -up);
          fence_async_shared();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.q_full[half]);
        }
        int all_lo, all_hi, unused;  // what all rows of this tile see
        {
          const int64_t row0 = static_cast<int64_t>(u.tile) * kUnitRows;
          const int last = min(u.live, half * 128 + 128) - 1;
          row_range(p, u.v, static_cast<int>((row0 + half * 128) / p.group), &unused, &all_hi);
          row_range(p, u.v, static_cast<int>((row0 + last) / p.group), &all_lo, &unused);
        }
        const int n = u.n, tok0 = u.t_first * kTile;
        for (int t = 0; t < n; ++t) {
          ok = ok && mbar_wait_warp(&sm.s_full[half], (mine + t) & 1, gave_up);
          tc_fence_after();
          const int tok = tok0 + t * kTile;
          const uint32_t ring = (before + t) & 3;
          const float *kf = sm.kfac[ring], *vlog = sm.vlog[ring];
          const uint32_t have = (sm.have[ring] & 0xfu) | ((sm.have[ring] >> 4) & 0xf0u);
          const uint32_t plain = (sm.plain[ring] & 0xfu) | ((sm.plain[ring] >> 4) & 0xf0u);
          const bool whole = tok >= all_lo && tok + kTile <= all_hi && have == 0xffu;
          // m moves to top for the rows of this warp: sums, accumulators and the weights of this tile's first
          // `stored` columns follow.
          auto raise = [&](float top, int stored) {
            const float mn = fmaxf(m, top);
            const float keep = mn == -INFINITY ? 1.f : exp2_fast(m - mn);
            m = mn;
            ref = m == -INFINITY ? -1e30f : m - kLift;
            l *= keep;
            if (t > 0) {
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
#pragma unroll 1
            for (int c = 0; c < stored; c += 16) {
              uint32_t y[8];
              tc_wait_st();
              tmem_ld(s_at + c / 2, y);
              tmem_wait(y);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&y[e]));
                y[e] = pack_f16(w.x * keep, w.y * keep);
              }
              tmem_st(s_at + c / 2, y);
            }
          };
          if (plain == 0xffu && p.scale_log2 > 0.f) {
            // 32 columns at a time, the next ones on their way.  Weights are taken against the maximum so far; only when
            // a sum of 16 of them shows that the maximum has grown too much is it looked for, and they are taken again.
            if (!whole) {  // scores that their row does not see become -inf
#pragma unroll 1
              for (int c = 0; c < 8; ++c) {
                const int first = tok + 16 * c, from = lo - first, to = (have >> c) & 1 ? hi - first : 0;
                if (!__any_sync(0xffffffffu, from > 0 || to < 16)) continue;
                uint32_t z[16];
                tmem_ld(s_at + c * 16, z);
                tmem_wait(z);
#pragma unroll
                for (int e = 0; e < 16; ++e) z[e] = e >= from && e < to ? z[e] : 0xff800000u;
                tmem_st(s_at + c * 16, z);
              }
              tc_wait_st();
            }
            uint32_t x[2][32];
            tmem_ld(s_at, x[0]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              tmem_wait(x[c & 1]);
              if (c < 3) tmem_ld(s_at + (c + 1) * 32, x[(c + 1) & 1]);
              uint32_t y[16];
              float2 sum[2];
              auto weights = [&](float ms) {
#pragma unroll
                for (int z = 0; z < 2; ++z) {  // 16 columns share their factors
                  const float f = fmaxf(kf[2 * c + z] * qs, 1e-37f), d = vlog[2 * c + z] - ms;  // not 0: masked scores are -inf
                  sum[z] = make_float2(0.f, 0.f);
#pragma unroll
                  for (int e = 0; e < 16; e += 2) {
                    const uint32_t* at = &x[c & 1][z * 16 + e];
                    float2 w = fma2(make_float2(__uint_as_float(at[0]), __uint_as_float(at[1])), make_float2(f, f), make_float2(d, d));
                    w.x = exp2_fast(w.x);
                    w.y = exp2_fast(w.y);
                    sum[z] = add2(sum[z], w);
                    y[(z * 16 + e) >> 1] = pack_f16(w.x, w.y);
                  }
                  sum[z].x += sum[z].y;
                }
              };
              weights(ref);
              if (__any_sync(0xffffffffu, fmaxf(sum[0].x, sum[1].x) > kSumLimit)) {
                float top = -INFINITY;
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                  const uint32_t* at = &x[c & 1][z * 16];
                  float best = fmaxf(__uint_as_float(at[0]), __uint_as_float(at[1]));
#pragma unroll
                  for (int e = 2; e < 16; e += 2) best = fmaxf(fmaxf(best, __uint_as_float(at[e])), __uint_as_float(at[e + 1]));
                  top = fmaxf(top, fmaf(best, kf[2 * c + z] * qs, vlog[2 * c + z]));
                }
                raise(top, c * 32);
                weights(ref);
              }
              l = fmaf(sum[0].x, sm.vinv[ring][2 * c], l);
              l = fmaf(sum[1].x, sm.vinv[ring][2 * c + 1], l);
              tmem_st(s_at + c * 16, y);
            }
          } else {
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t x[16], y[8];
              tmem_ld(s_at + c * 16, x);
              tmem_wait(x);
              const float f = kf[c] * qs, b = vlog[c], w = sm.vfac[ring][c];
              // columns [from, to) of these 16 are seen
              const int first = tok + 16 * c, from = lo - first, to = (have >> c) & 1 ? hi - first : 0;
              float top = -INFINITY;
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (e >= from && e < to) top = fmaxf(top, fmaf(__uint_as_float(x[e]), f, b));
              const bool grow = top > m + kLazy || (m == -INFINITY && top > m);
              if (__any_sync(0xffffffffu, grow)) raise(top, c * 16);
              const float ms = m == -INFINITY ? 0.f : m - kLift;
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                float p0 = exp2_fast(fmaf(__uint_as_float(x[e]), f, -ms));
                float p1 = exp2_fast(fmaf(__uint_as_float(x[e + 1]), f, -ms));
                p0 = e >= from && e < to ? p0 : 0.f;
                p1 = e + 1 >= from && e + 1 < to ? p1 : 0.f;
                l = fmaf(p0 + p1, 1.f / (1 << kSpare), l);
                // 0 where the row does not see the token, whatever its scale
                p0 = e >= from && e < to ? p0 * w : 0.f;
                p1 = e + 1 >= from && e + 1 < to ? p1 * w : 0.f;
                y[e >> 1] = pack_f16(p0, p1);
              }
              tmem_st(s_at + c * 8, y);
            }
          }
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_full[half]);
        }
        ok = ok && mbar_wait_warp(&sm.o_full[half], ends & 1, gave_up);
        tc_fence_after();
        mine += n;
        ++ends;
      }
      before += u.n;
      if (!ok) l = __uint_as_float(0x7fffffffu);  // a block that gave up leaves NaN, not stale memory

      // ---- this block's share of the unit -------------------------------------------
      auto place = [&](uint32_t row, uint16_t*& dst, float*& lse) {  // of a row's result
        const uint32_t i = row / p.group, j = row % p.group;
        dst = reinterpret_cast<uint16_t*>(p.out) + (u.v.first + i) * p.o_sr + (u.head * p.group + j) * p.o_sh;
        lse = p.lse == nullptr ? nullptr : p.lse + (static_cast<int64_t>(u.v.first + i) * p.nh + u.head) * p.group + j;
      };
      auto put = [&](uint16_t* dst, const float(&o)[16], float inv) {
        uint32_t y[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          if (p.q_bf16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(o[e] * inv, o[e + 1] * inv);
            y[e >> 1] = *reinterpret_cast<const uint32_t*>(&h);
          } else {
            y[e >> 1] = pack_f16(o[e] * inv, o[e + 1] * inv);
          }
        }
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
        if (lse != nullptr) *lse = sum > 0.f || sum != sum ? (mx + (log2f(sum) + (kSpare - kLift))) * 0.69314718055994531f : -INFINITY;
      };
      const bool split = u.ta > 0 || u.tb < u.len;
      constexpr int kFloats = kUnitRows * (HD + 2);  // of one partial sum: [HD][256], maxima, sums
      float* part = p.partial + (2 * static_cast<int64_t>(blockIdx.x) + (u.w_tiles > w_begin ? 1 : 0)) * kFloats;
      if (active) {
        uint16_t* dst = nullptr;
        float* lse = nullptr;
        if (on) place(row, dst, lse);
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        const bool nan_seen = CODE == MAK_CODE_E4M3 && u.n > 0 && *static_cast<volatile int*>(&sm.nan_seen);
#pragma unroll 1
        for (int d = 0; d < HD; d += 16) {
          uint32_t x[16];
          float o[16];
          if (u.n > 0) {
            tmem_ld(o_at + d, x);
            tmem_wait(x);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e)  // from 2^kLift to what l carries
            o[e] = u.n > 0 ? __uint_as_float(x[e]) * (1.f / (1 << kSpare)) : 0.f;
          if (CODE == MAK_CODE_E4M3 && nan_seen && on) {
            const uint32_t bad = nan_dims(p, u, row / p.group, d);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = bad >> e & 1 ? __uint_as_float(0x7fffffffu) : o[e];
          }
          if (split) {
#pragma unroll
            for (int e = 0; e < 16; ++e) part[(d + e) * kUnitRows + tid] = o[e];
          } else if (on) {
            put(dst + d, o, inv);
          }
        }
        if (split) {
          part[HD * kUnitRows + tid] = m;
          part[HD * kUnitRows + kUnitRows + tid] = l;
        } else if (on) {
          put_lse(lse, m, l);
        }
      }
      tc_fence_before();
      if (split) {
        const int first_block = static_cast<int>(u.w_tiles / chunk), last_block = static_cast<int>((u.w_tiles + u.len - 1) / chunk);
        const int slot0 = 2 * first_block + (u.w_tiles > first_block * chunk ? 1 : 0);
        soft_sync();
        if (tid == 0) {  // releases what the barrier has gathered
          int ticket;
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(ticket) : "l"(p.counters + slot0) : "memory");
          sm.last = ticket == last_block - first_block;
        }
        soft_sync();
        if (sm.last) {
          // Few rows leave several threads for each, which share its columns.  Four blocks' loads at a time.
          const int span = u.live > 128 ? 256 : u.live > 64 ? 128 : 64, mine_row = tid & (span - 1), cols = HD * span / kUnitRows;
          if (mine_row < u.live) {
            auto from = [&](int b) {
              return p.partial + (2 * static_cast<int64_t>(b) + (u.w_tiles > b * chunk ? 1 : 0)) * kFloats + mine_row;
            };
            float mx = -INFINITY, sum = 0.f;
#pragma unroll 4
            for (int b = first_block; b <= last_block; ++b) {
              const float pm = __ldcg(from(b) + HD * kUnitRows), pl = __ldcg(from(b) + HD * kUnitRows + kUnitRows);
              const float mn = fmaxf(mx, pm), ms = mn == -INFINITY ? 0.f : mn;
              sum = sum * exp2_fast(mx - ms) + pl * exp2_fast(pm - ms);
              mx = mn;
            }
            const float ms = mx == -INFINITY ? 0.f : mx, inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
            uint16_t* dst;
            float* lse;
            place(u.tile * kUnitRows + mine_row, dst, lse);
#pragma unroll 1
            for (int d = tid / span * cols, end = d + cols; d < end; d += 16) {
              float o[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = 0.f;
#pragma unroll 1
              for (int b = first_block; b <= last_block; b += 4) {
                float x[4][16], k[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                  const float* src = from(min(b + z, last_block));
                  k[z] = __ldcg(src + HD * kUnitRows);
#pragma unroll
                  for (int e = 0; e < 16; ++e) x[z][e] = __ldcg(src + (d + e) * kUnitRows);
                }
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                  k[z] = b + z <= last_block ? exp2_fast(k[z] - ms) : 0.f;
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[e] = b + z <= last_block ? fmaf(x[z][e], k[z], o[e]) : o[e];
                }
              }
              put(dst + d, o, inv);
            }
            if (tid < span) put_lse(lse, mx, sum);
          }
          if (tid == 0) p.counters[slot0] = 0;
        }
      }
      soft_sync();  // the unit is read
    }
  } else if (warp < 16) {
    regs_down<80>();
    // ---- codes to f16 in shared memory: K by the first four warps, V by the others ------------------
    const bool is_v = warp >= 12;
    const int w = warp & 3, mine = warp - 7;
    const int dlo = lane & 7, chunk16 = (w & 1) * 4 + (lane >> 3);
    const int d0 = (w >> 1) * (HD / 2) + dlo;
    constexpr int kIts = HD / 16;
    const uint32_t to = (chunk16 >> 2) * (HD * 128) + d0 * 128;
    const uint32_t c0 = ((((chunk16 & 3) * 2) ^ dlo) << 4), c1 = ((((chunk16 & 3) * 2 + 1) ^ dlo) << 4);
    uint8_t(*const buffers)[HD * 256] = is_v ? sm.v : sm.k;
    uint64_t *const full = is_v ? sm.v_full : sm.k_full, *const empty = is_v ? sm.v_empty : sm.k_empty;
    const int64_t stride = is_v ? p.v_sb : p.k_sb;
    uint4 x[kIts];
    uint32_t g = 0;  // tiles so far
    bool ok = true;
    if (lane == 0) sm.walk[mine] = walk;
    const Unit& u = sm.unit[mine];
    while (ok) {
      __syncwarp();
      if (lane == 0) sm.more[mine] = next_unit(p, plan, sm.walk[mine], sm.unit[mine]);
      __syncwarp();
      if (!sm.more[mine]) break;
      const int n = u.n, t_first = u.t_first, head = u.head;
      // Pieces outside need a look at their codes: those that some row does not see where a code of V may be NaN.
      constexpr bool kNan = CODE == MAK_CODE_E4M3;
      const int inner_lo = kNan && is_v ? u.all_lo : u.any_lo, inner_hi = kNan && is_v ? u.all_hi : u.any_hi;
      auto any_lo = [&]() { return kNan ? u.any_lo : inner_lo; };
      auto any_hi = [&]() { return kNan ? u.any_hi : inner_hi; };
      const uint8_t* base = (is_v ? p.value + head * p.v_sh : p.key + head * p.k_sh) + d0 * bs;
      const int32_t* table = p.tables + u.seq * p.table_stride;
      auto token = [&](int t) { return (t_first + t) * kTile + 16 * chunk16; };
      auto find = [&](int t) {
        const int kt = token(t);
        int pg = -1;
        if (t < n && kt < any_hi() && kt + 16 > any_lo()) pg = __ldg(table + (kt >> p.bs_log2));
        return pg >= p.num_blocks ? -1 : pg;
      };
      auto fetch = [&](int t, int pg) {
        const uint8_t* src = base + pg * stride + (token(t) & (bs - 1));
        if (pg >= 0) {
#pragma unroll
          for (int it = 0; it < kIts; ++it) x[it] = __ldg(reinterpret_cast<const uint4*>(src + it * 8 * bs));
        } else {
#pragma unroll
          for (int it = 0; it < kIts; ++it) x[it] = make_uint4(0, 0, 0, 0);
        }
      };
      float ks = 0.f, vs = 0.f;
      auto scales = [&](int pg) {
        ks = vs = 1.f;  // where there is no block nothing is seen
        if (!is_v && pg >= 0) {
          ks = __ldg(p.key_scale + pg * p.ks_sb + head * p.ks_sh);
          vs = __ldg(p.value_scale + pg * p.vs_sb + head * p.vs_sh);
        }
      };
      int page = find(0), next_page = find(1);
      if (n > 0) {
        fetch(0, page);
        scales(page);
      }
      for (int t = 0; t < n; ++t, ++g) {
        const int st = g & 1;
        ok = mbar_wait_warp_idle(&empty[st], ((g >> 1) & 1) ^ 1, gave_up);
        if (!ok) break;
        if (!is_v) {
          // the factors of tile g - 4 were last read before tile g - 2's scores were issued
          const bool fine = ks > 0.f && ks < INFINITY && vs >= 0x1p-110f && vs < INFINITY;
          if (dlo == 0 && w < 2) {
            sm.kfac[g & 3][chunk16] = ks;
            sm.vfac[g & 3][chunk16] = vs;
            // a scale of 0, or one that is no number, counts as 2^-100 in the maximum: its weights are right in the sum alone
            sm.vlog[g & 3][chunk16] = vs != 0.f && fabsf(vs) < INFINITY ? fmaxf(log2f(fabsf(vs)), kLeast) : -100.f;
            sm.vinv[g & 3][chunk16] = fine ? 1.f / (1 << kSpare) / vs : 0.f;
          }
          const uint32_t v1 = __ballot_sync(0xffffffffu, page >= 0), v2 = __ballot_sync(0xffffffffu, fine);
          if (lane == 0 && w < 2) {
            auto bits = [](uint32_t v) { return static_cast<uint8_t>((v & 1) | ((v >> 7) & 2) | ((v >> 14) & 4) | ((v >> 21) & 8)); };
            reinterpret_cast<uint8_t*>(&sm.have[g & 3])[w] = bits(v1);
            reinterpret_cast<uint8_t*>(&sm.plain[g & 3])[w] = bits(v2);
          }
        }
        const int kt = token(t);
        uint8_t* dst = buffers[st] + to;
        auto convert = [&](int it, uint4 z) {
          uint32_t y[8];
          codes4_to_f16<CODE>(z.x, &y[0], &y[1]);
          codes4_to_f16<CODE>(z.y, &y[2], &y[3]);
          codes4_to_f16<CODE>(z.z, &y[4], &y[5]);
          codes4_to_f16<CODE>(z.w, &y[6], &y[7]);
          *reinterpret_cast<uint4*>(dst + it * 1024 + c0) = make_uint4(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<uint4*>(dst + it * 1024 + c1) = make_uint4(y[4], y[5], y[6], y[7]);
        };
        uint32_t bad = 0;
        if (kt < inner_lo || kt + 16 > inner_hi) {
          if (!kNan || kt < any_lo() || kt + 16 > any_hi()) {
            // tokens that no row sees: their codes may be anything and become 0
            uint32_t mask[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              mask[q] = 0;
#pragma unroll
              for (int b = 0; b < 4; ++b)
                if (kt + 4 * q + b >= any_lo() && kt + 4 * q + b < any_hi()) mask[q] |= 0xffu << (8 * b);
            }
#pragma unroll
            for (int it = 0; it < kIts; ++it)
              x[it] = make_uint4(x[it].x & mask[0], x[it].y & mask[1], x[it].z & mask[2], x[it].w & mask[3]);
          }
          if (kNan && is_v) {
#pragma unroll
            for (int it = 0; it < kIts; ++it) bad |= nan_codes(x[it].x) | nan_codes(x[it].y) | nan_codes(x[it].z) | nan_codes(x[it].w);
          }
        }
#pragma unroll
        for (int it = 0; it < kIts; ++it) convert(it, x[it]);
        if (kNan && bad != 0) {
          // A weight of 0 times NaN would reach the rows that do not see the token: NaN becomes 0 here, and the rows that
          // see it get it with their results.
#pragma unroll 1
          for (int e = 0; e < kIts * 16; ++e) {
            uint16_t* h = reinterpret_cast<uint16_t*>(dst + (e >> 4) * 1024 + (e & 8 ? c1 : c0)) + (e & 7);
            if ((*h & 0x7fffu) > 0x7c00u) *h = 0;
          }
          *static_cast<volatile int*>(&sm.nan_seen) = 1;
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
        page = next_page;
        if (t + 1 < n) {
          fetch(t + 1, page);
          scales(page);
        }
        next_page = find(t + 2);
      }
    }
  } else {
    regs_down<64>();
    if (warp == 16 && lane == 0) {
      // ---- the tensor cores -------------------------------------------------------
      constexpr uint32_t kQk = instr_desc(kTile, 1, 0, false, true), kPv = instr_desc(HD, 1, 0, false, false);
      // Descriptors differ in their addresses alone, in units of 16 bytes: no carry leaves that field.
      const uint64_t q_desc = smem_desc(smem_addr(sm.q), 16, 1024, 7), k_desc = smem_desc(smem_addr(sm.k), HD * 128, 1024, 7);
      const uint64_t v_desc = smem_desc(smem_addr(sm.v), 16, 1024, 7);
      constexpr uint32_t kBuffer = HD * 256 / 16;
      auto scores = [&](int half, int st) {
        const uint64_t qd = q_desc + half * kBuffer, kd = k_desc + st * kBuffer;
        steps<HD / 16>([&](auto i) {
          constexpr int ks = decltype(i)::value;
          mma_ss_f16<(ks >> 2) * 1024 + (ks & 3) * 2, ks * 128>(tmem + half * 128, qd, kd, kQk, ks > 0);
        });
        tc_commit(&sm.s_full[half]);
      };
      uint32_t g = 0, mine[2] = {0, 0}, begins[2] = {0, 0};
      bool ok = true;
      sm.walk[9] = walk;
      const Unit& u = sm.unit[9];
      while (ok && next_unit(p, plan, sm.walk[9], sm.unit[9])) {
        const int n = u.n;
        if (n == 0) continue;
        const int halves = u.live > 128 ? 2 : 1;
        for (int half = 0; half < halves && ok; ++half) ok = mbar_wait(&sm.q_full[half], begins[half]++ & 1, gave_up);
        ok = ok && mbar_wait(&sm.k_full[g & 1], (g >> 1) & 1, gave_up);
        if (ok) {
          tc_fence_after();
          for (int half = 0; half < halves; ++half) scores(half, g & 1);
          tc_commit(&sm.k_empty[g & 1]);
        }
        for (int t = 0; t < n && ok; ++t, ++g) {
          const int st = g & 1;
          ok = mbar_wait(&sm.v_full[st], (g >> 1) & 1, gave_up);
          if (ok && t + 1 < n) ok = mbar_wait(&sm.k_full[st ^ 1], ((g + 1) >> 1) & 1, gave_up);
          for (int half = 0; half < halves && ok; ++half) {
            ok = mbar_wait(&sm.p_full[half], (mine[half] + t) & 1, gave_up);
            if (!ok) break;
            tc_fence_after();
            const uint64_t vd = v_desc + st * kBuffer;
            steps<kTile / 16>([&](auto i) {
              constexpr int ks = decltype(i)::value;
              mma_ts_f16<ks * 8, (ks >> 2) * (HD * 8) + (ks & 3) * 2>(tmem + 256 + half * HD, tmem + half * 128, vd, kPv, t > 0 || ks > 0);
            });
            if (half == halves - 1) tc_commit(&sm.v_empty[st]);
            if (t + 1 < n) {
              scores(half, st ^ 1);
              if (half == halves - 1) tc_commit(&sm.k_empty[st ^ 1]);
            } else {
              tc_commit(&sm.o_full[half]);
            }
          }
        }
        for (int half = 0; half < halves; ++half) mine[half] += n;
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
  if (warp == 16) {
    __syncwarp();
    tc_fence_after();
    tmem_free<512>(tmem);
  }
}

// Row tiles of all sequences, at most.
int64_t row_tiles(const BlockAttnParams& p) { return static_cast<int64_t>(p.num_rows) * p.group / kUnitRows + p.num_seqs; }

template <int HD, int CODE>
int launch_tc(const BlockAttnParams& p, Plan* plan, cudaStream_t st) {
  constexpr int kBytes = sizeof(TcSmem<HD>);
  static_assert(kBytes <= 227 * 1024, "shared memory of a block");
  const auto kernel = block_attn_tc_kernel<HD, CODE>;
  static bool ready[kMaxDevices] = {};
  if (int rc = prepare_kernel(kernel, kBytes, ready)) return rc;
  const int64_t items = row_tiles(p);
  if (int rc = launch_pdl("mak_block_attention", block_attn_plan_kernel, dim3(1), dim3(1024), 0, st, p, plan, static_cast<int>(items)))
    return rc;
  const int sms = sm_count();
  return launch_pdl("mak_block_attention", kernel, dim3(sms < kMaxGrid ? sms : kMaxGrid), dim3(kThreads), kBytes, st, p,
                    static_cast<const Plan*>(plan), static_cast<int>(items));
}

}  // namespace

int64_t block_attn_tc_partial_bytes() { return static_cast<int64_t>(2 * kMaxGrid) * kUnitRows * (128 + 2) * 4; }
bool block_attn_tc_fits(const BlockAttnParams& p) { return row_tiles(p) <= kMaxItems; }
int64_t block_attn_tc_plan_bytes() { return sizeof(Plan); }

int launch_block_attn_tc(const BlockAttnParams& p, int head_dim, int code, void* plan, cudaStream_t st) {
  Plan* at = static_cast<Plan*>(plan);
  if (head_dim == 64)
    return code == MAK_CODE_INT8 ? launch_tc<64, MAK_CODE_INT8>(p, at, st) : launch_tc<64, MAK_CODE_E4M3>(p, at, st);
  return code == MAK_CODE_INT8 ? launch_tc<128, MAK_CODE_INT8>(p, at, st) : launch_tc<128, MAK_CODE_E4M3>(p, at, st);
}

}  // namespace mak
