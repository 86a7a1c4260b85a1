// Attention over a paged 16-bit cache for few rows per sequence (single tokens, small trees), and the entry points.
//
// o = softmax(scale q K^T) V over the tokens that a row sees: a window and the first tokens, or the tokens before a tree
// of drafted ones and those that a row continues.  One pass over K and V with the running maximum m and sum l of a row;
// sums, statistics and accumulators are 32-bit.  A weight multiplies V as the sum of two 16-bit numbers, so it is good to
// 2^-16 (bfloat16) or 2^-22 (float16; lifted by 2^15, so that weights down to 2^-39 of the largest count).
//
// Bound by reading K and V.  A unit is 16 rows (tokens of a sequence times the query heads of a cache head) of one
// sequence and head, its work 16-token steps.  All units laid end to end are cut into equal runs, one per warp, whatever
// the lengths; a warp has its steps brought by TMA into a ring of its own, so no warp waits for another until its run ends.
// A unit cut by that leaves partial sums: the block joins those of its warps, the last block to arrive joins those of the
// blocks, both in order of position, so results do not depend on timing.
//
// Measured, calls in a graph, 8 cache heads of 128 in bfloat16 for 32 query heads: 64 requests of 256 to 4096 tokens with a
// window of 2048 85 us (5.1 TB/s of the 6.5 that a plain copy has), of which some 12 are the way to the first tile and the
// joins; one request that sees 4100 tokens 15.3 us, a chain of latencies (lengths, block ids, tiles, the block's join, the
// blocks'); three trees on 60000 to 100000 tokens, 4 heads, 102 us (5.1 TB/s).  12 warps with shorter rings: 98 us for the
// first; K and V by cp.async of single lines instead of TMA: 89.
#include "paged_attn_tc.cuh"
#include "tcgen05.cuh"

namespace mak {
namespace {

constexpr int kRows = 16;     // rows of a unit
constexpr int kStep = 16;     // tokens of a step: one page holds them
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxGrid = 148;
constexpr int kUnitCost = 2;  // a unit's beginning and end, in steps
constexpr int kMinRun = 2;    // steps that are worth another warp
constexpr int kQueue = 8;     // units between a warp's copies and its products, at most

struct Unit {
  PagedSeq v;
  Span s;
  int seq, head, tile, live;
  int ta, tb, len;  // this warp has steps [ta, tb) of len
  int64_t wt;       // where the unit's steps begin in all work
};

// What is left of a unit that a run's end cut.
struct Piece {
  int64_t wt;  // -1: none
  const float* at;
  int seq, head, tile, live, len, first;
};

template <int HD>
struct Smem {
  static constexpr int kStages = HD == 64 ? 6 : 3;
  static constexpr int kTileBytes = kStep * HD * 2;
  alignas(1024) uint8_t ring[kWarps][kStages][2 * kTileBytes];  // K, V: HD / 64 pieces of [16][64], lines of 128 bytes swizzled
  uint64_t full[kWarps][kStages];
  Unit queue[kWarps][kQueue];
  Piece pieces[2 * kWarps];
  int64_t before[kThreads + 1];  // work of the sequences of the threads before
  int64_t sums[kWarps];
  int join[2], gave_up;  // pieces of the units that this block joins, -1: none
};

__device__ __forceinline__ int tiles_of(const PagedParams& p, const PagedSeq& v) {
  return (v.rows * p.group + kRows - 1) / kRows;
}
__device__ __forceinline__ Span span_of_tile(const PagedParams& p, const PagedSeq& v, int tile, int* live) {
  const int row0 = tile * kRows;
  *live = min(v.rows * p.group - row0, kRows);
  return span_of<kStep>(p, v, row0 / p.group, (row0 + *live - 1) / p.group);
}
__device__ __forceinline__ int64_t work_of(const PagedParams& p, const PagedSeq& v) {
  int64_t sum = 0;
  const int tiles = tiles_of(p, v);
  for (int i = 0; i < tiles; ++i) {
    int live;
    sum += kUnitCost + max(span_of_tile(p, v, i, &live).tiles, 1);
  }
  return sum * p.nh;
}

// 64-bit division takes the time of a trip to memory; most fit 32 bits.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}

// A run: units one after another, the tiles of a (sequence, head) next to one another.
struct Walk {
  int64_t w, w_end, w0;  // w0: where the unit begins
  PagedSeq v;
  int seq, head, tile, tiles;
};
__device__ __forceinline__ bool next_unit(const PagedParams& p, Walk& k, Unit& u) {
  while (k.w < k.w_end) {
    int live;
    const Span s = span_of_tile(p, k.v, k.tile, &live);
    const int len = max(s.tiles, 1);
    const int64_t wt = k.w0 + kUnitCost;
    const int ta = static_cast<int>(max(k.w - wt, static_cast<int64_t>(0)));
    const int tb = static_cast<int>(min(k.w_end - wt, static_cast<int64_t>(len)));
    if (tb > ta) {
      u.v = k.v, u.s = s;
      u.seq = k.seq, u.head = k.head, u.tile = k.tile, u.live = live;
      u.ta = ta, u.tb = tb, u.len = len, u.wt = wt;
    }
    k.w0 = wt + len;
    k.w = k.w0;
    if (++k.tile == k.tiles) {
      k.tile = 0;
      if (++k.head == p.nh && k.w < k.w_end) {
        k.head = 0;
        do {
          k.v = paged_seq(p, ++k.seq);
          k.tiles = tiles_of(p, k.v);
        } while (k.tiles == 0);
      }
    }
    if (tb > ta) return true;
  }
  return false;
}

template <bool BF16>
__device__ __forceinline__ void store4(uint16_t* dst, float4 o, float f) {
  const uint32_t a = pack_two<BF16>(o.x * f, o.y * f), b = pack_two<BF16>(o.z * f, o.w * f);
  if ((reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(a, b);
  } else {
    dst[0] = static_cast<uint16_t>(a), dst[1] = static_cast<uint16_t>(a >> 16);
    dst[2] = static_cast<uint16_t>(b), dst[3] = static_cast<uint16_t>(b >> 16);
  }
}

// Four columns of a row's sum over some of its tokens.
struct Sum {
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(const Sum& y) {
    const float now = fmaxf(m, y.m);
    const float a = now == -INFINITY ? 1.f : shrink(m - now), b = now == -INFINITY ? 1.f : shrink(y.m - now);
    o.x = o.x * a + y.o.x * b, o.y = o.y * a + y.o.y * b, o.z = o.z * a + y.o.z * b, o.w = o.w * a + y.o.w * b;
    l = l * a + y.l * b;
    m = now;
  }
};

// Partial sums: [16][HD] accumulators, 16 maxima, 16 sums.
template <int HD>
constexpr int kPieceFloats = kRows * (HD + 2);

template <int HD, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) 
    paged_rows_kernel(const __grid_constant__ PagedParams p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  constexpr int kStages = Smem<HD>::kStages, kTileBytes = Smem<HD>::kTileBytes;
  constexpr int kPieces = HD / 64, kPiece = kStep * 128;  // of a step's K or V
  constexpr float kLift = BF16 ? 0.f : 15.f;    // log2 factor that weights carry
  extern __shared__ __align__(1024) uint8_t raw[];
  Smem<HD>& sm = *reinterpret_cast<Smem<HD>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
    sm.gave_up = 0;
    for (int i = 0; i < kWarps * kStages; ++i) mbar_init(&sm.full[0][0] + i, 1);
    mbar_init_fence();
  }
  pdl_wait();
  pdl_trigger();

  // ---- all work, and this warp's run ----------------------------------------------
  const int per = (p.num_seqs + kThreads - 1) / kThreads;
  const int s0 = min(tid * per, p.num_seqs), s1 = min(s0 + per, p.num_seqs);
  {
    int64_t mine = 0;
    for (int s = s0; s < s1; ++s) mine += work_of(p, paged_seq(p, s));
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) sm.sums[warp] = incl;
    __syncthreads();
    int64_t at = incl - mine;
#pragma unroll
    for (int i = 0; i < kWarps; ++i)
      if (i < warp) at += sm.sums[i];
    sm.before[tid] = at;
    if (tid == kThreads - 1) sm.before[kThreads] = at + mine;
    if (tid < 2 * kWarps) sm.pieces[tid].wt = -1;
    if (tid < 2) sm.join[tid] = -1;
    __syncthreads();
  }
  const int64_t total = sm.before[kThreads];
  int64_t run = divide(total + gridDim.x * kWarps - 1, gridDim.x * kWarps);
  if (run < kMinRun) run = kMinRun;
  const int64_t block_run = run * kWarps, block_begin = blockIdx.x * block_run;
  if (block_begin >= total) return;

  Walk walk;
  walk.w = block_begin + warp * run;
  walk.w_end = min(walk.w + run, total);
  if (walk.w < walk.w_end) {
    int lo = 0, n = kThreads;  // the last thread whose sequences begin at or before w
    while (n > 1) {
      const int step = (n + 31) >> 5, at = lo + lane * step;
      const uint32_t votes = __ballot_sync(0xffffffffu, at < lo + n && sm.before[min(at, kThreads)] <= walk.w);
      const int k = 31 - __clz(votes), end = lo + n;
      lo += k * step;
      n = min(step, end - lo);
    }
    int64_t at = sm.before[lo];
    walk.seq = min(lo * per, p.num_seqs - 1);
    for (;;) {
      walk.v = paged_seq(p, walk.seq);
      const int64_t work = work_of(p, walk.v);
      if (walk.w < at + work) {
        walk.tiles = tiles_of(p, walk.v);
        const int64_t one = divide(work, p.nh);
        walk.head = static_cast<int>(divide(walk.w - at, one));
        at += one * walk.head;
        break;
      }
      at += work;
      ++walk.seq;
    }
    walk.tile = 0;
    for (;;) {
      int live;
      const int len = kUnitCost + max(span_of_tile(p, walk.v, walk.tile, &live).tiles, 1);
      if (walk.w < at + len) break;
      at += len;
      ++walk.tile;
    }
    walk.w0 = at;
  }

  // ---- loads, some steps ahead of the products ---------------------------------------
  const uint32_t ring = shared_at(sm.ring[warp]);
  uint64_t* full = sm.full[warp];
  volatile int* gave_up = &sm.gave_up;
  Unit* queue = sm.queue[warp];
  int units_in = 0, left_in = 0;   // steps of the unit at hand that are left
  int tok_in = 0, jump_at = 0, jump = 0, tiles_in = 0, head_in = 0, next_id = -1;
  const int32_t* table_in = nullptr;
  bool more = true;
  const int inside = (1 << p.bs_log2) - 1;
  // Steps go up by 16 tokens, but for one jump from the first tokens to the window.
  auto enter = [&]() {
    Unit u;
    more = more && next_unit(p, walk, u);
    if (!more) return;
    __syncwarp();
    if (lane == 0) queue[units_in % kQueue] = u;
    __syncwarp();
    ++units_in;
    left_in = u.tb - u.ta, tiles_in = u.s.tiles, head_in = u.head;
    tok_in = tile_token<kStep>(u.s, u.ta);
    jump_at = u.ta < u.s.ns ? kStep * (u.s.ns - 1) : -1, jump = kStep * u.s.t0;
    table_in = p.tables + u.seq * p.table_stride;
    next_id = tiles_in > 0 ? __ldg(table_in + (tok_in >> p.bs_log2)) : -1;  // looked at when it is needed, a step later
  };
  int in = 0, stage_in = 0;  // steps loaded so far
  uint32_t there = 0;        // bit i: step i % 32 has a page
  bool ok = true;            // no wait has run out
  auto load = [&]() {
    if (more && left_in == 0) enter();
    if (!more) return;
    const int page = __shfl_sync(0xffffffffu, next_id, 0), tok = __shfl_sync(0xffffffffu, tok_in, 0), head = __shfl_sync(0xffffffffu, head_in, 0);
    const bool has = ok && page >= 0 && page < p.num_blocks;
    there = (there & ~(1u << (in & 31))) | (has ? 1u << (in & 31) : 0u);
    tok_in = tok_in == jump_at ? jump : tok_in + kStep;
    --left_in;
    next_id = left_in > 0 && tiles_in > 0 ? __ldg(table_in + (tok_in >> p.bs_log2)) : -1;
    if (has && elect_one()) {
      const uint32_t to = ring + stage_in * (2 * kTileBytes);
      uint64_t* bar = full + stage_in;
      mbar_arrive_expect(bar, 2 * kTileBytes);
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        box_load(to + c * kPiece, &k_map, c * 64, head, tok & inside, page, bar);
        box_load(to + kTileBytes + c * kPiece, &v_map, c * 64, head, tok & inside, page, bar);
      }
    }
    __syncwarp();
    ++in;
    stage_in = stage_in + 1 == kStages ? 0 : stage_in + 1;
  };
  if (walk.w < walk.w_end) {
    enter();
  } else {
    more = false;
  }
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load();

  // ---- products --------------------------------------------------------------------------
  const int r = lane >> 2, c2 = (lane & 3) * 2;  // this lane's rows r and r + 8, columns c2 and c2 + 1 of 8
  const float scale = fmaxf(fabsf(p.scale_log2), 1e-37f);  // not 0: masked scores are -inf
  const uint32_t sign = p.scale_log2 < 0.f ? 0x80008000u : 0u;
  int units_out = 0, out = 0, stage = 0;
  uint32_t phases = 0;  // bit of a stage: the parity of its next phase
  while (units_out < units_in) {
    const Unit& u = queue[units_out % kQueue];
    uint32_t qf[HD / 16][4];
    int64_t row_q[2];
    RowView see[2];
    int who[2];
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int x = r + 8 * z;
      const int row = u.tile * kRows + min(x, u.live - 1);
      who[z] = row / p.group;
      const int j = row - who[z] * p.group;
      row_q[z] = (static_cast<int64_t>(u.v.first) + who[z]) * p.q_sr + (static_cast<int64_t>(u.head) * p.group + j) * p.q_sh;
      see[z] = row_view(p, u.v, who[z]);
    }
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        qf[ks][e] = __ldg(reinterpret_cast<const uint32_t*>(p.q + row_q[e & 1] + ks * 16 + (e >> 1) * 8 + c2)) ^ sign;
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    const int ta = u.ta, tb = u.tb, live = u.live;
    const Span span = u.s;
    for (int j = ta; j < tb; ++j, ++out) {
      load();
      bool has = there >> (out & 31) & 1;
      if (has && !mbar_wait_warp(full + stage, phases >> stage & 1, gave_up)) {
        land<kStages>(full, out, in, there, phases);
        there = 0;
        has = ok = false;
      }
      if (has) {
        phases ^= 1u << stage;
        const int tok = tile_token<kStep>(span, j);
        const uint32_t at = ring + stage * (2 * kTileBytes);
        float s[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
        {
          const int t = ((lane >> 4) << 3) + (lane & 7), half = (lane >> 3) & 1;
          const uint32_t row = at + t * 128;
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            uint32_t b[4];
            load_matrix(row + (ks >> 2) * kPiece + (((2 * (ks & 3) + half) ^ (t & 7)) << 4), b);
            mma_16816<BF16>(s[0], qf[ks], b[0], b[1]);
            mma_16816<BF16>(s[1], qf[ks], b[2], b[3]);
          }
        }
        const bool whole = tile_whole<kStep>(span, tok);
        uint32_t bits[2] = {0xffffu, 0xffffu};  // tokens that the lane's rows see
        if (!whole) {
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            if (p.parents != nullptr) {
              bits[z] = tree_bits(p, u.v, who[z], tok) & 0xffffu;
            } else {
              auto below = [](int k) { return k >= kStep ? 0xffffu : k <= 0 ? 0u : (1u << k) - 1u; };
              bits[z] = below(see[z].hi - tok) & (~below(see[z].lo - tok) | below(p.sinks - tok));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                s[i][2 * z + e] = bits[z] >> (i * 8 + c2 + e) & 1 ? s[i][2 * z + e] : -INFINITY;
          }
        }
        float keep[2], ref[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          float top = fmaxf(fmaxf(s[0][2 * z], s[0][2 * z + 1]), fmaxf(s[1][2 * z], s[1][2 * z + 1]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * scale;
          const float now = fmaxf(m[z], top);
          keep[z] = now == m[z] ? 1.f : shrink(m[z] - now);
          ref[z] = now == -INFINITY ? 0.f : now - kLift;
          m[z] = now;
        }
        if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
          l[0] *= keep[0], l[1] *= keep[1];
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) o[i][0] *= keep[0], o[i][1] *= keep[0], o[i][2] *= keep[1], o[i][3] *= keep[1];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[i][e] = exp2_near(fmaf(s[i][e], scale, -ref[e >> 1]));
            l[e >> 1] += s[i][e];
          }
        const uint32_t values = at + kTileBytes;
        bool odd = false;
        if (!whole) {  // 0 times an infinite value is not 0: such a value is kept from the rows that do not see it
#pragma unroll 1
          for (int i = lane; i < kTileBytes / 16; i += 32) {
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(values + i * 16) : "memory");
            odd = odd || odd_two<BF16>(w[0]) || odd_two<BF16>(w[1]) || odd_two<BF16>(w[2]) || odd_two<BF16>(w[3]);
          }
          odd = __any_sync(0xffffffffu, odd);
        }
        if (!odd) {
          // A weight is the sum of the two.  Neither is 0 where an infinite value may be seen: 0 times it is no number.
          const uint32_t least = whole ? 0x00010001u : 0u;
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = s[e >> 1][(e & 1) * 2], b = s[e >> 1][(e & 1) * 2 + 1];
            hi[e] = cut_two<BF16>(a, b);
            const float2 f = unpack_two<BF16>(hi[e]);
            lo[e] = __vmaxu2(pack_two<BF16>(a - f.x, b - f.y), least);
            hi[e] = __vmaxu2(hi[e], least);
          }
          const int t = (((lane >> 3) & 1) << 3) + (lane & 7), half = lane >> 4;
          const uint32_t row = values + t * 128;
#pragma unroll
          for (int d = 0; d < HD / 16; ++d) {
            uint32_t b[4];
            load_matrix_t(row + (d >> 2) * kPiece + (((2 * (d & 3) + half) ^ (t & 7)) << 4), b);
            mma_16816<BF16>(o[2 * d], hi, b[0], b[1]);
            mma_16816<BF16>(o[2 * d + 1], hi, b[2], b[3]);
            mma_16816<BF16>(o[2 * d], lo, b[0], b[1]);
            mma_16816<BF16>(o[2 * d + 1], lo, b[2], b[3]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < kStep; ++t) {
            float w[2];
#pragma unroll
            for (int z = 0; z < 2; ++z)  // not 0 either
              w[z] = fmaxf(__shfl_sync(0xffffffffu, s[t >> 3][z * 2 + (t & 1)], (lane & ~3) | ((t & 7) >> 1)), 0x1p-126f);
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) {
              uint32_t x;
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(values + (d >> 3) * kPiece + t * 128 + (((d & 7) ^ (t & 7)) << 4) + c2 * 2) : "memory");
              const float2 f = unpack_two<BF16>(x);
              if (bits[0] >> t & 1) o[d][0] = fmaf(w[0], f.x, o[d][0]), o[d][1] = fmaf(w[0], f.y, o[d][1]);
              if (bits[1] >> t & 1) o[d][2] = fmaf(w[1], f.x, o[d][2]), o[d][3] = fmaf(w[1], f.y, o[d][3]);
            }
          }
        }
      }
      stage = stage + 1 == kStages ? 0 : stage + 1;
      __syncwarp();  // the stage is read
    }
    if (!ok) l[0] = l[1] = __uint_as_float(0x7fffffffu);  // a block that gave up leaves NaN

    // ---- this warp's share of the unit ----------------------------------------------------
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      l[z] += __shfl_xor_sync(0xffffffffu, l[z], 1);
      l[z] += __shfl_xor_sync(0xffffffffu, l[z], 2);
    }
    if (ta == 0 && tb == u.len) {
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        if (r + 8 * z >= live) continue;
        const int row = u.tile * kRows + r + 8 * z;
        const int64_t i = u.v.first + row / p.group, h = static_cast<int64_t>(u.head) * p.group + row % p.group;
        uint16_t* dst = static_cast<uint16_t*>(p.out) + i * p.o_sr + h * p.o_sh + c2;
        const float inv = l[z] > 0.f || l[z] != l[z] ? 1.f / l[z] : 0.f;
        const bool even = (reinterpret_cast<uintptr_t>(dst) & 3) == 0;
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) {
          const uint32_t w = pack_two<BF16>(o[d][2 * z] * inv, o[d][2 * z + 1] * inv);
          if (even) {
            *reinterpret_cast<uint32_t*>(dst + d * 8) = w;
          } else {
            dst[d * 8] = static_cast<uint16_t>(w);
            dst[d * 8 + 1] = static_cast<uint16_t>(w >> 16);
          }
        }
        if (p.lse != nullptr && (lane & 3) == 0)
          p.lse[i * p.nh * p.group + h] = l[z] > 0.f || l[z] != l[z] ? (m[z] - kLift + log2f(l[z])) * 0.69314718055994531f : -INFINITY;
      }
    } else {
      // The last piece of a run finds its place in the ring, which is empty by then.
      const bool final_piece = !more && units_out + 1 == units_in;
      const int slot = ta > 0 ? 0 : 1;  // a run begins inside one unit at most, and ends inside one
      float* part = final_piece ? reinterpret_cast<float*>(sm.ring[warp])
                                : p.partial + (static_cast<int64_t>(blockIdx.x) * (2 * kWarps) + warp * 2 + slot) * kPieceFloats<HD>;
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        if (r + 8 * z >= live) continue;
        float* dst = part + (r + 8 * z) * HD + c2;
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) *reinterpret_cast<float2*>(dst + d * 8) = make_float2(o[d][2 * z], o[d][2 * z + 1]);
        if ((lane & 3) == 0) {
          part[kRows * HD + r + 8 * z] = m[z];
          part[kRows * HD + kRows + r + 8 * z] = l[z];
        }
      }
      if (lane == 0) {
        Piece& x = sm.pieces[warp * 2 + slot];
        x.wt = u.wt, x.at = part;
        x.seq = u.seq, x.head = u.head, x.tile = u.tile, x.live = u.live, x.len = u.len, x.first = u.v.first;
      }
    }
    ++units_out;
    __syncwarp();
  }
  __syncthreads();

  // ---- pieces of the same unit: a warp for each unit, then the block for what other blocks have left ----------
  auto finish = [&](const Piece& x, int row_in, int d, const Sum& s) {
    const int row = x.tile * kRows + row_in;
    const int64_t i = x.first + row / p.group, h = static_cast<int64_t>(x.head) * p.group + row % p.group;
    const bool any = s.l > 0.f || s.l != s.l;
    store4<BF16>(static_cast<uint16_t*>(p.out) + i * p.o_sr + h * p.o_sh + d, s.o, any ? 1.f / s.l : 0.f);
    if (p.lse != nullptr && d == 0) p.lse[i * p.nh * p.group + h] = any ? (s.m - kLift + log2f(s.l)) * 0.69314718055994531f : -INFINITY;
  };
  auto of_block = [&](int64_t b, int64_t wt) {  // a block's sum of a unit that others share
    return p.partial + (static_cast<int64_t>(gridDim.x) * (2 * kWarps) + 2 * b + (wt > b * block_run ? 1 : 0)) * kPieceFloats<HD>;
  };
  {
    const int64_t wt_mine = lane < 2 * kWarps ? sm.pieces[lane].wt : -1;
    const uint32_t used = __ballot_sync(0xffffffffu, wt_mine >= 0);
    const uint32_t lower = used & ((1u << lane) - 1);
    const int64_t wt_before = __shfl_sync(0xffffffffu, wt_mine, lower ? 31 - __clz(lower) : 0);
    uint32_t heads = __ballot_sync(0xffffffffu, wt_mine >= 0 && (lower == 0 || wt_before != wt_mine));
    for (int k = 0; heads != 0; ++k) {
      const int g = __ffs(heads) - 1;
      heads &= heads - 1;
      if (k % kWarps != warp) continue;
      const uint32_t members = used & (heads ? (1u << (__ffs(heads) - 1)) - 1 : 0xffffffffu) & ~((1u << g) - 1);
      const Piece& x = sm.pieces[g];
      const int64_t wt = x.wt, first = divide(wt, block_run), last = divide(wt + x.len - 1, block_run);
      const int live = x.live;
      float* mine = of_block(blockIdx.x, wt);
      constexpr int kAcross = HD / 4, kDown = 32 / kAcross;  // lanes of a row, rows at once
      const int d = lane % kAcross * 4;
      for (int row0 = lane / kAcross; row0 < live; row0 += 4 * kDown) {
        Sum sum[4];
        for (uint32_t left = members; left != 0; left &= left - 1) {
          const float* at = sm.pieces[__ffs(left) - 1].at;
          Sum y[4];
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            const int row = min(row0 + z * kDown, live - 1);
            y[z].m = at[kRows * HD + row], y[z].l = at[kRows * HD + kRows + row];
            y[z].o = *reinterpret_cast<const float4*>(at + row * HD + d);
          }
#pragma unroll
          for (int z = 0; z < 4; ++z) sum[z].add(y[z]);
        }
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const int row = row0 + z * kDown;
          if (row >= live) continue;
          if (first == last) {
            finish(x, row, d, sum[z]);
          } else {
            *reinterpret_cast<float4*>(mine + row * HD + d) = sum[z].o;
            if (d == 0) mine[kRows * HD + row] = sum[z].m, mine[kRows * HD + kRows + row] = sum[z].l;
          }
        }
      }
      if (first != last) {
        __syncwarp();
        if (lane == 0) {  // releases what the warp has written
          int ticket;
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(ticket) : "l"(p.counters + first) : "memory");
          if (ticket == last - first) {
            sm.join[wt > block_begin ? 1 : 0] = g;
            p.counters[first] = 0;
          }
        }
      }
    }
  }
  __syncthreads();
  for (int which = 0; which < 2; ++which) {
    const int g = sm.join[which];
    if (g < 0) continue;
    const Piece& x = sm.pieces[g];
    const int64_t wt = x.wt, first = divide(wt, block_run), last = divide(wt + x.len - 1, block_run);
    const int items = x.live * (HD / 4);
    const int parts = items < kThreads ? kThreads / items : 1;  // of the blocks, for rows too few for all threads
    Sum* shared = reinterpret_cast<Sum*>(sm.ring);
    for (int i = tid; i < items * parts; i += kThreads) {
      const int item = i % items, part = i / items, row = item / (HD / 4), d = item % (HD / 4) * 4;
      Sum sum;
      for (int64_t b = first + part; b <= last; b += 4 * parts) {
        Sum y[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const float* at = of_block(min(b + z * parts, last), wt);
          y[z].m = __ldcg(at + kRows * HD + row), y[z].l = __ldcg(at + kRows * HD + kRows + row);
          y[z].o = __ldcg(reinterpret_cast<const float4*>(at + row * HD + d));
        }
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if (b + z * parts <= last) sum.add(y[z]);
      }
      if (parts == 1)
        finish(x, row, d, sum);
      else
        shared[i] = sum;
    }
    if (parts > 1) {
      __syncthreads();
      if (tid < items) {
        Sum sum;
        for (int part = 0; part < parts; ++part) sum.add(shared[part * items + tid]);
        finish(x, tid / (HD / 4), tid % (HD / 4) * 4, sum);
      }
    }
    __syncthreads();
  }
}

template <int HD, bool BF16>
int launch_rows(const PagedParams& p, const CUtensorMap& k, const CUtensorMap& v, const char* name, cudaStream_t st) {
  constexpr int kBytes = sizeof(Smem<HD>);
  static_assert(kBytes <= 227 * 1024, "shared memory of a block");
  static_assert(kRows * (HD + 2) * 4 <= Smem<HD>::kStages * 2 * Smem<HD>::kTileBytes, "a piece fits its warp's ring");
  static_assert(kQueue > Smem<HD>::kStages, "units in flight");
  const auto kernel = paged_rows_kernel<HD, BF16>;
  static bool ready[kPagedDevices] = {};
  if (int rc = paged_prepare(name, kernel, kBytes, ready)) return rc;
  const int sms = sm_count();
  return launch_pdl(name, kernel, dim3(sms < kMaxGrid ? sms : kMaxGrid), dim3(kThreads), kBytes, st, p, k, v);
}

int64_t plan_bytes() { return (paged_tc_plan_bytes() + 255) / 256 * 256; }
static_assert(kMaxGrid * 4 <= kPagedCounterBytes, "a counter per block");

}  // namespace

int check_paged_cache(const mak_paged_cache_desc& c, bool values, const char* name) {
  if (c.head_dim != 64 && c.head_dim != 128) return fail(MAK_E_UNSUPPORTED, "%s: head_dim must be 64 or 128, got %d", name, c.head_dim);
  if (c.block_size != 16 && c.block_size != 32 && c.block_size != 64 && c.block_size != 128)
    return fail(MAK_E_UNSUPPORTED, "%s: block_size must be 16, 32, 64 or 128, got %d", name, c.block_size);
  if (c.dtype != MAK_DT_F16 && c.dtype != MAK_DT_BF16) return fail(MAK_E_UNSUPPORTED, "%s: caches must be float16 or bfloat16", name);
  if (c.num_seqs < 0 || c.num_blocks < 0 || c.max_blocks < 0 || c.num_rows < 0 || c.num_heads <= 0)
    return fail(MAK_E_INVALID, "%s: negative size", name);
  if (c.num_seqs > 0x7fffffff || c.num_blocks > 0x7fffffff || c.num_rows > 0x7fffffff || c.max_blocks > 0x7fffffff / c.block_size)
    return fail(MAK_E_UNSUPPORTED, "%s: sequences, blocks, rows and tokens of a sequence are 32-bit counts", name);
  if (c.num_seqs > 0 && (c.context_lens == nullptr || (c.max_blocks > 0 && c.block_tables == nullptr)))
    return fail(MAK_E_INVALID, "%s: null block_tables or context_lens", name);
  if (c.num_blocks > 0 && (c.key == nullptr || (values && c.value == nullptr))) return fail(MAK_E_INVALID, "%s: null cache", name);
  uint64_t bits = reinterpret_cast<uintptr_t>(c.key), strides = static_cast<uint64_t>(c.key_stride_block | c.key_stride_token | c.key_stride_head);
  if (values) {
    bits |= reinterpret_cast<uintptr_t>(c.value);
    strides |= static_cast<uint64_t>(c.value_stride_block | c.value_stride_token | c.value_stride_head);
  }
  if ((bits & 15) || (strides & 7)) return fail(MAK_E_INVALID, "%s: caches need 16-byte aligned addresses and strides", name);
  return MAK_OK;
}

PagedParams paged_params(const mak_paged_cache_desc& c) {
  PagedParams p = {};
  p.key = static_cast<const uint16_t*>(c.key);
  p.value = static_cast<const uint16_t*>(c.value);
  p.k_sb = c.key_stride_block, p.k_st = c.key_stride_token, p.k_sh = c.key_stride_head;
  p.v_sb = c.value_stride_block, p.v_st = c.value_stride_token, p.v_sh = c.value_stride_head;
  p.tables = c.block_tables, p.ctx_lens = c.context_lens, p.starts = c.cu_seqlens;
  p.table_stride = c.table_stride, p.num_blocks = c.num_blocks;
  p.num_seqs = static_cast<int32_t>(c.num_seqs), p.max_blocks = static_cast<int32_t>(c.max_blocks);
  p.num_rows = static_cast<int32_t>(c.num_rows);
  p.nh = c.num_heads;
  p.bs_log2 = c.block_size == 16 ? 4 : c.block_size == 32 ? 5 : c.block_size == 64 ? 6 : 7;
  return p;
}

int check_paged_workspace(const void* workspace, int64_t bytes, const char* name) {
  if (workspace == nullptr || bytes < mak_paged_attention_workspace_bytes()) return fail(MAK_E_WORKSPACE, "%s: workspace missing or too small", name);
  // partial sums are read from it 16 bytes at a time, and the map of a pool without blocks has its address
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(MAK_E_WORKSPACE, "%s: the workspace must begin on 16 bytes", name);
  return MAK_OK;
}

PagedSpace paged_space(void* workspace) {
  char* at = static_cast<char*>(workspace);
  return {static_cast<int32_t*>(workspace), at + kPagedCounterBytes, plan_bytes(), reinterpret_cast<float*>(at + kPagedCounterBytes + plan_bytes())};
}

}  // namespace mak

using namespace mak;

extern "C" int64_t mak_paged_attention_workspace_bytes(void) {
  const int64_t few = static_cast<int64_t>(kMaxGrid) * (2 * kWarps + 2) * kPieceFloats<128> * 4, many = paged_tc_partial_bytes();
  return kPagedCounterBytes + plan_bytes() + (few > many ? few : many);
}

extern "C" int mak_paged_attention(const mak_paged_attn_desc* d, void* stream) {
  const char* name = "mak_paged_attention";
  if (d == nullptr) return fail(MAK_E_INVALID, "%s: null descriptor", name);
  const mak_paged_cache_desc& c = d->cache;
  if (int rc = check_paged_cache(c, true, name)) return rc;
  if (d->num_q_heads <= 0 || d->num_q_heads % c.num_heads)
    return fail(MAK_E_INVALID, "%s: %d query heads over %d cache heads", name, d->num_q_heads, c.num_heads);
  if (d->window < 0 || d->sinks < 0) return fail(MAK_E_INVALID, "%s: negative window or sinks", name);
  if (!std::isfinite(d->scale * 1.4426950408889634f)) return fail(MAK_E_INVALID, "%s: the scale is not finite", name);
  if (d->parents != nullptr && d->window) return fail(MAK_E_INVALID, "%s: a tree has no window", name);
  if (c.num_rows * d->num_q_heads / c.num_heads > 0x7fffffff - 256)
    return fail(MAK_E_UNSUPPORTED, "%s: rows times query heads of a cache head are a 32-bit count", name);
  if (c.num_seqs == 0 || c.num_rows == 0) return MAK_OK;
  if (d->q == nullptr || d->out == nullptr) return fail(MAK_E_INVALID, "%s: null q or out", name);
  if ((reinterpret_cast<uintptr_t>(d->q) & 15) || ((d->q_stride_row | d->q_stride_head) & 7))
    return fail(MAK_E_INVALID, "%s: q needs 16-byte aligned rows", name);
  if (int rc = check_paged_workspace(d->workspace, d->workspace_bytes, name)) return rc;
  PagedParams p = paged_params(c);
  p.parents = d->parents;
  p.q = static_cast<const uint16_t*>(d->q), p.out = d->out, p.lse = d->lse;
  p.q_sr = d->q_stride_row, p.q_sh = d->q_stride_head, p.o_sr = d->out_stride_row, p.o_sh = d->out_stride_head;
  p.group = d->num_q_heads / c.num_heads;
  p.window = d->window, p.sinks = d->window ? d->sinks : 0;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  const PagedSpace space = paged_space(d->workspace);
  p.counters = space.counters, p.partial = space.partial;
  cudaStream_t st = as_stream(stream);
  const bool bf16 = c.dtype == MAK_DT_BF16;
  // Rows that share a cache head, on average.  Few rows read K and V again for every 16; many rows wait for a unit's
  // longer beginning and end.  Few / many in us, 8 cache heads of 128 with 4 query heads: 16 sequences of 4096 tokens
  // 63 / 62 for 16 rows, 110 / 62 for 32 (heads of 64: 38 / 49, 61 / 49); 64 of 512 44 / 61, 55 / 61, 76 / 70 for 48; one of
  // 4096 25 / 27, 25 / 27, 35 / 48 for 128.  The average alone decides, which is not the faster kernel everywhere: one sequence's
  // 17 to 128 rows, and 32 rows of many short sequences, are taken up to a third slower than the other kernel would.
  const int64_t rows = c.num_rows * p.group / c.num_seqs;
  const bool many = rows > 16 && paged_tc_fits(p);
  const int tokens = many ? paged_tc_box(c.block_size) : kStep;
  CUtensorMap k, v;
  if (!paged_map(&k, p.key, p.k_sb, p.k_st, p.k_sh, p.num_blocks, p.nh, c.head_dim, c.block_size, bf16, tokens, d->workspace) ||
      !paged_map(&v, p.value, p.v_sb, p.v_st, p.v_sh, p.num_blocks, p.nh, c.head_dim, c.block_size, bf16, tokens, d->workspace))
    return fail(MAK_E_INVALID, "%s: the cache's strides make no tensor map", name);
  if (many) return launch_paged_tc(p, c.head_dim, bf16, name, k, v, space.plan, st);
  if (c.head_dim == 64) return bf16 ? launch_rows<64, true>(p, k, v, name, st) : launch_rows<64, false>(p, k, v, name, st);
  return bf16 ? launch_rows<128, true>(p, k, v, name, st) : launch_rows<128, false>(p, k, v, name, st);
}
