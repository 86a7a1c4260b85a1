// The attention weight that each cached token gathers: A[h, t] += sum over the rows that see token t, and over the query
// heads that share cache head h, of exp(scale q . k_t - lse), with the lse that the attention gave.
//
// Few rows: bound by reading K.  A warp takes 16 tokens of one sequence and head at a time (the same runs of all work for
// every warp as in the attention), keeps their K in shared memory and goes over the rows, 16 at a time; each token's sum
// has one writer, so results do not depend on timing.  Exponents are taken of scale s - lse in natural units, one
// rounding, which keeps a weight's error at that of its exponent.
//
// Measured, calls in a graph: 64 requests of 256 to 4096 tokens, one row, 8 cache heads of 128 in bfloat16 for 32 query heads
// 58 us (5.3 TB/s of the 6.5 that a plain copy has); 8 warps with longer rings took 78: a warp's way from a part's pages to
// its sums is latency, which more warps hide.
#include "paged_weights.cuh"
#include "tcgen05.cuh"

namespace mak {
namespace {

constexpr int kRows = 16;
constexpr int kStep = 16;
constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxGrid = 148;
constexpr int kMinRun = 2;
constexpr int kQueue = 16;  // parts between a warp's loads and its products, at most
constexpr float kLog2e = 1.4426950408889634f;

// Steps [ta, tb) of a (sequence, head) that a warp has.
struct Part {
  PagedSeq v;
  Span s;
  int seq, head, ta, tb;
};

template <int HD>
struct Smem {
  static constexpr int kStages = HD == 64 ? 6 : 3;
  static constexpr int kTileBytes = kStep * HD * 2;
  alignas(1024) uint8_t ring[kWarps][kStages][kTileBytes];  // HD / 64 pieces of [16][64], lines of 128 bytes swizzled
  alignas(16) float old[kWarps][kStages][kStep];            // sums so far
  uint64_t full[kWarps][kStages];
  Part queue[kWarps][kQueue];
  int64_t before[kThreads + 1];
  int64_t sums[kWarps];
  int gave_up;
};

__device__ __forceinline__ void copy4(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// Steps of a (sequence, head): the tokens that some row sees, or, where sums begin, all places of the row.
__device__ __forceinline__ Span all_rows(const PagedParams& p, const PagedSeq& v) {
  Span s = {};
  if (v.rows > 0) s = span_of<kStep>(p, v, 0, v.rows - 1);
  return s;
}
__device__ __forceinline__ int steps_of(const WeightParams& w, const PagedSeq& v, int s) {
  if (sum_row(w, s) < 0) return 0;
  return w.add ? all_rows(w.a, v).tiles : (w.max_tokens + kStep - 1) / kStep;
}

template <int HD, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) paged_weights_kernel(const __grid_constant__ WeightParams w, const __grid_constant__ CUtensorMap k_map) {
  constexpr int kStages = Smem<HD>::kStages, kTileBytes = Smem<HD>::kTileBytes;
  constexpr int kPieces = HD / 64, kPiece = kStep * 128;
  extern __shared__ __align__(1024) uint8_t raw[];
  Smem<HD>& sm = *reinterpret_cast<Smem<HD>*>(raw);
  const PagedParams& p = w.a;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  if (tid == 0) {
    sm.gave_up = 0;
    for (int i = 0; i < kWarps * kStages; ++i) mbar_init(&sm.full[0][0] + i, 1);
    mbar_init_fence();
  }
  pdl_wait();
  pdl_trigger();

  const int per = (p.num_seqs + kThreads - 1) / kThreads;
  const int s0 = min(tid * per, p.num_seqs), s1 = min(s0 + per, p.num_seqs);
  {
    int64_t mine = 0;
    for (int s = s0; s < s1; ++s) mine += static_cast<int64_t>(steps_of(w, paged_seq(p, s), s)) * p.nh;
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
    __syncthreads();
  }
  const int64_t total = sm.before[kThreads];
  int64_t run = (total + gridDim.x * kWarps - 1) / (gridDim.x * kWarps);
  if (run < kMinRun) run = kMinRun;
  int64_t left = (blockIdx.x * static_cast<int64_t>(kWarps) + warp) * run;  // begin, then steps that are left
  const int64_t end = min(left + run, total);
  if (left >= end) return;

  Part at;  // the part at hand
  int steps;
  {
    const int64_t begin = left;
    int lo = 0, n = kThreads;  // the last thread whose sequences begin at or before this warp's run
    while (n > 1) {
      const int step = (n + 31) >> 5, i = lo + lane * step;
      const uint32_t votes = __ballot_sync(0xffffffffu, i < lo + n && sm.before[min(i, kThreads)] <= begin);
      const int k = 31 - __clz(votes), last = lo + n;
      lo += k * step;
      n = min(step, last - lo);
    }
    int64_t first = sm.before[lo];
    at.seq = min(lo * per, p.num_seqs - 1);
    for (;;) {
      at.v = paged_seq(p, at.seq);
      steps = steps_of(w, at.v, at.seq);
      const int64_t work = static_cast<int64_t>(steps) * p.nh;
      if (begin < first + work) break;
      first += work;
      ++at.seq;
    }
    at.s = all_rows(p, at.v);
    at.head = static_cast<int>((begin - first) / steps);
    at.ta = static_cast<int>((begin - first) - static_cast<int64_t>(at.head) * steps);
    left = end - begin;
    at.tb = static_cast<int>(min(at.ta + left, static_cast<int64_t>(steps)));
  }

  // ---- loads, some steps ahead of the products ---------------------------------------
  const uint32_t ring = shared_at(sm.ring[warp]);
  uint64_t* full = sm.full[warp];
  volatile int* gave_up = &sm.gave_up;
  Part* queue = sm.queue[warp];
  int parts_in = 0, left_in = 0, in = 0, stage_in = 0;
  int tok_in = 0, jump_at = 0, jump = 0, any_lo = 0, any_hi = 0, head_in = 0, next_id = -1;
  uint32_t there = 0;  // bit i: step i % 32 has a page
  bool ok = true;      // no wait has run out
  const int32_t* table_in = nullptr;
  const float* old_in = nullptr;
  const int inside = (1 << p.bs_log2) - 1;
  auto look = [&]() {  // id of the next step's page, looked at a step later
    const bool any = tok_in < any_hi && (tok_in + kStep > any_lo || tok_in < p.sinks);
    next_id = left_in > 0 && any ? __ldg(table_in + (tok_in >> p.bs_log2)) : -1;
  };
  auto enter = [&]() {
    __syncwarp();
    if (lane == 0) queue[parts_in % kQueue] = at;
    __syncwarp();
    ++parts_in;
    left_in = at.tb - at.ta, head_in = at.head, any_lo = at.s.any_lo, any_hi = at.v.rows > 0 ? at.s.any_hi : 0;
    tok_in = w.add ? tile_token<kStep>(at.s, at.ta) : at.ta * kStep;
    jump_at = w.add && at.ta < at.s.ns ? kStep * (at.s.ns - 1) : -1, jump = kStep * at.s.t0;
    table_in = p.tables + at.seq * p.table_stride;
    old_in = w.sums + sum_row(w, at.seq) * w.sum_sr + at.head * w.sum_sh;
    look();
    left -= left_in;
    // the part after it
    if (left > 0) {
      at.ta = 0;
      if (++at.head == p.nh) {
        at.head = 0;
        do {
          at.v = paged_seq(p, ++at.seq);
          steps = steps_of(w, at.v, at.seq);
        } while (steps == 0);
        at.s = all_rows(p, at.v);
      }
      at.tb = static_cast<int>(min(left, static_cast<int64_t>(steps)));
    }
  };
  bool more = true;
  auto load = [&]() {
    if (more && left_in == 0) {
      if (left > 0)
        enter();
      else
        more = false;
    }
    if (more) {
      const int page = __shfl_sync(0xffffffffu, next_id, 0), tok = __shfl_sync(0xffffffffu, tok_in, 0), head = __shfl_sync(0xffffffffu, head_in, 0);
      const bool has = ok && page >= 0 && page < p.num_blocks;
      there = (there & ~(1u << (in & 31))) | (has ? 1u << (in & 31) : 0u);
      if (w.add && lane < kStep) {
        const bool fits = tok + lane < w.max_tokens;
        copy4(shared_at(&sm.old[warp][stage_in][lane]), fits ? old_in + tok + lane : w.sums, fits ? 4 : 0);
      }
      tok_in = tok_in == jump_at ? jump : tok_in + kStep;
      --left_in;
      look();
      if (has && elect_one()) {
        const uint32_t to = ring + stage_in * kTileBytes;
        mbar_arrive_expect(full + stage_in, kTileBytes);
#pragma unroll
        for (int c = 0; c < kPieces; ++c) box_load(to + c * kPiece, &k_map, c * 64, head, tok & inside, page, full + stage_in);
      }
      __syncwarp();
      ++in;
      stage_in = stage_in + 1 == kStages ? 0 : stage_in + 1;
    }
    copies_commit();
  };
  enter();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load();

  // ---- products --------------------------------------------------------------------------
  const int r = lane >> 2, c2 = (lane & 3) * 2;
  int out = 0, stage = 0;
  uint32_t phases = 0;  // bit of a stage: the parity of its next phase
  for (int parts_out = 0; parts_out < parts_in; ++parts_out) {
    const Part& u = queue[parts_out % kQueue];
    const int seq = u.seq, head = u.head, ta = u.ta, tb = u.tb;
    const PagedSeq v = u.v;
    const Span span = u.s;
    const int64_t all = static_cast<int64_t>(v.rows) * p.group;
    float* dst = w.sums + sum_row(w, seq) * w.sum_sr + head * w.sum_sh;
    uint32_t qf[HD / 16][4];
    float lse[2];
    RowView see[2];
    auto fetch = [&](int64_t row0) {  // rows row0 + r and row0 + r + 8
      int64_t row_q[2];
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const int64_t row = min(row0 + r + 8 * z, all - 1);
        const int i = static_cast<int>(row / p.group);
        const int64_t h = static_cast<int64_t>(head) * p.group + (row - static_cast<int64_t>(i) * p.group);
        row_q[z] = (static_cast<int64_t>(v.first) + i) * p.q_sr + h * p.q_sh;
        lse[z] = __ldg(w.lse + (static_cast<int64_t>(v.first) + i) * w.lse_sr + h);
        see[z] = row_view(p, v, i);
        if (row0 + r + 8 * z >= all) see[z].hi = 0;
      }
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          qf[ks][e] = __ldg(reinterpret_cast<const uint32_t*>(p.q + row_q[e & 1] + ks * 16 + (e >> 1) * 8 + c2));
    };
    const bool one = all <= kRows;  // 16 rows or fewer stay in registers from step to step
    if (one && all > 0) fetch(0);
    for (int j = ta; j < tb; ++j, ++out) {
      load();
      if (w.add) copies_wait<kStages - 1>();
      const int tok = w.add ? tile_token<kStep>(span, j) : j * kStep;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};  // tokens c2, c2 + 1, c2 + 8, c2 + 9
      bool has = there >> (out & 31) & 1;
      if (has && !mbar_wait_warp(full + stage, phases >> stage & 1, gave_up)) {
        land<kStages>(full, out, in, there, phases);
        there = 0;
        has = ok = false;
      }
      if (has) {
        phases ^= 1u << stage;
        const uint32_t tile = ring + stage * kTileBytes;
        int64_t row0 = 0;
        if (!one && tok >= p.sinks) {  // rows before the first that sees a token of the step: the one at position tok
          const int64_t i = static_cast<int64_t>(tok) - (v.ctx - v.rows);
          if (i > 0) row0 = i * p.group / kRows * kRows;
        }
        for (; row0 < all; row0 += kRows) {
          if (!one) fetch(row0);
          // rows of a window that have all left the step behind end the walk
          if (p.window > 0 && tok >= p.sinks && __all_sync(0xffffffffu, see[0].lo >= tok + kStep && see[1].lo >= tok + kStep)) break;
          float s[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
          const int t = ((lane >> 4) << 3) + (lane & 7), half = (lane >> 3) & 1;
          const uint32_t line = tile + t * 128;
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            uint32_t b[4];
            load_matrix(line + (ks >> 2) * kPiece + (((2 * (ks & 3) + half) ^ (t & 7)) << 4), b);
            mma_16816<BF16>(s[0], qf[ks], b[0], b[1]);
            mma_16816<BF16>(s[1], qf[ks], b[2], b[3]);
          }
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            auto below = [](int k) { return k >= kStep ? 0xffffu : k <= 0 ? 0u : (1u << k) - 1u; };
            const uint32_t bits = below(see[z].hi - tok) & (~below(see[z].lo - tok) | below(p.sinks - tok));
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // tokens c2, c2 + 1, c2 + 8, c2 + 9
              const float x = exp2_near(fmaf(s[i >> 1][2 * z + (i & 1)], w.scale, -lse[z]) * kLog2e);
              sum[i] += bits >> (c2 + (i & 1) + 8 * (i >> 1)) & 1 ? x : 0.f;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 4);
          sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 8);
          sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 16);
        }
      }
      if (!ok) sum[0] = sum[1] = sum[2] = sum[3] = __uint_as_float(0x7fffffffu);  // a warp that gave up leaves NaN
      __syncwarp();
      if (r < 2) {  // eight lanes, two tokens each
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int k = r * 8 + c2 + e, t = tok + k;
          const float x = r == 0 ? sum[e] : sum[2 + e];
          const bool seen = t < span.any_hi && (t >= span.any_lo || t < p.sinks);
          if (t >= w.max_tokens || (w.add && !seen)) continue;
          dst[t] = w.add ? sm.old[warp][stage][k] + x : x;
        }
      }
      stage = stage + 1 == kStages ? 0 : stage + 1;
      __syncwarp();  // the stage is read
    }
  }
}

template <int HD, bool BF16>
int launch_few(const WeightParams& w, const CUtensorMap& k, const char* name, cudaStream_t st) {
  constexpr int kBytes = sizeof(Smem<HD>);
  static_assert(kBytes <= 227 * 1024, "shared memory of a block");
  static_assert(kQueue > Smem<HD>::kStages + 1, "parts in flight");
  const auto kernel = paged_weights_kernel<HD, BF16>;
  static bool ready[kPagedDevices] = {};
  if (int rc = paged_prepare(name, kernel, kBytes, ready)) return rc;
  const int sms = sm_count();
  return launch_pdl(name, kernel, dim3(sms < kMaxGrid ? sms : kMaxGrid), dim3(kThreads), kBytes, st, w, k);
}

}  // namespace
}  // namespace mak

using namespace mak;

extern "C" int mak_paged_weights(const mak_paged_weights_desc* d, void* stream) {
  const char* name = "mak_paged_weights";
  if (d == nullptr) return fail(MAK_E_INVALID, "%s: null descriptor", name);
  const mak_paged_cache_desc& c = d->cache;
  if (int rc = check_paged_cache(c, false, name)) return rc;
  if (d->num_q_heads <= 0 || d->num_q_heads % c.num_heads)
    return fail(MAK_E_INVALID, "%s: %d query heads over %d cache heads", name, d->num_q_heads, c.num_heads);
  if (d->window < 0 || d->sinks < 0) return fail(MAK_E_INVALID, "%s: negative window or sinks", name);
  if (!std::isfinite(d->scale * 1.4426950408889634f)) return fail(MAK_E_INVALID, "%s: the scale is not finite", name);
  if (d->max_tokens < 0 || d->max_tokens > 0x7fffffff - 16 || d->sum_rows < 0)
    return fail(MAK_E_INVALID, "%s: sums of %lld rows of %lld tokens", name, static_cast<long long>(d->sum_rows),
                static_cast<long long>(d->max_tokens));
  if (c.num_rows * d->num_q_heads / c.num_heads > 0x7fffffff - 256)
    return fail(MAK_E_UNSUPPORTED, "%s: rows times query heads of a cache head are a 32-bit count", name);
  if (c.num_seqs == 0 || d->max_tokens == 0 || d->sum_rows == 0) return MAK_OK;
  if (d->sums == nullptr || (c.num_rows > 0 && (d->q == nullptr || d->lse == nullptr)))
    return fail(MAK_E_INVALID, "%s: null q, lse or sums", name);
  if ((reinterpret_cast<uintptr_t>(d->q) & 15) || ((d->q_stride_row | d->q_stride_head) & 7))
    return fail(MAK_E_INVALID, "%s: q needs 16-byte aligned rows", name);
  WeightParams w = {};
  w.a = paged_params(c);
  w.a.q = static_cast<const uint16_t*>(d->q);
  w.a.q_sr = d->q_stride_row, w.a.q_sh = d->q_stride_head;
  w.a.group = d->num_q_heads / c.num_heads;
  w.a.window = d->window, w.a.sinks = d->window ? d->sinks : 0;
  w.a.scale_log2 = d->scale * kLog2e;
  w.lse = d->lse, w.lse_sr = d->lse_stride_row;
  w.sums = d->sums, w.sum_sr = d->sum_stride_row, w.sum_sh = d->sum_stride_head, w.sum_rows = d->sum_rows;
  w.rows = d->rows;
  w.max_tokens = static_cast<int32_t>(d->max_tokens), w.add = d->accumulate != 0;
  w.scale = d->scale;
  if (int rc = check_paged_workspace(d->workspace, d->workspace_bytes, name)) return rc;
  const PagedSpace space = paged_space(d->workspace);
  w.a.counters = space.counters, w.a.partial = space.partial;
  cudaStream_t st = as_stream(stream);
  const bool bf16 = c.dtype == MAK_DT_BF16;
  // Rows that share a cache head, on average; a group has to fit the chunks of rows.  Few / many in us, 8 cache heads of 128
  // with 4 query heads: 16 sequences of 4096 tokens 33 / 80 for 16 rows, 97 / 80 for 32, 133 / 85 for 48 (heads of 64: 25 / 73,
  // 58 / 73, 77 / 78); 64 of 512 19 / 44, 51 / 44; one of 4096 11 / 14, 20 / 14.  The average alone decides: 17 to 32 rows with heads
  // of 64 are taken up to a quarter slower than the other kernel would.
  const bool many = c.num_rows * w.a.group / c.num_seqs > 16 && c.num_seqs * 8 <= space.plan_bytes && weights_tc_fits(w);
  CUtensorMap k;
  if (!paged_map(&k, w.a.key, w.a.k_sb, w.a.k_st, w.a.k_sh, w.a.num_blocks, w.a.nh, c.head_dim, c.block_size, bf16, many ? c.block_size : kStep,
                 d->workspace))
    return fail(MAK_E_INVALID, "%s: the cache's strides make no tensor map", name);
  if (many) return launch_weights_tc(w, c.head_dim, bf16, name, k, static_cast<int64_t*>(space.plan), st);
  if (c.head_dim == 64) return bf16 ? launch_few<64, true>(w, k, name, st) : launch_few<64, false>(w, k, name, st);
  return bf16 ? launch_few<128, true>(w, k, name, st) : launch_few<128, false>(w, k, name, st);
}
