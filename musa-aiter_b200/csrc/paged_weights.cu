// The attention weight that each cached token gathers: A[h, t] += sum over the rows that see token t, and over the query
// heads that share cache head h, of exp(scale q . k_t - lse), with the lse that the attention gave.
//
// Few rows: bound by reading K.  A warp takes 16 tokens of one sequence and head at a time (the same runs of all work for
// every warp as in the attention), keeps their K in shared memory and goes over the rows, 16 at a time; each token's sum
// has one writer, so results do not depend on timing.  Exponents are taken of scale s - lse in natural units, one
// rounding, which keeps a weight's error at that of its exponent.
#include "paged_weights.cuh"

namespace mak {
namespace {

constexpr int kRows = 16;
constexpr int kStep = 16;
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxGrid = 148;
constexpr int kMinRun = 2;
constexpr float kLog2e = 1.4426950408889634f;

template <int HD>
struct Smem {
  static constexpr int kStages = HD == 64 ? 8 : 4;
  static constexpr int kStage = kStep * HD * 2 + 64;  // K of a step, its sums so far
  alignas(128) uint8_t ring[kWarps][kStages][kStage];
  int64_t before[kThreads + 1];
  int64_t sums[kWarps];
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
__global__ void __launch_bounds__(kThreads, 1) paged_weights_kernel(const __grid_constant__ WeightParams w) {
  constexpr int kStages = Smem<HD>::kStages, kStage = Smem<HD>::kStage, kTileBytes = kStep * HD * 2;
  constexpr int kChunks = HD / 8, kCopies = kStep * kChunks / 32;
  extern __shared__ __align__(128) uint8_t raw[];
  Smem<HD>& sm = *reinterpret_cast<Smem<HD>*>(raw);
  const PagedParams& p = w.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
  const int64_t begin = (blockIdx.x * static_cast<int64_t>(kWarps) + warp) * run, end = min(begin + run, total);
  if (begin >= end) return;

  // A place in the run: sequence, head, step.
  struct Place {
    int seq, head, step, steps;
    PagedSeq v;
    Span s;
  };
  Place in;
  {
    int lo = 0, n = kThreads;  // the last thread whose sequences begin at or before this warp's run
    while (n > 1) {
      const int step = (n + 31) >> 5, at = lo + lane * step;
      const uint32_t votes = __ballot_sync(0xffffffffu, at < lo + n && sm.before[min(at, kThreads)] <= begin);
      const int k = 31 - __clz(votes), last = lo + n;
      lo += k * step;
      n = min(step, last - lo);
    }
    int64_t at = sm.before[lo];
    in.seq = min(lo * per, p.num_seqs - 1);
    for (;;) {
      in.v = paged_seq(p, in.seq);
      in.steps = steps_of(w, in.v, in.seq);
      const int64_t work = static_cast<int64_t>(in.steps) * p.nh;
      if (begin < at + work) break;
      at += work;
      ++in.seq;
    }
    in.s = all_rows(p, in.v);
    in.head = static_cast<int>((begin - at) / in.steps);
    in.step = static_cast<int>((begin - at) - static_cast<int64_t>(in.head) * in.steps);
  }
  auto advance = [&](Place& x) {
    if (++x.step < x.steps) return;
    x.step = 0;
    if (++x.head < p.nh) return;
    x.head = 0;
    do {
      if (++x.seq >= p.num_seqs) return;
      x.v = paged_seq(p, x.seq);
      x.steps = steps_of(w, x.v, x.seq);
    } while (x.steps == 0);
    x.s = all_rows(p, x.v);
  };
  auto token = [&](const Place& x) { return w.add ? tile_token<kStep>(x.s, x.step) : x.step * kStep; };
  auto any = [&](const Place& x, int tok) {  // whether some row may see a token of the step
    return x.s.tiles > 0 && tok < x.s.any_hi && (tok + kStep > x.s.any_lo || tok < p.sinks);
  };
  auto look = [&](const Place& x) {
    const int tok = token(x);
    return any(x, tok) ? page_of(p, p.tables + x.seq * p.table_stride, tok) : -1;
  };

  const uint32_t ring = shared_at(sm.ring[warp]);
  Place out = in;
  int page_in = look(in);
  int64_t copied = begin;
  uint32_t there = 0;
  auto copy = [&]() {
    if (copied < end) {
      const uint32_t slot = static_cast<uint32_t>(copied - begin);
      there = (there & ~(1u << (slot & 31))) | (page_in >= 0 ? 1u << (slot & 31) : 0u);
      const int tok0 = token(in);
      const uint32_t to = ring + (slot % kStages) * kStage;
      if (w.add && lane < kStep) {
        const bool has = tok0 + lane < w.max_tokens;
        const float* old = w.sums + sum_row(w, in.seq) * w.sum_sr + in.head * w.sum_sh + tok0 + lane;
        copy4(to + kTileBytes + lane * 4, has ? old : w.sums, has ? 4 : 0);
      }
      if (page_in >= 0) {
        const int64_t off = tok0 & ((1 << p.bs_log2) - 1);
        const uint16_t* k = p.key + page_in * p.k_sb + off * p.k_st + in.head * p.k_sh;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int t = (i * 32 + lane) / kChunks, c = (i * 32 + lane) % kChunks;
          copy16(to + t * (HD * 2) + ((c ^ (t & 7)) << 4), k + t * p.k_st + c * 8, 16);
        }
      }
      if (++copied < end) {
        advance(in);
        page_in = look(in);
      }
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) copy();

  const int r = lane >> 2, c2 = (lane & 3) * 2;
  uint32_t qf[HD / 16][4];
  float lse[2];
  RowView see[2];
  auto fetch = [&](int64_t row0, int64_t all) {  // rows row0 + r and row0 + r + 8
    int64_t row_q[2];
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int64_t row = min(row0 + r + 8 * z, all - 1);
      const int i = static_cast<int>(row / p.group);
      const int64_t h = static_cast<int64_t>(out.head) * p.group + (row - static_cast<int64_t>(i) * p.group);
      row_q[z] = (static_cast<int64_t>(out.v.first) + i) * p.q_sr + h * p.q_sh;
      lse[z] = __ldg(w.lse + (static_cast<int64_t>(out.v.first) + i) * w.lse_sr + h);
      see[z] = row_view(p, out.v, i);
      if (row0 + r + 8 * z >= all) see[z].hi = 0;
    }
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        qf[ks][e] = __ldg(reinterpret_cast<const uint32_t*>(p.q + row_q[e & 1] + ks * 16 + (e >> 1) * 8 + c2));
  };
  bool fresh = true;  // another sequence or head
  for (int64_t at = begin; at < end; ++at) {
    copy();
    copies_wait<kStages - 1>();
    __syncwarp();
    const uint32_t slot = static_cast<uint32_t>(at - begin);
    const uint32_t tile = ring + (slot % kStages) * kStage;
    const int tok = token(out);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};  // tokens c2, c2 + 1, c2 + 8, c2 + 9
    if (there >> (slot & 31) & 1) {
      const int64_t all = static_cast<int64_t>(out.v.rows) * p.group;
      int64_t row0 = 0;
      if (tok >= p.sinks) {  // rows before the first that sees a token of the step: the one at position tok
        const int64_t i = static_cast<int64_t>(tok) - (out.v.ctx - out.v.rows);
        if (i > 0) row0 = i * p.group / kRows * kRows;
      }
      for (; row0 < all; row0 += kRows) {
        // 16 rows or fewer stay in registers from step to step
        if (fresh || all > kRows) fetch(row0, all);
        fresh = false;
        // rows of a window that have all left the step behind end the walk
        if (p.window > 0 && tok >= p.sinks && __all_sync(0xffffffffu, see[0].lo >= tok + kStep && see[1].lo >= tok + kStep)) break;
        float s[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
        const int t = ((lane >> 4) << 3) + (lane & 7), half = (lane >> 3) & 1;
        const uint32_t line = tile + t * (HD * 2);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          uint32_t b[4];
          load_matrix(line + (((2 * ks + half) ^ (t & 7)) << 4), b);
          mma_16816<BF16>(s[0], qf[ks], b[0], b[1]);
          mma_16816<BF16>(s[1], qf[ks], b[2], b[3]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int z = e >> 1, mine = tok + i * 8 + c2 + (e & 1);
            const bool seen = mine < see[z].hi && (mine >= see[z].lo || mine < p.sinks);
            const float x = exp2_near(fmaf(s[i][e], w.scale, -lse[z]) * kLog2e);
            sum[i * 2 + (e & 1)] += seen ? x : 0.f;
          }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 4);
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 8);
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 16);
      }
    }
    if (r < 2) {  // eight lanes, two tokens each
      float* dst = w.sums + sum_row(w, out.seq) * w.sum_sr + out.head * w.sum_sh;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int t = tok + r * 8 + c2 + e;
        const float x = r == 0 ? sum[e] : sum[2 + e];
        const bool seen = t < out.s.any_hi && (t >= out.s.any_lo || t < p.sinks);
        if (t >= w.max_tokens || (w.add && !seen)) continue;
        float old = 0.f;
        if (w.add) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(old) : "r"(tile + kTileBytes + (t - tok) * 4) : "memory");
        dst[t] = old + x;
      }
    }
    __syncwarp();  // the stage is read
    if (at + 1 < end) {
      const int seq = out.seq, head = out.head;
      advance(out);
      fresh = fresh || out.seq != seq || out.head != head;
    }
  }
  copies_wait<0>();
}

template <int HD, bool BF16>
int launch_few(const WeightParams& w, const char* name, cudaStream_t st) {
  constexpr int kBytes = sizeof(Smem<HD>);
  static_assert(kBytes <= 227 * 1024, "shared memory of a block");
  const auto kernel = paged_weights_kernel<HD, BF16>;
  static bool ready[kPagedDevices] = {};
  if (int rc = paged_prepare(name, kernel, kBytes, ready)) return rc;
  const int sms = sm_count();
  return launch_pdl(name, kernel, dim3(sms < kMaxGrid ? sms : kMaxGrid), dim3(kThreads), kBytes, st, w);
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
  if (d->max_tokens < 0 || d->max_tokens > 0x7fffffff - 16 || d->sum_rows < 0)
    return fail(MAK_E_INVALID, "%s: sums of %lld rows of %lld tokens", name, static_cast<long long>(d->sum_rows),
                static_cast<long long>(d->max_tokens));
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
  if (d->workspace == nullptr || d->workspace_bytes < mak_paged_attention_workspace_bytes())
    return fail(MAK_E_WORKSPACE, "%s: workspace missing or too small", name);
  const PagedSpace space = paged_space(d->workspace);
  w.a.counters = space.counters, w.a.partial = space.partial;
  cudaStream_t st = as_stream(stream);
  const bool bf16 = c.dtype == MAK_DT_BF16;
  // Rows that share a cache head, on average.
  if (c.num_rows * w.a.group / c.num_seqs > 32 && c.num_seqs * 8 <= space.plan_bytes) {
    bool taken = false;
    const int rc = launch_weights_tc(w, c.head_dim, bf16, name, static_cast<int64_t*>(space.plan), st, &taken);
    if (rc != MAK_OK || taken) return rc;
  }
  if (c.head_dim == 64) return bf16 ? launch_few<64, true>(w, name, st) : launch_few<64, false>(w, name, st);
  return bf16 ? launch_few<128, true>(w, name, st) : launch_few<128, false>(w, name, st);
}
