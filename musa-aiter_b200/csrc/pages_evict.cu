// Eviction: rows of a paged 16-bit cache shrink to `keep` tokens, each layer and head keeping its own, those of the
// largest sums (the attention weight that a token has gathered); the first `sinks` and the last `recent` tokens stay.
//
// Of n candidates the k largest in 32 bits: the sums become whole numbers in the same order, and the k-th largest is
// found 8 bits at a time from counts; of equal ones the first stay.  The kept tokens then move to places 0 .. keep - 1
// in their order.  A token moves to a place at or before its own, and every place before those still to be read is free,
// so one walk in rising order works in place: a warp owns some columns of all tokens and loads a batch before it stores.
//
// Bound by moving the kept tokens (HBM); a block per layer, row and head; a second small launch returns the pages.
#include "common.cuh"

namespace mak {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 1024;  // tokens looked at between two moves
constexpr int kMaxLayers = 128;
constexpr int kMaxRequests = 8192;

struct EvictParams {
  const int32_t* tables;
  const int32_t* lens;
  const int32_t* refs;
  const int32_t* rows;
  int32_t* state;  // per request: 1 shrinks, 0 has nothing to give, -1 left alone
  float* sums;
  int64_t table_stride;
  int64_t sum_sl, sum_sr, sum_sh;
  int64_t k_sb, k_st, k_sh, v_sb, v_st, v_sh;  // elements
  int32_t num_rows, max_blocks, pages, bs, n, nh, head_dim, max_tokens;
  int32_t keep, sinks, recent, layer0;
  uint16_t* key[kMaxLayers];
  uint16_t* value[kMaxLayers];
};

// 1: request i shrinks, 0: it holds no more than `keep`, -1: it is left alone.  All threads of the block ask together.
__device__ int decide(const EvictParams& p, int i, int* len_out) {
  const int row = p.rows[i];
  *len_out = 0;
  bool again = false;  // the same row earlier in the list
  for (int j = threadIdx.x; j < i; j += kThreads) again = again || p.rows[j] == row;
  if (__syncthreads_or(again) || row < 0 || row >= p.num_rows) return 0;
  const int len = p.lens[row];
  if (len <= p.keep) return 0;
  if (len > p.max_tokens || (len - 1) / p.bs >= p.max_blocks) return -1;
  const int held = (len - 1) / p.bs + 1, written = p.keep > 0 ? (p.keep - 1) / p.bs + 1 : 0;
  bool bad = false;
  for (int j = threadIdx.x; j < held; j += kThreads) {
    const int page = p.tables[row * p.table_stride + j];
    bad = bad || page < 0 || page >= p.pages || (j < written && p.refs[page] > 1);
  }
  *len_out = len;
  return __syncthreads_or(bad) ? -1 : 1;
}

// Whole numbers in the order of the sums: NaN and -inf are lowest, both zeros are equal.
__device__ __forceinline__ uint32_t order_of(float x) {
  x = x == x ? x + 0.f : -INFINITY;
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <int LANES>  // 16-byte pieces of a token that a warp moves
__global__ void __launch_bounds__(kThreads) evict_kernel(const __grid_constant__ EvictParams p) {
  __shared__ int counts[256];
  __shared__ int warp_sums[kThreads / 32];
  __shared__ int32_t from[kChunk], to[kChunk];
  __shared__ uint32_t prefix_s;
  __shared__ int left_s;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.x % p.nh, i = blockIdx.x / p.nh, layer = blockIdx.y;
  int len;
  const int what = decide(p, i, &len);
  if (head == 0 && layer == 0 && p.layer0 == 0 && tid == 0) p.state[i] = what;
  if (what <= 0) return;
  const int row = p.rows[i];
  float* sums = p.sums + (p.layer0 + layer) * p.sum_sl + row * p.sum_sr + head * p.sum_sh;
  const int lo = min(p.sinks, len), hi = max(len - p.recent, lo);  // candidates
  const int want = p.keep - (lo + len - hi);                       // of them, these many stay

  // ---- the want-th largest: `prefix`, and how many equal to it stay -----------------
  uint32_t prefix = 0;
  int left = want;
  for (int shift = 24; shift >= 0; shift -= 8) {
    counts[tid] = 0;
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int t = lo + tid; t < hi; t += kThreads) {
      const uint32_t x = order_of(sums[t]);
      if ((x & mask) == (prefix & mask)) atomicAdd(&counts[x >> shift & 255], 1);
    }
    __syncthreads();
    if (warp == 0) {  // the byte: the largest b with at least `left` numbers at or above it
      int mine[8], sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += mine[e] = counts[255 - (lane * 8 + e)];
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      int above = incl - sum;
      if (left > above && left <= incl) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (left > above && left <= above + mine[e]) {
            prefix_s = prefix | static_cast<uint32_t>(255 - (lane * 8 + e)) << shift;
            left_s = left - above;
          }
          above += mine[e];
        }
      }
      if (want <= 0 && lane == 0) prefix_s = 0xffffffffu, left_s = 0;
    }
    __syncthreads();
    prefix = prefix_s;
    left = left_s;
    __syncthreads();
  }

  // ---- the walk ------------------------------------------------------------------------
  const int32_t* table = p.tables + row * p.table_stride;
  const bool is_v = warp >= kThreads / 64;
  uint16_t* base = (is_v ? p.value[layer] : p.key[layer]) + head * (is_v ? p.v_sh : p.k_sh);
  const int64_t sb = is_v ? p.v_sb : p.k_sb, st = is_v ? p.v_st : p.k_st;
  const int piece = (warp % (kThreads / 64)) * LANES + lane % LANES;
  base += piece * 8;
  auto at = [&](int slot) {
    const int page = slot / p.bs;
    return reinterpret_cast<uint4*>(base + page * sb + (slot - page * p.bs) * st);
  };
  int done = 0, ties = 0;  // tokens kept so far, numbers equal to the prefix so far
  constexpr int kPer = kChunk / kThreads;
  for (int t0 = 0; t0 < len; t0 += kChunk) {
    bool stay[kPer], tie[kPer];
    float x[kPer];
    int n_stay = 0, n_tie = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int t = t0 + tid * kPer + e;
      x[e] = t < len ? sums[t] : 0.f;
      const uint32_t o = order_of(x[e]);
      const bool candidate = t >= lo && t < hi;
      tie[e] = candidate && o == prefix && want > 0;
      stay[e] = t < len && (!candidate || (o > prefix && want > 0));
      n_stay += stay[e], n_tie += tie[e];
    }
    // both counts before this thread: at most 1024 each
    int packed = n_stay | n_tie << 16, incl = packed;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int before = incl - packed, all = 0;
#pragma unroll
    for (int z = 0; z < kThreads / 32; ++z) {
      if (z < warp) before += warp_sums[z];
      all += warp_sums[z];
    }
    int stays = before & 0xffff, tied = before >> 16;
    const int room = max(left - ties, 0);  // equal ones that still stay
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int t = t0 + tid * kPer + e;
      const bool tie_stays = tie[e] && tied < room;
      if (stay[e] || tie_stays) {
        const int mine = stays + min(tied, room), dst = done + mine;
        // slots stay below 2^31: the host has checked pages * block size
        from[mine] = dst == t ? -1 : table[t / p.bs] * p.bs + t % p.bs;
        to[mine] = table[dst / p.bs] * p.bs + dst % p.bs;
        if (dst != t) sums[dst] = x[e];  // at or before this chunk, which has been read
      }
      stays += stay[e], tied += tie[e];
    }
    const int kept = (all & 0xffff) + min(all >> 16, room);
    __syncthreads();
    constexpr int kTokens = 32 / LANES, kDeep = 8;
    for (int z = lane / LANES; z < ((kept + kTokens - 1) / kTokens) * kTokens; z += kTokens * kDeep) {
      uint4 v[kDeep];
      int32_t src[kDeep];
#pragma unroll
      for (int e = 0; e < kDeep; ++e) {
        const int k = z + e * kTokens;
        src[e] = k < kept ? from[k] : -1;
        if (src[e] >= 0) v[e] = *at(src[e]);
      }
      __syncwarp();
#pragma unroll
      for (int e = 0; e < kDeep; ++e)
        if (src[e] >= 0) *at(to[z + e * kTokens]) = v[e];
      __syncwarp();
    }
    done += kept;
    ties += all >> 16;
    __syncthreads();
  }
  for (int t = done + tid; t < p.max_tokens; t += kThreads) sums[t] = 0.f;
}

// Pages past the kept tokens return; lengths follow.
__global__ void __launch_bounds__(kThreads) evict_finish_kernel(int32_t* tables, int32_t* lens, int32_t* refs, const int32_t* rows,
                                                                const int32_t* state, int n, int64_t table_stride, int bs, int keep,
                                                                int32_t* left) {
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x;
  if (i == 0) {
    int alone = 0;
    for (int base = 0; base < n; base += kThreads) alone += __syncthreads_count(base + static_cast<int>(threadIdx.x) < n && state[base + threadIdx.x] < 0);
    if (threadIdx.x == 0) left[0] = alone;
  }
  if (state[i] <= 0) return;
  const int row = rows[i], len = lens[row];
  __syncthreads();
  if (threadIdx.x == 0) lens[row] = keep;
  for (int j = (keep + bs - 1) / bs + threadIdx.x; j <= (len - 1) / bs; j += kThreads) {
    atomicSub(refs + tables[row * table_stride + j], 1);
    tables[row * table_stride + j] = -1;
  }
}

}  // namespace
}  // namespace mak

using namespace mak;

extern "C" int mak_pages_evict(const mak_pages_desc* d, const mak_evict_desc* e, const int32_t* rows, int64_t n, int32_t* left, int32_t* state,
                               void* stream) {
  const char* name = "mak_pages_evict";
  if (d == nullptr || e == nullptr) return fail(MAK_E_INVALID, "%s: null descriptor", name);
  if (e->head_dim != 64 && e->head_dim != 128 && e->head_dim != 256)
    return fail(MAK_E_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256, got %d", name, e->head_dim);
  if (d->num_rows < 0 || d->max_blocks < 0 || d->num_pages < 0 || n < 0 || e->num_layers < 0 || e->num_heads <= 0 || d->block_size <= 0)
    return fail(MAK_E_INVALID, "%s: negative size", name);
  if (d->num_rows > 0x7fffffff || d->max_blocks > 0x7fffffff / d->block_size || d->num_pages > 0x7fffffff / d->block_size || n > kMaxRequests)
    return fail(MAK_E_UNSUPPORTED, "%s: rows, tokens of a row and slots of a pool are 32-bit counts, requests at most %d", name, kMaxRequests);
  if (e->keep < 1 || e->sinks < 0 || e->recent < 0 || static_cast<int64_t>(e->sinks) + e->recent > e->keep)
    return fail(MAK_E_INVALID, "%s: keep must be at least 1 and sinks + recent", name);
  if (e->max_tokens < 0 || e->max_tokens > 0x7fffffff - kChunk) return fail(MAK_E_INVALID, "%s: bad width of the sums", name);
  if (left == nullptr || (n > 0 && (rows == nullptr || state == nullptr))) return fail(MAK_E_INVALID, "%s: null rows, state or result", name);
  if (n > 0 && d->num_rows > 0 && (d->block_tables == nullptr || d->context_lens == nullptr))
    return fail(MAK_E_INVALID, "%s: null block_tables or context_lens", name);
  if (d->num_pages > 0 && d->ref_counts == nullptr) return fail(MAK_E_INVALID, "%s: null ref_counts", name);
  if (e->num_layers > 0 && (e->keys == nullptr || e->values == nullptr || e->sums == nullptr)) return fail(MAK_E_INVALID, "%s: null cache or sums", name);
  cudaStream_t st = as_stream(stream);
  if (n == 0 || e->num_layers == 0) {
    const cudaError_t rc = cudaMemsetAsync(left, 0, 4, st);
    return rc == cudaSuccess ? MAK_OK : cuda_fail(rc, name);
  }
  if (n * e->num_heads > 0x7fffffff) return fail(MAK_E_UNSUPPORTED, "%s: too many heads", name);
  uint64_t bits = 0;
  for (int64_t i = 0; i < e->num_layers; ++i) bits |= e->keys[i] | e->values[i];
  const uint64_t strides = static_cast<uint64_t>(e->key_stride_block | e->key_stride_token | e->key_stride_head | e->value_stride_block |
                                                 e->value_stride_token | e->value_stride_head);
  if ((bits & 15) || (strides & 7)) return fail(MAK_E_INVALID, "%s: caches need 16-byte aligned addresses and strides", name);
  EvictParams p = {};
  p.tables = d->block_tables, p.lens = d->context_lens, p.refs = d->ref_counts, p.rows = rows, p.state = state;
  p.sums = e->sums;
  p.table_stride = d->table_stride;
  p.sum_sl = e->sum_stride_layer, p.sum_sr = e->sum_stride_row, p.sum_sh = e->sum_stride_head;
  p.k_sb = e->key_stride_block, p.k_st = e->key_stride_token, p.k_sh = e->key_stride_head;
  p.v_sb = e->value_stride_block, p.v_st = e->value_stride_token, p.v_sh = e->value_stride_head;
  p.num_rows = static_cast<int32_t>(d->num_rows), p.max_blocks = static_cast<int32_t>(d->max_blocks);
  p.pages = static_cast<int32_t>(d->num_pages), p.bs = static_cast<int32_t>(d->block_size);
  p.n = static_cast<int32_t>(n), p.nh = e->num_heads, p.head_dim = e->head_dim;
  p.max_tokens = static_cast<int32_t>(e->max_tokens);
  p.keep = e->keep, p.sinks = e->sinks, p.recent = e->recent;
  for (int64_t at = 0; at < e->num_layers; at += kMaxLayers) {
    const int64_t layers = e->num_layers - at < kMaxLayers ? e->num_layers - at : kMaxLayers;
    p.layer0 = static_cast<int32_t>(at);
    for (int64_t i = 0; i < layers; ++i) {
      p.key[i] = reinterpret_cast<uint16_t*>(e->keys[at + i]);
      p.value[i] = reinterpret_cast<uint16_t*>(e->values[at + i]);
    }
    const dim3 grid(static_cast<unsigned>(n * e->num_heads), static_cast<unsigned>(layers));
    const auto kernel = e->head_dim == 64 ? evict_kernel<2> : e->head_dim == 128 ? evict_kernel<4> : evict_kernel<8>;
    if (int rc = launch_pdl(name, kernel, grid, dim3(kThreads), 0, st, p)) return rc;
  }
  return launch_pdl(name, evict_finish_kernel, dim3(static_cast<unsigned>(n)), dim3(kThreads), 0, st, d->block_tables, d->context_lens,
                    d->ref_counts, rows, static_cast<const int32_t*>(state), static_cast<int>(n), d->table_stride, p.bs, p.keep, left);
}
