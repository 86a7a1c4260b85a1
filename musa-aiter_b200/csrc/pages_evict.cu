// Eviction: rows of a paged 16-bit cache shrink to `keep` tokens, each layer and head keeping its own, those of the
// largest sums (the attention weight that a token has gathered); the first `sinks` and the last `recent` tokens stay.
//
// Of n candidates the k largest in 32 bits: the sums become whole numbers in the same order, and the k-th largest is
// found 8 bits at a time from counts; of equal ones the first stay.  The kept tokens then move to places 0 .. keep - 1
// in their order.  A token moves to a place at or before its own, and every place before those still to be read is free,
// so one walk in rising order works in place: the block loads a batch of tokens, their K and V whole, ahead of the one that
// it stores.
//
// Bound by moving the kept tokens: rows of 256 bytes at places of their own, read and written.  A block per layer, row and
// head; a second small launch returns the pages.  Measured: 16 requests of 1500 to 4096 tokens to 1024, 8 layers, 8 heads of
// 128: 246 us (4.5 TB/s of 6.5 that a plain copy has), of which a block's search for its tokens is a seventh; one request of
// 30000 tokens to 2000, 4 heads of 64: 65 us, four blocks' search (two thirds) and walk; with 8192 tokens to a list, not 4096,
// the walk has its batches in one row (81 to 68 us, together with counts of each lane for equal first bytes).  128 registers a
// thread, of which 8 words are spilled.  Batches of 64
// tokens and 2 blocks on an SM were the best of those tried: 32 tokens 352 to 413 us, 40 415, 48 344, 128 480; slices of 64
// or 128 bytes of each token to a warp, which needs no barrier, 374 and 362.
#include "common.cuh"

namespace mak {
namespace {

constexpr int kPer = 8;  // tokens of a thread that are looked at together
// Tokens that move together, at most.
constexpr int list_of(int threads) { return 2 * kPer * threads; }
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
  int32_t num_rows, max_blocks, pages, bs, nh, max_tokens;
  int32_t keep, sinks, recent, layer0;
  int32_t cached;   // sums of a row are kept in shared memory
  int32_t bs_log2;  // -1: no power of 2
  uint16_t* key[kMaxLayers];
  uint16_t* value[kMaxLayers];
};

// 1: request i shrinks, 0: it holds no more than `keep`, -1: it is left alone.  All threads of the block ask together.
template <int kThreads>
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

template <int HD, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 256 ? 2 : 1) evict_kernel(const __grid_constant__ EvictParams p) {
  constexpr int kChunk = kPer * kThreads, kList = list_of(kThreads);
  extern __shared__ __align__(16) int32_t shared[];  // cleared 16 bytes at a time
  int32_t *const from = shared, *const to = shared + kList;
  float* const cache = reinterpret_cast<float*>(shared + 2 * kList);
  __shared__ int counts[256];
  __shared__ int warp_sums[kThreads / 32];
  __shared__ uint32_t prefix_s;
  __shared__ int left_s;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int head = blockIdx.x % p.nh, i = blockIdx.x / p.nh, layer = blockIdx.y;
  int len;
  const int what = decide<kThreads>(p, i, &len);
  if (head == 0 && layer == 0 && p.layer0 == 0 && tid == 0) p.state[i] = what;
  if (what <= 0) return;
  const int row = p.rows[i];
  float* sums = p.sums + (p.layer0 + layer) * p.sum_sl + row * p.sum_sr + head * p.sum_sh;
  const int lo = min(p.sinks, len), hi = max(len - p.recent, lo);  // candidates
  const int want = p.keep - (lo + len - hi);                       // of them, these many stay

  // ---- sums of the row, sixteen loads of a thread at a time -----------------
  if (p.cached) {
    for (int t0 = tid; t0 < len; t0 += 16 * kThreads) {
      float x[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = t0 + e * kThreads < len ? sums[t0 + e * kThreads] : 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (t0 + e * kThreads < len) cache[t0 + e * kThreads] = x[e];
    }
    __syncthreads();
  }
  const float* from_sums = p.cached ? cache : sums;

  // ---- the want-th largest: `prefix`, and how many equal to it stay -----------------
  // A lane has counts of its own, in a bank of its own, where the lists will be: most sums share their first byte.
  uint32_t prefix = 0;
  int left = want;
  static_assert(2 * kList >= 256 * 32 && kThreads >= 256, "counts of each lane");
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int j = tid; j < 256 * 32 / 4; j += kThreads) reinterpret_cast<int4*>(shared)[j] = make_int4(0, 0, 0, 0);
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int first = lo; first < hi; first += 8 * kThreads) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int t = first + tid + e * kThreads;
        x[e] = t < hi ? from_sums[t] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t o = order_of(x[e]);
        if (first + tid + e * kThreads < hi && (o & mask) == (prefix & mask)) atomicAdd(&shared[(o >> shift & 255) * 32 + lane], 1);
      }
    }
    __syncthreads();
    if (tid < 256) {
      int sum = 0;
#pragma unroll
      for (int c = 0; c < 32; ++c) sum += shared[tid * 32 + ((c + lane) & 31)];
      counts[tid] = sum;
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
  // A kept token is HD / 8 pieces of 16 bytes of K and as many of V.
  constexpr int kPieces = HD / 4, kDeep = 8, kBatch = kThreads * kDeep / kPieces;
  const int piece = tid % kPieces;
  const bool is_v = piece >= kPieces / 2;
  uint16_t* base = (is_v ? p.value[layer] : p.key[layer]) + head * (is_v ? p.v_sh : p.k_sh) + (is_v ? piece - kPieces / 2 : piece) * 8;
  const int64_t sb = is_v ? p.v_sb : p.k_sb, st = is_v ? p.v_st : p.k_st;
  auto page_of = [&](int t) { return p.bs_log2 >= 0 ? t >> p.bs_log2 : t / p.bs; };
  auto at = [&](int slot) {
    const int page = page_of(slot);
    return reinterpret_cast<uint4*>(base + page * sb + (slot - page * p.bs) * st);
  };
  int done = 0, ties = 0;  // tokens kept so far, numbers equal to the prefix so far
  int listed = 0;          // of the kept ones, those that have not moved yet
  for (int t0 = 0; t0 < len; t0 += kChunk) {
    bool stay[kPer], tie[kPer];
    float x[kPer];
    int n_stay = 0, n_tie = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int t = t0 + tid * kPer + e;
      x[e] = t < len ? from_sums[t] : 0.f;
      const uint32_t o = order_of(x[e]);
      const bool candidate = t >= lo && t < hi;
      tie[e] = candidate && o == prefix && want > 0;
      stay[e] = t < len && (!candidate || (o > prefix && want > 0));
      n_stay += stay[e], n_tie += tie[e];
    }
    // both counts before this thread: at most kChunk each
    int packed = n_stay | n_tie << 16, incl = packed;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    constexpr int kWarps = kThreads / 32;
    int of_warps = lane < kWarps ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, of_warps, o);
      if (lane >= o) of_warps += up;
    }
    const int all = __shfl_sync(0xffffffffu, of_warps, kWarps - 1), earlier = __shfl_sync(0xffffffffu, of_warps, warp ? warp - 1 : 0);
    const int before = incl - packed + (warp ? earlier : 0);
    int stays = before & 0xffff, tied = before >> 16;
    const int room = max(left - ties, 0);  // equal ones that still stay
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int t = t0 + tid * kPer + e;
      const bool tie_stays = tie[e] && tied < room;
      if (stay[e] || tie_stays) {
        const int mine = stays + min(tied, room), dst = done + mine;
        from[listed + mine] = t;
        if (dst != t) sums[dst] = x[e];  // at or before this chunk, which has been read
      }
      stays += stay[e], tied += tie[e];
    }
    const int some = (all & 0xffff) + min(all >> 16, room);
    done += some;
    listed += some;
    ties += all >> 16;
    __syncthreads();
    if (t0 + kChunk < len && listed + kChunk <= kList) continue;
    // tokens to slots, which stay below 2^31: the host has checked pages * block size
    const int kept = listed, first = done - listed;
    listed = 0;
    for (int k0 = tid; k0 < kept; k0 += 4 * kThreads) {  // each entry is one thread's
      int t[4], a[4], b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = k0 + e * kThreads;
        if (k >= kept) break;
        t[e] = from[k];
        a[e] = table[page_of(t[e])], b[e] = table[page_of(first + k)];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = k0 + e * kThreads, d = first + k;
        if (k >= kept) break;
        from[k] = d == t[e] ? -1 : a[e] * p.bs + t[e] - page_of(t[e]) * p.bs;
        to[k] = b[e] * p.bs + d - page_of(d) * p.bs;
      }
    }
    __syncthreads();
    // The block loads a batch ahead of the one that it stores: places are taken in rising order, none at or past a source
    // that is still to be read.
    uint4 v[2][kDeep];
    auto source = [&](int z0, int e) {
      const int k = z0 + (tid + e * kThreads) / kPieces;
      return k < kept ? from[k] : -1;
    };
    auto fetch = [&](int which, int z0) {
#pragma unroll
      for (int e = 0; e < kDeep; ++e) {
        const int src = source(z0, e);
        if (src >= 0) v[which][e] = *at(src);
      }
    };
    auto put = [&](int which, int z0) {
      __syncthreads();  // the batch is loaded
#pragma unroll
      for (int e = 0; e < kDeep; ++e)
        if (source(z0, e) >= 0) *at(to[z0 + (tid + e * kThreads) / kPieces]) = v[which][e];
    };
    fetch(0, 0);
    for (int z = 0; z < kept; z += 2 * kBatch) {
      fetch(1, z + kBatch);
      put(0, z);
      fetch(0, z + 2 * kBatch);
      put(1, z + kBatch);
    }
    __syncthreads();
  }
  for (int t = done + tid; t < p.max_tokens; t += kThreads) sums[t] = 0.f;
}

// Pages past the kept tokens return; lengths follow.
constexpr int kFinish = 256;
__global__ void __launch_bounds__(kFinish) evict_finish_kernel(int32_t* tables, int32_t* lens, int32_t* refs, const int32_t* rows,
                                                                const int32_t* state, int n, int64_t table_stride, int bs, int keep,
                                                                int32_t* left) {
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x;
  if (i == 0) {
    int alone = 0;
    for (int base = 0; base < n; base += kFinish) alone += __syncthreads_count(base + static_cast<int>(threadIdx.x) < n && state[base + threadIdx.x] < 0);
    if (threadIdx.x == 0) left[0] = alone;
  }
  if (state[i] <= 0) return;
  const int row = rows[i], len = lens[row];
  __syncthreads();
  if (threadIdx.x == 0) lens[row] = keep;
  for (int j = (keep + bs - 1) / bs + threadIdx.x; j <= (len - 1) / bs; j += kFinish) {
    atomicSub(refs + tables[row * table_stride + j], 1);
    tables[row * table_stride + j] = -1;
  }
}

constexpr int kMostCached = 40960;  // next to the lists
static_assert(kMostCached * 4 + list_of(512) * 8 + 2048 <= 227 * 1024, "shared memory of a block");
constexpr int kMaxDevices = 64;

template <int HD, int kThreads>
int launch_evict(const EvictParams& p, dim3 grid, int bytes, const char* name, cudaStream_t st) {
  const auto kernel = evict_kernel<HD, kThreads>;
  static bool ready[kMaxDevices] = {};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && (device >= kMaxDevices || !ready[device])) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostCached * 4 + list_of(kThreads) * 8);
    if (e == cudaSuccess && device < kMaxDevices) ready[device] = true;
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return cuda_fail(e, name);
  }
  return launch_pdl(name, kernel, grid, dim3(kThreads), bytes + list_of(kThreads) * 8, st, p);
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
  if (e->max_tokens < 0 || e->max_tokens > 0x7fffffff - 65536) return fail(MAK_E_INVALID, "%s: bad width of the sums", name);
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
  p.nh = e->num_heads;
  p.max_tokens = static_cast<int32_t>(e->max_tokens);
  p.bs_log2 = (p.bs & (p.bs - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(p.bs)) : -1;
  p.keep = e->keep, p.sinks = e->sinks, p.recent = e->recent;
  for (int64_t at = 0; at < e->num_layers; at += kMaxLayers) {
    const int64_t layers = e->num_layers - at < kMaxLayers ? e->num_layers - at : kMaxLayers;
    p.layer0 = static_cast<int32_t>(at);
    for (int64_t i = 0; i < layers; ++i) {
      p.key[i] = reinterpret_cast<uint16_t*>(e->keys[at + i]);
      p.value[i] = reinterpret_cast<uint16_t*>(e->values[at + i]);
    }
    const dim3 grid(static_cast<unsigned>(n * e->num_heads), static_cast<unsigned>(layers));
    // Rows of up to 8192 tokens leave room for two blocks on an SM; longer ones are kept where there are few blocks.
    const int64_t blocks = n * e->num_heads * layers;
    p.cached = e->max_tokens <= 8192 || (e->max_tokens <= kMostCached && blocks <= sm_count());
    const int bytes = p.cached ? static_cast<int>(e->max_tokens) * 4 : 0;
    // Few blocks: more threads for the search.
    const bool few = blocks <= sm_count();
    const int rc = e->head_dim == 64    ? (few ? launch_evict<64, 512>(p, grid, bytes, name, st) : launch_evict<64, 256>(p, grid, bytes, name, st))
                   : e->head_dim == 128 ? (few ? launch_evict<128, 512>(p, grid, bytes, name, st) : launch_evict<128, 256>(p, grid, bytes, name, st))
                                        : (few ? launch_evict<256, 512>(p, grid, bytes, name, st) : launch_evict<256, 256>(p, grid, bytes, name, st));
    if (rc != MAK_OK) return rc;
  }
  return launch_pdl(name, evict_finish_kernel, dim3(static_cast<unsigned>(n)), dim3(kFinish), 0, st, d->block_tables, d->context_lens,
                    d->ref_counts, rows, static_cast<const int32_t*>(state), static_cast<int>(n), d->table_stride, p.bs, p.keep, left);
}
