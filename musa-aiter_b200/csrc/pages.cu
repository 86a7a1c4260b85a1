// Pages of a cache: growing, forking, freeing, compacting and copying them, with
// block tables and reference counts kept on the device and no read-back.
//
// Two launches at most.  The first, one block, scans the reference counts and
// decides which pages are handed out or moved (lowest free index first, in the
// order of the requests: a prefix sum over the requests meets a prefix sum over
// the free pages); it is bound by the latency of its loads.  The second moves the
// pages' bytes over all planes and updates tables and counts; it is bound by HBM.
//
// Measured.  4096 pages of 16 tokens, 8 layers (8 heads of 128, codes and scales), with holes, made dense: 94 us, 5.2
// TB/s of a copy's 6.47; 16 requests forked 4 times each, part-filled last pages copied: 10.1 us, 3.1 TB/s, two launches
// and the scan's loads; 64 requests freed in a pool of 32768: 2 to 3.6 us, one launch's latency.  The scan is one block's
// and goes over the pool 8192 counts at a time, one turn after another: 64 rows grown into the last 200 free pages of 4096,
// 32768 and 262144: 7.5, 10.9 and 45.5 us; pools of those sizes with 1 % of holes made dense (32-byte pages): 5.8, 12.1
// and 77.5 us.
#include "common.cuh"

namespace mak {
namespace {

constexpr int kPlan = 1024;      // threads of a planning block
constexpr int kPerThread = 8;    // reference counts of one thread per step
constexpr int kMaxRequests = 4096;
constexpr int kMaxPagePlanes = 128;

struct Pages {
  int32_t* tables;
  int32_t* lens;
  int32_t* refs;
  int64_t table_stride;
  int32_t rows, max_blocks, pages, bs;
};

// Exclusive prefix sum over the block, and the total.
__device__ __forceinline__ int block_scan(int x, int* shared, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) shared[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int v = lane < warps ? shared[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    shared[lane] = v;
  }
  __syncthreads();
  *total = shared[31];
  const int before = warp ? shared[warp - 1] : 0;
  __syncthreads();
  return before + incl - x;
}

// Reference counts of this thread's kPerThread pages from `at`; pages past the end read as in use.
__device__ __forceinline__ void load_refs(const Pages& p, int64_t at, int32_t (&r)[kPerThread]) {
  if (at + kPerThread <= p.pages && (reinterpret_cast<uintptr_t>(p.refs) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < kPerThread; i += 4) {
      const int4 v = *reinterpret_cast<const int4*>(p.refs + at + i);
      r[i] = v.x, r[i + 1] = v.y, r[i + 2] = v.z, r[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) r[i] = at + i < p.pages ? p.refs[at + i] : 1;
  }
}

// Calls take(rank, page) for the first `need` free pages in index order; returns how many there were.
template <typename F>
__device__ int take_free(const Pages& p, int need, int* shared, F take) {
  int done = 0;
  for (int64_t base = 0; base < p.pages && done < need; base += kPlan * kPerThread) {
    const int64_t at = base + threadIdx.x * kPerThread;
    int32_t r[kPerThread];
    load_refs(p, at, r);
    int n = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) n += r[i] <= 0;
    int total;
    int rank = done + block_scan(n, shared, &total);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (r[i] <= 0) {
        if (rank < need) take(rank, static_cast<int32_t>(at + i));
        ++rank;
      }
    done += total;
  }
  return min(done, need);
}

__device__ __forceinline__ int valid_len(const Pages& p, int row) {
  const int64_t room = static_cast<int64_t>(p.max_blocks) * p.bs;
  const int n = p.lens[row];
  return n < 0 ? 0 : n > room ? static_cast<int>(room) : n;
}

// moves[i] / moves[n + i]: source and new page of request i, -1 where there is none.
__global__ void __launch_bounds__(kPlan) fork_plan_kernel(Pages p, const int32_t* parents, const int32_t* children, int n,
                                                          int32_t* missing, int first_call, int32_t* src, int32_t* dst) {
  __shared__ int shared[32];
  __shared__ int16_t who[kMaxRequests];
  pdl_wait();
  pdl_trigger();
  int need = 0;
  for (int base = 0; base < n; base += kPlan) {
    const int i = base + threadIdx.x;
    int from = -1;
    if (i < n) {
      const int row = parents[i], child = children[i];
      if (row >= 0 && row < p.rows && child >= 0 && child < p.rows) {
        const int len = valid_len(p, row);
        if (len % p.bs) from = p.tables[row * p.table_stride + len / p.bs];
        if (from >= p.pages) from = -1;
      }
      src[i] = from;
      dst[i] = -1;
    }
    int total;
    const int at = need + block_scan(from >= 0, shared, &total);
    if (from >= 0) who[at] = static_cast<int16_t>(i);
    need += total;
  }
  __syncthreads();
  const int got = take_free(p, need, shared, [&](int rank, int32_t page) { dst[who[rank]] = page; });
  if (threadIdx.x == 0) missing[0] = (first_call ? 0 : missing[0]) + need - got;
}

// Rows' new pages go straight into their tables.
__global__ void __launch_bounds__(kPlan) grow_kernel(Pages p, const int32_t* rows, const int32_t* more, int n, int32_t* missing,
                                                     int first_call) {
  __shared__ int shared[32];
  __shared__ int before[kMaxRequests + 1];  // pages that the requests before i need
  __shared__ int lost;
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x == 0) lost = 0;
  int need = 0;
  for (int base = 0; base < n; base += kPlan) {
    const int i = base + threadIdx.x;
    int want = 0;
    if (i < n) {
      const int row = rows[i];
      if (row >= 0 && row < p.rows && more[i] > 0) {
        const int64_t len = valid_len(p, row);
        const int64_t end = min(len + more[i], static_cast<int64_t>(p.max_blocks) * p.bs);
        want = static_cast<int>((end + p.bs - 1) / p.bs - (len + p.bs - 1) / p.bs);
      }
    }
    int total;
    const int at = need + block_scan(want, shared, &total);
    if (i < n) before[i] = at;
    need += total;
  }
  if (threadIdx.x == 0) before[n] = need;
  __syncthreads();
  const int got = take_free(p, need, shared, [&](int rank, int32_t page) {
    int lo = 0, hi = n;  // the last i with before[i] <= rank
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= rank)
        lo = mid;
      else
        hi = mid;
    }
    const int row = rows[lo];
    const int old = (valid_len(p, row) + p.bs - 1) / p.bs;
    p.tables[row * p.table_stride + old + (rank - before[lo])] = page;
    p.refs[page] = 1;
  });
  __syncthreads();
  int short_of = 0;
  for (int i = threadIdx.x; i < n; i += kPlan) {
    const int row = rows[i];
    if (row < 0 || row >= p.rows || more[i] <= 0) continue;
    const int64_t len = valid_len(p, row);
    const int64_t old = (len + p.bs - 1) / p.bs;
    const int64_t given = max(0, min(before[i + 1], got) - before[i]);
    const int64_t end = min(len + more[i], (old + given) * p.bs);
    p.lens[row] = static_cast<int32_t>(end);
    short_of += static_cast<int>(len + more[i] - end);
  }
  atomicAdd(&lost, short_of);
  __syncthreads();
  if (threadIdx.x == 0) missing[0] = (first_call ? 0 : missing[0]) + lost;
}

__global__ void __launch_bounds__(256) free_kernel(Pages p, const int32_t* rows) {
  pdl_wait();
  pdl_trigger();
  const int row = rows[blockIdx.x];
  if (row < 0 || row >= p.rows) return;
  // Each entry is taken by one thread only, so a row named twice loses its pages once.
  for (int j = threadIdx.x; j < p.max_blocks; j += blockDim.x) {
    const int page = atomicExch(p.tables + row * p.table_stride + j, -1);
    if (page >= 0 && page < p.pages) atomicSub(p.refs + page, 1);
  }
  if (threadIdx.x == 0) p.lens[row] = 0;
}

// scratch: src[pages], dst[pages], rank[pages] (of a page that moves), count, live.
__global__ void __launch_bounds__(kPlan) compact_plan_kernel(Pages p, int32_t* live_out, int32_t* scratch) {
  __shared__ int shared[32];
  __shared__ int below;
  pdl_wait();
  pdl_trigger();
  int mine = 0;
  for (int64_t at = threadIdx.x * kPerThread; at < p.pages; at += kPlan * kPerThread) {
    int32_t r[kPerThread];
    load_refs(p, at, r);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) mine += at + i < p.pages && r[i] > 0;
  }
  int live;
  block_scan(mine, shared, &live);
  if (threadIdx.x == 0) below = live;
  __syncthreads();
  int32_t *src = scratch, *dst = scratch + p.pages, *rank = scratch + 2 * static_cast<int64_t>(p.pages);
  int seen = 0;
  for (int64_t base = 0; base < p.pages; base += kPlan * kPerThread) {
    const int64_t at = base + threadIdx.x * kPerThread;
    int32_t r[kPerThread];
    load_refs(p, at, r);
    int n = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) n += at + i < p.pages && r[i] > 0;
    int total;
    int before = seen + block_scan(n, shared, &total);
    // pages in use below index `live` stay; the first page past them learns how many those are
    if (live >= at && live < at + kPerThread) {
      int k = before;
      for (int i = 0; i < kPerThread; ++i)
        if (at + i < live) k += r[i] > 0;
      below = k;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int64_t page = at + i;
      if (page >= p.pages) break;
      if (r[i] > 0) {
        if (page >= live) {
          src[before - below] = static_cast<int32_t>(page);
          rank[page] = before - below;
        }
        ++before;
      } else if (page < live) {
        dst[page - before] = static_cast<int32_t>(page);
      }
    }
    seen += total;
  }
  if (threadIdx.x == 0) {
    scratch[3 * static_cast<int64_t>(p.pages)] = live - below;
    scratch[3 * static_cast<int64_t>(p.pages) + 1] = live;
    live_out[0] = live;
  }
}

// The planes of one launch in the order they are moved: first those of at least a chunk, each in
// whole chunks of 256 vectors (its last one part empty), then the small ones, their vectors end to
// end.  A warp moves a chunk of one page at a time, 8 vectors per lane in flight, so a page's
// indexes cost one look-up per 4 KB.
constexpr int kChunk = 256;
struct Planes {
  uint64_t ptr[kMaxPagePlanes];
  int64_t stride[kMaxPagePlanes];
  uint32_t vecs[kMaxPagePlanes];   // of one page
  uint32_t start[kMaxPagePlanes];  // big: first chunk; small: first vector
  int32_t big, planes;
  uint32_t big_chunks, small_vecs, chunks;
};

enum { kCopyOnly = 0, kFork = 1, kCompact = 2 };

struct Moves {
  const int32_t* src;
  const int32_t* dst;
  const int32_t* count;  // number of pairs on the device, or null: n
  int32_t n;
  int64_t pages;
  int32_t table_blocks;  // leading blocks that update tables and counts instead
};

// The last plane in [lo, hi) that starts at or before x.
__device__ __forceinline__ int plane_of(const Planes& pl, int lo, int hi, uint32_t x) {
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pl.start[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <typename V>
__device__ __forceinline__ void move_pages(const Planes& pl, const Moves& mv, int n, int64_t warp, int64_t warps) {
  const int lane = threadIdx.x & 31;
  const int64_t units = static_cast<int64_t>(n) * pl.chunks;
  for (int64_t u = warp; u < units; u += warps) {
    const int64_t pair = (units >> 32) == 0 ? static_cast<uint32_t>(u) / pl.chunks : u / pl.chunks;
    const uint32_t chunk = static_cast<uint32_t>(u - pair * pl.chunks);
    const int s = __ldg(mv.src + pair), d = __ldg(mv.dst + pair);
    if (s < 0 || d < 0 || s >= mv.pages || d >= mv.pages) continue;
    V x[8];
    if (chunk < pl.big_chunks) {
      const int i = plane_of(pl, 0, pl.big, chunk);
      const uint32_t first = (chunk - pl.start[i]) * kChunk, left = pl.vecs[i] - first;
      const V* from = reinterpret_cast<const V*>(pl.ptr[i] + s * pl.stride[i]) + first;
      V* to = reinterpret_cast<V*>(pl.ptr[i] + d * pl.stride[i]) + first;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k * 32 + lane < left) x[k] = from[k * 32 + lane];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k * 32 + lane < left) to[k * 32 + lane] = x[k];
    } else {
      const uint32_t first = (chunk - pl.big_chunks) * kChunk;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t v = first + k * 32 + lane;
        if (v < pl.small_vecs) {
          const int i = plane_of(pl, pl.big, pl.planes, v);
          const uint32_t in = v - pl.start[i];
          reinterpret_cast<V*>(pl.ptr[i] + d * pl.stride[i])[in] = reinterpret_cast<const V*>(pl.ptr[i] + s * pl.stride[i])[in];
        }
      }
    }
  }
}

template <int MODE>
__device__ __forceinline__ void update_tables(const Moves& mv, const Pages& p, int n, const int32_t* parents, const int32_t* children) {
  if constexpr (MODE == kFork) {
    for (int i = blockIdx.x; i < n; i += mv.table_blocks) {
      const int row = parents[i], child = children[i];
      if (row < 0 || row >= p.rows || child < 0 || child >= p.rows) continue;
      const int len = valid_len(p, row);
      const int full = len / p.bs, fresh = mv.dst[i];
      for (int j = threadIdx.x; j < p.max_blocks; j += blockDim.x) {
        int page = -1;
        if (j < full) {
          page = p.tables[row * p.table_stride + j];
          if (page >= 0 && page < p.pages) atomicAdd(p.refs + page, 1);
        } else if (j == full) {
          page = fresh;
        }
        p.tables[child * p.table_stride + j] = page;
      }
      if (threadIdx.x == 0) {
        if (fresh >= 0) p.refs[fresh] = 1;
        p.lens[child] = fresh < 0 ? full * p.bs : len;
      }
    }
  }
  if constexpr (MODE == kCompact) {
    const int32_t* rank = mv.src + 2 * mv.pages;
    const int live = mv.count[1];
    const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const int64_t step = static_cast<int64_t>(mv.table_blocks) * blockDim.x;
    for (int64_t i = first; i < static_cast<int64_t>(p.rows) * p.max_blocks; i += step) {
      int32_t* e = p.tables + (i / p.max_blocks) * p.table_stride + i % p.max_blocks;
      const int page = *e;
      // an entry that names a page nobody counts is left alone
      if (page >= live && page < p.pages && static_cast<uint32_t>(rank[page]) < static_cast<uint32_t>(n) && mv.src[rank[page]] == page)
        *e = mv.dst[rank[page]];
    }
    for (int64_t i = first; i < n; i += step) {
      p.refs[mv.dst[i]] = p.refs[mv.src[i]];
      p.refs[mv.src[i]] = 0;
    }
  }
}

template <int MODE, typename V>
__global__ void __launch_bounds__(256) pages_move_kernel(const __grid_constant__ Planes pl, const __grid_constant__ Moves mv,
                                                         const __grid_constant__ Pages p, const int32_t* parents,
                                                         const int32_t* children) {
  pdl_wait();
  pdl_trigger();
  const int n = mv.count != nullptr ? *mv.count : mv.n;
  if (static_cast<int>(blockIdx.x) < mv.table_blocks) {
    update_tables<MODE>(mv, p, n, parents, children);
    return;
  }
  const int64_t warps = static_cast<int64_t>(gridDim.x - mv.table_blocks) * 8;
  move_pages<V>(pl, mv, n, static_cast<int64_t>(blockIdx.x - mv.table_blocks) * 8 + (threadIdx.x >> 5), warps);
}

int check_pages(const mak_pages_desc* d, const char* name, Pages* out) {
  if (d == nullptr) return fail(MAK_E_INVALID, "%s: null descriptor", name);
  if (d->num_rows < 0 || d->max_blocks < 0 || d->num_pages < 0 || d->block_size <= 0)
    return fail(MAK_E_INVALID, "%s: bad size", name);
  if (d->num_rows > 0x7fffffff || d->num_pages > 0x3fffffff || d->block_size > 0x7fffffff ||
      d->max_blocks > 0x7fffffff / d->block_size)
    return fail(MAK_E_UNSUPPORTED, "%s: rows, pages and tokens of a row are 32-bit counts", name);
  if ((d->num_rows && d->max_blocks && d->block_tables == nullptr) || (d->num_pages && d->ref_counts == nullptr))
    return fail(MAK_E_INVALID, "%s: null pointer", name);
  *out = Pages{d->block_tables, d->context_lens, d->ref_counts, d->table_stride, static_cast<int32_t>(d->num_rows),
               static_cast<int32_t>(d->max_blocks), static_cast<int32_t>(d->num_pages), static_cast<int32_t>(d->block_size)};
  return MAK_OK;
}

int check_planes(const mak_pages_planes* pl, const char* name) {
  if (pl == nullptr || pl->num_planes < 0 || (pl->num_planes && (!pl->ptrs || !pl->strides || !pl->sizes)))
    return fail(MAK_E_INVALID, "%s: bad planes", name);
  if (pl->num_planes > MAK_MAX_PLANES) return fail(MAK_E_UNSUPPORTED, "%s: over %d planes", name, MAK_MAX_PLANES);
  for (int64_t i = 0; i < pl->num_planes; ++i) {
    if (pl->sizes[i] < 0 || pl->sizes[i] > 0x7fffffff || (pl->sizes[i] && pl->ptrs[i] == 0) || pl->strides[i] < pl->sizes[i])
      return fail(MAK_E_INVALID, "%s: plane %lld has page size %lld, stride %lld", name, static_cast<long long>(i),
                  static_cast<long long>(pl->sizes[i]), static_cast<long long>(pl->strides[i]));
  }
  return MAK_OK;
}

template <int MODE, typename V>
int launch_move(const Planes& pl, Moves mv, const Pages& p, const int32_t* parents, const int32_t* children, int64_t most, bool tables,
                const char* name, cudaStream_t st) {
  const auto kernel = pages_move_kernel<MODE, V>;
  static int per_sm = 0;
  if (per_sm == 0) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 256, 0) != cudaSuccess || n <= 0) n = 1;
    per_sm = n;
  }
  const int64_t room = static_cast<int64_t>(per_sm) * sm_count();
  int64_t copy = (most * pl.chunks + 7) / 8;
  copy = copy < room ? copy : room;
  mv.table_blocks = 0;
  if (tables && MODE == kFork) mv.table_blocks = static_cast<int32_t>(most < 256 ? most : 256);
  if (tables && MODE == kCompact) {
    const int64_t entries = static_cast<int64_t>(p.rows) * p.max_blocks + most;
    mv.table_blocks = static_cast<int32_t>((entries + 1023) / 1024 < 64 ? (entries + 1023) / 1024 : 64);
  }
  if (copy + mv.table_blocks == 0) return MAK_OK;
  return launch_pdl(name, kernel, dim3(static_cast<unsigned>(copy + mv.table_blocks)), dim3(256), 0, st, pl, mv, p, parents, children);
}

// Moves all planes, those of one alignment (16, 4 or 1 bytes) and at most kMaxPagePlanes to a launch;
// the last launch also updates the tables.
template <int MODE>
int launch_moves(const mak_pages_planes* pl, const Moves& mv, const Pages& p, const int32_t* parents, const int32_t* children,
                 int64_t most, const char* name, cudaStream_t st) {
  static const int kWidths[3] = {16, 4, 1};
  int64_t left = 0;
  for (int64_t i = 0; i < pl->num_planes; ++i) left += pl->sizes[i] > 0;
  Planes a;
  a.big = a.planes = 0;
  a.big_chunks = a.small_vecs = a.chunks = 0;
  if (left == 0) return launch_move<MODE, uint4>(a, mv, p, parents, children, most, true, name, st);
  for (int w = 0; w < 3 && left > 0; ++w) {
    const int width = kWidths[w];
    auto fits = [&](int64_t i) {
      const uint64_t bits = pl->ptrs[i] | static_cast<uint64_t>(pl->strides[i]) | static_cast<uint64_t>(pl->sizes[i]);
      return pl->sizes[i] > 0 && ((bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : 1) == width;
    };
    int64_t at = 0;
    while (at < pl->num_planes) {
      int64_t end = at;
      int got = 0;
      for (; end < pl->num_planes && got < kMaxPagePlanes; ++end) got += fits(end);
      if (got == 0) break;
      a.planes = a.big = 0;
      a.big_chunks = a.small_vecs = 0;
      for (int big = 1; big >= 0; --big) {
        for (int64_t i = at; i < end; ++i) {
          const uint32_t vecs = static_cast<uint32_t>(pl->sizes[i] / width);
          if (!fits(i) || (vecs >= kChunk) != (big == 1)) continue;
          a.ptr[a.planes] = pl->ptrs[i];
          a.stride[a.planes] = pl->strides[i];
          a.vecs[a.planes] = vecs;
          a.start[a.planes] = big ? a.big_chunks : a.small_vecs;
          if (big)
            a.big_chunks += (vecs + kChunk - 1) / kChunk;
          else
            a.small_vecs += vecs;
          ++a.planes;
        }
        if (big) a.big = a.planes;
      }
      a.chunks = a.big_chunks + (a.small_vecs + kChunk - 1) / kChunk;
      left -= got;
      const bool tables = MODE != kCopyOnly && left == 0;
      int rc;
      if (width == 16)
        rc = launch_move<MODE, uint4>(a, mv, p, parents, children, most, tables, name, st);
      else if (width == 4)
        rc = launch_move<MODE, uint32_t>(a, mv, p, parents, children, most, tables, name, st);
      else
        rc = launch_move<MODE, uint8_t>(a, mv, p, parents, children, most, tables, name, st);
      if (rc) return rc;
      at = end;
    }
  }
  return MAK_OK;
}

}  // namespace
}  // namespace mak

using namespace mak;

extern "C" int mak_pages_fork(const mak_pages_desc* pages, const mak_pages_planes* planes, const int32_t* parents,
                              const int32_t* children, int64_t n, int32_t* missing, int32_t* moves, void* stream) {
  const char* name = "mak_pages_fork";
  Pages p;
  if (int rc = check_pages(pages, name, &p)) return rc;
  if (int rc = check_planes(planes, name)) return rc;
  if (n < 0 || n > 0x3fffffff || missing == nullptr || (n && (!parents || !children || !moves || !p.lens)))
    return fail(MAK_E_INVALID, "%s: bad requests", name);
  cudaStream_t st = as_stream(stream);
  for (int64_t at = 0; at < n || at == 0; at += kMaxRequests) {
    const int here = static_cast<int>(n - at < kMaxRequests ? n - at : kMaxRequests);
    int32_t *src = moves + at, *dst = moves + n + at;
    if (int rc = launch_pdl(name, fork_plan_kernel, dim3(1), dim3(kPlan), 0, st, p, parents + at, children + at, here, missing,
                            at == 0, src, dst))
      return rc;
    if (here == 0) break;
    const Moves mv{src, dst, nullptr, here, p.pages, 0};
    if (int rc = launch_moves<kFork>(planes, mv, p, parents + at, children + at, here, name, st)) return rc;
  }
  return MAK_OK;
}

extern "C" int mak_pages_grow(const mak_pages_desc* pages, const int32_t* rows, const int32_t* new_tokens, int64_t n,
                              int32_t* missing, void* stream) {
  const char* name = "mak_pages_grow";
  Pages p;
  if (int rc = check_pages(pages, name, &p)) return rc;
  if (n < 0 || n > 0x7fffffff || missing == nullptr || (n && (!rows || !new_tokens || !p.lens)))
    return fail(MAK_E_INVALID, "%s: bad requests", name);
  cudaStream_t st = as_stream(stream);
  for (int64_t at = 0; at < n || at == 0; at += kMaxRequests) {
    const int here = static_cast<int>(n - at < kMaxRequests ? n - at : kMaxRequests);
    if (int rc = launch_pdl(name, grow_kernel, dim3(1), dim3(kPlan), 0, st, p, rows + at, new_tokens + at, here, missing, at == 0))
      return rc;
  }
  return MAK_OK;
}

extern "C" int mak_pages_free(const mak_pages_desc* pages, const int32_t* rows, int64_t n, void* stream) {
  const char* name = "mak_pages_free";
  Pages p;
  if (int rc = check_pages(pages, name, &p)) return rc;
  if (n < 0 || n > 0x7fffffff || (n && (!rows || !p.lens))) return fail(MAK_E_INVALID, "%s: bad requests", name);
  if (n == 0) return MAK_OK;
  return launch_pdl(name, free_kernel, dim3(static_cast<unsigned>(n)), dim3(256), 0, as_stream(stream), p, rows);
}

extern "C" int mak_pages_compact(const mak_pages_desc* pages, const mak_pages_planes* planes, int32_t* live, int32_t* scratch,
                                 void* stream) {
  const char* name = "mak_pages_compact";
  Pages p;
  if (int rc = check_pages(pages, name, &p)) return rc;
  if (int rc = check_planes(planes, name)) return rc;
  if (live == nullptr || scratch == nullptr) return fail(MAK_E_INVALID, "%s: null pointer", name);
  cudaStream_t st = as_stream(stream);
  if (int rc = launch_pdl(name, compact_plan_kernel, dim3(1), dim3(kPlan), 0, st, p, live, scratch)) return rc;
  const Moves mv{scratch, scratch + p.pages, scratch + 3 * static_cast<int64_t>(p.pages), 0, p.pages, 0};
  return launch_moves<kCompact>(planes, mv, p, nullptr, nullptr, p.pages / 2 + 1, name, st);
}

extern "C" int mak_pages_copy(const mak_pages_planes* planes, int64_t num_pages, const int32_t* src, const int32_t* dst, int64_t n,
                              void* stream) {
  const char* name = "mak_pages_copy";
  if (int rc = check_planes(planes, name)) return rc;
  if (num_pages < 0 || num_pages > 0x3fffffff || n < 0 || n > 0x7fffffff || (n && (!src || !dst)))
    return fail(MAK_E_INVALID, "%s: bad requests", name);
  if (n == 0) return MAK_OK;
  const Moves mv{src, dst, nullptr, static_cast<int32_t>(n), num_pages, 0};
  return launch_moves<kCopyOnly>(planes, mv, Pages{}, nullptr, nullptr, n, name, as_stream(stream));
}
