// Attention over a paged 16-bit cache [num_blocks][block_size][num_heads][head_dim]: what a row sees, and the
// parts that the kernels for few rows, for many rows and for accumulated weights share.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "common.cuh"
#include "tcgen05.cuh"

namespace mak {

struct PagedParams {
  const uint16_t* key;
  const uint16_t* value;
  int64_t k_sb, k_st, k_sh, v_sb, v_st, v_sh;  // elements: block, token, head
  const int32_t* tables;
  const int32_t* ctx_lens;
  const int32_t* starts;   // null: one row per sequence
  const int32_t* parents;  // tree of drafted tokens, or null
  int64_t table_stride;
  int64_t num_blocks;
  const uint16_t* q;
  void* out;
  float* lse;
  int64_t q_sr, q_sh, o_sr, o_sh;
  int32_t num_seqs, max_blocks, num_rows;
  int32_t nh, group, bs_log2, window, sinks;
  float scale_log2;  // scale * log2(e)
  int32_t* counters;
  float* partial;
};

// A sequence in a call.  first: the row index of its first row; rows: how many it has; ctx: its length, which positions
// are counted from even where the table holds less; room: the tokens that the table holds.
struct PagedSeq {
  int first, rows, ctx, room;
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int s) {
  PagedSeq v;
  int a = s, b = s + 1;
  if (p.starts != nullptr) {
    a = __ldg(p.starts + s);
    b = __ldg(p.starts + s + 1);
  }
  a = a < 0 ? 0 : a;
  b = b > p.num_rows ? p.num_rows : b;
  v.first = a;
  v.rows = b > a ? b - a : 0;
  v.ctx = max(__ldg(p.ctx_lens + s), 0);
  v.room = min(v.ctx, p.max_blocks << p.bs_log2);
  return v;
}

// Row i of a sequence sees the tokens t < hi with t >= lo or t < sinks; in a tree, of those at or past `base`, only the
// ones that it continues.
struct RowView {
  int lo, hi;
};
__device__ __forceinline__ RowView row_view(const PagedParams& p, const PagedSeq& v, int i) {
  const int pos = v.ctx - v.rows + i;
  RowView r;
  r.hi = max(min(pos + 1, v.room), 0);
  r.lo = p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;  // compared first: the difference alone may leave 32 bits
  return r;
}

// Bit e: row i of a tree sees token t0 + e, e < 32.  Its line of parents is walked down to t0: a parent is an earlier row
// of the sequence, anything else ends the line.
__device__ __forceinline__ uint32_t tree_bits(const PagedParams& p, const PagedSeq& v, int i, int t0) {
  const int base = v.ctx - v.rows;
  uint32_t bits = t0 >= base ? 0u : base - t0 >= 32 ? 0xffffffffu : (1u << (base - t0)) - 1u;
  for (int a = base - t0 >= 32 ? -1 : i; a >= 0 && base + a >= t0;) {
    const int e = base + a - t0;
    if (e < 32) bits |= 1u << e;
    const int up = __ldg(p.parents + v.first + a);
    a = up < a ? up : -1;
  }
  const int left = v.room - t0;
  return left >= 32 ? bits : left <= 0 ? 0u : bits & ((1u << left) - 1u);
}

// Tokens that the rows i0 .. i1 of a sequence see, as tiles of T tokens: `ns` tiles from 0 on (the first tokens that stay
// visible), then tiles from t0 on; `tiles` in all.  Tokens below any_lo and not below `sinks`, and from any_hi on, nobody
// sees; between all_lo and all_hi, and below all_sinks, everyone does.
struct Span {
  int any_lo, any_hi, all_lo, all_hi, all_sinks, ns, t0, tiles;
};
template <int T>
__device__ __forceinline__ Span span_of(const PagedParams& p, const PagedSeq& v, int i0, int i1) {
  Span s;
  const RowView a = row_view(p, v, i0), b = row_view(p, v, i1);
  s.any_lo = a.lo, s.any_hi = b.hi;
  s.all_lo = b.lo, s.all_hi = a.hi;
  if (p.parents != nullptr) {
    s.any_hi = v.room;
    s.all_hi = max(min(v.ctx - v.rows, v.room), 0);
  }
  s.all_sinks = min(p.sinks, s.all_hi);
  s.t0 = s.any_lo / T;
  s.ns = (min(p.sinks, s.any_hi) + T - 1) / T;
  s.tiles = s.ns;
  if (s.any_hi > s.any_lo) {  // else all windows lie past the table's tokens, and the first tokens are all there is
    s.ns = min(s.ns, s.t0);
    s.tiles = s.ns + (s.any_hi + T - 1) / T - s.t0;
  }
  return s;
}
// First token of tile j of a span.
template <int T>
__device__ __forceinline__ int tile_token(const Span& s, int j) {
  return T * (j < s.ns ? j : s.t0 + j - s.ns);
}
template <int T>
__device__ __forceinline__ bool tile_whole(const Span& s, int tok) {
  return tok + T <= s.all_sinks || (tok >= s.all_lo && tok + T <= s.all_hi);
}

// Page of a token, -1 where there is none.
__device__ __forceinline__ int page_of(const PagedParams& p, const int32_t* table, int tok) {
  const int page = __ldg(table + (tok >> p.bs_log2));
  return page >= 0 && page < p.num_blocks ? page : -1;
}

__device__ __forceinline__ float exp2_near(float x) {  // 2^x, 2 units in the last place
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x for x <= 0 as a factor of sums that may hold an infinite one, which stays infinite: not 0, however far apart maxima are.
// 2^-126 of a sum counts for nothing, and of an empty one is 0.
__device__ __forceinline__ float shrink(float x) { return fmaxf(exp2_near(x), 0x1p-126f); }

template <bool BF16>
__device__ __forceinline__ uint32_t pack_two(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// The same, cut off instead of rounded.
template <bool BF16>
__device__ __forceinline__ uint32_t cut_two(float a, float b) {
  uint32_t w;
  if constexpr (BF16)
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
  else
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
  return w;
}
template <bool BF16>
__device__ __forceinline__ float2 unpack_two(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ float to_float(uint16_t h) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
  return __half2float(__ushort_as_half(h));
}
// Whether either of two 16-bit values is infinite or NaN.
template <bool BF16>
__device__ __forceinline__ bool odd_two(uint32_t w) {
  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}

// Once per device: shared memory for a kernel's blocks.
constexpr int kPagedDevices = 64;
template <typename K>
int paged_prepare(const char* name, K kernel, int bytes, bool (&ready)[kPagedDevices]) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && device < kPagedDevices && ready[device]) return MAK_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return cuda_fail(e, name);
  }
  if (device < kPagedDevices) ready[device] = true;
  return MAK_OK;
}

// ---- 16 x 8 x 16 products on fragments in registers --------------------------------------------------------
__device__ __forceinline__ uint32_t shared_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void load_matrix(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void load_matrix_t(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Box of a 4-dimensional tensor map; a coordinate outside fills zeros.
__device__ __forceinline__ void box_load(uint32_t to, const void* map, int x, int y, int z, int v, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(v), "r"(shared_at(bar))
      : "memory");
}
// A warp's wait for the loads of steps [from, to) that have been issued (`there`, a bit for each of the last 32) ends when they
// have landed, or with its limit: after a wait that ran out, so that none lands later.
template <int STAGES>
__device__ __forceinline__ void land(uint64_t* full, int from, int to, uint32_t there, uint32_t phases) {
  for (int k = from; k < to; ++k)
    if (there >> (k & 31) & 1)
      for (uint32_t i = 0; i < kWaitLimit && !mbar_try(full + k % STAGES, phases >> (k % STAGES) & 1); ++i) {
      }
  __syncwarp();
}
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(is));
  return is != 0;
}

}  // namespace mak
