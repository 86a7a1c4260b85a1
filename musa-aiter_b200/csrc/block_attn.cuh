// Attention over a block-scaled 8-bit cache: the parts that the kernel for few
// rows and the kernel for many rows share.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace mak {

struct BlockAttnParams {
  const uint8_t* key;
  const uint8_t* value;
  const float* key_scale;
  const float* value_scale;
  int64_t k_sb, k_sh, v_sb, v_sh;          // bytes
  int64_t ks_sb, ks_sh, vs_sb, vs_sh;      // elements
  const int32_t* tables;
  const int32_t* ctx_lens;
  const int32_t* starts;  // null: one row per sequence
  int64_t table_stride;
  int64_t num_blocks;
  const void* q;
  void* out;
  float* lse;
  int64_t q_sr, q_sh, o_sr, o_sh;
  int32_t num_seqs, max_blocks, num_rows;
  int32_t nh, group, bs_log2, q_bf16, causal, window;
  float scale_log2;  // scale * log2(e)
  int32_t* counters;
  float* partial;
};

// What a sequence's rows see.  first: the row index of its first row; rows: how
// many it has; ctx: its length, which positions are counted from even where the
// table holds less; lo..hi: tokens that at least one of them sees, hi within the table.
struct SeqView {
  int first, rows, ctx, lo, hi;
};

__device__ __forceinline__ SeqView seq_view(const BlockAttnParams& p, int s) {
  SeqView v;
  const int ctx = max(__ldg(p.ctx_lens + s), 0);
  const int room = p.max_blocks << p.bs_log2;
  int a = s, b = s + 1;
  if (p.starts != nullptr) {
    a = __ldg(p.starts + s);
    b = __ldg(p.starts + s + 1);
  }
  a = a < 0 ? 0 : a;
  b = b > p.num_rows ? p.num_rows : b;
  v.first = a;
  v.rows = b > a ? b - a : 0;
  v.ctx = ctx;
  v.hi = min(ctx, room);
  const int before = ctx - v.rows;  // the first row's position
  v.lo = p.window > 0 && before >= p.window ? before - p.window + 1 : 0;
  return v;
}

// Tokens [lo, hi) that row i of the sequence sees.
__device__ __forceinline__ void row_range(const BlockAttnParams& p, const SeqView& v, int i, int* lo, int* hi) {
  const int pos = v.ctx - v.rows + i;
  *hi = p.causal ? max(min(pos + 1, v.hi), 0) : v.hi;
  *lo = p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;  // compared first: the difference alone may leave 32 bits
}

// Two 8-bit codes (low / high half of w as b0, b1 pairs) to two f16: every int8
// and every finite E4M3 value is exact in f16.
template <int CODE>
__device__ __forceinline__ void codes4_to_f16(uint32_t w, uint32_t* lo, uint32_t* hi) {
  if constexpr (CODE == MAK_CODE_INT8) {
    // 0x6400 | u is 1024 + u in f16, u = code + 128
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
    *lo = *reinterpret_cast<const uint32_t*>(&x);
    *hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(*lo), "=r"(*hi)
        : "r"(w));
  }
}

// Bit 7 of each byte of w that is an E4M3 NaN (0x7f or 0xff).
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Once per device: shared memory for a kernel's blocks.
constexpr int kMaxDevices = 64;
template <typename K>
int prepare_kernel(K kernel, int bytes, bool (&ready)[kMaxDevices]) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && device < kMaxDevices && ready[device]) return MAK_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return cuda_fail(e, "mak_block_attention");
  }
  if (device < kMaxDevices) ready[device] = true;
  return MAK_OK;
}

// [num_blocks][num_heads][head_dim][block_size] bytes as boxes of one head of one block, lines of
// block_size bytes swizzled.
int cache_map(CUtensorMap* map, const uint8_t* base, int64_t sb, int64_t sh, int64_t num_blocks, int nh, int hd, int bs);

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two 32-bit operations in one instruction, each rounded as its scalar form.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n .reg .b64 w, x, y, z;\n mov.b64 w, {%2, %3};\n mov.b64 x, {%4, %5};\n mov.b64 y, {%6, %7};\n fma.rn.f32x2 z, w, x, y;\n"
      " mov.b64 {%0, %1}, z;\n}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace mak
