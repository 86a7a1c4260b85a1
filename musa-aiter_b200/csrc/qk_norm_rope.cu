// Norms of queries and keys for each head with the position rotation in the same pass, and their gradient.
//
// n = x (mean x^2 + eps)^-1/2 over a head, y = R (n w): R turns pairs of the first rot_dim columns by the angle of the
// token's position.  Backward, with g = R^T grad: dw = sum g n over tokens and heads, h = g w,
// dx = r (h - n mean(h n)), r = (mean x^2 + eps)^-1/2.  All in 32 bits, results rounded once.
//
// Bound by HBM: forward reads x and writes y, backward reads x and grad and writes dx.  A head is held by hd / 16 lanes
// (rounded up to a power of two), 16 columns each as two 16-byte pieces that hold both halves of their pairs, so the
// rotation needs no exchange and the norm log2(lanes) of them.  A block has heads of q or of k alone: the weights, and in
// the backward pass the sums of dw, stay in registers; the angles stay over several heads of a token.
//
// Measured, 16411 tokens, 32 + 8 heads of 128 in bfloat16: forward 72 us (4.7 TB/s of the 6.5 that a plain copy has), backward
// 101 us (5.0 TB/s) and 7 us for the sums over the blocks; 64 tokens 3.9 us, one launch's latency.  Heads of q and k mixed in a
// block, weights read anew for each: 260 us for all three, 180 now.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace mak {
namespace {

constexpr int kThreads = 256;

struct NormParams {
  mak_qk_norm_rope_desc d;
  int32_t lanes;                // of a head: a power of two
  int32_t per_group;            // a token's heads in groups
  int32_t q_groups, k_groups;
  int32_t q_blocks, k_blocks;   // the first ones have heads of q
  int32_t wide_angles;          // rows of the tables begin on 16 bytes
};

template <int DT>
__device__ __forceinline__ void unpack8(const uint4& r, float* x) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == MAK_DT_BF16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float* x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == MAK_DT_BF16) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    } else {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Columns of a lane: two pieces of eight.  Split pairs: 8 j and its partners half a rotation further; pairs next to one
// another, and columns that stay: 16 j and the eight behind.
template <bool INTER>
__device__ __forceinline__ void columns(const mak_qk_norm_rope_desc& d, int j, int* a, int* b, bool* turns) {
  *turns = 16 * j < d.rot_dim;
  *a = !INTER && *turns ? 8 * j : 16 * j;
  *b = !INTER && *turns ? d.rot_dim / 2 + 8 * j : 16 * j + 8;
}

// cos and sin of the lane's eight pairs; 1 and 0 where it turns nothing.
template <bool INTER>
__device__ __forceinline__ void angles(const NormParams& p, int64_t t, int j, bool turns, float (&c)[8], float (&s)[8]) {
  const mak_qk_norm_rope_desc& d = p.d;
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
  if (!turns) return;
  const int64_t pos = load_index(d.positions, d.pos_dtype == MAK_DT_I64, t);
  if (pos < 0 || pos >= d.max_positions) return;
  const float *cs = d.cos + pos * d.cos_stride + 8 * j, *sn = d.sin + pos * d.sin_stride + 8 * j;
  if (p.wide_angles) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(cs)), b = __ldg(reinterpret_cast<const float4*>(cs) + 1);
    const float4 e = __ldg(reinterpret_cast<const float4*>(sn)), f = __ldg(reinterpret_cast<const float4*>(sn) + 1);
    c[0] = a.x, c[1] = a.y, c[2] = a.z, c[3] = a.w, c[4] = b.x, c[5] = b.y, c[6] = b.z, c[7] = b.w;
    s[0] = e.x, s[1] = e.y, s[2] = e.z, s[3] = e.w, s[4] = f.x, s[5] = f.y, s[6] = f.z, s[7] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __ldg(cs + i), s[i] = __ldg(sn + i);
  }
}
// Pairs of the lane's 16 values: (i, 8 + i) split, (2 i, 2 i + 1) next to one another.  `sign` -1: back.
template <bool INTER>
__device__ __forceinline__ void turn(float (&x)[16], const float (&c)[8], const float (&s)[8], float sign) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int u = INTER ? 2 * i : i, v = INTER ? 2 * i + 1 : 8 + i;
    const float a = x[u], b = x[v], sn = sign * s[i];
    x[u] = a * c[i] - b * sn;
    x[v] = a * sn + b * c[i];
  }
}
__device__ __forceinline__ void weights(const mak_qk_norm_rope_desc& d, const void* w, int a, int b, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int at = i < 8 ? a + i : b + i - 8;
    x[i] = d.weight_dtype == MAK_DT_F32    ? __ldg(static_cast<const float*>(w) + at)
           : d.weight_dtype == MAK_DT_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[at])
                                           : __half2float(static_cast<const __half*>(w)[at]);
  }
}
__device__ __forceinline__ float over_lanes(float x, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <int DT, bool INTER, bool BACK>
__global__ void __launch_bounds__(kThreads, 2) qk_norm_rope_kernel(const __grid_constant__ NormParams p) {
  const mak_qk_norm_rope_desc& d = p.d;
  extern __shared__ float shared[];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & (p.lanes - 1), per_block = kThreads / p.lanes;
  int ca, cb;
  bool turns;
  columns<INTER>(d, lane, &ca, &cb, &turns);
  const bool on = 16 * lane < d.head_dim;
  const bool isq = static_cast<int>(blockIdx.x) < p.q_blocks;
  const int block = isq ? blockIdx.x : blockIdx.x - p.q_blocks, blocks = isq ? p.q_blocks : p.k_blocks;
  const int groups = isq ? p.q_groups : p.k_groups, all_heads = isq ? d.q_heads : d.k_heads;
  const int64_t st = isq ? d.q_stride_token : d.k_stride_token, sh = isq ? d.q_stride_head : d.k_stride_head;
  const int64_t ot = isq ? d.qo_stride_token : d.ko_stride_token, oh = isq ? d.qo_stride_head : d.ko_stride_head;
  const int64_t gt = isq ? d.gq_stride_token : d.gk_stride_token, gh = isq ? d.gq_stride_head : d.gk_stride_head;
  const uint16_t* x0 = static_cast<const uint16_t*>(isq ? d.q : d.k);
  const uint16_t* g0 = static_cast<const uint16_t*>(isq ? d.grad_q : d.grad_k);
  uint16_t* o0 = static_cast<uint16_t*>(isq ? d.q_out : d.k_out);
  const int64_t items = d.tokens * groups;
  float w[16], dw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = dw[i] = 0.f;
  if (on && items > 0) weights(d, isq ? d.q_weight : d.k_weight, ca, cb, w);
  const float inv = 1.f / d.head_dim;
  // lanes without columns, and items past the last, take part in the sums with zeros
  for (int64_t first = static_cast<int64_t>(block) * per_block; first < items; first += static_cast<int64_t>(blocks) * per_block) {
    const int64_t item = min(first + threadIdx.x / p.lanes, items - 1);
    const bool live = on && first + threadIdx.x / p.lanes < items;
    const int64_t t = (items >> 31) == 0 ? static_cast<uint32_t>(item) / static_cast<uint32_t>(groups) : item / groups;
    const int h0 = static_cast<int>(item - t * groups) * p.per_group, heads = min(p.per_group, all_heads - h0);
    const uint16_t* src = x0 + t * st + h0 * sh;
    const uint16_t* grad = g0 + t * gt + h0 * gh;
    uint16_t* dst = o0 + t * ot + h0 * oh;
    float c[8], s[8];
    if (live) angles<INTER>(p, t, lane, turns, c, s);
    constexpr int kDeep = BACK ? 2 : 4;
    for (int h = 0; h < p.per_group; h += kDeep) {
      uint4 xa[kDeep], xb[kDeep], ga[kDeep], gb[kDeep];
#pragma unroll
      for (int z = 0; z < kDeep; ++z) {
        xa[z] = xb[z] = ga[z] = gb[z] = make_uint4(0, 0, 0, 0);
        if (!live || h + z >= heads) continue;
        xa[z] = __ldcs(reinterpret_cast<const uint4*>(src + (h + z) * sh + ca));
        xb[z] = __ldcs(reinterpret_cast<const uint4*>(src + (h + z) * sh + cb));
        if constexpr (BACK) {
          ga[z] = __ldcs(reinterpret_cast<const uint4*>(grad + (h + z) * gh + ca));
          gb[z] = __ldcs(reinterpret_cast<const uint4*>(grad + (h + z) * gh + cb));
        }
      }
#pragma unroll
      for (int z = 0; z < kDeep; ++z) {
        float x[16];
        unpack8<DT>(xa[z], x);
        unpack8<DT>(xb[z], x + 8);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum = fmaf(x[i], x[i], sum);
        const float r = rsqrtf(over_lanes(sum, p.lanes) * inv + d.eps);
        const bool mine = live && h + z < heads;
        if constexpr (!BACK) {
          if (!mine) continue;
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = x[i] * r * w[i];
          turn<INTER>(x, c, s, 1.f);
        } else {
          float g[16];
          unpack8<DT>(ga[z], g);
          unpack8<DT>(gb[z], g + 8);
          float along = 0.f;
          if (mine) {
            turn<INTER>(g, c, s, -1.f);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              x[i] *= r;
              dw[i] = fmaf(g[i], x[i], dw[i]);
              g[i] *= w[i];
              along = fmaf(g[i], x[i], along);
            }
          }
          along = over_lanes(along, p.lanes) * inv;
          if (!mine) continue;
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = r * (g[i] - x[i] * along);
        }
        __stcs(reinterpret_cast<uint4*>(dst + (h + z) * oh + ca), pack8<DT>(x));
        __stcs(reinterpret_cast<uint4*>(dst + (h + z) * oh + cb), pack8<DT>(x + 8));
      }
    }
  }
  if constexpr (BACK) {
    // the block's sums of dw, in a fixed order
#pragma unroll
    for (int i = 0; i < 16; ++i) shared[threadIdx.x * 16 + i] = dw[i];
    __syncthreads();
    for (int at = threadIdx.x; at < p.lanes * 16; at += kThreads) {
      const int j = at >> 4, i = at & 15;
      if (16 * j >= d.head_dim) continue;
      float sum = 0.f;
      for (int b = 0; b < per_block; ++b) sum += shared[(b * p.lanes + j) * 16 + i];
      int a, b;
      bool t;
      columns<INTER>(d, j, &a, &b, &t);
      d.partial[static_cast<int64_t>(blockIdx.x) * d.head_dim + (i < 8 ? a + i : b + i - 8)] = sum;
    }
  }
}

// dw: the blocks' sums in a fixed order, a warp per column.
__global__ void __launch_bounds__(kThreads) qk_norm_sum_kernel(const __grid_constant__ NormParams p) {
  const mak_qk_norm_rope_desc& d = p.d;
  pdl_wait();
  pdl_trigger();
  const int at = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (at >= 2 * d.head_dim) return;
  const bool isq = at < d.head_dim;
  const int col = isq ? at : at - d.head_dim, end = isq ? p.q_blocks : p.q_blocks + p.k_blocks;
  float sum = 0.f;
#pragma unroll 8
  for (int b = (isq ? 0 : p.q_blocks) + lane; b < end; b += 32) sum += d.partial[static_cast<int64_t>(b) * d.head_dim + col];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane) return;
  void* dst = isq ? d.grad_q_weight : d.grad_k_weight;
  if (d.weight_dtype == MAK_DT_F32)
    static_cast<float*>(dst)[col] = sum;
  else if (d.weight_dtype == MAK_DT_BF16)
    static_cast<__nv_bfloat16*>(dst)[col] = __float2bfloat16_rn(sum);
  else
    static_cast<__half*>(dst)[col] = __float2half_rn(sum);
}

constexpr int kMaxBlocks = 148 * 2;  // of a backward pass

template <int DT, bool INTER>
int launch(const NormParams& p, bool back, const char* name, cudaStream_t st) {
  const int smem = back ? kThreads * 16 * 4 : 0;
  if (!back) return launch_pdl(name, qk_norm_rope_kernel<DT, INTER, false>, dim3(p.q_blocks + p.k_blocks), dim3(kThreads), smem, st, p);
  if (int rc = launch_pdl(name, qk_norm_rope_kernel<DT, INTER, true>, dim3(p.q_blocks + p.k_blocks), dim3(kThreads), smem, st, p)) return rc;
  return launch_pdl(name, qk_norm_sum_kernel, dim3((2 * p.d.head_dim + kThreads / 32 - 1) / (kThreads / 32)), dim3(kThreads), 0, st, p);
}

}  // namespace
}  // namespace mak

using namespace mak;

extern "C" int64_t mak_qk_norm_rope_partial_floats(int32_t head_dim) { return static_cast<int64_t>(kMaxBlocks + 2) * head_dim; }

extern "C" int mak_qk_norm_rope(const mak_qk_norm_rope_desc* d, void* stream) {
  const char* name = "mak_qk_norm_rope";
  if (d == nullptr) return fail(MAK_E_INVALID, "%s: null descriptor", name);
  const bool back = d->grad_q != nullptr || d->grad_k != nullptr;
  if (d->dtype != MAK_DT_F16 && d->dtype != MAK_DT_BF16) return fail(MAK_E_UNSUPPORTED, "%s: q and k must be float16 or bfloat16", name);
  if (d->weight_dtype != MAK_DT_F32 && d->weight_dtype != d->dtype)
    return fail(MAK_E_UNSUPPORTED, "%s: weights must be float32 or of the type of q and k", name);
  if (!valid_index_dtype(d->pos_dtype)) return fail(MAK_E_INVALID, "%s: positions must be int32 or int64", name);
  if (d->head_dim < 16 || d->head_dim > 256 || d->head_dim % 16)
    return fail(MAK_E_UNSUPPORTED, "%s: head_dim must be a multiple of 16 up to 256, got %d", name, d->head_dim);
  if (d->rot_dim < 0 || d->rot_dim > d->head_dim || d->rot_dim % 16)
    return fail(MAK_E_UNSUPPORTED, "%s: the rotated columns must be a multiple of 16, at most head_dim, got %d", name, d->rot_dim);
  if (d->tokens < 0 || d->q_heads < 0 || d->k_heads < 0 || d->max_positions < 0) return fail(MAK_E_INVALID, "%s: negative size", name);
  if (back && (d->grad_q_weight == nullptr || d->grad_k_weight == nullptr || d->partial == nullptr))
    return fail(MAK_E_INVALID, "%s: null gradient", name);
  const bool any = d->tokens > 0 && d->q_heads + d->k_heads > 0;
  if (!any && !back) return MAK_OK;
  if (any) {
    if ((d->q_heads && (d->q == nullptr || d->q_out == nullptr)) || (d->k_heads && (d->k == nullptr || d->k_out == nullptr)) ||
        d->q_weight == nullptr || d->k_weight == nullptr || d->positions == nullptr ||
        (d->rot_dim && d->max_positions && (d->cos == nullptr || d->sin == nullptr)) ||
        (back && ((d->q_heads && d->grad_q == nullptr) || (d->k_heads && d->grad_k == nullptr))))
      return fail(MAK_E_INVALID, "%s: null tensor", name);
    uint64_t bits = 0, strides = 0;
    if (d->q_heads) {
      bits |= reinterpret_cast<uintptr_t>(d->q) | reinterpret_cast<uintptr_t>(d->q_out) | reinterpret_cast<uintptr_t>(d->grad_q);
      strides |= d->q_stride_token | d->q_stride_head | d->qo_stride_token | d->qo_stride_head | (back ? d->gq_stride_token | d->gq_stride_head : 0);
    }
    if (d->k_heads) {
      bits |= reinterpret_cast<uintptr_t>(d->k) | reinterpret_cast<uintptr_t>(d->k_out) | reinterpret_cast<uintptr_t>(d->grad_k);
      strides |= d->k_stride_token | d->k_stride_head | d->ko_stride_token | d->ko_stride_head | (back ? d->gk_stride_token | d->gk_stride_head : 0);
    }
    if ((bits & 15) || (strides & 7)) return fail(MAK_E_INVALID, "%s: rows need 16-byte alignment", name);
  }
  NormParams p = {};
  p.d = *d;
  p.lanes = 1;
  while (p.lanes * 16 < d->head_dim) p.lanes *= 2;
  // As many heads to a lane as leave every SM some 512 threads, eight at most.
  const int64_t heads = static_cast<int64_t>(d->q_heads) + d->k_heads;
  int per = 8;
  while (per > 1 && d->tokens * heads * p.lanes / per < static_cast<int64_t>(sm_count()) * 512) per /= 2;
  p.per_group = per;
  p.q_groups = (d->q_heads + per - 1) / per;
  p.k_groups = (d->k_heads + per - 1) / per;
  const int64_t per_block = kThreads / p.lanes;
  int64_t q_blocks = (d->tokens * p.q_groups + per_block - 1) / per_block, k_blocks = (d->tokens * p.k_groups + per_block - 1) / per_block;
  if (q_blocks + k_blocks > 0x7fffffff) return fail(MAK_E_UNSUPPORTED, "%s: too many heads", name);
  if (back && q_blocks + k_blocks > kMaxBlocks) {  // the blocks by the heads that they have
    const int64_t all = q_blocks + k_blocks;
    k_blocks = k_blocks ? (k_blocks * kMaxBlocks + all - 1) / all : 0;
    q_blocks = q_blocks ? (k_blocks < kMaxBlocks ? kMaxBlocks - k_blocks : 1) : 0;
  }
  if (q_blocks + k_blocks == 0) q_blocks = 1;
  p.q_blocks = static_cast<int32_t>(q_blocks), p.k_blocks = static_cast<int32_t>(k_blocks);
  p.wide_angles = d->cos_stride % 4 == 0 && d->sin_stride % 4 == 0 &&
                  ((reinterpret_cast<uintptr_t>(d->cos) | reinterpret_cast<uintptr_t>(d->sin)) & 15) == 0;
  cudaStream_t st = as_stream(stream);
  if (d->dtype == MAK_DT_BF16)
    return d->interleaved ? launch<MAK_DT_BF16, true>(p, back, name, st) : launch<MAK_DT_BF16, false>(p, back, name, st);
  return d->interleaved ? launch<MAK_DT_F16, true>(p, back, name, st) : launch<MAK_DT_F16, false>(p, back, name, st);
}
