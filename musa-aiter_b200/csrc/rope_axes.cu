// Rotary positions with several axes (time, height, width): each pair of a head
// takes its angle from the position along its own axis; q and k in one launch,
// forward or with the angles negated (the gradient).
//
// (y1, y2) = (x1 c - x2 s, x1 s + x2 c) in 32 bits, rounded once.  Memory-bound:
// a thread keeps the cos / sin of its pairs in registers over several heads and
// moves 16 bytes at a time.
//
// Measured.  16384 tokens of 32 + 8 heads of 128 as views of one projection: 61 us, 5.6 TB/s of a copy's 6.47; 64
// tokens: 2.6 to 2.8 us, one launch's latency (positions, angles, heads).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace mak {
namespace {

struct RopeAxesParams {
  mak_rope_axes_desc d;
  int32_t slots;      // 16-byte pieces of a head that one thread each takes (two pieces for split pairs)
  int32_t rot_slots;  // of these, the ones that rotate
  int32_t groups;     // threads per (token, slot)
  int32_t per_group;  // heads of one thread
};

template <int DT>
__device__ __forceinline__ void unpack8(const uint4& r, float (&x)[8]) {
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
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
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

// Thread: one token, one slot, per_group heads.  Split pairs: slot j < rot / 16
// holds x[8 j .. 8 j + 8) and its partners half a rotation further; interleaved:
// slot j < rot / 8 holds pairs 4 j .. 4 j + 4.  Further slots are copied.
template <int DT, bool INTER>
__global__ void __launch_bounds__(256) rope_axes_kernel(const __grid_constant__ RopeAxesParams p) {
  constexpr int kPairs = INTER ? 4 : 8;
  const mak_rope_axes_desc& d = p.d;
  const int64_t per_token = static_cast<int64_t>(p.slots) * p.groups;
  const int64_t idx = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x;
  pdl_wait();
  pdl_trigger();
  if (idx >= d.tokens * per_token) return;
  const int64_t t = idx / per_token;
  const int in = static_cast<int>(idx - t * per_token);
  const int slot = in % p.slots, grp = in / p.slots;
  const int heads = d.q_heads + d.k_heads;
  const int h0 = grp * p.per_group, h1 = min(h0 + p.per_group, heads);
  const int half = d.rot_dim / 2;
  const bool rotates = slot < p.rot_slots;
  const int at = rotates ? slot * 8 : d.rot_dim + (slot - p.rot_slots) * 8;
  float c[kPairs], s[kPairs];
  if (rotates) {
    const int pair0 = slot * kPairs;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int pair = pair0 + i;
      const int64_t pos = load_index(d.positions, d.pos_dtype == MAK_DT_I64, d.pair_axis[pair] * d.pos_stride + t);
      c[i] = 1.f, s[i] = 0.f;
      if (pos >= 0 && pos < d.max_positions) {
        c[i] = __ldg(d.cos + pos * d.cos_stride + pair);
        s[i] = __ldg(d.sin + pos * d.sin_stride + pair);
      }
      if (d.inverse) s[i] = -s[i];
    }
  }
  // kDeep heads' loads in flight
  constexpr int kDeep = INTER ? 8 : 4;
  for (int h = h0; h < h1; h += kDeep) {
    uint4 r1[kDeep], r2[kDeep];
#pragma unroll
    for (int z = 0; z < kDeep; ++z) {
      if (h + z >= h1) break;
      const bool isq = h + z < d.q_heads;
      const int hh = isq ? h + z : h + z - d.q_heads;
      const uint16_t* src = static_cast<const uint16_t*>(isq ? d.q : d.k) + t * (isq ? d.q_stride_token : d.k_stride_token) +
                            hh * (isq ? d.q_stride_head : d.k_stride_head) + at;
      r1[z] = __ldcs(reinterpret_cast<const uint4*>(src));
      if (!INTER && rotates) r2[z] = __ldcs(reinterpret_cast<const uint4*>(src + half));
    }
#pragma unroll
    for (int z = 0; z < kDeep; ++z) {
      if (h + z >= h1) break;
      const bool isq = h + z < d.q_heads;
      const int hh = isq ? h + z : h + z - d.q_heads;
      uint16_t* dst = static_cast<uint16_t*>(isq ? d.q_out : d.k_out) + t * (isq ? d.qo_stride_token : d.ko_stride_token) +
                      hh * (isq ? d.qo_stride_head : d.ko_stride_head) + at;
      if (!rotates) {
        __stcs(reinterpret_cast<uint4*>(dst), r1[z]);
        continue;
      }
      float x[8], y[8];
      unpack8<DT>(r1[z], x);
      if constexpr (INTER) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[2 * i] = x[2 * i] * c[i] - x[2 * i + 1] * s[i];
          y[2 * i + 1] = x[2 * i] * s[i] + x[2 * i + 1] * c[i];
        }
        __stcs(reinterpret_cast<uint4*>(dst), pack8<DT>(y));
      } else {
        float x2[8], y2[8];
        unpack8<DT>(r2[z], x2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = x[i] * c[i] - x2[i] * s[i];
          y2[i] = x[i] * s[i] + x2[i] * c[i];
        }
        __stcs(reinterpret_cast<uint4*>(dst), pack8<DT>(y));
        __stcs(reinterpret_cast<uint4*>(dst + half), pack8<DT>(y2));
      }
    }
  }
}

}  // namespace
}  // namespace mak

using namespace mak;

extern "C" int mak_rope_axes(const mak_rope_axes_desc* desc, void* stream) {
  const char* name = "mak_rope_axes";
  if (desc == nullptr) return fail(MAK_E_INVALID, "%s: null descriptor", name);
  RopeAxesParams p = {};
  p.d = *desc;
  mak_rope_axes_desc& d = p.d;
  if (d.k == nullptr) d.k_heads = 0;
  if (d.tokens < 0 || d.q_heads < 0 || d.k_heads < 0 || d.axes <= 0 || d.max_positions < 0)
    return fail(MAK_E_INVALID, "%s: bad size", name);
  if (d.dtype != MAK_DT_F16 && d.dtype != MAK_DT_BF16) return fail(MAK_E_UNSUPPORTED, "%s: float16 or bfloat16 only", name);
  if (!valid_index_dtype(d.pos_dtype)) return fail(MAK_E_INVALID, "%s: positions must be int32 or int64", name);
  if (d.head_dim <= 0 || d.head_dim % 8 || d.rot_dim <= 0 || d.rot_dim % (d.interleaved ? 8 : 16) || d.rot_dim > d.head_dim ||
      d.rot_dim / 2 > MAK_ROPE_MAX_PAIRS)
    return fail(MAK_E_UNSUPPORTED, "%s: head_dim %d / rot_dim %d", name, d.head_dim, d.rot_dim);
  for (int i = 0; i < d.rot_dim / 2; ++i)
    if (d.pair_axis[i] >= d.axes) return fail(MAK_E_INVALID, "%s: pair %d has axis %d of %d", name, i, d.pair_axis[i], d.axes);
  const int heads = d.q_heads + d.k_heads;
  if (d.tokens == 0 || heads == 0) return MAK_OK;
  if ((d.q_heads && (d.q == nullptr || d.q_out == nullptr)) || (d.k_heads && d.k_out == nullptr) || d.positions == nullptr ||
      (d.max_positions && (d.cos == nullptr || d.sin == nullptr)))
    return fail(MAK_E_INVALID, "%s: null pointer", name);
  const uint64_t addr = (d.q_heads ? reinterpret_cast<uintptr_t>(d.q) | reinterpret_cast<uintptr_t>(d.q_out) : 0) |
                        (d.k_heads ? reinterpret_cast<uintptr_t>(d.k) | reinterpret_cast<uintptr_t>(d.k_out) : 0);
  int64_t strides = 0;
  if (d.q_heads) strides |= d.q_stride_token | d.q_stride_head | d.qo_stride_token | d.qo_stride_head;
  if (d.k_heads) strides |= d.k_stride_token | d.k_stride_head | d.ko_stride_token | d.ko_stride_head;
  if ((addr & 15) || (strides & 7)) return fail(MAK_E_INVALID, "%s: rows need 16-byte alignment", name);
  p.rot_slots = d.rot_dim / (d.interleaved ? 8 : 16);
  p.slots = p.rot_slots + (d.head_dim - d.rot_dim) / 8;
  // A thread takes up to 8 heads, as many as leave each SM 128 threads: it reads its angles once for all of them.
  // 40 heads of 128, tokens: us with 1, 4 and 8 heads a thread: 64: 2.8, 3.4, 4.2; 256: 5.2, 3.4, 4.2;
  // 1024: 13.0, 6.7, 6.3; 4096: 50, 19, 16.5; 16384: 202, 72, 61.
  const int64_t threads = d.tokens * p.slots * heads;
  int64_t per = threads / (static_cast<int64_t>(sm_count()) * 128);
  per = per < 1 ? 1 : per > 8 ? 8 : per;
  p.per_group = static_cast<int32_t>(per);
  p.groups = (heads + p.per_group - 1) / p.per_group;
  const int64_t blocks = (d.tokens * p.slots * p.groups + 255) / 256;
  if (blocks > 0x7fffffff) return fail(MAK_E_UNSUPPORTED, "%s: too many tokens for one call", name);
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
  cudaStream_t st = as_stream(stream);
  if (d.dtype == MAK_DT_BF16)
    return d.interleaved ? launch_pdl(name, rope_axes_kernel<MAK_DT_BF16, true>, grid, block, 0, st, p)
                         : launch_pdl(name, rope_axes_kernel<MAK_DT_BF16, false>, grid, block, 0, st, p);
  return d.interleaved ? launch_pdl(name, rope_axes_kernel<MAK_DT_F16, true>, grid, block, 0, st, p)
                       : launch_pdl(name, rope_axes_kernel<MAK_DT_F16, false>, grid, block, 0, st, p);
}
