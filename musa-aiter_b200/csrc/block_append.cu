// The writer of a block-scaled 8-bit cache: k / v rows into the last positions of
// their sequences, each (block, head) tile with one scale.
//
// Mathematics.  m = max |x| over the finite values written to the tile;
// s = m / Qmax for a tile the call begins, else max(s_old, m / Qmax);
// code = round(x / s), and where s grew the codes that stay become
// round(code * (s_old / s)).  Every step is an IEEE operation in 32 bits (the
// quotient x / s by reciprocal, remainder and one correction, which rounds
// exactly: P. Markstein, IA-64 and Elementary Functions, 2000).
//
// Layout.  One warp owns one tile [head_dim][block_size] of K or V, so nothing is
// shared and a tile is read at most once and written once.  A lane holds
// head_dim / 32 neighbouring dims of 16 tokens: its loads are a piece of a token's
// row, its stores whole 16-byte pieces of the tile's rows.
//
// Measured.  8 prompts of 900 to 4096 tokens, 8 heads of 128, bf16 to E4M3, blocks of 16: 22.3 us, 3.5 TB/s of a copy's
// 6.47; f16 the same, f32 29.6 us, 4.3 TB/s.  Neither instructions nor HBM bound it alone: 15 instructions for 32 values
// keep 0.53 of the issue slots busy, and of 8.2 cycles between two of a warp's 2.6 go to loads (lengths, block id and
// rows come one after another, a tile a warp, 17 warps per SM) and 1.8 to waits of fixed length.  64 requests of one
// token, into blocks that held some: 4.1 to 4.3 us, latency (length, block id, rows and old codes, new codes).
#include "block_attn.cuh"

namespace mak {

int check_block_cache(const mak_block_cache_desc& c, const char* name);

namespace {

constexpr int kWarpsPerBlock = 4;

struct AppendParams {
  uint8_t* cache[2];
  float* scale[2];
  const void* x[2];
  int64_t c_sb[2], c_sh[2], s_sb[2], s_sh[2], x_sr[2], x_sh[2];
  const int32_t* tables;
  const int32_t* ctx_lens;
  const int32_t* starts;
  int64_t table_stride, num_blocks, items;
  int32_t num_seqs, max_blocks, num_rows, nh, bs_log2;
};

// N neighbouring values of one row as they are stored.
template <int DT, int N>
struct Raw {
  static constexpr int kWords = DT == MAK_DT_F32 ? N : N / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    const uint32_t* p = static_cast<const uint32_t*>(base) + (DT == MAK_DT_F32 ? at : at / 2);
    if constexpr (kWords == 1) {
      w[0] = __ldg(p);
    } else if constexpr (kWords == 2) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + i));
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  // Magnitudes order as their bits do: the largest of those seen so far, for 16-bit types two at a time.
  __device__ __forceinline__ void top(uint32_t& m) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      m = DT == MAK_DT_F32 ? max(m, w[i] & 0x7fffffffu) : __vmaxu2(m, w[i] & 0x7fff7fffu);
  }
  static constexpr uint32_t kInf = DT == MAK_DT_F32 ? 0x7f800000u : DT == MAK_DT_BF16 ? 0x7f80u : 0x7c00u;
  // Of the two halves of m.
  static __device__ __forceinline__ uint32_t widest(uint32_t m) { return DT == MAK_DT_F32 ? m : max(m & 0xffffu, m >> 16); }
  static __device__ __forceinline__ float value(uint32_t bits) {
    if constexpr (DT == MAK_DT_F32)
      return __uint_as_float(bits);
    else if constexpr (DT == MAK_DT_BF16)
      return __uint_as_float(bits << 16);
    else
      return __half2float(__ushort_as_half(static_cast<uint16_t>(bits)));
  }
  // Non-finite values to 0.
  __device__ __forceinline__ void finite() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (DT == MAK_DT_F32) {
        if ((w[i] & kInf) == kInf) w[i] = 0;
      } else {
        if ((w[i] & kInf) == kInf) w[i] &= 0xffff0000u;
        if ((w[i] >> 16 & kInf) == kInf) w[i] &= 0xffffu;
      }
    }
  }
  // Values 2 i and 2 i + 1.
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (DT == MAK_DT_F32)
      return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else if constexpr (DT == MAK_DT_BF16)
      return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    else
      return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  }
};

template <int CODE>
__device__ __forceinline__ float code_value(uint32_t byte) {
  if constexpr (CODE == MAK_CODE_INT8) {
    return static_cast<float>(static_cast<int>(static_cast<int8_t>(byte)));
  } else {
    uint32_t h;
    asm("{\n .reg .b16 a;\n cvt.u16.u32 a, %1;\n cvt.rn.f16x2.e4m3x2 %0, a;\n}" : "=r"(h) : "r"(byte));
    return __half2float(__ushort_as_half(static_cast<uint16_t>(h)));
  }
}

// Four values to four code bytes; int8: values of at most 127.5 in magnitude.
template <int CODE>
__device__ __forceinline__ uint32_t to_codes(const float (&v)[4]) {
  if constexpr (CODE == MAK_CODE_INT8) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // adding 1.5 * 2^23 rounds to a whole number in the low bits
      b[i] = __float_as_uint(v[i] + 12582912.f);
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  } else {
    uint32_t r;
    asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n"
        " mov.b32 %0, {l, h};\n}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]));
    return r;
  }
}

// A block of the cache that the call writes.
struct Target {
  int64_t item, row;  // row: packed row of offset 0 (may lie before the sequence's first)
  int page, off0, off1;  // offsets [off0, off1) are written; page < 0: none
  bool begun;
};

__device__ __forceinline__ Target find_target(const AppendParams& p, int64_t item, int lane) {
  Target t;
  t.item = item;
  t.page = -1;
  const int bs = 1 << p.bs_log2;
  // Slots floor(starts[s] / bs) + 2 s ... belong to sequence s: at least as many as it
  // can touch blocks, whatever its position.  Slots before the first sequence's, whose rows
  // need not begin at 0, are nobody's.
  int s, row0, rows, nth;
  if (p.starts == nullptr) {
    s = static_cast<int>(item), row0 = s, rows = 1, nth = 0;
  } else {
    int lo = 0, n = p.num_seqs;  // the last s in [lo, lo + n) with slot(s) <= item
    while (n > 1) {
      const int step = (n + 31) >> 5;
      const int at = lo + lane * step;
      bool ok = false;
      if (at < lo + n) ok = (max(__ldg(p.starts + at), 0) >> p.bs_log2) + 2 * static_cast<int64_t>(at) <= item;
      const uint32_t votes = __ballot_sync(0xffffffffu, ok);
      const int k = votes == 0 ? 0 : 31 - __clz(votes);
      const int end = lo + n;
      lo += k * step;
      n = min(step, end - lo);
    }
    s = lo;
    row0 = max(__ldg(p.starts + s), 0);
    rows = min(__ldg(p.starts + s + 1), p.num_rows) - row0;
    nth = static_cast<int>(item - (row0 >> p.bs_log2) - 2 * static_cast<int64_t>(s));
    if (nth < 0) return t;
  }
  const int64_t ctx = __ldg(p.ctx_lens + s);
  const int64_t first = ctx - rows;  // position of the call's first row
  if (rows <= 0 || first < 0) return t;
  const int64_t block = (first >> p.bs_log2) + nth;
  const int64_t start = block << p.bs_log2;
  if (start >= ctx || block >= p.max_blocks) return t;
  const int page = __ldg(p.tables + s * p.table_stride + block);
  if (page < 0 || page >= p.num_blocks) return t;
  t.page = page;
  t.begun = start >= first;
  t.off0 = t.begun ? 0 : static_cast<int>(first - start);
  t.off1 = static_cast<int>(min(ctx - start, static_cast<int64_t>(bs)));
  t.row = row0 + start - first;
  return t;
}

// Blocks per SM by the words a lane holds of a row: 16-bit rows of head_dim 64 and 128 fit five times (prompt
// writes 24.3 us with four, 22.5 with five, 21.8 with six, 24.2 with eight; a decode step 3.95, 4.19, 4.47, 5.15).
constexpr int blocks_per_sm_of(int words) { return words <= 2 ? 5 : words <= 4 ? 3 : 2; }

// One warp, one tile: its first 16 tokens (all of them for 16-token blocks), old scale and codes are loaded
// at once and stay in registers.
template <int HD, int CODE, int DT>
__global__ void __launch_bounds__(32 * kWarpsPerBlock, blocks_per_sm_of(Raw<DT, HD / 32>::kWords)) block_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kDims = HD / 32;
  constexpr float kMost = CODE == MAK_CODE_INT8 ? 127.f : 448.f;
  using R = Raw<DT, kDims>;
  const int lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  const int64_t unit = blockIdx.x * static_cast<int64_t>(kWarpsPerBlock) + (threadIdx.x >> 5);
  if (unit >= p.items * p.nh * 2) return;
  const int kv = static_cast<int>(unit & 1);
  const int64_t pair = unit >> 1;
  const int64_t item = (pair >> 32) == 0 ? static_cast<uint32_t>(pair) / static_cast<uint32_t>(p.nh) : pair / p.nh;
  const int head = static_cast<int>(pair - item * p.nh);
  const Target t = find_target(p, item, lane);
  if (t.page < 0) return;
  const int bs = 1 << p.bs_log2;
  const void* x = p.x[kv];
  const int64_t x_step = p.x_sr[kv];
  const int64_t x_at = t.row * x_step + head * p.x_sh[kv] + lane * kDims;  // offset 0, this lane's dims
  uint8_t* tile = p.cache[kv] + t.page * p.c_sb[kv] + head * p.c_sh[kv] + static_cast<int64_t>(lane * kDims) * bs;
  float* scale = p.scale[kv] + t.page * p.s_sb[kv] + head * p.s_sh[kv];

  R raw[16];
  auto load16 = [&](int c0) {
    const int64_t at = x_at + c0 * x_step;
    if (c0 >= t.off0 && c0 + 16 <= t.off1) {
#pragma unroll
      for (int b = 0; b < 16; ++b) raw[b].load(x, at + b * x_step);
    } else {
#pragma unroll
      for (int b = 0; b < 16; ++b) {
        raw[b].clear();
        if (c0 + b >= t.off0 && c0 + b < t.off1) raw[b].load(x, at + b * x_step);
      }
    }
  };
  const int first = t.off0 & ~15;
  load16(first);
  float old = 0.f;
  uint4 codes[kDims];
  if (!t.begun) {
    old = *scale;
#pragma unroll
    for (int i = 0; i < kDims; ++i) codes[i] = *reinterpret_cast<const uint4*>(tile + static_cast<int64_t>(i) * bs + first);
    if (!(old > 0.f) || old == INFINITY) old = 0.f;
  }
  uint32_t most = 0;
  int held = first;  // the 16 tokens in registers
  bool odd = false;  // non-finite values seen
  for (int c0 = first; c0 < t.off1; c0 += 16) {
    if (c0 != held) load16(c0), held = c0;
    uint32_t m = 0;
#pragma unroll
    for (int b = 0; b < 16; ++b) raw[b].top(m);
    if (R::widest(m) >= R::kInf) {
      odd = true;
      m = 0;
#pragma unroll
      for (int b = 0; b < 16; ++b) {
        raw[b].finite();
        raw[b].top(m);
      }
    }
    most = max(most, R::widest(m));
  }
  const float top = R::value(__reduce_max_sync(0xffffffffu, most));
  const float mine = top < 0x1p-100f ? 0.f : __fdiv_rn(top, kMost);
  const float now = fmaxf(old, mine);
  const bool grew = now > old;
  if (lane == 0 && (t.begun || grew || old == 0.f)) *scale = now;
  const float safe = now > 0.f ? now : 1.f;
  const float ratio = grew ? __fdiv_rn(old, safe) : 1.f;
  // x / s as (x 2^k) / (s 2^k): away from the ends of the exponent range the remainder is exact, and what
  // 2^-64 rounds off of an x is nothing beside an s above 2^60
  const float adj = safe < 0x1p-60f ? 0x1p64f : safe > 0x1p60f ? 0x1p-64f : 1.f;
  const float div = safe * adj, inv = __frcp_rn(div);

  for (int c0 = 0; c0 < bs; c0 += 16) {
    const bool fresh = c0 < t.off1 && c0 + 16 > t.off0;
    if (!fresh && !t.begun && !grew) continue;
    uint32_t w[kDims][4];
    if (t.begun) {
#pragma unroll
      for (int i = 0; i < kDims; ++i) w[i][0] = w[i][1] = w[i][2] = w[i][3] = 0;
    } else {
#pragma unroll
      for (int i = 0; i < kDims; ++i) {
        uint4 z = codes[i];
        if (c0 != first) z = *reinterpret_cast<const uint4*>(tile + static_cast<int64_t>(i) * bs + c0);
        w[i][0] = z.x, w[i][1] = z.y, w[i][2] = z.z, w[i][3] = z.w;
      }
      if (grew) {
#pragma unroll
        for (int i = 0; i < kDims; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              v[b] = __fmul_rn(code_value<CODE>((w[i][q] >> (8 * b)) & 0xffu), ratio);
              if (CODE == MAK_CODE_INT8) v[b] = fmaxf(v[b], -127.f);  // -128 is not the writer's
            }
            w[i][q] = to_codes<CODE>(v);
          }
      }
    }
    if (fresh) {
      if (c0 != held) {
        load16(c0), held = c0;
        if (odd) {
#pragma unroll
          for (int b = 0; b < 16; ++b) raw[b].finite();
        }
      }
      const float2 zero = make_float2(0.f, 0.f);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t mask = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (c0 + 4 * q + b >= t.off0 && c0 + 4 * q + b < t.off1) mask |= 0xffu << (8 * b);
#pragma unroll
        for (int i = 0; i < kDims; i += 2) {
          float y[2][4];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const float2 v = fma2(raw[4 * q + b].pair(i / 2), make_float2(adj, adj), zero), q0 = fma2(v, make_float2(inv, inv), zero);
            const float2 z = fma2(fma2(q0, make_float2(-div, -div), v), make_float2(inv, inv), q0);
            y[0][b] = z.x;
            y[1][b] = z.y;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) w[i + e][q] = (w[i + e][q] & ~mask) | (to_codes<CODE>(y[e]) & mask);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kDims; ++i)
      *reinterpret_cast<uint4*>(tile + static_cast<int64_t>(i) * bs + c0) = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
  }
}

template <int HD, int CODE>
int launch_append(const AppendParams& p, int dtype, dim3 grid, cudaStream_t st) {
  const dim3 block(32 * kWarpsPerBlock);
  const char* name = "mak_block_append";
  if (dtype == MAK_DT_F16) return launch_pdl(name, block_append_kernel<HD, CODE, MAK_DT_F16>, grid, block, 0, st, p);
  if (dtype == MAK_DT_BF16) return launch_pdl(name, block_append_kernel<HD, CODE, MAK_DT_BF16>, grid, block, 0, st, p);
  return launch_pdl(name, block_append_kernel<HD, CODE, MAK_DT_F32>, grid, block, 0, st, p);
}

template <int HD>
int launch_append_code(const AppendParams& p, int code, int dtype, dim3 grid, cudaStream_t st) {
  return code == MAK_CODE_INT8 ? launch_append<HD, MAK_CODE_INT8>(p, dtype, grid, st)
                               : launch_append<HD, MAK_CODE_E4M3>(p, dtype, grid, st);
}

}  // namespace
}  // namespace mak

using namespace mak;

extern "C" int mak_block_append(const mak_block_cache_desc* cache, const void* k, const void* v, int64_t k_stride_row,
                                int64_t k_stride_head, int64_t v_stride_row, int64_t v_stride_head, int32_t dtype, void* stream) {
  const char* name = "mak_block_append";
  if (cache == nullptr) return fail(MAK_E_INVALID, "%s: null descriptor", name);
  const mak_block_cache_desc& c = *cache;
  if (int rc = check_block_cache(c, name)) return rc;
  if (dtype != MAK_DT_F16 && dtype != MAK_DT_BF16 && dtype != MAK_DT_F32)
    return fail(MAK_E_UNSUPPORTED, "%s: k / v must be float16, bfloat16 or float32", name);
  if (c.num_seqs == 0 || c.num_rows == 0) return MAK_OK;
  if (k == nullptr || v == nullptr) return fail(MAK_E_INVALID, "%s: null k or v", name);
  const uint64_t align = 16 / dtype_bytes(dtype);
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) ||
      (static_cast<uint64_t>(k_stride_row | k_stride_head | v_stride_row | v_stride_head) & (align - 1)))
    return fail(MAK_E_INVALID, "%s: k / v need 16-byte aligned rows", name);
  AppendParams p = {};
  p.cache[0] = static_cast<uint8_t*>(c.key), p.cache[1] = static_cast<uint8_t*>(c.value);
  p.scale[0] = c.key_scale, p.scale[1] = c.value_scale;
  p.x[0] = k, p.x[1] = v;
  p.c_sb[0] = c.key_stride_block, p.c_sb[1] = c.value_stride_block;
  p.c_sh[0] = c.key_stride_head, p.c_sh[1] = c.value_stride_head;
  p.s_sb[0] = c.key_scale_stride_block, p.s_sb[1] = c.value_scale_stride_block;
  p.s_sh[0] = c.key_scale_stride_head, p.s_sh[1] = c.value_scale_stride_head;
  p.x_sr[0] = k_stride_row, p.x_sr[1] = v_stride_row;
  p.x_sh[0] = k_stride_head, p.x_sh[1] = v_stride_head;
  p.tables = c.block_tables, p.ctx_lens = c.context_lens, p.starts = c.cu_seqlens;
  p.table_stride = c.table_stride, p.num_blocks = c.num_blocks;
  p.num_seqs = static_cast<int32_t>(c.num_seqs), p.max_blocks = static_cast<int32_t>(c.max_blocks);
  p.num_rows = static_cast<int32_t>(c.num_rows), p.nh = c.num_heads;
  p.bs_log2 = c.block_size == 16 ? 4 : c.block_size == 32 ? 5 : c.block_size == 64 ? 6 : 7;
  p.items = c.cu_seqlens == nullptr ? c.num_seqs : (c.num_rows >> p.bs_log2) + 2 * c.num_seqs;
  const int64_t blocks = (p.items * p.nh * 2 + kWarpsPerBlock - 1) / kWarpsPerBlock;
  if (blocks > 0x7fffffff) return fail(MAK_E_UNSUPPORTED, "%s: too many rows for one call", name);
  const dim3 grid(static_cast<unsigned>(blocks));
  cudaStream_t st = as_stream(stream);
  if (c.head_dim == 64) return launch_append_code<64>(p, c.code_type, dtype, grid, st);
  if (c.head_dim == 128) return launch_append_code<128>(p, c.code_type, dtype, grid, st);
  return launch_append_code<256>(p, c.code_type, dtype, grid, st);
}
