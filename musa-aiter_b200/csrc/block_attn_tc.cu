// Attention over a block-scaled 8-bit cache for many rows per sequence (prompts):
// the products on the tcgen05 tensor cores, everything else hidden behind them.
//
// Mathematics as in block_attn.cu: S = q . codes with q and codes in f16 (codes
// exactly, a bf16 row of q by a power of two), the K scale and the softmax scale
// multiplied on in 32 bits, weights p * (V scale / largest V scale of the unit) *
// 2^6 rounded once to f16, sums in 32 bits.  The running maximum of a row is only
// moved when it grew by more than 2^8: weights then stay below 2^14, the result is
// the same, and the accumulators in TMEM are rarely rescaled.
//
// A block takes 256 rows of one cache head (heads of the group next to one another,
// so a K / V tile serves all of them) as two tiles of 128, and walks the cache in
// tiles of 128 tokens.  Roles:
//   warps 0-3, 4-7   softmax of row tile 0 / 1, a thread per row (TMEM lane)
//   warps 8-11       codes to f16, shared memory to shared memory
//   warp 12          one thread issues all tcgen05.mma
//   warp 13          block ids, scales, and the copies of the codes to shared memory
// While one row tile's scores are exponentiated the tensor cores work for the other.
//
// Layout.  The cache tile is [head_dim][tokens], tokens contiguous.  Converted to f16
// it is stored as it is, in 128-byte swizzled lines of 64 tokens: K is read from there
// as an MN-major operand and V as a K-major one, so no element is ever transposed.
// Scores and weights share TMEM columns: the product with V of a tile is issued
// before the next scores of the same rows overwrite them.
#include "block_attn.cuh"
#include "tcgen05.cuh"

namespace mak {
namespace {

constexpr int kTile = 128;                // tokens per step
constexpr int kUnitRows = 256;            // rows of a block
constexpr int kThreads = 512;
constexpr float kLazy = 8.f;              // log2 growth of a row's maximum that is tolerated

template <int HD>
struct TcSmem {
  alignas(1024) uint8_t q[2][HD * 256];  // 128 rows: HD / 64 pieces of [128][64]
  alignas(1024) uint8_t k[2][HD * 256];  // 128 tokens: 2 pieces of [HD][64]
  alignas(1024) uint8_t v[2][HD * 256];
  alignas(128) uint8_t k_raw[HD * 128], v_raw[HD * 128];  // codes as they come: [block][HD][block_size]
  alignas(16) float kfac[4][8], vfac[4][8];  // per 16 tokens of a tile: K scale, weight of a unit of V
  alignas(16) float vlog[4][8], vinv[4][8];  // log2 and reciprocal of the latter
  uint32_t have[4], plain[4];                // bit c: piece c has a block; its factors are positive and finite
  alignas(8) uint64_t kr_full, kr_empty, vr_full, vr_empty, q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], spare;
  uint32_t tmem;
  float vmax[4];
  int unit_seq, unit_tile;
  int gave_up;
};

template <int HD, int CODE>
__global__ void __launch_bounds__(kThreads, 1) block_attn_tc_kernel(const __grid_constant__ BlockAttnParams p,
                                                                           const __grid_constant__ CUtensorMap kmap,
                                                                           const __grid_constant__ CUtensorMap vmap) {
  extern __shared__ __align__(1024) uint8_t raw[];
  TcSmem<HD>& sm = *reinterpret_cast<TcSmem<HD>*>(raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();

  // ---- which rows -------------------------------------------------------------
  // Units of sequence s take the numbers floor(starts[s] * group / 256) + s and up, at
  // least as many as it has tiles.  Later units see more tokens: they come first.
  const int head = blockIdx.x % p.nh;
  const int64_t item = gridDim.x / p.nh - 1 - blockIdx.x / p.nh;
  if (warp == 0) {
    int lo = 0, n = p.num_seqs;
    while (n > 1) {
      const int step = (n + 31) >> 5;
      const int at = lo + lane * step;
      bool ok = false;
      if (at < lo + n) {
        const int64_t row = p.starts != nullptr ? max(__ldg(p.starts + at), 0) : at;
        ok = row * p.group / kUnitRows + at <= item;
      }
      const uint32_t votes = __ballot_sync(0xffffffffu, ok);
      const int k = votes == 0 ? 0 : 31 - __clz(votes);
      const int end = lo + n;
      lo += k * step;
      n = min(step, end - lo);
    }
    if (lane == 0) {
      const int64_t row = p.starts != nullptr ? max(__ldg(p.starts + lo), 0) : lo;
      sm.unit_seq = lo;
      sm.unit_tile = static_cast<int>(item - row * p.group / kUnitRows - lo);
      sm.gave_up = 0;
      mbar_init(&sm.spare, 1);
      mbar_init(&sm.kr_full, 1);
      mbar_init(&sm.vr_full, 1);
      mbar_init(&sm.kr_empty, 4);
      mbar_init(&sm.vr_empty, 4);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sm.q_full[i], 4);
        mbar_init(&sm.k_full[i], 4);
        mbar_init(&sm.v_full[i], 4);
        mbar_init(&sm.k_empty[i], 1);
        mbar_init(&sm.v_empty[i], 1);
        mbar_init(&sm.s_full[i], 1);
        mbar_init(&sm.p_full[i], 4);
        mbar_init(&sm.o_full[i], 1);
      }
      mbar_init_fence();
    }
  }
  __syncthreads();
  const int seq = sm.unit_seq;
  const SeqView v = seq_view(p, seq);
  const int rows_total = v.rows * p.group;
  const int64_t row0 = static_cast<int64_t>(sm.unit_tile) * kUnitRows;
  if (row0 >= rows_total) return;
  if (warp == 12) {
    tmem_alloc<512>(&sm.tmem);
  }
  const int live = static_cast<int>(min(static_cast<int64_t>(kUnitRows), rows_total - row0));
  const int halves = live > 128 ? 2 : 1;
  int any_lo, any_hi, unused;
  row_range(p, v, static_cast<int>(row0 / p.group), &any_lo, &unused);
  row_range(p, v, static_cast<int>((row0 + live - 1) / p.group), &unused, &any_hi);
  const int t0 = any_lo / kTile;
  const int tiles = any_hi > any_lo ? (any_hi + kTile - 1) / kTile - t0 : 0;
  const int32_t* table = p.tables + seq * p.table_stride;
  const int bs = 1 << p.bs_log2;

  // largest V scale of the unit's pages
  if (warp >= 8 && warp < 12 && tiles > 0) {
    float top = 0.f;
    for (int b = (any_lo >> p.bs_log2) + tid - 256; b <= (any_hi - 1) >> p.bs_log2; b += 128) {
      const int page = __ldg(table + b);
      if (page >= 0 && page < p.num_blocks) top = fmaxf(top, fabsf(__ldg(p.value_scale + page * p.vs_sb + head * p.vs_sh)));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) sm.vmax[warp - 8] = top;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const float vref = tiles > 0 ? fmaxf(fmaxf(sm.vmax[0], sm.vmax[1]), fmaxf(sm.vmax[2], sm.vmax[3])) : 0.f;
  volatile int* gave_up = &sm.gave_up;

  if (warp < 8) {
    regs_up<184>();  // with 80 and 64 below: what the block was launched with
    // ---- softmax ----------------------------------------------------------------
    const int half = warp >> 2;
    const int r = tid & 127;
    const int64_t row = row0 + half * 128 + r;
    if (half < halves) {
      const bool on = row < rows_total;
      const int i = on ? static_cast<int>(row / p.group) : 0, j = on ? static_cast<int>(row % p.group) : 0;
      float qs = 0.f;
      {  // this row of q to f16
        uint4 x[HD / 8];
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < HD / 8; ++e) {
          x[e] = make_uint4(0, 0, 0, 0);
          if (on)
            x[e] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + (v.first + i) * p.q_sr +
                                                        (head * p.group + j) * p.q_sh + e * 8));
        }
        int up = 0;
        if (p.q_bf16) {
#pragma unroll
          for (int e = 0; e < HD / 8; ++e)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t b = (&x[e].x)[w];
              top = fmaxf(top, fmaxf(fabsf(__uint_as_float(b << 16)), fabsf(__uint_as_float(b & 0xffff0000u))));
            }
          if (top > 0.f && top < __uint_as_float(0x7f800000u)) up = 14 - ilogbf(top);
          const int up1 = up / 2, up2 = up - up1;
          const float f1 = __uint_as_float(static_cast<uint32_t>(127 + up1) << 23);
          const float f2 = __uint_as_float(static_cast<uint32_t>(127 + up2) << 23);
#pragma unroll
          for (int e = 0; e < HD / 8; ++e)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t& b = (&x[e].x)[w];
              b = pack_f16(__uint_as_float(b << 16) * f1 * f2, __uint_as_float(b & 0xffff0000u) * f1 * f2);
            }
        }
#pragma unroll
        for (int e = 0; e < HD / 8; ++e)
          *reinterpret_cast<uint4*>(sm.q[half] + (e >> 3) * 16384 + r * 128 + (((e & 7) ^ (r & 7)) << 4)) = x[e];
        qs = ldexpf(p.scale_log2, -up);
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full[half]);
      }
      int lo = 0, hi = 0;
      if (on) row_range(p, v, i, &lo, &hi);
      int all_lo, all_hi;  // what all rows of this tile see
      {
        const int last = min(live, half * 128 + 128) - 1;
        row_range(p, v, static_cast<int>((row0 + half * 128) / p.group), &unused, &all_hi);
        row_range(p, v, static_cast<int>((row0 + last) / p.group), &all_lo, &unused);
      }
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t s_at = tmem + lanes + half * 128;
      const uint32_t o_at = tmem + lanes + 256 + half * HD;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int t = 0; t < tiles; ++t) {
        ok = mbar_wait_warp(&sm.s_full[half], t & 1, gave_up);
        if (!ok) break;
        tc_fence_after();
        const int tok = (t0 + t) * kTile;
        const float* kf = sm.kfac[t & 3];
        const uint32_t have = sm.have[t & 3];
        const bool whole = tok >= all_lo && tok + kTile <= all_hi && sm.plain[t & 3] == 0xffu && p.scale_log2 > 0.f;
        uint32_t x[4][32];  // whole: the row's scores stay in registers
        float top = -INFINITY;
        if (whole) {
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld(s_at + c * 32, x[c]);
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_wait(x[c]);
          float tops[8];  // 16 columns share a factor, which is positive: it can wait
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint32_t* at = &x[c >> 1][(c & 1) * 16];
            tops[c] = fmaxf(__uint_as_float(at[0]), __uint_as_float(at[1]));
#pragma unroll
            for (int e = 2; e < 16; e += 2) tops[c] = fmaxf(fmaxf(tops[c], __uint_as_float(at[e])), __uint_as_float(at[e + 1]));
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) top = fmaxf(top, tops[c] * (kf[c] * qs));
        } else {
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t y[16];
            tmem_ld(s_at + c * 16, y);
            tmem_wait(y);
            const float f = kf[c] * qs;
            // columns [from, to) of these 16 are seen
            const int first = tok + 16 * c, from = lo - first, to = (have >> c) & 1 ? hi - first : 0;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (e >= from && e < to) top = fmaxf(top, __uint_as_float(y[e]) * f);
          }
        }
        const bool grow = top > m + kLazy || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, grow)) {
          const float mn = fmaxf(m, top);
          const float keep = mn == -INFINITY ? 1.f : exp2_fast(m - mn);
          m = mn;
          l *= keep;
          if (t > 0) {
#pragma unroll 1
            for (int c = 0; c < HD / 16; ++c) {
              uint32_t o[16];
              tmem_ld(o_at + c * 16, o);
              tmem_wait(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
              tmem_st(o_at + c * 16, o);
            }
          }
        }
        const float ms = m == -INFINITY ? 0.f : m;
        if (whole) {
          // 2^(x f - m) b' as one power of 2; the sum of the weights without b' is taken per 16 columns
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t y[16];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const float f = kf[2 * c + z] * qs, d = sm.vlog[t & 3][2 * c + z] - ms;
              float2 sum = make_float2(0.f, 0.f);
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                const uint32_t* at = &x[c][z * 16 + e];
                float2 w = fma2(make_float2(__uint_as_float(at[0]), __uint_as_float(at[1])), make_float2(f, f), make_float2(d, d));
                w.x = exp2_fast(w.x);
                w.y = exp2_fast(w.y);
                sum = add2(sum, w);
                y[(z * 16 + e) >> 1] = pack_f16(w.x, w.y);
              }
              l = fmaf(sum.x + sum.y, sm.vinv[t & 3][2 * c + z], l);
            }
            tmem_st(s_at + c * 16, y);
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t x16[16], y[8];
            tmem_ld(s_at + c * 16, x16);
            tmem_wait(x16);
            const float f = kf[c] * qs, w = sm.vfac[t & 3][c];
            const int first = tok + 16 * c, from = lo - first, to = (have >> c) & 1 ? hi - first : 0;
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              float a = exp2_fast(fmaf(__uint_as_float(x16[e]), f, -ms));
              float b = exp2_fast(fmaf(__uint_as_float(x16[e + 1]), f, -ms));
              a = e >= from && e < to ? a : 0.f;
              b = e + 1 >= from && e + 1 < to ? b : 0.f;
              l += a + b;
              y[e >> 1] = pack_f16(a * w, b * w);
            }
            tmem_st(s_at + c * 8, y);
          }
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[half]);
      }
      if (ok && tiles > 0) {
        ok = mbar_wait_warp(&sm.o_full[half], 0, gave_up);
        tc_fence_after();
      }
      // a block that gave up leaves NaN, not stale memory
      const float bad = __uint_as_float(0x7fffffffu);
      const bool some = l > 0.f || l != l;
      const float inv = some ? vref * (1.f / 64.f) / l : 0.f;
      const int64_t at = (v.first + i) * p.o_sr + (head * p.group + j) * p.o_sh;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t x[32];
        if (tiles > 0 && ok) {
          tmem_ld(o_at + c * 32, x);
          tmem_wait(x);
        }
        if (on) {
          uint32_t y[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float a = some ? __uint_as_float(x[e]) * inv : 0.f, b = some ? __uint_as_float(x[e + 1]) * inv : 0.f;
            if (!ok) a = b = bad;
            if (p.q_bf16) {
              const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
              y[e >> 1] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
              y[e >> 1] = pack_f16(a, b);
            }
          }
          uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + at + c * 32;
          if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) reinterpret_cast<uint4*>(dst)[e] = make_uint4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              dst[2 * e] = static_cast<uint16_t>(y[e]);
              dst[2 * e + 1] = static_cast<uint16_t>(y[e] >> 16);
            }
          }
        }
      }
      if (on && p.lse != nullptr)
        p.lse[static_cast<int64_t>(v.first + i) * p.nh * p.group + head * p.group + j] =
            !ok ? bad : some ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
    }
  } else if (warp < 12) {
    regs_down<80>();
    // ---- codes to f16 in shared memory -------------------------------------------
    // Piece i of the raw codes (16 tokens of one head_dim row) is 16 bytes at 16 i: pieces of a block's
    // line first, then rows, then blocks.
    const int id0 = tid - 256;
    const int per_log2 = p.bs_log2 - 4;
    constexpr int kIts = HD / 16;
    auto convert = [&](uint8_t* dst, int it, uint4 z) {
      const int id = it * 128 + id0;
      const int d = (id >> per_log2) & (HD - 1);
      const int chunk = ((id >> per_log2) / HD << per_log2) | (id & ((1 << per_log2) - 1));
      uint32_t y[8];
      codes4_to_f16<CODE>(z.x, &y[0], &y[1]);
      codes4_to_f16<CODE>(z.y, &y[2], &y[3]);
      codes4_to_f16<CODE>(z.z, &y[4], &y[5]);
      codes4_to_f16<CODE>(z.w, &y[6], &y[7]);
      uint8_t* line = dst + (chunk >> 2) * (HD * 128) + d * 128;
      const uint32_t c0 = ((chunk & 3) * 2) ^ (d & 7);
      *reinterpret_cast<uint4*>(line + (c0 << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<uint4*>(line + ((c0 ^ 1) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
    };
    auto tile = [&](const uint8_t* src, uint8_t* dst, int t, uint64_t* raw_full, uint64_t* raw_empty, uint64_t* empty, uint64_t* full) {
      if (!mbar_wait_warp(raw_full, t & 1, gave_up)) return false;
      uint4 x[kIts];
#pragma unroll
      for (int it = 0; it < kIts; ++it) x[it] = reinterpret_cast<const uint4*>(src)[it * 128 + id0];
      const int tok = (t0 + t) * kTile;
      if (tok < any_lo || tok + kTile > any_hi || sm.have[t & 3] != 0xffu) {
        // tokens that no row sees, or without a block: their codes may be anything and become 0
#pragma unroll
        for (int it = 0; it < kIts; ++it) {
          const int id = it * 128 + id0;
          const int chunk = ((id >> per_log2) / HD << per_log2) | (id & ((1 << per_log2) - 1));
          const int first = tok + 16 * chunk;
          uint32_t* words = &x[it].x;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t mask = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b)
              if (first + 4 * q + b >= any_lo && first + 4 * q + b < any_hi) mask |= 0xffu << (8 * b);
            words[q] = (sm.have[t & 3] >> chunk) & 1 ? words[q] & mask : 0u;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(raw_empty);
      if (!mbar_wait_warp(empty, ((t >> 1) & 1) ^ 1, gave_up)) return false;
#pragma unroll
      for (int it = 0; it < kIts; ++it) convert(dst, it, x[it]);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
      return true;
    };
    for (int t = 0; t < tiles; ++t) {
      const int st = t & 1;
      if (!tile(sm.k_raw, sm.k[st], t, &sm.kr_full, &sm.kr_empty, &sm.k_empty[st], &sm.k_full[st])) break;
      if (!tile(sm.v_raw, sm.v[st], t, &sm.vr_full, &sm.vr_empty, &sm.v_empty[st], &sm.v_full[st])) break;
    }
  } else {
    regs_down<64>();
    if (warp == 12 && lane == 0 && tiles > 0) {
      // ---- the tensor cores -------------------------------------------------------
      constexpr uint32_t kQk = instr_desc(kTile, 1, 0, false, true), kPv = instr_desc(HD, 1, 0, false, false);
      // Descriptors differ in their addresses alone, in units of 16 bytes: no carry leaves that field.
      const uint64_t q_desc = smem_desc(smem_addr(sm.q), 16, 1024, 7), k_desc = smem_desc(smem_addr(sm.k), HD * 128, 1024, 7);
      const uint64_t v_desc = smem_desc(smem_addr(sm.v), 16, 1024, 7);
      constexpr uint32_t kBuffer = HD * 256 / 16;
      auto scores = [&](int half, int st) {
        const uint64_t qd = q_desc + half * kBuffer, kd = k_desc + st * kBuffer;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
          mma_ss_f16(tmem + half * 128, qd + (ks >> 2) * 1024 + (ks & 3) * 2, kd + ks * 128, kQk, ks > 0);
        tc_commit(&sm.s_full[half]);
      };
      bool ok = true;
      for (int half = 0; half < halves && ok; ++half) ok = mbar_wait(&sm.q_full[half], 0, gave_up);
      ok = ok && mbar_wait(&sm.k_full[0], 0, gave_up);
      if (ok) {
        tc_fence_after();
        for (int half = 0; half < halves; ++half) scores(half, 0);
        tc_commit(&sm.k_empty[0]);
      }
      for (int t = 0; t < tiles && ok; ++t) {
        const int st = t & 1;
        ok = mbar_wait(&sm.v_full[st], (t >> 1) & 1, gave_up);
        if (ok && t + 1 < tiles) ok = mbar_wait(&sm.k_full[st ^ 1], ((t + 1) >> 1) & 1, gave_up);
        for (int half = 0; half < halves && ok; ++half) {
          ok = mbar_wait(&sm.p_full[half], t & 1, gave_up);
          if (!ok) break;
          tc_fence_after();
          const uint64_t vd = v_desc + st * kBuffer;
#pragma unroll
          for (int ks = 0; ks < kTile / 16; ++ks)
            mma_ts_f16(tmem + 256 + half * HD, tmem + half * 128 + ks * 8, vd + (ks >> 2) * (HD * 8) + (ks & 3) * 2, kPv, t > 0 || ks > 0);
          if (half == halves - 1) tc_commit(&sm.v_empty[st]);
          if (t + 1 < tiles) {
            scores(half, st ^ 1);
            if (half == halves - 1) tc_commit(&sm.k_empty[st ^ 1]);
          } else {
            tc_commit(&sm.o_full[half]);
          }
        }
      }
      if (!ok) {  // let what was issued end before the TMEM is given back
        tc_commit(&sm.spare);
        for (uint32_t i = 0; i < kWaitLimit && !mbar_try(&sm.spare, 0); ++i) {
        }
      }
    } else if (warp == 13 && tiles > 0) {
      // ---- copies of the codes, a lane per 16 tokens (lanes 8 and up idle) ---------
      const int piece = lane & 7;
      const uint32_t per_line = bs >> 4, bytes = HD * bs;
      const bool leads = lane < 8 && piece % per_line == 0;
      const uint32_t k_to = smem_addr(sm.k_raw) + piece * (HD * 16), v_to = smem_addr(sm.v_raw) + piece * (HD * 16);
      auto find = [&](int t) {
        const int tk = ((t0 + t) * kTile + 16 * piece) & ~(bs - 1);  // the block's first token
        int pg = -1;
        if (lane < 8 && t < tiles && tk < any_hi && tk + bs > any_lo) pg = __ldg(table + (tk >> p.bs_log2));
        return pg >= p.num_blocks ? -1 : pg;
      };
      auto scale = [&](const float* from, int pg, int64_t sb, int64_t sh) { return pg >= 0 ? __ldg(from + pg * sb + head * sh) : 0.f; };
      int page = find(0), page1 = find(1);
      float ks = scale(p.key_scale, page, p.ks_sb, p.ks_sh), vs = scale(p.value_scale, page, p.vs_sb, p.vs_sh);
      uint32_t k_sent = 0, v_sent = 0;
      for (int t = 0; t < tiles; ++t) {
        const uint32_t parity = (t & 1) ^ 1;
        const uint32_t led = __popc(__ballot_sync(0xffffffffu, leads && page >= 0)) * bytes;
        if (!mbar_wait_warp(&sm.kr_empty, parity, gave_up)) break;
        if (leads && page >= 0) {
          if (p.bs_log2 == 4)
            bulk_load(k_to, p.key + page * p.k_sb + head * p.k_sh, bytes, &sm.kr_full);
          else
            tensor_load(k_to, &kmap, head, page, &sm.kr_full);
        }
        // Their place was tile t - 4's.  Codes of tile t - 1 have been taken, so V of tile t - 2 has been
        // stored, for which the products of tile t - 4 had to be done, and its factors read before them.
        const float w = vref > 0.f ? vs / vref * 64.f : 0.f;
        const bool fine = page >= 0 && ks > 0.f && ks < INFINITY && w > 0.f && w < INFINITY;
        const uint32_t have = __ballot_sync(0xffffffffu, page >= 0) & 0xffu, plain = __ballot_sync(0xffffffffu, fine) & 0xffu;
        if (lane < 8) {
          sm.kfac[t & 3][piece] = ks;
          sm.vfac[t & 3][piece] = w;
          sm.vlog[t & 3][piece] = fine ? log2f(w) : 0.f;
          sm.vinv[t & 3][piece] = fine ? 1.f / w : 0.f;
        }
        if (lane == 0) {
          sm.have[t & 3] = have;
          sm.plain[t & 3] = plain;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect(&sm.kr_full, led);
        ++k_sent;
        if (!mbar_wait_warp(&sm.vr_empty, parity, gave_up)) break;
        if (leads && page >= 0) {
          if (p.bs_log2 == 4)
            bulk_load(v_to, p.value + page * p.v_sb + head * p.v_sh, bytes, &sm.vr_full);
          else
            tensor_load(v_to, &vmap, head, page, &sm.vr_full);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect(&sm.vr_full, led);
        ++v_sent;
        page = page1;
        ks = scale(p.key_scale, page, p.ks_sb, p.ks_sh);
        vs = scale(p.value_scale, page, p.vs_sb, p.vs_sh);
        page1 = find(t + 2);
      }
      // copies in flight end before the block does
      for (uint32_t z = 0; k_sent > 0 && z < kWaitLimit && !mbar_try(&sm.kr_full, (k_sent - 1) & 1); ++z) {
      }
      for (uint32_t z = 0; v_sent > 0 && z < kWaitLimit && !mbar_try(&sm.vr_full, (v_sent - 1) & 1); ++z) {
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    __syncwarp();
    tc_fence_after();
    tmem_free<512>(tmem);
  }
}

template <int HD, int CODE>
int launch_tc(const BlockAttnParams& p, cudaStream_t st) {
  constexpr int kBytes = sizeof(TcSmem<HD>);
  static_assert(kBytes <= 227 * 1024, "shared memory of a block");
  static bool set = false;
  if (!set) {
    const cudaError_t e = cudaFuncSetAttribute(block_attn_tc_kernel<HD, CODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return cuda_fail(e, "mak_block_attention");
    }
    set = true;
  }
  CUtensorMap maps[2] = {};
  if (p.bs_log2 > 4 && p.num_blocks > 0) {
    if (int rc = cache_map(&maps[0], p.key, p.k_sb, p.k_sh, p.num_blocks, p.nh, HD, 1 << p.bs_log2, false)) return rc;
    if (int rc = cache_map(&maps[1], p.value, p.v_sb, p.v_sh, p.num_blocks, p.nh, HD, 1 << p.bs_log2, false)) return rc;
  }
  const int64_t items = static_cast<int64_t>(p.num_rows) * p.group / kUnitRows + p.num_seqs;
  if (items * p.nh > 0x7fffffff) return fail(MAK_E_UNSUPPORTED, "mak_block_attention: too many rows for one call");
  return launch_pdl("mak_block_attention", block_attn_tc_kernel<HD, CODE>, dim3(static_cast<unsigned>(items * p.nh)), dim3(kThreads),
                    kBytes, st, p, maps[0], maps[1]);
}

}  // namespace

int launch_block_attn_tc(const BlockAttnParams& p, int head_dim, int code, cudaStream_t st) {
  if (head_dim == 64)
    return code == MAK_CODE_INT8 ? launch_tc<64, MAK_CODE_INT8>(p, st) : launch_tc<64, MAK_CODE_E4M3>(p, st);
  return code == MAK_CODE_INT8 ? launch_tc<128, MAK_CODE_INT8>(p, st) : launch_tc<128, MAK_CODE_E4M3>(p, st);
}

}  // namespace mak
