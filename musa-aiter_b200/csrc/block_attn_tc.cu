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
//   warps 8-11       load codes, convert to f16, store to shared memory
//   warp 12          one thread issues all tcgen05.mma
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
  float kfac[4][8], vfac[4][8];          // per 16 tokens of a tile
  uint32_t chunks[4];                    // 16-token pieces that have a page: 0-3 in byte 0, 4-7 in byte 1
  alignas(8) uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], spare;
  uint32_t tmem;
  float vmax[4];
  int unit_seq, unit_tile;
  int gave_up;
};

template <int HD, int CODE>
__global__ void __launch_bounds__(kThreads, 1) block_attn_tc_kernel(const __grid_constant__ BlockAttnParams p) {
  extern __shared__ uint8_t raw[];
  TcSmem<HD>& sm = *reinterpret_cast<TcSmem<HD>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
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
    regs_up<176>();  // with 104 and 56 below: what the block was launched with
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
        const float* vf = sm.vfac[t & 3];
        const uint32_t have = (sm.chunks[t & 3] & 0xfu) | ((sm.chunks[t & 3] >> 4) & 0xf0u);
        const bool whole = tok >= all_lo && tok + kTile <= all_hi && have == 0xffu;
        // the row's scores stay in registers: scaled, then exponentiated
        uint32_t x[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld(s_at + c * 32, x[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_wait(x[c]);
        if (whole) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float f = kf[c] * qs;
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              uint32_t* at = &x[c >> 1][(c & 1) * 16 + e];
              const float2 y = mul2(make_float2(__uint_as_float(at[0]), __uint_as_float(at[1])), make_float2(f, f));
              at[0] = __float_as_uint(y.x);
              at[1] = __float_as_uint(y.y);
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float f = kf[c] * qs;
            // columns [from, to) of these 16 are seen
            const int first = tok + 16 * c;
            const int from = lo - first, to = (have >> c) & 1 ? hi - first : 0;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              uint32_t& at = x[c >> 1][(c & 1) * 16 + e];
              at = e >= from && e < to ? __float_as_uint(__uint_as_float(at) * f) : 0xff800000u;
            }
          }
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            tops[c] = fmaxf(fmaxf(tops[c], __uint_as_float(x[c][e])), __uint_as_float(x[c][e + 1]));
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
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
        const float2 shift = make_float2(-ms, -ms);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t y[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float w = vf[2 * c + (e >> 4)];
            float2 a = add2(make_float2(__uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1])), shift);
            a.x = exp2_fast(a.x);
            a.y = exp2_fast(a.y);
            sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], a);
            a = mul2(a, make_float2(w, w));
            y[e >> 1] = pack_f16(a.x, a.y);
          }
          tmem_st(s_at + c * 16, y);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
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
    regs_down<104>();
    // ---- codes to f16 in shared memory -------------------------------------------
    const int w = warp - 8;
    const int dlo = lane & 7, chunk = (w & 1) * 4 + (lane >> 3);
    const int d0 = (w >> 1) * (HD / 2) + dlo;
    constexpr int kIts = HD / 16;
    const uint8_t* kb = p.key + head * p.k_sh + static_cast<int64_t>(d0) * bs;
    const uint8_t* vb = p.value + head * p.v_sh + static_cast<int64_t>(d0) * bs;
    const uint32_t to = (chunk >> 2) * (HD * 128) + d0 * 128;
    const uint32_t c0 = ((((chunk & 3) * 2) ^ dlo) << 4), c1 = ((((chunk & 3) * 2 + 1) ^ dlo) << 4);
    uint4 kx[kIts], vx[kIts];
    float ks = 0.f, vs = 0.f;
    int page = -1, next_page = -1;
    auto find = [&](int t) {
      const int kt = (t0 + t) * kTile + 16 * chunk;
      int pg = -1;
      if (t < tiles && kt < any_hi && kt + 16 > any_lo) pg = __ldg(table + (kt >> p.bs_log2));
      return pg >= p.num_blocks ? -1 : pg;
    };
    auto fetch = [&](const uint8_t* base, int64_t stride, int t, int pg, uint4(&x)[kIts]) {
      const int kt = (t0 + t) * kTile + 16 * chunk;
      const uint8_t* src = base + pg * stride + (kt & (bs - 1));
#pragma unroll
      for (int it = 0; it < kIts; ++it) {
        x[it] = make_uint4(0, 0, 0, 0);
        if (pg >= 0) x[it] = __ldg(reinterpret_cast<const uint4*>(src + static_cast<int64_t>(it * 8) * bs));
      }
    };
    auto store = [&](uint8_t* dst, int t, const uint4(&x)[kIts]) {
      const int kt = (t0 + t) * kTile + 16 * chunk;
      uint32_t mask[4] = {~0u, ~0u, ~0u, ~0u};
      const bool edge = kt < any_lo || kt + 16 > any_hi;
      if (edge) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          mask[q] = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (kt + 4 * q + b >= any_lo && kt + 4 * q + b < any_hi) mask[q] |= 0xffu << (8 * b);
        }
      }
      auto convert = [&](int it, uint4 z) {
        uint32_t y[8];
        codes4_to_f16<CODE>(z.x, &y[0], &y[1]);
        codes4_to_f16<CODE>(z.y, &y[2], &y[3]);
        codes4_to_f16<CODE>(z.z, &y[4], &y[5]);
        codes4_to_f16<CODE>(z.w, &y[6], &y[7]);
        uint8_t* line = dst + to + it * 1024;
        *reinterpret_cast<uint4*>(line + c0) = make_uint4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<uint4*>(line + c1) = make_uint4(y[4], y[5], y[6], y[7]);
      };
      if (edge) {
#pragma unroll
        for (int it = 0; it < kIts; ++it)
          convert(it, make_uint4(x[it].x & mask[0], x[it].y & mask[1], x[it].z & mask[2], x[it].w & mask[3]));
      } else {
#pragma unroll
        for (int it = 0; it < kIts; ++it) convert(it, x[it]);
      }
    };
    auto scales = [&]() {
      ks = vs = 0.f;
      if (page >= 0) {
        ks = __ldg(p.key_scale + page * p.ks_sb + head * p.ks_sh);
        vs = __ldg(p.value_scale + page * p.vs_sb + head * p.vs_sh);
      }
    };
    if (tiles > 0) {
      page = find(0);
      next_page = find(1);
      fetch(kb, p.k_sb, 0, page, kx);
      fetch(vb, p.v_sb, 0, page, vx);
      scales();
    }
    for (int t = 0; t < tiles; ++t) {
      const int st = t & 1;
      const uint32_t parity = ((t >> 1) & 1) ^ 1;
      if (!mbar_wait_warp(&sm.k_empty[st], parity, gave_up)) break;
      // the factors of tile t - 4 were last read before tile t - 2's scores were issued
      if (dlo == 0 && w < 2) {
        sm.kfac[t & 3][chunk] = ks;
        sm.vfac[t & 3][chunk] = vref > 0.f ? vs / vref * 64.f : 0.f;
      }
      const uint32_t votes = __ballot_sync(0xffffffffu, page >= 0);
      if (lane == 0 && w < 2) {
        const uint32_t bits = (votes & 1) | ((votes >> 7) & 2) | ((votes >> 14) & 4) | ((votes >> 21) & 8);
        reinterpret_cast<uint8_t*>(&sm.chunks[t & 3])[w] = static_cast<uint8_t>(bits);
      }
      store(sm.k[st], t, kx);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.k_full[st]);
      page = next_page;
      if (t + 1 < tiles) fetch(kb, p.k_sb, t + 1, page, kx);
      next_page = find(t + 2);
      if (!mbar_wait_warp(&sm.v_empty[st], parity, gave_up)) break;
      store(sm.v[st], t, vx);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.v_full[st]);
      if (t + 1 < tiles) {
        fetch(vb, p.v_sb, t + 1, page, vx);
        scales();
      }
    }
  } else {
    regs_down<56>();
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
  constexpr int kBytes = sizeof(TcSmem<HD>) + 1024;
  static bool set = false;
  if (!set) {
    const cudaError_t e = cudaFuncSetAttribute(block_attn_tc_kernel<HD, CODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return cuda_fail(e, "mak_block_attention");
    }
    set = true;
  }
  const int64_t items = static_cast<int64_t>(p.num_rows) * p.group / kUnitRows + p.num_seqs;
  if (items * p.nh > 0x7fffffff) return fail(MAK_E_UNSUPPORTED, "mak_block_attention: too many rows for one call");
  return launch_pdl("mak_block_attention", block_attn_tc_kernel<HD, CODE>, dim3(static_cast<unsigned>(items * p.nh)), dim3(kThreads),
                    kBytes, st, p);
}

}  // namespace

int launch_block_attn_tc(const BlockAttnParams& p, int head_dim, int code, cudaStream_t st) {
  if (head_dim == 64)
    return code == MAK_CODE_INT8 ? launch_tc<64, MAK_CODE_INT8>(p, st) : launch_tc<64, MAK_CODE_E4M3>(p, st);
  return code == MAK_CODE_INT8 ? launch_tc<128, MAK_CODE_INT8>(p, st) : launch_tc<128, MAK_CODE_E4M3>(p, st);
}

}  // namespace mak
