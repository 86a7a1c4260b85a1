// Attention over a paged cache held in 8 bits with one scale per block and head,
// for few rows per sequence (decoding, checking drafted tokens).
//
// Mathematics.  With codes k, v and scales a, b per (block, head):
//   S[t] = scale * a(t) * (q . k[t]),   o = sum_t 2^(S'[t] - m) b(t) v[t] / sum_t 2^(S'[t] - m)
// with S' = S * log2(e) and the running maximum m.  The matrix instructions see
// the codes themselves, exact in f16; a multiplies a finished product and b the
// weight of a token, both in 32 bits, so a scale costs one multiplication per
// token and not one per element.
//
// q in f16: a row of bf16 is multiplied by a power of two that brings its
// largest magnitude to [2^14, 2^15); values that fall out of f16's normal range
// by that are below 2^-28 of the largest and err by at most 2^-39 of it.
// Weights in f16: p * b(t) / b_max * 2^15, at most 2^15, rounded once (2^-12
// relative); b_max is the largest scale met so far and rescales with m.  The
// sum of the weights is taken in 32 bits before that rounding.
//
// Layout.  A warp takes 128 tokens at a time.  K is the A operand of
// m16n8k16 with tokens as rows and V the A operand with head_dim as rows; the
// rows of q (the heads that share a cache head, times the rows of a sequence)
// are the 8 columns.  A lane's 16-byte load is 16 tokens of one head_dim row,
// so neighbouring lanes cover 4 rows of K (8 of V) in full sectors, and since
// the order of the contracted index is free as long as both operands agree, the
// loaded bytes become fragments in place: no shared memory for K or V.
//
// Work.  All (sequence, head, row group) units laid end to end as 128-token
// tiles are cut into equal runs, one per block, whatever the lengths; a block
// finds its run from the lengths alone.  A unit cut by that leaves partial sums
// (maximum, sum, accumulators) and the last block to arrive joins them.
#include "block_attn.cuh"

namespace mak {
namespace {

constexpr int kTile = 128;       // tokens per warp step
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxGrid = 148 * 8;  // blocks of the largest grid; the workspace has two partial sums for each
constexpr int kMaxRows = 16;
constexpr int kMaxDim = 256;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Asynchronous 16-byte copy to shared memory; bytes = 0 stores zeros and reads nothing.
__device__ __forceinline__ void copy_async(uint32_t to, const uint8_t* from, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Tiles of a unit of sequence v (at least one, so that empty rows are written).
__device__ __forceinline__ int unit_tiles(const SeqView& v) {
  const int t0 = v.lo / kTile, t1 = (v.hi + kTile - 1) / kTile;
  return t1 > t0 ? t1 - t0 : 1;
}

template <int NROWS>
__device__ __forceinline__ int64_t seq_work(const BlockAttnParams& p, const SeqView& v) {
  if (v.rows == 0) return 0;
  const int64_t groups = (static_cast<int64_t>(v.rows) * p.group + NROWS - 1) / NROWS;
  return groups * p.nh * unit_tiles(v);
}

// Each lane's loads go through its own slots of a ring: the lane that copies 16 bytes
// in is the one that reads them, so no barrier is needed, and the loads in flight cost
// no registers.  Loads come in groups of 4 per lane, head_dim / 16 groups for K of a tile
// and as many for V; each group that is consumed makes room for the one kRing further on,
// so V follows K and K of the next tile follows V.  The loops are rolled as far as the
// accumulators allow: unrolled whole, waiting for instructions cost more than the work.
constexpr int kRing = 4;  // groups

template <int HD, int NT>
struct Smem {
  static constexpr int kRows = 8 * NT;
  static constexpr int kPStride = 64 * 2 + 16;  // bytes between rows of the weights of 64 tokens
  union {
    uint4 ring[kWarps][4 * kRing][32];
    float acc[kWarps][kRows][HD + 1];
  };
  uint8_t weights[kWarps][kRows * kPStride];
  alignas(16) __half q[kRows][HD + 16];
  float m[kWarps][kRows];
  float l[kWarps][kRows];
  float qscale[kRows];
  int64_t scan[kWarps];
  int64_t begin_base;
  int begin_seq;
  int last;
};

template <int HD, int NT, int CODE>
__global__ void __launch_bounds__(kThreads, HD == 256 ? 1 : NT == 1 ? 3 : 2)
    block_attn_rows_kernel(const __grid_constant__ BlockAttnParams p) {
  constexpr int kRows = 8 * NT;
  constexpr int kSteps = HD / 16;  // groups of 4 loads of one lane per tile of K (and of V)
  extern __shared__ __align__(16) uint8_t raw[];
  Smem<HD, NT>& sm = *reinterpret_cast<Smem<HD, NT>*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  pdl_wait();
  pdl_trigger();

  // ---- the run of this block ------------------------------------------------
  const int per = (p.num_seqs + kThreads - 1) / kThreads;
  const int s0 = min(tid * per, p.num_seqs), s1 = min(s0 + per, p.num_seqs);
  int64_t mine = 0;
  for (int s = s0; s < s1; ++s) mine += seq_work<kRows>(p, seq_view(p, s));
  int64_t incl = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sm.scan[warp] = incl;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) incl += sm.scan[w];
    total += sm.scan[w];
  }
  int64_t chunk = (total + gridDim.x - 1) / gridDim.x;
  if (chunk < kWarps) chunk = kWarps;  // a tile for each warp before another block joins
  const int64_t w_begin = blockIdx.x * chunk;
  const int64_t w_end = min(w_begin + chunk, total);
  if (w_begin >= w_end) return;
  if (incl - mine <= w_begin && w_begin < incl) {
    int64_t base = incl - mine;
    for (int s = s0; s < s1; ++s) {
      const int64_t w = seq_work<kRows>(p, seq_view(p, s));
      if (w_begin < base + w) {
        sm.begin_seq = s;
        sm.begin_base = base;
        break;
      }
      base += w;
    }
  }
  __syncthreads();
  int seq = sm.begin_seq;
  int64_t base = sm.begin_base;

  int64_t w = w_begin;
  while (w < w_end) {
    SeqView v = seq_view(p, seq);
    int64_t sw = seq_work<kRows>(p, v);
    while (w >= base + sw) {
      base += sw;
      v = seq_view(p, ++seq);
      sw = seq_work<kRows>(p, v);
    }
    const int tiles = unit_tiles(v);
    const int64_t unit = (w - base) / tiles;
    const int64_t unit_w0 = base + unit * tiles;
    const int ta = static_cast<int>(w - unit_w0);
    const int tb = static_cast<int>(min(w_end - unit_w0, static_cast<int64_t>(tiles)));
    const int rows_total = v.rows * p.group;
    const int groups = (rows_total + kRows - 1) / kRows;
    const int head = static_cast<int>(unit / groups);
    const int row0 = static_cast<int>(unit % groups) * kRows;  // row i * group + j: row i, query head j of the group

    // ---- q rows: f16, contracted index in fragment order ---------------------
    __syncthreads();  // the last unit's readers are done
    {
      constexpr int kLanes = HD / 8;            // lanes of one row
      constexpr int kPass = kThreads / kLanes;  // rows at once
      const int part = tid % kLanes;
#pragma unroll
      for (int r0 = 0; r0 < kRows; r0 += kPass) {
        const int r = r0 + tid / kLanes;
        const bool on = r < kRows && row0 + r < rows_total;
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (on) {
          const int i = (row0 + r) / p.group, j = (row0 + r) % p.group;
          raw = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + (v.first + i) * p.q_sr +
                                                     (head * p.group + j) * p.q_sh + part * 8));
        }
        float x[8];
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (p.q_bf16) {
            x[2 * e] = __uint_as_float(words[e] << 16);
            x[2 * e + 1] = __uint_as_float(words[e] & 0xffff0000u);
          } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&words[e]));
            x[2 * e] = f.x;
            x[2 * e + 1] = f.y;
          }
          top = fmaxf(top, fmaxf(fabsf(x[2 * e]), fabsf(x[2 * e + 1])));
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // 2^up brings top to [2^14, 2^15); bf16 only, f16 is taken as it is
        int up = 0;
        if (p.q_bf16 && top > 0.f && top < __uint_as_float(0x7f800000u)) up = 14 - (ilogbf(top));
        const int up1 = up / 2, up2 = up - up1;  // two steps: 2^up itself may leave the exponent range
        const float f1 = __uint_as_float(static_cast<uint32_t>(127 + up1) << 23);
        const float f2 = __uint_as_float(static_cast<uint32_t>(127 + up2) << 23);
        if (r < kRows) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            // d = 16 ks + 4 jj + cc sits at 16 ks + 4 cc + jj
            const int d = part * 8 + e;
            sm.q[r][(d & ~15) + (d & 3) * 4 + ((d >> 2) & 3)] = __float2half_rn(x[e] * f1 * f2);
          }
          if (part == 0) sm.qscale[r] = ldexpf(p.scale_log2, -up);
        }
      }
    }
    __syncthreads();
    float qs[NT][2];
    int lo[NT][2], hi[NT][2];
    int all_lo = 0, all_hi = 0x7fffffff, any_lo = 0x7fffffff, any_hi = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = n * 8 + 2 * c + e;
        qs[n][e] = sm.qscale[r];
        lo[n][e] = hi[n][e] = 0;
        if (row0 + r < rows_total) row_range(p, v, (row0 + r) / p.group, &lo[n][e], &hi[n][e]);
      }
    }
    {  // tokens that all rows of the group see, and that any sees
      const int i0 = row0 / p.group, i1 = min(row0 + kRows, rows_total) - 1;
      int l0, h0, l1, h1;
      row_range(p, v, i0, &l0, &h0);
      row_range(p, v, i1 / p.group, &l1, &h1);
      all_lo = l1;
      all_hi = h0;
      any_lo = l0;
      any_hi = h1;
    }

    float acc[NT][HD / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][i][e] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
    float vref = 0.f;
    const int32_t* table = p.tables + seq * p.table_stride;
    const uint8_t* kbase = p.key + head * p.k_sh;
    const uint8_t* vbase = p.value + head * p.v_sh;
    const int bs = 1 << p.bs_log2;
    const int tile0 = v.hi > v.lo ? v.lo / kTile : 0;
    // tiles of this warp: t, t + kWarps, ... below t_end, all of which some row sees
    int t = ta + warp, t_end = tb;
    if (any_hi > any_lo) {
      t_end = min(t_end, (any_hi + kTile - 1) / kTile - tile0);
      const int skip = any_lo / kTile - tile0 - t;
      if (skip > 0) t += (skip + kWarps - 1) / kWarps * kWarps;
    } else {
      t_end = 0;
    }
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(&sm.ring[warp][0][lane]));
    // Block of this lane's 16 tokens of K (chunk g) of tile i, -1 where there is none.
    auto find = [&](int i) {
      const int kt = (tile0 + i) * kTile + 16 * g;
      int page = -1;
      if (i < t_end && kt < any_hi && kt + 16 > any_lo) page = __ldg(table + (kt >> p.bs_log2));
      return page >= p.num_blocks ? -1 : page;
    };
    int page = find(t), page1 = find(t + kWarps);
    float ksc = 0.f, vsc = 0.f;
    auto scales = [&](int pg, float* a, float* b) {
      *a = *b = 0.f;
      if (pg >= 0) {
        *a = __ldg(p.key_scale + pg * p.ks_sb + head * p.ks_sh);
        *b = __ldg(p.value_scale + pg * p.vs_sb + head * p.vs_sh);
      }
    };
    const int in_block = (16 * g) & (bs - 1);  // a tile starts at a block's start
    const uint8_t* kp = page >= 0 ? kbase + page * p.k_sb + in_block + c * bs : kbase;
    uint32_t kn = page >= 0 ? 16 : 0;
    // group i of K: rows 16 i + 4 jj + c of this lane's chunk
    auto load_k = [&](int slot, int i, const uint8_t* from, uint32_t bytes) {
      const uint8_t* at = from + (bytes ? 16 * i * bs : 0);
      const int step = bytes ? 4 * bs : 0;
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) copy_async(ring + (4 * slot + jj) * 512, at + jj * step, bytes);
    };
    if (t < t_end) {
#pragma unroll
      for (int i = 0; i < kRing; ++i) {
        load_k(i, i, kp, kn);
        copy_commit();
      }
      scales(page, &ksc, &vsc);
    }

    for (; t < t_end; t += kWarps) {
      const int tok = (tile0 + t) * kTile;
      const int kt = tok + 16 * g;
      // V of this tile: chunk 4 hf + c
      const uint8_t* vp[2];
      uint32_t vn[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int vpage = __shfl_sync(0xffffffffu, page, (4 * hf + c) * 4);
        vn[hf] = vpage >= 0 ? 16 : 0;
        vp[hf] = vpage >= 0 ? vbase + vpage * p.v_sb + ((64 * hf + 16 * c) & (bs - 1)) + g * bs : vbase;
      }
      // the next tile
      const int page2 = find(t + 2 * kWarps);
      const bool more = t + kWarps < t_end;
      const uint8_t* kp1 = page1 >= 0 ? kbase + page1 * p.k_sb + in_block + c * bs : kbase;
      const uint32_t kn1 = page1 >= 0 ? 16 : 0;
      float ksc1, vsc1;
      scales(page1, &ksc1, &vsc1);

      float s[NT][8][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][i][e] = 0.f;
      // group i of V: rows 32 pair + 8 e + g of chunk 4 hf + c
      auto load_v = [&](int slot, int hf, int pair) {
        const uint8_t* at = hf ? vp[1] : vp[0];
        const uint32_t bytes = hf ? vn[1] : vn[0];
        const int step = bytes ? 8 * bs : 0;
        at += 4 * pair * step;
#pragma unroll
        for (int e = 0; e < 4; ++e) copy_async(ring + (4 * slot + e) * 512, at + e * step, bytes);
      };
#pragma unroll 1
      for (int k0 = 0; k0 < kSteps; k0 += kRing) {
#pragma unroll
        for (int u = 0; u < kRing; ++u) {
          const int ks = k0 + u;
          copy_wait<kRing - 1>();
          uint4 x[4];
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) x[jj] = sm.ring[warp][4 * u + jj][lane];
          uint2 qf[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) qf[n] = *reinterpret_cast<const uint2*>(&sm.q[n * 8 + g][ks * 16 + c * 4]);
#pragma unroll
          for (int wd = 0; wd < 4; ++wd) {
            const uint32_t x0 = (&x[0].x)[wd], x1 = (&x[1].x)[wd], x2 = (&x[2].x)[wd], x3 = (&x[3].x)[wd];
            uint32_t a[4], b[4];
            // tokens 4 wd, 4 wd + 1 -> row pair (g, g + 8) of tile 2 wd
            codes4_to_f16<CODE>(__byte_perm(x0, x1, 0x5140), &a[0], &a[1]);
            codes4_to_f16<CODE>(__byte_perm(x2, x3, 0x5140), &a[2], &a[3]);
            codes4_to_f16<CODE>(__byte_perm(x0, x1, 0x7362), &b[0], &b[1]);
            codes4_to_f16<CODE>(__byte_perm(x2, x3, 0x7362), &b[2], &b[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_f16(s[n][2 * wd], a[0], a[1], a[2], a[3], qf[n].x, qf[n].y);
              mma_f16(s[n][2 * wd + 1], b[0], b[1], b[2], b[3], qf[n].x, qf[n].y);
            }
          }
          if (k0 + kRing < kSteps)
            load_k(u, ks + kRing, kp, kn);
          else
            load_v(u, u / (kSteps / 2), u % (kSteps / 2));
          copy_commit();
        }
      }
      // s[n][i][2 * r + e]: token kt + 2 i + r, column 2 c + e
      const bool whole = tok >= all_lo && tok + kTile <= all_hi;
      float vmax = fabsf(vsc);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
      const float vnew = fmaxf(vref, vmax);
      const float vkeep = vnew > vref ? vref / vnew : 1.f;
      const float vfac = vnew > 0.f ? vsc / vnew * 32768.f : 0.f;
      vref = vnew;
      bool moved = false;
      float keep[NT][2];
      uint32_t wt[NT][2][8];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2] = {qs[n][0] * ksc, qs[n][1] * ksc};
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = s[n][i][e] * f[e & 1];
            if (!whole || page < 0) {
              const int at = kt + 2 * i + (e >> 1);
              if (page < 0 || at < lo[n][e & 1] || at >= hi[n][e & 1]) x = -INFINITY;
            }
            s[n][i][e] = x;
            top[e & 1] = fmaxf(top[e & 1], x);
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], o));
          const float mn = fmaxf(m[n][e], top[e]);
          const float ms = mn == -INFINITY ? 0.f : mn;
          keep[n][e] = exp2_fast(m[n][e] - ms);
          l[n][e] *= keep[n][e];
          keep[n][e] *= vkeep;
          moved |= keep[n][e] != 1.f;
          m[n][e] = mn;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float w0 = exp2_fast(s[n][i][e] - ms), w1 = exp2_fast(s[n][i][2 + e] - ms);
            l[n][e] += w0 + w1;
            wt[n][e][i] = pack_f16(w0 * vfac, w1 * vfac);
          }
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < HD / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][i][e] *= keep[n][e & 1];
      }
      uint8_t* wrow = sm.weights[warp];
#pragma unroll 1
      for (int hf = 0; hf < 2; ++hf) {
        // weights of 64 tokens from the score layout to the operand layout
        if ((g >> 2) == hf) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint4* dst = reinterpret_cast<uint4*>(wrow + (n * 8 + 2 * c + e) * Smem<HD, NT>::kPStride + (g & 3) * 32);
              dst[0] = make_uint4(wt[n][e][0], wt[n][e][1], wt[n][e][2], wt[n][e][3]);
              dst[1] = make_uint4(wt[n][e][4], wt[n][e][5], wt[n][e][6], wt[n][e][7]);
            }
        }
        __syncwarp();
        uint32_t pf[NT][4][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4* src = reinterpret_cast<const uint4*>(wrow + (n * 8 + g) * Smem<HD, NT>::kPStride + c * 32);
          const uint4 a = src[0], b = src[1];
          pf[n][0][0] = a.x, pf[n][0][1] = a.y, pf[n][1][0] = a.z, pf[n][1][1] = a.w;
          pf[n][2][0] = b.x, pf[n][2][1] = b.y, pf[n][3][0] = b.z, pf[n][3][1] = b.w;
        }
        __syncwarp();
        // tokens of this chunk that some row sees; the others' codes may be anything and count as 0
        const int vt = tok + 64 * hf + 16 * c;
        const int first = any_lo - vt, last = any_hi - vt;
#pragma unroll
        for (int i2 = 0; i2 < kSteps / 2; ++i2) {
          // HD 64 has two groups to a half: their slots go by the half
          const int slot = kSteps / 2 >= kRing ? i2 % kRing : hf * (kSteps / 2) + i2;
          copy_wait<kRing - 1>();
          uint4 x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = sm.ring[warp][4 * slot + e][lane];
#pragma unroll
          for (int i1 = 0; i1 < 2; ++i1) {
            const int i = 2 * i2 + i1;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
              uint32_t y0 = (&x[2 * i1].x)[q4], y1 = (&x[2 * i1 + 1].x)[q4];
              if (!whole) {
                uint32_t mask = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b)
                  if (4 * q4 + b >= first && 4 * q4 + b < last) mask |= 0xffu << (8 * b);
                y0 &= mask;
                y1 &= mask;
              }
              uint32_t a[4];
              codes4_to_f16<CODE>(y0, &a[0], &a[2]);
              codes4_to_f16<CODE>(y1, &a[1], &a[3]);
#pragma unroll
              for (int n = 0; n < NT; ++n) mma_f16(acc[n][i], a[0], a[1], a[2], a[3], pf[n][q4][0], pf[n][q4][1]);
            }
          }
          const int next = hf * (kSteps / 2) + i2 + kRing;  // group of V, or past the last one of the next tile's K
          if (next < kSteps)
            load_v(slot, next / (kSteps / 2), next % (kSteps / 2));
          else if (more)
            load_k(slot, next - kSteps, kp1, kn1);
          copy_commit();
        }
      }
      page = page1, page1 = page2;
      kp = kp1, kn = kn1;
      ksc = ksc1, vsc = vsc1;
    }
    copy_wait<0>();

    // ---- join the warps --------------------------------------------------------
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o);
    __syncthreads();  // the ring is read, its space takes the accumulators
    const float unit_scale = vref * (1.f / 32768.f);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sm.acc[warp][n * 8 + 2 * c + (e & 1)][16 * i + g + 8 * (e >> 1)] = acc[n][i][e] * unit_scale;
      if (g == 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sm.m[warp][n * 8 + 2 * c + e] = m[n][e];
          sm.l[warp][n * 8 + 2 * c + e] = l[n][e];
        }
      }
    }
    __syncthreads();
    const bool single = ta == 0 && tb == tiles;
    const int first_block = static_cast<int>(unit_w0 / chunk);
    const int last_block = static_cast<int>((unit_w0 + tiles - 1) / chunk);
    const int live = min(kRows, rows_total - row0);
    constexpr int kStep = kRows * (HD + 2);  // floats of one partial sum
    float* part = nullptr;
    if (!single) part = p.partial + (2 * static_cast<int64_t>(blockIdx.x) + (unit_w0 > w_begin ? 1 : 0)) * kStep;
    for (int idx = tid; idx < live * HD; idx += kThreads) {
      const int r = idx / HD, d = idx % HD;
      float mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) mx = fmaxf(mx, sm.m[x][r]);
      const float ms = mx == -INFINITY ? 0.f : mx;
      float o = 0.f, sum = 0.f;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        const float k = exp2_fast(sm.m[x][r] - ms);
        o += k * sm.acc[x][r][d];
        sum += k * sm.l[x][r];
      }
      if (single) {
        const int i = (row0 + r) / p.group, j = head * p.group + (row0 + r) % p.group;
        const float y = sum > 0.f || sum != sum ? o / sum : 0.f;
        const int64_t at = (v.first + i) * p.o_sr + j * p.o_sh + d;
        if (p.q_bf16)
          reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
        else
          reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(y);
        if (d == 0 && p.lse != nullptr)
          p.lse[static_cast<int64_t>(v.first + i) * p.nh * p.group + j] =
              sum > 0.f || sum != sum ? (mx + log2f(sum)) * 0.69314718055994531f : -INFINITY;
      } else {
        part[r * HD + d] = o;
        if (d == 0) {
          part[kRows * HD + r] = mx;
          part[kRows * HD + kRows + r] = sum;
        }
      }
    }
    if (!single) {
      __threadfence();
      __syncthreads();
      const int slot0 = 2 * first_block + (unit_w0 > first_block * chunk ? 1 : 0);
      const int blocks = last_block - first_block + 1;
      if (tid == 0) sm.last = atomicAdd(p.counters + slot0, 1) == blocks - 1;
      __syncthreads();
      if (sm.last) {
        __threadfence();
        for (int idx = tid; idx < live * (HD / 4); idx += kThreads) {
          const int r = idx / (HD / 4), d = idx % (HD / 4) * 4;
          float mx = -INFINITY, sum = 0.f;
          float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
          for (int b = first_block; b <= last_block; ++b) {
            const float* src = p.partial + (2 * static_cast<int64_t>(b) + (unit_w0 > b * chunk ? 1 : 0)) * kStep;
            const float pm = __ldcg(src + kRows * HD + r), pl = __ldcg(src + kRows * HD + kRows + r);
            const float4 po = __ldcg(reinterpret_cast<const float4*>(src + r * HD + d));
            const float mn = fmaxf(mx, pm);
            const float ms = mn == -INFINITY ? 0.f : mn;
            const float k0 = exp2_fast(mx - ms), k1 = exp2_fast(pm - ms);
            o[0] = o[0] * k0 + po.x * k1;
            o[1] = o[1] * k0 + po.y * k1;
            o[2] = o[2] * k0 + po.z * k1;
            o[3] = o[3] * k0 + po.w * k1;
            sum = sum * k0 + pl * k1;
            mx = mn;
          }
          const int i = (row0 + r) / p.group, j = head * p.group + (row0 + r) % p.group;
          const bool some = sum > 0.f || sum != sum;
          const int64_t at = (v.first + i) * p.o_sr + j * p.o_sh + d;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = some ? o[e] / sum : 0.f;
            if (p.q_bf16)
              reinterpret_cast<__nv_bfloat16*>(p.out)[at + e] = __float2bfloat16_rn(y);
            else
              reinterpret_cast<__half*>(p.out)[at + e] = __float2half_rn(y);
          }
          if (d == 0 && p.lse != nullptr)
            p.lse[static_cast<int64_t>(v.first + i) * p.nh * p.group + j] =
                some ? (mx + log2f(sum)) * 0.69314718055994531f : -INFINITY;
        }
        if (tid == 0) p.counters[slot0] = 0;
      }
    }
    w = unit_w0 + tb;
  }
}

template <int HD, int NT, int CODE>
int launch_rows(const BlockAttnParams& p, cudaStream_t st) {
  const void* fn = reinterpret_cast<const void*>(&block_attn_rows_kernel<HD, NT, CODE>);
  constexpr int kBytes = sizeof(Smem<HD, NT>);
  static int per_sm = 0;
  if (per_sm == 0) {
    const cudaError_t e =
        cudaFuncSetAttribute(block_attn_rows_kernel<HD, NT, CODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return cuda_fail(e, "mak_block_attention");
    }
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, kThreads, kBytes) != cudaSuccess || n <= 0) n = 1;
    per_sm = n;
  }
  int64_t grid = per_sm * sm_count();
  if (grid > kMaxGrid) grid = kMaxGrid;
  // no more blocks than there can be work for: kWarps tiles each
  const int64_t seq_tiles = ((static_cast<int64_t>(p.max_blocks) << p.bs_log2) + kTile - 1) / kTile + 1;
  const int64_t groups = static_cast<int64_t>(p.num_rows) * p.group / (8 * NT) + p.num_seqs;
  const int64_t most = (groups * p.nh * seq_tiles + kWarps - 1) / kWarps;
  if (most < grid) grid = most;
  return launch_pdl("mak_block_attention", block_attn_rows_kernel<HD, NT, CODE>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), kBytes, st, p);
}

template <int HD, int NT>
int launch_rows_code(const BlockAttnParams& p, int code, cudaStream_t st) {
  return code == MAK_CODE_INT8 ? launch_rows<HD, NT, MAK_CODE_INT8>(p, st) : launch_rows<HD, NT, MAK_CODE_E4M3>(p, st);
}

constexpr int64_t kCounterBytes = (2 * kMaxGrid * 4 + 255) / 256 * 256;

}  // namespace

int launch_block_attn_tc(const BlockAttnParams& p, int head_dim, int code, cudaStream_t st);

int check_block_cache(const mak_block_cache_desc& c, const char* name) {
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
    return fail(MAK_E_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256, got %d", name, c.head_dim);
  if (c.block_size != 16 && c.block_size != 32 && c.block_size != 64 && c.block_size != 128)
    return fail(MAK_E_UNSUPPORTED, "%s: block_size must be 16, 32, 64 or 128, got %d", name, c.block_size);
  if (c.code_type != MAK_CODE_INT8 && c.code_type != MAK_CODE_E4M3)
    return fail(MAK_E_INVALID, "%s: unknown code type %d", name, c.code_type);
  if (c.num_seqs < 0 || c.num_blocks < 0 || c.max_blocks < 0 || c.num_rows < 0 || c.num_heads <= 0)
    return fail(MAK_E_INVALID, "%s: negative size", name);
  if (c.num_seqs > 0x7fffffff || c.num_blocks > 0x7fffffff || c.num_rows > 0x7fffffff ||
      c.max_blocks > 0x7fffffff / c.block_size)
    return fail(MAK_E_UNSUPPORTED, "%s: sequences, blocks, rows and tokens of a sequence are 32-bit counts", name);
  if (c.num_seqs > 0 && (c.context_lens == nullptr || (c.max_blocks > 0 && c.block_tables == nullptr)))
    return fail(MAK_E_INVALID, "%s: null block_tables or context_lens", name);
  if (c.num_blocks > 0 && (c.key == nullptr || c.value == nullptr || c.key_scale == nullptr || c.value_scale == nullptr))
    return fail(MAK_E_INVALID, "%s: null cache", name);
  const uint64_t bits = reinterpret_cast<uintptr_t>(c.key) | reinterpret_cast<uintptr_t>(c.value) |
                        static_cast<uint64_t>(c.key_stride_block | c.key_stride_head | c.value_stride_block | c.value_stride_head);
  if (bits & 15) return fail(MAK_E_INVALID, "%s: caches need 16-byte aligned addresses and block / head strides", name);
  return MAK_OK;
}

}  // namespace mak

using namespace mak;

extern "C" int64_t mak_block_attention_workspace_bytes(void) {
  return kCounterBytes + static_cast<int64_t>(2 * kMaxGrid) * kMaxRows * (kMaxDim + 2) * 4;
}

extern "C" int mak_block_attention(const mak_block_attn_desc* d, void* stream) {
  const char* name = "mak_block_attention";
  if (d == nullptr) return fail(MAK_E_INVALID, "%s: null descriptor", name);
  const mak_block_cache_desc& c = d->cache;
  if (int rc = check_block_cache(c, name)) return rc;
  if (d->q_dtype != MAK_DT_F16 && d->q_dtype != MAK_DT_BF16)
    return fail(MAK_E_UNSUPPORTED, "%s: q must be float16 or bfloat16", name);
  if (d->num_q_heads <= 0 || d->num_q_heads % c.num_heads)
    return fail(MAK_E_INVALID, "%s: %d query heads over %d cache heads", name, d->num_q_heads, c.num_heads);
  if (d->window < 0 || (d->window > 0 && !d->causal))
    return fail(MAK_E_INVALID, "%s: a window needs causal attention", name);
  if (c.num_seqs == 0 || c.num_rows == 0) return MAK_OK;
  if (d->q == nullptr || d->out == nullptr) return fail(MAK_E_INVALID, "%s: null q or out", name);
  if ((reinterpret_cast<uintptr_t>(d->q) & 15) || ((d->q_stride_row | d->q_stride_head) & 7))
    return fail(MAK_E_INVALID, "%s: q needs 16-byte aligned rows", name);
  if (d->workspace == nullptr || d->workspace_bytes < mak_block_attention_workspace_bytes())
    return fail(MAK_E_WORKSPACE, "%s: workspace missing or too small", name);
  BlockAttnParams p = {};
  p.key = static_cast<const uint8_t*>(c.key);
  p.value = static_cast<const uint8_t*>(c.value);
  p.key_scale = c.key_scale;
  p.value_scale = c.value_scale;
  p.k_sb = c.key_stride_block, p.k_sh = c.key_stride_head;
  p.v_sb = c.value_stride_block, p.v_sh = c.value_stride_head;
  p.ks_sb = c.key_scale_stride_block, p.ks_sh = c.key_scale_stride_head;
  p.vs_sb = c.value_scale_stride_block, p.vs_sh = c.value_scale_stride_head;
  p.tables = c.block_tables;
  p.ctx_lens = c.context_lens;
  p.starts = c.cu_seqlens;
  p.table_stride = c.table_stride;
  p.num_blocks = c.num_blocks;
  p.q = d->q, p.out = d->out, p.lse = d->lse;
  p.q_sr = d->q_stride_row, p.q_sh = d->q_stride_head, p.o_sr = d->out_stride_row, p.o_sh = d->out_stride_head;
  p.num_seqs = static_cast<int32_t>(c.num_seqs);
  p.max_blocks = static_cast<int32_t>(c.max_blocks);
  p.num_rows = static_cast<int32_t>(c.num_rows);
  p.nh = c.num_heads;
  p.group = d->num_q_heads / c.num_heads;
  p.bs_log2 = c.block_size == 16 ? 4 : c.block_size == 32 ? 5 : c.block_size == 64 ? 6 : 7;
  p.q_bf16 = d->q_dtype == MAK_DT_BF16;
  p.causal = d->causal != 0;
  p.window = d->window;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.counters = static_cast<int32_t*>(d->workspace);
  p.partial = reinterpret_cast<float*>(static_cast<char*>(d->workspace) + kCounterBytes);
  cudaStream_t st = as_stream(stream);
  // Rows that share a cache head, on average: more than 8 fill a second set of columns.
  const int64_t rows = c.num_rows * p.group / c.num_seqs;
  if (rows >= 64 && c.head_dim <= 128) return launch_block_attn_tc(p, c.head_dim, c.code_type, st);
  const bool wide = rows > 8 && c.head_dim < 256;
  if (c.head_dim == 64) return wide ? launch_rows_code<64, 2>(p, c.code_type, st) : launch_rows_code<64, 1>(p, c.code_type, st);
  if (c.head_dim == 128) return wide ? launch_rows_code<128, 2>(p, c.code_type, st) : launch_rows_code<128, 1>(p, c.code_type, st);
  return launch_rows_code<256, 1>(p, c.code_type, st);
}
