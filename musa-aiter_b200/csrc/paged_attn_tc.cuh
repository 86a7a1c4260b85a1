// The kernel for many rows of the attention over paged 16-bit caches, as its entry point calls it, and what it shares with that of
// the attention weights.
#pragma once

#include <utility>

#include "paged_attn.cuh"
#include "tcgen05.cuh"

namespace mak {

constexpr int64_t kPagedCounterBytes = 4096;  // of a workspace, at its beginning

int64_t paged_tc_partial_bytes();
int64_t paged_tc_plan_bytes();
bool paged_tc_fits(const PagedParams& p);
int paged_tc_box(int bs);  // tokens of the boxes that it loads
int launch_paged_tc(const PagedParams& p, int head_dim, bool bf16, const char* name, const CUtensorMap& k, const CUtensorMap& v, void* plan,
                    cudaStream_t st);
// A plane [num_blocks][block_size][num_heads][head_dim] as boxes of `tokens` tokens of one head, 64 columns of them, lines of
// 128 bytes swizzled.  `none`: an address for a plane without blocks.  False where strides make no tensor map.
bool paged_map(CUtensorMap* map, const uint16_t* base, int64_t sb, int64_t st, int64_t sh, int64_t num_blocks, int nh, int hd, int bs, bool bf16,
               int tokens, const void* none);
// A tensor map over 16-bit elements; strides in bytes.
bool paged_encode(CUtensorMap* map, const void* base, int rank, const int64_t* dims, const int64_t* strides, const uint32_t* box, bool bf16);

// Of the entry points.
int check_paged_cache(const mak_paged_cache_desc& c, bool values, const char* name);
int check_paged_workspace(const void* workspace, int64_t bytes, const char* name);
PagedParams paged_params(const mak_paged_cache_desc& c);
struct PagedSpace {
  int32_t* counters;
  void* plan;
  int64_t plan_bytes;
  float* partial;
};
PagedSpace paged_space(void* workspace);

// ---- of the kernels for many rows ----------------------------------------------
// f(0), f(1) ... f(N - 1) with the number as a constant.
template <int N, typename F, int... I>
__device__ __forceinline__ void steps_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void steps(F f) {
  steps_of<N>(f, std::make_integer_sequence<int, N>());
}

// A warp's wait for a phase of a barrier, asleep for up to 0.1 ms at a time: a loop of short looks takes issue slots from
// the warps that compute.  False when it did not complete in a second or so, or another role gave up.
__device__ __forceinline__ bool wait_warp(uint64_t* b, uint32_t parity, volatile int* gave_up) {
  uint32_t ok = 0;
  for (uint32_t i = 0; i < (1u << 14); ++i) {
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_addr(b)), "r"(parity), "r"(100000)
        : "memory");
    if (ok || *gave_up) break;
  }
  if (!ok) *gave_up = 1;
  return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 z, x, y;\n mov.b64 {%0, %1}, z;\n}"
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
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

}  // namespace mak
