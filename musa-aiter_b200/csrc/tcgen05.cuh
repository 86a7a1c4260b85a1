// Inline PTX of the tcgen05 tensor cores, tensor memory, mbarriers and bulk copies.
#pragma once

#include <cstdint>

namespace mak {

constexpr uint32_t kWaitLimit = 1u << 22;  // polls of a barrier before a block gives up

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(count));
}
__device__ __forceinline__ void mbar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_addr(b)), "r"(parity)
      : "memory");
  return ok != 0;
}
// False when the barrier did not complete within the limit, or another role gave up.
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, volatile int* gave_up) {
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    if (mbar_try(b, parity)) return true;
    if ((i & 255) == 255 && *gave_up) return false;
  }
  *gave_up = 1;
  return false;
}
// The same for a whole warp, with one answer.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* b, uint32_t parity, volatile int* gave_up) {
  return __all_sync(0xffffffffu, mbar_wait(b, parity, gave_up));
}

// For warps with time to spare: between looks they leave the issue slots to others.
__device__ __forceinline__ bool mbar_wait_warp_idle(uint64_t* b, uint32_t parity, volatile int* gave_up) {
  bool ok = false;
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    ok = mbar_try(b, parity);
    if (ok) break;
    __nanosleep(100);
    if ((i & 255) == 255 && *gave_up) break;
  }
  if (!ok) *gave_up = 1;
  return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(b)) : "memory");
}
// Generic writes to shared memory become visible to the tensor cores and the copy engine.
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Registers of the threads of a warpgroup from here on.
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int COLS>
__device__ __forceinline__ void tmem_alloc(uint32_t* at) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(at)), "n"(COLS) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <int COLS>
__device__ __forceinline__ void tmem_free(uint32_t at) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "n"(COLS));
}

// D (TMEM) = or += A (shared memory) * B (shared memory)
#define MAK_MMA_SS(NAME, KIND)                                                                                                 \
  __device__ __forceinline__ void NAME(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {                     \
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::" KIND " [%0], %1, %2, %3, p;\n}" \
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add)                                                               \
                 : "memory");                                                                                                  \
  }
MAK_MMA_SS(mma_ss_f8, "f8f6f4")
MAK_MMA_SS(mma_ss_i8, "i8")
#undef MAK_MMA_SS
// The same in f16 with constants added to the descriptors: written so that the compiler does not keep
// every sum in a register of its own.
template <int A, int B>
__device__ __forceinline__ void mma_ss_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %4, 0;\n add.u64 x, %1, %5;\n add.u64 y, %2, %6;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(add), "n"(A), "n"(B)
      : "memory");
}
// D (TMEM, f32) = or += A (TMEM, f16) * B (shared memory, f16)
template <int A, int B>
__device__ __forceinline__ void mma_ts_f16(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b32 x;\n .reg .b64 y;\n setp.ne.b32 p, %4, 0;\n add.u32 x, %1, %5;\n add.u64 y, %2, %6;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add), "n"(A), "n"(B)
      : "memory");
}

#define MAK_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define MAK_W8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])
#define MAK_RW8(a, i) "+r"(a[i]), "+r"(a[i + 1]), "+r"(a[i + 2]), "+r"(a[i + 3]), "+r"(a[i + 4]), "+r"(a[i + 5]), "+r"(a[i + 6]), "+r"(a[i + 7])

__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&v)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at));
}
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : MAK_R8(v, 0) : "r"(at));
}
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : MAK_R8(v, 0), MAK_R8(v, 8)
               : "r"(at));
}
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : MAK_R8(v, 0), MAK_R8(v, 8), MAK_R8(v, 16), MAK_R8(v, 24)
      : "r"(at));
}
// Wait for this thread's loads from TMEM; the registers are named so that nothing uses them before.
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[4]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3])::"memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : MAK_RW8(v, 0)::"memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : MAK_RW8(v, 0), MAK_RW8(v, 8)::"memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : MAK_RW8(v, 0), MAK_RW8(v, 8), MAK_RW8(v, 16), MAK_RW8(v, 24)::"memory");
}
__device__ __forceinline__ void tmem_st(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::MAK_W8(v, 0),
      MAK_W8(v, 8), "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t at, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::MAK_W8(v, 0), "r"(at) : "memory");
}
#undef MAK_R8
#undef MAK_W8
#undef MAK_RW8

// Shared-memory matrix descriptor; strides in bytes.  Swizzle by the bytes of a line.
__device__ __forceinline__ uint64_t smem_desc(uint32_t at, uint32_t lbo, uint32_t sbo, int line_log2) {
  const uint64_t kind = line_log2 == 7 ? 2 : line_log2 == 6 ? 4 : line_log2 == 5 ? 6 : 0;
  return static_cast<uint64_t>((at >> 4) & 0x3fff) | (static_cast<uint64_t>((lbo >> 4) & 0x3fff) << 16) |
         (static_cast<uint64_t>((sbo >> 4) & 0x3fff) << 32) | (1ull << 46) | (kind << 61);
}
// Instruction descriptor, M = 128.  Formats of A and B: f16 0; E4M3 0; s8 1.  Accumulator: f32 1, s32 2.
constexpr uint32_t instr_desc(int n, int acc, int fmt, bool a_mn_major, bool b_mn_major) {
  return (static_cast<uint32_t>(acc) << 4) | (static_cast<uint32_t>(fmt) << 7) | (static_cast<uint32_t>(fmt) << 10) |
         (a_mn_major ? 1u << 15 : 0u) | (b_mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(128 >> 4) << 24);
}

// Contiguous copy from global to shared memory: both 16-byte aligned, a multiple of 16 bytes.
__device__ __forceinline__ void bulk_load(uint32_t to, const void* from, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from),
               "r"(bytes), "r"(smem_addr(bar))
               : "memory");
}
// Box of a 4-dimensional tensor map from coordinates (0, 0, y, z).
__device__ __forceinline__ void tensor_load(uint32_t to, const void* map, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %3, %4}], [%5];" ::"r"(to),
      "l"(map), "r"(0), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}

}  // namespace mak
