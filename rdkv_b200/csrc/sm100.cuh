// mbarriers, tiled TMA copies, tensor memory and the fifth-generation tensor cores: the instructions the paged
// attention kernels use, one function each.
#pragma once

#include <cuda.h>   // CUtensorMap and its enums (the encoder itself is looked up through the runtime)

#include "rdkv_common.cuh"

namespace rdkv {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ float exp2_approx(float x) {          // 2^x, one instruction (relative error 2^-22; 2^-inf = 0)
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void store_global(uint64_t addr, const uint4& v) {
  asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

__device__ __forceinline__ uint32_t now_ns() {                  // (wraps after 4.3 s)
  uint32_t t;
  asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
  return t;
}

// ── mbarrier ────────────────────────────────────────────────────────────────
__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_arrive_tx(uint32_t bar, uint32_t bytes) {   // arrive and expect `bytes` of copies
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits for the barrier's phase `parity`, for `limit` nanoseconds (under 2^32) once a first try has failed; false if it did not complete.
// A limit of time, not of tries: a try that fails takes 1 us (it sleeps on the barrier), but nothing promises that.  Waits end within
// microseconds to a few milliseconds; WAIT_NS is far above both.  (No limit at all left: a wait that is not over with the first try has run out.)
constexpr uint32_t WAIT_NS = 2000000000u;
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, uint32_t limit) {
  if (bar_try(bar, parity)) return true;
  for (const uint32_t start = now_ns(); now_ns() - start < limit;)
    if (bar_try(bar, parity)) return true;
  return false;
}
// The same for a whole warp: all its lanes go on, or none does.
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, uint32_t parity, uint32_t limit) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity, limit));
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ── dependent launches ──────────────────────────────────────────────────────
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ── TMA ─────────────────────────────────────────────────────────────────────
// One box of a 4-D tensor map into shared memory; its bytes are counted on the mbarrier.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* tm, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* tm, int c0, int c1, int c2, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
               : "memory");
}

// ── tensor memory and tcgen05 ───────────────────────────────────────────────
// Shared-memory matrix descriptors of operands laid down with the 128-byte swizzle.  Bits [0,14) start address / 16,
// [16,30) leading-dimension offset / 16, [32,46) stride-dimension offset / 16, [46,48) version 1, [61,64) 2 = 128-byte swizzle.
// K-major (rows of 64 16-bit elements along K, 8 rows 1024 bytes apart): the leading offset is not used.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// MN-major (a row of 64 16-bit elements along N for every step of K, 8 steps 1024 bytes apart): `panel` bytes to the next 64 of N.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr, uint32_t panel) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)(panel >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Instruction descriptor of a dense 16-bit MMA of 128 x n with fp32 accumulation: bits [4,6) accumulator 1 = fp32, [7,10) and
// [10,13) operand types (0 = fp16, 1 = bf16), 16: B is MN-major, [17,23) N / 8, [24,29) M / 16.
template <bool BF16>
__device__ __forceinline__ constexpr uint32_t mma_idesc(int n, bool b_mn_major) {
  return 1u << 4 | (BF16 ? 1u : 0u) << 7 | (BF16 ? 1u : 0u) << 10 | (b_mn_major ? 1u : 0u) << 16 | (uint32_t)(n >> 3) << 17 |
         (uint32_t)(128 >> 4) << 24;
}
// The whole warp comes here with the same values, one elected lane issues: control flow and operands stay uniform, which
// is what the instruction wants (issued from inside a one-lane branch, each cost about 150 cycles instead of under 64).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void mma_ss(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {   // A in shared memory
  asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t elected, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {   // A in tensor memory
  asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t elected, uint32_t bar) {   // the barrier gets an arrival once the MMAs issued so far are done
  asm volatile("{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n"
               ::"r"(bar), "r"(elected) : "memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define RDKV_R8(v, i) "=r"((v)[i]), "=r"((v)[i + 1]), "=r"((v)[i + 2]), "=r"((v)[i + 3]), "=r"((v)[i + 4]), "=r"((v)[i + 5]), "=r"((v)[i + 6]), "=r"((v)[i + 7])
#define RDKV_S8(v, i) "r"((v)[i]), "r"((v)[i + 1]), "r"((v)[i + 2]), "r"((v)[i + 3]), "r"((v)[i + 4]), "r"((v)[i + 5]), "r"((v)[i + 6]), "r"((v)[i + 7])
// 32 consecutive 32-bit columns of this thread's row (lane i of warp w: row 32*(w&3)+i).  The wait is part of the statement, so
// that no use of the registers can move ahead of it.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : RDKV_R8(v, 0), RDKV_R8(v, 8), RDKV_R8(v, 16), RDKV_R8(v, 24)
      : "r"(taddr)
      : "memory");
}
// 64 columns.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, "
      "%46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : RDKV_R8(v, 0), RDKV_R8(v, 8), RDKV_R8(v, 16), RDKV_R8(v, 24), RDKV_R8(v, 32), RDKV_R8(v, 40), RDKV_R8(v, 48), RDKV_R8(v, 56)
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
      "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n"
      ::"r"(taddr), RDKV_S8(v, 0), RDKV_S8(v, 8), RDKV_S8(v, 16), RDKV_S8(v, 24)
      : "memory");
}
#undef RDKV_R8
#undef RDKV_S8

__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* tm) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tm)) : "memory");
}

// The driver's tensor-map encoder, found through the runtime (the library does not link the driver).
using TensorMapEncoder = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                      const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                      CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline TensorMapEncoder tensor_map_encoder() {
  static const TensorMapEncoder fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &res) != cudaSuccess || res != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      return (TensorMapEncoder) nullptr;
    }
    return reinterpret_cast<TensorMapEncoder>(p);
  }();
  return fn;
}

}  // namespace rdkv
