// tcgen05.cuh -- what the tcgen05 kernels share: fences, tensor-memory loads
// and stores, the single-CTA matrix instructions, their descriptors, and the
// tensor maps of their TMA loads.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "kyro_internal.cuh"
#include "ptx.cuh"

namespace kyro {
namespace tc {

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
      "%29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st1(uint32_t taddr, uint32_t r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(r) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(taddr));
}
// one column, waited for
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  tmem_ld_wait();
  return r;
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Shared-memory matrix descriptors (tcgen05 format: version 1, 128-byte
// swizzle).  K-major (rows of 64 contiguous bf16 along K): the stride between
// 8-row groups is 1024 B and the leading offset is unused (16 B).  MN-major
// (64 contiguous bf16 along N): the leading offset steps between 64-column
// slabs along N, the stride between 8-row groups along K.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)((lbo >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFF) << 32;
  d |= (uint64_t)1 << 46;  // descriptor version (sm_100)
  d |= (uint64_t)2 << 61;  // SWIZZLE_128B
  return d;
}

// The two words of such a descriptor: the high one depends on the layout
// alone, the low one holds the address (in 16 bytes), so the next operand of
// a row of products is one 32-bit addition away.  A matrix instruction takes
// 64 cycles at M = N = 128; building both descriptors anew for each takes its
// one issuing thread about 110.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) {
  return (saddr >> 4) | ((lbo >> 4) << 16);
}

// Instruction descriptor of kind::f16: bf16 A and B, fp32 accumulate, of m x
// n; b_mn selects an MN-major B.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool b_mn) {
  return (1u << 4)              // D fp32
         | (1u << 7)            // A bf16
         | (1u << 10)           // B bf16
         | ((b_mn ? 1u : 0u) << 16)
         | ((uint32_t)(n >> 3) << 17)
         | ((uint32_t)(m >> 4) << 24);
}

// ---------------------------------------------------------------- one CTA
__device__ __forceinline__ void tmem_alloc1(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem),
               "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish1() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc1(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
               : "memory");
}
// D (+)= A[smem] * B[smem], 16 deep (descriptors by their low words)
__device__ __forceinline__ void umma1_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                         uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}
// D (+)= A[tmem] * B[smem], 16 deep
__device__ __forceinline__ void umma1_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                         uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}
// Arrive on `bar` when every MMA issued so far is done.
__device__ __forceinline__ void umma1_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
               : "memory");
}
// Shared memory written by this thread becomes visible to TMA and the MMAs.
__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Every wait ends: after kWaitBudget cycles it sets *err, flags
// KYRO_DEV_WAIT_TIMEOUT and returns false.  The wait sleeps in the barrier
// (up to kWaitNap ns at a time): a warp that polls takes issue slots from the
// warps that compute on its scheduler (600 of 2200 cycles of a step, where a
// matrix warp polled beside two warps of kv_scores_kernel).  Without Nap it
// polls: tree_attention_tc_kernel takes 618.4 us that way at 32 sequences of 8192
// slots and 64 nodes, and 621.0 asleep.
constexpr long long kWaitBudget = 2000000000ll;
constexpr uint32_t kWaitNap = 1000000;
__device__ __forceinline__ bool nap_bar(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity), "r"(kWaitNap)
      : "memory");
  return done != 0;
}
template <bool Nap = true>
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, int* err,
                                         uint32_t* status) {
  if constexpr (Nap) {
    if (nap_bar(bar, parity)) return true;
    const long long t0 = clock64();
    do {
      if (nap_bar(bar, parity)) return true;
    } while (clock64() - t0 <= kWaitBudget);
  } else {
    if (kyro::ptx::mbar_wait_bounded(bar, parity, kWaitBudget)) return true;
  }
  *(volatile int*)err = 1;
  kyro::dev::flag(status, KYRO_DEV_WAIT_TIMEOUT);
  return false;
}

// The same for a whole warp: every lane gets the same answer, so that no lane
// leaves the others behind at a warp-wide instruction.
__device__ __forceinline__ bool wait_bar_warp(uint32_t bar, uint32_t parity, int* err,
                                              uint32_t* status) {
  return __all_sync(0xffffffffu, wait_bar(bar, parity, err, status));
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Maximum of a row's 128 scores (raw units): four max3 chains.
__device__ __forceinline__ float row_max128(const uint32_t (&r)[128]) {
  float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
  for (int i = 0; i < 128; i += 8) {
    m0 = fmax3(m0, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
    m1 = fmax3(m1, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
    m2 = fmax3(m2, __uint_as_float(r[i + 4]), __uint_as_float(r[i + 5]));
    m3 = fmax3(m3, __uint_as_float(r[i + 6]), __uint_as_float(r[i + 7]));
  }
  return fmax3(fmax3(m0, m1, m2), m3, -INFINITY);
}

// ---------------------------------------------------------------- tensor maps
inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// 3-D bf16 map with 128-byte swizzle: dims (innermost first), strides of the
// outer two dims in bytes, box (64, box1, box2).
inline int make_map3(CUtensorMap* map, const void* ptr, uint64_t d0, uint64_t d1, uint64_t d2,
              uint64_t s1, uint64_t s2, uint32_t box1, uint32_t box2) {
  auto enc = encode_fn();
  if (!enc) return kyro::set_error(KYRO_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {d0, d1, d2};
  cuuint64_t strides[2] = {s1, s2};
  cuuint32_t box[3] = {64, box1, box2};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims,
                         strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return kyro::set_error(KYRO_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return KYRO_OK;
}


// The pages of one K or V cache, [rows = blocks * Hkv][16 tokens][D] bf16, as
// (64 dims, 16 tokens, D / 64 slabs, rows): one box is a page, its slabs one
// after the other in shared memory.
inline int make_page_map(CUtensorMap* map, const void* ptr, int d, uint64_t rows) {
  auto enc = encode_fn();
  if (!enc) return kyro::set_error(KYRO_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[4] = {64, 16, (cuuint64_t)(d / 64), rows};
  cuuint64_t strides[3] = {(cuuint64_t)d * 2, 128, (cuuint64_t)d * 32};
  cuuint32_t box[4] = {64, 16, (cuuint32_t)(d / 64), 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims,
                         strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return kyro::set_error(KYRO_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return KYRO_OK;
}

}  // namespace tc
}  // namespace kyro
