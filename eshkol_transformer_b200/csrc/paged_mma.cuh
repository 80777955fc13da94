// Warp matrix pieces, copies, exponentials and stores that the kernels of the paged
// attention share, and what launches those on mma.sync.
#pragma once

#include <type_traits>

#include "attention_tc.cuh"
#include "paged.cuh"

namespace etb {
namespace paged {

// ---- warp matrix pieces -----------------------------------------------------------------

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                      uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo + r with hi, lo TF32 values, |r| <= 2^-22 |x|
__device__ __forceinline__ void pair_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(__uint_as_float(x)));
  const float rest = __uint_as_float(x) - __uint_as_float(hi);
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(rest));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool full) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(full ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two neighbouring outputs; one store where the address allows it.
template <typename T>
__device__ __forceinline__ void store2(T* dst, float a, float b) {
  if ((reinterpret_cast<uintptr_t>(dst) & (2 * sizeof(T) - 1)) == 0) {
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<float2*>(dst) = make_float2(a, b);
    else
      *reinterpret_cast<uint32_t*>(dst) = pack2<T>(a, b);
  } else {
    dst[0] = from_f32<T>(a);
    dst[1] = from_f32<T>(b);
  }
}

// ---- exponentials -----------------------------------------------------------------------

// 2^x of two finite values on the FMA pipe (x <= 15, under -126 as -126): x =
// n + f with n rounded to nearest, 2^f by its polynomial of degree 4 of least
// relative error on |f| <= 1/2 (2.7e-6), n added to the exponent.
__device__ __forceinline__ uint64_t power2(uint64_t x) {
  const float2 v = unpk(x);
  x = pk(fmaxf(v.x, -126.0f), fmaxf(v.y, -126.0f));
  const uint64_t m = add2(x, twice(12582912.0f));  // 1.5 2^23: n in the low bits
  const uint64_t f = fma2(add2(m, twice(-12582912.0f)), twice(-1.0f), x);
  uint64_t y = twice(9.5701013e-3f);
  y = fma2(y, f, twice(5.5917859e-2f));
  y = fma2(y, f, twice(2.4024744e-1f));
  y = fma2(y, f, twice(6.9312179e-1f));
  y = fma2(y, f, twice(9.9999928e-1f));
  const float2 mm = unpk(m), yy = unpk(y);
  return pk(__int_as_float(__float_as_int(yy.x) + (__float_as_int(mm.x) << 23)),
            __int_as_float(__float_as_int(yy.y) + (__float_as_int(mm.y) << 23)));
}

// ---- launching --------------------------------------------------------------------------

// Padded head_dim of the kernels: 32, 64, 128 or 256.
inline int padded(int64_t dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

constexpr int kMostPerSm = 4;  // resident thread blocks per SM that the workspace allows for

// Resident thread blocks of a kernel per SM (at most kMostPerSm), per device
// (the attribute that admits its shared memory is set on the way).
template <auto Kernel>
int resident_blocks(int threads, int smem) {
  static std::atomic<int> known[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64) {
    const int n = known[dev].load(std::memory_order_relaxed);
    if (n > 0) return n;
  }
  cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  int n = 0;
  cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kernel, threads, smem);
  n = n < 1 ? 1 : n > kMostPerSm ? kMostPerSm : n;
  if (dev >= 0 && dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

}  // namespace paged
}  // namespace etb
