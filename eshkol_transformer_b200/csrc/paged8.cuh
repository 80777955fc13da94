// Pieces of the 8-bit paged cache that its append and attention kernels share.
#pragma once

#include "paged.cuh"

namespace etb {
namespace paged {

// A row's scale lies at page * page_stride + head * head_stride + slot * token_stride.
struct Scales {
  float* keys;
  float* values;
  int64_t page_stride, head_stride, token_stride;
};

// The element offset of a key's row in the pools and the offset of its scale; -1 for
// a page outside the pool.
struct Row8 {
  int64_t element, scale;
};
__device__ __forceinline__ Row8 row_of(const Pools& P, const Scales& S, const Batch& B, int b, int h,
                                       int key) {
  const int column = quotient(key, P.by_page), slot = key - column * P.page_size;
  const int64_t page = B.table[(int64_t)b * B.columns + column];
  if (page < 0 || page >= P.pages) return Row8{-1, -1};
  return Row8{page * P.page_stride + h * P.head_stride + slot * P.token_stride,
              page * S.page_stride + h * S.head_stride + slot * S.token_stride};
}

// A word of four e4m3 elements as binary16 pairs (exact).
__device__ __forceinline__ void halves_of(uint32_t four, uint32_t& low, uint32_t& high) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n"
      : "=r"(low), "=r"(high)
      : "r"(four));
}

struct Attend8Args {
  AttendArgs a;
  Scales scales;
};

int32_t check_cache8(const et_b200_paged_cache8_v1* c, et_kernel_error* e, const char* op);
Pools pools_of(const et_b200_paged_cache8_v1* c);
Scales scales_of(const et_b200_paged_cache8_v1* c);
// A map of a byte pool for boxes of `wide` (64 or 128, swizzled as wide as that) dims x
// box_rows slots, as pool_map's; false for pools it cannot describe.
bool pool8_map(CUtensorMap* map, void* pool, const et_b200_paged_cache8_v1* c, int wide,
               int box_rows);
// Whether the scales of neighbouring slots can be copied in whole 16-byte pieces.
bool scales_copy(const et_b200_paged_cache8_v1* c);
// The tcgen05 kernel (paged_attention8_tc.cu): its thread blocks, 0 where it does not
// take the cache (nothing is launched).  Its workspace is within attend_tc_workspace.
int attend8_tc(const et_b200_paged_cache8_v1* c, Attend8Args& a, void* ws, cudaStream_t stream);

// 2^e of a row of queries: the largest magnitude times it lies in [2^14, 2^15) (1 for
// rows of zeros and rows that are not finite).
__device__ __forceinline__ int query_exponent(float top) {
  const int b = (int)(__float_as_uint(top) >> 23);
  return b == 255 || top == 0.0f ? 0 : min(141 - b, 126);
}

// One untiled copy to shared memory: both addresses 16-byte aligned, whole 16-byte pieces.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

}  // namespace paged
}  // namespace etb
