// Appending keys and values to an 8-bit paged cache (et_b200_paged_append8_v1).
//
// A row x (one head of one token, of the keys k' = R(pos) k in f32) becomes e4m3
// elements x / s and its scale s = 2^e, the least power of two with max|x| <= 448 s:
// x / s is exact, so an element is rounded once, and the attention's products with s
// are exact too.  Every byte is read once; a lane takes 8 dims, a group of lanes as
// many as a row has (a power of two up to 32) a row of K and the row of V beside it,
// whose maxima they exchange by shuffles.  The rows are requested before the chain
// offsets, length, page, tables is followed, as in the append of wider types (paged_kv.cu).
// 11 ragged prompts (15,600 tokens, 8 heads x 128, bf16 or f16, 98 MB): 28.2 us on the device where
// the inputs come from memory, 3.5 TB/s (24.7 us where the L2 holds a part of them from the call
// before); f32 (162 MB) 40.5 us, 4.0 TB/s.  Issue slots are 65 % busy (rotation, maxima, conversion)
// while a warp waits 2 of its 7 cycles an instruction for its loads.  A warp a token of 4 rows a
// lane; with the L2's help, four tokens a warp 30.6 us, two rows or one a lane 28 to 34.  One token:
// 7.4 us a call (the host), 3.9 us on the device.
#include <type_traits>

#include "attention_tc.cuh"
#include "paged8.cuh"

namespace etb {
namespace {

using namespace paged;

constexpr int WARPS = 4;

// 8 elements from src as f32; VEC: it can be read in 16-byte pieces.
template <typename T, bool VEC>
struct Eight {
  static constexpr int PIECES = sizeof(T) / 2;
  union {
    uint4 v[PIECES];
    T x[8];
  };
  __device__ __forceinline__ void load(const T* src) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < PIECES; i++) v[i] = __ldcs(reinterpret_cast<const uint4*>(src) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = src[i];
    }
  }
};

// The larger magnitude; NaN if either is.
__device__ __forceinline__ float larger(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}
// The scale of a row whose largest magnitude is `top` (448 = 1.75 2^8), and its inverse: a
// power of two between 2^-126 and 2^120, so exact, and in range; 0 for rows of zeros and
// rows that are not finite.
__device__ __forceinline__ float scale_of_row(float top, float& inverse) {
  const uint32_t u = __float_as_uint(top);
  const int e = max((int)((u + 0x1fffffu) >> 23) - 8, 1);  // biased; + 1 above 1.75
  const bool some = top > 0.0f && u < 0x7f800000u;
  inverse = some ? __uint_as_float((uint32_t)(254 - e) << 23) : 0.0f;
  return some ? __uint_as_float((uint32_t)e << 23) : top == 0.0f ? 0.0f : NAN;
}
__device__ __forceinline__ uint32_t two_e4m3(float low, float high) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(high), "f"(low));
  return r;
}
// The stored elements of 8 values: x / s; zeros under the scale NaN.
__device__ __forceinline__ uint2 quantised(const float (&x)[8], float s, float inv) {
  if (s != s) return make_uint2(0, 0);
  return make_uint2(two_e4m3(x[0] * inv, x[1] * inv) | two_e4m3(x[2] * inv, x[3] * inv) << 16,
                    two_e4m3(x[4] * inv, x[5] * inv) | two_e4m3(x[6] * inv, x[7] * inv) << 16);
}

// A warp takes a token and `ROWS` times 32 / lanes of its heads; lanes = 2^lane_bits
// to a row.
constexpr int ROWS = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * WARPS)
paged_append8_kernel(Pools P, Scales S, Batch B, Rope R, uint8_t* __restrict__ keys,
                     uint8_t* __restrict__ values, const T* __restrict__ k, int64_t k_stride,
                     const T* __restrict__ v, int64_t v_stride, int lane_bits) {
  const int lane = threadIdx.x & 31;
  const int64_t token = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (token >= B.tokens) {
    // a block behind the last token (there is one where there is a status word)
    // looks at the metadata of every request, also of those that store nothing
    if ((int64_t)blockIdx.x * WARPS >= B.tokens && blockIdx.y == 0)
      for (int b = threadIdx.x; b < B.batch; b += 32 * WARPS)
        if (const int bad = load_request(B, b).bad) report(B.status, bad);
    return;
  }
  const int lanes = 1 << lane_bits, at_once = 32 >> lane_bits;
  const int h0 = blockIdx.y * ROWS * at_once + (lane >> lane_bits), d = 8 * (lane & (lanes - 1));
  Eight<T, VEC> kx[ROWS], vx[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    const int h = h0 + i * at_once;
    if (h < P.kv_heads && d < P.head_dim) {
      kx[i].load(k + token * k_stride + (int64_t)h * P.head_dim + d);
      vx[i].load(v + token * v_stride + (int64_t)h * P.head_dim + d);
    }
  }
  // the request whose rows hold this token: the last b with offsets[b] <= token
  const int b = warp_count(B.offsets, B.batch + 1, token, true) - 1;
  if (b < 0 || b >= B.batch) return;  // a row of no request
  const Request r = load_request(B, b);
  if (r.bad != 0 && lane == 0) report(B.status, r.bad);
  if (token < r.first || token >= r.first + r.n) return;
  const int64_t pos = (int64_t)r.len - r.n + (token - r.first);
  if (pos < 0) return;
  const Row8 at = row_of(P, S, B, b, 0, (int)pos);
  if (at.element < 0) {
    if (lane == 0) report(B.status, ET_B200_PAGED_BAD_PAGE);
    return;
  }
  float cs[4] = {1.0f, 1.0f, 1.0f, 1.0f}, sn[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (R.cos != nullptr && d < P.head_dim) {
    const int64_t row = rope_row(R, pos, B.status) * (P.head_dim / 2) + d / 2;
    if (((reinterpret_cast<uintptr_t>(R.cos) | reinterpret_cast<uintptr_t>(R.sin)) & 15) == 0) {
      const float4 c = __ldg(reinterpret_cast<const float4*>(R.cos + row));
      const float4 s = __ldg(reinterpret_cast<const float4*>(R.sin + row));
      cs[0] = c.x, cs[1] = c.y, cs[2] = c.z, cs[3] = c.w;
      sn[0] = s.x, sn[1] = s.y, sn[2] = s.z, sn[3] = s.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        cs[j] = __ldg(R.cos + row + j);
        sn[j] = __ldg(R.sin + row + j);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; i++) {
    const int h = h0 + i * at_once;
    const bool some = h < P.kv_heads && d < P.head_dim;
    float x[8], y[8], top[2] = {0.0f, 0.0f};
    if (h0 - (lane >> lane_bits) + i * at_once >= P.kv_heads) break;  // for the whole warp
    if (some) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        x[j] = to_f32<T>(kx[i].x[j]);
        y[j] = to_f32<T>(vx[i].x[j]);
      }
      if (R.cos != nullptr) {
#pragma unroll
        for (int j = 0; j < 4; j++) rotate(x[2 * j], x[2 * j + 1], cs[j], sn[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        top[0] = larger(top[0], x[j]);
        top[1] = larger(top[1], y[j]);
      }
    }
    for (int o = 1; o < lanes; o <<= 1) {
#pragma unroll
      for (int j = 0; j < 2; j++) top[j] = larger(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
    }
    if (some) {
      float ki, vi;
      const float ks = scale_of_row(top[0], ki), vs = scale_of_row(top[1], vi);
      const int64_t e = at.element + h * P.head_stride + d;
      *reinterpret_cast<uint2*>(keys + e) = quantised(x, ks, ki);
      *reinterpret_cast<uint2*>(values + e) = quantised(y, vs, vi);
      if (d == 0) {
        S.keys[at.scale + h * S.head_stride] = ks;
        S.values[at.scale + h * S.head_stride] = vs;
      }
    }
  }
}

template <typename T>
void launch_append8(const et_b200_paged_cache8_v1* c, const Batch& B, const Rope& R, const void* k,
                    int64_t ks, const void* v, int64_t vs, cudaStream_t stream) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                         (uintptr_t)(ks * (int64_t)sizeof(T)) | (uintptr_t)(vs * (int64_t)sizeof(T));
  int lane_bits = 0;
  while ((8 << lane_bits) < c->head_dim) lane_bits++;
  const int heads = ROWS * (32 >> lane_bits);
  const unsigned check = B.status != nullptr ? 1 : 0;  // a block behind the last token
  const dim3 grid((unsigned)((B.tokens + WARPS - 1) / WARPS) + check,
                  (unsigned)((c->kv_heads + heads - 1) / heads));
  auto go = [&](auto vec) {
    paged_append8_kernel<T, decltype(vec)::value><<<grid, 32 * WARPS, 0, stream>>>(
        pools_of(c), scales_of(c), B, R, static_cast<uint8_t*>(c->keys),
        static_cast<uint8_t*>(c->values), static_cast<const T*>(k), ks, static_cast<const T*>(v), vs,
        lane_bits);
  };
  if ((bits & 15) == 0) go(std::true_type{}); else go(std::false_type{});
  count_launch();
}

}  // namespace

namespace paged {

int32_t check_cache8(const et_b200_paged_cache8_v1* c, et_kernel_error* e, const char* op) {
  if (c == nullptr || c->struct_size < sizeof(et_b200_paged_cache8_v1))
    return set_error(e, ET_KERNEL_ERROR_VERSION_MISMATCH, ET_KERNEL_CODE_INVALID_STRUCT_SIZE, op,
                     "8-bit paged cache descriptor is missing or truncated");
  if (c->dtype > ET_B200_DTYPE_BF16)
    return set_error(e, ET_KERNEL_ERROR_DTYPE_MISMATCH, ET_KERNEL_CODE_INVALID_ENUM, op,
                     "unknown element type of the tensors beside the 8-bit paged cache");
  if (c->pages < 1 || c->pages > INT32_MAX || c->page_size < 1 || c->page_size > (1 << 20) ||
      c->kv_heads < 1 || c->kv_heads > 4096 || c->head_dim < 16 || c->head_dim > 256 ||
      c->head_dim % 16 != 0)
    return set_error(e, ET_KERNEL_ERROR_SHAPE_MISMATCH, ET_KERNEL_CODE_INVALID_SHAPE, op,
                     "8-bit paged cache shape is outside its limits (head_dim: a multiple of 16 up "
                     "to 256)");
  if (!strides_nest(c->page_size, c->kv_heads, c->head_dim, c->pages, c->page_stride, c->head_stride,
                    c->token_stride) ||
      !strides_nest(c->page_size, c->kv_heads, 1, c->pages, c->scale_page_stride,
                    c->scale_head_stride, c->scale_token_stride))
    return set_error(e, ET_KERNEL_ERROR_NONCONTIGUOUS, ET_KERNEL_CODE_INVALID_BUFFER, op,
                     "8-bit paged cache strides overlap or are out of range");
  if (c->keys == nullptr || c->values == nullptr || c->key_scales == nullptr ||
      c->value_scales == nullptr)
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_NULL_ARGUMENT, op,
                     "both pools of the 8-bit paged cache and their scales are required");
  if (!aligned_to(16, c->keys, c->values) || !aligned_to(4, c->key_scales, c->value_scales) ||
      (c->page_stride | c->head_stride | c->token_stride) % 16 != 0)
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_INVALID_BUFFER, op,
                     "8-bit pools must be 16-byte aligned with strides of whole 16-byte pieces, "
                     "scales aligned to their elements");
  return 0;
}

bool pool8_map(CUtensorMap* map, void* pool, const et_b200_paged_cache8_v1* c, int wide,
               int box_rows) {
  const int64_t rows = c->page_size;
  if (rows < 8 || (rows & (rows - 1)) != 0 || encode_fn() == nullptr ||
      c->page_stride >= (int64_t)1 << 40 || c->head_stride >= (int64_t)1 << 40)
    return false;
  const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->page_size,
                              (cuuint64_t)c->kv_heads, (cuuint64_t)c->pages};
  const cuuint64_t strides[3] = {(cuuint64_t)c->token_stride, (cuuint64_t)c->head_stride,
                                 (cuuint64_t)c->page_stride};
  const cuuint32_t box[4] = {(cuuint32_t)wide, (cuuint32_t)box_rows, 1, 1}, one[4] = {1, 1, 1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, pool, dims, strides, box, one,
                     CU_TENSOR_MAP_INTERLEAVE_NONE,
                     wide == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool scales_copy(const et_b200_paged_cache8_v1* c) {
  return aligned_to(16, c->key_scales, c->value_scales) && c->scale_token_stride == 1 &&
         (c->scale_page_stride | c->scale_head_stride) % 4 == 0;
}

Pools pools_of(const et_b200_paged_cache8_v1* c) {
  return Pools{c->pages, c->page_stride, c->head_stride, c->token_stride, (int)c->page_size,
               (int)c->kv_heads, (int)c->head_dim, divisor_of((uint32_t)c->page_size)};
}
Scales scales_of(const et_b200_paged_cache8_v1* c) {
  return Scales{c->key_scales, c->value_scales, c->scale_page_stride, c->scale_head_stride,
                c->scale_token_stride};
}

}  // namespace paged
}  // namespace etb

using namespace etb;
using namespace etb::paged;

extern "C" int32_t et_b200_paged_append8_v1(const et_b200_paged_cache8_v1* c,
                                            const et_b200_paged_batch_v1* b,
                                            const et_b200_paged_rope_v1* rope, const void* k,
                                            int64_t k_stride, const void* v, int64_t v_stride,
                                            void* stream, et_kernel_error* e) {
  const char* op = "paged-append8";
  if (int32_t r = check_cache8(c, e, op)) return r;
  if (int32_t r = check_batch(b, c->page_size, e, op)) return r;
  if (int32_t r = check_rope(rope, e, op)) return r;
  if (b->tokens > 0 && b->batch > 0) {
    const int64_t size = c->dtype == ET_B200_DTYPE_F32 ? 4 : 2;
    if (int32_t r = check_new_rows(k, k_stride, v, v_stride, c->kv_heads * c->head_dim, size, e, op))
      return r;
    const Batch B = batch_of(b, c->page_size);
    const Rope R = rope_of(rope);
    auto st = static_cast<cudaStream_t>(stream);
    if (c->dtype == ET_B200_DTYPE_F32) launch_append8<float>(c, B, R, k, k_stride, v, v_stride, st);
    else if (c->dtype == ET_B200_DTYPE_F16) launch_append8<__half>(c, B, R, k, k_stride, v, v_stride, st);
    else launch_append8<__nv_bfloat16>(c, B, R, k, k_stride, v, v_stride, st);
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return cuda_error(e, status, op);
  }
  if (e) memset(e, 0, sizeof(*e));
  return 0;
}
