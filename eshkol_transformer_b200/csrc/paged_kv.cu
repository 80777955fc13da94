// Appending keys and values to a paged cache (et_b200_paged_append_v1).
//
// k'(pos) = R(pos) k with R the pairwise rotation (x0 c - x1 s, x0 s + x1 c),
// written with v to slot pos % page_size of the request's page.  Pure data
// movement: every byte is read once and written once.  The latency of its loads
// bounds it: of the data in large steps (four 16-byte pieces of K and V in flight a
// lane), of the chain offsets, length, page, tables in small ones.  One warp takes
// one token and 32 VPL 16-byte pieces of its keys and values; the pieces are
// requested before the chain is followed, so the two latencies overlap, and the
// request is found by a 32-ary search of the whole warp (two load rounds up to 1,024
// requests).  Measured: 27.5 us for 32 MB of keys and values from 11 prompts (4.7
// TB/s read and written, the writes to L2), 2.8 us for one token; fewer pieces per
// lane with more resident warps took 28 to 30 us.
#include <type_traits>

#include "attention_tc.cuh"
#include "paged.cuh"

namespace etb {
namespace {

using namespace paged;

constexpr int VPL = 4;  // 16-byte pieces of K and of V per lane
constexpr int WARPS = 4;

template <typename T, bool VEC>
__device__ __forceinline__ uint4 load_piece(const T* src) {
  if constexpr (VEC) {
    return __ldcs(reinterpret_cast<const uint4*>(src));
  } else {
    constexpr int N = 16 / sizeof(T);
    union { uint4 v; T x[N]; } u;
#pragma unroll
    for (int i = 0; i < N; i++) u.x[i] = src[i];
    return u.v;
  }
}

// VEC: rows of k and v can be read as 16-byte pieces.
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * WARPS)
paged_append_kernel(Pools P, Batch B, Rope R, T* __restrict__ keys, T* __restrict__ values,
                    const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v,
                    int64_t v_stride) {
  constexpr int N = 16 / sizeof(T);
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
  const int row_pieces = P.kv_heads * P.head_dim / N;
  const int piece0 = blockIdx.y * 32 * VPL + lane;
  uint4 kp[VPL], vp[VPL];
#pragma unroll
  for (int i = 0; i < VPL; i++) {
    const int p = piece0 + 32 * i;
    if (p < row_pieces) {
      kp[i] = load_piece<T, VEC>(k + token * k_stride + (int64_t)p * N);
      vp[i] = load_piece<T, VEC>(v + token * v_stride + (int64_t)p * N);
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
  const int64_t base = key_offset(P, B, b, 0, (int)pos);
  if (base < 0) {
    if (lane == 0) report(B.status, ET_B200_PAGED_BAD_PAGE);
    return;
  }
  const int half = P.head_dim / 2;
  const float* ct = nullptr;
  const float* st = nullptr;
  if (R.cos != nullptr) {
    const int64_t row = rope_row(R, pos, B.status) * half;
    ct = R.cos + row;
    st = R.sin + row;
  }
#pragma unroll
  for (int i = 0; i < VPL; i++) {
    const int p = piece0 + 32 * i;
    if (p >= row_pieces) break;
    const int e = p * N, h = e / P.head_dim, d = e - h * P.head_dim;
    const int64_t at = base + h * P.head_stride + d;
    if (ct != nullptr) {
      union { uint4 v; T x[N]; } u;
      u.v = kp[i];
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        float x0 = to_f32<T>(u.x[j]), x1 = to_f32<T>(u.x[j + 1]);
        rotate(x0, x1, __ldg(ct + (d + j) / 2), __ldg(st + (d + j) / 2));
        u.x[j] = from_f32<T>(x0);
        u.x[j + 1] = from_f32<T>(x1);
      }
      kp[i] = u.v;
    }
    *reinterpret_cast<uint4*>(keys + at) = kp[i];
    *reinterpret_cast<uint4*>(values + at) = vp[i];
  }
}

template <typename T>
void launch_append(const et_b200_paged_cache_v1* c, const Pools& P, const Batch& B, const Rope& R,
                   const void* k, int64_t ks, const void* v, int64_t vs, cudaStream_t stream) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                         (uintptr_t)(ks * (int64_t)sizeof(T)) | (uintptr_t)(vs * (int64_t)sizeof(T));
  const int pieces = P.kv_heads * P.head_dim / (int)(16 / sizeof(T));
  const unsigned check = B.status != nullptr ? 1 : 0;  // a block behind the last token
  const dim3 grid((unsigned)((B.tokens + WARPS - 1) / WARPS) + check, (unsigned)((pieces + 32 * VPL - 1) / (32 * VPL)));
  auto go = [&](auto vec) {
    paged_append_kernel<T, decltype(vec)::value><<<grid, 32 * WARPS, 0, stream>>>(
        P, B, R, static_cast<T*>(c->keys), static_cast<T*>(c->values), static_cast<const T*>(k), ks,
        static_cast<const T*>(v), vs);
  };
  if ((bits & 15) == 0) go(std::true_type{}); else go(std::false_type{});
  count_launch();
}

}  // namespace

namespace paged {

// Whether no stride lets two rows of a pool share a place: the smallest nesting is
// token < head < page or head < token < page.  Far strides are refused too.
bool strides_nest(int64_t page_size, int64_t kv_heads, int64_t row, int64_t pages, int64_t ps,
                  int64_t hs, int64_t ts) {
  if (ts < 1 || hs < 1 || ps < 1 || ts > (int64_t)1 << 31 || hs > (int64_t)1 << 36 ||
      ps > INT64_MAX / 8 / pages)
    return false;
  return (ts >= row && hs >= (page_size - 1) * ts + row &&
          ps >= (kv_heads - 1) * hs + (page_size - 1) * ts + row) ||
         (hs >= row && ts >= (kv_heads - 1) * hs + row &&
          ps >= (page_size - 1) * ts + (kv_heads - 1) * hs + row);
}

int32_t check_cache(const et_b200_paged_cache_v1* c, et_kernel_error* e, const char* op) {
  if (c == nullptr || c->struct_size < sizeof(et_b200_paged_cache_v1))
    return set_error(e, ET_KERNEL_ERROR_VERSION_MISMATCH, ET_KERNEL_CODE_INVALID_STRUCT_SIZE, op,
                     "paged cache descriptor is missing or truncated");
  if (c->dtype > ET_B200_DTYPE_BF16)
    return set_error(e, ET_KERNEL_ERROR_DTYPE_MISMATCH, ET_KERNEL_CODE_INVALID_ENUM, op,
                     "unknown element type of the paged cache");
  if (c->pages < 1 || c->pages > INT32_MAX || c->page_size < 1 || c->page_size > (1 << 20) ||
      c->kv_heads < 1 || c->kv_heads > 4096 || c->head_dim < 8 || c->head_dim > 256 ||
      c->head_dim % 8 != 0)
    return set_error(e, ET_KERNEL_ERROR_SHAPE_MISMATCH, ET_KERNEL_CODE_INVALID_SHAPE, op,
                     "paged cache shape is outside its limits (head_dim: a multiple of 8 up to "
                     "256)");
  const int64_t size = c->dtype == ET_B200_DTYPE_F32 ? 4 : 2;
  const int64_t hs = c->head_stride, ts = c->token_stride, ps = c->page_stride;
  if (!strides_nest(c->page_size, c->kv_heads, c->head_dim, c->pages, ps, hs, ts))
    return set_error(e, ET_KERNEL_ERROR_NONCONTIGUOUS, ET_KERNEL_CODE_INVALID_BUFFER, op,
                     "paged cache strides overlap or are out of range");
  if (c->keys == nullptr || c->values == nullptr)
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_NULL_ARGUMENT, op,
                     "both pools of the paged cache are required");
  if (((reinterpret_cast<uintptr_t>(c->keys) | reinterpret_cast<uintptr_t>(c->values)) & 15) != 0 ||
      ((ts * size) | (hs * size) | (ps * size)) % 16 != 0)
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_INVALID_BUFFER, op,
                     "pools must be 16-byte aligned with strides of whole 16-byte pieces");
  return 0;
}

int32_t check_batch(const et_b200_paged_batch_v1* b, int64_t page_size, et_kernel_error* e,
                    const char* op) {
  if (b == nullptr || b->struct_size < sizeof(et_b200_paged_batch_v1))
    return set_error(e, ET_KERNEL_ERROR_VERSION_MISMATCH, ET_KERNEL_CODE_INVALID_STRUCT_SIZE, op,
                     "paged batch descriptor is missing or truncated");
  if (b->batch < 0 || b->batch > (1 << 20) || b->tokens < 0 || b->tokens > (1 << 26) ||
      b->table_columns < 1 || b->table_columns > kMostCapacity / page_size || b->max_new < 0 ||
      b->max_length < 0)
    return set_error(e, ET_KERNEL_ERROR_SHAPE_MISMATCH, ET_KERNEL_CODE_INVALID_SHAPE, op,
                     "paged batch is outside its limits (a page table holds fewer than 2^31 - "
                     "4096 keys)");
  if (b->batch > 0 && (b->offsets == nullptr || b->lengths == nullptr || b->page_table == nullptr))
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_NULL_ARGUMENT, op,
                     "offsets, lengths and the page table are required");
  if (!aligned_to(8, b->offsets, b->lengths) || !aligned_to(4, b->page_table, b->status))
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_INVALID_BUFFER, op,
                     "offsets, lengths, the page table and the status word must be aligned to "
                     "their elements");
  return 0;
}

int32_t check_new_rows(const void* k, int64_t k_stride, const void* v, int64_t v_stride, int64_t row,
                       int64_t size, et_kernel_error* e, const char* op) {
  if (k == nullptr || v == nullptr)
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_NULL_ARGUMENT, op,
                     "k and v are required");
  if (k_stride < row || v_stride < row || k_stride > (int64_t)1 << 31 ||
      v_stride > (int64_t)1 << 31)
    return set_error(e, ET_KERNEL_ERROR_NONCONTIGUOUS, ET_KERNEL_CODE_INVALID_BUFFER, op,
                     "rows of k and v overlap or lie too far apart");
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % size != 0)
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_INVALID_BUFFER, op,
                     "k and v must be aligned to their elements");
  return 0;
}

int32_t check_rope(const et_b200_paged_rope_v1* r, et_kernel_error* e, const char* op) {
  if (r == nullptr || (r->cos == nullptr && r->sin == nullptr)) return 0;
  if (r->cos == nullptr || r->sin == nullptr)
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_NULL_ARGUMENT, op,
                     "RoPE needs both the cosine and the sine table");
  if (r->rows < 1)
    return set_error(e, ET_KERNEL_ERROR_SHAPE_MISMATCH, ET_KERNEL_CODE_INVALID_SHAPE, op,
                     "RoPE tables have no rows");
  if (!aligned_to(4, r->cos, r->sin))
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_INVALID_BUFFER, op,
                     "RoPE tables must be aligned to their elements");
  return 0;
}

bool pool_map(CUtensorMap* map, void* pool, const et_b200_paged_cache_v1* c, int wide, int box_rows,
              bool swizzled) {
  const int64_t rows = c->page_size, size = c->dtype == ET_B200_DTYPE_F32 ? 4 : 2;
  if (rows < 8 || (rows & (rows - 1)) != 0 || encode_fn() == nullptr ||
      c->page_stride * size >= (int64_t)1 << 40 || c->head_stride * size >= (int64_t)1 << 40)
    return false;
  const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->page_size,
                              (cuuint64_t)c->kv_heads, (cuuint64_t)c->pages};
  const cuuint64_t strides[3] = {(cuuint64_t)(c->token_stride * size),
                                 (cuuint64_t)(c->head_stride * size),
                                 (cuuint64_t)(c->page_stride * size)};
  const cuuint32_t box[4] = {(cuuint32_t)wide, (cuuint32_t)box_rows, 1, 1}, one[4] = {1, 1, 1, 1};
  const auto type = c->dtype == ET_B200_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                    : c->dtype == ET_B200_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return encode_fn()(map, type, 4, pool, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     !swizzled            ? CU_TENSOR_MAP_SWIZZLE_NONE
                     : wide * size == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                         : CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

Pools pools_of(const et_b200_paged_cache_v1* c) {
  return Pools{c->pages, c->page_stride, c->head_stride, c->token_stride, (int)c->page_size,
               (int)c->kv_heads, (int)c->head_dim, divisor_of((uint32_t)c->page_size)};
}
Batch batch_of(const et_b200_paged_batch_v1* b, int64_t page_size) {
  return Batch{b->offsets, b->lengths, b->page_table, b->status, b->tokens, b->table_columns,
               (int)b->batch, (int)(b->table_columns * page_size)};
}
Rope rope_of(const et_b200_paged_rope_v1* r) {
  return r == nullptr ? Rope{nullptr, nullptr, 0} : Rope{r->cos, r->sin, r->rows};
}

}  // namespace paged
}  // namespace etb

using namespace etb;
using namespace etb::paged;

extern "C" int32_t et_b200_paged_append_v1(const et_b200_paged_cache_v1* c,
                                           const et_b200_paged_batch_v1* b,
                                           const et_b200_paged_rope_v1* rope, const void* k,
                                           int64_t k_stride, const void* v, int64_t v_stride,
                                           void* stream, et_kernel_error* e) {
  const char* op = "paged-append";
  if (int32_t r = check_cache(c, e, op)) return r;
  if (int32_t r = check_batch(b, c->page_size, e, op)) return r;
  if (int32_t r = check_rope(rope, e, op)) return r;
  const int64_t row = c->kv_heads * c->head_dim, size = c->dtype == ET_B200_DTYPE_F32 ? 4 : 2;
  if (b->tokens > 0 && b->batch > 0) {
    if (int32_t r = check_new_rows(k, k_stride, v, v_stride, row, size, e, op)) return r;
    const Pools P = pools_of(c);
    const Batch B = batch_of(b, c->page_size);
    const Rope R = rope_of(rope);
    auto st = static_cast<cudaStream_t>(stream);
    if (c->dtype == ET_B200_DTYPE_F32) launch_append<float>(c, P, B, R, k, k_stride, v, v_stride, st);
    else if (c->dtype == ET_B200_DTYPE_F16) launch_append<__half>(c, P, B, R, k, k_stride, v, v_stride, st);
    else launch_append<__nv_bfloat16>(c, P, B, R, k, k_stride, v, v_stride, st);
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return cuda_error(e, status, op);
  }
  if (e) memset(e, 0, sizeof(*e));
  return 0;
}
