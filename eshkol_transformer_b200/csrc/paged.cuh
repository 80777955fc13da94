// Pieces the paged-cache kernels share: kernel arguments, safe reads of a
// request's device metadata, element conversions and the division of the
// attention's work among the thread blocks.
#pragma once

#include <cuda_bf16.h>

#include "ops.cuh"
#include "tcgen05.cuh"

namespace etb {
namespace paged {

// The arithmetic on a request's metadata also runs on the host (its tests).
#define ETB_HD __host__ __device__ __forceinline__
template <typename I> ETB_HD I least_of(I a, I b) { return a < b ? a : b; }
template <typename I> ETB_HD I most_of(I a, I b) { return a > b ? a : b; }

// Division by a fixed d: for 0 <= n < 2^31, n / d = n m >> (31 + l) with l =
// ceil(log2 d) and m = ceil(2^(31 + l) / d) (Granlund & Montgomery, 1994: m
// exceeds 2^(31 + l) / d by less than 2^l / d, which n < 2^31 cannot carry
// into the quotient).
struct Divisor {
  uint32_t d, m;
  int shift;  // l - 1, of the product's upper half
};
inline Divisor divisor_of(uint32_t d) {
  int l = 0;
  while (((uint64_t)1 << l) < d) l++;
  if (l == 0) return Divisor{1, 0, 0};
  return Divisor{d, (uint32_t)((((uint64_t)1 << (31 + l)) + d - 1) / d), l - 1};
}
ETB_HD int quotient(int n, const Divisor& v) {
  return v.m == 0 ? n : (int)((uint32_t)(((uint64_t)(uint32_t)n * v.m) >> 32) >> v.shift);
}

struct Pools {
  int64_t pages, page_stride, head_stride, token_stride;
  int page_size, kv_heads, head_dim;
  Divisor by_page;
};
// Most keys of a page table: positions, rounded up to whole blocks of keys and of
// look-ups, stay 32-bit numbers.
constexpr int64_t kMostCapacity = INT32_MAX - 4096;
struct Batch {
  const int64_t* offsets;
  const int64_t* lengths;
  const int32_t* table;
  int* status;
  int64_t tokens, columns;
  int batch, capacity;  // capacity = columns * page_size
};
struct Rope {
  const float* cos;
  const float* sin;
  int64_t rows;
};

__device__ __forceinline__ void report(int* status, int bit) {
  if (status != nullptr) atomicOr(status, bit);
}

// A block's abort word is also the error word of its bounded waits (role_wait,
// mbar_wait): the one that runs out sets it, whichever role waits, the other roles'
// waits then give up, and who comes last tells the caller.
__device__ __forceinline__ void report_abort(int* status, volatile int* abort) {
  if (*abort != 0) report(status, ET_B200_PAGED_TIMEOUT);
}

// A request's new tokens (rows first .. first + n - 1 of the tensors) and its
// length, clamped to the tensors and the page table; `bad` holds the status
// bits of what had to be clamped.
struct Request {
  int64_t first;
  int n, len, bad;
};
ETB_HD Request load_request(const Batch& B, int b) {
  const int64_t o0 = B.offsets[b], o1 = B.offsets[b + 1], l = B.lengths[b];
  const int64_t a = least_of(most_of(o0, (int64_t)0), B.tokens);
  const int64_t e = least_of(most_of(o1, a), B.tokens);
  const int64_t len = least_of(most_of(l, (int64_t)0), (int64_t)B.capacity);
  return Request{a, (int)(e - a), (int)len,
                 ((a != o0 || e != o1) ? ET_B200_PAGED_BAD_OFFSET : 0) |
                     (len != l ? ET_B200_PAGED_BAD_LENGTH : 0)};
}

// Element offset of slot 0 dims of `key` (0 <= key < capacity) of request b
// in the pools for head h; -1 for a page outside the pool.
ETB_HD int64_t key_offset(const Pools& P, const Batch& B, int b, int h,
                                              int key) {
  const int column = quotient(key, P.by_page), slot = key - column * P.page_size;
  const int64_t page = B.table[(int64_t)b * B.columns + column];
  if (page < 0 || page >= P.pages) return -1;
  return page * P.page_stride + h * P.head_stride + slot * P.token_stride;
}

// ---- element types ------------------------------------------------------------------

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) {
  return __float2half_rn(x);
}
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// ---- pairs of f32 in one register pair: two operations per instruction ----------------

__device__ __forceinline__ uint64_t pk(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpk(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t twice(float a) { return pk(a, a); }

// RoPE of the pair (x0, x1) in the reference's rounding order
// (native/a2_attention_provider.c:792-935).
__device__ __forceinline__ void rotate(float& x0, float& x1, float c, float s) {
  const float a = rn_mul(x0, c), b = rn_mul(x1, s), d = rn_mul(x0, s), e = rn_mul(x1, c);
  x0 = rn_sub(a, b);
  x1 = rn_add(d, e);
}
// The table row of a position: the last one for positions beyond the tables.
__device__ __forceinline__ int64_t rope_row(const Rope& R, int64_t pos, int* status) {
  if (pos >= R.rows) {
    report(status, ET_B200_PAGED_BAD_ROPE);
    return R.rows - 1;
  }
  return pos;
}

// ---- division of the attention's work -------------------------------------------------
//
// The rows of one (request, kv head) are its new tokens times the group of
// query heads, token-major (row r: token r / group, head r % group), cut into
// tiles of 2^row_bits; a tile walks the keys its last token sees in blocks of
// 2^key_bits.  A unit is one (tile, block); the units of all requests, ordered by
// request, head, tile, block, are divided evenly among the thread blocks
// whatever the lengths are.  A tile cut by such a border leaves partial sums,
// which a second kernel joins.
// Rows and keys are powers of two; tokens times group stay below 2^31.
struct Tiling {
  int row_bits, key_bits, group, kv_heads;
  Divisor by_group;
};
inline Tiling tiling_of(int row_bits, int key_bits, int group, int kv_heads) {
  return Tiling{row_bits, key_bits, group, kv_heads, divisor_of((uint32_t)group)};
}
ETB_HD int tile_count(const Tiling& t, const Request& r) {
  return (r.n * t.group + (1 << t.row_bits) - 1) >> t.row_bits;
}
// Keys that the last row of a tile sees (0 when it stands before position 0).
ETB_HD int tile_visible(const Tiling& t, const Request& r, int tile) {
  const int last = least_of((tile + 1) << t.row_bits, r.n * t.group) - 1;
  return most_of(0, r.len - r.n + quotient(last, t.by_group) + 1);
}
ETB_HD int tile_units(const Tiling& t, const Request& r, int tile) {
  return most_of(1, (tile_visible(t, r, tile) + (1 << t.key_bits) - 1) >> t.key_bits);
}
ETB_HD int64_t head_units(const Tiling& t, const Request& r) {
  const int tiles = tile_count(t, r);
  int64_t s = 0;
  for (int i = 0; i < tiles; i++) s += tile_units(t, r, i);
  return s;
}

// Where a thread block stands: block `blk` of `nblk` of a tile.
struct Place {
  Request r;
  int b, h, tile, tiles, blk, nblk;
};
ETB_HD void enter_tile(const Tiling& t, Place& p) {
  p.blk = 0;
  p.nblk = tile_units(t, p.r, p.tile);
}
// The next unit; past the last one of the batch b == B.batch.
ETB_HD void advance(const Tiling& t, const Batch& B, Place& p) {
  if (++p.blk < p.nblk) return;
  if (++p.tile == p.tiles) {
    p.tile = 0;
    if (++p.h == t.kv_heads) {
      p.h = 0;
      do {
        if (++p.b >= B.batch) return;
        p.r = load_request(B, p.b);
      } while (p.r.n == 0);
      p.tiles = tile_count(t, p.r);
    }
  }
  enter_tile(t, p);
}

struct Share {
  int64_t units;  // of this thread block
  int64_t per;    // of every thread block but the last
};
// This block's share of the units and where it begins; every thread of the
// NT-thread block calls it and gets the same.
template <int NT>
struct DivideRoom {  // shared memory
  int64_t warp_sum[NT / 32];
  int64_t found[2];
  Request request;
};
template <int NT>
__device__ Share divide(const Tiling& t, const Batch& B, int64_t least, Place& p,
                        DivideRoom<NT>& room) {
  int64_t* warp_sum_s = room.warp_sum;
  int64_t* found_s = room.found;
  Request& request_s = room.request;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Request mine_r{0, 0, 0, 0};
  int64_t per_head = 0;
  auto units_of = [&](int b) -> int64_t {
    if (b >= B.batch) return 0;
    mine_r = load_request(B, b);
    if (mine_r.bad != 0 && blockIdx.x == 0) report(B.status, mine_r.bad);
    return (per_head = head_units(t, mine_r)) * t.kv_heads;
  };
  // inclusive scan over the block; *all receives the block's sum
  auto scan = [&](int64_t v, int64_t* all) -> int64_t {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) warp_sum_s[warp] = v;
    __syncthreads();
    int64_t before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; w++) {
      if (w < warp) before += warp_sum_s[w];
      sum += warp_sum_s[w];
    }
    *all = sum;
    return v + before;
  };
  int64_t total = 0, mine = 0, incl = 0;
  for (int base = 0; base < B.batch; base += NT) {
    int64_t all;
    mine = units_of(base + tid);
    incl = scan(mine, &all);
    total += all;
  }
  Share s;
  s.per = max(least, total < INT32_MAX - (int)gridDim.x
                         ? (int64_t)(((uint32_t)total + gridDim.x - 1) / gridDim.x)
                         : (total + gridDim.x - 1) / gridDim.x);
  const int64_t u0 = (int64_t)blockIdx.x * s.per;
  s.units = max((int64_t)0, min(total - u0, s.per));
  p.b = B.batch;
  if (s.units == 0) return s;
  if (tid == 0) found_s[0] = B.batch;
  __syncthreads();
  int64_t before = 0;
  for (int base = 0; base < B.batch; base += NT) {
    int64_t all;
    if (B.batch > NT) {
      mine = units_of(base + tid);
      incl = scan(mine, &all);
    } else {
      all = total;
    }
    const int64_t from = before + incl - mine;
    if (from <= u0 && u0 < from + mine) {
      found_s[0] = base + tid;
      int64_t rest = u0 - from;
      int h = 0;
      for (; rest >= per_head; rest -= per_head) h++;
      found_s[1] = ((int64_t)h << 48) | rest;  // units of a head stay below 2^45
      request_s = mine_r;
    }
    before += all;
    if (u0 < before) break;
  }
  __syncthreads();
  p.b = (int)found_s[0];
  if (p.b >= B.batch) {  // the lengths changed between the two passes: nothing is followed
    s.units = 0;
    return s;
  }
  int64_t rest = found_s[1] & (((int64_t)1 << 48) - 1);
  p.h = (int)(found_s[1] >> 48);
  p.r = request_s;
  p.tiles = tile_count(t, p.r);
  p.tile = 0;
  enter_tile(t, p);
  while (rest >= p.nblk) {
    rest -= p.nblk;
    p.tile++;
    enter_tile(t, p);
  }
  p.blk = (int)rest;
  return s;
}

// ---- joining of cut tiles --------------------------------------------------------------
//
// Workspace: per thread block a Cut (the tile it began and did not finish,
// parts == 0 for none), then two slots of partial results: slot 0 for the
// tile it continued, slot 1 for the tile it began.  A slot holds the
// unnormalised sums [rows][dim] relative to the row's maximum, the maxima
// (base 2) and the sums of exponentials.
struct Cut {
  int64_t first;
  int n, h, tile, parts;
};
struct Joint {
  Cut* cuts;
  float* sums;   // [blocks][2][rows][dim]
  float* stats;  // [blocks][2][2][rows]: maxima, sums of exponentials
};
constexpr size_t kCutBytes = 64;
__host__ __device__ inline size_t joint_bytes(int blocks, int rows, int dim) {
  return (size_t)blocks * (kCutBytes + 2 * sizeof(float) * (size_t)rows * (dim + 2));
}
inline Joint joint_of(void* ws, int blocks, int rows, int dim) {
  Joint j;
  j.cuts = static_cast<Cut*>(ws);
  j.sums = reinterpret_cast<float*>(static_cast<char*>(ws) + (size_t)blocks * kCutBytes);
  j.stats = j.sums + (size_t)blocks * 2 * rows * dim;
  return j;
}

struct AttendArgs {
  Pools pools;
  Batch batch;
  Rope rope;
  Tiling tiling;
  Joint joint;
  const void* keys;
  const void* values;
  const void* q;
  void* o;
  float* lse;
  int64_t q_stride, o_stride, least;
  int q_heads, sms;  // SMs of the device
  float scale_log2;  // log2(e) / sqrt(head_dim), and 1 / q_factor
  // 1/2 for rotated f16 queries, whose elements reach sqrt(2) times the largest f16;
  // else 1
  float q_factor;
};

// ---- TMA from the pools ---------------------------------------------------------------

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// Map of a pool for boxes of `wide` dims (swizzled: of 64 or 128 bytes, and as
// wide as that) x box_rows slots of one head of one page; dims beyond head_dim and pages
// outside the pool read as zeros.  False for pools it cannot describe (pages
// that are no power of two of at least 8 slots, far strides).
bool pool_map(CUtensorMap* map, void* pool, const et_b200_paged_cache_v1* c, int wide, int box_rows,
              bool swizzled = true);

// Host pieces of the entry points.
template <typename... P>
inline bool aligned_to(uintptr_t bytes, P... pointers) {
  return ((reinterpret_cast<uintptr_t>(pointers) | ...) & (bytes - 1)) == 0;
}
int32_t check_cache(const et_b200_paged_cache_v1* c, et_kernel_error* e, const char* op);
int32_t check_batch(const et_b200_paged_batch_v1* b, const et_b200_paged_cache_v1* c,
                    et_kernel_error* e, const char* op);
int32_t check_rope(const et_b200_paged_rope_v1* r, et_kernel_error* e, const char* op);
Pools pools_of(const et_b200_paged_cache_v1* c);
Batch batch_of(const et_b200_paged_batch_v1* b, const et_b200_paged_cache_v1* c);
Rope rope_of(const et_b200_paged_rope_v1* r);
// `most` thread blocks, or fewer where the host's sizes leave fewer units.
inline int thread_blocks(const AttendArgs& a, int most, int rows, int keys) {
  const int64_t tiles = (a.batch.tokens * a.tiling.group / rows + a.batch.batch) * a.pools.kv_heads;
  const int64_t blocks = (a.batch.capacity + keys - 1) / keys;
  return blocks < most && tiles * blocks < most ? (int)(tiles * blocks) : most;
}
// The tcgen05 kernel (paged_attention_tc.cu): launches it and returns its
// thread blocks, 0 where it does not take the cache (nothing is launched).
size_t attend_tc_workspace(int dim_padded, int sms);
int attend_tc(const et_b200_paged_cache_v1* c, AttendArgs& a, void* ws, cudaStream_t stream);
// The same for f32 caches (paged_attention_f32.cu); its workspace is within
// attend_tc_workspace.
int attend_f32(const et_b200_paged_cache_v1* c, AttendArgs& a, void* ws, cudaStream_t stream);

}  // namespace paged
}  // namespace etb
