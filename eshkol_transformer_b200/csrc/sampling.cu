// Sampling one token per row of logits (et_b200_sample_v1).
//
// Weights w(x) = exp((x - M) / temperature), M the row's maximum, as 2^-40
// fixed point: integer sums are the same in every order, so cumulative sums,
// cuts and draws are deterministic whatever the thread layout.  A cut (top-k,
// top-p) is a pair (key, index): the tokens above a logit, and of those equal
// to it the ones up to an index; it is found by radix selection on the
// monotone integer image of the logits, counting tokens or adding their
// weights per digit.  The draw inverts the running sum in vocabulary order.
#include <math.h>

#include <type_traits>

#include "paged.cuh"

namespace etb {
namespace {

using paged::to_f32;

constexpr int NT = 512, WARPS = NT / 32;
constexpr int BINS = 2048;
constexpr int FRACTION = 40;  // weights are multiples of 2^-40

// Monotone integer image of a logit; NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  if (x != x) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr uint32_t kKeyMinusInf = 0x007fffffu;  // key_of(-inf)

struct Scale {
  float max, hi, lo;  // hi + lo = log2(e) / temperature
};

// exp((x - max) / temperature) 2^40, rounded.  t = (x - max) (hi + lo) keeps
// the rounding errors of the difference and the products, 2^t = 2^n 2^f with
// 2^f - 1 by its series (|f| <= 1/2, terms up to f^7: 5e-9), so the relative
// error stays near 3e-8 whatever the size of the logits.
__device__ __forceinline__ uint64_t weight_of(float x, const Scale& s) {
  if (!(x > -INFINITY)) return 0;
  if (s.max == INFINITY) return x == INFINITY ? 1ull << FRACTION : 0;
  const float d = x - s.max;
  const float t = d * s.hi;
  if (!(t >= -(float)(FRACTION + 1))) return 0;
  const float bb = d - x;
  const float e = (x - (d - bb)) - (s.max + bb);
  const float rest = fmaf(d, s.hi, -t) + fmaf(d, s.lo, e * s.hi);
  const float n = rintf(t);
  const float f = (t - n) + rest;
  float y = 1.5252734e-5f;
  y = fmaf(y, f, 1.5403530e-4f);
  y = fmaf(y, f, 1.3333558e-3f);
  y = fmaf(y, f, 9.6181291e-3f);
  y = fmaf(y, f, 5.5504109e-2f);
  y = fmaf(y, f, 2.4022651e-1f);
  y = fmaf(y, f, 6.9314718e-1f);
  y *= f;
  const int k = FRACTION + (int)n;  // -1 .. 40
  const float p = __uint_as_float((uint32_t)(127 + k) << 23);
  const int64_t whole = k >= 0 ? (int64_t)1 << k : 0;
  return (uint64_t)(k >= 0 ? whole + __float2ll_rn(y * p) : __float2ll_rn(fmaf(y, p, p)));
}

struct Shared {
  uint32_t low[BINS], high[BINS];
  uint64_t warp[WARPS];
  uint64_t found[3];
};

__device__ __forceinline__ uint64_t warp_scan(uint64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
// Inclusive sum over the block up to this thread; *all: the block's.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, Shared& sm, uint64_t* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan(v);
  __syncthreads();
  if (lane == 31) sm.warp[warp] = v;
  __syncthreads();
  uint64_t before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < WARPS; w++) {
    if (w < warp) before += sm.warp[w];
    sum += sm.warp[w];
  }
  *all = sum;
  return v + before;
}

struct Cut {
  uint32_t key;   // tokens above it are kept,
  int64_t index;  // and those equal to it up to this index
};
__device__ __forceinline__ bool kept(const Cut& c, uint32_t key, int i) {
  return key > c.key || (key == c.key && i <= c.index);
}

// First index at which the running sum of weight(i), in index order, reaches
// aim(total); aim is at least 1 and at most the total.
template <typename Weight, typename Aim>
__device__ int in_order(int n, Shared& sm, Weight weight, Aim aim) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int span = (n + WARPS - 1) / WARPS;
  const int w0 = min(n, warp * span), w1 = min(n, w0 + span);
  uint64_t sum = 0;
  for (int i = w0 + lane; i < w1; i += 32) sum += weight(i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) sm.warp[warp] = sum;
  __syncthreads();
  uint64_t total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; w++) total += sm.warp[w];
  uint64_t rest = aim(total);
  int at = 0;
  while (at < WARPS - 1 && rest > sm.warp[at]) rest -= sm.warp[at++];
  const int s0 = min(n, at * span), s1 = min(n, s0 + span);
  const int each = (span + NT - 1) / NT;
  const int t0 = min(s1, s0 + tid * each), t1 = min(s1, t0 + each);
  uint64_t mine = 0, all;
  for (int i = t0; i < t1; i++) mine += weight(i);
  const uint64_t incl = block_scan(mine, sm, &all);
  if (incl - mine < rest && rest <= incl) {
    uint64_t run = incl - mine;
    int i = t0;
    for (; i < t1; i++) {
      run += weight(i);
      if (run >= rest) break;
    }
    sm.found[0] = (uint64_t)i;
    sm.found[1] = total;
  }
  __syncthreads();
  return (int)sm.found[0];
}

// Lowers `cut` to the shortest prefix of the ranking (logit descending, index
// ascending) of the tokens it keeps whose weights reach aim(total) (0: all).
// unit(key) is the weight of a token with that key.
template <typename Key, typename Unit, typename Aim>
__device__ void select(int n, Shared& sm, Cut& cut, Key key_at, Unit unit, Aim aim) {
  const int tid = threadIdx.x;
  uint32_t prefix = 0;
  uint64_t rest = 0, tied = 0;
#pragma unroll
  for (int level = 0; level < 3; level++) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
    const int above = level == 0 ? 32 : level == 1 ? 21 : 10;
    const uint32_t mask = level == 2 ? 1023u : 2047u;
    __syncthreads();
    for (int i = tid; i < BINS; i += NT) sm.low[i] = sm.high[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const uint32_t key = key_at(i);
      if (level > 0 && (key >> above) != prefix) continue;
      if (!kept(cut, key, i)) continue;
      const uint64_t w = unit(key);
      if (w == 0) continue;
      const uint32_t bin = (key >> shift) & mask;
      const uint32_t lo = (uint32_t)w;
      const uint32_t old = atomicAdd(&sm.low[bin], lo);
      const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
      if (hi != 0) atomicAdd(&sm.high[bin], hi);
    }
    __syncthreads();
    uint64_t bins[BINS / NT], mine = 0, all;
#pragma unroll
    for (int j = 0; j < BINS / NT; j++) {
      const int bin = BINS - 1 - (tid * (BINS / NT) + j);
      bins[j] = ((uint64_t)sm.high[bin] << 32) | sm.low[bin];
      mine += bins[j];
    }
    const uint64_t incl = block_scan(mine, sm, &all);
    if (level == 0) {
      rest = aim(all);
      if (rest == 0 || rest > all) return;
    }
    uint64_t run = incl - mine;
    if (run < rest && rest <= incl) {
#pragma unroll
      for (int j = 0; j < BINS / NT; j++) {
        if (run < rest && rest <= run + bins[j]) {
          sm.found[0] = (uint64_t)(BINS - 1 - (tid * (BINS / NT) + j));
          sm.found[1] = rest - run;
          sm.found[2] = bins[j];
        }
        run += bins[j];
      }
    }
    __syncthreads();
    prefix = level == 0 ? (uint32_t)sm.found[0]
                        : (prefix << (level == 1 ? 11 : 10)) | (uint32_t)sm.found[0];
    rest = sm.found[1];
    tied = sm.found[2];
  }
  // `prefix` is the key of the last kept token; of its ties the first
  // ceil(rest / unit) by index stay
  const Cut old = cut;
  const uint64_t one = unit(prefix);
  const uint64_t count = (rest + one - 1) / one;
  cut.key = prefix;
  cut.index = INT64_MAX;
  if (count * one < tied) {
    const uint32_t tie = prefix;
    cut.index = in_order(
        n, sm,
        [&](int i) -> uint64_t {
          const uint32_t key = key_at(i);
          return key == tie && kept(old, key, i) ? 1u : 0u;
        },
        [&](uint64_t) { return count; });
  } else if (old.key == prefix) {
    cut.index = old.index;
  }
}

__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

template <typename T>
__global__ void __launch_bounds__(NT)
sample_kernel(const T* __restrict__ logits, int64_t row_stride, int n,
              const float* __restrict__ uniform, const float* __restrict__ temperature,
              const int64_t* __restrict__ top_k, const float* __restrict__ top_p,
              const float* __restrict__ min_p, int64_t* __restrict__ ids,
              float* __restrict__ logprobs) {
  __shared__ Shared sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * row_stride;
  auto key_at = [&](int i) { return key_of(to_f32<T>(x[i])); };

  // the largest logit, of equal ones the first
  uint64_t best = 0;
  for (int i = tid; i < n; i += NT) {
    const uint64_t v = ((uint64_t)key_at(i) << 32) | (0xffffffffu - (uint32_t)i);
    best = max(best, v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) sm.warp[warp] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; w++) best = max(best, sm.warp[w]);
  const uint32_t best_key = (uint32_t)(best >> 32);
  const int64_t best_index = (int64_t)(0xffffffffu - (uint32_t)best);
  if (best_key <= kKeyMinusInf) {
    if (tid == 0) {
      ids[row] = -1;
      if (logprobs != nullptr) logprobs[row] = -INFINITY;
    }
    return;
  }
  const float temp = temperature != nullptr ? temperature[row] : 1.0f;
  if (!(temp > 0x1p-100f)) {
    if (tid == 0) {
      ids[row] = best_index;
      if (logprobs != nullptr) logprobs[row] = 0.0f;
    }
    return;
  }
  const double per = 1.4426950408889634 / (double)temp;
  Scale sc;
  sc.max = value_of(best_key);
  sc.hi = (float)per;
  sc.lo = (float)(per - (double)sc.hi);

  auto unit = [&](uint32_t key) { return weight_of(value_of(key), sc); };
  Cut cut{kKeyMinusInf, -1};
  const int64_t k = top_k != nullptr ? top_k[row] : 0;
  if (k > 0 && k < n)
    select(n, sm, cut, key_at, [](uint32_t) -> uint64_t { return 1; },
           [&](uint64_t all) { return (uint64_t)k < all ? (uint64_t)k : 0ull; });
  const float share = top_p != nullptr ? top_p[row] : 1.0f;
  if (share < 1.0f)
    select(n, sm, cut, key_at, unit, [&](uint64_t all) {
      const double aim = ceil((double)share * (double)all);
      return aim > 1.0 ? (uint64_t)aim : 1ull;
    });
  const float low = min_p != nullptr ? min_p[row] : 0.0f;
  if (low > 0.0f && sc.max < INFINITY) {
    const double least = (double)sc.max + (double)temp * log((double)fminf(low, 1.0f));
    float f = (float)least;
    if ((double)f < least) f = nextafterf(f, INFINITY);
    const uint32_t key = key_of(f);
    if (key > cut.key) cut = Cut{key, INT64_MAX};
  }

  const double u = (double)uniform[row];
  uint64_t total = 0;
  const int id = in_order(
      n, sm,
      [&](int i) -> uint64_t {
        const uint32_t key = key_at(i);
        return kept(cut, key, i) ? unit(key) : 0;
      },
      [&](uint64_t all) {
        total = all;
        const double aim = u > 0.0 ? u * (double)all : 0.0;
        return aim < (double)all ? min((uint64_t)aim + 1, all) : all;
      });
  if (tid == 0) {
    ids[row] = id;
    if (logprobs != nullptr) {
      const double d = sc.max == INFINITY ? 0.0 : (double)to_f32<T>(x[id]) - (double)sc.max;
      logprobs[row] = (float)(d / (double)temp - log((double)total * 0x1p-40));
    }
  }
}

}  // namespace
}  // namespace etb

using namespace etb;

extern "C" int32_t et_b200_sample_v1(const et_b200_sampling_v1* s, const void* logits,
                                     const float* uniform, int64_t* ids, float* logprobs,
                                     void* stream, et_kernel_error* e) {
  const char* op = "sample";
  if (s == nullptr || s->struct_size < sizeof(et_b200_sampling_v1))
    return set_error(e, ET_KERNEL_ERROR_VERSION_MISMATCH, ET_KERNEL_CODE_INVALID_STRUCT_SIZE, op,
                     "sampling descriptor is missing or truncated");
  if (s->dtype > ET_B200_DTYPE_BF16)
    return set_error(e, ET_KERNEL_ERROR_DTYPE_MISMATCH, ET_KERNEL_CODE_INVALID_ENUM, op,
                     "unknown element type of the logits");
  if (s->rows < 0 || s->rows > INT32_MAX || s->vocabulary < 1 || s->vocabulary > (1 << 22) ||
      s->row_stride < s->vocabulary || s->row_stride > (int64_t)1 << 31)
    return set_error(e, ET_KERNEL_ERROR_SHAPE_MISMATCH, ET_KERNEL_CODE_INVALID_SHAPE, op,
                     "rows, vocabulary or row stride are outside their limits");
  if (s->rows > 0) {
    if (logits == nullptr || uniform == nullptr || ids == nullptr)
      return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_NULL_ARGUMENT, op,
                       "logits, uniform numbers and ids are required");
    const uintptr_t size = s->dtype == ET_B200_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % size != 0)
      return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_INVALID_BUFFER, op,
                       "logits must be aligned to their elements");
    auto st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto t) {
      using T = decltype(t);
      sample_kernel<T><<<(unsigned)s->rows, NT, 0, st>>>(
          static_cast<const T*>(logits), s->row_stride, (int)s->vocabulary, uniform,
          s->temperature, s->top_k, s->top_p, s->min_p, ids, logprobs);
    };
    if (s->dtype == ET_B200_DTYPE_F32) go(float{});
    else if (s->dtype == ET_B200_DTYPE_F16) go(__half{});
    else go(__nv_bfloat16{});
    count_launch();
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return cuda_error(e, status, op);
  }
  if (e) memset(e, 0, sizeof(*e));
  return 0;
}
