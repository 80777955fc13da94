// Sampling one token per row of logits (et_b200_sample_v1).
//
// Weights w(x) = exp((x - M) / temperature), M the row's maximum, as 2^-35
// fixed point: integer sums are the same in every order, so cumulative sums,
// cuts and draws are deterministic whatever the thread layout.  A cut (top-k,
// top-p) is a pair (logit, index): the tokens above a logit, and of those
// equal to it the ones up to an index.  The draw inverts the running sum in
// vocabulary order.
//
// A row is read from memory once, into the shared memory of a cluster of
// thread blocks (each a contiguous slice; as many as the slices need, more
// when there are few rows), while its maximum is formed.  Then
//  - a small top-k (or a small vocabulary) becomes a list: every slice pushes
//    what reaches a lower bound of the row's k-th largest logit (from the maxima
//    of its threads) to one block, which ranks it, cuts it by all filters, adds
//    up what is left in the order of the vocabulary and draws;
//  - otherwise a cut is found from a histogram (tokens or weights) over 1,024
//    steps of the logit, the border's step is gathered and ranked, and the draw
//    adds the kept weights slice by slice, warp by warp.
// Greedy rows take 30 us for 256 rows of 128,259 bf16 logits, 10 us of it reading at
// the copy rate and the rest the thread blocks' set-up, which nothing overlaps.
// Otherwise it is instructions, 58 per logit without a filter (128 rows of 50,257:
// 26.7 us) and 150 with a nucleus (three passes evaluate the weights), issued in half
// to 60 % of the cycles between the cluster's barriers, and for few rows the latency
// of the steps that one thread block or cluster takes alone.
// Rows for which the list or the border's step overflows (thousands of equal
// logits) or the slices do not fit are selected by radix from memory.
#include <math.h>

#include <cooperative_groups.h>

#include <type_traits>

#include "paged.cuh"

namespace etb {
namespace {

using paged::add2;
using paged::fma2;
using paged::pk;
using paged::to_f32;
using paged::twice;
using paged::unpk;
namespace cg = cooperative_groups;

constexpr int NT = 512, WARPS = NT / 32;
constexpr int BINS = 2048;

// Monotone integer image of a logit; NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  if (x != x) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr uint32_t kKeyMinusInf = 0x007fffffu;  // key_of(-inf)

// log2(e) / temperature = hi + lo.  shift = M (hi + lo) = shift_hi + shift_lo
// with shift_hi a multiple of 2^-8 below 2^15 (narrow), so that n + shift_hi
// is exact for the integers n of the exponents; low: logits below have weight
// 0 whatever they are.
struct Scale {
  float max, hi, lo, shift, shift_hi, shift_lo, low;
  bool narrow;
};
__device__ __forceinline__ Scale scale_of(float max, double per) {
  Scale s;
  s.max = max;
  s.hi = (float)per;
  s.lo = (float)(per - (double)s.hi);
  const double shift = (double)max * per;
  s.narrow = fabs(shift) < 32000.0 && s.hi > 0x1p-60f;
  const double grid = rint(shift * 256.0) / 256.0;
  s.shift = (float)shift;
  s.shift_hi = (float)grid;
  s.shift_lo = (float)(shift - grid);
  s.low = max - 64.0f / s.hi;
  return s;
}

constexpr float kRound = 12582912.0f;  // 1.5 2^23: adding it rounds to an integer
// 2^f = 1 + f (c1 + f (c2 + ...)), ck = ln(2)^k / k! to k = 7: |f| <= 1/2, error
// 5e-9.  exp((x - max) / temperature) = 2^t, t = (x - max) (hi + lo) = n + f; f is
// accurate to about 2^-25 because its one large difference is an fma whose
// other operand is exact.  Relative error near 6e-8 whatever the size of the
// logits.
__device__ __forceinline__ float power_of(float x, const Scale& s) {
  float n, f;
  if (s.narrow) {
    x = fmaxf(x, s.low);  // NaN too
    n = (fmaf(x, s.hi, -s.shift) + kRound) - kRound;
    f = fmaf(x, s.hi, -n - s.shift_hi) + fmaf(x, s.lo, -s.shift_lo);
  } else {
    if (!(x > -INFINITY)) return 0.0f;
    if (s.max == INFINITY) return x == INFINITY ? 1.0f : 0.0f;
    const float d = x - s.max;
    if (d == -INFINITY) {  // further apart than the largest f32: of weight at such temperatures only
      const float t = fmaf(x, s.hi, -s.max * s.hi);
      n = rintf(fmaxf(t, -64.0f));
      f = t < -64.0f ? 0.0f : t - n;
    } else {
      const float t = d * s.hi;
      if (!(t >= -64.0f)) return 0.0f;
      const float bb = d - x, e = (x - (d - bb)) - (s.max + bb);
      n = rintf(t);
      f = (t - n) + (fmaf(d, s.hi, -t) + fmaf(d, s.lo, e * s.hi));
    }
  }
  float y = 1.5252734e-5f;
  y = fmaf(y, f, 1.5403530e-4f);
  y = fmaf(y, f, 1.3333558e-3f);
  y = fmaf(y, f, 9.6181291e-3f);
  y = fmaf(y, f, 5.5504109e-2f);
  y = fmaf(y, f, 2.4022651e-1f);
  y = fmaf(y, f, 6.9314718e-1f);
  y = fmaf(y, f, 1.0f);
  return __int_as_float(__float_as_int(y) + ((int)n << 23));
}
// The weight in units of 2^-35.
__device__ __forceinline__ uint64_t weight_of(float x, const Scale& s) {
  return __float2ull_rn(power_of(x, s) * 0x1p35f);
}

// Sums of weights of up to 64 logits at a time, exact in f32: each is rounded
// to multiples of 2^-17 (sums below 2^6) and the rest to multiples of 2^-35
// (below 2^-12); both together round it as weight_of does.  Two logits per
// packed instruction (narrow scales).
struct Sum64 {
  uint64_t coarse, fine;  // f32 pairs
};
// power_of of two logits at once (narrow scales)
__device__ __forceinline__ uint64_t powers_of(float a, float b, const Scale& s) {
  const uint64_t x = pk(fmaxf(a, s.low), fmaxf(b, s.low)), hi = twice(s.hi), minus = twice(-1.0f);
  const uint64_t m = add2(fma2(x, hi, twice(-s.shift)), twice(kRound));
  const uint64_t n = add2(m, twice(-kRound));
  const uint64_t f = add2(fma2(x, hi, fma2(n, minus, twice(-s.shift_hi))),
                          fma2(x, twice(s.lo), twice(-s.shift_lo)));
  uint64_t y = twice(1.5252734e-5f);
  y = fma2(y, f, twice(1.5403530e-4f));
  y = fma2(y, f, twice(1.3333558e-3f));
  y = fma2(y, f, twice(9.6181291e-3f));
  y = fma2(y, f, twice(5.5504109e-2f));
  y = fma2(y, f, twice(2.4022651e-1f));
  y = fma2(y, f, twice(6.9314718e-1f));
  y = fma2(y, f, twice(1.0f));
  // the integers n lie in the low bits of m
  const float2 yy = unpk(y), mm = unpk(m);
  return pk(__int_as_float(__float_as_int(yy.x) + (__float_as_int(mm.x) << 23)),
            __int_as_float(__float_as_int(yy.y) + (__float_as_int(mm.y) << 23)));
}
__device__ __forceinline__ void add_weights(Sum64& sum, float a, float b, const Scale& s) {
  const uint64_t w = powers_of(a, b, s), minus = twice(-1.0f);
  const uint64_t q = add2(add2(w, twice(96.0f)), twice(-96.0f));
  const uint64_t r = fma2(q, minus, w);
  const uint64_t r2 = add2(add2(r, twice(0x1.8p-12f)), twice(-0x1.8p-12f));
  sum.coarse = add2(sum.coarse, q);
  sum.fine = add2(sum.fine, r2);
}
__device__ __forceinline__ uint64_t flush(Sum64& sum) {
  const float2 c = unpk(sum.coarse), f = unpk(sum.fine);
  const int64_t v = ((int64_t)__float2int_rn((c.x + c.y) * 0x1p17f) << 18) +
                    (int64_t)__float2int_rn(f.x * 0x1p35f) + (int64_t)__float2int_rn(f.y * 0x1p35f);
  sum.coarse = sum.fine = 0;
  return (uint64_t)v;
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

// A row's parameters, and what of them takes long double precision arithmetic
// (formed while the logits arrive).
struct Filters {
  float temperature, top_p, min_p;
  int64_t top_k;
  double uniform, per, fall;  // log2(e) / temperature, temperature ln(min_p)
};
struct Args {
  const float* uniform;
  const float* temperature;
  const int64_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* ids;
  float* logprobs;
  int64_t row_stride;
  int n, slice;  // tokens of a row, of a slice
};
__device__ __forceinline__ Filters filters_of(const Args& a, int64_t row) {
  Filters f;
  f.temperature = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  f.top_k = a.top_k != nullptr ? a.top_k[row] : 0;
  f.top_p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
  f.min_p = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  f.uniform = (double)a.uniform[row];
  f.per = 1.4426950408889634 / (double)f.temperature;
  // at an infinite temperature every logit weighs 1, which is no less than min_p
  f.fall = !(f.min_p > 0.0f) ? 0.0
           : f.temperature == INFINITY ? -(double)INFINITY
                                       : (double)f.temperature * log((double)fminf(f.min_p, 1.0f));
  return f;
}
// What the running sum has to reach: the first integer above u total, inside
// [1, total].
__device__ __forceinline__ uint64_t draw_aim(double u, uint64_t total) {
  const double aim = u > 0.0 ? u * (double)total : 0.0;
  return aim < (double)total ? min((uint64_t)aim + 1, total) : total;
}
// What the ranked weights have to reach for a share p of `total`.
__device__ __forceinline__ uint64_t share_aim(float p, uint64_t total) {
  const double aim = ceil((double)p * (double)total);
  return aim > 1.0 ? (uint64_t)aim : 1ull;
}
// The least logit that min_p keeps (-inf: no limit).
__device__ __forceinline__ float least_logit(const Filters& f, float max) {
  if (!(f.min_p > 0.0f) || max == INFINITY) return -INFINITY;
  const double least = (double)max + f.fall;
  const float x = (float)least;
  return (double)x < least ? nextafterf(x, INFINITY) : x;
}
__device__ __forceinline__ void answer(const Args& a, int64_t row, int id, float x,
                                       const Filters& f, const Scale& sc, uint64_t total) {
  a.ids[row] = id;
  if (a.logprobs == nullptr) return;
  const double d = sc.max == INFINITY ? 0.0 : (double)x - (double)sc.max;
  // ln(total / w(max)) of the ratio's exponent and mantissa: 1e-7 absolute
  const float ratio = (float)total / (float)weight_of(sc.max, sc);
  int k;
  float m = frexpf(ratio, &k);
  if (m < 0.70710678f) {  // around 1, so that a ratio of 1 is exactly 0
    m *= 2.0f;
    k--;
  }
  a.logprobs[row] = (float)((d * f.per - (double)k) * 0.6931471805599453 - (double)logf(m));
}

// One thread block draws for a row in global memory: radix selection.
template <typename T>
__device__ void sample_row(const T* x, const Args& a, int64_t row, const Filters& flt,
                           const Scale& sc, Shared& sm) {
  const int n = a.n;
  auto key_at = [&](int i) { return key_of(to_f32<T>(x[i])); };
  auto unit = [&](uint32_t key) { return weight_of(value_of(key), sc); };
  Cut cut{kKeyMinusInf, -1};
  if (flt.top_k > 0 && flt.top_k < n)
    select(n, sm, cut, key_at, [](uint32_t) -> uint64_t { return 1; },
           [&](uint64_t all) { return (uint64_t)flt.top_k < all ? (uint64_t)flt.top_k : 0ull; });
  if (flt.top_p < 1.0f)
    select(n, sm, cut, key_at, unit, [&](uint64_t all) { return share_aim(flt.top_p, all); });
  const uint32_t least = key_of(least_logit(flt, sc.max));
  if (least > cut.key) cut = Cut{least, INT64_MAX};
  uint64_t total = 0;
  const int id = in_order(
      n, sm,
      [&](int i) -> uint64_t {
        const uint32_t key = key_at(i);
        return kept(cut, key, i) ? unit(key) : 0;
      },
      [&](uint64_t all) {
        total = all;
        return draw_aim(flt.uniform, all);
      });
  if (threadIdx.x == 0) answer(a, row, id, to_f32<T>(x[id]), flt, sc, total);
}

// ---- rows in the shared memory of a cluster ------------------------------------------------

constexpr int LIST = 1024;       // entries of a list, steps of a histogram
constexpr float kTopSteps = 40.0f;  // steps per unit of the logit for a large top-k

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// The largest value of a 16-byte piece; NaN only where all are.
template <typename T>
__device__ __forceinline__ float piece_max(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                 fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    union { uint32_t w; T2 h; } a, b, c, d;
    a.w = v.x; b.w = v.y; c.w = v.z; d.w = v.w;
    const T2 m = __hmax2(__hmax2(a.h, b.h), __hmax2(c.h, d.h));
    return fmaxf(to_f32<T>(m.x), to_f32<T>(m.y));
  }
}

// A slice of n logits in shared memory, stored at their global address modulo
// 16, so that whole 16-byte pieces copy and read as such.
template <typename T>
struct Slice {
  static constexpr int N = 16 / sizeof(T);
  const T* x;               // in shared memory
  int n, head, pieces;      // tokens before the first whole piece, whole pieces
  // f(i, value) for every token that may reach `least`, in no particular order
  // (16-byte pieces without one are skipped)
  template <typename F>
  __device__ __forceinline__ void each_from(float least, F f) const {
    for (int p = threadIdx.x; p < pieces; p += NT) {
      union { uint4 v; T x[N]; } u;
      u.v = *reinterpret_cast<const uint4*>(x + head + p * N);
      if (piece_max<T>(u.v) >= least)
#pragma unroll
        for (int k = 0; k < N; k++) f(head + p * N + k, to_f32<T>(u.x[k]));
    }
    const int t = threadIdx.x, tail = head + pieces * N;
    if (t < head) f(t, to_f32<T>(x[t]));
    else if (t >= 32 && tail + t - 32 < n) f(tail + t - 32, to_f32<T>(x[tail + t - 32]));
  }
  // f(i, values) for every piece of N tokens from i that may reach `least`;
  // what is no whole piece comes with the rest of its values -inf
  template <typename F>
  __device__ __forceinline__ void each_piece(float least, F f) const {
    for (int p = threadIdx.x; p < pieces + 2; p += NT) {
      float v[N], top = -INFINITY;
      int i = head + p * N;
      if (p < pieces) {
        union { uint4 v; T x[N]; } u;
        u.v = *reinterpret_cast<const uint4*>(x + i);
#pragma unroll
        for (int k = 0; k < N; k++) v[k] = to_f32<T>(u.x[k]);
      } else {
        i = p == pieces ? 0 : head + pieces * N;
        const int end = p == pieces ? head : n;
#pragma unroll
        for (int k = 0; k < N; k++) v[k] = i + k < end ? to_f32<T>(x[i + k]) : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < N; k++) top = fmaxf(top, v[k]);
      if (top >= least) f(i, v);
    }
  }
  // f(i, value) for every token, in no particular order
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int p = threadIdx.x; p < pieces; p += NT) {
      union { uint4 v; T x[N]; } u;
      u.v = *reinterpret_cast<const uint4*>(x + head + p * N);
#pragma unroll
      for (int k = 0; k < N; k++) f(head + p * N + k, to_f32<T>(u.x[k]));
    }
    const int t = threadIdx.x, tail = head + pieces * N;
    if (t < head) f(t, to_f32<T>(x[t]));
    else if (t >= 32 && tail + t - 32 < n) f(tail + t - 32, to_f32<T>(x[tail + t - 32]));
  }
};

// Sorts a[0 .. n), n a power of two, descending.
__device__ void sort_descending(uint64_t* a, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += NT) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const uint64_t u = a[lo], v = a[hi];
        if ((u < v) == ((lo & size) == 0)) {
          a[lo] = v;
          a[hi] = u;
        }
      }
    }
  __syncthreads();
}
// Pads a list of n entries with zeros to a power of two; that power.
__device__ int pad_list(uint64_t* a, int n) {
  int size = 32;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += NT) a[i] = 0;
  return size;
}
__device__ __forceinline__ uint64_t entry_of(float x, int index) {
  return ((uint64_t)key_of(x) << 32) | (0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ float entry_value(uint64_t e) { return value_of((uint32_t)(e >> 32)); }
__device__ __forceinline__ int entry_index(uint64_t e) { return (int)(0xffffffffu - (uint32_t)e); }

struct Border {
  float value;  // tokens above it are kept,
  int index;    // and those equal to it up to this index
};
__device__ __forceinline__ bool kept(const Border& b, float x, int i) {
  return x > b.value || (x == b.value && i <= b.index);
}

struct Room {
  union {
    struct { uint64_t list[LIST], all[LIST]; };  // a block's list, the cluster's
    struct { uint32_t low[LIST], high[LIST]; };  // a histogram
    Shared radix;
  };
  uint64_t warp[WARPS];
  uint64_t found[4];
  float top, bound;
  int count, keep, step, before;
  Border border;
  uint64_t total;
};

// Inclusive sum over the block; *all: the block's.
__device__ __forceinline__ uint64_t room_scan(uint64_t v, Room& rm, uint64_t* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan(v);
  __syncthreads();
  if (lane == 31) rm.warp[warp] = v;
  __syncthreads();
  uint64_t before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < WARPS; w++) {
    if (w < warp) before += rm.warp[w];
    sum += rm.warp[w];
  }
  *all = sum;
  return v + before;
}

// A value that at least k of the threads' maxima (`mine`, `top` the largest)
// reach, so a lower bound of the k-th largest logit of the slice, and not many
// more than 5 k / 4: histograms of 256 steps over the maxima, each into the
// border's step of the one before.  -inf where fewer than k are finite.
__device__ float top_bound(float mine, float top, int k, Room& rm) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t* bins = rm.low;
  const bool some = mine > -INFINITY;
  float low = some ? mine : INFINITY, bound = -INFINITY, high = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  __syncthreads();
  if (lane == 0) rm.warp[warp] = (uint64_t)__float_as_uint(low);
  if (__syncthreads_count(some) < k) return -INFINITY;
#pragma unroll
  for (int w = 0; w < WARPS; w++) low = fminf(low, __uint_as_float((uint32_t)rm.warp[w]));
  bound = low;  // all of them reach it
  int above = 0;  // maxima over `high`
  for (int round = 0; round < 4; round++) {
    const float width = (high - low) * (1.0f / 256.0f), inv = 1.0f / width;
    if (!(width > 0.0f) || !(width < INFINITY) || !(inv < INFINITY)) break;
    if (tid < 256) bins[tid] = 0;
    __syncthreads();
    if (some && mine >= low && mine <= high) atomicAdd(&bins[min(255, (int)((high - mine) * inv))], 1u);
    __syncthreads();
    if (warp == 0) {
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) sum += c[j] = bins[lane * 8 + j];
      uint32_t run = (uint32_t)warp_scan(sum) - sum, before = 0;
      int step = 255;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (step == 255 && above + (int)(run + c[j]) >= k) {
          step = lane * 8 + j;
          before = run;
        }
        run += c[j];
      }
      const int first = __reduce_min_sync(0xffffffffu, step);
      if (step == first) rm.step = first, rm.before = (int)before;
    }
    __syncthreads();
    const int step = rm.step, before = rm.before;
    const float edge = high - ((float)step + 1.01f) * width;
    const int reach = __syncthreads_count(some && mine >= edge);
    if (reach < k) break;  // the steps are finer than the values' rounding
    bound = fmaxf(bound, edge);
    if (reach <= k + k / 4 + 16) break;
    above += before;
    high -= (float)step * width;
    low = edge;
  }
  __syncthreads();
  return bound;
}

// Adds a token to the cluster's list in rank 0 (dropped when it is full).
__device__ __forceinline__ void push(Room* to, uint64_t entry) {
  const int at = atomicAdd(&to->count, 1);
  if (at < LIST) to->all[at] = entry;
}

// Ranks the n <= NT entries of rm.all, their weights in rm.list: every entry
// is compared with all others, the NT threads sharing an entry's comparisons
// in groups of `parts` neighbouring lanes.  That takes n^2 / NT steps without a
// barrier, where sorting takes some log(n)^2 / 2 with one each.
struct Ranking {
  int parts;      // threads per entry
  int entry;      // of this thread's group
  bool mine;      // the entry exists
};
__device__ __forceinline__ Ranking ranking_of(int n) {
  Ranking r;
  r.parts = 1;
  while (r.parts < 32 && r.parts * 2 * n <= NT) r.parts *= 2;
  r.entry = threadIdx.x / r.parts;
  r.mine = r.entry < n;
  return r;
}
// The number and the weights of the entries for which `before(other)` holds.
template <typename Before>
__device__ __forceinline__ void count_before(const Ranking& r, int n, const Room& rm, Before before,
                                             int* number, uint64_t* mass) {
  int c = 0;
  uint64_t m = 0;
  if (r.mine)
#pragma unroll 4
    for (int j = threadIdx.x % r.parts; j < n; j += r.parts) {
      const uint64_t other = rm.all[j], w = rm.list[j];
      const bool b = before(other);
      c += b ? 1 : 0;
      m += b ? w : 0;
    }
  for (int o = 1; o < r.parts; o <<= 1) {
    c += __shfl_xor_sync(0xffffffffu, c, o);
    m += __shfl_xor_sync(0xffffffffu, m, o);
  }
  *number = c;
  *mass = m;
}

// Rank 0: cuts the list of n entries by all filters and draws (n <= NT).
__device__ void draw_from_short_list(int n, const Args& a, int64_t row, const Filters& flt,
                                     const Scale& sc, Room& rm) {
  const int tid = threadIdx.x;
  rm.list[tid] = tid < n ? weight_of(entry_value(rm.all[tid]), sc) : 0;
  __syncthreads();
  const Ranking r = ranking_of(n);
  const uint64_t e = r.mine ? rm.all[r.entry] : 0, w = r.mine ? rm.list[r.entry] : 0;
  const float x = entry_value(e);
  const bool first = r.mine && tid % r.parts == 0;  // speaks for its entry
  int rank;
  uint64_t before, all;
  count_before(r, n, rm, [&](uint64_t other) { return other > e; }, &rank, &before);
  const int k = flt.top_k > 0 && flt.top_k < n ? (int)flt.top_k : n;
  room_scan(first && rank < k ? w : 0, rm, &all);
  const uint64_t aim = flt.top_p < 1.0f ? share_aim(flt.top_p, all) : all;
  const bool keep = first && rank < k && (before < aim || rank == 0) && x >= least_logit(flt, sc.max);
  room_scan(keep ? w : 0, rm, &all);  // its barriers also end the reading of the weights
  if (first && !keep) rm.list[r.entry] = 0;
  __syncthreads();
  const uint64_t to = draw_aim(flt.uniform, all);
  int unused;
  uint64_t run;  // indexes are stored inverted
  count_before(r, n, rm, [&](uint64_t other) { return (uint32_t)other > (uint32_t)e; }, &unused, &run);
  if (keep && run < to && to <= run + w) answer(a, row, entry_index(e), x, flt, sc, all);
}

// The same for any list, by sorting.
__device__ void draw_from_list(int n, const Args& a, int64_t row, const Filters& flt,
                               const Scale& sc, Room& rm) {
  if (n <= NT) return draw_from_short_list(n, a, row, flt, sc, rm);
  constexpr int PER = LIST / NT;
  const int tid = threadIdx.x;
  const int size = pad_list(rm.all, n);
  sort_descending(rm.all, size);
  if (flt.top_k > 0 && flt.top_k < n) n = (int)flt.top_k;
  uint64_t w[PER], mine = 0, all;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int i = tid * PER + j;
    w[j] = i < n ? weight_of(entry_value(rm.all[i]), sc) : 0;
    mine += w[j];
  }
  uint64_t run = room_scan(mine, rm, &all) - mine;
  const uint64_t aim = flt.top_p < 1.0f ? share_aim(flt.top_p, all) : all;
  const float least = least_logit(flt, sc.max);
  if (tid == 0) rm.keep = 0;
  __syncthreads();
  int keep = 0;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int i = tid * PER + j;
    if (i < n && (run < aim || i == 0) && entry_value(rm.all[i]) >= least) keep++;
    run += w[j];
  }
  keep = __reduce_add_sync(0xffffffffu, keep);
  if ((tid & 31) == 0 && keep) atomicAdd(&rm.keep, keep);
  __syncthreads();
  n = rm.keep;  // what is kept is a prefix of the ranking
  __syncthreads();
  // by index, ascending: entries (~index, logit bits), descending
  for (int i = tid; i < n; i += NT) {
    const uint64_t e = rm.all[i];
    rm.all[i] = (e << 32) | (e >> 32);
  }
  sort_descending(rm.all, pad_list(rm.all, n));
  mine = 0;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int i = tid * PER + j;
    w[j] = i < n ? weight_of(value_of((uint32_t)rm.all[i]), sc) : 0;
    mine += w[j];
  }
  run = room_scan(mine, rm, &all) - mine;
  const uint64_t to = draw_aim(flt.uniform, all);
#pragma unroll
  for (int j = 0; j < PER; j++) {
    if (run < to && to <= run + w[j]) {
      const uint64_t e = rm.all[tid * PER + j];
      answer(a, row, (int)(0xffffffffu - (uint32_t)(e >> 32)), value_of((uint32_t)e), flt, sc, all);
    }
    run += w[j];
  }
}

// Sums over the blocks of a cluster of a value that each has in rm.total.
__device__ __forceinline__ uint64_t cluster_total(cg::cluster_group& cluster, Room& rm,
                                                  unsigned blocks) {
  uint64_t all = 0;
#pragma unroll
  for (unsigned b = 0; b < 8; b++)
    if (b < blocks) all += cluster.map_shared_rank(&rm, b)->total;
  return all;
}

// What a cut adds up: tokens or weights.
struct Tokens {
  __device__ __forceinline__ uint64_t operator()(float x) const { return x > -INFINITY; }
  __device__ __forceinline__ void both(float x, float y, uint64_t (&w)[2]) const {
    w[0] = x > -INFINITY;
    w[1] = y > -INFINITY;
  }
};
struct Weights {
  Scale sc;
  __device__ __forceinline__ uint64_t operator()(float x) const { return weight_of(x, sc); }
  __device__ __forceinline__ void both(float x, float y, uint64_t (&w)[2]) const {
    if (sc.narrow) {
      // rounded as add_weights does; the integers lie in the sums' low bits
      const uint64_t p = powers_of(x, y, sc), c = add2(p, twice(96.0f));
      const uint64_t r = fma2(add2(c, twice(-96.0f)), twice(-1.0f), p);
      const float2 cc = unpk(c), ff = unpk(add2(r, twice(0x1.8p-12f)));
      const int base = __float_as_int(96.0f), fine = __float_as_int(0x1.8p-12f);
      w[0] = ((uint64_t)(__float_as_int(cc.x) - base) << 18) + (int64_t)(__float_as_int(ff.x) - fine);
      w[1] = ((uint64_t)(__float_as_int(cc.y) - base) << 18) + (int64_t)(__float_as_int(ff.y) - fine);
    } else {
      w[0] = weight_of(x, sc);
      w[1] = weight_of(y, sc);
    }
  }
};

// Lowers `border` to the shortest prefix of the ranking of the tokens it keeps
// whose units reach `to` (at least 1, at most their sum); tokens under `least`
// are known to lie behind it.  `per` histogram steps per unit of the logit.
// False (in every block of the cluster) when the border's step holds more
// tokens than a list or `least` was not low enough.
template <typename T, typename Unit>
__device__ bool cluster_cut(cg::cluster_group& cluster, Room& rm, unsigned rank, unsigned blocks,
                            const Slice<T>& slice, int first, float max, float per, float least,
                            Border& border, const Unit unit, uint64_t to) {
  constexpr bool COUNT = std::is_same_v<Unit, Tokens>;
  constexpr int PER = LIST / NT;
  const int tid = threadIdx.x;
  // steps of 1 / per of the logit, falling; the last takes all below
  auto step_of = [&](float x) {
    const float t = (max - x) * per;
    return t > 0.0f ? (int)fminf(t, (float)(LIST - 1)) : 0;
  };
  least = fmaxf(least, border.value);
  // (since the caller's last cluster.sync nobody reads or writes this block's
  // histogram or list)
  for (int i = tid; i < LIST; i += NT) rm.low[i] = rm.high[i] = 0;
  __syncthreads();
  const bool every = border.value == -INFINITY && least > -INFINITY;
  auto add = [&](float x, uint64_t w) {
    // `least` is finite for weights: steps need no bounds but the rounding's
    const int step = COUNT ? step_of(x) : min((int)((max - x) * per), LIST - 1);
    if (COUNT) {
      atomicAdd(&rm.low[step], (uint32_t)w);
      return;
    }
    const uint32_t lo = (uint32_t)w, old = atomicAdd(&rm.low[step], lo);
    const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
    if (hi != 0) atomicAdd(&rm.high[step], hi);
  };
  slice.each_piece(least, [&](int i, const float (&v)[Slice<T>::N]) {
#pragma unroll
    for (int k = 0; k < Slice<T>::N; k += 2) {
      const bool a = v[k] >= least && (every || kept(border, v[k], first + i + k));
      const bool b = v[k + 1] >= least && (every || kept(border, v[k + 1], first + i + k + 1));
      if (a || b) {
        uint64_t w[2];
        unit.both(v[k], v[k + 1], w);
        if (a) add(v[k], w[0]);
        if (b) add(v[k + 1], w[1]);
      }
    }
  });
  cluster.sync();
  static_assert(PER == 2, "two steps per thread");
  uint64_t bins[PER] = {0, 0}, all;
#pragma unroll
  for (unsigned b = 0; b < 8; b++)
    if (b < blocks) {
      const Room* r = cluster.map_shared_rank(&rm, b);
      const uint2 lo = *reinterpret_cast<const uint2*>(&r->low[2 * tid]);
      bins[0] += lo.x;
      bins[1] += lo.y;
      if (!COUNT) {
        const uint2 hi = *reinterpret_cast<const uint2*>(&r->high[2 * tid]);
        bins[0] += (uint64_t)hi.x << 32;
        bins[1] += (uint64_t)hi.y << 32;
      }
    }
  uint64_t run = room_scan(bins[0] + bins[1], rm, &all) - bins[0] - bins[1];
  if (tid == 0) rm.count = 0, rm.found[0] = LIST;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; j++) {
    if (run < to && to <= run + bins[j]) {
      rm.found[0] = (uint64_t)(tid * PER + j);
      rm.found[1] = to - run;
    }
    run += bins[j];
  }
  cluster.sync();  // every block is done with the histograms: the list takes their place
  const int step = (int)rm.found[0];
  const uint64_t rest = rm.found[1];
  if (step >= LIST) return false;
  Room* head = cluster.map_shared_rank(&rm, 0);
  // below the step's lower edge whatever step_of rounds
  const float from = step == LIST - 1 ? least
                                      : fmaxf(least, max - ((float)step + 1.01f) / per - fabsf(max) * 1e-6f);
  slice.each_from(from, [&](int i, float x) {
    if (x >= from && step_of(x) == step && kept(border, x, first + i)) push(head, entry_of(x, first + i));
  });
  cluster.sync();
  if (rank == 0) {
    const int n = rm.count;
    if (tid == 0) rm.border = Border{NAN, 0};
    __syncthreads();
    if (n <= NT) {
      rm.list[tid] = tid < n ? unit(entry_value(rm.all[tid])) : 0;
      __syncthreads();
      const Ranking r = ranking_of(n);
      const uint64_t e = r.mine ? rm.all[r.entry] : 0;
      int unused;
      uint64_t before;
      count_before(r, n, rm, [&](uint64_t other) { return other > e; }, &unused, &before);
      if (r.mine && before < rest && rest <= before + rm.list[r.entry])
        rm.border = Border{entry_value(e), entry_index(e)};
    } else if (n <= LIST) {
      sort_descending(rm.all, pad_list(rm.all, n));
      uint64_t w[PER], mine = 0;
#pragma unroll
      for (int j = 0; j < PER; j++) {
        const int i = tid * PER + j;
        w[j] = i < n ? unit(entry_value(rm.all[i])) : 0;
        mine += w[j];
      }
      run = room_scan(mine, rm, &all) - mine;
#pragma unroll
      for (int j = 0; j < PER; j++) {
        if (run < rest && rest <= run + w[j]) {
          const uint64_t e = rm.all[tid * PER + j];
          rm.border = Border{entry_value(e), entry_index(e)};
        }
        run += w[j];
      }
    }
  }
  cluster.sync();
  const Border found = head->border;
  if (!(found.value == found.value)) return false;
  border = found;
  return true;
}

// The block's weights that `border` keeps: their sum, the sums per warp in
// rm.warp; warp w takes the tokens from span_of(w) to span_of(w + 1).
template <typename T>
__device__ __forceinline__ int span_of(const Slice<T>& s, int w) {
  if (w == 0) return 0;
  if (w >= WARPS) return s.n;
  return s.head + min(s.pieces, w * ((s.pieces + WARPS - 1) / WARPS)) * Slice<T>::N;
}
template <typename T>
__device__ uint64_t block_weights(const Slice<T>& s, int first, const Border& border,
                                  const Scale& sc, Room& rm) {
  constexpr int N = Slice<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (s.pieces + WARPS - 1) / WARPS;
  const int p0 = min(s.pieces, warp * each), p1 = min(s.pieces, p0 + each);
  auto weight_at = [&](int i) -> uint64_t {
    const float v = to_f32<T>(s.x[i]);
    return kept(border, v, first + i) ? weight_of(v, sc) : 0;
  };
  uint64_t sum = 0;
  if (sc.narrow) {
    const bool every = border.value == -INFINITY;
    Sum64 part{0, 0};
    int in = 0;
    for (int p = p0 + lane; p < p1; p += 32) {
      union { uint4 v; T x[N]; } u;
      u.v = *reinterpret_cast<const uint4*>(s.x + s.head + p * N);
      float v[N], top = -INFINITY;
#pragma unroll
      for (int k = 0; k < N; k++) {
        v[k] = to_f32<T>(u.x[k]);
        top = fmaxf(top, v[k]);
      }
      if (!every) {
        if (!(top >= border.value)) continue;
        const int i = first + s.head + p * N;
#pragma unroll
        for (int k = 0; k < N; k++) v[k] = kept(border, v[k], i + k) ? v[k] : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < N; k += 2) add_weights(part, v[k], v[k + 1], sc);
      if ((in += N) == 64) {
        sum += flush(part);
        in = 0;
      }
    }
    sum += flush(part);
  } else {
    for (int p = p0 + lane; p < p1; p += 32) {
      union { uint4 v; T x[N]; } u;
      u.v = *reinterpret_cast<const uint4*>(s.x + s.head + p * N);
      float top = to_f32<T>(u.x[0]);
#pragma unroll
      for (int k = 1; k < N; k++) top = fmaxf(top, to_f32<T>(u.x[k]));
      if (top >= border.value)
#pragma unroll
        for (int k = 0; k < N; k++) {
          const float v = to_f32<T>(u.x[k]);
          if (kept(border, v, first + s.head + p * N + k)) sum += weight_of(v, sc);
        }
    }
  }
  if (warp == 0 && lane < s.head) sum += weight_at(lane);
  const int tail = s.head + s.pieces * N;
  if (warp == WARPS - 1 && tail + lane < s.n) sum += weight_at(tail + lane);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) rm.warp[warp] = sum;
  __syncthreads();
  uint64_t here = 0;
#pragma unroll
  for (int w = 0; w < WARPS; w++) here += rm.warp[w];
  return here;
}

template <typename T>
__global__ void __launch_bounds__(NT, 2) sample_cluster_kernel(const T* __restrict__ logits, Args a) {
  extern __shared__ __align__(16) uint8_t slice_smem[];
  __shared__ Room rm;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned rank = cluster.block_rank(), blocks = cluster.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / blocks;
  const T* x = logits + row * a.row_stride;
  const Filters flt = filters_of(a, row);

  // this block's slice, and its maximum while it arrives
  const int first = min(a.n, (int)rank * a.slice);
  Slice<T> slice;
  slice.n = min(a.n, first + a.slice) - first;
  const uintptr_t at = reinterpret_cast<uintptr_t>(x + first);
  const int off = (int)(at & 15);
  slice.head = min(slice.n, off == 0 ? 0 : (16 - off) / (int)sizeof(T));
  slice.pieces = (slice.n - slice.head) / Slice<T>::N;
  T* mine = reinterpret_cast<T*>(slice_smem + off);
  slice.x = mine;
  const uint32_t dst = (uint32_t)__cvta_generic_to_shared(mine + slice.head);
  const T* src = x + first + slice.head;
  constexpr int PARTS = 4;
  const int part = (slice.pieces + PARTS - 1) / PARTS;
#pragma unroll
  for (int g = 0; g < PARTS; g++) {
    const int end = min(slice.pieces, (g + 1) * part);
    for (int p = g * part + tid; p < end; p += NT) cp16(dst + 16u * p, src + p * Slice<T>::N);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  float top = -INFINITY;
  {
    const int tail = slice.head + slice.pieces * Slice<T>::N;
    if (tid < slice.head) {
      mine[tid] = x[first + tid];
      top = to_f32<T>(mine[tid]);
    } else if (tid >= 32 && tail + tid - 32 < slice.n) {
      mine[tail + tid - 32] = x[first + tail + tid - 32];
      top = to_f32<T>(mine[tail + tid - 32]);
    }
    top = fmaxf(top, -INFINITY);  // NaN is no maximum
  }
#pragma unroll
  for (int g = 0; g < PARTS; g++) {
    if (g == 0) asm volatile("cp.async.wait_group 3;" ::: "memory");
    if (g == 1) asm volatile("cp.async.wait_group 2;" ::: "memory");
    if (g == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    if (g == 3) asm volatile("cp.async.wait_group 0;" ::: "memory");
    const int end = min(slice.pieces, (g + 1) * part);
    for (int p = g * part + tid; p < end; p += NT) {  // the pieces this thread copied
      union { uint4 v; T x[Slice<T>::N]; } u;
      u.v = *reinterpret_cast<const uint4*>(mine + slice.head + p * Slice<T>::N);
      top = fmaxf(top, piece_max<T>(u.v));
    }
  }
  const float thread_top = top;
  top = warp_max(top);
  if (lane == 0) rm.warp[warp] = (uint64_t)__float_as_uint(top);
  if (tid == 0) rm.count = 0;
  __syncthreads();
  float block_top = -INFINITY;
#pragma unroll
  for (int w = 0; w < WARPS; w++) block_top = fmaxf(block_top, __uint_as_float((uint32_t)rm.warp[w]));
  if (tid == 0) rm.top = block_top;
  cluster.sync();
  float max = -INFINITY;
  for (unsigned b = 0; b < blocks; b++) max = fmaxf(max, cluster.map_shared_rank(&rm, b)->top);

  // no block leaves while another may read or write its shared memory
  if (max == -INFINITY) {
    if (rank == 0 && tid == 0) {
      a.ids[row] = -1;
      if (a.logprobs != nullptr) a.logprobs[row] = -INFINITY;
    }
    cluster.sync();
    return;
  }
  if (!(flt.temperature > 0x1p-100f)) {  // the first of the largest
    int best = INT32_MAX;
    if (block_top == max)
      slice.each([&](int i, float v) { if (v == max) best = min(best, first + i); });
    best = __reduce_min_sync(0xffffffffu, best);
    __syncthreads();
    if (lane == 0) rm.warp[warp] = (uint64_t)best;
    cluster.sync();
    if (rank == 0 && warp == 0) {
      for (unsigned i = lane; i < blocks * WARPS; i += 32)
        best = min(best, (int)cluster.map_shared_rank(&rm, i / WARPS)->warp[i % WARPS]);
      best = __reduce_min_sync(0xffffffffu, best);
      if (lane == 0) {
        a.ids[row] = best;
        if (a.logprobs != nullptr) a.logprobs[row] = 0.0f;
      }
    }
    cluster.sync();
    return;
  }
  const Scale sc = scale_of(max, flt.per);
  const bool top_k = flt.top_k > 0 && flt.top_k < a.n;

  // ---- a list
  bool listed = a.n <= LIST;
  float bound = -INFINITY;
  if (!listed && top_k && flt.top_k <= NT / 2) {
    // What k / blocks tokens of every slice reach, k tokens of the row reach;
    // where a slice has fewer, what k tokens of one slice reach.
    bound = top_bound(thread_top, block_top, ((int)flt.top_k + (int)blocks - 1) / (int)blocks, rm);
    auto exchange = [&](bool least) {
      if (tid == 0) rm.bound = bound;
      cluster.sync();
#pragma unroll
      for (unsigned b = 0; b < 8; b++)
        if (b < blocks) {
          const float other = cluster.map_shared_rank(&rm, b)->bound;
          bound = least ? fminf(bound, other) : fmaxf(bound, other);
        }
    };
    exchange(true);
    if (blocks > 1 && bound == -INFINITY) {
      bound = top_bound(thread_top, block_top, (int)flt.top_k, rm);
      cluster.sync();  // the first bounds are read
      exchange(false);
    }
    listed = true;
  }
  if (listed) {
    Room* head = cluster.map_shared_rank(&rm, 0);
    slice.each_from(bound, [&](int i, float v) {
      if (v > -INFINITY && v >= bound) push(head, entry_of(v, first + i));
    });
    cluster.sync();
    const int n = head->count;
    if (n <= LIST) {
      // only rank 0 has work left, in its own memory; it waits until the others
      // have read its count
      cluster.sync();
      if (rank == 0) draw_from_list(n, a, row, flt, sc, rm);
      return;
    }
  }

  // ---- cuts from histograms
  Border border{-INFINITY, -1};
  bool good = true;
  if (top_k) {
    // how many there are to rank
    int some = 0;
    slice.each([&](int, float v) { some += v > -INFINITY; });
    some = __reduce_add_sync(0xffffffffu, some);
    __syncthreads();
    if (lane == 0) rm.warp[warp] = (uint64_t)some;
    __syncthreads();
    if (tid == 0) {
      uint64_t t = 0;
      for (int w = 0; w < WARPS; w++) t += rm.warp[w];
      rm.total = t;
    }
    cluster.sync();
    if ((uint64_t)flt.top_k < cluster_total(cluster, rm, blocks))
      good = cluster_cut<T>(cluster, rm, rank, blocks, slice, first, max, kTopSteps, -INFINITY, border,
                            Tokens{}, (uint64_t)flt.top_k);
    else
      cluster.sync();  // the totals are read
  }
  if (good && flt.top_p < 1.0f) {
    const uint64_t here = block_weights(slice, first, border, sc, rm);
    if (tid == 0) rm.total = here;
    cluster.sync();
    const uint64_t all = cluster_total(cluster, rm, blocks);
    const uint64_t to = share_aim(flt.top_p, all);
    // The tokens from the border down weigh more than the mass that may go, so
    // the border's weight is over its share of a token; a little less, for the
    // rounding of weights (half a unit) and logits.
    const double gone = (double)(all - to) / (double)a.n;
    float least = -INFINITY;
    if (max < INFINITY)
      least = (float)((double)max + (double)flt.temperature * log(fmax(gone - 0.51, 0.49) * (0.999 * 0x1p-35))) -
              fabsf(max) * 1e-6f;
    // all steps between the maximum and `least`
    const float per = fminf((float)(LIST - 1) / fmaxf(max - least, 0.0f), 1e30f);
    good = cluster_cut<T>(cluster, rm, rank, blocks, slice, first, max, per, least, border,
                          Weights{sc}, to);
  }
  if (!good) {
    cluster.sync();  // the border is read: the others may leave
    if (rank == 0) sample_row<T>(x, a, row, flt, sc, rm.radix);
    return;
  }
  const float least = least_logit(flt, sc.max);
  if (least > border.value) border = Border{least, INT32_MAX};

  // ---- the draw: running sums by block, warp, lane
  const uint64_t here = block_weights(slice, first, border, sc, rm);
  if (tid == 0) rm.total = here;
  cluster.sync();
  const uint64_t all = cluster_total(cluster, rm, blocks);
  uint64_t before = 0;
  for (unsigned b = 0; b < rank; b++) before += cluster.map_shared_rank(&rm, b)->total;
  cluster.sync();  // nothing of another block is read any more
  const uint64_t to = draw_aim(flt.uniform, all);
  if (before < to && to <= before + here) {
    uint64_t rest = to - before;
    int w = 0;
    while (w < WARPS - 1 && rest > rm.warp[w]) rest -= rm.warp[w++];
    __syncthreads();
    auto weight_at = [&](int i) -> uint64_t {
      const float v = to_f32<T>(slice.x[i]);
      return kept(border, v, first + i) ? weight_of(v, sc) : 0;
    };
    const int s0 = span_of(slice, w), s1 = span_of(slice, w + 1);
    const int each = (s1 - s0 + NT - 1) / NT;
    const int t0 = min(s1, s0 + tid * each), t1 = min(s1, t0 + each);
    uint64_t mine_sum = 0, unused;
    for (int i = t0; i < t1; i++) mine_sum += weight_at(i);
    uint64_t run = room_scan(mine_sum, rm, &unused) - mine_sum;
    if (run < rest && rest <= run + mine_sum) {
      int i = t0;
      for (; i < t1; i++) {
        run += weight_at(i);
        if (run >= rest) break;
      }
      answer(a, row, first + i, to_f32<T>(slice.x[i]), flt, sc, all);
    }
  }
}

// Vocabularies beyond the shared memory of a cluster.
template <typename T>
__global__ void __launch_bounds__(NT) sample_kernel(const T* __restrict__ logits, Args a) {
  __shared__ Shared sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * a.row_stride;
  const Filters flt = filters_of(a, row);
  // the largest logit, of equal ones the first
  uint64_t best = 0;
  for (int i = tid; i < n; i += NT)
    best = max(best, ((uint64_t)key_of(to_f32<T>(x[i])) << 32) | (0xffffffffu - (uint32_t)i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) sm.warp[warp] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; w++) best = max(best, sm.warp[w]);
  const uint32_t best_key = (uint32_t)(best >> 32);
  const bool none = best_key <= kKeyMinusInf;
  if (none || !(flt.temperature > 0x1p-100f)) {
    if (tid == 0) {
      a.ids[row] = none ? -1 : (int64_t)(0xffffffffu - (uint32_t)best);
      if (a.logprobs != nullptr) a.logprobs[row] = none ? -INFINITY : 0.0f;
    }
    return;
  }
  sample_row<T>(x, a, row, flt, scale_of(value_of(best_key), flt.per), sm);
}

// Clusters of as few thread blocks as hold a row (two of them per SM), and of
// up to 8 while that leaves SMs idle and a slice keeps 4,096 logits.
template <typename T>
cudaError_t launch(const T* logits, Args a, int64_t rows, cudaStream_t stream) {
  constexpr int kSliceBytes = 96 * 1024;
  int blocks = 1;
  auto slice_of = [&](int b) { return ((a.n + b - 1) / b + 15) / 16 * 16; };
  while (blocks < 8 && (int64_t)slice_of(blocks) * (int)sizeof(T) > kSliceBytes) blocks *= 2;
  if ((int64_t)slice_of(blocks) * (int)sizeof(T) > 208 * 1024 || rows * blocks > INT32_MAX) {
    sample_kernel<T><<<(unsigned)rows, NT, 0, stream>>>(logits, a);
    count_launch();
    return cudaGetLastError();
  }
  while (blocks < 8 && rows * blocks * 2 <= 2 * sm_count() && slice_of(2 * blocks) >= 4096) blocks *= 2;
  a.slice = slice_of(blocks);
  const int smem = a.slice * (int)sizeof(T) + 32;
  cudaError_t st = cudaFuncSetAttribute(sample_cluster_kernel<T>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, 209 * 1024);
  if (st != cudaSuccess) return st;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * blocks));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  st = cudaLaunchKernelEx(&cfg, sample_cluster_kernel<T>, logits, a);
  count_launch();
  return st;
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
    using paged::aligned_to;
    if (!aligned_to(size, logits) || !aligned_to(8, ids, s->top_k) ||
        !aligned_to(4, uniform, logprobs, s->temperature, s->top_p, s->min_p))
      return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_INVALID_BUFFER, op,
                       "logits and the rows' values must be aligned to their elements");
    auto st = static_cast<cudaStream_t>(stream);
    const Args a{uniform, s->temperature, s->top_k, s->top_p, s->min_p, ids, logprobs,
                 s->row_stride, (int)s->vocabulary, 0};
    cudaError_t status;
    if (s->dtype == ET_B200_DTYPE_F32)
      status = launch(static_cast<const float*>(logits), a, s->rows, st);
    else if (s->dtype == ET_B200_DTYPE_F16)
      status = launch(static_cast<const __half*>(logits), a, s->rows, st);
    else
      status = launch(static_cast<const __nv_bfloat16*>(logits), a, s->rows, st);
    if (status != cudaSuccess) return cuda_error(e, status, op);
  }
  if (e) memset(e, 0, sizeof(*e));
  return 0;
}
