// Verification of drafted tokens (et_b200_verify_v1).
//
// Proposal x of row r is accepted if u q(x) < p(x); the first row that is not
// accepted draws from max(p - q, 0), the last row from p.  Only that row of p and q is
// read in full, so at most 8 bytes a token of the vocabulary and request.  A cluster
// of thread blocks takes a request: each finds the row (a value of p and q per
// proposal), sums its share of segments of 1,024 tokens in f64, a warp a segment; all
// segments' sums come together in every block, whose scan finds the segment of the
// draw, and one warp walks it.  Segments, and with them all orders of summation, depend
// on the vocabulary alone.
// 64 requests of 5 rows of 128,259 (66 MB): 19.3 us on the device, other inputs each time, 3.4 TB/s;
// without draft distributions (33 MB) 17.5 us.  A thread block an SM holds two segments a warp,
// so the start, the cluster's barriers (3.5 of the 13 cycles between two instructions of a warp)
// and the conversions to f64 stand beside the reading, and take as long for half the bytes.  One
// request of 32,768: 9.5 us, the latency of those steps.
#include <math.h>

#include <cooperative_groups.h>

#include <type_traits>

#include "paged.cuh"

namespace etb {
namespace {

namespace cg = cooperative_groups;
using paged::aligned_to;
using paged::report;

constexpr int NT = 512, WARPS = NT / 32;
constexpr int SEG = 1024;  // tokens of a segment
constexpr int64_t kMostVocabulary = 1 << 22;

struct VerifyArgs {
  const float* target;
  const float* draft;
  const int64_t* offsets;
  const int64_t* drafts;
  const float* accept;
  const float* draw;
  int64_t* ids;
  int64_t* accepted;
  int* status;
  int64_t tokens, target_stride, draft_stride;
  int n, segs;  // tokens of the vocabulary, its segments
};

// A probability as the rules read it: NaN and negative ones are 0, the largest is 1.
__device__ __forceinline__ float probability(float p) { return p > 0.0f ? fminf(p, 1.0f) : 0.0f; }
// max(p - q, 0), in 32 bits: a conversion to 64 costs four times a difference (64 requests 28 us
// with two, 22 with one).  Each is off by at most 2^-24 of itself, a draw's border by 2^-24 of the
// running sum before it.
__device__ __forceinline__ double weight(float p, float q) {
  return (double)fmaxf(probability(p) - probability(q), 0.0f);
}

// The weights that the request's token is drawn from.
struct Rest {
  const float* p;
  const float* q;  // or null
  int without;     // a token of weight 0 (a proposal made without chance), or -1
};

__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The weights of segment s, added up by a warp: whole lines whatever the rows' alignment
// (an odd vocabulary has rows at every multiple of 4 bytes), 16 loads of a lane and row out
// together.
__device__ double segment(const VerifyArgs& a, const Rest& rest, int s) {
  constexpr int J = 16;
  const int lane = threadIdx.x & 31;
  double sum = 0.0;
#pragma unroll 1
  for (int i0 = s * SEG + lane; i0 < (s + 1) * SEG && i0 - lane < a.n; i0 += 32 * J) {
    float x[J], y[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
      const int i = i0 + 32 * j;
      x[j] = i < a.n && i != rest.without ? __ldcs(rest.p + i) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < J; j++) {
      const int i = i0 + 32 * j;
      y[j] = rest.q != nullptr && i < a.n ? __ldcs(rest.q + i) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < J; j++) sum += weight(x[j], y[j]);
  }
  return warp_total(sum);
}

__global__ void __launch_bounds__(NT, 2) verify_kernel(VerifyArgs a) {
  extern __shared__ double sums[];  // [segs]: this block's share at its place, then all
  __shared__ double warp_s[WARPS];
  __shared__ int stop_s, found_s;
  __shared__ double before_s;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned rank = cluster.block_rank(), blocks = cluster.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / blocks;
  const int64_t o0 = a.offsets[b], o1 = a.offsets[b + 1];
  const int64_t first = min(max(o0, (int64_t)0), a.tokens), end = min(max(o1, first), a.tokens);
  if ((first != o0 || end != o1) && rank == 0 && tid == 0) report(a.status, ET_B200_PAGED_BAD_OFFSET);
  const int n = (int)(end - first);
  if (n == 0) {
    if (rank == 0 && tid == 0) a.accepted[b] = 0;
    return;
  }
  auto sound = [&](int64_t x) { return x >= 0 && x < a.n; };

  // ---- the first row whose proposal is not accepted, or the last row
  if (tid == 0) stop_s = n - 1;
  __syncthreads();
  int mine = n - 1;
  for (int i = tid; i < mine; i += NT) {
    const int64_t r = first + i, x = a.drafts[r];
    bool good = false;
    if (sound(x)) {
      const double p = probability(a.target[r * a.target_stride + x]);
      const double q = a.draft != nullptr ? probability(a.draft[r * a.draft_stride + x]) : 1.0f;
      good = (double)a.accept[r] * q < p;
    }
    if (!good) mine = i;
  }
  mine = __reduce_min_sync(0xffffffffu, mine);
  if (lane == 0 && mine < n - 1) atomicMin(&stop_s, mine);
  __syncthreads();
  const int stop = stop_s;
  const int64_t row = first + stop;
  Rest rest{a.target + row * a.target_stride, nullptr, -1};
  if (stop < n - 1 && sound(a.drafts[row])) {
    if (a.draft != nullptr) rest.q = a.draft + row * a.draft_stride;
    else rest.without = (int)a.drafts[row];
  }

  // ---- the draw
  const int each = (a.segs + (int)blocks - 1) / (int)blocks;
  const int s0 = min(a.segs, (int)rank * each), s1 = min(a.segs, s0 + each);
  int64_t id = -1;
  for (int attempt = 0; attempt < 2; attempt++) {
    for (int s = s0 + warp; s < s1; s += WARPS) {
      const double sum = segment(a, rest, s);
      if (lane == 0) sums[s] = sum;
    }
    cluster.sync();
    for (int s = tid; s < a.segs; s += NT) {
      const unsigned from = (unsigned)(s / each);
      if (from != rank) sums[s] = cluster.map_shared_rank(sums, from)[s];
    }
    // every block waits for this before it leaves or begins again; the first draws meanwhile
    cluster.barrier_arrive();
    // the sums that a thread scans are neighbours, gathered by others once they are more than NT
    __syncthreads();
    // running sums of `per` segments a thread
    const int per = (a.segs + NT - 1) / NT, t0 = min(a.segs, tid * per), t1 = min(a.segs, t0 + per);
    double own = 0.0;
    for (int s = t0; s < t1; s++) own += sums[s];
    double incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_s[warp] = incl;
    if (tid == 0) found_s = a.segs;
    __syncthreads();
    double before = 0.0, total = 0.0;
    for (int w = 0; w < WARPS; w++) {
      if (w < warp) before += warp_s[w];
      total += warp_s[w];
    }
    if (total > 0.0) {
      if (rank != 0) break;
      const double u = a.draw[b], aim = u > 0.0 ? u * total : 0.0;
      // the first segment whose running sum exceeds the aim; rounding, or an aim of the
      // total, may leave none: then the last that weighs something
      double run = before + (incl - own);
      int at = a.segs, last = -1;
      for (int s = t0; s < t1; s++) {
        const double next = run + sums[s];
        if (at == a.segs && sums[s] > 0.0 && next > aim) at = s;
        if (sums[s] > 0.0) last = s;
        run = next;
      }
      const int lowest = __reduce_min_sync(0xffffffffu, at);
      if (lane == 0 && lowest < a.segs) atomicMin(&found_s, lowest);
      __syncthreads();
      int seg = found_s;
      __syncthreads();
      const bool none = seg == a.segs;
      if (none) {
        if (tid == 0) found_s = -1;
        __syncthreads();
        if (last >= 0) atomicMax(&found_s, last);
        __syncthreads();
        seg = found_s;
      } else if (t0 <= seg && seg < t1) {
        double start = before + (incl - own);
        for (int s = t0; s < seg; s++) start += sums[s];
        before_s = start;
      }
      __syncthreads();
      if (warp == 0) {
        // the tokens in order: rounds of 128, 4 neighbours a lane
        const double left = none ? INFINITY : aim - before_s;
        constexpr int J = 4;  // rounds whose loads go out together
        double go = 0.0;
        int hit = INT32_MAX, some = -1;
#pragma unroll 1
        for (int i0 = seg * SEG + 4 * lane; i0 < (seg + 1) * SEG + 4 * lane; i0 += 128 * J) {
          float x[J][4], y[J][4];
#pragma unroll
          for (int j = 0; j < J; j++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const int i = i0 + 128 * j + k;
              x[j][k] = i < a.n && i != rest.without ? rest.p[i] : 0.0f;
              y[j][k] = i < a.n && rest.q != nullptr ? rest.q[i] : 0.0f;
            }
#pragma unroll
          for (int j = 0; j < J; j++) {
            double w[4], sum = 0.0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
              w[k] = weight(x[j][k], y[j][k]);
              sum += w[k];
              if (w[k] > 0.0) some = i0 + 128 * j + k;
            }
            double upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double v = __shfl_up_sync(0xffffffffu, upto, o);
              if (lane >= o) upto += v;
            }
            double run_in = go + (upto - sum);
#pragma unroll
            for (int k = 0; k < 4; k++) {
              run_in += w[k];
              if (w[k] > 0.0 && run_in > left) hit = min(hit, i0 + 128 * j + k);
            }
            go += __shfl_sync(0xffffffffu, upto, 31);
          }
        }
        hit = __reduce_min_sync(0xffffffffu, hit);
        const int behind = __reduce_max_sync(0xffffffffu, some);
        if (lane == 0) found_s = hit != INT32_MAX ? hit : behind;
      }
      __syncthreads();
      id = found_s;
      break;
    }
    if (rest.q == nullptr && rest.without < 0) break;  // p has no mass either
    rest.q = nullptr;
    rest.without = -1;
    cluster.barrier_wait();
  }
  cluster.barrier_wait();
  if (rank != 0) return;
  for (int i = tid; i < n; i += NT)
    a.ids[first + i] = i < stop ? a.drafts[first + i] : i == stop ? id : -1;
  if (tid == 0) a.accepted[b] = stop;
}

cudaError_t launch_verify(const VerifyArgs& a, int64_t batch, cudaStream_t stream) {
  // up to 8 thread blocks a request while they fit the device at once (two an SM) and each
  // warp keeps a segment
  int blocks = 1;
  while (blocks < 8 && batch * blocks * 2 <= 2 * sm_count() && a.segs >= 2 * blocks * WARPS) blocks *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(batch * blocks));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = (size_t)a.segs * sizeof(double);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t st = cudaLaunchKernelEx(&cfg, verify_kernel, a);
  count_launch();
  return st;
}

}  // namespace
}  // namespace etb

using namespace etb;

extern "C" int32_t et_b200_verify_v1(const et_b200_verification_v1* s, const float* target,
                                     const float* draft, int64_t* ids, int64_t* accepted,
                                     void* stream, et_kernel_error* e) {
  const char* op = "verify";
  if (s == nullptr || s->struct_size < sizeof(et_b200_verification_v1))
    return set_error(e, ET_KERNEL_ERROR_VERSION_MISMATCH, ET_KERNEL_CODE_INVALID_STRUCT_SIZE, op,
                     "verification descriptor is missing or truncated");
  const int64_t most = (int64_t)1 << 31;
  if (s->batch < 0 || s->batch > (1 << 20) || s->tokens < 0 || s->tokens > (1 << 26) ||
      s->vocabulary < 1 || s->vocabulary > kMostVocabulary || s->target_stride < s->vocabulary ||
      s->target_stride > most ||
      (draft != nullptr && (s->draft_stride < s->vocabulary || s->draft_stride > most)))
    return set_error(e, ET_KERNEL_ERROR_SHAPE_MISMATCH, ET_KERNEL_CODE_INVALID_SHAPE, op,
                     "batch, tokens, vocabulary or row strides are outside their limits");
  if (s->batch > 0) {
    if (s->offsets == nullptr || s->draw_uniform == nullptr || accepted == nullptr ||
        (s->tokens > 0 && (target == nullptr || s->drafts == nullptr || s->accept_uniform == nullptr ||
                           ids == nullptr)))
      return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_NULL_ARGUMENT, op,
                       "offsets, drafts, uniform numbers, target probabilities, ids and accepted "
                       "are required");
    if (!aligned_to(8, s->offsets, s->drafts, ids, accepted) ||
        !aligned_to(4, s->accept_uniform, s->draw_uniform, s->status, target, draft))
      return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_INVALID_BUFFER, op,
                       "arrays must be aligned to their elements");
    const VerifyArgs a{target, draft, s->offsets, s->drafts, s->accept_uniform, s->draw_uniform, ids,
                 accepted, s->status, s->tokens, s->target_stride, s->draft_stride,
                 (int)s->vocabulary, (int)((s->vocabulary + SEG - 1) / SEG)};
    const cudaError_t status = launch_verify(a, s->batch, static_cast<cudaStream_t>(stream));
    if (status != cudaSuccess) return cuda_error(e, status, op);
  }
  if (e) memset(e, 0, sizeof(*e));
  return 0;
}
