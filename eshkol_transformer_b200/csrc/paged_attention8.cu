// Causal attention of new tokens over an 8-bit paged cache
// (et_b200_paged_attention8_v1): the kernels for any page size, head_dim and type.
//
// With rows k_j = a_j k^_j and v_j = b_j v^_j (k^, v^ of e4m3, a and b scales),
//   o = sum_j 2^(s_j - m) b_j v^_j / sum_j 2^(s_j - m),  s_j = log2(e) scale a_j q'.k^_j.
// The division of the work, the copies and the joining are those of
// paged_attention.cu; elements become binary16 (exact) on their way to mma.sync, so
// what is read of the cache is head_dim + 4 bytes a row.  The scales of keys multiply
// the scores; those of values move into the weights: with b_j = 2^x_j c_j, c_j below 2,
// the operand of P V is 2^(s_j - m + x_j - D) c_j, D a whole number near the largest
// s_j - m + x_j so far, so that value rows of any magnitudes stand side by side, and
// o's sums are multiplied by 2^D where a tile ends.  Queries are binary16 times 2^-e of
// their row.  At f32 queries and weights carry the residual of that rounding (22 bits), at
// f16 the queries do.  At bf16 11 bits of a query stand beside results of 8: over 64 requests to 8,192
// keys the output is 1.68e-3 off 64 bits (norms), with sums in 32 bits throughout 1.64e-3, both the
// output's own rounding; the residual would bring the two from 1.1e-3 to 2e-4 of each other for
// 2 % of single tokens' time and 21 % of drafts' (72 us to 87).
//
// Tiles of 8 or 16 rows (few8_kernel): products have the keys as rows, S^T = K Q^T and
// O^T = V^T P^T with the queries as 8 or 16 columns, and warps split the keys of a block:
// what is converted (every byte once, by the warp that uses it) is the operand of all
// rows, a step of few queries has no idle rows, and o takes dim x 8 sums.  A thread's four
// neighbouring bytes of a key are the two register pairs that a 16-deep product wants
// if dims are numbered that way, which the queries' layout follows; of V the transposed
// load brings two dims of two keys, which one byte permutation turns into two pairs of
// keys, rows of an even and an odd dim.  Weights change from a result's to an operand's
// layout by 8 x 8 transposes of the register files.
// Tiles of 64 rows (many8_kernel, chunks that the tcgen05 kernel does not take): four warps
// convert a block together to binary16 tiles first, then take 16 rows and all keys each.
//
// Single tokens are read at 5.0 TB/s (64 requests of up to 8,192 keys, 32 / 8 heads x 128,
// bf16, 697 MB: 140 us, 76 % of the copy rate); a block of 128 keys then waits for bytes
// (2.7 of the 6.7 cycles between two instructions of a warp), issue slots are 41 % busy.  Three
// thread blocks an SM with two stages each hide that best: two with three stages 177 us,
// four of 64 keys 151.  Rows of 64 dims take 69 us for 64 requests of up to 4,000 keys (174 MB, 2.5
// TB/s): the work of a key is that of 128 dims (78 us) for half its bytes, and a stage holds half as
// many (a warp waits 3.9 of its 7.8 cycles an instruction for memory, issue slots 41 %).  f32 of 128
// dims takes 87 us, its residuals' products and conversions (issue slots 51 %); 256 dims 147 us, two
// thread blocks an SM (35 %); without TMA 97 us, copies in the arithmetic warps (54 %).  Drafts (32 requests of 5 tokens, 20 rows a head, to 4,000 keys:
// 71 us, 2.5 TB/s) read the cache twice, from the L2 the second time, and are bound by
// the latency of a step's chain (conversion, products, exponentials, products; issue
// slots 41 %, tensor pipe 19 %): tiles of 8 rows 76 us, of 32 rows as two warps' halves 107.
// many8_kernel: 512 tokens over 6,000 keys, 32 / 8 heads x 128 bf16, pages of 24: 344 us,
// 140 TFLOP/s; two blocks an SM (254 registers), whose conversion, products and
// exponentials follow one another (issue slots 47 %, tensor pipe 27 %).
#include <math.h>

#include <type_traits>

#include "paged8.cuh"
#include "paged_mma.cuh"

namespace etb {
namespace {

using namespace paged;

// log2 of the largest weight: D is within 1/2 of the largest exponent, c below 2
constexpr float kShift = 13.0f;

// ROWS queries of a tile, WARPS warps, all (WK == WARPS: few8_kernel) or one of them (many8_kernel,
// tiles of binary16 in shared memory) along the BK keys of a block; PER_SM thread blocks whose
// registers have to fit an SM.
template <typename T, int DH_, int ROWS_, int WARPS_, int WK_, int BK_, int STAGES_, int PER_SM_>
struct Shape8 {
  static constexpr int DH = DH_, BM = ROWS_, WARPS = WARPS_, WK = WK_, BK = BK_, STAGES = STAGES_,
                       PER_SM = PER_SM_;
  static constexpr int NT = 32 * WARPS, KW = BK / WK;
  static constexpr bool CONVERT = WK == 1;
  static constexpr bool QLO = !std::is_same_v<T, __nv_bfloat16>, PLO = sizeof(T) == 4;
  static constexpr int ROW = DH, PIECES = ROW / 16;  // bytes of one key
  static constexpr int TILE = BK * ROW, STAGE = 2 * TILE;
  static constexpr int TILE_Q = BM * DH * 2, TILE_16 = BK * DH * 2;
  static constexpr int Q = STAGES * STAGE;
  static constexpr int CONV = Q + TILE_Q * (QLO ? 2 : 1);
  static constexpr int SCALES = CONV + (CONVERT ? 2 * TILE_16 : 0);  // [STAGES][keys, values][BK]
  static constexpr int RING = STAGES + 1;  // blocks with known pages
  static constexpr int PAGES = SCALES + STAGES * 2 * BK * 4;
  static constexpr int QMUL = PAGES + RING * (BK * 4 + 16);
  static constexpr int JOIN = QMUL + BM * 4;
  static constexpr int BARS = JOIN + WK * BM * 8;
  static constexpr int SMEM = BARS + 2 * STAGES * 8 + 16;
  static constexpr int CHUNK = ROW < 128 ? ROW : 128, CHUNKS = ROW / CHUNK;
  static constexpr int bits(int n) { return n <= 1 ? 0 : 1 + bits(n / 2); }
  static_assert(1 << bits(BM) == BM && 1 << bits(BK) == BK, "powers of two");
  static_assert(KW % 16 == 0 && DH % 64 == 0, "whole products");
  static_assert(CONVERT || WK / 2 * BM * DH * 4 <= STAGE, "the joining of warps reuses a stage");
  static_assert(PER_SM * (SMEM + 2048) <= 233472 && BARS % 8 == 0, "shared memory");
  // byte of 16-byte piece c of a row of bytes in a tile of BK rows: the swizzle of the
  // TMA boxes, 64 or 128 bytes wide
  __device__ static uint32_t at8(int row, int c) {
    if constexpr (PIECES >= 8)
      return (uint32_t)((c >> 3) * BK * 128 + row * 128 + (((c & 7) ^ (row & 7)) << 4));
    else
      return (uint32_t)(row * ROW + ((c ^ ((row >> 1) & 3)) << 4));
  }
  // the same of a row of binary16 in a tile of R rows
  template <int R>
  __device__ static uint32_t at16(int row, int c) {
    return (uint32_t)((c >> 3) * R * 128 + row * 128 + (((c & 7) ^ (row & 7)) << 4));
  }
};

// Barriers of the stages (full: 1 arrival; empty: one per arithmetic warp) and the
// block's abort word.
template <typename S>
struct Bars {
  uint32_t at;
  __device__ explicit Bars(uint32_t base) : at(base + S::BARS) {}
  __device__ uint32_t full(int st) const { return at + 8u * (uint32_t)st; }
  __device__ uint32_t empty(int st) const { return at + 8u * (uint32_t)(S::STAGES + st); }
  __device__ static int* abort_word(uint8_t* smem) {
    return reinterpret_cast<int*>(smem + S::BARS + 2 * S::STAGES * 8);
  }
  __device__ void init(uint8_t* smem) const {
    for (int i = 0; i < S::STAGES; i++) {
      mbar_init(full(i), 1);
      mbar_init(empty(i), S::WARPS);
    }
    *abort_word(smem) = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
};

// ---- the copying warp: bytes by TMA, scales by untiled copies, page by page ---------------
template <typename S>
__device__ void copy_blocks(const CUtensorMap& k_map, const CUtensorMap& v_map, const Attend8Args& args,
                            int box_bits, Place p, int units, uint8_t* smem) {
  constexpr int BK = S::BK;
  const AttendArgs& a = args.a;
  const int lane = threadIdx.x & 31;
  const uint32_t base = smem_u32(smem);
  const Bars<S> bars(base);
  int* abort_word = Bars<S>::abort_word(smem);
  volatile int* abort = abort_word;
  float* scales_s = reinterpret_cast<float*>(smem + S::SCALES);
  int fetched = 0;
  const int per_block = BK >> box_bits, per_bits = S::bits(BK) - box_bits;
  auto page_of = [&](const Place& k) {  // of this lane's box; -2 for none, -1 for a bad page
    const int key = k.blk * BK + (lane << box_bits);
    if (lane >= per_block || key >= tile_visible(a.tiling, k.r, k.tile)) return -2;
    const int page = a.batch.table[(int64_t)k.b * a.batch.columns + quotient(key, a.pools.by_page)];
    if (page >= 0 && page < a.pools.pages) return page;
    report(a.batch.status, ET_B200_PAGED_BAD_PAGE);
    return -1;  // outside the map: filled with zeros
  };
  int page = units > 0 ? page_of(p) : -2;
  for (int u = 0; u < units; u++) {
    const int st = u % S::STAGES, key0 = p.blk * BK, h = p.h, now = page;
    if (u >= S::STAGES &&
        !__all_sync(0xffffffffu, role_wait(bars.empty(st), (uint32_t)((u / S::STAGES - 1) & 1), abort_word, abort)))
      break;
    const int boxes = __popc(__ballot_sync(0xffffffffu, now != -2));
    const int sound = __popc(__ballot_sync(0xffffffffu, now >= 0));
    float* sc = scales_s + st * 2 * BK + (lane << box_bits);
    if (now == -1) {
      for (int i = 0; i < 1 << box_bits; i++) sc[i] = sc[BK + i] = 0.0f;
      fence_async_smem();  // before a later block's copy to these places
    }
    __syncwarp();
    if (lane == 0)
      mbar_expect_tx(bars.full(st), (uint32_t)((boxes << box_bits) * S::ROW * 2 + (sound << box_bits) * 8));
    __syncwarp();
    if (now >= 0) {
      const int key = key0 + (lane << box_bits);
      const int slot = key - quotient(key, a.pools.by_page) * a.pools.page_size;
      const int64_t off = now * args.scales.page_stride + h * args.scales.head_stride + slot;
      bulk_load(smem_u32(sc), args.scales.keys + off, 4u << box_bits, bars.full(st));
      bulk_load(smem_u32(sc + BK), args.scales.values + off, 4u << box_bits, bars.full(st));
    }
    const uint32_t dst = base + (uint32_t)st * S::STAGE;
    for (int i0 = 0; i0 < per_block * S::CHUNKS * 2; i0 += 32) {
      const int i = i0 + lane, box = i & (per_block - 1), c = i >> per_bits;  // K's chunks, then V's
      const int from = __shfl_sync(0xffffffffu, now, box);
      if (c < S::CHUNKS * 2 && from != -2) {
        const int key = key0 + (box << box_bits), chunk = c % S::CHUNKS;
        const int slot = key - quotient(key, a.pools.by_page) * a.pools.page_size;
        tma_load_4d(dst + (uint32_t)(c / S::CHUNKS) * S::TILE + (uint32_t)chunk * BK * S::CHUNK +
                        (uint32_t)(box << box_bits) * S::CHUNK,
                    c < S::CHUNKS ? &k_map : &v_map, bars.full(st), chunk * S::CHUNK, slot, h, from);
      }
      __syncwarp();
    }
    fetched = u + 1;
    advance(a.tiling, a.batch, p);
    if (u + 1 < units) page = page_of(p);
  }
  // every copy has landed before the block releases its memory
  for (int u = max(0, fetched - S::STAGES); u < fetched; u++)
    mbar_wait(bars.full(u % S::STAGES), (uint32_t)((u / S::STAGES) & 1), abort_word);
  if (lane == 0) report_abort(a.batch.status, abort);
}

// ---- copies by the arithmetic warps, for what TMA does not take ---------------------------
// The pages of a block's keys are looked up one block ahead of its copies.
template <typename S>
struct Copies {
  struct Ahead { int key0, h, unused[2]; };
  const Attend8Args& args;
  uint8_t* smem;
  Place kp;
  int units, looked = 0;
  __device__ Copies(const Attend8Args& x, uint8_t* s, const Place& p, int n) : args(x), smem(s), kp(p), units(n) {}
  __device__ int* pages(int u) const { return reinterpret_cast<int*>(smem + S::PAGES) + u % S::RING * S::BK; }
  __device__ Ahead& ahead(int u) const {
    return reinterpret_cast<Ahead*>(smem + S::PAGES + S::RING * S::BK * 4)[u % S::RING];
  }
  __device__ void look_up() {  // pages of block `looked`
    const AttendArgs& a = args.a;
    if (looked < units) {
      const int visible = tile_visible(a.tiling, kp.r, kp.tile);
      if (threadIdx.x == 0) ahead(looked) = Ahead{kp.blk * S::BK, kp.h, {0, 0}};
      for (int i = threadIdx.x; i < S::BK; i += S::NT) {
        const int key = kp.blk * S::BK + i;
        int page = -1;
        if (key < visible) {
          page = a.batch.table[(int64_t)kp.b * a.batch.columns + quotient(key, a.pools.by_page)];
          if (page < 0 || page >= a.pools.pages) {
            report(a.batch.status, ET_B200_PAGED_BAD_PAGE);
            page = -1;
          }
        }
        pages(looked)[i] = page;
      }
      advance(a.tiling, a.batch, kp);
    }
    looked++;
  }
  __device__ void issue(int u) const {  // copies of unit u into stage u % STAGES
    const AttendArgs& a = args.a;
    if (u < units) {
      const uint32_t st = smem_u32(smem) + (uint32_t)(u % S::STAGES) * S::STAGE;
      const uint32_t sc = smem_u32(smem) + S::SCALES + (uint32_t)(u % S::STAGES) * 2 * S::BK * 4;
      const Ahead at = ahead(u);
      auto slot_of = [&](int row) {
        const int key = at.key0 + row;
        return key - quotient(key, a.pools.by_page) * a.pools.page_size;
      };
      for (int i = threadIdx.x; i < S::BK * S::PIECES; i += S::NT) {
        const int row = i / S::PIECES, c = i % S::PIECES, page = pages(u)[row];
        const bool full = page >= 0 && c * 16 < a.pools.head_dim;
        const int64_t e = !full ? 0
                                : page * a.pools.page_stride + at.h * a.pools.head_stride +
                                      slot_of(row) * a.pools.token_stride + c * 16;
        const uint32_t dst = st + S::at8(row, c);
        cp16(dst, static_cast<const uint8_t*>(a.keys) + e, full);
        cp16(dst + S::TILE, static_cast<const uint8_t*>(a.values) + e, full);
      }
      for (int row = threadIdx.x; row < S::BK; row += S::NT) {
        const int page = pages(u)[row];
        const int64_t e = page < 0 ? 0
                                   : page * args.scales.page_stride + at.h * args.scales.head_stride +
                                         slot_of(row) * args.scales.token_stride;
        const int bytes = page < 0 ? 0 : 4;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(sc + 4u * row),
                     "l"(args.scales.keys + e), "r"(bytes) : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(sc + 4u * (S::BK + row)),
                     "l"(args.scales.values + e), "r"(bytes) : "memory");
      }
    }
    cp_commit();
  }
  __device__ void begin() {
#pragma unroll
    for (int s = 0; s < S::STAGES; s++) look_up();
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S::STAGES - 1; s++) issue(s);
  }
  __device__ void next(int u) {  // block u has arrived; every warp is done with block u - 1
    cp_wait<S::STAGES - 2>();
    __syncthreads();
    issue(u + S::STAGES - 1);
    look_up();
  }
};

// ---- queries ----------------------------------------------------------------------------
// The rows of the tile at p, rotated: 8 lanes to a row find its largest magnitude, then
// binary16 of the row times 2^e, and the factor of its scores in qmul.
template <typename T, typename S>
__device__ void load_queries(const AttendArgs& a, const Place& p, uint8_t* smem) {
  constexpr int DH = S::DH, BM = S::BM;
  const int lane = threadIdx.x & 31, dim = a.pools.head_dim, group = a.tiling.group;
  float* qmul = reinterpret_cast<float*>(smem + S::QMUL);
  const int first_row = p.tile << a.tiling.row_bits, rows = min(BM, p.r.n * group - first_row);
  constexpr int PAIRS = DH / 16;  // of a lane: its pairs are 8 apart, so neighbours read neighbours
#pragma unroll 1
  for (int r = threadIdx.x / 8; r < (BM + 3) / 4 * 4; r += S::NT / 8) {
    T x[PAIRS][2];
    float cs[PAIRS], sn[PAIRS];
    const int t = quotient(first_row + r, a.tiling.by_group), j = first_row + r - t * group;
    const int pos = p.r.len - p.r.n + t;
    const bool turn = a.rope.cos != nullptr && pos >= 0 && r < rows;
    const int64_t tab = turn ? rope_row(a.rope, pos, a.batch.status) * (dim / 2) : 0;
    const T* src = static_cast<const T*>(a.q) + (p.r.first + t) * a.q_stride +
                   (int64_t)(p.h * group + j) * dim;
#pragma unroll
    for (int i = 0; i < PAIRS; i++) {
      const int d = 2 * ((lane & 7) + 8 * i);
      x[i][0] = x[i][1] = from_f32<T>(0.0f);
      cs[i] = 1.0f;
      sn[i] = 0.0f;
      if (r < rows && d < dim) {
        x[i][0] = src[d];
        x[i][1] = src[d + 1];
        if (turn) {
          cs[i] = __ldg(a.rope.cos + tab + d / 2);
          sn[i] = __ldg(a.rope.sin + tab + d / 2);
        }
      }
    }
    float y[PAIRS][2], top = 0.0f;
#pragma unroll
    for (int i = 0; i < PAIRS; i++) {
      y[i][0] = to_f32<T>(x[i][0]);
      y[i][1] = to_f32<T>(x[i][1]);
      if (turn) rotate(y[i][0], y[i][1], cs[i], sn[i]);
      top = fmaxf(top, fmaxf(fabsf(y[i][0]), fabsf(y[i][1])));
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int e = query_exponent(top);
    const float by = exp2_int(e);
    if ((lane & 7) == 0) qmul[r] = a.scale_log2 * exp2_int(-e);
#pragma unroll
    for (int i = 0; i < PAIRS; i++) {
      const int d = 2 * ((lane & 7) + 8 * i);
      // the place of the pair among its 16 dims: as it is, or as the fragments of K
      // number them (dims 4 t + {0, 1} at 2 t, 4 t + {2, 3} at 8 + 2 t)
      const int in = (d & 15) / 2, to = S::CONVERT ? in : (in >> 1) + 4 * (in & 1);
      const uint32_t at = S::template at16<BM>(r, 2 * (d >> 4) + (to >> 2)) + 4 * (to & 3);
      const float y0 = y[i][0] * by, y1 = y[i][1] * by;
      const __half2 hi = __floats2half2_rn(y0, y1);
      *reinterpret_cast<__half2*>(smem + S::Q + at) = hi;
      if constexpr (S::QLO) {
        const float2 f = __half22float2(hi);
        *reinterpret_cast<__half2*>(smem + S::Q + S::TILE_Q + at) = __floats2half2_rn(y0 - f.x, y1 - f.y);
      }
    }
  }
}

// A value's scale b = 2^x c as (x, c), c below 2 (0 for a scale that is not finite).
__device__ __forceinline__ void scale_parts(float b, float& x, float& c) {
  const int e = (int)(__float_as_uint(b) >> 23) & 255, top = min(e, 253);
  x = (float)(top - 127);
  c = e == 255 ? 0.0f : b * __uint_as_float((uint32_t)(254 - top) << 23);
}
// The scale of a key's scores: NaN if either of its scales is not finite, so that the row
// makes NaN of the queries that see it, and of no other.
__device__ __forceinline__ float key_scale(float k, float v) { return fmaf(k + v, 0.0f, k); }
// The running maximum m of s, `big` of s + x, sum l and exponent D of a row of queries, and
// their change by a block whose maxima are top and tob.
struct RowState {
  float m, big, l, d;
  __device__ __forceinline__ void clear() {
    m = big = -INFINITY;
    l = d = 0.0f;
  }
  // returns what the row's sums of P V are to be multiplied by; from: m, or 0 at -inf
  __device__ __forceinline__ float raise(float top, float tob, float& from) {
    const float now = fmaxf(m, top);
    big = fmaxf(big, tob);
    from = now == -INFINITY ? 0.0f : now;
    const float next = now == -INFINITY ? 0.0f : rintf(big - now), fall = m - from;
    l *= ex2(fall);
    const float factor = ex2(fall + (d - next));
    m = now;
    d = next;
    return factor;
  }
  // 2^(D - kShift) in two factors
  __device__ __forceinline__ void scale(float& f0, float& f1) const {
    f0 = ex2(fmaxf(d - kShift, -120.0f));
    f1 = ex2(fminf(d - kShift + 120.0f, 0.0f));
  }
};

__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// d += (hi + lo) b of 16-deep products; SUM: the tensor pipe's accumulation truncates, so
// they are added in f32
template <bool LO, bool SUM>
__device__ __forceinline__ void product(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&hi)[2],
                                        const uint32_t (&lo)[2]) {
  if constexpr (SUM) {
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (LO) mma16<__half>(part, a, lo[0], lo[1]);
    mma16<__half>(part, a, hi[0], hi[1]);
#pragma unroll
    for (int e = 0; e < 4; e++) d[e] += part[e];
  } else {
    if constexpr (LO) mma16<__half>(d, a, lo[0], lo[1]);
    mma16<__half>(d, a, hi[0], hi[1]);
  }
}

// ---- few rows ----------------------------------------------------------------------------

template <typename T, typename S, bool TMA>
__global__ void __launch_bounds__(S::NT + (TMA ? 32 : 0), S::PER_SM)
few8_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
            const __grid_constant__ Attend8Args args, int box_bits) {
  constexpr int DH = S::DH, BM = S::BM, BK = S::BK, KW = S::KW, NT = S::NT, WK = S::WK;
  static_assert(WK == S::WARPS, "every warp takes all rows");
  constexpr int NQ = BM / 8, KG = KW / 16;  // columns of 8 queries, rows of 16 keys
  constexpr bool QLO = S::QLO, PLO = S::PLO;
  const AttendArgs& a = args.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* scales_s = reinterpret_cast<float*>(smem + S::SCALES);
  const float* qmul = reinterpret_cast<const float*>(smem + S::QMUL);
  float* join_m = reinterpret_cast<float*>(smem + S::JOIN);
  float* join_l = join_m + WK * BM;
  const uint32_t base = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, wk = tid >> 5;
  const int dim = a.pools.head_dim, group = a.tiling.group;
  const int g = lane >> 2, t2 = 2 * (lane & 3);  // a result's row (and row + 8), its columns
  // lets the joining kernel start its launch; it waits for this one's results
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Bars<S> bars(base);
  int* abort_word = Bars<S>::abort_word(smem);
  volatile int* abort = abort_word;
  if (TMA && tid == 0) bars.init(smem);

  Place p;
  __shared__ DivideRoom<NT + (TMA ? 32 : 0)> room;
  const Share share = divide(a.tiling, a.batch, a.least, p, room);
  __syncthreads();
  const int units = (int)share.units;
  if (TMA && wk == WK) {
    copy_blocks<S>(k_map, v_map, args, box_bits, p, units, smem);
    return;
  }
  Cut cut{0, 0, 0, 0, 0};
  if (units > 0) {
    Copies<S> copies(args, smem, p, units);
    if constexpr (!TMA) copies.begin();
    load_queries<T, S>(a, p, smem);
    named_sync(1, NT);

    float o[DH / 16][NQ][4];  // dims 16 i + 2 g + {0, 1} (e / 2) of queries 8 n + t2 + {0, 1} (e % 2)
    RowState row[NQ][2];
    float mul[NQ][2];
    int vis[NQ][2], vis_min = 0;
    bool whole = false;  // this block began the tile
    bool ok = true;
    for (int u = 0; u < units; u++) {
      const int st = u % S::STAGES;
      if constexpr (TMA) {
        // after a wait that ran out the loop still ends, in step with the other warps
        if (ok)
          ok = __all_sync(0xffffffffu, role_wait(bars.full(st), (uint32_t)((u / S::STAGES) & 1),
                                                 abort_word, abort));
      } else {
        copies.next(u);
      }
      if (u == 0 || p.blk == 0) {  // a new tile
        whole = p.blk == 0;
        const int first_row = p.tile << a.tiling.row_bits, rows = min(BM, p.r.n * group - first_row);
        if (u > 0) {
          if (TMA) named_sync(1, NT);  // every warp is done with the last tile's queries
          load_queries<T, S>(a, p, smem);
          named_sync(1, NT);
        }
#pragma unroll
        for (int i = 0; i < DH / 16; i++)
#pragma unroll
          for (int n = 0; n < NQ; n++) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const int r = 8 * n + t2 + c;
            row[n][c].clear();
            mul[n][c] = qmul[r];
            vis[n][c] = r < rows ? max(0, p.r.len - p.r.n + quotient(first_row + r, a.tiling.by_group) + 1) : 0;
          }
        // keys that every row sees; what rows without a query see does not matter
        vis_min = max(0, p.r.len - p.r.n + quotient(first_row, a.tiling.by_group) + 1);
      }
      const uint32_t kt = base + (uint32_t)st * S::STAGE, vt = kt + S::TILE;
      const float* ks_s = scales_s + st * 2 * BK;
      const float* vs_s = ks_s + BK;
      const bool tile_ends = p.blk + 1 == p.nblk;
      // slots behind the tile's keys may hold anything: this warp's rows of V
      const int valid = tile_ends ? tile_visible(a.tiling, p.r, p.tile) - p.blk * BK : BK;
      if (valid < (wk + 1) * KW) {
        for (int r = max(valid, wk * KW); r < (wk + 1) * KW; r++)
          for (int c = lane; c < S::PIECES; c += 32)
            sts128(vt + S::at8(r, c), make_float4(0.f, 0.f, 0.f, 0.f));
        __syncwarp();
      }

      // ---- scores of this warp's KW keys
      float s[KG][NQ][4];
#pragma unroll
      for (int k = 0; k < KG; k++)
#pragma unroll
        for (int n = 0; n < NQ; n++) s[k][n][0] = s[k][n][1] = s[k][n][2] = s[k][n][3] = 0.0f;
#pragma unroll
      for (int d = 0; d < DH / 32; d++) {  // 32 dims
        uint32_t qh[NQ][4], ql[NQ][4];     // pairs of two 16-deep products
#pragma unroll
        for (int n = 0; n < NQ; n++) {
          const uint32_t at = base + S::Q + S::template at16<BM>(8 * n + (lane & 7), 4 * d + (lane >> 3));
          ldsm4(qh[n], at);
          if constexpr (QLO) ldsm4(ql[n], at + S::TILE_Q);
        }
#pragma unroll
        for (int k = 0; k < KG; k++) {
          uint32_t kb[4];  // of the lower 16 dims the lower and the upper 8 keys, of the upper 16 dims
          ldsm4(kb, kt + S::at8(wk * KW + 16 * k + (lane & 15), 2 * d + (lane >> 4)));
#pragma unroll
          for (int i = 0; i < 2; i++) {
            uint32_t x[4];
            halves_of(kb[2 * i], x[0], x[2]);
            halves_of(kb[2 * i + 1], x[1], x[3]);
#pragma unroll
            for (int n = 0; n < NQ; n++) {
              const uint32_t hi[2] = {qh[n][2 * i], qh[n][2 * i + 1]};
              uint32_t lo[2] = {0, 0};
              if constexpr (QLO) lo[0] = ql[n][2 * i], lo[1] = ql[n][2 * i + 1];
              product<QLO, PLO>(s[k][n], x, hi, lo);
            }
          }
        }
      }
      // ---- scores times their keys' scales, running maxima; value scales as 2^x c
      const int key0 = p.blk * BK + wk * KW;
      const bool full = key0 + KW <= vis_min;
      float xv[KG][2], cv[KG][2];
      float top[NQ][2], tob[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; n++) top[n][0] = top[n][1] = tob[n][0] = tob[n][1] = -INFINITY;
#pragma unroll
      for (int k = 0; k < KG; k++)
#pragma unroll
        for (int h = 0; h < 2; h++) {  // key g, key g + 8
          const int in = wk * KW + 16 * k + 8 * h + g;
          scale_parts(in < valid ? vs_s[in] : 0.0f, xv[k][h], cv[k][h]);
          const float ks = key_scale(ks_s[in], vs_s[in]);
#pragma unroll
          for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
              float y = s[k][n][2 * h + c] * (ks * mul[n][c]);
              if (!full && key0 + 16 * k + 8 * h + g >= vis[n][c]) y = -INFINITY;
              s[k][n][2 * h + c] = y;
              top[n][c] = fmaxf(top[n][c], y);
              tob[n][c] = fmaxf(tob[n][c], y + xv[k][h]);
            }
        }
      bool changed = false;
      float factor[NQ][2], from[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; n++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            top[n][c] = fmaxf(top[n][c], __shfl_xor_sync(0xffffffffu, top[n][c], x));
            tob[n][c] = fmaxf(tob[n][c], __shfl_xor_sync(0xffffffffu, tob[n][c], x));
          }
          factor[n][c] = row[n][c].raise(top[n][c], tob[n][c], from[n][c]);
          changed |= factor[n][c] != 1.0f;
        }
      if (__any_sync(0xffffffffu, changed)) {
#pragma unroll
        for (int i = 0; i < DH / 16; i++)
#pragma unroll
          for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[i][n][e] *= factor[n][e & 1];
      }
      // ---- weights, as operands: keys t2 + {0, 1} (+ 8) of query g
      uint32_t ph[KG][NQ][2], pl[KG][NQ][2];
#pragma unroll
      for (int k = 0; k < KG; k++)
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float w[2];
#pragma unroll
            for (int c = 0; c < 2; c++) {
              const float y = s[k][n][2 * h + c] - from[n][c];
              row[n][c].l += ex2(y);
              w[c] = ex2(y + (xv[k][h] - (row[n][c].d - kShift))) * cv[k][h];
            }
            const __half2 x = __floats2half2_rn(w[0], w[1]);
            ph[k][n][h] = transposed(*reinterpret_cast<const uint32_t*>(&x));
            if constexpr (PLO) {
              const float2 f = __half22float2(x);
              pl[k][n][h] = transposed(pack2<__half>(w[0] - f.x, w[1] - f.y));
            }
          }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int k = 0; k < KG; k++)
#pragma unroll
        for (int d = 0; d < DH / 32; d++) {
          uint32_t vb[4];  // of the lower 16 dims the lower and the upper 8 keys, of the upper 16 dims
          ldsm4t(vb, vt + S::at8(wk * KW + 16 * k + (lane & 15), 2 * d + (lane >> 4)));
#pragma unroll
          for (int i = 0; i < 2; i++) {
            // bytes (key, dim): 00 01 10 11 -> 00 10 | 01 11: keys paired, even dim, odd dim
            uint32_t x[4];
            halves_of(__byte_perm(vb[2 * i], 0, 0x3120), x[0], x[1]);
            halves_of(__byte_perm(vb[2 * i + 1], 0, 0x3120), x[2], x[3]);
#pragma unroll
            for (int n = 0; n < NQ; n++) {
              uint32_t lo[2] = {0, 0};
              if constexpr (PLO) lo[0] = pl[k][n][0], lo[1] = pl[k][n][1];
              product<PLO, PLO>(o[2 * d + i][n], x, ph[k][n], lo);
            }
          }
        }

      if (tile_ends || u + 1 == units) {
        // ---- the warps' parts: relative to the largest of their maxima, then added up
        float l[NQ][2], m[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            float v = row[n][c].l;
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
            if (g == 0) {
              join_m[wk * BM + 8 * n + t2 + c] = row[n][c].m;
              join_l[wk * BM + 8 * n + t2 + c] = v;
            }
          }
        named_sync(1, NT);  // every warp is done with the stage, too
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const int r = 8 * n + t2 + c;
            float all = -INFINITY;
#pragma unroll
            for (int w = 0; w < WK; w++) all = fmaxf(all, join_m[w * BM + r]);
            const float ref = all == -INFINITY ? 0.0f : all;
            l[n][c] = 0.0f;
#pragma unroll
            for (int w = 0; w < WK; w++) l[n][c] += ex2(join_m[w * BM + r] - ref) * join_l[w * BM + r];
            m[n][c] = all;
            float f0, f1;
            row[n][c].scale(f0, f1);
            f1 *= ex2(row[n][c].m - ref);
#pragma unroll
            for (int i = 0; i < DH / 16; i++) {
              o[i][n][c] = o[i][n][c] * f0 * f1;
              o[i][n][2 + c] = o[i][n][2 + c] * f0 * f1;
            }
          }
        float4* merge = reinterpret_cast<float4*>(smem + st * S::STAGE);
#pragma unroll
        for (int half = WK / 2; half > 0; half >>= 1) {
          if (half < WK / 2) named_sync(1, NT);
          if (wk >= half && wk < 2 * half) {
#pragma unroll
            for (int i = 0; i < DH / 16; i++)
#pragma unroll
              for (int n = 0; n < NQ; n++)
                merge[((wk - half) * (DH / 16 * NQ) + i * NQ + n) * 32 + lane] =
                    make_float4(o[i][n][0], o[i][n][1], o[i][n][2], o[i][n][3]);
          }
          named_sync(1, NT);
          if (wk < half) {
#pragma unroll
            for (int i = 0; i < DH / 16; i++)
#pragma unroll
              for (int n = 0; n < NQ; n++) {
                const float4 x = merge[(wk * (DH / 16 * NQ) + i * NQ + n) * 32 + lane];
                o[i][n][0] += x.x;
                o[i][n][1] += x.y;
                o[i][n][2] += x.z;
                o[i][n][3] += x.w;
              }
          }
        }
        const bool done = whole && tile_ends;
        if (wk == 0) {
          const int slot = 2 * (int)blockIdx.x + (whole ? 1 : 0);
#pragma unroll
          for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
              const int r = 8 * n + t2 + c, at = (p.tile << a.tiling.row_bits) + r;
              if (done) {
                if (at < p.r.n * group) {
                  const int by = quotient(at, a.tiling.by_group), h = p.h * group + at - by * group;
                  const int64_t t = p.r.first + by;
                  const float inv = l[n][c] > 0.0f ? 1.0f / l[n][c] : 0.0f;
                  T* dst = static_cast<T*>(a.o) + t * a.o_stride + (int64_t)h * dim + 2 * g;
#pragma unroll
                  for (int i = 0; i < DH / 16; i++)
                    if (16 * i < dim) store2<T>(dst + 16 * i, o[i][n][c] * inv, o[i][n][2 + c] * inv);
                  if (a.lse != nullptr && g == 0)
                    a.lse[t * a.q_heads + h] = l[n][c] > 0.0f ? m[n][c] * kLn2 + logf(l[n][c]) : -INFINITY;
                }
              } else {
                float* dst = a.joint.sums + ((int64_t)slot * BM + r) * DH + 2 * g;
#pragma unroll
                for (int i = 0; i < DH / 16; i++)
                  *reinterpret_cast<float2*>(dst + 16 * i) = make_float2(o[i][n][c], o[i][n][2 + c]);
                if (g == 0) {
                  a.joint.stats[(int64_t)slot * 2 * BM + r] = m[n][c];
                  a.joint.stats[((int64_t)slot * 2 + 1) * BM + r] = l[n][c];
                }
              }
            }
        }
        if (whole && !tile_ends) {
          const int64_t rest = p.nblk - p.blk - 1;
          cut = Cut{p.r.first, p.r.n, p.h, p.tile, 1 + (int)((rest + share.per - 1) / share.per)};
        }
      }
      if constexpr (TMA) {
        if (tile_ends || u + 1 == units) fence_async_smem();  // plain writes before the next copy
        __syncwarp();
        if (lane == 0) mbar_arrive(bars.empty(st));
      }
      advance(a.tiling, a.batch, p);
    }
    if constexpr (TMA) {
      if (!ok && lane == 0) report_abort(a.batch.status, abort);
    } else {
      cp_wait<0>();
    }
  }
  if (tid == 0) a.joint.cuts[blockIdx.x] = cut;
}

// ---- more rows ---------------------------------------------------------------------------

template <typename T, typename S, bool TMA>
__global__ void __launch_bounds__(S::NT + (TMA ? 32 : 0), S::PER_SM)
many8_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
             const __grid_constant__ Attend8Args args, int box_bits) {
  constexpr int DH = S::DH, BM = S::BM, BK = S::BK, NT = S::NT;
  constexpr bool QLO = S::QLO, PLO = S::PLO;
  static_assert(S::CONVERT && BM == 16 * S::WARPS, "16 rows a warp");
  const AttendArgs& a = args.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* scales_s = reinterpret_cast<float*>(smem + S::SCALES);
  const float* qmul = reinterpret_cast<const float*>(smem + S::QMUL);
  const uint32_t base = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int dim = a.pools.head_dim, group = a.tiling.group;
  // lets the joining kernel start its launch; it waits for this one's results
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Bars<S> bars(base);
  int* abort_word = Bars<S>::abort_word(smem);
  volatile int* abort = abort_word;
  if (TMA && tid == 0) bars.init(smem);

  Place p;
  __shared__ DivideRoom<NT + (TMA ? 32 : 0)> room;
  const Share share = divide(a.tiling, a.batch, a.least, p, room);
  __syncthreads();
  const int units = (int)share.units;
  if (TMA && warp == S::WARPS) {
    copy_blocks<S>(k_map, v_map, args, box_bits, p, units, smem);
    return;
  }
  Cut cut{0, 0, 0, 0, 0};
  if (units > 0) {
    Copies<S> copies(args, smem, p, units);
    if constexpr (!TMA) copies.begin();
    load_queries<T, S>(a, p, smem);
    named_sync(1, NT);

    float o[DH / 8][4];
    RowState row[2];
    float mul[2];
    int vis[2], vis_min = 0;
    bool whole = false;  // this block began the tile
    bool ok = true;
    for (int u = 0; u < units; u++) {
      const int st = u % S::STAGES;
      if constexpr (TMA) {
        // after a wait that ran out the loop still ends, in step with the other warps
        if (ok)
          ok = __all_sync(0xffffffffu, role_wait(bars.full(st), (uint32_t)((u / S::STAGES) & 1),
                                                 abort_word, abort));
      } else {
        copies.next(u);
      }
      if (u == 0 || p.blk == 0) {  // a new tile
        whole = p.blk == 0;
        const int first_row = p.tile << a.tiling.row_bits, rows = min(BM, p.r.n * group - first_row);
        if (u > 0) {
          if (TMA) named_sync(1, NT);  // every warp is done with the last tile's queries
          load_queries<T, S>(a, p, smem);
          named_sync(1, NT);
        }
#pragma unroll
        for (int i = 0; i < DH / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int r = warp * 16 + lane / 4 + 8 * i;
          row[i].clear();
          mul[i] = qmul[r];
          vis[i] = r < rows ? max(0, p.r.len - p.r.n + quotient(first_row + r, a.tiling.by_group) + 1) : 0;
        }
        // keys that every row sees; what rows without a query see does not matter
        vis_min = max(0, p.r.len - p.r.n + quotient(first_row, a.tiling.by_group) + 1);
      }
      const uint32_t kt = base + (uint32_t)st * S::STAGE, vt = kt + S::TILE;
      const float* ks_s = scales_s + st * 2 * BK;
      const float* vs_s = ks_s + BK;
      const bool tile_ends = p.blk + 1 == p.nblk;
      // slots behind the tile's keys may hold anything
      const int valid = tile_ends ? tile_visible(a.tiling, p.r, p.tile) - p.blk * BK : BK;
      named_sync(1, NT);  // every warp is done with the last block's tiles
      for (int i = tid; i < BK * S::PIECES * 2; i += NT) {
        const int c = i % S::PIECES, r = i / S::PIECES % BK, v = i / (S::PIECES * BK);
        float4 raw = lds128((v ? vt : kt) + S::at8(r, c));
        if (v && r >= valid) raw = make_float4(0.f, 0.f, 0.f, 0.f);
        uint32_t h[8];
        halves_of(__float_as_uint(raw.x), h[0], h[1]);
        halves_of(__float_as_uint(raw.y), h[2], h[3]);
        halves_of(__float_as_uint(raw.z), h[4], h[5]);
        halves_of(__float_as_uint(raw.w), h[6], h[7]);
        const uint32_t to = base + S::CONV + (uint32_t)(v * S::TILE_16);
#pragma unroll
        for (int j = 0; j < 2; j++)
          sts128(to + S::template at16<BK>(r, 2 * c + j),
                 make_float4(__uint_as_float(h[4 * j]), __uint_as_float(h[4 * j + 1]),
                             __uint_as_float(h[4 * j + 2]), __uint_as_float(h[4 * j + 3])));
      }
      named_sync(1, NT);

      // ---- scores
      float s[BK / 8][4];
#pragma unroll
      for (int i = 0; i < BK / 8; i++) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
      // d += (hi + lo) b, as product() with the operands' parts exchanged
      auto add = [&](auto with_lo, float (&d)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                     uint32_t b0, uint32_t b1) {
        constexpr bool LO = decltype(with_lo)::value;
        if constexpr (PLO) {
          float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          if constexpr (LO) mma16<__half>(part, lo, b0, b1);
          mma16<__half>(part, hi, b0, b1);
#pragma unroll
          for (int e = 0; e < 4; e++) d[e] += part[e];
        } else {
          if constexpr (LO) mma16<__half>(d, lo, b0, b1);
          mma16<__half>(d, hi, b0, b1);
        }
      };
#pragma unroll
      for (int ks = 0; ks < DH / 16; ks++) {
        uint32_t qh[4], ql[4];
        const uint32_t at = base + S::Q + S::template at16<BM>(warp * 16 + (lane & 15), 2 * ks + (lane >> 4));
        ldsm4(qh, at);
        if constexpr (QLO) ldsm4(ql, at + S::TILE_Q);
#pragma unroll
        for (int n = 0; n < BK / 16; n++) {
          uint32_t kb[4];
          ldsm4(kb, base + S::CONV + S::template at16<BK>(16 * n + ((lane >> 4) << 3) + (lane & 7),
                                                           2 * ks + ((lane >> 3) & 1)));
          add(std::bool_constant<QLO>{}, s[2 * n], qh, ql, kb[0], kb[1]);
          add(std::bool_constant<QLO>{}, s[2 * n + 1], qh, ql, kb[2], kb[3]);
        }
      }
      // ---- scores times their keys' scales, running maxima (rows lane / 4 and lane / 4 + 8)
      const int key0 = p.blk * BK;
      const bool full = key0 + BK <= vis_min;
      float top[2] = {-INFINITY, -INFINITY}, tob[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < BK / 8; i++) {
        const int in = 8 * i + 2 * (lane & 3);
        float2 ks = *reinterpret_cast<const float2*>(ks_s + in);
        const float2 vb = *reinterpret_cast<const float2*>(vs_s + in);
        ks = make_float2(key_scale(ks.x, vb.x), key_scale(ks.y, vb.y));
        float xv[2], c;
        scale_parts(in < valid ? vb.x : 0.0f, xv[0], c);
        scale_parts(in + 1 < valid ? vb.y : 0.0f, xv[1], c);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float y = s[i][e] * ((e & 1 ? ks.y : ks.x) * mul[e >> 1]);
          s[i][e] = full || key0 + in + (e & 1) < vis[e >> 1] ? y : -INFINITY;
          top[e >> 1] = fmaxf(top[e >> 1], s[i][e]);
          tob[e >> 1] = fmaxf(tob[e >> 1], s[i][e] + xv[e & 1]);
        }
      }
      float factor[2], from[2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
          top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], x));
          tob[i] = fmaxf(tob[i], __shfl_xor_sync(0xffffffffu, tob[i], x));
        }
        factor[i] = row[i].raise(top[i], tob[i], from[i]);
      }
      if (__any_sync(0xffffffffu, factor[0] != 1.0f || factor[1] != 1.0f)) {
#pragma unroll
        for (int i = 0; i < DH / 8; i++) {
          o[i][0] *= factor[0];
          o[i][1] *= factor[0];
          o[i][2] *= factor[1];
          o[i][3] *= factor[1];
        }
      }
      // ---- weights and o += P V
#pragma unroll
      for (int kk = 0; kk < BK / 16; kk++) {
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int in = 16 * kk + 8 * i + 2 * (lane & 3);
          const float2 vb = *reinterpret_cast<const float2*>(vs_s + in);
          float xv[2], cv[2];
          scale_parts(in < valid ? vb.x : 0.0f, xv[0], cv[0]);
          scale_parts(in + 1 < valid ? vb.y : 0.0f, xv[1], cv[1]);
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float w[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const float y = s[2 * kk + i][2 * h + e] - from[h];
              row[h].l += ex2(y);
              w[e] = ex2(y + (xv[e] - (row[h].d - kShift))) * cv[e];
            }
            const __half2 x = __floats2half2_rn(w[0], w[1]);
            ph[2 * i + h] = *reinterpret_cast<const uint32_t*>(&x);
            if constexpr (PLO) {
              const float2 f = __half22float2(x);
              pl[2 * i + h] = pack2<__half>(w[0] - f.x, w[1] - f.y);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < DH / 16; n++) {
          uint32_t vb[4];
          ldsm4t(vb, base + S::CONV + S::TILE_16 +
                         S::template at16<BK>(16 * kk + (lane & 15), 2 * n + (lane >> 4)));
          add(std::bool_constant<PLO>{}, o[2 * n], ph, pl, vb[0], vb[1]);
          add(std::bool_constant<PLO>{}, o[2 * n + 1], ph, pl, vb[2], vb[3]);
        }
      }

      if (tile_ends || u + 1 == units) {
        const bool done = whole && tile_ends;
        const int slot = 2 * (int)blockIdx.x + (whole ? 1 : 0);
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float l = row[i].l, f0, f1;
          l += __shfl_xor_sync(0xffffffffu, l, 1);
          l += __shfl_xor_sync(0xffffffffu, l, 2);
          row[i].scale(f0, f1);
          const int r = warp * 16 + lane / 4 + 8 * i, at = (p.tile << a.tiling.row_bits) + r;
          if (done) {
            if (at < p.r.n * group) {
              const int by = quotient(at, a.tiling.by_group), h = p.h * group + at - by * group;
              const int64_t t = p.r.first + by;
              const float inv = l > 0.0f ? 1.0f / l : 0.0f;
              T* dst = static_cast<T*>(a.o) + t * a.o_stride + (int64_t)h * dim;
#pragma unroll
              for (int n = 0; n < DH / 8; n++) {
                const int d = 8 * n + 2 * (lane & 3);
                if (d < dim) store2<T>(dst + d, o[n][2 * i] * f0 * f1 * inv, o[n][2 * i + 1] * f0 * f1 * inv);
              }
              if (a.lse != nullptr && (lane & 3) == 0)
                a.lse[t * a.q_heads + h] = l > 0.0f ? row[i].m * kLn2 + logf(l) : -INFINITY;
            }
          } else {
            float* dst = a.joint.sums + ((int64_t)slot * BM + r) * DH;
#pragma unroll
            for (int n = 0; n < DH / 8; n++)
              *reinterpret_cast<float2*>(dst + 8 * n + 2 * (lane & 3)) =
                  make_float2(o[n][2 * i] * f0 * f1, o[n][2 * i + 1] * f0 * f1);
            if ((lane & 3) == 0) {
              a.joint.stats[(int64_t)slot * 2 * BM + r] = row[i].m;
              a.joint.stats[((int64_t)slot * 2 + 1) * BM + r] = l;
            }
          }
        }
        if (whole && !tile_ends) {
          const int64_t rest = p.nblk - p.blk - 1;
          cut = Cut{p.r.first, p.r.n, p.h, p.tile, 1 + (int)((rest + share.per - 1) / share.per)};
        }
      }
      if constexpr (TMA) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bars.empty(st));
      }
      advance(a.tiling, a.batch, p);
    }
    if constexpr (TMA) {
      if (!ok && lane == 0) report_abort(a.batch.status, abort);
    } else {
      cp_wait<0>();
    }
  }
  if (tid == 0) a.joint.cuts[blockIdx.x] = cut;
}

// ---- launching --------------------------------------------------------------------------

int padded8(int64_t dim) { return dim <= 64 ? 64 : padded(dim); }

template <typename T, typename S>
int launch_shape8(const et_b200_paged_cache8_v1* c, Attend8Args& x, void* ws, cudaStream_t stream) {
  AttendArgs& a = x.a;
  int box_bits = 0;
  while ((2 << box_bits) <= (c->page_size < S::BK ? c->page_size : S::BK)) box_bits++;
  CUtensorMap k_map, v_map;
  const bool tma = scales_copy(c) && pool8_map(&k_map, c->keys, c, S::CHUNK, 1 << box_bits) &&
                   pool8_map(&v_map, c->values, c, S::CHUNK, 1 << box_bits);
  auto go = [&](auto with_tma) {
    constexpr bool TMA = decltype(with_tma)::value;
    constexpr auto kernel = [] {
      if constexpr (S::CONVERT) return &many8_kernel<T, S, TMA>;
      else return &few8_kernel<T, S, TMA>;
    }();
    const int threads = S::NT + (TMA ? 32 : 0);
    const int blocks = thread_blocks(a, resident_blocks<kernel>(threads, S::SMEM) * a.sms, S::BM, S::BK);
    a.tiling = tiling_of(S::bits(S::BM), S::bits(S::BK), a.tiling.group, a.pools.kv_heads);
    a.least = 1;
    a.joint = joint_of(ws, blocks, S::BM, S::DH);
    kernel<<<blocks, threads, S::SMEM, stream>>>(k_map, v_map, x, box_bits);
    count_launch();
    return blocks;
  };
  return tma ? go(std::true_type{}) : go(std::false_type{});
}

// How a step's rows per kv head are taken.  One or two columns of 8 queries: few8_kernel
// alone.  More: tiles of 16, each of which reads the cache (from the L2 after the
// first), against one pass of attend8_tc, whose time is that of its conversion whatever the
// rows, or of many8_kernel, where that does not take the cache.  us for 20, 32, 48, 64, 96, 128 rows,
// 32 requests of up to 4,000 keys:
//   32 / 8 heads x 128, bf16: tiles of 16 rows 75, 104, 141, 174, 239, 308; attend8_tc 142, 148,
//     159, 164, 175, 180.  f32: 104, 145, 207, 248, 352, 466 and 198, 203, 213, 220, 229, 242.
//   16 heads x 64 of group 1, f32: 148, 181, 248, 308, 428, 544 and 311, 318, 327, 336, 349, 357.
// Against many8_kernel:
//   32 / 8 x 128, pages of 24, bf16: 86, 123, 173, 212, 297, 382 and 169, 170, 172, 174, 255, 289.
//     f32: 103, 148, 208, 255, 362, 468 (192 rows: 680) and 280, 281, 284, 286, 415, 480 (684).
//   32 / 8 x 64, pages of 24, f32: 71, 101, 136, 169, 234, 300 and 156, 156, 157, 159, 234, 265.
//   32 / 8 x 256, bf16: 134, 196, 280, 348, 505, 652 and 327, 329, 341, 341, 499, 573.  f32: 204, 300, 427,
//     539, 801, 1,016 (192 rows: 1,528; 256: 2,033) and 618, 621, 638, 640, 955, 1,101 (1,599; 1,958).
template <typename T, int DH>
int launch_dim8(const et_b200_paged_cache8_v1* c, Attend8Args& x, int64_t rows, void* ws,
                cudaStream_t stream) {
  constexpr bool F32 = sizeof(T) == 4;
  if constexpr (DH == 256) {
    if (rows <= 8) return launch_shape8<T, Shape8<T, DH, 8, 4, 4, 64, 3, 2>>(c, x, ws, stream);
    if (rows <= (F32 ? 192 : 48))
      return launch_shape8<T, Shape8<T, DH, 16, 4, 4, 128, 3, 1>>(c, x, ws, stream);
    return launch_shape8<T, Shape8<T, DH, 64, 4, 1, 64, 2, 1>>(c, x, ws, stream);
  } else {
    if (rows <= 8) return launch_shape8<T, Shape8<T, DH, 8, 4, 4, 128, 2, 3>>(c, x, ws, stream);
    using Sixteen = Shape8<T, DH, 16, 4, 4, 128, 3, 2>;
    if (rows <= (F32 && DH == 64 ? 64 : 48)) return launch_shape8<T, Sixteen>(c, x, ws, stream);
    if (const int blocks = attend8_tc(c, x, ws, stream)) return blocks;
    if (F32 && DH == 128 && rows <= 192) return launch_shape8<T, Sixteen>(c, x, ws, stream);
    return launch_shape8<T, Shape8<T, DH, 64, 4, 1, 64, 2, 2>>(c, x, ws, stream);
  }
}

template <typename T>
int launch_type8(const et_b200_paged_cache8_v1* c, Attend8Args& x, int64_t rows, void* ws,
                 cudaStream_t stream) {
  switch (padded8(c->head_dim)) {
    case 64: return launch_dim8<T, 64>(c, x, rows, ws, stream);
    case 128: return launch_dim8<T, 128>(c, x, rows, ws, stream);
    default: return launch_dim8<T, 256>(c, x, rows, ws, stream);
  }
}

}  // namespace
}  // namespace etb

using namespace etb;
using namespace etb::paged;

extern "C" {

size_t et_b200_paged_attention8_workspace_bytes_v1(const et_b200_paged_cache8_v1* c,
                                                   int64_t q_heads) {
  if (check_cache8(c, nullptr, "paged-attention8-workspace") || !heads_fit(c->kv_heads, q_heads))
    return 0;
  return attention_workspace(padded8(c->head_dim), sm_count());
}

int32_t et_b200_paged_attention8_v1(const et_b200_paged_cache8_v1* c,
                                    const et_b200_paged_batch_v1* b,
                                    const et_b200_paged_rope_v1* rope, int64_t q_heads,
                                    const void* q, int64_t q_stride, void* o, int64_t o_stride,
                                    float* lse, void* workspace, size_t bytes, void* stream,
                                    et_kernel_error* e) {
  const char* op = "paged-attention8";
  if (int32_t r = check_cache8(c, e, op)) return r;
  if (int32_t r = check_batch(b, c->page_size, e, op)) return r;
  if (int32_t r = check_rope(rope, e, op)) return r;
  if (!heads_fit(c->kv_heads, q_heads))
    return set_error(e, ET_KERNEL_ERROR_SHAPE_MISMATCH, ET_KERNEL_CODE_INVALID_SHAPE, op,
                     "q_heads must be a multiple of the cache's kv_heads, up to 65536");
  if (b->tokens > 0 && b->batch > 0) {
    const int sms = sm_count();
    if (int32_t r = check_attention(b, c->head_dim, c->dtype == ET_B200_DTYPE_F32 ? 4 : 2, q_heads,
                                    q, q_stride, o, o_stride, lse, workspace, bytes,
                                    attention_workspace(padded8(c->head_dim), sms), e, op))
      return r;
    Attend8Args x{};
    AttendArgs& a = x.a;
    x.scales = scales_of(c);
    a.pools = pools_of(c);
    a.batch = batch_of(b, c->page_size);
    a.rope = rope_of(rope);
    a.tiling.group = (int)(q_heads / c->kv_heads);
    a.keys = c->keys;
    a.values = c->values;
    a.q = q;
    a.o = o;
    a.lse = lse;
    a.q_stride = q_stride;
    a.o_stride = o_stride;
    a.q_heads = (int)q_heads;
    a.sms = sms;
    a.q_factor = 1.0f;
    a.scale_log2 = kLog2e / sqrtf((float)c->head_dim);
    auto st = static_cast<cudaStream_t>(stream);
    const int64_t rows = least_of(b->max_new, (int64_t)INT32_MAX) * a.tiling.group;
    const int blocks = c->dtype == ET_B200_DTYPE_F32   ? launch_type8<float>(c, x, rows, workspace, st)
                       : c->dtype == ET_B200_DTYPE_F16 ? launch_type8<__half>(c, x, rows, workspace, st)
                                                       : launch_type8<__nv_bfloat16>(c, x, rows, workspace, st);
    join_parts(a, c->dtype, padded8(c->head_dim), blocks, rows, st);
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return cuda_error(e, status, op);
  }
  if (e) memset(e, 0, sizeof(*e));
  return 0;
}

}  // extern "C"
