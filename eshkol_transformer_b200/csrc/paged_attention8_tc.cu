// Attention of chunks of new tokens over an 8-bit paged cache on tcgen05: head_dim up to
// 128, pages of a power of two of at least 8 slots.
//
// The mathematics are those of paged_attention8.cu, tiles and roles those of
// paged_attention_tc.cu (256 rows as two halves, blocks of 128 keys, a warpgroup of
// probabilities and a product warp a half), with four more warps that turn each
// block's bytes into the binary16 tiles that the products read.  They also apply the
// scales, so the probabilities' loop knows nothing of them: rows of K times 2^(6 - E)
// with E the largest exponent of the block's scales, a constant of the block's scores;
// rows of V times 2^(6 - F) with F the largest exponent of the tile's blocks so far, by
// whose growth O is rescaled together with a new maximum.  With scales that are
// powers of two that is exact down to 2^-21 of the largest (binary16 holds 2^-24 to
// 2^15, an element 2^-9 to 448); other scales round each element to 11 bits.
// Queries are binary16 times 2^-e of their row, weights binary16 times 2^11 below a
// standing maximum that allows 2^4: 11 bits, more than a bf16 result keeps (queries with their residual do not
// fit shared memory beside two halves of 128 dims).  At f32 both carry
// the residual of that rounding (22 bits, two products instead of one), and the products of a
// block are added to f32 sums in tensor memory.
//
// 4,096 tokens over 12,000 keys (32 / 8 heads x 128, bf16): 930 us, 720 TFLOP/s, 43 % of the
// matrix rate (810 to 840 with the conversion's arithmetic left out).  Bound by the chain
// of a block (scores to probabilities 3,000 to 3,500 cycles, conversion 1,250 beside it), with
// issue slots 46 % and the tensor pipe 34 % busy, the roles' code beyond the instruction cache
// (stalls for it 0.5 a warp's instruction; placement moves the time by 5 %).  Four ragged f32
// prompts to 1,024 (16 heads x 64): 78 us with the joining, of 7 blocks in two tiles a thread
// block half in queries (6.5 us a tile) and outputs (4 us), issue slots 28 % busy.  f32 at 128
// dims: 2,048 tokens over 6,000 keys (32 / 8 heads) 635 us, tiles of one half (1,771 us by
// mma.sync).
// Measured and not kept: a warp that computes the scales' factors ahead (978 to 1,130 us),
// probabilities in rolled loops (1,216 to 1,327), the halves along the keys for few rows (140 to
// 180 us for 20 to 128 rows where this takes 135 to 175), loads of the queries two or three
// steps ahead (prompts 83 and 85 us) or prefetched into the L2 (83).
// Waits are bounded; one that runs out raises a CTA-wide abort, copies and
// products in flight are waited for and TMEM is released.
#include <math.h>

#include <type_traits>

#include "attention_f16.cuh"
#include "paged8.cuh"
#include "paged_mma.cuh"

namespace etb {
namespace {

using namespace paged;
using namespace f16att;

constexpr int HALF = 128, BK = 128;
// warps 0-7 probabilities; 8, 9 products, 10 copies; 12-15 conversion.  Registers of
// the warpgroups out of 512 x 128.
constexpr int MMA_WARP = 8, LOAD_WARP = 10, CONVERT_WARP = 12, THREADS = 512;
constexpr int kWideRegs = 200, kLeanRegs = 56, kConvertRegs = 56;
static_assert(256 * kWideRegs + 128 * (kLeanRegs + kConvertRegs) <= THREADS * 128, "registers at launch");
constexpr float kJump = 4.0f, kShift = 11.0f;  // weights reach 2^15
constexpr int RING = 8;  // blocks whose exponents are kept: more than conversion runs ahead
constexpr int kNone = -1000;  // the exponent of no scale
constexpr int kMarked = 4096;  // added to E of a block with keys that make NaN

// PAIRS: queries and weights with their residuals (f32)
template <int DH, bool PAIRS>
struct Layout {
  // halves of 128 rows; f32 at 128 dims has one, as its sums take the other's tensor memory
  static constexpr int HALVES = PAIRS && DH == 128 ? 1 : 2;
  static constexpr int SLOT = BK * DH * 2;  // one block of K or V in binary16
  static constexpr int SLOTS = DH == 128 ? 3 : 6;
  static constexpr int RAW = BK * DH;       // one block of K or V in bytes
  static constexpr int RAWS = DH == 128 ? 4 : PAIRS ? 6 : 8;
  static constexpr int TILE_Q = HALF * DH * 2 * (PAIRS ? 2 : 1);
  static constexpr int Q = SLOTS * SLOT;
  static constexpr int BYTES = Q + HALVES * TILE_Q;
  static constexpr int SCALES = BYTES + RAWS * RAW;  // [block % (RAWS / 2)][keys, values][BK]
  static constexpr int BARS = SCALES + RAWS * BK * 4;
  static constexpr int SMEM = BARS + 512;
  // TMEM: scores of the halves (P over the first 64 columns, its residual over the others),
  // outputs, with PAIRS their sums over blocks
  static constexpr uint32_t S0 = 0, O0 = 256, SUM0 = O0 + HALVES * DH, COLS = 512;
  static_assert(SUM0 + (PAIRS ? HALVES * DH : 0) <= COLS && SMEM <= 232448, "TMEM and shared memory");
};

// Whether `v` holds for all `threads` threads of a named barrier.
__device__ __forceinline__ bool named_all(int id, int threads, bool v) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %3, 0;\n\t"
      "bar.red.and.pred p, %1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(all)
      : "r"(id), "r"(threads), "r"((uint32_t)v)
      : "memory");
  return all != 0;
}

// x 2^e in two steps, e from -252 to 252
__device__ __forceinline__ float times_power(float x, int e) {
  const int h = e / 2;
  return x * exp2_int(h) * exp2_int(e - h);
}

template <typename T, int DH>
__global__ void __launch_bounds__(THREADS, 1)
paged_attention8_tc_kernel(const __grid_constant__ CUtensorMap k_map,
                           const __grid_constant__ CUtensorMap v_map, Attend8Args args, int box_rows) {
  constexpr bool PAIRS = sizeof(T) == 4;
  using L = Layout<DH, PAIRS>;
  constexpr int SLOTS = L::SLOTS, RAWS = L::RAWS, TILE = L::HALVES * HALF;
  const AttendArgs& a = args.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* scales_s = reinterpret_cast<float*>(smem + L::SCALES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  enum { FULL = 0, EMPTY = FULL + SLOTS, RAWFULL = EMPTY + SLOTS, RAWEMPTY = RAWFULL + RAWS,
         SFULL = RAWEMPTY + RAWS, PREADY = SFULL + 2, QREADY = PREADY + 2, ODONE = QREADY + 2,
         DRAIN = ODONE + 2, TURN = DRAIN + 2, EXPS = TURN + 2, NBARS = EXPS + RING };
  const uint32_t bar0 = smem_u32(bars);
  auto B_ = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  int* exps = reinterpret_cast<int*>(bars + NBARS);  // [RING][E, F]
  int* found = exps + 2 * RING;                      // [E, F, NaN][4 warps]
  uint32_t* tslot = reinterpret_cast<uint32_t*>(found + 12);
  int* abort_word = reinterpret_cast<int*>(tslot + 1);
  static_assert(NBARS * 8 + (2 * RING + 12 + 2) * 4 <= 512, "room behind the tiles");
  volatile int* abort = abort_word;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_u32(smem);
  const int group = a.tiling.group, dim = a.pools.head_dim;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (tid == 0) {
    for (int i = 0; i < NBARS; i++)
      mbar_init(B_(i), i < EMPTY                       ? 128
                       : i < RAWFULL                   ? 2
                       : i >= RAWEMPTY && i < SFULL    ? 4
                       : i >= PREADY && i < ODONE      ? HALF
                                                       : 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) tmem_alloc(smem_u32(tslot), L::COLS);
  Place p;
  // the rows of Q are written behind the barrier below
  const Share share = divide(a.tiling, a.batch, a.least, p,
                             *reinterpret_cast<DivideRoom<THREADS>*>(smem + L::Q));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  // blocks of the tile at p that fall into this share, and its rows
  int64_t left = share.units;
  auto blocks_here = [&]() { return (int)min((int64_t)(p.nblk - p.blk), left); };
  auto rows_here = [&]() {
    return min(TILE, p.r.n * group - p.tile * TILE);
  };
  auto next_tile = [&](int done) {
    left -= done;
    p.blk += done - 1;
    advance(a.tiling, a.batch, p);
  };
  auto wait = [&](int i, uint32_t parity) {
    return role_wait(B_(i), parity & 1u, abort_word, abort);
  };

  if (warp >= CONVERT_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegs));
    // ---- bytes into binary16, rows times their scales
    const int c = tid - 32 * CONVERT_WARP;  // this thread's key of a block's scales
    // A thread takes 16-byte pieces of rows that share their place among 8, so its addresses
    // differ by constants; lanes 4 apart take rows r and r ^ 5, whose pieces lie in
    // different banks, both of the bytes and of what is written.
    constexpr int GROUPS = DH / 64;                                  // of 4 pieces
    constexpr int APART = DH == 128 ? 16 : 32, ROUNDS = BK / APART;  // rows from one to the next
    const int quarter = DH == 128 ? (lane >> 4) + 2 * (warp & 1) : lane >> 3 & 3;
    const int r0 = 8 * (DH == 128 ? warp >> 1 & 1 : warp & 3) + ((lane & 4) ? quarter ^ 5 : quarter);
    const int in = lane & 3, piece = in + 4 * (GROUPS > 1 ? lane >> 3 & 1 : 0);
    const uint32_t from = base + L::BYTES + (uint32_t)r0 * DH +
                          (uint32_t)((DH == 128 ? piece ^ (r0 & 7) : piece ^ (r0 >> 1 & 3)) << 4);
    const uint32_t to = base + (uint32_t)(piece / 4) * BK * 128u + (uint32_t)r0 * 128u;
    const uint32_t to0 = to + (uint32_t)(((2 * in) ^ (r0 & 7)) << 4);
    const uint32_t to1 = to + (uint32_t)(((2 * in + 1) ^ (r0 & 7)) << 4);
    uint32_t n = 0;
    // a wait of one warp that runs out ends the four together, at their next barrier
    bool ok = true, live = true;
    while (live && left > 0) {
      const int nb = blocks_here(), visible = tile_visible(a.tiling, p.r, p.tile);
      int high = kNone;  // F
      for (int j = 0; j < nb; j++, n++) {
        // the scales of both come with V, whose slot says when theirs is free
        if (ok) ok = wait(RAWFULL + 2 * n % RAWS, 2 * n / RAWS);
        if (ok) ok = wait(RAWFULL + (2 * n + 1) % RAWS, (2 * n + 1) / RAWS);
        ok = __all_sync(0xffffffffu, ok);
        const int valid = visible - (p.blk + j) * BK;
        uint32_t* factors = reinterpret_cast<uint32_t*>(scales_s + n % (RAWS / 2) * 2 * BK);
        int e[2];
        float s[2];
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 2; i++) {
          s[i] = c < valid ? __uint_as_float(factors[i * BK + c]) : 0.0f;
          const int x = (int)(__float_as_uint(s[i]) >> 23) & 255;
          bad |= x == 255;
          e[i] = s[i] == 0.0f || x == 255 ? kNone : min(max(x, 1) - 127, 126);
          const int top = __reduce_max_sync(0xffffffffu, e[i]);
          if (lane == 0) found[4 * i + (warp & 3)] = top;
        }
        const bool any = __any_sync(0xffffffffu, bad);
        if (lane == 0) found[8 + (warp & 3)] = any;
        live = named_all(1, 128, ok);
        if (!live) break;
#pragma unroll
        for (int i = 0; i < 2; i++) e[i] = max(max(found[4 * i], found[4 * i + 1]), max(found[4 * i + 2], found[4 * i + 3]));
        if (e[0] == kNone) e[0] = 0;
        high = max(high, e[1]);
        e[1] = high == kNone ? 0 : high;
        // in place of the scales: their products, as pairs of binary16.  A key with a scale that
        // is not finite makes NaN of its scores, which those that do not see it drop.
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const __half2 f = __float2half2_rn(bad ? (i == 0 ? NAN : 0.0f) : s[i] * exp2_int(-e[i]) * 64.0f);
          factors[i * BK + c] = *reinterpret_cast<const uint32_t*>(&f);
        }
        if (c == 0) {
          exps[2 * (n % RING)] = e[0] + ((found[8] | found[9] | found[10] | found[11]) ? kMarked : 0);
          exps[2 * (n % RING) + 1] = e[1];
          mbar_arrive(B_(EXPS + n % RING));
        }
        named_sync(1, 128);
#pragma unroll 1
        for (int kv = 0; kv < 2; kv++) {
          const uint32_t count = 2 * n + kv, slot = count % SLOTS, round = count / SLOTS;
          const uint32_t st = count % RAWS;
          if (round > 0) ok = __all_sync(0xffffffffu, wait(EMPTY + slot, round - 1));
          if (!ok) break;  // live until the next barrier
          const uint32_t raw = from + st * L::RAW, out = slot * L::SLOT;
          const uint32_t* factor = factors + kv * BK + r0;
          constexpr int BATCH = 2;  // rows whose loads go out together
#pragma unroll 1
          for (int i0 = 0; i0 < ROUNDS; i0 += BATCH) {
            float4 x[BATCH];
            uint32_t f[BATCH];
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
              x[k] = lds128(raw + (uint32_t)((i0 + k) * APART * DH));
              f[k] = factor[(i0 + k) * APART];
            }
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
              uint32_t h[8];
              halves_of(__float_as_uint(x[k].x), h[0], h[1]);
              halves_of(__float_as_uint(x[k].y), h[2], h[3]);
              halves_of(__float_as_uint(x[k].z), h[4], h[5]);
              halves_of(__float_as_uint(x[k].w), h[6], h[7]);
#pragma unroll
              for (int e = 0; e < 8; e++) asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(h[e]) : "r"(f[k]));
              if (valid < BK && r0 + (i0 + k) * APART >= valid)  // slots behind the keys may hold anything
#pragma unroll
                for (int e = 0; e < 8; e++) h[e] = 0;
              const uint32_t at = out + (uint32_t)((i0 + k) * APART * 128);
              sts128(to0 + at, make_float4(__uint_as_float(h[0]), __uint_as_float(h[1]),
                                           __uint_as_float(h[2]), __uint_as_float(h[3])));
              sts128(to1 + at, make_float4(__uint_as_float(h[4]), __uint_as_float(h[5]),
                                           __uint_as_float(h[6]), __uint_as_float(h[7])));
            }
          }
          fence_async_smem();
          mbar_arrive(B_(FULL + slot));
          __syncwarp();
          if (lane == 0) mbar_arrive(B_(RAWEMPTY + st));
        }
      }
      next_tile(nb);
    }
  } else if (warp >= MMA_WARP) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLeanRegs));
  if (warp == LOAD_WARP) {
    // ---- bytes and scales of K and V, page by page: lanes 0 to 15 K, the others V
    uint32_t n = 0, count = 0;
    bool ok = true;
    while (ok && left > 0) {
      const int nb = blocks_here(), visible = tile_visible(a.tiling, p.r, p.tile);
      for (int j = 0; j < nb; j++) {
        const int key0 = (p.blk + j) * BK;
        const int boxes = max(0, (min(visible - key0, BK) + box_rows - 1) / box_rows);
        // each lane looks up the box it will load (at most 16 pages of 8 keys)
        const int mine = lane % 16, v = lane / 16;
        int page = -1, slot = 0;
        if (mine < boxes) {
          const int key = key0 + mine * box_rows, column = quotient(key, a.pools.by_page);
          slot = key - column * a.pools.page_size;
          page = a.batch.table[(int64_t)p.b * a.batch.columns + column];
          if (page < 0 || page >= a.pools.pages) {
            report(a.batch.status, ET_B200_PAGED_BAD_PAGE);
            page = -1;  // outside the map: filled with zeros
          }
        }
#pragma unroll
        for (int kv = 0; kv < 2; kv++, count++) {
          const uint32_t st = count % RAWS, round = count / RAWS, bar = B_(RAWFULL + st);
          if (round > 0) ok = wait(RAWEMPTY + st, round - 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          uint32_t bytes = (uint32_t)(boxes * box_rows * DH);
          float* scales = scales_s + (n % (RAWS / 2) * 2 + v) * BK + mine * box_rows;
          if (kv == 1) {
            if (mine < boxes && page < 0)
              for (int i = 0; i < box_rows; i++) scales[i] = 0.0f;
            bytes += (uint32_t)(__popc(__ballot_sync(0xffffffffu, page >= 0)) * box_rows * 4);
            __syncwarp();
          }
          if (lane == 0) mbar_expect_tx(bar, bytes);
          __syncwarp();
          if (kv == 1 && page >= 0)
            bulk_load(smem_u32(scales),
                      (v ? args.scales.values : args.scales.keys) + page * args.scales.page_stride +
                          p.h * args.scales.head_stride + slot,
                      4u * box_rows, bar);
          if (v == kv && mine < boxes)
            tma_load_4d(base + L::BYTES + st * L::RAW + (uint32_t)(mine * box_rows) * DH,
                        v ? &v_map : &k_map, bar, 0, slot, p.h, page);
        }
        if (!ok) break;
        n++;
      }
      next_tile(nb);
    }
    // every copy has landed before the CTA releases its memory
    if (lane == 0)
      for (uint32_t i = count > RAWS ? count - RAWS : 0; i < count; i++)
        mbar_wait(B_(RAWFULL + i % RAWS), (i / RAWS) & 1u, abort_word);
  } else if (warp < LOAD_WARP) {
    // ---- products of half t.  A half without rows goes along with the slots.
    const int t = warp - MMA_WARP;
    constexpr uint32_t idesc_s = idesc_f16_m128(BK, 0);
    constexpr uint32_t idesc_o = idesc_f16_m128(DH, 1);
    const uint32_t q = base + L::Q + (uint32_t)t * L::TILE_Q;
    const uint32_t s_at = tmem + L::S0 + 128u * t, o_at = tmem + L::O0 + (uint32_t)(DH * t);
    uint32_t count = 0, items = 0, steps = 0, turns = 0;
    bool ok = true;
    // the halves' products go out in turns while both have rows
    auto my_turn = [&](bool both) { return !both || (t == 0 && turns == 0) || wait(TURN + t, turns - 1 + t); };
    auto pass_on = [&](bool both) {
      if (both) {
        mbar_arrive(B_(TURN + 1 - t));
        turns++;
      }
    };
    auto scores = [&](uint32_t slot) {
      const uint32_t k = base + slot * L::SLOT;
#pragma unroll
      for (int i = 0; i < DH / 16; i++) {
        if constexpr (PAIRS)
          umma_f16(s_at, kdesc16<HALF>(q + HALF * DH * 2, i), kdesc16<BK>(k, i), idesc_s, i > 0 ? 1u : 0u);
        umma_f16(s_at, kdesc16<HALF>(q, i), kdesc16<BK>(k, i), idesc_s, PAIRS || i > 0 ? 1u : 0u);
      }
      umma_commit(B_(SFULL + t));
    };
    while (ok && left > 0) {
      const int nb = blocks_here();
      const bool rows = rows_here() > HALF * t, both = rows_here() > HALF;
      uint32_t ks = count % SLOTS;
      ok = wait(FULL + ks, count / SLOTS);
      count++;
      if (ok && rows) ok = wait(QREADY + t, items);
      if (ok) ok = my_turn(both);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      if (lane == 0) {
        if (rows) scores(ks);
        pass_on(both);
        umma_commit(B_(EMPTY + ks));
      }
      turns = __shfl_sync(0xffffffffu, turns, 0);
      for (int j = 0; j < nb; j++) {
        const uint32_t vs = count % SLOTS, vt = base + vs * L::SLOT;
        ok = __all_sync(0xffffffffu, wait(FULL + vs, count / SLOTS));
        if (!ok) break;
        count++;
        const bool more = j + 1 < nb;
        if (more) {
          ks = count % SLOTS;
          ok = wait(FULL + ks, count / SLOTS);
          count++;
        }
        if (ok && rows) ok = wait(PREADY + t, steps);
        if (ok) ok = my_turn(both);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          if (rows) {
#pragma unroll
            for (int i = 0; i < BK / 16; i++) {
              const uint32_t more_of_it = (!PAIRS && j > 0) || i > 0 ? 1u : 0u;
              if constexpr (PAIRS) {
                umma_f16_ts(o_at, s_at + 64u + 8u * i, mdesc16<BK>(vt, i), idesc_o, more_of_it);
                umma_f16_ts(o_at, s_at + 8u * i, mdesc16<BK>(vt, i), idesc_o, 1u);
              } else {
                umma_f16_ts(o_at, s_at + 8u * i, mdesc16<BK>(vt, i), idesc_o, more_of_it);
              }
            }
            if (more) scores(ks);
            else umma_commit(B_(ODONE + t));
          }
          pass_on(both);
          umma_commit(B_(EMPTY + vs));
          if (more) umma_commit(B_(EMPTY + ks));
        }
        turns = __shfl_sync(0xffffffffu, turns, 0);
        steps += rows ? 1 : 0;
      }
      items += rows ? 1 : 0;
      next_tile(nb);
    }
    if (lane == 0) {
      umma_commit(B_(DRAIN + t));
      mbar_wait(B_(DRAIN + t), 0u, abort_word);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWideRegs));
    // ---- probabilities: half t, one row per thread
    const int t = warp >> 2, row = tid & (HALF - 1);
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_at = lanes + L::S0 + 128u * t, o_at = lanes + L::O0 + (uint32_t)(DH * t);
    const uint32_t sum_at = lanes + L::SUM0 + (uint32_t)(DH * t);
    constexpr int SIZE = (int)sizeof(T);
    const bool q_vec = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * SIZE)) & 15) == 0;
    const bool rope_vec = ((reinterpret_cast<uintptr_t>(a.rope.cos) | reinterpret_cast<uintptr_t>(a.rope.sin)) & 15) == 0;
    const bool o_vec = ((reinterpret_cast<uintptr_t>(a.o) | (uintptr_t)(a.o_stride * SIZE)) & 15) == 0;
    uint32_t items = 0, steps = 0, n = 0;
    bool ok = true;
    Cut cut{0, 0, 0, 0, 0};
    while (ok && left > 0) {
      const int nb = blocks_here(), rows = rows_here() - HALF * t;
      const bool whole = p.blk == 0, ends = p.blk + nb == p.nblk;
      if (whole && !ends) {
        const int64_t rest = p.nblk - nb;
        cut = Cut{p.r.first, p.r.n, p.h, p.tile, 1 + (int)((rest + share.per - 1) / share.per)};
      }
      if (rows > 0) {
        const int first_row = p.tile * TILE + HALF * t, g = first_row + row;
        const bool valid = row < rows;
        const int token = quotient(g, a.tiling.by_group), head = p.h * group + g - token * group;
        const int pos = p.r.len - p.r.n + token;
        const int vis = valid ? max(0, pos + 1) : 0;
        // keys that every row of this warp sees (invalid rows follow the last valid one)
        const int vis_warp = __shfl_sync(0xffffffffu, max(0, pos + 1), 0);
        // a warp without rows only keeps its barriers; its lanes of the products hold anything
        const bool live = (warp & 3) * 32 < rows;
        // ---- the warp's rows of Q, rotated and times 2^e, into the swizzled tile: 8 lanes a
        // row, whole lines, 4 rows' loads ahead of their use.  Rolled, as whatever runs once a
        // tile is: its instructions have to be fetched each time.
        float row_scale = 0.0f;
        if (live) {
          constexpr int P = DH / 64;  // 8 dims of a lane
          const uint32_t tile = base + L::Q + (uint32_t)t * L::TILE_Q;
          union Piece { uint4 v[SIZE / 2]; T x[8]; };
          Piece u[P], u_next[P];
          float4 cs[P], sn[P], cs_next[P], sn_next[P];
          auto load = [&](int r, Piece (&u)[P], float4 (&cs)[P], float4 (&sn)[P]) {
            const int gr = first_row + r;
            const int tk = quotient(gr, a.tiling.by_group), at_pos = p.r.len - p.r.n + tk;
            const bool some = r < rows;
            const T* src = static_cast<const T*>(a.q) + (p.r.first + tk) * a.q_stride +
                           (int64_t)(p.h * group + gr - tk * group) * dim;
            const int64_t tab = some && a.rope.cos != nullptr && at_pos >= 0
                                    ? rope_row(a.rope, at_pos, a.batch.status) * (dim / 2) : -1;
#pragma unroll
            for (int i = 0; i < P; i++) {
              const int d = 8 * ((lane & 7) + 8 * i);
#pragma unroll
              for (int e = 0; e < SIZE / 2; e++) u[i].v[e] = make_uint4(0, 0, 0, 0);
              cs[i] = make_float4(1.f, 1.f, 1.f, 1.f);
              sn[i] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (some && d < dim) {
                if (q_vec) {
#pragma unroll
                  for (int e = 0; e < SIZE / 2; e++) u[i].v[e] = __ldg(reinterpret_cast<const uint4*>(src + d) + e);
                } else {
#pragma unroll
                  for (int e = 0; e < 8; e++) u[i].x[e] = src[d + e];
                }
                if (tab >= 0) {
                  const float *ct = a.rope.cos + tab + d / 2, *st = a.rope.sin + tab + d / 2;
                  if (rope_vec) {
                    cs[i] = __ldg(reinterpret_cast<const float4*>(ct));
                    sn[i] = __ldg(reinterpret_cast<const float4*>(st));
                  } else {
                    cs[i] = make_float4(__ldg(ct), __ldg(ct + 1), __ldg(ct + 2), __ldg(ct + 3));
                    sn[i] = make_float4(__ldg(st), __ldg(st + 1), __ldg(st + 2), __ldg(st + 3));
                  }
                }
              }
            }
          };
          const int row0 = (warp & 3) * 32 + (lane >> 3);
          load(row0, u_next, cs_next, sn_next);
#pragma unroll 1
          for (int r0 = 0; r0 < 32 && (warp & 3) * 32 + r0 < rows; r0 += 4) {
#pragma unroll
            for (int i = 0; i < P; i++) {
              u[i] = u_next[i];
              cs[i] = cs_next[i];
              sn[i] = sn_next[i];
            }
            const int r = row0 + r0;
            load(r + 4, u_next, cs_next, sn_next);  // rows past the last read nothing
            float y[P][8], top = 0.0f;
#pragma unroll
            for (int i = 0; i < P; i++) {
              const float cc[4] = {cs[i].x, cs[i].y, cs[i].z, cs[i].w};
              const float ss[4] = {sn[i].x, sn[i].y, sn[i].z, sn[i].w};
#pragma unroll
              for (int e = 0; e < 4; e++) {
                y[i][2 * e] = to_f32<T>(u[i].x[2 * e]);
                y[i][2 * e + 1] = to_f32<T>(u[i].x[2 * e + 1]);
                if (a.rope.cos != nullptr) rotate(y[i][2 * e], y[i][2 * e + 1], cc[e], ss[e]);
                top = fmaxf(top, fmaxf(fabsf(y[i][2 * e]), fabsf(y[i][2 * e + 1])));
              }
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = query_exponent(top);
            const float by = exp2_int(e);
            // to the thread that owns the row
            const float back = __shfl_sync(0xffffffffu, a.scale_log2 * exp2_int(-e), 8 * (lane & 3));
            if (lane / 4 == r0 / 4) row_scale = back;
#pragma unroll
            for (int i = 0; i < P; i++) {
              const int c = (lane & 7) + 8 * i;
              const uint32_t at = tile + (uint32_t)(c >> 3) * HALF * 128u + (uint32_t)r * 128u +
                                  ((((uint32_t)c & 7u) ^ (uint32_t)(r & 7)) << 4);
              float hi[4], lo[4];
#pragma unroll
              for (int k = 0; k < 4; k++) pair2(y[i][2 * k] * by, y[i][2 * k + 1] * by, hi[k], lo[k]);
              sts128(at, make_float4(hi[0], hi[1], hi[2], hi[3]));
              if constexpr (PAIRS) sts128(at + HALF * DH * 2, make_float4(lo[0], lo[1], lo[2], lo[3]));
            }
          }
          fence_async_smem();
          tc_fence_before();
        }
        mbar_arrive(B_(QREADY + t));
        float m = -INFINITY, l = 0.0f;
        int high = 0;  // F
        for (int j = 0; ok && j < nb; j++) {
          const uint32_t at = (n + j) % RING;
          // the exponents are there before the scores, but only these keep in step with a half
          // that had no rows for a while
          ok = wait(SFULL + t, steps);
          if (ok) ok = wait(EXPS + at, (n + j) / RING);
          // no less than the least normal number: 0 times a masked score is NaN
          const int e = exps[2 * at];
          const bool marked = e > kMarked / 2;
          const float scale = fmaxf(times_power(row_scale, e - 6 - (marked ? kMarked : 0)), 0x1p-126f);
          const int now = exps[2 * at + 1], grown = j > 0 ? now - high : 0;
          high = now;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          steps++;
          if (!live) {
            mbar_arrive(B_(PREADY + t));
            continue;
          }
          tc_fence_after();
          uint32_t r[4][32];
#pragma unroll
          for (int c = 0; c < 4; c++) tmem_ld32_nowait(s_at + 32 * c, r[c]);
          tmem_wait_ld_pin<true>(r[0]);
          tmem_wait_ld_pin<false>(r[1]);
          tmem_wait_ld_pin<false>(r[2]);
          tmem_wait_ld_pin<false>(r[3]);
          const int key0 = (p.blk + j) * BK;
          const bool masked = key0 + BK > vis_warp;
          if (masked) {
            const int seen = vis - key0;
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
              for (int i = 0; i < 32; i++)
                if (32 * c + i >= seen) r[c][i] = 0xff800000u;  // -inf
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 4; c++)
#pragma unroll
            for (int i = 0; i < 32; i++) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(r[c][i]));
          const float bmax = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
          const bool jump = bmax > m + kJump || (m == -INFINITY && bmax > -INFINITY);
          float factor = jump ? ex2(m - bmax) : 1.0f;  // 0 while m is -inf
          if (jump) {
            m = bmax;
            l *= factor;
          }
          factor *= ex2((float)-grown);
          // the scores' barrier also says that the last P V is complete
          if constexpr (PAIRS) {
            // the tensor pipe's f32 accumulation truncates: the products of a block are added to
            // the sums here (no slower than one accumulator of many blocks; error of prompts of
            // up to 1,024 tokens 1.0e-6 with eight blocks, 0.6e-6 with one)
            if (j > 0) {
#pragma unroll 1
              for (int c = 0; c < DH; c += 32) {
                float o[32], x[32];
                tmem_ld32(o_at + c, o);
                if (j > 1) {
                  tmem_ld32(sum_at + c, x);
#pragma unroll
                  for (int i = 0; i < 32; i++) o[i] += x[i];
                }
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] *= factor;
                tmem_st32(sum_at + c, o);
              }
              tmem_wait_st();
            }
          } else if (j > 0 && (__any_sync(0xffffffffu, jump) || grown != 0)) {
#pragma unroll
            for (int c = 0; c < DH / 32; c++) {
              float o[32];
              tmem_ld32(o_at + 32 * c, o);
#pragma unroll
              for (int i = 0; i < 32; i++) o[i] *= factor;
              tmem_st32(o_at + 32 * c, o);
            }
          }
          const float from = (m == -INFINITY ? 0.0f : m) - kShift;
          // a quarter of the exponentials on the FMA pipe (as in paged_attention_tc.cu);
          // blocks with masked scores (-inf) or NaN all on the special function unit
          uint64_t sum[2] = {0, 0};
          auto powers = [&](int c, auto some_masked) {
            float w[16];
            [[maybe_unused]] float w_lo[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
              uint64_t x = fma2(pk(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1])),
                                twice(scale), twice(-from));
              if (!PAIRS && !decltype(some_masked)::value && (i & 3) == 3) {
                x = power2(x);
              } else {
                const float2 v = unpk(x);
                x = pk(ex2(v.x), ex2(v.y));
              }
              sum[i & 1] = add2(sum[i & 1], x);
              const float2 v = unpk(x);
              if constexpr (PAIRS) pair2(v.x, v.y, w[i], w_lo[i]);
              else w[i] = __uint_as_float(pack2<__half>(v.x, v.y));
            }
            tmem_st16(s_at + 16 * c, w);
            if constexpr (PAIRS) tmem_st16(s_at + 64 + 16 * c, w_lo);
          };
          if (masked || marked || PAIRS) {
#pragma unroll
            for (int c = 0; c < 4; c++) powers(c, std::true_type{});
          } else {
#pragma unroll
            for (int c = 0; c < 4; c++) powers(c, std::false_type{});
          }
          const float2 all = unpk(add2(sum[0], sum[1]));
          l += all.x + all.y;
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(B_(PREADY + t));
        }
        if (ok) ok = __all_sync(0xffffffffu, wait(ODONE + t, items));
        items++;
        if (ok && live) {
          tc_fence_after();
          const bool done = whole && ends;
          const int h2 = (high - 6) / 2;
          const float f0 = (done ? l > 0.0f ? 1.0f / l : 0.0f : 1.0f) * exp2_int(h2), f1 = exp2_int(high - 6 - h2);
          T* dst = static_cast<T*>(a.o) + (p.r.first + token) * a.o_stride + (int64_t)head * dim;
          const int slot = 2 * (int)blockIdx.x + (whole ? 1 : 0), r = HALF * t + row;
          float* part = a.joint.sums + ((int64_t)slot * TILE + r) * DH;
#pragma unroll 1
          for (int c = 0; c < DH; c += 32) {
            float o[32];
            __syncwarp();
            tmem_ld32(o_at + c, o);
            if (PAIRS && nb > 1) {
              float x[32];
              tmem_ld32(sum_at + c, x);
#pragma unroll
              for (int i = 0; i < 32; i++) o[i] += x[i];
            }
            if (!valid) continue;
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] = o[i] * f0 * f1;
            if (done) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                if (c + i >= dim) break;
                union { uint4 v[SIZE / 2]; T x[8]; } u;
#pragma unroll
                for (int k = 0; k < 8; k++) u.x[k] = from_f32<T>(o[i + k]);
                if (o_vec) {
#pragma unroll
                  for (int k = 0; k < SIZE / 2; k++) reinterpret_cast<uint4*>(dst + c + i)[k] = u.v[k];
                } else {
#pragma unroll
                  for (int k = 0; k < 8; k++) dst[c + i + k] = u.x[k];
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<float4*>(part + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
          }
          if (valid) {
            if (!done) {
              a.joint.stats[(int64_t)slot * 2 * TILE + r] = m - kShift;
              a.joint.stats[((int64_t)slot * 2 + 1) * TILE + r] = l;
            } else if (a.lse != nullptr) {
              a.lse[(p.r.first + token) * a.q_heads + head] = l > 0.0f ? (m - kShift) * kLn2 + logf(l) : -INFINITY;
            }
          }
          tc_fence_before();  // O is read before the next tile's QREADY
        }
      }
      n += nb;
      next_tile(nb);
    }
    if (tid == 0) a.joint.cuts[blockIdx.x] = cut;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, L::COLS);
    if (lane == 0) report_abort(a.batch.status, abort);
  }
}

template <typename T, int DH>
int launch_tc8(const et_b200_paged_cache8_v1* c, Attend8Args& x, void* ws, cudaStream_t stream) {
  using L = Layout<DH, sizeof(T) == 4>;
  AttendArgs& a = x.a;
  const int box_rows = (int)(c->page_size < BK ? c->page_size : BK);
  CUtensorMap k_map, v_map;
  if (!scales_copy(c) || !pool8_map(&k_map, c->keys, c, DH, box_rows) ||
      !pool8_map(&v_map, c->values, c, DH, box_rows))
    return 0;
  constexpr int TILE = L::HALVES * HALF;
  const int blocks = thread_blocks(a, a.sms, TILE, BK);
  a.tiling = tiling_of(L::HALVES == 2 ? 8 : 7, 7, a.tiling.group, a.pools.kv_heads);
  static_assert(HALF == 1 << 7 && BK == 1 << 7, "tiling");
  a.least = 2;
  a.joint = joint_of(ws, blocks, TILE, DH);
  cudaFuncSetAttribute(paged_attention8_tc_kernel<T, DH>,
                       cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
  paged_attention8_tc_kernel<T, DH><<<blocks, THREADS, L::SMEM, stream>>>(k_map, v_map, x, box_rows);
  count_launch();
  return blocks;
}

}  // namespace

namespace paged {

int attend8_tc(const et_b200_paged_cache8_v1* c, Attend8Args& x, void* ws, cudaStream_t stream) {
  if (c->head_dim > 128) return 0;
  if (c->dtype == ET_B200_DTYPE_F32)
    return c->head_dim <= 64 ? launch_tc8<float, 64>(c, x, ws, stream)
                             : launch_tc8<float, 128>(c, x, ws, stream);
  if (c->dtype == ET_B200_DTYPE_F16)
    return c->head_dim <= 64 ? launch_tc8<__half, 64>(c, x, ws, stream)
                             : launch_tc8<__half, 128>(c, x, ws, stream);
  return c->head_dim <= 64 ? launch_tc8<__nv_bfloat16, 64>(c, x, ws, stream)
                           : launch_tc8<__nv_bfloat16, 128>(c, x, ws, stream);
}

}  // namespace paged
}  // namespace etb
