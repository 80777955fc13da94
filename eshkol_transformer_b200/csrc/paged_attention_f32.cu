// Attention of chunks of new tokens over a paged f32 cache on tcgen05:
// head_dim up to 128, pages of a power of two of at least 8 slots.
//
// The mathematics and the division of the work are those of
// paged_attention.cu; operands are binary16 pairs x 2^e = hi + lo (22
// significant bits) and every product is hi hi + hi lo + lo hi, as in the dense
// attention (attention_f16.cu).  The exponents are per row: of a query (a
// constant of its thread), of a key (a factor of its column of scores), and of
// a value row, which moves into the weight: with v_j = v^_j 2^g_j,
//   o = sum_j 2^(s_j + g_j - M) v^_j / sum_j 2^(s_j + g_j - M) 2^-g_j,
// M the running maximum of s_j + g_j, so cached rows of any magnitude need no
// pass of their own.  Where values of 2^24 and more stand beside far smaller ones,
// a key whose 2^(s_j + g_j - M) is flushed to zero may still have a share of the
// denominator: such keys are added to it by themselves (kFar below).
//
// A tile is 128 rows (TMEM lanes), a block 64 keys.  One warp copies raw K and V
// tiles by TMA, two teams of four warps turn them into pairs (a row by all lanes of
// a warp: maximum, exponent, split) in shared memory, a team for K and one for V: K's
// slot is free again when its scores are done, V's when its P V is, so the next
// scores never wait for a conversion.  One warp issues S = Q K^T up to a block ahead
// of another one's O += P V, and 2 threads per row (4 at more than 64 dims) form
// the probabilities, whose pair replaces the scores in TMEM.  A single warp per
// scheduler issues an instruction of such code every five or six cycles, so both
// kinds of arithmetic have at least two.  P hi times [V hi | V lo] is one product of
// N = 2 head_dim; the halves of O are added when it is read.  The tensor pipe's f32
// accumulation truncates, so every CHUNK blocks O moves to f32 sums in the
// workspace.
// Four ragged prompts of up to 1,024 tokens (16 heads x 64) take 96 to 102 us by
// machine (307 us on mma.sync), the same with 9,000 keys of history 600 us.  3,000 to
// 3,500 cycles per block of 64 keys and 11,000 per tile for its queries and output:
// instructions bound it, and their cache, which the roles' code together overflows
// (100 KB; 8 % of its requests miss), so what runs seldom or waits anyway is not
// unrolled, and a few instructions more or less move the time by some per cent.
// Waits are bounded as in paged_attention_tc.cu.
#include <math.h>

#include <type_traits>

#include "attention_f16.cuh"
#include "paged.cuh"

namespace etb {
namespace {

using namespace paged;
using namespace f16att;

constexpr int ROWS = 128, BK = 64;
constexpr int TEAM = 4;  // warps that convert K, and as many for V
constexpr float kJump = 8.0f;   // log2 of the largest P the standing maximum allows
constexpr float kShift = 7.0f;  // P carries 2^7: at most 2^15
constexpr int CHUNK = 8;        // blocks whose products one TMEM accumulator adds

template <int DH>
struct Layout {
  static constexpr int PARTS = DH / 32, KEYS = BK / PARTS;  // threads of a row, keys of one
  static constexpr int SOFT = ROWS * PARTS, CONVERT_WARP = SOFT / 32, MMA_WARP = CONVERT_WARP + 2 * TEAM,
                       LOAD_WARP = MMA_WARP + 2, THREADS = 32 * (MMA_WARP + 4);
  // registers of the warpgroups: probabilities, conversion, the rest
  static constexpr int REGS = DH == 128 ? 72 : 96, SOFT_REGS = DH == 128 ? 88 : 136,
                       CONVERT_REGS = DH == 128 ? 56 : 72, LEAN_REGS = DH == 128 ? 40 : 48;
  static_assert(SOFT * SOFT_REGS + 256 * CONVERT_REGS + 128 * LEAN_REGS <= THREADS * REGS &&
                    THREADS * REGS <= 65536, "registers at launch");
  static constexpr int RAW = BK * DH * 4;             // one raw tile of K or V
  static constexpr int RAWS = DH == 128 ? 2 : 6;      // tiles in the ring: K, V, K, V, ...
  static constexpr int KT = BK * DH * 2;              // one binary16 tile
  static constexpr int PAIR = 2 * KT;                 // hi, lo
  static constexpr int VS = DH == 128 ? 2 : 3;        // slots of V (of K: 2)
  static constexpr int KP = RAWS * RAW, VP = KP + 2 * PAIR;
  static constexpr int QLO = VP + VS * PAIR;
  static constexpr int V_FACTORS = QLO + ROWS * DH * 2;     // [VS][2][BK]: exponents and factors
  static constexpr int K_FACTORS = V_FACTORS + VS * 2 * BK * 4;  // [3][BK]
  static constexpr int V_LEAST = K_FACTORS + 3 * BK * 4;      // [VS][TEAM]: least exponents so far
  static constexpr int SHARED_ROWS = V_LEAST + VS * TEAM * 4;  // [2][ROWS]: what a row's threads exchange
  static constexpr int BARS = SHARED_ROWS + 2 * ROWS * 4;
  static constexpr int SMEM = BARS + 8 * (2 * RAWS + 2 * VS + 13) + 8;
  static constexpr uint32_t S0 = 0, QH = 128, O = 192, COLS = 512;
  static_assert(O + 2 * DH <= COLS && QH + DH / 2 <= O && SMEM <= 232448, "TMEM and shared memory");
};

// e with 2^13 <= amax 2^e < 2^14; `most` for a row of zeros (any e describes it,
// and a large one keeps it out of the maximum) and for rows below 2^(13 - most).
__device__ __forceinline__ int row_exponent(float amax, int most = 100) {
  return min(most, 13 - ((int)(__float_as_uint(amax) >> 23) - 127));
}
// Of values: a key adds at most 2^(kShift + kJump + 80) to its row's sum of weights,
// so 2^31 keys stay inside f32.
constexpr int kMostOfV = 80;
// A weight 2^(s_j + g_j - M + kShift) that f32 flushes to zero adds nothing to the
// numerator, but 2^-g_j of it belongs to the sum of weights.  Beside the row k that
// M stands for it is below 2^(-133 - g_j + g_k), so below 2^-44 while g_k < 10 (values
// under 2^24); from there on (kFar: exponents e = -g) such keys are added by themselves.
constexpr int kFar = -10;

__device__ __forceinline__ float tmem_ld1(uint32_t addr) {
  uint32_t v;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(v) : "r"(addr) : "memory");
  return __uint_as_float(v);
}

// A float's bits in an order of integers, and back.
__device__ __forceinline__ int ordered_bits(float x) {
  const int i = __float_as_int(x);
  return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float from_ordered(int i) {
  return __int_as_float(i ^ ((i >> 31) & 0x7fffffff));
}

template <int DH>
__global__ void __launch_bounds__(Layout<DH>::THREADS, 1)
paged_attention_f32_kernel(const __grid_constant__ CUtensorMap k_map,
                           const __grid_constant__ CUtensorMap v_map, AttendArgs a, int box_rows) {
  using L = Layout<DH>;
  constexpr int CONVERT_WARP = L::CONVERT_WARP, MMA_WARP = L::MMA_WARP;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* v_factors = reinterpret_cast<float*>(smem + L::V_FACTORS);
  float* k_factors = reinterpret_cast<float*>(smem + L::K_FACTORS);
  int* v_least = reinterpret_cast<int*>(smem + L::V_LEAST);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  enum {
    RAWFULL = 0, RAWEMPTY = L::RAWS, KFULL = 2 * L::RAWS, VFULL = KFULL + 3, SFULL = VFULL + L::VS,
    PREADY = SFULL + 2, PVDONE = PREADY + 2, KFREE = PVDONE + L::VS, QREADY = KFREE + 3,
    DRAIN = QREADY + 1, NBARS = DRAIN + 2
  };
  const uint32_t bar0 = smem_u32(bars);
  auto B_ = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + NBARS);
  int* abort_word = reinterpret_cast<int*>(tslot + 1);
  volatile int* abort = abort_word;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_u32(smem);
  const int group = a.tiling.group, dim = a.pools.head_dim;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (tid == 0) {
    for (int i = 0; i < NBARS; i++)
      mbar_init(B_(i), (i >= RAWEMPTY && i < SFULL) ? TEAM
                       : (i >= KFREE && i < QREADY) ? CONVERT_WARP
                       : (i == PREADY || i == PREADY + 1 || i == QREADY) ? L::SOFT : 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) tmem_alloc(smem_u32(tslot), L::COLS);
  Place p;
  const Share share = divide(a.tiling, a.batch, a.least, p,
                             *reinterpret_cast<DivideRoom<L::THREADS>*>(smem + L::QLO));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  int64_t left = share.units;
  auto blocks_here = [&]() { return (int)min((int64_t)(p.nblk - p.blk), left); };
  auto next_tile = [&](int done) {
    left -= done;
    p.blk += done - 1;
    advance(a.tiling, a.batch, p);
  };
  auto wait = [&](int i, uint32_t parity) {
    return role_wait(B_(i), parity & 1u, abort_word, abort);
  };
  auto pv_done = [&](uint32_t block) { return PVDONE + (int)(block % L::VS); };
  uint32_t n = 0;  // blocks so far, of all tiles: slot n & 1, round n >> 1

  if (warp >= MMA_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::LEAN_REGS));
  if (warp == L::LOAD_WARP) {
    // ---- raw tiles, page by page
    uint32_t count = 0;
    bool ok = true;
    while (ok && left > 0) {
      const int nb = blocks_here(), visible = tile_visible(a.tiling, p.r, p.tile);
      for (int j = 0; ok && j < nb; j++) {
        const int key0 = (p.blk + j) * BK;
        const int boxes = max(0, (min(visible - key0, BK) + box_rows - 1) / box_rows);  // at most 8
        int page = -1, slot = 0;
        if (lane < boxes) {
          const int key = key0 + lane * box_rows, column = quotient(key, a.pools.by_page);
          slot = key - column * a.pools.page_size;
          page = a.batch.table[(int64_t)p.b * a.batch.columns + column];
          if (page < 0 || page >= a.pools.pages) {
            report(a.batch.status, ET_B200_PAGED_BAD_PAGE);
            page = -1;  // outside the map: filled with zeros
          }
        }
#pragma unroll 1
        for (int kv = 0; kv < 2; kv++) {
          const uint32_t s = count % L::RAWS, round = count / L::RAWS;
          if (ok && round > 0) ok = wait(RAWEMPTY + s, round - 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(B_(RAWFULL + s), (uint32_t)(boxes * box_rows * DH * 4));
          __syncwarp();
          if (lane < boxes)
            tma_load_4d(base + s * L::RAW + (uint32_t)(lane * box_rows) * DH * 4u,
                        kv == 0 ? &k_map : &v_map, B_(RAWFULL + s), 0, slot, p.h, page);
          count++;
        }
      }
      next_tile(nb);
    }
    // every copy has landed before the CTA releases its memory
    if (lane == 0)
      for (uint32_t c = count > L::RAWS ? count - L::RAWS : 0; c < count; c++)
        mbar_wait(B_(RAWFULL + c % L::RAWS), (c / L::RAWS) & 1u, abort_word);
  } else if (warp == MMA_WARP) {
    // ---- S = Q K^T, up to a block ahead of P V
    constexpr uint32_t idesc_s = idesc_f16_m128(BK, 0);
    uint32_t items = 0;
    bool ok = true;
    while (ok && left > 0) {
      const int nb = blocks_here();
      ok = wait(QREADY, items++);
      for (int j = 0; j < nb; j++, n++) {
        const uint32_t slot = n & 1u;
        if (ok) ok = wait(KFULL + n % 3u, n / 3u);
        if (ok && n >= 2) ok = wait(pv_done(n - 2), (n - 2) / L::VS);  // the slot held P of block n - 2
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t k = base + L::KP + slot * L::PAIR, d = tmem + L::S0 + 64u * slot;
#pragma unroll 1
          for (int i = 0; i < DH / 16; i++) {
            const uint64_t kh = kdesc16<BK>(k, i);
            umma_f16(d, kdesc16<ROWS>(base + L::QLO, i), kh, idesc_s, i > 0 ? 1u : 0u);
            umma_f16_ts(d, tmem + L::QH + 8u * i, kdesc16<BK>(k + L::KT, i), idesc_s, 1u);
            umma_f16_ts(d, tmem + L::QH + 8u * i, kh, idesc_s, 1u);
          }
          umma_commit(B_(SFULL + (int)slot));
        }
      }
      next_tile(nb);
    }
    if (lane == 0) {
      umma_commit(B_(DRAIN));
      mbar_wait(B_(DRAIN), 0u, abort_word);
    }
  } else if (warp == MMA_WARP + 1) {
    // ---- O += P V
    constexpr uint32_t idesc_o = idesc_f16_m128(DH, 1), idesc_o2 = idesc_f16_m128(2 * DH, 1);
    bool ok = true;
    while (ok && left > 0) {
      const int nb = blocks_here();
      for (int j = 0; j < nb; j++, n++) {
        const uint32_t slot = n & 1u;
        ok = __all_sync(0xffffffffu, wait(PREADY + slot, n >> 1));
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t v = base + L::VP + n % L::VS * L::PAIR;
          const uint32_t pa = tmem + L::S0 + 64u * slot;
#pragma unroll 1
          for (int i = 0; i < BK / 16; i++) {
            const uint64_t vd = mdesc16<BK>(v, i);  // V lo lies one chunk stride behind V hi
            const uint32_t hi = pa + 16u * i;
            umma_f16_ts(tmem + L::O, hi, vd, idesc_o2, (j % CHUNK != 0 || i > 0) ? 1u : 0u);
            umma_f16_ts(tmem + L::O, hi + 8u, vd, idesc_o, 1u);
          }
          umma_commit(B_(pv_done(n)));
        }
      }
      next_tile(nb);
    }
    if (lane == 0) {
      umma_commit(B_(DRAIN + 1));
      mbar_wait(B_(DRAIN + 1), 0u, abort_word);
    }
  }
  } else if (warp >= CONVERT_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::CONVERT_REGS));
    // ---- raw rows into pairs: a team of warps for K, one for V; a warp takes 16
    // rows, a row at a time all its lanes.  A slot of K is free once its scores are
    // done, one of V once its P V is.  The factors of K outlive their slot by the
    // probabilities, so they have three.
    constexpr int W = DH / 32, AT_ONCE = DH == 64 ? 8 : 4;  // dims of a lane, rows at once
    const int kv = (warp - CONVERT_WARP) / TEAM, row0 = 16 * ((warp - CONVERT_WARP) % TEAM);
    const int most = kv == 0 ? 100 : kMostOfV;
    bool ok = true;
    while (ok && left > 0) {
      const int nb = blocks_here(), visible = tile_visible(a.tiling, p.r, p.tile);
      int least = most;  // exponent of this warp's rows of the tile so far
#pragma unroll 1
      for (int j = 0; j < nb; j++, n++) {
        const int valid = visible - (p.blk + j) * BK;
        const uint32_t s = (2 * n + kv) % L::RAWS, third = n % 3u;
        const uint32_t v_slot = n % L::VS;
        const uint32_t conv = base + (kv == 0 ? L::KP + (n & 1u) * L::PAIR : L::VP + v_slot * L::PAIR);
        if (kv == 0) {
          if (n >= 2) ok = wait(SFULL + (n & 1u), (n >> 1) - 1);
          if (ok && n >= 3) ok = wait(KFREE + third, n / 3u - 1);
        } else if (n >= L::VS) {
          ok = wait(PVDONE + v_slot, n / L::VS - 1);
        }
        if (ok) ok = wait(RAWFULL + s, (2 * n + kv) / L::RAWS);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        // AT_ONCE rows at a time: loads, then maxima, then stores
        const uint32_t raw = base + s * L::RAW + (uint32_t)(row0 * DH + W * lane) * 4u;
        const uint32_t to = conv + (uint32_t)(lane * W / 64) * BK * 128u + (uint32_t)row0 * 128u;
        int mine = 0;  // exponent of row row0 + lane
#pragma unroll 1
        for (int r0 = 0; r0 < 16; r0 += AT_ONCE) {
          float2 x[AT_ONCE][W / 2];
          uint32_t m[AT_ONCE];
#pragma unroll
          for (int k = 0; k < AT_ONCE; k++) {
            const uint32_t from = raw + (uint32_t)((r0 + k) * DH) * 4u;
            if constexpr (W == 4) {
              const float4 y = lds128(from);
              x[k][0] = make_float2(y.x, y.y);
              x[k][1] = make_float2(y.z, y.w);
            } else {
              asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(x[k][0].x), "=f"(x[k][0].y) : "r"(from) : "memory");
            }
            if (row0 + r0 + k >= valid)  // slots behind may hold anything
#pragma unroll
              for (int i = 0; i < W / 2; i++) x[k][i] = make_float2(0.f, 0.f);
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < W / 2; i++) top = fmaxf(top, fmaxf(fabsf(x[k][i].x), fabsf(x[k][i].y)));
            m[k] = __float_as_uint(top);
          }
#pragma unroll
          for (int k = 0; k < AT_ONCE; k++) m[k] = __reduce_max_sync(0xffffffffu, m[k]);
#pragma unroll
          for (int k = 0; k < AT_ONCE; k++) {
            const int r = r0 + k, e = row_exponent(__uint_as_float(m[k]), most);
            const uint64_t sc = twice(exp2_int(e));
            mine = lane == r ? e : mine;
            uint32_t hi[W / 2], lo[W / 2];
#pragma unroll
            for (int i = 0; i < W / 2; i++) {
              const uint64_t y = mul2(pk(x[k][i].x, x[k][i].y), sc);
              const float2 f = unpk(y);
              const __half2 h = __floats2half2_rn(f.x, f.y);
              const float2 hf = __half22float2(h), rest = unpk(fma2(pk(hf.x, hf.y), twice(-1.0f), y));
              const __half2 l = __floats2half2_rn(rest.x, rest.y);
              hi[i] = *reinterpret_cast<const uint32_t*>(&h);
              lo[i] = *reinterpret_cast<const uint32_t*>(&l);
            }
            // byte 2 W lane of the row's 128 (of each 64 dims), 16-byte pieces swizzled
            const uint32_t byte = 2u * W * ((uint32_t)lane % (64 / W)), at = to + 128u * r + (byte ^ (uint32_t)((AT_ONCE == 8 ? k : r & 7) << 4));
            if constexpr (W == 4) {
              asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(hi[0]), "r"(hi[W / 2 - 1]) : "memory");
              asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + L::KT), "r"(lo[0]), "r"(lo[W / 2 - 1]) : "memory");
            } else {
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(hi[0]) : "memory");
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + L::KT), "r"(lo[0]) : "memory");
            }
          }
        }
        if (lane < 16) {
          if (kv == 0) {
            k_factors[third * BK + row0 + lane] = exp2_int(-mine);
          } else {
            float* f = v_factors + v_slot * 2 * BK + row0 + lane;
            f[0] = (float)-mine;
            f[BK] = exp2_int(mine);
          }
        }
        if (kv == 1) {
          least = min(least, __reduce_min_sync(0xffffffffu, lane < 16 ? mine : most));
          if (lane == 0) v_least[v_slot * TEAM + row0 / 16] = least;
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(B_(RAWEMPTY + s));
          mbar_arrive(B_(kv == 0 ? KFULL + third : VFULL + v_slot));
        }
      }
      next_tile(nb);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::SOFT_REGS));
    // ---- probabilities: thread `which` of a row takes keys KEYS which .. of a block
    constexpr int PARTS = L::PARTS, KEYS = L::KEYS;
    const int quarter = warp & 3, which = warp >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t o_at = lanes + L::O;
    uint8_t* q_lo = smem + L::QLO;
    uint8_t* shared_rows = smem + L::SHARED_ROWS;
    int* row_max = reinterpret_cast<int*>(shared_rows);        // [2][ROWS], of ordered_bits
    float* row_value = reinterpret_cast<float*>(shared_rows);  // [ROWS], before a tile
    // behind a tile the memory of a quarter's queries passes on its row sums
    // [PARTS][32], then its output, 16 columns of 32 rows per warp at a time
    float* row_sums = reinterpret_cast<float*>(q_lo + quarter * 4096);
    const uint32_t stage = smem_u32(q_lo + (which >> 1) * ROWS * 128 + quarter * 4096 + (which & 1) * 2048);
    auto row_sync = [&]() { named_sync(1 + quarter, 32 * PARTS); };
    const bool q_vec = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * 4)) & 15) == 0;
    const bool rope_vec = ((reinterpret_cast<uintptr_t>(a.rope.cos) | reinterpret_cast<uintptr_t>(a.rope.sin)) & 7) == 0;
    const bool o_vec = ((reinterpret_cast<uintptr_t>(a.o) | (uintptr_t)(a.o_stride * 4)) & 15) == 0;
    bool ok = true;
    Cut cut{0, 0, 0, 0, 0};
    // after a wait that ran out the loops still end, in step with the other threads
    // of the row
    while (left > 0) {
      const int nb = blocks_here(), rows = min(ROWS, p.r.n * group - p.tile * ROWS);
      const bool whole = p.blk == 0, ends = p.blk + nb == p.nblk, done = whole && ends;
      if (whole && !ends) {
        const int64_t rest = p.nblk - nb;
        cut = Cut{p.r.first, p.r.n, p.h, p.tile, 1 + (int)((rest + share.per - 1) / share.per)};
      }
      const int g = p.tile * ROWS + row;
      const bool valid = row < rows;
      const int token = quotient(g, a.tiling.by_group), head = p.h * group + g - token * group;
      const int pos = p.r.len - p.r.n + token, vis = valid ? max(0, pos + 1) : 0;
      const int vis_warp = __shfl_sync(0xffffffffu, max(0, pos + 1), 0);
      float cq = 0.0f;
      // ---- the warp's rows of Q, rotated: 8 lanes a row, whole lines.  hi passes
      // through the tile of lo on its way into TMEM (a row per lane), then lo takes
      // the tile.
      {
        constexpr int P = DH / 32;  // 16-byte pieces of a lane
        const uint32_t tile = smem_u32(q_lo);
        constexpr int FOURS = 32 / PARTS / 4, G = DH == 128 ? 1 : FOURS;  // groups of 4 rows; in flight
        const int own = quarter * 32 + which * (32 / PARTS) + (lane >> 3);    // this lane's row of the first
        auto unit_at = [&](int r, int i) {
          const int c = (lane & 7) + 8 * i;  // 8-byte unit of the row
          return tile + (uint32_t)(c >> 4) * ROWS * 128u + (uint32_t)r * 128u +
                 (((((uint32_t)c & 15u) >> 1) ^ (uint32_t)(r & 7)) << 4) + (uint32_t)(c & 1) * 8u;
        };
        float low[FOURS][P][2];
#pragma unroll
        for (int g0 = 0; g0 < FOURS; g0 += G) {
          // all loads first: rows and dims that are not there read the tensor's or
          // the table's beginning
          float4 x[G][P];
          float2 cs[G][P], sn[G][P];
#pragma unroll
          for (int k = 0; k < G; k++) {
            const int r = own + 4 * (g0 + k), gr = p.tile * ROWS + r;
            const int t = quotient(gr, a.tiling.by_group), at_pos = p.r.len - p.r.n + t;
            const float* src = static_cast<const float*>(a.q);
            if (r < rows) src += (p.r.first + t) * a.q_stride + (int64_t)(p.h * group + gr - t * group) * dim;
            const int64_t tab = r < rows && at_pos >= 0 ? min((int64_t)at_pos, a.rope.rows - 1) * (dim / 2) : 0;
#pragma unroll
            for (int i = 0; i < P; i++) {
              const int d = 4 * ((lane & 7) + 8 * i), from = d < dim ? d : 0;
              if (q_vec) x[k][i] = __ldg(reinterpret_cast<const float4*>(src + from));
              else x[k][i] = make_float4(__ldg(src + from), __ldg(src + from + 1), __ldg(src + from + 2), __ldg(src + from + 3));
              if (a.rope.cos != nullptr) {
                const float *ct = a.rope.cos + tab + from / 2, *st = a.rope.sin + tab + from / 2;
                if (rope_vec) {
                  cs[k][i] = __ldg(reinterpret_cast<const float2*>(ct));
                  sn[k][i] = __ldg(reinterpret_cast<const float2*>(st));
                } else {
                  cs[k][i] = make_float2(__ldg(ct), __ldg(ct + 1));
                  sn[k][i] = make_float2(__ldg(st), __ldg(st + 1));
                }
              }
            }
          }
#pragma unroll
          for (int k = 0; k < G; k++) {
            const int r = own + 4 * (g0 + k);
            const int at_pos = p.r.len - p.r.n + quotient(p.tile * ROWS + r, a.tiling.by_group);
            const bool turned = r < rows && at_pos >= 0 && a.rope.cos != nullptr;
            if (turned && at_pos >= a.rope.rows) report(a.batch.status, ET_B200_PAGED_BAD_ROPE);
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < P; i++) {
              if (r >= rows || 4 * ((lane & 7) + 8 * i) >= dim) x[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
              m = abs_max4(m, x[k][i]);
            }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            // a rotated pair is at most sqrt(2) times its larger element: below 2^14.5
            const int e = row_exponent(m);
            const float sc = exp2_int(e);
            if ((lane & 7) == 0) row_value[r] = a.scale_log2 * exp2_int(-e);
#pragma unroll
            for (int i = 0; i < P; i++) {
              float4 v = x[k][i];
              if (turned) {
                rotate(v.x, v.y, cs[k][i].x, sn[k][i].x);
                rotate(v.z, v.w, cs[k][i].y, sn[k][i].y);
              }
              float h0, h1;
              pair2(v.x * sc, v.y * sc, h0, low[g0 + k][i][0]);
              pair2(v.z * sc, v.w * sc, h1, low[g0 + k][i][1]);
              asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(unit_at(r, i)), "f"(h0), "f"(h1) : "memory");
            }
          }
        }
        // hi is complete: this thread's 16 columns of its row
        row_sync();
        cq = row_value[row];
        static_assert(16 * PARTS == DH / 2, "columns of a thread");
        {
          float v[16];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t u = 4u * which + (uint32_t)i;
            const float4 f = lds128(tile + (u >> 3) * ROWS * 128u + (uint32_t)row * 128u +
                                    (((u & 7u) ^ (uint32_t)(row & 7)) << 4));
            v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
          }
          tmem_st16(lanes + L::QH + (uint32_t)(16 * which), v);
        }
        tmem_wait_st();
        row_sync();
        if (which == 0) row_max[row] = row_max[ROWS + row] = ordered_bits(-INFINITY);
#pragma unroll
        for (int k = 0; k < FOURS; k++)
#pragma unroll
          for (int i = 0; i < P; i++)
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(unit_at(own + 4 * k, i)),
                         "f"(low[k][i][0]), "f"(low[k][i][1]) : "memory");
      }
      {
        fence_async_smem();
        tc_fence_before();
        mbar_arrive(B_(QREADY));
        row_sync();  // row_max is set
      }
      // What leaves TMEM between chunks, 32 columns from o_col of a row per thread:
      // piece by piece, the threads side by side.  (A row per thread in place, every
      // store reaches 32 lines and keeps the other warps from shared memory.)
      constexpr int SIDE = 4 * ROWS * PARTS;
      float* scratch = a.joint.stats + (int64_t)gridDim.x * 4 * ROWS +
                       (int64_t)blockIdx.x * ROWS * DH + 4 * (which * ROWS + row);
      float m = -INFINITY, l = 0.0f, m_part = -INFINITY, most = -INFINITY;
      bool have_part = false;
      static_assert(DH / PARTS == 32, "columns of a thread");
      const int o_col = 32 * which;
      // O so far, relative to m, with what the scratch holds
      auto read_o = [&](float (&v)[32]) {
        float v2[32];
        tmem_ld32(o_at + (uint32_t)o_col, v);
        tmem_ld32(o_at + (uint32_t)(DH + o_col), v2);
        const float f = have_part ? ex2(m_part - (m == -INFINITY ? 0.0f : m)) : 0.0f;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          if (have_part) y = *reinterpret_cast<const float4*>(scratch + i / 4 * SIDE);
          v[i] = (v[i] + v2[i]) + f * y.x;
          v[i + 1] = (v[i + 1] + v2[i + 1]) + f * y.y;
          v[i + 2] = (v[i + 2] + v2[i + 2]) + f * y.z;
          v[i + 3] = (v[i + 3] + v2[i + 3]) + f * y.w;
        }
      };
      for (int j = 0; j < nb; j++, n++) {
        if (j > 0 && j % CHUNK == 0) {  // move O out: the next product starts a new accumulator
          if (ok) ok = __all_sync(0xffffffffu, wait(pv_done(n - 1), (n - 1) / L::VS));
          tc_fence_after();
          float v[32];
          read_o(v);
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(scratch + i / 4 * SIDE) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          have_part = true;
          m_part = m == -INFINITY ? 0.0f : m;
        }
        if (ok) ok = wait(KFULL + n % 3u, n / 3u) && wait(VFULL + n % L::VS, n / L::VS);  // the factors
        if (ok) ok = wait(SFULL + (n & 1u), n >> 1);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        const uint32_t s_at = lanes + L::S0 + 64u * (n & 1u);
        const int key0 = (p.blk + j) * BK;
        const bool masked = key0 + BK > vis_warp;
        const int seen = vis - key0 - KEYS * which;
        const uint32_t kf_at = smem_u32(k_factors + n % 3u * BK + KEYS * which);
        const uint32_t vf_at = smem_u32(v_factors + n % L::VS * 2 * BK + KEYS * which);
        // this thread's scores in base 2, exponents of their values added
        uint64_t s2[KEYS / 2];
        {
          const uint64_t cq2 = twice(cq);
#pragma unroll
          for (int h = 0; h < KEYS; h += 16) {
            float s[16];
            tmem_ld16(s_at + (uint32_t)(KEYS * which + h), s);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 kf = lds128(kf_at + 4u * (h + i)), ge = lds128(vf_at + 4u * (h + i));
              s2[(h + i) / 2] = fma2(mul2(pk(s[i], s[i + 1]), cq2), pk(kf.x, kf.y), pk(ge.x, ge.y));
              s2[(h + i) / 2 + 1] = fma2(mul2(pk(s[i + 2], s[i + 3]), cq2), pk(kf.z, kf.w), pk(ge.z, ge.w));
            }
          }
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < KEYS / 2; i++) {
            const float2 v = unpk(s2[i]);
            s2[i] = pk(2 * i >= seen ? -INFINITY : v.x, 2 * i + 1 >= seen ? -INFINITY : v.y);
          }
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < KEYS / 2; i++) {
          const float2 v = unpk(s2[i]);
          top[i & 3] = fmaxf(top[i & 3], fmaxf(v.x, v.y));
        }
        // the row's maximum over its threads, in f32: probabilities relative to a
        // bound above it would leave binary16.  Each thread adds the largest of all
        // its blocks so far to one of two places in turn, so what block n - 2 left
        // there is no larger than block n's; block n - 1's is in the other, and who
        // reads that is here before anyone writes it again.
        most = fmaxf(most, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
        int* shared_max = row_max + (n & 1u) * ROWS + row;
        atomicMax(shared_max, ordered_bits(most));
        row_sync();
        const float bmax = from_ordered(*reinterpret_cast<volatile int*>(shared_max));
        const bool jump = bmax > m + kJump;
        const int4 far_v = *reinterpret_cast<const int4*>(v_least + n % L::VS * TEAM);
        const bool far = min(min(far_v.x, far_v.y), min(far_v.z, far_v.w)) <= kFar;
        if (__any_sync(0xffffffffu, jump || far)) {
          const float factor = jump ? ex2(m - bmax) : 1.0f;  // 0 while m is -inf
          if (jump) {
            l = scaled(l, m - bmax);
            m = bmax;
          }
          if (j % CHUNK != 0) {  // O holds products of this chunk: rescale it once they are complete
            if (ok) ok = __all_sync(0xffffffffu, wait(pv_done(n - 1), (n - 1) / L::VS));
            tc_fence_after();
#pragma unroll 1
            for (int c = 2 * which; c < 2 * which + 2; c++) {
              float o[32];
              tmem_ld32(o_at + 32u * c, o);
#pragma unroll
              for (int i = 0; i < 32; i++) o[i] *= factor;
              tmem_st32(o_at + 32u * c, o);
            }
          }
          if (far) {  // the sum of weights of the keys that the loop below flushes to zero
            const float* kf = k_factors + n % 3u * BK + KEYS * which;
            const float* ge = v_factors + n % L::VS * 2 * BK + KEYS * which;
            const float below = (m == -INFINITY ? 0.0f : m) - kShift;
#pragma unroll 1
            for (int i = 0; i < KEYS; i++) {
              const float x = fmaf(tmem_ld1(s_at + (uint32_t)(KEYS * which + i)) * cq, kf[i], ge[i]) - below;
              if (i < seen && x < -126.0f) l += ex2(x - ge[i]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(B_(KFREE + n % 3u));
        const float from = (m == -INFINITY ? 0.0f : m) - kShift;
        uint64_t sum2[2] = {0, 0};
        const uint64_t from2 = twice(-from);
#pragma unroll
        for (int h = 0; h < KEYS; h += 16) {
          float pair[16];  // hi of 16 keys, then lo
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float4 vf = lds128(vf_at + 4u * (BK + h + 2 * i));
#pragma unroll
            for (int k = 0; k < 2; k++) {
              const float2 x = unpk(add2(s2[h / 2 + i + k], from2));
              const uint64_t w = pk(ex2(x.x), ex2(x.y));
              sum2[k] = fma2(w, k == 0 ? pk(vf.x, vf.y) : pk(vf.z, vf.w), sum2[k]);
              const float2 w2 = unpk(w);
              const __half2 h2 = __floats2half2_rn(w2.x, w2.y);
              const float2 hf = __half22float2(h2), rest = unpk(add2(w, pk(-hf.x, -hf.y)));
              const __half2 l2 = __floats2half2_rn(rest.x, rest.y);
              pair[i + k] = __uint_as_float(*reinterpret_cast<const uint32_t*>(&h2));
              pair[8 + i + k] = __uint_as_float(*reinterpret_cast<const uint32_t*>(&l2));
            }
          }
          tmem_st16(s_at + (uint32_t)(KEYS * which + h), pair);  // over these keys' scores
        }
        const float2 all = unpk(add2(sum2[0], sum2[1]));
        l += all.x + all.y;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(B_(PREADY + (n & 1u)));
      }
      // the row's sum, over the queries: the scores are done with them
      row_sums[which * 32 + lane] = l;
      row_sync();
      l = 0.0f;
#pragma unroll
      for (int i = 0; i < PARTS; i++) l += row_sums[i * 32 + lane];
      row_sync();  // read before the outputs are written there
      if (ok) ok = __all_sync(0xffffffffu, wait(pv_done(n - 1), (n - 1) / L::VS));
      if (ok) {
        tc_fence_after();
        const float inv = !done ? 1.0f : l > 0.0f ? 1.0f / l : 0.0f;
        const int slot = 2 * (int)blockIdx.x + (whole ? 1 : 0);
        float* mine = done ? static_cast<float*>(a.o) + (p.r.first + token) * a.o_stride + (int64_t)head * dim
                           : a.joint.sums + ((int64_t)slot * ROWS + row) * DH;
        float* to[4];  // rows lane / 4 + 8 k of the warp: four lanes write 16 columns of one
#pragma unroll
        for (int k = 0; k < 4; k++)
          to[k] = reinterpret_cast<float*>(
              __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), 8 * k + (lane >> 2)));
        const int width = done ? dim : DH;
        const bool vec = !done || o_vec;
        float o[32];
        read_o(o);
#pragma unroll
        for (int h = 0; h < 32; h += 16) {
#pragma unroll
          for (int i = 0; i < 4; i++)
            sts128(stage + 64u * lane + ((i ^ ((uint32_t)lane >> 1 & 3u)) << 4),
                   make_float4(o[h + 4 * i] * inv, o[h + 4 * i + 1] * inv, o[h + 4 * i + 2] * inv, o[h + 4 * i + 3] * inv));
          __syncwarp();
          const int d = o_col + h + 4 * (lane & 3);
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const uint32_t r = 8u * k + ((uint32_t)lane >> 2);
            const float4 v = lds128(stage + 64u * r + ((((uint32_t)lane & 3u) ^ (r >> 1 & 3u)) << 4));
            if (quarter * 32 + (int)r < rows && d < width) {
              if (vec) {
                *reinterpret_cast<float4*>(to[k] + d) = v;
              } else {
                to[k][d] = v.x;
                to[k][d + 1] = v.y;
                to[k][d + 2] = v.z;
                to[k][d + 3] = v.w;
              }
            }
          }
          __syncwarp();
        }
        if (valid && which == 0) {
          // weights are relative to m - kShift
          if (!done) {
            a.joint.stats[(int64_t)slot * 2 * ROWS + row] = m - kShift;
            a.joint.stats[((int64_t)slot * 2 + 1) * ROWS + row] = l;
          } else if (a.lse != nullptr) {
            a.lse[(p.r.first + token) * a.q_heads + head] =
                l > 0.0f ? (m - kShift) * kLn2 + logf(l) : -INFINITY;
          }
        }
        tc_fence_before();  // O is read before the next tile's QREADY
      }
      row_sync();  // the stage is read before the next tile's queries are written there
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

template <int DH>
int launch_f32(const et_b200_paged_cache_v1* c, AttendArgs& a, void* ws, cudaStream_t stream) {
  using L = Layout<DH>;
  const int box_rows = (int)(c->page_size < BK ? c->page_size : BK);
  CUtensorMap k_map, v_map;
  if (!pool_map(&k_map, c->keys, c, DH, box_rows, false) ||
      !pool_map(&v_map, c->values, c, DH, box_rows, false))
    return 0;
  a.tiling = tiling_of(7, 6, a.tiling.group, a.pools.kv_heads);
  static_assert(ROWS == 1 << 7 && BK == 1 << 6, "tiling");
  const int blocks = thread_blocks(a, a.sms, ROWS, BK);
  a.least = 2;
  a.joint = joint_of(ws, blocks, ROWS, DH);
  cudaFuncSetAttribute(paged_attention_f32_kernel<DH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       L::SMEM);
  paged_attention_f32_kernel<DH><<<blocks, L::THREADS, L::SMEM, stream>>>(k_map, v_map, a, box_rows);
  count_launch();
  return blocks;
}

}  // namespace

namespace paged {

int attend_f32(const et_b200_paged_cache_v1* c, AttendArgs& a, void* ws, cudaStream_t stream) {
  if (c->dtype != ET_B200_DTYPE_F32 || c->head_dim > 128) return 0;
  return c->head_dim <= 64 ? launch_f32<64>(c, a, ws, stream) : launch_f32<128>(c, a, ws, stream);
}

}  // namespace paged
}  // namespace etb
