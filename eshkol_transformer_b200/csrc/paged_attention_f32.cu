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
// pass of their own.
//
// A tile is 128 rows (TMEM lanes), a block 64 keys.  Warp 18 copies raw K and V
// tiles by TMA, warps 8-15 turn them into pairs (a row by DH / 4 lanes: maximum,
// exponent, split) in shared memory, warp 16 issues S = Q K^T up to a block ahead
// of warp 17's O += P V, warps 0-7 (two threads per row, 32 keys each) form the
// probabilities, whose pair replaces the scores in TMEM.  A single warp per
// scheduler issues an instruction of such code every five or six cycles, so both
// kinds of arithmetic have two.  P hi times
// [V hi | V lo] is one product of N = 2 head_dim; the halves of O are added
// when it is read.  The tensor pipe's f32 accumulation truncates, so every
// CHUNK blocks O moves to f32 sums in the workspace (each thread its row).
// Four ragged prompts of up to 1,024 tokens (16 heads x 64) take 113 us (307 us on
// mma.sync): 3,700 cycles per block of 64 keys, bound by the probabilities'
// instructions.  Waits are bounded as in paged_attention_tc.cu.
#include <math.h>

#include <type_traits>

#include "attention_f16.cuh"
#include "paged.cuh"

namespace etb {
namespace {

using namespace paged;
using namespace f16att;

constexpr int ROWS = 128, BK = 64;
constexpr int SOFT = 256, CONVERT_WARP = 8, MMA_WARP = 16, LOAD_WARP = 18, THREADS = 640;
// registers of the warpgroups: probabilities, conversion, the rest
constexpr int kSoftRegs = 136, kConvertRegs = 72, kLeanRegs = 48;
static_assert(256 * kSoftRegs + 256 * kConvertRegs + 128 * kLeanRegs <= THREADS * 96, "registers at launch");
constexpr float kJump = 8.0f;   // log2 of the largest P the standing maximum allows
constexpr float kShift = 7.0f;  // P carries 2^7: at most 2^15
constexpr int CHUNK = 8;        // blocks whose products one TMEM accumulator adds

__device__ int g_wait_error;  // bounded waits that gave up (the status word tells the caller)

template <int DH>
struct Layout {
  static constexpr int RAW = BK * DH * 4;             // one raw tile of K or V
  static constexpr int RAWS = DH == 128 ? 2 : 6;      // tiles in the ring: K, V, K, V, ...
  static constexpr int KT = BK * DH * 2;              // one binary16 tile
  static constexpr int PAIRS = 4 * KT;                // K hi, K lo, V hi, V lo
  static constexpr int CONV = RAWS * RAW;
  static constexpr int QLO = CONV + 2 * PAIRS;
  static constexpr int V_FACTORS = QLO + ROWS * DH * 2;     // [2][2][BK]: exponents and factors
  static constexpr int K_FACTORS = V_FACTORS + 2 * 2 * BK * 4;  // [3][BK]
  static constexpr int SHARED_ROWS = K_FACTORS + 3 * BK * 4;  // what a row's threads exchange
  static constexpr int BARS = SHARED_ROWS + 1024;
  static constexpr int SMEM = BARS + 216;
  static constexpr uint32_t S0 = 0, QH = 128, O = 192, COLS = 512;
  static_assert(O + 2 * DH <= COLS && QH + DH / 2 <= O && SMEM <= 232448, "TMEM and shared memory");
};

// e with 2^13 <= amax 2^e < 2^14; 100 for a row of zeros (any e describes it,
// and a large one keeps it out of the maximum) and for rows below 2^-87.
__device__ __forceinline__ int row_exponent(float amax) {
  return min(100, 13 - ((int)(__float_as_uint(amax) >> 23) - 127));
}

template <int DH>
__global__ void __launch_bounds__(THREADS, 1)
paged_attention_f32_kernel(const __grid_constant__ CUtensorMap k_map,
                           const __grid_constant__ CUtensorMap v_map, AttendArgs a, int box_rows) {
  using L = Layout<DH>;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* v_factors = reinterpret_cast<float*>(smem + L::V_FACTORS);
  float* k_factors = reinterpret_cast<float*>(smem + L::K_FACTORS);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  enum {
    RAWFULL = 0, RAWEMPTY = 6, KFULL = 12, VFULL = 14, SFULL = 16, PREADY = 18, PVDONE = 20,
    QREADY = 22, DRAIN = 23, NBARS = 25
  };
  const uint32_t bar0 = smem_u32(bars);
  auto B_ = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + NBARS);
  volatile int* abort = reinterpret_cast<volatile int*>(tslot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_u32(smem);
  const int group = a.tiling.group, dim = a.pools.head_dim;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (tid == 0) {
    for (int i = 0; i < NBARS; i++)
      mbar_init(B_(i), (i >= RAWEMPTY && i < SFULL) ? MMA_WARP - CONVERT_WARP
                       : (i == PREADY || i == PREADY + 1 || i == QREADY) ? SOFT : 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) tmem_alloc(smem_u32(tslot), L::COLS);
  Place p;
  const Share share = divide(a.tiling, a.batch, a.least, p,
                             *reinterpret_cast<DivideRoom<THREADS>*>(smem + L::QLO));
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
    return role_wait(B_(i), parity & 1u, &g_wait_error, abort);
  };
  uint32_t n = 0;  // blocks so far, of all tiles: slot n & 1, round n >> 1

  if (warp >= MMA_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLeanRegs));
  if (warp == LOAD_WARP) {
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
#pragma unroll
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
        mbar_wait(B_(RAWFULL + c % L::RAWS), (c / L::RAWS) & 1u, &g_wait_error);
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
        if (ok) ok = wait(KFULL + slot, n >> 1);
        if (ok && n >= 2) ok = wait(PVDONE + slot, (n >> 1) - 1);  // the slot held P of block n - 2
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t k = base + L::CONV + slot * L::PAIRS, d = tmem + L::S0 + 64u * slot;
#pragma unroll
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
      mbar_wait(B_(DRAIN), 0u, &g_wait_error);
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
          const uint32_t v = base + L::CONV + slot * L::PAIRS + 2u * L::KT;
          const uint32_t pa = tmem + L::S0 + 64u * slot;
#pragma unroll
          for (int i = 0; i < BK / 16; i++) {
            const uint64_t vd = mdesc16<BK>(v, i);  // V lo lies one chunk stride behind V hi
            const uint32_t hi = pa + 32u * (i / 2) + 8u * (i % 2);
            umma_f16_ts(tmem + L::O, hi, vd, idesc_o2, (j % CHUNK != 0 || i > 0) ? 1u : 0u);
            umma_f16_ts(tmem + L::O, hi + 16u, vd, idesc_o, 1u);
          }
          umma_commit(B_(PVDONE + (int)slot));
        }
      }
      next_tile(nb);
    }
    if (lane == 0) {
      umma_commit(B_(DRAIN + 1));
      mbar_wait(B_(DRAIN + 1), 0u, &g_wait_error);
    }
  }
  } else if (warp >= CONVERT_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegs));
    // ---- raw rows into pairs; warp w takes rows w RW, w RW + 1, ... of each 8 RW.  A
    // slot of K is free once its scores are done, one of V (and of the scores) once
    // its P V is: K is a block ahead by then and the next scores need not wait.  The
    // factors of K outlive their slot by the probabilities, so they have three.
    constexpr int LANES = DH / 4, RW = 32 / LANES;  // lanes per row, rows of a warp at once
    const int sub = lane / LANES, col = lane % LANES;
    uint32_t count = 0;  // tiles: K, V, K, V, ...
    bool ok = true;
    while (ok && left > 0) {
      const int nb = blocks_here(), visible = tile_visible(a.tiling, p.r, p.tile);
#pragma unroll 1
      for (int i = 0; i < 2 * nb; i++, count++) {
        const int kv = i & 1, valid = visible - (p.blk + (i >> 1)) * BK;
        const uint32_t s = count % L::RAWS, block = count >> 1;
        const uint32_t conv = base + L::CONV + (block & 1u) * L::PAIRS + (uint32_t)kv * 2u * L::KT;
        float* vf = v_factors + (block & 1u) * 2 * BK;
        float* kf = k_factors + block % 3u * BK;
        if (block >= 2) ok = wait((kv == 0 ? SFULL : PVDONE) + (block & 1u), (block >> 1) - 1);
        if (ok) ok = wait(RAWFULL + s, count / L::RAWS);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        // four rows at once: loads, then maxima, then stores
        constexpr int STEP = 8 * RW, AT_ONCE = 4;
#pragma unroll 1
        for (int r0 = 0; r0 < BK; r0 += AT_ONCE * STEP) {
          const int row0 = r0 + (warp - CONVERT_WARP) * RW + sub;
          float4 x[AT_ONCE];
          float m[AT_ONCE];
#pragma unroll
          for (int k = 0; k < AT_ONCE; k++) {
            const int row = row0 + k * STEP;
            x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row < valid) x[k] = lds128(base + s * L::RAW + (uint32_t)(row * DH + 4 * col) * 4u);
            m[k] = abs_max4(0.0f, x[k]);
          }
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) m[k] = fmaxf(m[k], __shfl_xor_sync(0xffffffffu, m[k], o));
#pragma unroll
          for (int k = 0; k < AT_ONCE; k++) {
            const int row = row0 + k * STEP;
            const uint32_t piece = ((uint32_t)col & 15u) >> 1;
            const uint32_t to = conv + (uint32_t)(col >> 4) * BK * 128u + (uint32_t)row * 128u +
                                ((piece ^ (uint32_t)(row & 7)) << 4) + (uint32_t)(col & 1) * 8u;
            const int e = row_exponent(m[k]);
            const float sc = exp2_int(e);
            float h0, l0, h1, l1;
            pair2(x[k].x * sc, x[k].y * sc, h0, l0);
            pair2(x[k].z * sc, x[k].w * sc, h1, l1);
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(h0), "f"(h1) : "memory");
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(to + L::KT), "f"(l0), "f"(l1) : "memory");
            if (col == 0) {
              if (kv == 0) {
                kf[row] = exp2_int(-e);
              } else {
                vf[row] = (float)-e;
                vf[BK + row] = sc;
              }
            }
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(B_(RAWEMPTY + s));
          mbar_arrive(B_((kv == 0 ? KFULL : VFULL) + (block & 1u)));
        }
      }
      next_tile(nb);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    // ---- probabilities: two threads per row, keys 32 half .. 32 half + 31 of a block
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    __nv_bfloat16* row_max = reinterpret_cast<__nv_bfloat16*>(smem + L::SHARED_ROWS);  // [2][2][ROWS]
    float* row_value = reinterpret_cast<float*>(smem + L::SHARED_ROWS);                // [ROWS], between tiles
    auto pair_sync = [&]() { named_sync(1 + quarter, 64); };
    const bool q_vec = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * 4)) & 15) == 0;
    const bool rope_vec = ((reinterpret_cast<uintptr_t>(a.rope.cos) | reinterpret_cast<uintptr_t>(a.rope.sin)) & 7) == 0;
    const bool o_vec = ((reinterpret_cast<uintptr_t>(a.o) | (uintptr_t)(a.o_stride * 4)) & 15) == 0;
    bool ok = true;
    Cut cut{0, 0, 0, 0, 0};
    // after a wait that ran out the loops still end, in step with the other thread
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
      // ---- the warp's 16 rows of Q, rotated: 8 lanes a row, whole lines.  hi passes
      // through the tile of lo on its way into TMEM (a row per lane), then lo takes
      // the tile.
      {
        constexpr int P = DH / 32;  // 16-byte pieces of a lane
        const uint32_t tile = base + L::QLO;
        constexpr int G = 2;  // groups of 4 rows whose loads are in flight
        auto unit_at = [&](int r, int i) {
          const int c = (lane & 7) + 8 * i;  // 8-byte unit of the row
          return tile + (uint32_t)(c >> 4) * ROWS * 128u + (uint32_t)r * 128u +
                 (((((uint32_t)c & 15u) >> 1) ^ (uint32_t)(r & 7)) << 4) + (uint32_t)(c & 1) * 8u;
        };
        float low[4][P][2];
#pragma unroll
        for (int g0 = 0; g0 < 4; g0 += G) {
          // all loads first: rows and dims that are not there read the tensor's or
          // the table's beginning
          float4 x[G][P];
          float2 cs[G][P], sn[G][P];
#pragma unroll
          for (int k = 0; k < G; k++) {
            const int r = quarter * 32 + half * 16 + 4 * (g0 + k) + (lane >> 3), gr = p.tile * ROWS + r;
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
            const int r = quarter * 32 + half * 16 + 4 * (g0 + k) + (lane >> 3);
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
        // hi is complete: this thread's half of its row
        pair_sync();
        cq = row_value[row];
#pragma unroll
        for (int w = 0; w < DH / 4; w += 16) {
          float v[16];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t u = (uint32_t)(half * (DH / 4) + w) / 4u + (uint32_t)i;
            const float4 f = lds128(tile + (u >> 3) * ROWS * 128u + (uint32_t)row * 128u +
                                    (((u & 7u) ^ (uint32_t)(row & 7)) << 4));
            v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
          }
          tmem_st16(lanes + L::QH + (uint32_t)(half * (DH / 4) + w), v);
        }
        tmem_wait_st();
        pair_sync();
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
          for (int i = 0; i < P; i++)
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(unit_at(quarter * 32 + half * 16 + 4 * k + (lane >> 3), i)),
                         "f"(low[k][i][0]), "f"(low[k][i][1]) : "memory");
      }
      {
        fence_async_smem();
        tc_fence_before();
        mbar_arrive(B_(QREADY));
      }
      float* part = a.joint.sums + ((int64_t)(2 * (int)blockIdx.x + (whole ? 1 : 0)) * ROWS + row) * DH;
      float m = -INFINITY, l = 0.0f, m_part = -INFINITY;
      bool have_part = false;
      // O so far, relative to m, into v (32 columns from 32 c), with what the workspace holds
      auto read_o = [&](int c, float (&v)[32]) {
        float v2[32];
        tmem_ld32(lanes + L::O + 32u * c, v);
        tmem_ld32(lanes + L::O + (uint32_t)DH + 32u * c, v2);
        const float f = have_part ? ex2(m_part - (m == -INFINITY ? 0.0f : m)) : 0.0f;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          if (have_part) y = *reinterpret_cast<const float4*>(part + 32 * c + i);
          v[i] = (v[i] + v2[i]) + f * y.x;
          v[i + 1] = (v[i + 1] + v2[i + 1]) + f * y.y;
          v[i + 2] = (v[i + 2] + v2[i + 2]) + f * y.z;
          v[i + 3] = (v[i + 3] + v2[i + 3]) + f * y.w;
        }
      };
      auto write_part = [&](int c, const float (&v)[32]) {
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<float4*>(part + 32 * c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      };
      for (int j = 0; j < nb; j++, n++) {
        if (j > 0 && j % CHUNK == 0) {  // move O out: the next product starts a new accumulator
          if (ok) ok = __all_sync(0xffffffffu, wait(PVDONE + ((n - 1) & 1u), (n - 1) >> 1));
          tc_fence_after();
#pragma unroll 1
          for (int c = half * (DH / 64); c < (half + 1) * (DH / 64); c++) {
            float v[32];
            read_o(c, v);
            write_part(c, v);
          }
          have_part = true;
          m_part = m == -INFINITY ? 0.0f : m;
        }
        if (ok) ok = wait(VFULL + (n & 1u), n >> 1);  // the factors of both: K's come first
        if (ok) ok = wait(SFULL + (n & 1u), n >> 1);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        const uint32_t s_at = lanes + L::S0 + 64u * (n & 1u);
        const int key0 = (p.blk + j) * BK;
        const bool masked = key0 + BK > vis_warp;
        const int seen = vis - key0 - 32 * half;
        const uint32_t kf_at = smem_u32(k_factors + n % 3u * BK) + 128u * (uint32_t)half;
        const uint32_t vf_at = smem_u32(v_factors + (n & 1u) * 2 * BK) + 128u * (uint32_t)half;
        // this thread's scores in base 2, exponents of their values added
        uint64_t s2[16];
        {
          float s[32];
          tmem_ld32(s_at + 32u * half, s);
          const uint64_t cq2 = twice(cq);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 kf = lds128(kf_at + 4u * i), ge = lds128(vf_at + 4u * i);
            s2[i / 2] = fma2(mul2(pk(s[i], s[i + 1]), cq2), pk(kf.x, kf.y), pk(ge.x, ge.y));
            s2[i / 2 + 1] = fma2(mul2(pk(s[i + 2], s[i + 3]), cq2), pk(kf.z, kf.w), pk(ge.z, ge.w));
          }
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const float2 v = unpk(s2[i]);
            s2[i] = pk(2 * i >= seen ? -INFINITY : v.x, 2 * i + 1 >= seen ? -INFINITY : v.y);
          }
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float2 v = unpk(s2[i]);
          top[i & 3] = fmaxf(top[i & 3], fmaxf(v.x, v.y));
        }
        // the row's maximum over both threads, rounded up: any bound serves both
        __nv_bfloat16* shared_max = row_max + (n & 1u) * 2 * ROWS;
        const __nv_bfloat16 own = __float2bfloat16_ru(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
        shared_max[half * ROWS + row] = own;
        pair_sync();
        const float bmax = fmaxf(__bfloat162float(own), __bfloat162float(shared_max[(1 - half) * ROWS + row]));
        const bool jump = bmax > m + kJump;
        if (__any_sync(0xffffffffu, jump)) {
          const float factor = jump ? ex2(m - bmax) : 1.0f;  // 0 while m is -inf
          if (jump) {
            m = bmax;
            l *= factor;
          }
          if (j % CHUNK != 0) {  // O holds products of this chunk: rescale it once they are complete
            if (ok) ok = __all_sync(0xffffffffu, wait(PVDONE + ((n - 1) & 1u), (n - 1) >> 1));
            tc_fence_after();
#pragma unroll 1
            for (int c = half * (DH / 32); c < (half + 1) * (DH / 32); c++) {
              float o[32];
              tmem_ld32(lanes + L::O + 32u * c, o);
#pragma unroll
              for (int i = 0; i < 32; i++) o[i] *= factor;
              tmem_st32(lanes + L::O + 32u * c, o);
            }
          }
        }
        const float from = (m == -INFINITY ? 0.0f : m) - kShift;
        uint64_t sum2[2] = {0, 0};
        const uint64_t from2 = twice(-from);
        float hi[16], lo[16];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float4 vf = lds128(vf_at + 4u * (BK + 2 * i));
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const float2 x = unpk(add2(s2[i + k], from2));
            const uint64_t w = pk(ex2(x.x), ex2(x.y));
            sum2[k] = fma2(w, k == 0 ? pk(vf.x, vf.y) : pk(vf.z, vf.w), sum2[k]);
            const float2 w2 = unpk(w);
            const __half2 h = __floats2half2_rn(w2.x, w2.y);
            const float2 hf = __half22float2(h), rest = unpk(add2(w, pk(-hf.x, -hf.y)));
            const __half2 l2 = __floats2half2_rn(rest.x, rest.y);
            hi[i + k] = __uint_as_float(*reinterpret_cast<const uint32_t*>(&h));
            lo[i + k] = __uint_as_float(*reinterpret_cast<const uint32_t*>(&l2));
          }
        }
        // over the columns of these keys' scores: hi, then lo
        tmem_st16(s_at + 32u * half, hi);
        tmem_st16(s_at + 32u * half + 16u, lo);
        const float2 all = unpk(add2(sum2[0], sum2[1]));
        l += all.x + all.y;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(B_(PREADY + (n & 1u)));
      }
      if (ok) ok = __all_sync(0xffffffffu, wait(PVDONE + ((n - 1) & 1u), (n - 1) >> 1));
      pair_sync();  // the last maxima are read
      if (half == 1) row_value[row] = l;
      pair_sync();
      if (half == 0) {
        l += row_value[row];
        row_value[row] = l;
      }
      pair_sync();
      l = row_value[row];
      pair_sync();  // read before the next tile's queries write there
      if (ok) {
        tc_fence_after();
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        float* dst = static_cast<float*>(a.o) + (p.r.first + token) * a.o_stride + (int64_t)head * dim;
        const int slot = 2 * (int)blockIdx.x + (whole ? 1 : 0);
#pragma unroll 1
        for (int c = half * (DH / 64); c < (half + 1) * (DH / 64); c++) {
          float o[32];
          read_o(c, o);
          if (!valid) continue;
          if (done) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const int d = 32 * c + i;
              if (d >= dim) break;
              if (o_vec)
                *reinterpret_cast<float4*>(dst + d) =
                    make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
              else
#pragma unroll
                for (int k = 0; k < 4; k++) dst[d + k] = o[i + k] * inv;
            }
          } else {
            write_part(c, o);
          }
        }
        if (valid && half == 0) {
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
      next_tile(nb);
    }
    if (tid == 0) {
      if (!ok) report(a.batch.status, ET_B200_PAGED_TIMEOUT);
      a.joint.cuts[blockIdx.x] = cut;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, L::COLS);
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
  paged_attention_f32_kernel<DH><<<blocks, THREADS, L::SMEM, stream>>>(k_map, v_map, a, box_rows);
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
