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
// A tile is 128 rows (TMEM lanes), a block 64 keys.  Warp 10 copies raw K and V
// tiles by TMA, warps 4-7 turn them into pairs (a row by DH / 4 lanes: maximum,
// exponent, split) in shared memory, warp 8 issues S = Q K^T up to a block ahead
// of warp 9's O += P V, warps 0-3 (one row per thread) form the
// probabilities, whose pair replaces the scores in TMEM.  P hi times
// [V hi | V lo] is one product of N = 2 head_dim; the halves of O are added
// when it is read.  The tensor pipe's f32 accumulation truncates, so every
// CHUNK blocks O moves to f32 sums in the workspace (each thread its row).
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
constexpr int CONVERT_WARP = 4, MMA_WARP = 8, LOAD_WARP = 10, THREADS = 384;
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
  static constexpr int FACTORS = QLO + ROWS * DH * 2;  // [2][3][BK]: of K, exponents and factors of V
  static constexpr int BARS = FACTORS + 2 * 3 * BK * 4;
  static constexpr int SMEM = BARS + 256 + 1024;
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
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  float* factors = reinterpret_cast<float*>(smem + L::FACTORS);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  enum {
    RAWFULL = 0, RAWEMPTY = 6, CONVFULL = 12, CONVEMPTY = 14, SFULL = 16, PREADY = 18, PVDONE = 20,
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
      mbar_init(B_(i), (i >= RAWEMPTY && i < CONVEMPTY) ? 4
                       : (i == PREADY || i == PREADY + 1 || i == QREADY) ? ROWS : 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) tmem_alloc(smem_u32(tslot), L::COLS);
  Place p;
  const Share share = divide<THREADS>(a.tiling, a.batch, a.least, p);
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
        if (ok) ok = wait(CONVFULL + slot, n >> 1);
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
            umma_f16_ts(tmem + L::O, pa + 8u * i, vd, idesc_o2, (j % CHUNK != 0 || i > 0) ? 1u : 0u);
            umma_f16_ts(tmem + L::O, pa + 32u + 8u * i, vd, idesc_o, 1u);
          }
          umma_commit(B_(PVDONE + (int)slot));
          umma_commit(B_(CONVEMPTY + (int)slot));
        }
      }
      next_tile(nb);
    }
    if (lane == 0) {
      umma_commit(B_(DRAIN + 1));
      mbar_wait(B_(DRAIN + 1), 0u, &g_wait_error);
    }
  } else if (warp >= CONVERT_WARP && warp < MMA_WARP) {
    // ---- raw rows into pairs; warp w takes rows w RW, w RW + 1, ... of each 4 RW
    constexpr int LANES = DH / 4, RW = 32 / LANES;  // lanes per row, rows of a warp at once
    const int sub = lane / LANES, col = lane % LANES;
    uint32_t count = 0;
    bool ok = true;
    while (ok && left > 0) {
      const int nb = blocks_here(), visible = tile_visible(a.tiling, p.r, p.tile);
      for (int j = 0; j < nb; j++, n++) {
        const int valid = visible - (p.blk + j) * BK;
        const uint32_t conv = base + L::CONV + (n & 1u) * L::PAIRS;
        float* f = factors + (n & 1u) * 3 * BK;
        if (n >= 2) ok = wait(CONVEMPTY + (n & 1u), (n >> 1) - 1);
        const uint32_t sk = count % L::RAWS, sv = (count + 1) % L::RAWS;
        if (ok) ok = wait(RAWFULL + sk, count / L::RAWS);
        if (ok) ok = wait(RAWFULL + sv, (count + 1) / L::RAWS);
        count += 2;
        // rows of both tiles at once: loads, then maxima, then stores
        constexpr int STEP = 4 * RW, AT_ONCE = 4;
#pragma unroll 1
        for (int r0 = 0; r0 < BK && ok; r0 += AT_ONCE * STEP) {
          const int row0 = r0 + (warp - CONVERT_WARP) * RW + sub;
          float4 x[2][AT_ONCE];
          float m[2][AT_ONCE];
#pragma unroll
          for (int kv = 0; kv < 2; kv++)
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) {
              const int row = row0 + k * STEP;
              x[kv][k] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (row < valid)
                x[kv][k] = lds128(base + (kv == 0 ? sk : sv) * L::RAW + (uint32_t)(row * DH + 4 * col) * 4u);
              m[kv][k] = abs_max4(0.0f, x[kv][k]);
            }
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < 2 * AT_ONCE; i++)
              m[i & 1][i >> 1] = fmaxf(m[i & 1][i >> 1], __shfl_xor_sync(0xffffffffu, m[i & 1][i >> 1], o));
#pragma unroll
          for (int k = 0; k < AT_ONCE; k++) {
            const int row = row0 + k * STEP;
            const uint32_t piece = ((uint32_t)col & 15u) >> 1;
            const uint32_t at = conv + (uint32_t)(col >> 4) * BK * 128u + (uint32_t)row * 128u +
                                ((piece ^ (uint32_t)(row & 7)) << 4) + (uint32_t)(col & 1) * 8u;
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
              const int e = row_exponent(m[kv][k]);
              const float sc = exp2_int(e);
              float h0, l0, h1, l1;
              pair2(x[kv][k].x * sc, x[kv][k].y * sc, h0, l0);
              pair2(x[kv][k].z * sc, x[kv][k].w * sc, h1, l1);
              const uint32_t to = at + (uint32_t)kv * 2u * L::KT;
              asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(h0), "f"(h1) : "memory");
              asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(to + L::KT), "f"(l0), "f"(l1)
                           : "memory");
              if (col == 0) {
                if (kv == 0) {
                  f[row] = exp2_int(-e);
                } else {
                  f[BK + row] = (float)-e;
                  f[2 * BK + row] = sc;
                }
              }
            }
          }
        }
        __syncwarp();
        if (ok && lane == 0) {
          mbar_arrive(B_(RAWEMPTY + sk));
          mbar_arrive(B_(RAWEMPTY + sv));
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(B_(CONVFULL + (n & 1u)));
      }
      next_tile(nb);
    }
  } else if (warp < CONVERT_WARP) {
    // ---- probabilities, one row per thread
    const int row = tid;
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const bool q_vec = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * 4)) & 15) == 0;
    const bool rope_vec = ((reinterpret_cast<uintptr_t>(a.rope.cos) | reinterpret_cast<uintptr_t>(a.rope.sin)) & 7) == 0;
    const bool o_vec = ((reinterpret_cast<uintptr_t>(a.o) | (uintptr_t)(a.o_stride * 4)) & 15) == 0;
    bool ok = true;
    Cut cut{0, 0, 0, 0, 0};
    while (ok && left > 0) {
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
        const uint32_t tile = base + L::QLO;
        constexpr int G = DH == 128 ? 2 : 4;  // groups of 4 rows whose loads are in flight
        auto unit_at = [&](int r, int i) {
          const int c = (lane & 7) + 8 * i;  // 8-byte unit of the row
          return tile + (uint32_t)(c >> 4) * ROWS * 128u + (uint32_t)r * 128u +
                 (((((uint32_t)c & 15u) >> 1) ^ (uint32_t)(r & 7)) << 4) + (uint32_t)(c & 1) * 8u;
        };
#pragma unroll 1
        for (int pass = 0; pass < 16; pass += G) {
        const int g0 = pass & 7;
        if (pass == 8) {  // hi is complete
          __syncwarp();
          tile_row16_to_tmem<DH>(tile, row, lanes, L::QH);
          tmem_wait_st();
          __syncwarp();
        }
          float4 x[G][P];
          float2 cs[G][P], sn[G][P];
#pragma unroll
          for (int k = 0; k < G; k++) {
            const int r = warp * 32 + 4 * (g0 + k) + (lane >> 3), gr = p.tile * ROWS + r;
            const int t = quotient(gr, a.tiling.by_group), at_pos = p.r.len - p.r.n + t;
            const bool some = r < rows;
            const float* src = static_cast<const float*>(a.q) + (p.r.first + t) * a.q_stride +
                               (int64_t)(p.h * group + gr - t * group) * dim;
            const int64_t tab = some && a.rope.cos != nullptr && at_pos >= 0
                                    ? rope_row(a.rope, at_pos, a.batch.status) * (dim / 2) : -1;
#pragma unroll
            for (int i = 0; i < P; i++) {
              const int d = 4 * ((lane & 7) + 8 * i);
              x[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
              cs[k][i] = make_float2(1.f, 1.f);
              sn[k][i] = make_float2(0.f, 0.f);
              if (some && d < dim) {
                if (q_vec) x[k][i] = __ldg(reinterpret_cast<const float4*>(src + d));
                else x[k][i] = make_float4(__ldg(src + d), __ldg(src + d + 1), __ldg(src + d + 2), __ldg(src + d + 3));
                if (tab >= 0) {
                  const float *ct = a.rope.cos + tab + d / 2, *st = a.rope.sin + tab + d / 2;
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
          }
#pragma unroll
          for (int k = 0; k < G; k++) {
            const int r = warp * 32 + 4 * (g0 + k) + (lane >> 3);
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < P; i++) m = abs_max4(m, x[k][i]);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            // a rotated pair is at most sqrt(2) times its larger element: below 2^14.5
            const int e = row_exponent(m);
            const float sc = exp2_int(e);
            const int mine = __shfl_sync(0xffffffffu, e, (lane & 3) * 8);
            if ((lane >> 2) == g0 + k) cq = a.scale_log2 * exp2_int(-mine);
#pragma unroll
            for (int i = 0; i < P; i++) {
              float4 v = x[k][i];
              if (a.rope.cos != nullptr) {
                rotate(v.x, v.y, cs[k][i].x, sn[k][i].x);
                rotate(v.z, v.w, cs[k][i].y, sn[k][i].y);
              }
              float h0, l0, h1, l1;
              pair2(v.x * sc, v.y * sc, h0, l0);
              pair2(v.z * sc, v.w * sc, h1, l1);
              asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(unit_at(r, i)),
                           "f"(pass < 8 ? h0 : l0), "f"(pass < 8 ? h1 : l1) : "memory");
            }
          }
        }
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
      for (int j = 0; ok && j < nb; j++, n++) {
        if (j > 0 && j % CHUNK == 0) {  // move O out: the next product starts a new accumulator
          ok = __all_sync(0xffffffffu, wait(PVDONE + ((n - 1) & 1u), (n - 1) >> 1));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < DH / 32; c++) {
            float v[32];
            read_o(c, v);
            write_part(c, v);
          }
          have_part = true;
          m_part = m == -INFINITY ? 0.0f : m;
        }
        ok = wait(CONVFULL + (n & 1u), n >> 1);  // the factors
        if (ok) ok = wait(SFULL + (n & 1u), n >> 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t s_at = lanes + L::S0 + 64u * (n & 1u);
        const int key0 = (p.blk + j) * BK;
        const bool masked = key0 + BK > vis_warp;
        const int seen = vis - key0;
        const uint32_t f_at = smem_u32(factors + (n & 1u) * 3 * BK);
        // scores of 32 keys in base 2, exponents of their values added; computed for
        // the maximum and again for the weights: half the code of keeping all 64
        // (instruction fetches were a quarter of this kernel's stalls)
        auto scores = [&](int c, float (&s)[32]) {
          tmem_ld32(s_at + 32u * c, s);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 kf = lds128(f_at + 4u * (32 * c + i)), ge = lds128(f_at + 4u * (BK + 32 * c + i));
            s[i] = fmaf(s[i] * cq, kf.x, ge.x);
            s[i + 1] = fmaf(s[i + 1] * cq, kf.y, ge.y);
            s[i + 2] = fmaf(s[i + 2] * cq, kf.z, ge.z);
            s[i + 3] = fmaf(s[i + 3] * cq, kf.w, ge.w);
          }
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; i++)
              if (32 * c + i >= seen) s[i] = -INFINITY;
          }
        };
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int c = 0; c < 2; c++) {
          float s[32];
          scores(c, s);
#pragma unroll
          for (int i = 0; i < 32; i++) top[i & 3] = fmaxf(top[i & 3], s[i]);
        }
        const float bmax = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        const bool jump = bmax > m + kJump;
        if (__any_sync(0xffffffffu, jump)) {
          const float factor = jump ? ex2(m - bmax) : 1.0f;  // 0 while m is -inf
          if (jump) {
            m = bmax;
            l *= factor;
          }
          if (j % CHUNK != 0) {  // O holds products of this chunk: rescale it once they are complete
            ok = __all_sync(0xffffffffu, wait(PVDONE + ((n - 1) & 1u), (n - 1) >> 1));
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 2 * DH / 32; c++) {
              float o[32];
              tmem_ld32(lanes + L::O + 32u * c, o);
#pragma unroll
              for (int i = 0; i < 32; i++) o[i] *= factor;
              tmem_st32(lanes + L::O + 32u * c, o);
            }
          }
        }
        const float from = (m == -INFINITY ? 0.0f : m) - kShift;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        // the pairs of the first 32 keys wait in registers: they replace scores that
        // the second pass still reads
        float hi[16], lo[16], hi0[16], lo0[16];
#pragma unroll 1
        for (int c = 0; c < 2; c++) {
          float s[32];
          scores(c, s);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 vf = lds128(f_at + 4u * (2 * BK + 32 * c + i));
            const float w0 = ex2(s[i] - from), w1 = ex2(s[i + 1] - from);
            const float w2 = ex2(s[i + 2] - from), w3 = ex2(s[i + 3] - from);
            sum[0] = fmaf(w0, vf.x, sum[0]);
            sum[1] = fmaf(w1, vf.y, sum[1]);
            sum[2] = fmaf(w2, vf.z, sum[2]);
            sum[3] = fmaf(w3, vf.w, sum[3]);
            pair2(w0, w1, hi[i / 2], lo[i / 2]);
            pair2(w2, w3, hi[i / 2 + 1], lo[i / 2 + 1]);
          }
          if (c == 0)
#pragma unroll
            for (int i = 0; i < 16; i++) {
              hi0[i] = hi[i];
              lo0[i] = lo[i];
            }
        }
        tmem_st16(s_at, hi0);
        tmem_st16(s_at + 32u, lo0);
        tmem_st16(s_at + 16u, hi);
        tmem_st16(s_at + 48u, lo);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(B_(PREADY + (n & 1u)));
      }
      if (ok) ok = __all_sync(0xffffffffu, wait(PVDONE + ((n - 1) & 1u), (n - 1) >> 1));
      if (ok) {
        tc_fence_after();
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        float* dst = static_cast<float*>(a.o) + (p.r.first + token) * a.o_stride + (int64_t)head * dim;
        const int slot = 2 * (int)blockIdx.x + (whole ? 1 : 0);
#pragma unroll 1
        for (int c = 0; c < DH / 32; c++) {
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
        if (valid) {
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
  const int blocks = thread_blocks(a, sm_count(), ROWS, BK);
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
