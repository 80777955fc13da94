// Attention of chunks of new tokens over a paged cache on tcgen05: f16 / bf16,
// head_dim up to 128, pages of a power of two of at least 8 slots.
//
// The mathematics and the division of the work are those of
// paged_attention.cu.  A tile is 256 rows (row: token x query head of the
// group) as two halves of 128 TMEM lanes, a block 128 keys.  K and V blocks
// arrive page by page through 4-D TMA maps of the pools (dim, slot, head,
// page) into a ring of slots that both halves read, which halves the L2
// traffic per product.  Each half has a thread that issues P V of a block and
// the next Q K^T behind it (one thread for both left the tensor pipe idle for
// 1,100 of 3,950 cycles per pair of blocks between barriers); the two take
// turns, which keeps the halves out of step: while the pipe works on one half, the
// other half's four warps (one row per thread, no exchange between threads) turn
// scores into probabilities, written over the scores in TMEM as the A operand of P V.
// The row maximum stands until a block exceeds it by 2^8 (2^4 at f16; the sums stay far
// inside f32), so O is rescaled in TMEM only then.
// A 4,096-token chunk over 12,000 keys (32 / 8 heads x 128, bf16) takes 725 us, 920
// TFLOP/s; a pair of half-blocks 3,520 cycles, 1,550 of them probabilities.  The
// products alone take 2,750 (the pipe's rate would allow some 2,050: Q K^T reads both
// 128-row operands from shared memory), the hand-off of scores and probabilities the
// rest.
// Fewer bits, by choice: the rotated queries and the probabilities are rounded to the
// cache's type (sums of weights are not).  The queries' residual would take 64 KB of
// shared memory (two of the five slots at head_dim 128) and half as many score products
// again.  Error of that chunk against 64 bits 2.9e-3 of the result, 1.7e-3 of it the
// rounding of the output alone; each of the two roundings adds some 1.5e-3 to 1.9e-3 in
// squares.
// Waits are bounded; one that runs out raises a CTA-wide abort, copies and
// products in flight are waited for and TMEM is released.
#include <math.h>

#include <type_traits>

#include "attention_f16.cuh"
#include "paged_mma.cuh"

namespace etb {
namespace {

using namespace paged;
using namespace f16att;

constexpr int HALF = 128, BK = 128;
// warps 0-7 probabilities; 8, 9 products, 10 copies (11 fills the warpgroup, whose
// registers above kLeanRegs go to the other two: 256 x 208 + 128 x 88 = 384 x 168)
constexpr int MMA_WARP = 8, LOAD_WARP = 10, THREADS = 384;
constexpr int kWideRegs = 208, kLeanRegs = 88;
static_assert(256 * kWideRegs + 128 * kLeanRegs <= THREADS * 168, "registers at launch");

template <int DH>
struct Layout {
  static constexpr int SLOT = BK * DH * 2;           // one block of K or V
  static constexpr int SLOTS = DH == 128 ? 5 : 8;
  static constexpr int Q = SLOTS * SLOT;              // two halves of 128 rows
  static constexpr int BARS = Q + 2 * HALF * DH * 2;
  static constexpr int SMEM = BARS + 512 + 1024;
  // TMEM: scores of the halves (P over the first 64 columns), outputs
  static constexpr uint32_t S0 = 0, O0 = 256, COLS = 512;
  static_assert(O0 + 2 * DH <= COLS && SMEM <= 232448, "TMEM and shared memory");
};

template <typename T, int DH>
__global__ void __launch_bounds__(THREADS, 1)
paged_attention_tc_kernel(const __grid_constant__ CUtensorMap k_map,
                          const __grid_constant__ CUtensorMap v_map, AttendArgs a, int box_rows) {
  using L = Layout<DH>;
  constexpr int SLOTS = L::SLOTS;
  // log2 of the largest P the standing maximum allows, and what P carries on top: at
  // f16 at most 2^15 together, so that its least normal number is 2^-25 of the standing
  // maximum (without it many unlikely keys behind a likely one lost their bits)
  constexpr float kJump = std::is_same_v<T, __half> ? 4.0f : 8.0f;
  constexpr float kShift = std::is_same_v<T, __half> ? 11.0f : 0.0f;
  constexpr uint32_t kType = std::is_same_v<T, __nv_bfloat16> ? (1u << 7) | (1u << 10) : 0u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  enum { FULL = 0, EMPTY = 8, SFULL = 16, PREADY = 18, QREADY = 20, ODONE = 22, DRAIN = 24, TURN = 26, NBARS = 28 };
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
      mbar_init(B_(i), (i >= PREADY && i < ODONE) ? HALF : (i >= EMPTY && i < SFULL) ? 2 : 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) tmem_alloc(smem_u32(tslot), L::COLS);
  Place p;
  __shared__ DivideRoom<THREADS> room;
  const Share share = divide(a.tiling, a.batch, a.least, p, room);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  // blocks of the tile at p that fall into this share, and whether it has rows
  // for the second half
  int64_t left = share.units;
  auto blocks_here = [&]() { return (int)min((int64_t)(p.nblk - p.blk), left); };
  auto rows_here = [&]() {
    return min(2 * HALF, p.r.n * group - p.tile * 2 * HALF);
  };
  auto next_tile = [&](int done) {
    left -= done;
    p.blk += done - 1;
    advance(a.tiling, a.batch, p);
  };
  auto wait = [&](int i, uint32_t parity) {
    return role_wait(B_(i), parity & 1u, abort_word, abort);
  };

  if (warp >= MMA_WARP) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLeanRegs));
  if (warp == LOAD_WARP) {
    // ---- K and V blocks, page by page
    uint32_t count = 0;  // slots filled: K, V, K, V, ...
    bool ok = true;
    const int boxes_per_tile = DH / 64;
    while (ok && left > 0) {
      const int nb = blocks_here(), visible = tile_visible(a.tiling, p.r, p.tile);
      for (int j = 0; ok && j < nb; j++) {
        const int key0 = (p.blk + j) * BK;
        const int boxes = (min(visible - key0, BK) + box_rows - 1) / box_rows;
        // each lane looks up the boxes it will load (at most 16 pages of 8 keys)
        const int mine = lane % 16;
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
        for (int kv = 0; kv < 2; kv++) {
          const uint32_t s = count % SLOTS, round = count / SLOTS;
          if (round > 0) ok = wait(EMPTY + s, round - 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint32_t bar = B_(FULL + s), dst = base + s * L::SLOT;
          if (lane == 0) mbar_expect_tx(bar, (uint32_t)(max(boxes, 0) * box_rows * DH * 2));
          __syncwarp();
          if (mine < boxes && lane / 16 < boxes_per_tile)
            tma_load_4d(dst + (uint32_t)(lane / 16) * BK * 128u + (uint32_t)(mine * box_rows) * 128u,
                        kv == 0 ? &k_map : &v_map, bar, 64 * (lane / 16), slot, p.h, page);
          count++;
        }
      }
      next_tile(nb);
    }
    // every copy has landed before the CTA releases its memory
    if (lane == 0)
      for (uint32_t c = count > SLOTS ? count - SLOTS : 0; c < count; c++)
        mbar_wait(B_(FULL + c % SLOTS), (c / SLOTS) & 1u, abort_word);
  } else if (warp < LOAD_WARP) {
    // ---- products of half t.  A half without rows goes along with the slots.
    const int t = warp - MMA_WARP;
    constexpr uint32_t idesc_s = idesc_f16_m128(BK, 0) | kType;
    constexpr uint32_t idesc_o = idesc_f16_m128(DH, 1) | kType;
    const uint32_t q = base + L::Q + (uint32_t)t * (HALF * DH * 2);
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
      for (int i = 0; i < DH / 16; i++)
        umma_f16(s_at, kdesc16<HALF>(q, i), kdesc16<BK>(k, i), idesc_s, i > 0 ? 1u : 0u);
      umma_commit(B_(SFULL + t));
    };
    while (ok && left > 0) {
      const int nb = blocks_here();
      const bool rows = rows_here() > HALF * t, both = rows_here() > HALF;
      const int visible = tile_visible(a.tiling, p.r, p.tile);
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
        const int valid = visible - (p.blk + j) * BK;
        if (valid < BK && rows) {  // slots behind the visible keys may hold anything
          for (int i = max(valid, 0) * 8 + lane; i < BK * 8; i += 32)
#pragma unroll
            for (int c = 0; c < DH / 64; c++)
              sts128(vt + (uint32_t)c * BK * 128u + (uint32_t)i * 16u, make_float4(0.f, 0.f, 0.f, 0.f));
          fence_async_smem();
          __syncwarp();
        }
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
            for (int i = 0; i < BK / 16; i++)
              umma_f16_ts(o_at, s_at + 8u * i, mdesc16<BK>(vt, i), idesc_o, (j > 0 || i > 0) ? 1u : 0u);
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
    const float scale = a.scale_log2;
    const bool q_vec = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_stride * 2)) & 15) == 0;
    const bool rope_vec = ((reinterpret_cast<uintptr_t>(a.rope.cos) | reinterpret_cast<uintptr_t>(a.rope.sin)) & 15) == 0;
    const bool o_vec = ((reinterpret_cast<uintptr_t>(a.o) | (uintptr_t)(a.o_stride * 2)) & 15) == 0;
    uint32_t items = 0, steps = 0;
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
        const int g = p.tile * 2 * HALF + HALF * t + row;
        const bool valid = row < rows;
        const int token = quotient(g, a.tiling.by_group), head = p.h * group + g - token * group;
        const int pos = p.r.len - p.r.n + token;
        const int vis = valid ? max(0, pos + 1) : 0;
        // keys that every row of this warp sees (invalid rows follow the last valid one)
        const int vis_warp = __shfl_sync(0xffffffffu, max(0, pos + 1), 0);
        // ---- the warp's rows of Q, rotated, into the swizzled tile: 8 lanes a row,
        // whole lines, 8 rows' loads in flight
        {
          constexpr int P = DH / 64;  // 16-byte pieces of a lane
          const int first_row = p.tile * 2 * HALF + HALF * t;
          const uint32_t tile = base + L::Q + (uint32_t)t * (HALF * DH * 2);
          for (int r0 = 0; r0 < 32; r0 += 8) {
            union Piece { uint4 v; T x[8]; };
            Piece u[2][P];
            float4 cs[2][P], sn[2][P];
#pragma unroll
            for (int k = 0; k < 2; k++) {
              const int r = (warp & 3) * 32 + r0 + 4 * k + (lane >> 3), gr = first_row + r;
              const int tk = quotient(gr, a.tiling.by_group), at_pos = p.r.len - p.r.n + tk;
              const bool some = r < rows;
              const T* src = static_cast<const T*>(a.q) + (p.r.first + tk) * a.q_stride +
                             (int64_t)(p.h * group + gr - tk * group) * dim;
              const int64_t tab = some && a.rope.cos != nullptr && at_pos >= 0
                                      ? rope_row(a.rope, at_pos, a.batch.status) * (dim / 2) : -1;
#pragma unroll
              for (int i = 0; i < P; i++) {
                const int d = 8 * ((lane & 7) + 8 * i);
                u[k][i].v = make_uint4(0, 0, 0, 0);
                cs[k][i] = make_float4(1.f, 1.f, 1.f, 1.f);
                sn[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (some && d < dim) {
                  if (q_vec) u[k][i].v = __ldg(reinterpret_cast<const uint4*>(src + d));
                  else
#pragma unroll
                    for (int e = 0; e < 8; e++) u[k][i].x[e] = src[d + e];
                  if (tab >= 0) {
                    const float *ct = a.rope.cos + tab + d / 2, *st = a.rope.sin + tab + d / 2;
                    if (rope_vec) {
                      cs[k][i] = __ldg(reinterpret_cast<const float4*>(ct));
                      sn[k][i] = __ldg(reinterpret_cast<const float4*>(st));
                    } else {
                      cs[k][i] = make_float4(__ldg(ct), __ldg(ct + 1), __ldg(ct + 2), __ldg(ct + 3));
                      sn[k][i] = make_float4(__ldg(st), __ldg(st + 1), __ldg(st + 2), __ldg(st + 3));
                    }
                  }
                }
              }
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
              const int r = (warp & 3) * 32 + r0 + 4 * k + (lane >> 3);
#pragma unroll
              for (int i = 0; i < P; i++) {
                const int c = (lane & 7) + 8 * i;
                if (a.rope.cos != nullptr) {
                  const float cc[4] = {cs[k][i].x, cs[k][i].y, cs[k][i].z, cs[k][i].w};
                  const float ss[4] = {sn[k][i].x, sn[k][i].y, sn[k][i].z, sn[k][i].w};
#pragma unroll
                  for (int e = 0; e < 4; e++) {
                    float x0 = to_f32<T>(u[k][i].x[2 * e]), x1 = to_f32<T>(u[k][i].x[2 * e + 1]);
                    rotate(x0, x1, cc[e], ss[e]);
                    if constexpr (std::is_same_v<T, __half>) {
                      x0 *= a.q_factor;
                      x1 *= a.q_factor;
                    }
                    u[k][i].x[2 * e] = from_f32<T>(x0);
                    u[k][i].x[2 * e + 1] = from_f32<T>(x1);
                  }
                }
                sts128(tile + (uint32_t)(c >> 3) * HALF * 128u + (uint32_t)r * 128u +
                           ((((uint32_t)c & 7u) ^ (uint32_t)(r & 7)) << 4),
                       *reinterpret_cast<const float4*>(&u[k][i].v));
              }
            }
          }
          fence_async_smem();
          tc_fence_before();
          mbar_arrive(B_(QREADY + t));
        }
        float m = -INFINITY, l = 0.0f;
        for (int j = 0; ok && j < nb; j++) {
          ok = __all_sync(0xffffffffu, wait(SFULL + t, steps));
          if (!ok) break;
          steps++;
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
          if (__any_sync(0xffffffffu, jump)) {
            const float factor = jump ? ex2(m - bmax) : 1.0f;  // 0 while m is -inf
            if (jump) {
              m = bmax;
              l *= factor;
            }
            if (j > 0) {
              // the scores' barrier also says that the last P V is complete
#pragma unroll
              for (int c = 0; c < DH / 32; c++) {
                float o[32];
                tmem_ld32(o_at + 32 * c, o);
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] *= factor;
                tmem_st32(o_at + 32 * c, o);
              }
            }
          }
          const float from = (m == -INFINITY ? 0.0f : m) - kShift;
          // a quarter of the exponentials on the FMA pipe, the others on the special
          // function unit (8 cycles per warp; the 4,096-token chunk: 783 us with all
          // of them there, 757 with a quarter on the FMA pipe, 800 with half);
          // blocks with masked scores (-inf) all on the latter
          uint64_t sum[2] = {0, 0};
          auto powers = [&](int c, auto some_masked) {
            float w[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
              uint64_t x = fma2(pk(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1])),
                                twice(scale), twice(-from));
              if (!decltype(some_masked)::value && (i & 3) == 3) {
                x = power2(x);
              } else {
                const float2 v = unpk(x);
                x = pk(ex2(v.x), ex2(v.y));
              }
              sum[i & 1] = add2(sum[i & 1], x);
              const float2 v = unpk(x);
              w[i] = __uint_as_float(pack2<T>(v.x, v.y));
            }
            tmem_st16(s_at + 16 * c, w);
          };
          if (masked) {
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
        if (ok) {
          tc_fence_after();
          const bool done = whole && ends;
          const float inv = l > 0.0f ? 1.0f / l : 0.0f;
          T* dst = static_cast<T*>(a.o) + (p.r.first + token) * a.o_stride + (int64_t)head * dim;
          const int slot = 2 * (int)blockIdx.x + (whole ? 1 : 0), r = HALF * t + row;
          float* part = a.joint.sums + ((int64_t)slot * 2 * HALF + r) * DH;
#pragma unroll
          for (int c = 0; c < DH / 32; c++) {
            float o[32];
            tmem_ld32(o_at + 32 * c, o);
            if (!valid) continue;
            if (done) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                const int d = 32 * c + i;
                if (d >= dim) break;
                union { uint4 v; uint32_t w[4]; T x[8]; } u;
#pragma unroll
                for (int k = 0; k < 4; k++) u.w[k] = pack2<T>(o[i + 2 * k] * inv, o[i + 2 * k + 1] * inv);
                if (o_vec) *reinterpret_cast<uint4*>(dst + d) = u.v;
                else
#pragma unroll
                  for (int k = 0; k < 8; k++) dst[d + k] = u.x[k];
              }
            } else {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<float4*>(part + 32 * c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
          }
          if (valid) {
            if (!done) {
              a.joint.stats[(int64_t)slot * 4 * HALF + r] = m - kShift;
              a.joint.stats[((int64_t)slot * 2 + 1) * 2 * HALF + r] = l;
            } else if (a.lse != nullptr) {
              a.lse[(p.r.first + token) * a.q_heads + head] = l > 0.0f ? (m - kShift) * kLn2 + logf(l) : -INFINITY;
            }
          }
          tc_fence_before();  // O is read before the next tile's QREADY
        }
      }
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
int launch_tc(const et_b200_paged_cache_v1* c, AttendArgs& a, void* ws, cudaStream_t stream) {
  using L = Layout<DH>;
  const int box_rows = (int)(c->page_size < BK ? c->page_size : BK);
  CUtensorMap k_map, v_map;
  if (!pool_map(&k_map, c->keys, c, 64, box_rows) || !pool_map(&v_map, c->values, c, 64, box_rows))
    return 0;
  const int blocks = thread_blocks(a, a.sms, 2 * HALF, BK);
  a.tiling = tiling_of(8, 7, a.tiling.group, a.pools.kv_heads);
  static_assert(2 * HALF == 1 << 8 && BK == 1 << 7, "tiling");
  a.least = 2;
  a.joint = joint_of(ws, blocks, 2 * HALF, DH);
  cudaFuncSetAttribute(paged_attention_tc_kernel<T, DH>,
                       cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
  paged_attention_tc_kernel<T, DH><<<blocks, THREADS, L::SMEM, stream>>>(k_map, v_map, a, box_rows);
  count_launch();
  return blocks;
}

}  // namespace

namespace paged {

size_t attend_tc_workspace(int dim_padded, int sms) {
  return dim_padded > 128 ? 0 : joint_bytes(sms, 2 * HALF, dim_padded < 64 ? 64 : dim_padded);
}

int attend_tc(const et_b200_paged_cache_v1* c, AttendArgs& a, void* ws, cudaStream_t stream) {
  if (c->dtype == ET_B200_DTYPE_F32 || c->head_dim > 128) return 0;
  if (c->dtype == ET_B200_DTYPE_F16)
    return c->head_dim <= 64 ? launch_tc<__half, 64>(c, a, ws, stream)
                             : launch_tc<__half, 128>(c, a, ws, stream);
  return c->head_dim <= 64 ? launch_tc<__nv_bfloat16, 64>(c, a, ws, stream)
                           : launch_tc<__nv_bfloat16, 128>(c, a, ws, stream);
}

}  // namespace paged
}  // namespace etb
