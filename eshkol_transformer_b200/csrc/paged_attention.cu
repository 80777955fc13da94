// Causal attention of new tokens over a paged cache
// (et_b200_paged_attention_v1): the kernel for any page size, head_dim and
// type, and the joining of cut tiles.
//
// o = sum_j p_j v_j / sum_j p_j, p_j = 2^(s_j - m), s_j = log2(e) scale q'.k_j,
// m the running maximum.  A thread block takes its share of the (tile, block)
// units (paged.cuh): tiles of 16 WM rows, blocks of BK keys.  K and V arrive
// in a ring of STAGES blocks, rows XOR-swizzled by 16-byte pieces (so ldmatrix
// and the f32 reads of V are free of bank conflicts): pages of a power of two
// of at least 8 slots by TMA from a warp of its own, which keeps copies,
// look-ups and block-wide barriers out of the arithmetic warps; any other page
// size by 16-byte cp.async, the key addresses of a block looked up one block
// ahead of its copies.  Warp (wm, wk) takes 16 rows and BK / WK keys of each block
// with its own maxima, sums and accumulators (mma.sync m16n8k16, or for f32 m16n8k8
// as 3xTF32: hi hi + hi lo + lo hi of operands rounded to TF32 pairs), which are
// joined where a tile ends.  At f16 and bf16 the queries carry their rounding's
// residual (the products are not what bounds it); the probabilities are rounded to
// the cache's type, which adds a third to the error of the output's own rounding.
// With few rows (a decoding step) reading the cache bounds it: one tile of 16 rows,
// warps split along the keys.  Measured: 64 requests of up to 8,192 keys (32 / 8
// heads x 128, bf16, 1.35 GB) 230 to 248 us by machine, 5.4 to 5.8 TB/s (274 us with
// cp.async where it took 231); one token over 300 f32 keys 9.6 us with the joining
// kernel.
#include <math.h>

#include <type_traits>

#include "paged_mma.cuh"

namespace etb {
namespace {

using namespace paged;

// ---- the kernel -------------------------------------------------------------------------

template <typename T, int DH_, int WM_, int WK_, int BK_, int STAGES_>
struct Shape {
  static constexpr int DH = DH_, WM = WM_, WK = WK_, BK = BK_, STAGES = STAGES_;
  static constexpr int NT = 32 * WM * WK, BM = 16 * WM, KW = BK / WK;
  static constexpr int ROW = DH * (int)sizeof(T), PIECES = ROW / 16;  // of one key
  static constexpr int TILE = BK * ROW, STAGE = 2 * TILE;
  static constexpr int TILE_Q = BM * ROW;
  static constexpr int Q_BYTES = TILE_Q * (sizeof(T) == 4 ? 1 : 2);  // f16, bf16: with their residuals
  static constexpr int MERGE = (WK - 1) * BM * DH * 4;
  static constexpr int RING = STAGES + 1;  // blocks with known key addresses
  static constexpr int KOFF = STAGES * STAGE + Q_BYTES;
  static constexpr int JOIN = KOFF + RING * BK * 8;
  static constexpr int BARS = JOIN + WK * BM * 8;
  static constexpr int SMEM = BARS + 2 * STAGES * 8 + 16;
  // a row in shared memory: chunks of 128 bytes (one of 64 at 4 pieces), each
  // [BK] (or [BM]) rows with the TMA swizzle of that width
  static constexpr int CHUNK = ROW < 128 ? ROW : 128, CHUNKS = ROW / CHUNK;
  static constexpr int WIDE = CHUNK / (int)sizeof(T);  // elements of a chunk
  static constexpr int PER_SM = 2 * (SMEM + 2048) <= 233472 ? 2 : 1;  // blocks the registers must allow
  static constexpr int bits(int n) { return n <= 1 ? 0 : 1 + bits(n / 2); }
  static_assert(1 << bits(BM) == BM && 1 << bits(BK) == BK, "powers of two");
  static_assert(KW % 16 == 0 && BK <= NT * 2, "keys per warp");
  static_assert(MERGE <= STAGE, "the joining of warps reuses a stage");
  static_assert(SMEM <= 232448, "shared memory");
  // byte of 16-byte piece c of a row in a tile of R rows
  template <int R>
  __device__ static uint32_t at(int row, int c) {
    if constexpr (PIECES >= 8)
      return (uint32_t)((c >> 3) * R * 128 + row * 128 + (((c & 7) ^ (row & 7)) << 4));
    else
      return (uint32_t)(row * ROW + ((c ^ ((row >> 1) & 3)) << 4));
  }
};

template <typename T, typename S, bool TMA>
__global__ void __launch_bounds__(S::NT + (TMA ? 32 : 0), S::PER_SM)
paged_attention_kernel(const __grid_constant__ CUtensorMap k_map,
                       const __grid_constant__ CUtensorMap v_map, AttendArgs a, int box_bits) {
  constexpr int DH = S::DH, BM = S::BM, BK = S::BK, KW = S::KW, NT = S::NT, WK = S::WK;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int KSTEP = F32 ? 8 : 16;  // dims (or keys) per matrix instruction
  // f16 probabilities carry 2^15: their least normal number is then 2^-29 of the largest
  constexpr float kShift = std::is_same_v<T, __half> ? 15.0f : 0.0f;
  extern __shared__ __align__(1024) uint8_t smem[];
  int64_t* koff = reinterpret_cast<int64_t*>(smem + S::KOFF);
  float* join_m = reinterpret_cast<float*>(smem + S::JOIN);
  float* join_l = join_m + WK * BM;
  const uint32_t base = smem_u32(smem);
  const uint32_t qs = base + S::STAGES * S::STAGE;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wm = warp / WK, wk = warp % WK;
  const int dim = a.pools.head_dim, group = a.tiling.group;
  const T* keys = static_cast<const T*>(a.keys);
  const T* values = static_cast<const T*>(a.values);
  // lets the joining kernel start its launch; it waits for this one's results
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // TMA: barriers of a stage (full, empty), 1 and one per arithmetic warp arrivals
  const uint32_t bars = base + S::BARS;
  auto full_bar = [&](int st) { return bars + 8u * (uint32_t)st; };
  auto empty_bar = [&](int st) { return bars + 8u * (uint32_t)(S::STAGES + st); };
  int* abort_word = reinterpret_cast<int*>(smem + S::BARS + 2 * S::STAGES * 8);
  volatile int* abort = abort_word;
  if (TMA && tid == 0) {
    for (int i = 0; i < S::STAGES; i++) {
      mbar_init(full_bar(i), 1);
      mbar_init(empty_bar(i), NT / 32);
    }
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }

  Place p;
  __shared__ DivideRoom<NT + (TMA ? 32 : 0)> room;
  const Share share = divide(a.tiling, a.batch, a.least, p, room);
  __syncthreads();
  if (TMA && warp == NT / 32) {
    // ---- the copying warp
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
    int page = share.units > 0 ? page_of(p) : -2;
    for (int u = 0; u < (int)share.units; u++) {
      const int st = u % S::STAGES, key0 = p.blk * BK, h = p.h, now = page;
      if (u >= S::STAGES && !__all_sync(0xffffffffu, role_wait(empty_bar(st), (uint32_t)((u / S::STAGES - 1) & 1),
                                                               abort_word, abort)))
        break;
      const int boxes = __popc(__ballot_sync(0xffffffffu, now != -2));
      if (lane == 0) mbar_expect_tx(full_bar(st), (uint32_t)((boxes << box_bits) * S::ROW * 2));
      __syncwarp();
      const uint32_t dst = base + (uint32_t)st * S::STAGE;
      for (int i0 = 0; i0 < per_block * S::CHUNKS * 2; i0 += 32) {
        const int i = i0 + lane, box = i & (per_block - 1), c = i >> per_bits;  // K's chunks, then V's
        const int from = __shfl_sync(0xffffffffu, now, box);
        if (c < S::CHUNKS * 2 && from != -2) {
          const int key = key0 + (box << box_bits), chunk = c % S::CHUNKS;
          const int slot = key - quotient(key, a.pools.by_page) * a.pools.page_size;
          tma_load_4d(dst + (uint32_t)(c / S::CHUNKS) * S::TILE + (uint32_t)chunk * BK * S::CHUNK +
                          (uint32_t)(box << box_bits) * S::CHUNK,
                      c < S::CHUNKS ? &k_map : &v_map, full_bar(st), chunk * S::WIDE, slot, h, from);
        }
        __syncwarp();
      }
      fetched = u + 1;
      advance(a.tiling, a.batch, p);
      if (u + 1 < (int)share.units) page = page_of(p);
    }
    // every copy has landed before the block releases its memory
    for (int u = max(0, fetched - S::STAGES); u < fetched; u++)
      mbar_wait(full_bar(u % S::STAGES), (uint32_t)((u / S::STAGES) & 1), abort_word);
    if (lane == 0) report_abort(a.batch.status, abort);
    return;
  }
  Cut cut{0, 0, 0, 0, 0};
  if (share.units > 0) {
    const int units = (int)share.units;
    Place kp = p;        // the block whose key addresses are looked up next
    int looked = 0;
    auto look_up = [&]() {  // addresses of block `looked` into slot looked % RING
      if (looked < units) {
        const int visible = tile_visible(a.tiling, kp.r, kp.tile);
        for (int i = tid; i < BK; i += NT) {
          const int key = kp.blk * BK + i;
          int64_t off = -1;
          if (key < visible) {
            off = key_offset(a.pools, a.batch, kp.b, kp.h, key);
            if (off < 0) report(a.batch.status, ET_B200_PAGED_BAD_PAGE);
          }
          koff[looked % S::RING * BK + i] = off;
        }
        advance(a.tiling, a.batch, kp);
      }
      looked++;
    };
    auto issue = [&](int u) {  // copies of unit u into stage u % STAGES
      if (u < units) {
        const uint32_t st = base + (uint32_t)(u % S::STAGES) * S::STAGE;
        for (int i = tid; i < BK * S::PIECES; i += NT) {
          const int row = i / S::PIECES, c = i % S::PIECES;
          const int64_t off = koff[u % S::RING * BK + row];
          const bool full = off >= 0 && c * (16 / (int)sizeof(T)) < dim;
          const int64_t e = full ? off + c * (16 / (int)sizeof(T)) : 0;
          const uint32_t dst = st + S::template at<BK>(row, c);
          cp16(dst, keys + e, full);
          cp16(dst + S::TILE, values + e, full);
        }
      }
      cp_commit();
    };
    if constexpr (!TMA) {
#pragma unroll
      for (int s = 0; s < S::STAGES; s++) look_up();
      __syncthreads();
#pragma unroll
      for (int s = 0; s < S::STAGES - 1; s++) issue(s);
    }

    auto load_queries = [&]() {  // the rows of the tile at p, rotated
      const int first_row = p.tile << a.tiling.row_bits, rows = min(BM, p.r.n * group - first_row);
      constexpr int PAIRS = BM * DH / 2, AT_ONCE = S::WM == 1 ? 8 : 1;  // loads in flight per thread
#pragma unroll(S::WM == 1 ? 1 : 4)
      for (int i0 = tid; i0 < PAIRS; i0 += NT * AT_ONCE) {
        T x[AT_ONCE][2];
        float cs[AT_ONCE], sn[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; k++) {
          const int i = i0 + k * NT, r = i / (DH / 2), d = 2 * (i % (DH / 2));
          x[k][0] = x[k][1] = from_f32<T>(0.0f);
          cs[k] = 1.0f;
          sn[k] = 0.0f;
          if (i < PAIRS && r < rows && d < dim) {
            const int t = quotient(first_row + r, a.tiling.by_group), j = first_row + r - t * group;
            const T* src = static_cast<const T*>(a.q) + (p.r.first + t) * a.q_stride +
                           (int64_t)(p.h * group + j) * dim + d;
            x[k][0] = src[0];
            x[k][1] = src[1];
            const int pos = p.r.len - p.r.n + t;
            if (a.rope.cos != nullptr && pos >= 0) {
              const int64_t at = rope_row(a.rope, pos, a.batch.status) * (dim / 2) + d / 2;
              cs[k] = __ldg(a.rope.cos + at);
              sn[k] = __ldg(a.rope.sin + at);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; k++) {
          const int i = i0 + k * NT, r = i / (DH / 2), d = 2 * (i % (DH / 2));
          if (i >= PAIRS) break;
          float x0 = to_f32<T>(x[k][0]), x1 = to_f32<T>(x[k][1]);
          if (a.rope.cos != nullptr) rotate(x0, x1, cs[k], sn[k]);
          if constexpr (std::is_same_v<T, __half>) {
            x0 *= a.q_factor;
            x1 *= a.q_factor;
          }
          const uint32_t at = S::template at<BM>(r, d * (int)sizeof(T) / 16) + (d * (int)sizeof(T)) % 16;
          T* dst = reinterpret_cast<T*>(smem + S::STAGES * S::STAGE + at);
          dst[0] = from_f32<T>(x0);
          dst[1] = from_f32<T>(x1);
          if constexpr (!F32) {  // and what the rounding left
            T* low = reinterpret_cast<T*>(smem + S::STAGES * S::STAGE + S::TILE_Q + at);
            low[0] = from_f32<T>(x0 - to_f32<T>(dst[0]));
            low[1] = from_f32<T>(x1 - to_f32<T>(dst[1]));
          }
        }
      }
    };
    load_queries();
    named_sync(1, NT);

    float o[DH / 8][4];
    float m[2], l[2];
    int vis[2], vis_min = 0;
    bool whole = false;  // this block began the tile
    bool ok = true;
    for (int u = 0; u < units; u++) {
      const int st = u % S::STAGES;
      if constexpr (TMA) {
        // after a wait that ran out the loop still ends, in step with the other warps
        if (ok)
          ok = __all_sync(0xffffffffu, role_wait(full_bar(st), (uint32_t)((u / S::STAGES) & 1),
                                                 abort_word, abort));
      } else {
        cp_wait<S::STAGES - 2>();
        __syncthreads();  // stage u is complete; stage u - 1 and its addresses are free
        issue(u + S::STAGES - 1);
        look_up();
      }
      const bool first = u == 0 || p.blk == 0;
      if (first) {  // a new tile
        whole = p.blk == 0;
        const int rows = min(BM, p.r.n * group - (p.tile << a.tiling.row_bits));
        if (u > 0) {
          if (TMA) named_sync(1, NT);  // every warp is done with the last tile's queries
          load_queries();
        }
#pragma unroll
        for (int i = 0; i < DH / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; i++) {
          m[i] = -INFINITY;
          l[i] = 0.0f;
          const int r = wm * 16 + lane / 4 + 8 * i, g = (p.tile << a.tiling.row_bits) + r;
          vis[i] = r < rows ? max(0, p.r.len - p.r.n + quotient(g, a.tiling.by_group) + 1) : 0;
        }
        vis_min = rows == BM ? max(0, p.r.len - p.r.n +
                                          quotient(p.tile << a.tiling.row_bits, a.tiling.by_group) + 1)
                             : 0;
        if (u > 0) named_sync(1, NT);
      }
      const uint32_t kt = base + (uint32_t)st * S::STAGE, vt = kt + S::TILE;
      if (TMA && p.blk + 1 == p.nblk) {
        // slots behind the tile's keys may hold anything: this warp's rows of V
        const int valid = tile_visible(a.tiling, p.r, p.tile) - p.blk * BK;
        if (valid < (wk + 1) * KW) {
          for (int row = max(valid, wk * KW); row < (wk + 1) * KW; row++)
            for (int c = lane; c < S::PIECES; c += 32)
              sts128(vt + S::template at<BK>(row, c), make_float4(0.f, 0.f, 0.f, 0.f));
          __syncwarp();
        }
      }

      // scores of this warp's KW keys
      float s[KW / 8][4];
#pragma unroll
      for (int i = 0; i < KW / 8; i++) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < DH / KSTEP; ks++) {
        uint32_t qa[4];
        ldsm4(qa, qs + S::template at<BM>(wm * 16 + (lane & 15), 2 * ks + (lane >> 4)));
        uint32_t qh[4], ql[4];
        if constexpr (F32) {
#pragma unroll
          for (int i = 0; i < 4; i++) pair_tf32(qa[i], qh[i], ql[i]);
        } else {
          ldsm4(ql, qs + S::TILE_Q + S::template at<BM>(wm * 16 + (lane & 15), 2 * ks + (lane >> 4)));
        }
#pragma unroll
        for (int n = 0; n < KW / 16; n++) {
          uint32_t kb[4];
          ldsm4(kb, kt + S::template at<BK>(wk * KW + 16 * n + ((lane >> 4) << 3) + (lane & 7),
                               2 * ks + ((lane >> 3) & 1)));
          if constexpr (F32) {
            uint32_t kh[4], kl[4];
#pragma unroll
            for (int i = 0; i < 4; i++) pair_tf32(kb[i], kh[i], kl[i]);
#pragma unroll
            for (int i = 0; i < 2; i++) {
              // the tensor pipe's accumulation truncates: eight dims at a time, added in f32
              float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma_tf32(part, ql, kh[2 * i], kh[2 * i + 1]);
              mma_tf32(part, qh, kl[2 * i], kl[2 * i + 1]);
              mma_tf32(part, qh, kh[2 * i], kh[2 * i + 1]);
#pragma unroll
              for (int e = 0; e < 4; e++) s[2 * n + i][e] += part[e];
            }
          } else {
            mma16<T>(s[2 * n], ql, kb[0], kb[1]);
            mma16<T>(s[2 * n + 1], ql, kb[2], kb[3]);
            mma16<T>(s[2 * n], qa, kb[0], kb[1]);
            mma16<T>(s[2 * n + 1], qa, kb[2], kb[3]);
          }
        }
      }
      // running maxima, probabilities (rows lane / 4 and lane / 4 + 8)
      const int key0 = p.blk * BK + wk * KW;
      const bool full = key0 + KW <= vis_min;
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < KW / 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int key = key0 + 8 * i + 2 * (lane & 3) + (e & 1);
          s[i][e] = full || key < vis[e >> 1] ? s[i][e] * a.scale_log2 : -INFINITY;
          top[e >> 1] = fmaxf(top[e >> 1], s[i][e]);
        }
      float factor[2], from[2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        const float now = fmaxf(m[i], top[i]);
        from[i] = now == -INFINITY ? 0.0f : now;
        factor[i] = ex2(m[i] - from[i]);
        m[i] = now;
        l[i] *= factor[i];
      }
#pragma unroll
      for (int i = 0; i < KW / 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          s[i][e] = ex2(s[i][e] - (from[e >> 1] - kShift));
          l[e >> 1] += s[i][e];
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
      // o += P V
      if constexpr (F32) {
        // key 2 (lane % 4) + {0, 1} of each 8 stands at matrix k lane % 4 + {0, 4},
        // so the score registers are the A operand as they lie
#pragma unroll
        for (int kk = 0; kk < KW / 8; kk++) {
          uint32_t ph[4], pl[4];
#pragma unroll
          for (int i = 0; i < 4; i++)
            pair_tf32(__float_as_uint(s[kk][((i & 1) << 1) | (i >> 1)]), ph[i], pl[i]);
          const int row = wk * KW + 8 * kk + 2 * (lane & 3);
#pragma unroll
          for (int n = 0; n < DH / 8; n++) {
            const int d = 8 * n + lane / 4;
            uint32_t vh[2], vl[2];
#pragma unroll
            for (int i = 0; i < 2; i++)
              pair_tf32(lds32(vt + S::template at<BK>(row + i, d / 4) + 4 * (d & 3)), vh[i], vl[i]);
            // eight keys at a time, as above
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma_tf32(part, pl, vh[0], vh[1]);
            mma_tf32(part, ph, vl[0], vl[1]);
            mma_tf32(part, ph, vh[0], vh[1]);
#pragma unroll
            for (int i = 0; i < 4; i++) o[n][i] += part[i];
          }
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < KW / 16; kk++) {
          uint32_t pa[4];
#pragma unroll
          for (int i = 0; i < 4; i++)
            pa[i] = pack2<T>(s[2 * kk + (i >> 1)][2 * (i & 1)], s[2 * kk + (i >> 1)][2 * (i & 1) + 1]);
#pragma unroll
          for (int n = 0; n < DH / 16; n++) {
            uint32_t vb[4];
            ldsm4t(vb, vt + S::template at<BK>(wk * KW + 16 * kk + (lane & 15), 2 * n + (lane >> 4)));
            mma16<T>(o[2 * n], pa, vb[0], vb[1]);
            mma16<T>(o[2 * n + 1], pa, vb[2], vb[3]);
          }
        }
      }

      const bool tile_ends = p.blk + 1 == p.nblk;
      if (tile_ends || u + 1 == units) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
          l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
        const int r0 = wm * 16 + lane / 4;
        if constexpr (WK > 1) {
          named_sync(1, NT);  // every warp is done with the stage
          float* merge = reinterpret_cast<float*>(smem + st * S::STAGE);
          if ((lane & 3) == 0) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              join_m[wk * BM + r0 + 8 * i] = m[i];
              join_l[wk * BM + r0 + 8 * i] = l[i];
            }
          }
          if (wk > 0) {
            float* mine = merge + ((wk - 1) * S::WM + wm) * 16 * DH + lane * 4;
#pragma unroll
            for (int n = 0; n < DH / 8; n++)
              *reinterpret_cast<float4*>(mine + n * 128) = make_float4(o[n][0], o[n][1], o[n][2], o[n][3]);
          }
          named_sync(1, NT);
          if (wk == 0) {
            float f[WK][2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
              float all = m[i];
#pragma unroll
              for (int w = 1; w < WK; w++) all = fmaxf(all, join_m[w * BM + r0 + 8 * i]);
              const float ref = all == -INFINITY ? 0.0f : all;
              f[0][i] = ex2(m[i] - ref);
              l[i] *= f[0][i];
#pragma unroll
              for (int w = 1; w < WK; w++) {
                f[w][i] = ex2(join_m[w * BM + r0 + 8 * i] - ref);
                l[i] += f[w][i] * join_l[w * BM + r0 + 8 * i];
              }
              m[i] = all;
            }
#pragma unroll
            for (int n = 0; n < DH / 8; n++) {
#pragma unroll
              for (int e = 0; e < 4; e++) o[n][e] *= f[0][e >> 1];
#pragma unroll
              for (int w = 1; w < WK; w++) {
                const float4 x = *reinterpret_cast<const float4*>(
                    merge + ((w - 1) * S::WM + wm) * 16 * DH + n * 128 + lane * 4);
                o[n][0] += f[w][0] * x.x;
                o[n][1] += f[w][0] * x.y;
                o[n][2] += f[w][1] * x.z;
                o[n][3] += f[w][1] * x.w;
              }
            }
          }
        }
        const bool done = whole && tile_ends;
        if (wk == 0) {
          const int slot = 2 * (int)blockIdx.x + (whole ? 1 : 0);
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const int r = r0 + 8 * i, g = (p.tile << a.tiling.row_bits) + r;
            if (done) {
              if (g < p.r.n * group) {
                const int by = quotient(g, a.tiling.by_group), h = p.h * group + g - by * group;
                const int64_t t = p.r.first + by;
                const float inv = l[i] > 0.0f ? 1.0f / l[i] : 0.0f;
                T* dst = static_cast<T*>(a.o) + t * a.o_stride + (int64_t)h * dim;
#pragma unroll
                for (int n = 0; n < DH / 8; n++) {
                  const int d = 8 * n + 2 * (lane & 3);
                  if (d < dim) store2<T>(dst + d, o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
                }
                if (a.lse != nullptr && (lane & 3) == 0)
                  a.lse[t * a.q_heads + h] = l[i] > 0.0f ? (m[i] - kShift) * kLn2 + logf(l[i]) : -INFINITY;
              }
            } else {
              float* dst = a.joint.sums + ((int64_t)slot * BM + r) * DH;
#pragma unroll
              for (int n = 0; n < DH / 8; n++)
                *reinterpret_cast<float2*>(dst + 8 * n + 2 * (lane & 3)) =
                    make_float2(o[n][2 * i], o[n][2 * i + 1]);
              if ((lane & 3) == 0) {
                a.joint.stats[(int64_t)slot * 2 * BM + r] = m[i] - kShift;
                a.joint.stats[((int64_t)slot * 2 + 1) * BM + r] = l[i];
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
        if (lane == 0) mbar_arrive(empty_bar(st));
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

// Joins the parts of the tiles that the thread blocks blockIdx.x, blockIdx.x +
// gridDim.x, ... (of `blocks`) of the attention began and did not finish;
// blockIdx.y takes its share of the rows.  A large tile of up to 8 parts takes the lanes
// that read a row in 16-byte pieces per row (with the tcgen05 kernels' many rows and two
// or three parts, rows in turn took 35 us of the f32 prompts' 154; a warp a row of 64 dims
// 15 us where this takes 11); more parts take the block: warp w
// parts w, w + 8, ..., 4 dims per lane, several parts' loads in flight, and
// shared memory adds the warps up in order.
constexpr int JOIN_WARPS = 8;
template <typename T, int DH>
__global__ void __launch_bounds__(32 * JOIN_WARPS) paged_join_kernel(AttendArgs a, int blocks) {
  constexpr int V = DH >= 128 ? DH / 32 : 4, LANES = DH / V;  // dims per lane, lanes used
  __shared__ float sums[JOIN_WARPS][DH];
  __shared__ float totals[JOIN_WARPS];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int rows = 1 << a.tiling.row_bits, group = a.tiling.group;
  const int dim = a.pools.head_dim, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int c = blockIdx.x; c < blocks; c += gridDim.x) {
    const Cut cut = a.joint.cuts[c];
    if (cut.parts == 0) continue;
    auto slot_of = [&](int part) { return part == 0 ? 2 * c + 1 : 2 * (c + part); };
    if (rows > 16 && cut.parts <= JOIN_WARPS) {
      // 16 bytes of a part at a time, so as many rows as the warp has lanes for at once
      constexpr int W = DH / 32 > 4 ? DH / 32 : 4, LANES_ROW = DH / W, AT_ONCE = 32 / LANES_ROW;
      const int sub = lane / LANES_ROW, in = lane % LANES_ROW;
      for (int r0 = (blockIdx.y * JOIN_WARPS + warp) * AT_ONCE; r0 < rows; r0 += gridDim.y * JOIN_WARPS * AT_ONCE) {
        const int r = r0 + sub, g = (cut.tile << a.tiling.row_bits) + r;
        if (g - sub >= cut.n * group) break;
        const bool mine = in < cut.parts;
        const int64_t s = mine ? slot_of(in) : 0;
        const float m1 = mine ? a.joint.stats[s * 2 * rows + r] : -INFINITY;
        const float l1 = mine ? a.joint.stats[(s * 2 + 1) * rows + r] : 0.0f;
        float m = m1;
#pragma unroll
        for (int o = 1; o < LANES_ROW; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float ref = m == -INFINITY ? 0.0f : m;
        const float f1 = ex2(m1 - ref), lf = scaled(l1, m1 - ref);
        // in the order of the parts, as below
        float l = 0.0f, x[W];
#pragma unroll
        for (int k = 0; k < W; k++) x[k] = 0.0f;
#pragma unroll 2
        for (int i = 0; i < cut.parts; i++) {
          const float f = __shfl_sync(0xffffffffu, f1, sub * LANES_ROW + i);
          l += __shfl_sync(0xffffffffu, lf, sub * LANES_ROW + i);
          const float* src = a.joint.sums + ((int64_t)slot_of(i) * rows + r) * DH + in * W;
#pragma unroll
          for (int k = 0; k < W; k += 4) {
            const float4 y = *reinterpret_cast<const float4*>(src + k);
            x[k] += f * y.x; x[k + 1] += f * y.y; x[k + 2] += f * y.z; x[k + 3] += f * y.w;
          }
        }
        if (g >= cut.n * group) continue;
        const int by = quotient(g, a.tiling.by_group), h = cut.h * group + g - by * group;
        const int64_t t = cut.first + by;
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        T* dst = static_cast<T*>(a.o) + t * a.o_stride + (int64_t)h * dim + in * W;
#pragma unroll
        for (int k = 0; k < W; k += 2)
          if (in * W + k < dim) store2<T>(dst + k, x[k] * inv, x[k + 1] * inv);
        if (a.lse != nullptr && in == 0)
          a.lse[t * a.q_heads + h] = l > 0.0f ? m * kLn2 + logf(l) : -INFINITY;
      }
      continue;
    }
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
      const int g = (cut.tile << a.tiling.row_bits) + r;
      if (g >= cut.n * group) break;
      float m = -INFINITY;
      for (int i = lane; i < cut.parts; i += 32)
        m = fmaxf(m, a.joint.stats[(int64_t)slot_of(i) * 2 * rows + r]);
      m = warp_max(m);
      const float ref = m == -INFINITY ? 0.0f : m;
      float l = 0.0f, x[V];
#pragma unroll
      for (int k = 0; k < V; k++) x[k] = 0.0f;
#pragma unroll 4
      for (int i = warp; i < cut.parts; i += JOIN_WARPS) {
        const int64_t s = slot_of(i);
        const float below = a.joint.stats[s * 2 * rows + r] - ref, f = ex2(below);
        l += scaled(a.joint.stats[(s * 2 + 1) * rows + r], below);
        if (lane < LANES) {
          const float* src = a.joint.sums + (s * rows + r) * DH + lane * V;
#pragma unroll
          for (int k = 0; k < V; k += 4) {
            const float4 y = *reinterpret_cast<const float4*>(src + k);
            x[k] += f * y.x; x[k + 1] += f * y.y; x[k + 2] += f * y.z; x[k + 3] += f * y.w;
          }
        }
      }
      if (lane < LANES)
#pragma unroll
        for (int k = 0; k < V; k++) sums[warp][lane * V + k] = x[k];
      if (lane == 0) totals[warp] = l;
      __syncthreads();
      const int d = 2 * threadIdx.x, by = quotient(g, a.tiling.by_group), h = cut.h * group + g - by * group;
      const int64_t t = cut.first + by;
      if (d < dim || threadIdx.x == 0) {
        float total = 0.0f, y0 = 0.0f, y1 = 0.0f;
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; w++) {
          total += totals[w];
          y0 += sums[w][d];
          y1 += sums[w][d + 1];
        }
        const float inv = total > 0.0f ? 1.0f / total : 0.0f;
        store2<T>(static_cast<T*>(a.o) + t * a.o_stride + (int64_t)h * dim + d, y0 * inv, y1 * inv);
        if (a.lse != nullptr && threadIdx.x == 0)
          a.lse[t * a.q_heads + h] = total > 0.0f ? m * kLn2 + logf(total) : -INFINITY;
      }
      __syncthreads();
    }
  }
}

// ---- launching --------------------------------------------------------------------------

template <typename T, int DH>
void launch_join(const AttendArgs& a, int blocks, int64_t rows, cudaStream_t stream) {
  if (cudaPeekAtLastError() != cudaSuccess) return;  // no parts were left to join
  cudaLaunchConfig_t cfg{};
  // a row per thread block for as many rows as a tile is likely to have (the
  // kernel walks any number)
  cfg.gridDim = dim3(blocks < a.sms ? blocks : a.sms, rows < 1 ? 1 : rows < 16 ? rows : 16);
  cfg.blockDim = dim3(32 * JOIN_WARPS);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, paged_join_kernel<T, DH>, a, blocks);
  count_launch();
}

template <typename T, typename S>
void launch_shape(const et_b200_paged_cache_v1* c, AttendArgs& a, int64_t max_new, void* ws,
                  cudaStream_t stream) {
  int box_bits = 0;
  while ((2 << box_bits) <= (c->page_size < S::BK ? c->page_size : S::BK)) box_bits++;
  CUtensorMap k_map, v_map;
  const bool tma = pool_map(&k_map, c->keys, c, S::WIDE, 1 << box_bits) &&
                   pool_map(&v_map, c->values, c, S::WIDE, 1 << box_bits);
  const int sms = a.sms;
  const int resident = tma ? resident_blocks<paged_attention_kernel<T, S, true>>(S::NT + 32, S::SMEM)
                           : resident_blocks<paged_attention_kernel<T, S, false>>(S::NT, S::SMEM);
  const int blocks = thread_blocks(a, resident * sms, S::BM, S::BK);
  a.tiling = tiling_of(S::bits(S::BM), S::bits(S::BK), a.tiling.group, a.pools.kv_heads);
  a.least = 1;
  a.joint = joint_of(ws, blocks, S::BM, S::DH);
  if (tma)
    paged_attention_kernel<T, S, true><<<blocks, S::NT + 32, S::SMEM, stream>>>(k_map, v_map, a, box_bits);
  else
    paged_attention_kernel<T, S, false><<<blocks, S::NT, S::SMEM, stream>>>(k_map, v_map, a, box_bits);
  count_launch();
  launch_join<T, S::DH>(a, blocks, max_new * a.tiling.group, stream);
}

template <typename T, int DH>
void launch_dim(const et_b200_paged_cache_v1* c, AttendArgs& a, int64_t max_new, void* ws,
                cudaStream_t stream) {
  constexpr bool F32 = sizeof(T) == 4;
  // up to 16 rows per kv head: one row tile, warps along the keys; more: 64-row
  // tiles, every warp walks all keys
  if (max_new * a.tiling.group <= 16) {
    if constexpr (F32 && DH == 256) launch_shape<T, Shape<T, DH, 1, 2, 32, 3>>(c, a, max_new, ws, stream);
    else launch_shape<T, Shape<T, DH, 1, 4, 64, 3>>(c, a, max_new, ws, stream);
  } else {
    if constexpr (F32 && DH == 256) launch_shape<T, Shape<T, DH, 4, 1, 32, 2>>(c, a, max_new, ws, stream);
    else launch_shape<T, Shape<T, DH, 4, 1, 64, 2>>(c, a, max_new, ws, stream);
  }
}

template <typename T>
void launch_type(const et_b200_paged_cache_v1* c, AttendArgs& a, int64_t max_new, void* ws,
                 cudaStream_t stream) {
  {
    if (max_new * a.tiling.group > 16) {
      const int blocks = sizeof(T) == 2 ? attend_tc(c, a, ws, stream) : attend_f32(c, a, ws, stream);
      if (blocks > 0)
        return c->head_dim <= 64 ? launch_join<T, 64>(a, blocks, 16, stream)
                                 : launch_join<T, 128>(a, blocks, 16, stream);
    }
  }
  switch (padded(a.pools.head_dim)) {
    case 32: return launch_dim<T, 32>(c, a, max_new, ws, stream);
    case 64: return launch_dim<T, 64>(c, a, max_new, ws, stream);
    case 128: return launch_dim<T, 128>(c, a, max_new, ws, stream);
    default: return launch_dim<T, 256>(c, a, max_new, ws, stream);
  }
}

template <typename T>
void join_type(const AttendArgs& a, int dim_padded, int blocks, int64_t rows, cudaStream_t stream) {
  switch (dim_padded) {
    case 64: return launch_join<T, 64>(a, blocks, rows, stream);
    case 128: return launch_join<T, 128>(a, blocks, rows, stream);
    default: return launch_join<T, 256>(a, blocks, rows, stream);
  }
}

}  // namespace

namespace paged {

size_t attention_workspace(int64_t head_dim, int sms) {
  const int dim = padded(head_dim);
  const size_t plain = joint_bytes(kMostPerSm * sms, 64, dim), tc = attend_tc_workspace(dim, sms);
  return plain > tc ? plain : tc;
}

bool heads_fit(int64_t kv_heads, int64_t q_heads) {
  return q_heads >= 1 && q_heads <= 65536 && q_heads % kv_heads == 0;
}

int32_t check_attention(const et_b200_paged_batch_v1* b, int64_t head_dim, int64_t size,
                        int64_t q_heads, const void* q, int64_t q_stride, const void* o,
                        int64_t o_stride, const float* lse, const void* workspace, size_t bytes,
                        size_t need, et_kernel_error* e, const char* op) {
  const int64_t row = q_heads * head_dim;
  if (q == nullptr || o == nullptr)
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_NULL_ARGUMENT, op,
                     "q and o are required");
  if (q_stride < row || o_stride < row || q_stride > (int64_t)1 << 31 ||
      o_stride > (int64_t)1 << 31)
    return set_error(e, ET_KERNEL_ERROR_NONCONTIGUOUS, ET_KERNEL_CODE_INVALID_BUFFER, op,
                     "rows of q or o overlap or lie too far apart");
  if (!aligned_to(size, q, o) || !aligned_to(4, lse))
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_INVALID_BUFFER, op,
                     "q, o and lse must be aligned to their elements");
  if (b->tokens * q_heads > INT32_MAX - 4096)
    return set_error(e, ET_KERNEL_ERROR_SHAPE_MISMATCH, ET_KERNEL_CODE_INVALID_SHAPE, op,
                     "tokens times q_heads must stay below 2^31");
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0 ||
      bytes < need)
    return set_error(e, ET_KERNEL_ERROR_INVALID_ARGUMENT, ET_KERNEL_CODE_BUFFER_TOO_SMALL, op,
                     "workspace is smaller than the call's workspace_bytes_v1 asks for or not "
                     "256-byte aligned");
  return 0;
}

void join_parts(const AttendArgs& a, uint32_t dtype, int dim_padded, int blocks, int64_t rows,
                cudaStream_t stream) {
  if (dtype == ET_B200_DTYPE_F32) join_type<float>(a, dim_padded, blocks, rows, stream);
  else if (dtype == ET_B200_DTYPE_F16) join_type<__half>(a, dim_padded, blocks, rows, stream);
  else join_type<__nv_bfloat16>(a, dim_padded, blocks, rows, stream);
}

}  // namespace paged
}  // namespace etb

using namespace etb;
using namespace etb::paged;

extern "C" {

size_t et_b200_paged_attention_workspace_bytes_v1(const et_b200_paged_cache_v1* c,
                                                  int64_t q_heads) {
  if (check_cache(c, nullptr, "paged-attention-workspace") || !heads_fit(c->kv_heads, q_heads)) return 0;
  return attention_workspace(c->head_dim, sm_count());
}

int32_t et_b200_paged_attention_v1(const et_b200_paged_cache_v1* c,
                                   const et_b200_paged_batch_v1* b,
                                   const et_b200_paged_rope_v1* rope, int64_t q_heads,
                                   const void* q, int64_t q_stride, void* o, int64_t o_stride,
                                   float* lse, void* workspace, size_t bytes, void* stream,
                                   et_kernel_error* e) {
  const char* op = "paged-attention";
  if (int32_t r = check_cache(c, e, op)) return r;
  if (int32_t r = check_batch(b, c->page_size, e, op)) return r;
  if (int32_t r = check_rope(rope, e, op)) return r;
  if (!heads_fit(c->kv_heads, q_heads))
    return set_error(e, ET_KERNEL_ERROR_SHAPE_MISMATCH, ET_KERNEL_CODE_INVALID_SHAPE, op,
                     "q_heads must be a multiple of the cache's kv_heads, up to 65536");
  if (b->tokens > 0 && b->batch > 0) {
    const int sms = sm_count();
    if (int32_t r = check_attention(b, c->head_dim, c->dtype == ET_B200_DTYPE_F32 ? 4 : 2, q_heads,
                                    q, q_stride, o, o_stride, lse, workspace, bytes,
                                    attention_workspace(c->head_dim, sms), e, op))
      return r;
    AttendArgs a{};
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
    a.q_factor = c->dtype == ET_B200_DTYPE_F16 && a.rope.cos != nullptr ? 0.5f : 1.0f;
    a.scale_log2 = kLog2e / sqrtf((float)c->head_dim) / a.q_factor;
    auto st = static_cast<cudaStream_t>(stream);
    const int64_t max_new = least_of(b->max_new, (int64_t)INT32_MAX);  // times group fits
    if (c->dtype == ET_B200_DTYPE_F32) launch_type<float>(c, a, max_new, workspace, st);
    else if (c->dtype == ET_B200_DTYPE_F16) launch_type<__half>(c, a, max_new, workspace, st);
    else launch_type<__nv_bfloat16>(c, a, max_new, workspace, st);
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return cuda_error(e, status, op);
  }
  if (e) memset(e, 0, sizeof(*e));
  return 0;
}

}  // extern "C"
