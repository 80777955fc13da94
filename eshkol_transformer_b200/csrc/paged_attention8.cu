// Causal attention of new tokens over an 8-bit paged cache
// (et_b200_paged_attention8_v1): the kernel for any page size, head_dim and type.
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
// f16 the queries do.
//
// Up to 16 rows (WK > 1) warps split the keys and convert fragments as they load them:
// a thread's four neighbouring bytes of a key are the two register pairs that a 16-deep
// product wants if dims are numbered that way, which the queries' layout follows; of V the
// transposed load brings two dims of two keys, which one byte permutation turns into
// two pairs of keys, for two products whose columns are the even and the odd dims.
// More rows (WK == 1): four warps convert a block together to binary16 tiles first.
#include <math.h>

#include <type_traits>

#include "paged8.cuh"
#include "paged_mma.cuh"

namespace etb {
namespace {

using namespace paged;

// log2 of the largest weight: D is within 1/2 of the largest exponent, c below 2
constexpr float kShift = 13.0f;

template <typename T, int DH_, int WM_, int WK_, int BK_, int STAGES_>
struct Shape8 {
  static constexpr int DH = DH_, WM = WM_, WK = WK_, BK = BK_, STAGES = STAGES_;
  static constexpr int NT = 32 * WM * WK, BM = 16 * WM, KW = BK / WK;
  static constexpr bool CONVERT = WK == 1;  // tiles of binary16 in shared memory
  static constexpr bool QLO = !std::is_same_v<T, __nv_bfloat16>, PLO = sizeof(T) == 4;
  static constexpr int ROW = DH, PIECES = ROW / 16;  // bytes of one key
  static constexpr int TILE = BK * ROW, STAGE = 2 * TILE;
  static constexpr int TILE_Q = BM * DH * 2, TILE_16 = BK * DH * 2;
  static constexpr int Q = STAGES * STAGE;
  static constexpr int CONV = Q + TILE_Q * (QLO ? 2 : 1);
  static constexpr int SCALES = CONV + (CONVERT ? 2 * TILE_16 : 0);  // [STAGES][keys, values][BK]
  static constexpr int MERGE = (WK - 1) * BM * DH * 4;
  static constexpr int RING = STAGES + 1;  // blocks with known pages
  static constexpr int PAGES = SCALES + STAGES * 2 * BK * 4;
  static constexpr int QMUL = PAGES + RING * (BK * 4 + 16);
  static constexpr int JOIN = QMUL + BM * 4;
  static constexpr int BARS = JOIN + WK * BM * 8;
  static constexpr int SMEM = BARS + 2 * STAGES * 8 + 16;
  static constexpr int CHUNK = ROW < 128 ? ROW : 128, CHUNKS = ROW / CHUNK;
  static constexpr int PER_SM = 2 * (SMEM + 2048) <= 233472 ? 2 : 1;  // blocks the registers must allow
  static constexpr int bits(int n) { return n <= 1 ? 0 : 1 + bits(n / 2); }
  static_assert(1 << bits(BM) == BM && 1 << bits(BK) == BK, "powers of two");
  static_assert(KW % 16 == 0 && DH % 64 == 0, "whole products");
  static_assert(MERGE <= STAGE, "the joining of warps reuses a stage");
  static_assert(SMEM <= 232448 && BARS % 8 == 0, "shared memory");
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

template <typename T, typename S, bool TMA>
__global__ void __launch_bounds__(S::NT + (TMA ? 32 : 0), S::PER_SM)
paged_attention8_kernel(const __grid_constant__ CUtensorMap k_map,
                        const __grid_constant__ CUtensorMap v_map, Attend8Args args, int box_bits) {
  constexpr int DH = S::DH, BM = S::BM, BK = S::BK, KW = S::KW, NT = S::NT, WK = S::WK;
  constexpr bool CONVERT = S::CONVERT, QLO = S::QLO, PLO = S::PLO;
  const AttendArgs& a = args.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* scales_s = reinterpret_cast<float*>(smem + S::SCALES);
  float* qmul = reinterpret_cast<float*>(smem + S::QMUL);
  float* join_m = reinterpret_cast<float*>(smem + S::JOIN);
  float* join_l = join_m + WK * BM;
  const uint32_t base = smem_u32(smem);
  const uint32_t qs = base + S::Q;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wm = warp / WK, wk = warp % WK;
  const int dim = a.pools.head_dim, group = a.tiling.group;
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
      const int sound = __popc(__ballot_sync(0xffffffffu, now >= 0));
      float* sc = scales_s + st * 2 * BK + (lane << box_bits);
      if (now == -1)
        for (int i = 0; i < 1 << box_bits; i++) sc[i] = sc[BK + i] = 0.0f;
      __syncwarp();
      if (lane == 0)
        mbar_expect_tx(full_bar(st), (uint32_t)((boxes << box_bits) * S::ROW * 2 + (sound << box_bits) * 8));
      __syncwarp();
      if (now >= 0) {
        const int key = key0 + (lane << box_bits);
        const int slot = key - quotient(key, a.pools.by_page) * a.pools.page_size;
        const int64_t off = now * args.scales.page_stride + h * args.scales.head_stride + slot;
        bulk_load(smem_u32(sc), args.scales.keys + off, 4u << box_bits, full_bar(st));
        bulk_load(smem_u32(sc + BK), args.scales.values + off, 4u << box_bits, full_bar(st));
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
                      c < S::CHUNKS ? &k_map : &v_map, full_bar(st), chunk * S::CHUNK, slot, h, from);
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
    // without TMA: the pages of a block's keys, looked up one block ahead of its copies
    struct Ahead { int key0, h, unused[2]; };
    int* pages_s = reinterpret_cast<int*>(smem + S::PAGES);
    Ahead* ahead_s = reinterpret_cast<Ahead*>(smem + S::PAGES + S::RING * BK * 4);
    Place kp = p;
    int looked = 0;
    auto look_up = [&]() {  // pages of block `looked` into slot looked % RING
      if (looked < units) {
        const int visible = tile_visible(a.tiling, kp.r, kp.tile), at = looked % S::RING;
        if (tid == 0) ahead_s[at] = Ahead{kp.blk * BK, kp.h, {0, 0}};
        for (int i = tid; i < BK; i += NT) {
          const int key = kp.blk * BK + i;
          int page = -1;
          if (key < visible) {
            page = a.batch.table[(int64_t)kp.b * a.batch.columns + quotient(key, a.pools.by_page)];
            if (page < 0 || page >= a.pools.pages) {
              report(a.batch.status, ET_B200_PAGED_BAD_PAGE);
              page = -1;
            }
          }
          pages_s[at * BK + i] = page;
        }
        advance(a.tiling, a.batch, kp);
      }
      looked++;
    };
    auto issue = [&](int u) {  // copies of unit u into stage u % STAGES
      if (u < units) {
        const uint32_t st = base + (uint32_t)(u % S::STAGES) * S::STAGE;
        const uint32_t sc = base + S::SCALES + (uint32_t)(u % S::STAGES) * 2 * BK * 4;
        const Ahead at = ahead_s[u % S::RING];
        auto slot_of = [&](int row) {
          const int key = at.key0 + row;
          return key - quotient(key, a.pools.by_page) * a.pools.page_size;
        };
        for (int i = tid; i < BK * S::PIECES; i += NT) {
          const int row = i / S::PIECES, c = i % S::PIECES, page = pages_s[u % S::RING * BK + row];
          const bool full = page >= 0 && c * 16 < dim;
          const int64_t e = !full ? 0
                                  : page * a.pools.page_stride + at.h * a.pools.head_stride +
                                        slot_of(row) * a.pools.token_stride + c * 16;
          const uint32_t dst = st + S::at8(row, c);
          cp16(dst, static_cast<const uint8_t*>(a.keys) + e, full);
          cp16(dst + S::TILE, static_cast<const uint8_t*>(a.values) + e, full);
        }
        for (int row = tid; row < BK; row += NT) {
          const int page = pages_s[u % S::RING * BK + row];
          const int64_t e = page < 0 ? 0
                                     : page * args.scales.page_stride + at.h * args.scales.head_stride +
                                           slot_of(row) * args.scales.token_stride;
          const int bytes = page < 0 ? 0 : 4;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(sc + 4u * row),
                       "l"(args.scales.keys + e), "r"(bytes) : "memory");
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(sc + 4u * (BK + row)),
                       "l"(args.scales.values + e), "r"(bytes) : "memory");
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

    // the rows of the tile at p, rotated: 8 lanes to a row, a row's lanes find its
    // largest magnitude, then binary16 of the row times 2^e
    auto load_queries = [&]() {
      const int first_row = p.tile << a.tiling.row_bits, rows = min(BM, p.r.n * group - first_row);
      constexpr int PAIRS = DH / 16;  // of a lane: its pairs are 8 apart, so neighbours read neighbours
#pragma unroll 1
      for (int r = tid / 8; r < BM; r += NT / 8) {
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
          const int in = (d & 15) / 2, to = CONVERT ? in : (in >> 1) + 4 * (in & 1);
          const uint32_t at = S::template at16<BM>(r, 2 * (d >> 4) + (to >> 2)) + 4 * (to & 3);
          const float y0 = y[i][0] * by, y1 = y[i][1] * by;
          const __half2 hi = __floats2half2_rn(y0, y1);
          *reinterpret_cast<__half2*>(smem + S::Q + at) = hi;
          if constexpr (QLO) {
            const float2 f = __half22float2(hi);
            *reinterpret_cast<__half2*>(smem + S::Q + S::TILE_Q + at) = __floats2half2_rn(y0 - f.x, y1 - f.y);
          }
        }
      }
    };
    load_queries();
    named_sync(1, NT);

    float o[DH / 8][4];
    // maxima of s and of s + x so far, sums of 2^(s - m), exponents D of o
    float m[2], l[2], big[2], dexp[2], mul[2];
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
        __syncthreads();  // stage u is complete; stage u - 1 and its pages are free
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
          named_sync(1, NT);
        }
#pragma unroll
        for (int i = 0; i < DH / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; i++) {
          m[i] = big[i] = -INFINITY;
          l[i] = dexp[i] = 0.0f;
          const int r = wm * 16 + lane / 4 + 8 * i, g = (p.tile << a.tiling.row_bits) + r;
          vis[i] = r < rows ? max(0, p.r.len - p.r.n + quotient(g, a.tiling.by_group) + 1) : 0;
          mul[i] = qmul[r];
        }
        vis_min = rows == BM ? max(0, p.r.len - p.r.n +
                                          quotient(p.tile << a.tiling.row_bits, a.tiling.by_group) + 1)
                             : 0;
      }
      const uint32_t kt = base + (uint32_t)st * S::STAGE, vt = kt + S::TILE;
      const float* ks_s = scales_s + st * 2 * BK;
      const float* vs_s = ks_s + BK;
      const bool tile_ends = p.blk + 1 == p.nblk;
      // slots behind the tile's keys may hold anything
      const int valid = tile_ends ? tile_visible(a.tiling, p.r, p.tile) - p.blk * BK : BK;
      if constexpr (CONVERT) {
        named_sync(1, NT);  // every warp is done with the last block's tiles
        for (int i = tid; i < BK * S::PIECES * 2; i += NT) {
          const int c = i % S::PIECES, row = i / S::PIECES % BK, v = i / (S::PIECES * BK);
          float4 raw = lds128((v ? vt : kt) + S::at8(row, c));
          if (v && row >= valid) raw = make_float4(0.f, 0.f, 0.f, 0.f);
          uint32_t h[8];
          halves_of(__float_as_uint(raw.x), h[0], h[1]);
          halves_of(__float_as_uint(raw.y), h[2], h[3]);
          halves_of(__float_as_uint(raw.z), h[4], h[5]);
          halves_of(__float_as_uint(raw.w), h[6], h[7]);
          const uint32_t to = base + S::CONV + (uint32_t)(v * S::TILE_16);
#pragma unroll
          for (int j = 0; j < 2; j++)
            sts128(to + S::template at16<BK>(row, 2 * c + j),
                   make_float4(__uint_as_float(h[4 * j]), __uint_as_float(h[4 * j + 1]),
                               __uint_as_float(h[4 * j + 2]), __uint_as_float(h[4 * j + 3])));
        }
        named_sync(1, NT);
      } else if (valid < (wk + 1) * KW) {  // this warp's rows of V
        for (int row = max(valid, wk * KW); row < (wk + 1) * KW; row++)
          for (int c = lane; c < S::PIECES; c += 32)
            sts128(vt + S::at8(row, c), make_float4(0.f, 0.f, 0.f, 0.f));
        __syncwarp();
      }

      // scores of this warp's KW keys
      float s[KW / 8][4];
#pragma unroll
      for (int i = 0; i < KW / 8; i++) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
      auto product = [&](float (&d)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4], uint32_t b0,
                         uint32_t b1) {
        if constexpr (PLO) {
          // the tensor pipe's accumulation truncates: 16 dims at a time, added in f32
          float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma16<__half>(part, lo, b0, b1);
          mma16<__half>(part, hi, b0, b1);
#pragma unroll
          for (int e = 0; e < 4; e++) d[e] += part[e];
        } else {
          if constexpr (QLO) mma16<__half>(d, lo, b0, b1);
          mma16<__half>(d, hi, b0, b1);
        }
      };
      auto query = [&](int ks, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
        const uint32_t at = S::template at16<BM>(wm * 16 + (lane & 15), 2 * ks + (lane >> 4));
        ldsm4(hi, qs + at);
        if constexpr (QLO) ldsm4(lo, qs + S::TILE_Q + at);
      };
      if constexpr (CONVERT) {
        const uint32_t k16 = base + S::CONV;
#pragma unroll
        for (int ks = 0; ks < DH / 16; ks++) {
          uint32_t qa[4], ql[4];
          query(ks, qa, ql);
#pragma unroll
          for (int n = 0; n < KW / 16; n++) {
            uint32_t kb[4];
            ldsm4(kb, k16 + S::template at16<BK>(16 * n + ((lane >> 4) << 3) + (lane & 7),
                                                 2 * ks + ((lane >> 3) & 1)));
            product(s[2 * n], qa, ql, kb[0], kb[1]);
            product(s[2 * n + 1], qa, ql, kb[2], kb[3]);
          }
        }
      } else {
#pragma unroll
        for (int k2 = 0; k2 < DH / 32; k2++) {  // 32 dims
          uint32_t qa[2][4], ql[2][4];
          query(2 * k2, qa[0], ql[0]);
          query(2 * k2 + 1, qa[1], ql[1]);
#pragma unroll
          for (int n = 0; n < KW / 16; n++) {
            uint32_t kb[4];  // 16 keys: pieces 2 k2 and 2 k2 + 1 of the lower 8, of the upper 8
            ldsm4(kb, kt + S::at8(wk * KW + 16 * n + ((lane >> 4) << 3) + (lane & 7),
                                  2 * k2 + ((lane >> 3) & 1)));
#pragma unroll
            for (int i = 0; i < 4; i++) {
              uint32_t b0, b1;
              halves_of(kb[i], b0, b1);
              product(s[2 * n + (i >> 1)], qa[i & 1], ql[i & 1], b0, b1);
            }
          }
        }
      }
      // scores times their keys' scales; value scales as 2^x c; running maxima (rows lane
      // / 4 and lane / 4 + 8)
      const int key0 = p.blk * BK + wk * KW;
      const bool full = key0 + KW <= vis_min;
      float xv[KW / 8][2], cv[KW / 8][2];
      float top[2] = {-INFINITY, -INFINITY}, tob[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < KW / 8; i++) {
        const int in = wk * KW + 8 * i + 2 * (lane & 3);
        const float2 ka = *reinterpret_cast<const float2*>(ks_s + in);
        const float2 vb = *reinterpret_cast<const float2*>(vs_s + in);
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float b = in + e < valid ? (e ? vb.y : vb.x) : 0.0f;
          const int x = min((int)(__float_as_uint(b) >> 23) & 255, 253);
          xv[i][e] = (float)(x - 127);
          cv[i][e] = b * __uint_as_float((uint32_t)(254 - x) << 23);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int key = key0 + 8 * i + 2 * (lane & 3) + (e & 1);
          const float y = s[i][e] * ((e & 1 ? ka.y : ka.x) * mul[e >> 1]);
          s[i][e] = full || key < vis[e >> 1] ? y : -INFINITY;
          top[e >> 1] = fmaxf(top[e >> 1], s[i][e]);
          tob[e >> 1] = fmaxf(tob[e >> 1], s[i][e] + xv[i][e & 1]);
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
        const float now = fmaxf(m[i], top[i]);
        big[i] = fmaxf(big[i], tob[i]);
        from[i] = now == -INFINITY ? 0.0f : now;
        const float d = now == -INFINITY ? 0.0f : rintf(big[i] - now), fall = m[i] - from[i];
        l[i] *= ex2(fall);
        factor[i] = ex2(fall + (dexp[i] - d));
        m[i] = now;
        dexp[i] = d;
      }
#pragma unroll
      for (int i = 0; i < KW / 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float y = s[i][e] - from[e >> 1];
          l[e >> 1] += ex2(y);
          s[i][e] = ex2(y + (xv[i][e & 1] - (dexp[e >> 1] - kShift))) * cv[i][e & 1];
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
#pragma unroll
      for (int kk = 0; kk < KW / 16; kk++) {
        uint32_t pa[4], pl[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float x = s[2 * kk + (i >> 1)][2 * (i & 1)], y = s[2 * kk + (i >> 1)][2 * (i & 1) + 1];
          const __half2 h = __floats2half2_rn(x, y);
          pa[i] = *reinterpret_cast<const uint32_t*>(&h);
          if constexpr (PLO) {
            const float2 f = __half22float2(h);
            pl[i] = pack2<__half>(x - f.x, y - f.y);
          }
        }
        auto weigh = [&](float (&d)[4], uint32_t b0, uint32_t b1) {
          if constexpr (PLO) {  // 16 keys at a time, as above
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma16<__half>(part, pl, b0, b1);
            mma16<__half>(part, pa, b0, b1);
#pragma unroll
            for (int e = 0; e < 4; e++) d[e] += part[e];
          } else {
            mma16<__half>(d, pa, b0, b1);
          }
        };
        if constexpr (CONVERT) {
          const uint32_t v16 = base + S::CONV + S::TILE_16;
#pragma unroll
          for (int n = 0; n < DH / 16; n++) {
            uint32_t vb[4];
            ldsm4t(vb, v16 + S::template at16<BK>(16 * kk + (lane & 15), 2 * n + (lane >> 4)));
            weigh(o[2 * n], vb[0], vb[1]);
            weigh(o[2 * n + 1], vb[2], vb[3]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < DH / 32; n++) {
            uint32_t vb[4];  // pieces 2 n and 2 n + 1, of each the lower and the upper 8 keys
            ldsm4t(vb, vt + S::at8(wk * KW + 16 * kk + (lane & 15), 2 * n + (lane >> 4)));
#pragma unroll
            for (int i = 0; i < 2; i++) {
              // bytes (key, dim): 00 01 10 11 -> 00 10 | 01 11: keys paired, even dim, odd dim
              uint32_t even[2], odd[2];
              halves_of(__byte_perm(vb[2 * i], 0, 0x3120), even[0], odd[0]);
              halves_of(__byte_perm(vb[2 * i + 1], 0, 0x3120), even[1], odd[1]);
              weigh(o[4 * n + 2 * i], even[0], even[1]);
              weigh(o[4 * n + 2 * i + 1], odd[0], odd[1]);
            }
          }
        }
      }

      // two neighbouring outputs at a time: f(dim, value, value) for row half i
      auto each_pair = [&](int i, auto f) {
#pragma unroll
        for (int n = 0; n < DH / 16; n++) {
          const int t = lane & 3;
          if constexpr (CONVERT) {
            f(16 * n + 2 * t, o[2 * n][2 * i], o[2 * n][2 * i + 1]);
            f(16 * n + 8 + 2 * t, o[2 * n + 1][2 * i], o[2 * n + 1][2 * i + 1]);
          } else {
            f(16 * n + 4 * t, o[2 * n][2 * i], o[2 * n + 1][2 * i]);
            f(16 * n + 4 * t + 2, o[2 * n][2 * i + 1], o[2 * n + 1][2 * i + 1]);
          }
        }
      };
      if (tile_ends || u + 1 == units) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
          l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
        // o relative to m alone
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const float d = dexp[i] - kShift, f0 = ex2(fmaxf(d, -120.0f)), f1 = ex2(fminf(d + 120.0f, 0.0f));
#pragma unroll
          for (int n = 0; n < DH / 8; n++) {
            o[n][2 * i] = o[n][2 * i] * f0 * f1;
            o[n][2 * i + 1] = o[n][2 * i + 1] * f0 * f1;
          }
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
                each_pair(i, [&](int d, float x, float y) {
                  if (d < dim) store2<T>(dst + d, x * inv, y * inv);
                });
                if (a.lse != nullptr && (lane & 3) == 0)
                  a.lse[t * a.q_heads + h] = l[i] > 0.0f ? m[i] * kLn2 + logf(l[i]) : -INFINITY;
              }
            } else {
              float* dst = a.joint.sums + ((int64_t)slot * BM + r) * DH;
              each_pair(i, [&](int d, float x, float y) {
                *reinterpret_cast<float2*>(dst + d) = make_float2(x, y);
              });
              if ((lane & 3) == 0) {
                a.joint.stats[(int64_t)slot * 2 * BM + r] = m[i];
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
  const int resident = tma ? resident_blocks<paged_attention8_kernel<T, S, true>>(S::NT + 32, S::SMEM)
                           : resident_blocks<paged_attention8_kernel<T, S, false>>(S::NT, S::SMEM);
  const int blocks = thread_blocks(a, resident * a.sms, S::BM, S::BK);
  a.tiling = tiling_of(S::bits(S::BM), S::bits(S::BK), a.tiling.group, a.pools.kv_heads);
  a.least = 1;
  a.joint = joint_of(ws, blocks, S::BM, S::DH);
  if (tma)
    paged_attention8_kernel<T, S, true><<<blocks, S::NT + 32, S::SMEM, stream>>>(k_map, v_map, x, box_bits);
  else
    paged_attention8_kernel<T, S, false><<<blocks, S::NT, S::SMEM, stream>>>(k_map, v_map, x, box_bits);
  count_launch();
  return blocks;
}

template <typename T, int DH>
int launch_dim8(const et_b200_paged_cache8_v1* c, Attend8Args& x, bool few, void* ws,
                cudaStream_t stream) {
  // few rows: one tile of 16, warps along the keys; more: tiles of 64, every warp all keys
  if (few) return launch_shape8<T, Shape8<T, DH, 1, 4, 128, 3>>(c, x, ws, stream);
  return launch_shape8<T, Shape8<T, DH, 4, 1, 64, 2>>(c, x, ws, stream);
}

template <typename T>
int launch_type8(const et_b200_paged_cache8_v1* c, Attend8Args& x, bool few, void* ws,
                 cudaStream_t stream) {
  if (!few && sizeof(T) == 2)
    if (const int blocks = attend8_tc(c, x, ws, stream)) return blocks;
  switch (padded8(c->head_dim)) {
    case 64: return launch_dim8<T, 64>(c, x, few, ws, stream);
    case 128: return launch_dim8<T, 128>(c, x, few, ws, stream);
    default: return launch_dim8<T, 256>(c, x, few, ws, stream);
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
    const bool few = rows <= 16;
    const int blocks = c->dtype == ET_B200_DTYPE_F32   ? launch_type8<float>(c, x, few, workspace, st)
                       : c->dtype == ET_B200_DTYPE_F16 ? launch_type8<__half>(c, x, few, workspace, st)
                                                       : launch_type8<__nv_bfloat16>(c, x, few, workspace, st);
    join_parts(a, c->dtype, padded8(c->head_dim), blocks, few ? rows : 16, st);
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return cuda_error(e, status, op);
  }
  if (e) memset(e, 0, sizeof(*e));
  return 0;
}

}  // extern "C"
