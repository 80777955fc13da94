// Host run of the paged kernels' metadata arithmetic (csrc/paged.cuh): what
// leads outside the pools or tensors is clamped or refused, and walking the
// units of a batch visits every (request, head, tile, block) once, in order.
#include <stdio.h>

#include <vector>

#include "paged.cuh"

using namespace etb::paged;

#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main() {
  const int64_t offsets[] = {0, 3, 3, 9, 7, 40, -5, 12};
  const int64_t lengths[] = {5, 0, 100, 2, -1, 1ll << 40, 33};
  const int32_t table[7 * 3] = {0, 1, 2, 9, -1, 1 << 30, 3, 4, 5, 6, 7, 8, 0, 0, 0, 8, 9, 10, -7, 1, 2};
  Batch B{};
  B.offsets = offsets;
  B.lengths = lengths;
  B.table = table;
  B.tokens = 20;
  B.columns = 3;
  B.batch = 7;
  B.capacity = 30;
  for (int b = 0; b < 7; b++) {
    const Request r = load_request(B, b);
    CHECK(r.first >= 0 && r.n >= 0 && r.first + r.n <= B.tokens && r.len >= 0 && r.len <= B.capacity);
  }
  CHECK(load_request(B, 0).bad == 0 && load_request(B, 1).n == 0);
  CHECK(load_request(B, 2).bad == ET_B200_PAGED_BAD_LENGTH && load_request(B, 2).len == 30);
  CHECK(load_request(B, 3).bad == ET_B200_PAGED_BAD_OFFSET && load_request(B, 3).n == 0);
  CHECK(load_request(B, 4).bad == (ET_B200_PAGED_BAD_OFFSET | ET_B200_PAGED_BAD_LENGTH));
  CHECK(load_request(B, 4).n == 13);
  CHECK(load_request(B, 5).bad == (ET_B200_PAGED_BAD_OFFSET | ET_B200_PAGED_BAD_LENGTH));
  CHECK(load_request(B, 6).bad == (ET_B200_PAGED_BAD_OFFSET | ET_B200_PAGED_BAD_LENGTH));

  for (uint32_t d : {1u, 2u, 3u, 7u, 16u, 24u, 1000u, 65536u, (1u << 20) - 1, 1u << 20}) {
    const Divisor v = divisor_of(d);
    for (int64_t n = 0; n < (1ll << 31); n += 1 + n / 50) CHECK(quotient((int)n, v) == (int)(n / d));
    for (int64_t k = 1; k * d < (1ll << 31); k += 1 + k / 20)
      CHECK(quotient((int)(k * d), v) == k && quotient((int)(k * d) - 1, v) == k - 1);
    CHECK(quotient(INT32_MAX, v) == (int)(INT32_MAX / d));
  }

  Pools P{};
  P.pages = 10;
  P.page_size = 10;
  P.by_page = divisor_of(10);
  P.kv_heads = 2;
  P.head_dim = 8;
  P.token_stride = 8;
  P.head_stride = 80;
  P.page_stride = 160;
  for (int b = 0; b < 7; b++)
    for (int h = 0; h < 2; h++)
      for (int key = 0; key < 30; key++) {
        const int64_t at = key_offset(P, B, b, h, key);
        const int page = table[b * 3 + key / 10];
        if (page < 0 || page >= 10) CHECK(at == -1);
        else CHECK(at == page * 160 + h * 80 + key % 10 * 8 && at + 8 <= 10 * 160);
      }
  P.pages = 1 << 24;  // offsets beyond 32 bits
  P.page_stride = 1 << 20;
  const int32_t far = (1 << 24) - 1;
  Batch F = B;
  F.table = &far;
  F.columns = 1;
  CHECK(key_offset(P, F, 0, 1, 9) == (int64_t)far * (1 << 20) + 80 + 72);

  // walks: empty requests, more new tokens than keys, groups that straddle tiles
  const int64_t off2[] = {0, 0, 1, 1, 38, 45, 45, 300};
  const int64_t len2[] = {0, 900, 12, 37, 3, 0, 4000};
  Batch W{};
  W.offsets = off2;
  W.lengths = len2;
  W.tokens = 300;
  W.columns = 4096;
  W.batch = 7;
  W.capacity = 4096;
  for (int group : {1, 3, 8})
    for (int bits : {4, 6, 8}) {
      const int rows = 1 << bits;
      const Tiling t = tiling_of(bits, 6, group, 2);
      int64_t total = 0;
      for (int b = 0; b < 7; b++) total += head_units(t, load_request(W, b)) * 2;
      Place p{};
      p.b = -1;
      p.tiles = 1;  // the last unit of a request before the first
      p.h = 1;
      p.nblk = 1;
      int64_t seen = 0, rows_seen = 0;
      for (advance(t, W, p); p.b < W.batch; advance(t, W, p)) {
        seen++;
        CHECK(p.r.n > 0 && p.h < 2 && p.tile < tile_count(t, p.r) && p.blk < p.nblk);
        CHECK(p.blk == 0 || p.blk * 64 < tile_visible(t, p.r, p.tile));
        CHECK(p.blk + 1 < p.nblk || p.nblk * 64 >= tile_visible(t, p.r, p.tile));
        if (p.blk == 0)
          rows_seen += least_of(rows, p.r.n * group - p.tile * rows);
        CHECK(seen <= total);
      }
      CHECK(seen == total && rows_seen == 300 * group * 2);
    }
  printf("ok\n");
  return 0;
}
