// Host run of the paged kernels' arithmetic at the largest page table they accept:
// the number of thread blocks, the blocks of keys of the longest request and the keys
// that the last of them looks up.
#include <stdio.h>

#include "paged.cuh"

using namespace etb::paged;

#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main() {
  const int most = (int)kMostCapacity;
  const int64_t offsets[] = {0, 40};
  for (int page : {1, 8, 64, 1 << 20}) {
    const int columns = most / page, capacity = columns * page;
    for (int64_t length : {(int64_t)capacity, (int64_t)INT64_MAX, (int64_t)capacity - 130, (int64_t)70}) {
      Batch B{};
      B.offsets = offsets;
      B.lengths = &length;
      B.tokens = 40;
      B.columns = columns;
      B.batch = 1;
      B.capacity = capacity;
      const Request r = load_request(B, 0);
      CHECK(r.len == (length < capacity ? length : capacity) && r.n == 40);
      for (int key_bits : {5, 6, 7}) {
        AttendArgs a{};
        a.batch = B;
        a.pools.kv_heads = 1;
        a.tiling = tiling_of(7, key_bits, 2, 1);
        const int blocks = thread_blocks(a, 148, 128, 1 << key_bits);
        CHECK(blocks > 0 && blocks <= 148);
        const int units = tile_units(a.tiling, r, 0), keys = 1 << key_bits;
        CHECK(units == ((int64_t)r.len + keys - 1) / keys);
        // a lane's key of the last block, and of the block that is looked up ahead of it
        CHECK((int64_t)units * keys + 31 * 64 < INT32_MAX);
        CHECK(quotient(r.len - 1, divisor_of((uint32_t)page)) < columns);
      }
    }
  }
  printf("ok\n");
  return 0;
}
