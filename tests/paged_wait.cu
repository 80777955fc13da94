// Bounded waits as the paged kernels use them (csrc/paged.cuh), on a barrier that
// nothing completes (some two seconds each): the wait that runs out ends the other
// warps' waits, from whatever warp it stands in, and is reported; waits on complete
// barriers succeed.
#include <stdio.h>

#include "attention_tc.cuh"
#include "paged.cuh"

using namespace etb;
using namespace etb::paged;

__global__ void waits(int* status, int* result) {
  __shared__ uint64_t bars[2];
  __shared__ int abort_s;
  volatile int* abort = &abort_s;
  const int warp = threadIdx.x / 32;
  const uint32_t never = smem_u32(&bars[0]), done = smem_u32(&bars[1]);
  if (threadIdx.x == 0) {
    mbar_init(never, 1);
    mbar_init(done, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    mbar_arrive(done);
  }
  __syncthreads();
  bool ok = true;
  if (warp == 1) ok = role_wait(never, 0, &abort_s, abort);
  if (warp == 2) {  // begins half a limit later and ends with the other
    const long long start = clock64();
    while (clock64() - start < kWaitCycles / 2) {}
    ok = role_wait(never, 0, &abort_s, abort);
    if (threadIdx.x % 32 == 0) result[7] = clock64() - start < kWaitCycles * 5 / 4;
  }
  if (warp == 3) ok = role_wait(done, 0, &abort_s, abort);
  if (threadIdx.x % 32 == 0) result[warp] = ok;
  __syncthreads();
  if (threadIdx.x == 0) {
    result[4] = *abort;
    report_abort(status, abort);
    result[5] = mbar_wait(done, 0, &abort_s);   // although aborted
    result[6] = mbar_wait(never, 0, &abort_s);
  }
}

__global__ void drains(int* status, int* result) {
  __shared__ uint64_t bar;
  __shared__ int abort_s;
  volatile int* abort = &abort_s;
  mbar_init(smem_u32(&bar), 1);
  *abort = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  result[0] = mbar_wait(smem_u32(&bar), 0, &abort_s);
  result[1] = *abort;
  report_abort(status, abort);
}

#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main() {
  int *device, host[9];
  CHECK(cudaMalloc(&device, sizeof(host)) == cudaSuccess);
  for (int with_status = 1; with_status >= 0; with_status--) {
    int* status = with_status ? device + 8 : nullptr;
    CHECK(cudaMemset(device, 0, sizeof(host)) == cudaSuccess);
    waits<<<1, 128>>>(status, device);
    CHECK(cudaMemcpy(host, device, sizeof(host), cudaMemcpyDeviceToHost) == cudaSuccess);
    CHECK(host[0] == 1 && host[1] == 0 && host[2] == 0 && host[3] == 1 && host[4] != 0);
    CHECK(host[5] == 1 && host[6] == 0 && host[7] == 1);
    CHECK(host[8] == (with_status ? ET_B200_PAGED_TIMEOUT : 0));
    CHECK(cudaMemset(device, 0, sizeof(host)) == cudaSuccess);
    drains<<<1, 1>>>(status, device);
    CHECK(cudaMemcpy(host, device, sizeof(host), cudaMemcpyDeviceToHost) == cudaSuccess);
    CHECK(host[0] == 0 && host[1] != 0 && host[8] == (with_status ? ET_B200_PAGED_TIMEOUT : 0));
  }
  printf("ok\n");
  return 0;
}
