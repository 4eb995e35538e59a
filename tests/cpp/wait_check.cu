// The bounded waits of tcgen05.cuh on a GPU, each with a limit of a few milliseconds: a wait ends
// when its barrier completes; one that nothing arrives on gives up, sets the abort flag and
// returns, and so do the CTA's other waits then. Settling waits for copies in flight whatever
// the abort flag says, and has a limit too. Prints "ok".
#include <cstdio>

#include "../../qora-llm_b200/csrc/tcgen05.cuh"

using namespace qora;

constexpr unsigned long long kLimit = 3000000;  // ns

// Thread 0 waits on a barrier on which thread 32 arrives (arrive != 0) after a third of the
// limit; thread 64 waits behind it on one that nothing arrives on.
__global__ void wait_kernel(int arrive, int* out) {
  __shared__ uint64_t bars[2];
  __shared__ volatile int abort_flag;
  if (threadIdx.x == 0) {
    ptx::mbar_init(&bars[0], 1);
    ptx::mbar_init(&bars[1], 1);
    ptx::fence_mbar_init();
    abort_flag = 0;
  }
  __syncthreads();
  const uint64_t t0 = ptx::globaltimer();
  if (threadIdx.x == 0) {
    out[0] = umma::wait_bar(&bars[0], 0, kLimit, &abort_flag);
    out[1] = abort_flag;
    out[2] = (int)((ptx::globaltimer() - t0) / 1000);  // us
  } else if (threadIdx.x == 32 && arrive) {
    while (ptx::globaltimer() - t0 < kLimit / 3) {
    }
    ptx::mbar_arrive(&bars[0]);
  } else if (threadIdx.x == 64 && !arrive) {
    out[3] = umma::wait_bar(&bars[1], 0, 100 * kLimit, &abort_flag);  // ends by the flag
    out[4] = (int)((ptx::globaltimer() - t0) / 1000);
  }
  __syncthreads();
}

// A bulk copy under way when the CTA has already given up: settling waits for it, so that the
// data is there; settling on a barrier that nothing arrives on ends at the limit.
__global__ void settle_kernel(const int* src, int* out) {
  __shared__ alignas(128) int data[8192];
  __shared__ uint64_t bars[2];
  if (threadIdx.x == 0) {
    ptx::mbar_init(&bars[0], 1);
    ptx::mbar_init(&bars[1], 1);
    ptx::fence_mbar_init();
    data[8191] = -1;
    ptx::fence_proxy_async();
    ptx::mbar_arrive_expect_tx(&bars[0], sizeof(data));
    ptx::bulk_g2s(data, src, sizeof(data), &bars[0]);
    out[0] = umma::settle_bar(&bars[0], 0, 1000 * kLimit);
    out[1] = data[8191];
    const uint64_t t0 = ptx::globaltimer();
    out[2] = umma::settle_bar(&bars[1], 0, kLimit);
    out[3] = (int)((ptx::globaltimer() - t0) / 1000);
  }
}

int main() {
  int *out, *src;
  if (cudaMallocManaged(&out, 5 * sizeof(int)) != cudaSuccess || cudaMalloc(&src, 8192 * sizeof(int)) != cudaSuccess ||
      cudaMemset(src, 5, 8192 * sizeof(int)) != cudaSuccess)
    return std::printf("no device memory\n"), 1;
  for (int arrive = 0; arrive < 2; ++arrive) {
    wait_kernel<<<1, 96>>>(arrive, out);
    if (cudaDeviceSynchronize() != cudaSuccess || out[0] != arrive || out[1] != !arrive || out[2] < (arrive ? 990 : 2900) ||
        (!arrive && (out[3] != 0 || out[4] < 2900 || out[4] > 100000)))
      return std::printf("FAIL arrive=%d: ended %d, abort %d, %d us; behind it %d, %d us\n", arrive, out[0], out[1], out[2], out[3],
                         out[4]),
             1;
  }
  settle_kernel<<<1, 32>>>(src, out);
  if (cudaDeviceSynchronize() != cudaSuccess || out[0] != 1 || out[1] != 0x05050505 || out[2] != 0 || out[3] < 2900)
    return std::printf("FAIL settle: %d, data %x; %d, %d us\n", out[0], out[1], out[2], out[3]), 1;
  std::printf("ok\n");
  return 0;
}
