// The bounded waits of tcgen05.cuh on a GPU, each with a limit of a few milliseconds: a wait
// whose partner reports progress outlasts the limit and ends when the barrier completes; one
// without progress gives up, sets the abort flag and returns. Prints "ok".
#include <cstdio>

#include "../../qora-llm_b200/csrc/tcgen05.cuh"

using namespace qora;

constexpr unsigned long long kLimit = 3000000;  // ns

// Thread 0 waits; thread 32 raises the counter every limit / 10 for `rounds`, then arrives
// (arrive != 0) or leaves the barrier as it is.
__global__ void wait_kernel(int rounds, int arrive, int counted, int* out) {
  __shared__ uint64_t bar;
  __shared__ volatile int abort_flag;
  __shared__ volatile unsigned progress;
  if (threadIdx.x == 0) {
    ptx::mbar_init(&bar, 1);
    ptx::fence_mbar_init();
    abort_flag = 0;
    progress = 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint64_t t0 = ptx::globaltimer();
    out[0] = umma::wait_bar(&bar, 0, kLimit, &abort_flag, counted ? &progress : nullptr);
    out[1] = abort_flag;
    out[2] = (int)((ptx::globaltimer() - t0) / 1000);  // us
  } else if (threadIdx.x == 32) {
    for (int i = 0; i < rounds; ++i) {
      const uint64_t t0 = ptx::globaltimer();
      while (ptx::globaltimer() - t0 < kLimit / 10) {
      }
      progress = progress + 1;
    }
    if (arrive) ptx::mbar_arrive(&bar);
  }
  __syncthreads();
}

int main() {
  int* out;
  if (cudaMallocManaged(&out, 3 * sizeof(int)) != cudaSuccess) return std::printf("no device memory\n"), 1;
  struct Case {
    int rounds, arrive, counted, ended, least_us;
  };
  // five limits of work with progress; the same unseen; progress that stops; at once
  const Case cases[] = {{50, 1, 1, 1, 10000}, {50, 1, 0, 0, 2900}, {20, 0, 1, 0, 8000}, {0, 1, 1, 1, 0}};
  for (const Case& c : cases) {
    wait_kernel<<<1, 64>>>(c.rounds, c.arrive, c.counted, out);
    if (cudaDeviceSynchronize() != cudaSuccess) return std::printf("FAIL launch\n"), 1;
    if (out[0] != c.ended || out[1] != !c.ended || out[2] < c.least_us) {
      std::printf("FAIL rounds=%d arrive=%d counted=%d: ended %d, abort %d, %d us\n", c.rounds, c.arrive, c.counted, out[0],
                  out[1], out[2]);
      return 1;
    }
  }
  std::printf("ok\n");
  return 0;
}
