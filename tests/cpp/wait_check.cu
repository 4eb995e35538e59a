// The bounded waits of tcgen05.cuh on a GPU, each with a limit of a few milliseconds: a wait
// whose partner renews the mark outlasts the limit and ends when the barrier completes; one
// that is not renewed gives up, sets the abort flag and returns. Settling waits for copies in
// flight and has a limit too. Prints "ok".
#include <cstdio>

#include "../../qora-llm_b200/csrc/tcgen05.cuh"

using namespace qora;

constexpr unsigned long long kLimit = 3000000;  // ns

// Thread 0 waits; thread 32 renews the mark every limit / 10 for `rounds`, then arrives
// (arrive != 0) or leaves the barrier as it is.
__global__ void wait_kernel(int rounds, int arrive, int counted, int* out) {
  __shared__ uint64_t bar;
  __shared__ volatile int abort_flag;
  __shared__ volatile uint64_t mark;
  if (threadIdx.x == 0) {
    ptx::mbar_init(&bar, 1);
    ptx::fence_mbar_init();
    abort_flag = 0;
    mark = 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint64_t t0 = ptx::globaltimer();
    out[0] = umma::wait_bar(&bar, 0, kLimit, &abort_flag, counted ? &mark : nullptr);
    out[1] = abort_flag;
    out[2] = (int)((ptx::globaltimer() - t0) / 1000);  // us
  } else if (threadIdx.x == 32) {
    for (int i = 0; i < rounds; ++i) {
      const uint64_t t0 = ptx::globaltimer();
      while (ptx::globaltimer() - t0 < kLimit / 10) {
      }
      mark = ptx::globaltimer();
    }
    if (arrive) ptx::mbar_arrive(&bar);
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
  if (cudaMallocManaged(&out, 4 * sizeof(int)) != cudaSuccess || cudaMalloc(&src, 8192 * sizeof(int)) != cudaSuccess ||
      cudaMemset(src, 5, 8192 * sizeof(int)) != cudaSuccess)
    return std::printf("no device memory\n"), 1;
  struct Case {
    int rounds, arrive, counted, ended, least_us;
  };
  // five limits of work with marks; the same unseen; marks that stop; at once
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
  settle_kernel<<<1, 32>>>(src, out);
  if (cudaDeviceSynchronize() != cudaSuccess || out[0] != 1 || out[1] != 0x05050505 || out[2] != 0 || out[3] < 2900)
    return std::printf("FAIL settle: %d, data %x; %d, %d us\n", out[0], out[1], out[2], out[3]), 1;
  std::printf("ok\n");
  return 0;
}
