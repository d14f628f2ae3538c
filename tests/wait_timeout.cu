// A kernel that waits for a barrier as the attention's do. Nobody completes the barrier, so the wait gives up, unless
// `complete`; then it reports and gives its tensor memory back.
#include "tcgen05.cuh"

namespace {

__global__ void __launch_bounds__(128) wait_kernel(bool complete, int32_t* status, int32_t* waited) {
  using namespace b200tbe;
  __shared__ uint64_t bar;
  __shared__ uint32_t tmem_base;
  __shared__ int dead_word;
  const int warp = threadIdx.x / 32;
  volatile int* dead = &dead_word;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    dead_word = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(&tmem_base, 512);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (complete && threadIdx.x == 0) mbar_arrive(&bar);
  __syncwarp();
  const bool ok = warp_wait(&bar, 0, dead);
  waited[blockIdx.x * blockDim.x + threadIdx.x] = ok;
  __syncthreads();
  report(&dead_word, status);
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_free(tmem_base, 512);
}

}  // namespace

extern "C" __attribute__((visibility("default"))) int wait_out(int blocks, int complete, int32_t* status, int32_t* waited, void* stream) {
  wait_kernel<<<blocks, 128, 0, static_cast<cudaStream_t>(stream)>>>(complete != 0, status, waited);
  return b200tbe::launch_status();
}
