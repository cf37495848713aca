// The device's side of a look at the status word (take_status, status.h).
#include "kernels.cuh"

namespace esmb200 {
namespace {

__global__ void exchange_status_kernel(uint32_t* status, uint32_t* held) { *held = atomicExch(status, 0u); }

}  // namespace

cudaError_t launch_exchange_status(uint32_t* status, uint32_t* held, cudaStream_t s) {
  exchange_status_kernel<<<1, 1, 0, s>>>(status, held);
  return cudaGetLastError();
}

}  // namespace esmb200
