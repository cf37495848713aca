// The 4-bit Linear's kernels for float16 activations (linear_w4_kernel.cuh).
#include "linear_w4_kernel.cuh"

namespace esmb200 {

cudaError_t launch_linear_w4_f16(const LinearW4Args& a, cudaStream_t s) {
  return w4::linear<__half>(a, s);
}

}  // namespace esmb200
