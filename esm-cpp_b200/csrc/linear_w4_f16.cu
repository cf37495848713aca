// The 4-bit Linear's kernels for float16 activations (linear_w4_kernel.cuh).
#include "linear_w4_kernel.cuh"

namespace esmb200 {

cudaError_t launch_linear_w4_f16(const LinearW4Args& a, cudaStream_t s) {
  return w4::linear<__half>(a, s);
}

size_t linear_w4_workspace_f16(int M, int K, int group) { return w4::workspace<__half>(M, K, group); }

}  // namespace esmb200
