// The 4-bit Linear's kernels for bfloat16 activations (linear_w4_kernel.cuh).
#include "linear_w4_kernel.cuh"

namespace esmb200 {

cudaError_t launch_linear_w4_bf16(const LinearW4Args& a, cudaStream_t s) {
  return w4::linear<__nv_bfloat16>(a, s);
}

size_t linear_w4_workspace_bf16(int M, int K, int group) { return w4::workspace<__nv_bfloat16>(M, K, group); }

}  // namespace esmb200
