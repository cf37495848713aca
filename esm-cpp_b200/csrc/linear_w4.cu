// A Linear with 4-bit weights and group scales for few activation rows:
//   out[m, n] = sum_k x[m, k] * (q[n, k] - z[n, k / G]) * s[n, k / G] + bias[n]
// One warp per weight row: the lanes take the row's bytes (two columns each)
// in turn; products and sums in float32.
#include "common.cuh"
#include "dtype.cuh"
#include "kernels.cuh"

namespace esmb200 {
namespace {

template <typename T>
__global__ void __launch_bounds__(256) linear_w4_simple_kernel(LinearW4Args a) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= a.N) return;
  const uint8_t* w = a.W + static_cast<long>(n) * a.ldw;
  for (int m = blockIdx.y; m < a.M; m += gridDim.y) {
    const T* x = static_cast<const T*>(a.x) + static_cast<long>(m) * a.ldx;
    float sum = 0.0f;
    for (int k = 2 * lane; k < a.K; k += 64) {
      const int g = k / a.group;
      const float s = load_typed(a.scales, static_cast<long>(n) * a.lds + g, a.scale_type);
      const int z = a.zeros ? a.zeros[static_cast<long>(n) * a.ldz + g] : 8;
      const int byte = w[k >> 1];
      // The scale goes to the weight, not to the sum: x near the type's largest
      // value times q - z would overflow before a small scale brings it back.
      sum = __fmaf_rn(to_f32(x[k]), __fmul_rn(static_cast<float>((byte & 15) - z), s), sum);
      if (k + 1 < a.K)
        sum = __fmaf_rn(to_f32(x[k + 1]), __fmul_rn(static_cast<float>((byte >> 4) - z), s), sum);
    }
    sum = warp_sum(sum);
    if (lane == 0) {
      if (a.bias) sum = __fadd_rn(sum, a.bias[n]);
      static_cast<T*>(a.out)[static_cast<long>(m) * a.ldo + n] = from_f32<T>(sum);
    }
  }
}

}  // namespace

cudaError_t launch_linear_w4(const LinearW4Args& a, cudaStream_t s) {
  if (a.M <= 0 || a.N <= 0) return cudaSuccess;
  const dim3 grid((a.N + 7) / 8, a.M < 65535 ? a.M : 65535);
  if (a.type == kF32) return launch_pdl(linear_w4_simple_kernel<float>, grid, dim3(256), 0, s, a);
  if (a.type == kF16) return launch_pdl(linear_w4_simple_kernel<__half>, grid, dim3(256), 0, s, a);
  return launch_pdl(linear_w4_simple_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, a);
}

}  // namespace esmb200
