// Attention of one query token per sequence over a paged K/V cache:
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q.k_t - max),
// over the last `window` (or all) keys of the sequence; query head h reads
// key/value head h / (q_heads / kv_heads).  One warp per (sequence, query
// head), one pass with a running maximum and sum, all in float32.
#include "common.cuh"
#include "dtype.cuh"
#include "kernels.cuh"
#include "paged.h"

namespace esmb200 {
namespace {

constexpr int kPerLane = 8;  // head_dim <= 256

template <typename T>
__global__ void __launch_bounds__(128) attention_decode_simple_kernel(AttentionDecodeArgs a) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long row = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<long>(a.B) * a.q_heads) return;
  const int b = static_cast<int>(row / a.q_heads), h = static_cast<int>(row % a.q_heads);
  const PagedKV& kv = a.kv;
  const int hk = h / (a.q_heads / kv.heads);
  const KeyRange r = key_range(a.lens[b], kv.max_pages, kv.page_size, a.window);
  bool bad = r.bad != 0;
  const T* q = static_cast<const T*>(a.q) + b * a.q_seq + h * a.q_head;
  float qr[kPerLane], o[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int d = lane + 32 * i;
    qr[i] = d < kv.dh ? to_f32(q[d]) : 0.0f;
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int t = r.first; t < r.end; ++t) {
    const int page = kv.table[b * kv.table_stride + t / kv.page_size];
    if (page < 0 || page >= kv.num_pages) {
      bad = true;
      continue;
    }
    const int slot = t % kv.page_size;
    const T* k = static_cast<const T*>(kv.k) + page * kv.k_page + slot * kv.k_slot + hk * kv.k_head;
    const T* v = static_cast<const T*>(kv.v) + page * kv.v_page + slot * kv.v_slot + hk * kv.v_head;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (lane + 32 * i < kv.dh) s = __fmaf_rn(qr[i], to_f32(k[lane + 32 * i]), s);
    s = __fmul_rn(warp_sum(s), a.scale);
    const float m2 = fmaxf(m, s);
    const float c = m == -INFINITY ? 0.0f : expf(m - m2);
    const float p = s == -INFINITY ? 0.0f : expf(s - m2);
    l = __fmaf_rn(l, c, p);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (lane + 32 * i < kv.dh) o[i] = __fmaf_rn(p, to_f32(v[lane + 32 * i]), __fmul_rn(o[i], c));
    m = m2;
  }
  if (bad && lane == 0) atomicOr(a.status, kStatusBadIndex);
  const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
#pragma unroll
  for (int i = 0; i < kPerLane; ++i)
    if (lane + 32 * i < kv.dh)
      static_cast<T*>(a.out)[row * kv.dh + lane + 32 * i] = from_f32<T>(__fmul_rn(o[i], inv));
  if (a.lse != nullptr && lane == 0) a.lse[row] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace

size_t attention_decode_workspace(int, int, int, int, int) { return 0; }

cudaError_t launch_attention_decode(const AttentionDecodeArgs& a, cudaStream_t s) {
  if (a.B <= 0) return cudaSuccess;
  const long rows = static_cast<long>(a.B) * a.q_heads;
  const dim3 grid(static_cast<unsigned>((rows + 3) / 4));
  if (a.kv.type == kF32)
    return launch_pdl(attention_decode_simple_kernel<float>, grid, dim3(128), 0, s, a);
  if (a.kv.type == kF16)
    return launch_pdl(attention_decode_simple_kernel<__half>, grid, dim3(128), 0, s, a);
  return launch_pdl(attention_decode_simple_kernel<__nv_bfloat16>, grid, dim3(128), 0, s, a);
}

}  // namespace esmb200
