// New keys and values into a paged cache, RoPE applied on the way, and the
// rotated queries beside them: one pass over q, k and v instead of a rotation,
// a conversion and a scatter.
//
// Rotation (the rotate-half form of rope_varlen_kernel, elementwise.cu) by the
// table row of the token's cache position, over the first `rot` of a head's
// dh elements, half = rot / 2:
//   x'[i] = x[i] c[i] - x[half + i] s[i],  x'[half + i] = x[half + i] c[i] + x[i] s[i]
// in float32, rounded once to the cache's type.
//
// Bound by HBM: every byte of q, k, v is read once and written once.  A block
// takes TB consecutive tokens: its first TB threads find each token's
// sequence, position and page once, then thread (x, y) takes chunk x of every
// head y, y + ny, ... so that a table row is loaded once per token and thread,
// not once per head.  Chunks are V elements: a pair (i, half + i) inside the
// rotated part, single ones behind it; v takes the same chunks unrotated.
#include "common.cuh"
#include "dtype.cuh"
#include "kernels.cuh"
#include "paged.h"

namespace esmb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;  // tokens per block

template <typename Tin, typename Tc, int V>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(KvAppendArgs a, int tb, int nx) {
  __shared__ Place s_place[kMaxTokens];
  pdl_wait();
  pdl_trigger();
  const PagedKV& kv = a.kv;
  const int t0 = blockIdx.x * tb;
  if (threadIdx.x < tb) {
    const int t = t0 + threadIdx.x;
    Place p = {-1, 0, 0, 0};
    if (t < a.T)
      p = append_place(a.cu, a.B, a.lens, kv.table, kv.table_stride, kv.max_pages, kv.page_size,
                       kv.num_pages, a.rot > 0 ? a.table_len : -1, t);
    if (p.bad) atomicOr(a.status, kStatusBadIndex);
    s_place[threadIdx.x] = p;
  }
  __syncthreads();

  const int tx = threadIdx.x & (nx - 1), ty = threadIdx.x / nx, ny = kThreads / nx;
  const int half = a.rot / 2;
  const int pairs = half / V, chunks = pairs + (kv.dh - a.rot) / V;
  const int hq = a.q_out != nullptr ? a.q_heads : 0;
  const int heads = hq + 2 * kv.heads;
  for (int j = 0; j < tb; ++j) {
    const Place p = s_place[j];
    if (p.page < 0) continue;
    const long t = t0 + j;
    for (int i = tx; i < chunks; i += nx) {
      const bool pair = i < pairs;
      const int at = pair ? i * V : a.rot + (i - pairs) * V;
      float c[V], sn[V];
      if (pair) {
        Vec<float, V> cv, sv;
        cv.load(a.cos_t + static_cast<long>(p.pos) * a.rot + at);
        sv.load(a.sin_t + static_cast<long>(p.pos) * a.rot + at);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          c[e] = cv.e[e];
          sn[e] = sv.e[e];
        }
      }
      for (int h = ty; h < heads; h += ny) {
        const Tin* src;
        Tc* dst;
        bool turn = pair;
        if (h < hq) {
          src = static_cast<const Tin*>(a.q) + t * a.q_tok + h * a.q_head;
          dst = static_cast<Tc*>(a.q_out) + (t * hq + h) * kv.dh;
        } else if (h < hq + kv.heads) {
          const int hk = h - hq;
          src = static_cast<const Tin*>(a.k) + t * a.k_tok + hk * a.k_head;
          dst = static_cast<Tc*>(kv.k) + p.page * kv.k_page + p.slot * kv.k_slot + hk * kv.k_head;
        } else {
          const int hk = h - hq - kv.heads;
          src = static_cast<const Tin*>(a.v) + t * a.v_tok + hk * a.v_head;
          dst = static_cast<Tc*>(kv.v) + p.page * kv.v_page + p.slot * kv.v_slot + hk * kv.v_head;
          turn = false;
        }
        Vec<Tin, V> lo, hi;
        Vec<Tc, V> lo2, hi2;
        lo.load(src + at);
        if (pair) hi.load(src + at + half);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float x = to_f32(lo.e[e]);
          if (turn) {
            const float y = to_f32(hi.e[e]);
            lo2.e[e] = from_f32<Tc>(__fmaf_rn(-y, sn[e], __fmul_rn(x, c[e])));
            hi2.e[e] = from_f32<Tc>(__fmaf_rn(y, c[e], __fmul_rn(x, sn[e])));
          } else {
            lo2.e[e] = from_f32<Tc>(x);
            if (pair) hi2.e[e] = from_f32<Tc>(to_f32(hi.e[e]));
          }
        }
        lo2.store(dst + at);
        if (pair) hi2.store(dst + at + half);
      }
    }
  }
}

// Whether rows that start at p and step by the strides (elements of `size`
// bytes) all start on `bytes`-byte boundaries.
bool aligned(const void* p, int bytes, int size, long s0, long s1, long s2 = 0) {
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(s0 * size) |
                           static_cast<uintptr_t>(s1 * size) | static_cast<uintptr_t>(s2 * size)) &
                          (bytes - 1)) == 0;
}

template <int V>
bool fits(const KvAppendArgs& a, int in_size, int c_size) {
  const int half = a.rot / 2, bi = V * in_size < 16 ? V * in_size : 16,
            bc = V * c_size < 16 ? V * c_size : 16;
  return half % V == 0 && (a.kv.dh - a.rot) % V == 0 &&
         aligned(a.q, bi, in_size, a.q_tok, a.q_head) && aligned(a.k, bi, in_size, a.k_tok, a.k_head) &&
         aligned(a.v, bi, in_size, a.v_tok, a.v_head) && aligned(a.q_out, bc, c_size, a.kv.dh, 0) &&
         aligned(a.kv.k, bc, c_size, a.kv.k_page, a.kv.k_slot, a.kv.k_head) &&
         aligned(a.kv.v, bc, c_size, a.kv.v_page, a.kv.v_slot, a.kv.v_head) &&
         (a.rot == 0 || (aligned(a.cos_t, 16, 4, a.rot, 0) && aligned(a.sin_t, 16, 4, a.rot, 0)));
}

template <typename Tin, typename Tc, int V>
cudaError_t launch(const KvAppendArgs& a, cudaStream_t s) {
  const int chunks = a.rot / 2 / V + (a.kv.dh - a.rot) / V;
  int nx = 1;
  while (nx < chunks && nx < 32) nx *= 2;
  const int tb = a.T >= 148 * 8 * kMaxTokens ? kMaxTokens : 1;
  return launch_pdl(kv_append_kernel<Tin, Tc, V>, dim3((a.T + tb - 1) / tb), dim3(kThreads), 0, s, a,
                    tb, nx);
}

template <typename Tin, typename Tc>
cudaError_t dispatch(const KvAppendArgs& a, cudaStream_t s) {
  const int is = sizeof(Tin), cs = sizeof(Tc);
  if (fits<8>(a, is, cs)) return launch<Tin, Tc, 8>(a, s);
  if (fits<4>(a, is, cs)) return launch<Tin, Tc, 4>(a, s);
  return launch<Tin, Tc, 1>(a, s);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendArgs& a, cudaStream_t s) {
  if (a.T <= 0 || a.B <= 0) return cudaSuccess;
  if (a.type == kF16) return dispatch<__half, __half>(a, s);
  if (a.type == kBF16) return dispatch<__nv_bfloat16, __nv_bfloat16>(a, s);
  if (a.kv.type == kF16) return dispatch<float, __half>(a, s);
  if (a.kv.type == kBF16) return dispatch<float, __nv_bfloat16>(a, s);
  return dispatch<float, float>(a, s);
}

}  // namespace esmb200
