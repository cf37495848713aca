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
// takes `tb` consecutive tokens: its first threads find each token's sequence,
// position and page once, then every thread keeps one token and one item of a
// head row -- a pair of V-element chunks, (i, half + i) inside the rotated
// part, the two halves of the rest behind it -- and takes it of every ny-th
// head, so that a table row's part is loaded once per thread and not once per
// head.  The loads of two (16-bit inputs) or four heads are in flight before
// the first store, and 64 registers allow four blocks per SM.  v takes the same
// items unrotated.
//
// Measured on a B200: 26k prompt tokens of 20 heads of 64, float32 into
// bfloat16 (755 MB), 122 us, 6.2 TB/s, 94% of the copy rate; 32k bfloat16 tokens
// of 32/8 heads of 128, half rotated (801 MB), 146 us, 84%; 256 single tokens
// 4.4 us.
#include "common.cuh"
#include "dtype.cuh"
#include "kernels.cuh"
#include "paged.h"

namespace esmb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;  // tokens per block

template <typename Tin, typename Tc, int V>
__global__ void __launch_bounds__(kThreads, 4) kv_append_kernel(KvAppendArgs a, int tb, int nx) {
  __shared__ Place s_place[kMaxTokens];
  pdl_wait();
  pdl_trigger();
  const PagedKV& kv = a.kv;
  const int t0 = blockIdx.x * tb;
  // Thread: item fastest, then head, then token.
  const int tx = threadIdx.x & (nx - 1), row = threadIdx.x / nx, ny = kThreads / (nx * tb);
  const int ty = row % ny, j = row / ny;
  const long t = static_cast<long>(t0) + j;
  const int half = a.rot / 2, rest = kv.dh - a.rot;
  const bool halves = rest / 2 % V == 0 && rest % 2 == 0;  // the rest goes in pairs too
  const int pairs = half / V, items = pairs + (halves ? rest / 2 / V : rest / V);
  const int hq = a.q_out != nullptr ? a.q_heads : 0;
  const int heads = hq + 2 * kv.heads;
  const Tin* const q = static_cast<const Tin*>(a.q) + t * a.q_tok;
  const Tin* const k = static_cast<const Tin*>(a.k) + t * a.k_tok;
  const Tin* const v = static_cast<const Tin*>(a.v) + t * a.v_tok;
  constexpr int kBatch = sizeof(Tin) == 4 ? 4 : 2;  // heads in flight
  Vec<Tin, V> x[kBatch], y[kBatch];
  auto first_of = [&](int i) { return i < pairs ? i * V : a.rot + (i - pairs) * V; };
  auto load = [&](int i, int h0) {
    const int at = first_of(i), at2 = at + (i < pairs ? half : rest / 2);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int h = h0 + u * ny, hk = h - hq;
      if (h >= heads) break;
      const Tin* src = h < hq         ? q + h * a.q_head
                       : hk < kv.heads ? k + hk * a.k_head
                                       : v + (hk - kv.heads) * a.v_head;
      x[u].load(src + at);
      if (i < pairs || halves) y[u].load(src + at2);
    }
  };
  // The first loads are on their way while the tokens' places are found.
  const bool active = j < tb && t < a.T && tx < items;
  if (active && ty < heads) load(tx, ty);
  if (threadIdx.x < tb) {
    Place p = {-1, 0, 0, 0};
    if (t0 + threadIdx.x < a.T)
      p = append_place(a.cu, a.B, a.lens, kv.table, kv.table_stride, kv.max_pages, kv.page_size,
                       kv.num_pages, a.rot > 0 ? a.table_len : -1, t0 + threadIdx.x);
    if (p.bad) atomicOr(a.status, kStatusBadIndex);
    s_place[threadIdx.x] = p;
  }
  __syncthreads();
  if (!active) return;
  const Place p = s_place[j];
  if (p.page < 0) return;
  Tc* const qo = static_cast<Tc*>(a.q_out) + t * hq * kv.dh;
  Tc* const ko = static_cast<Tc*>(kv.k) + p.page * kv.k_page + p.slot * kv.k_slot;
  Tc* const vo = static_cast<Tc*>(kv.v) + p.page * kv.v_page + p.slot * kv.v_slot;
  for (int i = tx; i < items; i += nx) {
    const bool rotated = i < pairs, two = rotated || halves;
    const int at = first_of(i), at2 = at + (rotated ? half : rest / 2);
    Vec<float, V> c, s;
    if (rotated) {
      c.load(a.cos_t + static_cast<long>(p.pos) * a.rot + at);
      s.load(a.sin_t + static_cast<long>(p.pos) * a.rot + at);
    }
    for (int h0 = ty; h0 < heads; h0 += kBatch * ny) {
      if (i > tx || h0 > ty) load(i, h0);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int h = h0 + u * ny, hk = h - hq;
        if (h >= heads) break;
        Tc* dst = h < hq         ? qo + static_cast<long>(h) * kv.dh
                  : hk < kv.heads ? ko + hk * kv.k_head
                                  : vo + (hk - kv.heads) * kv.v_head;
        const bool turn = rotated && hk < kv.heads;
        Vec<Tc, V> x2, y2;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float lo = to_f32(x[u].e[e]);
          if (turn) {
            const float hi = to_f32(y[u].e[e]);
            x2.e[e] = from_f32<Tc>(__fmaf_rn(-hi, s.e[e], __fmul_rn(lo, c.e[e])));
            y2.e[e] = from_f32<Tc>(__fmaf_rn(hi, c.e[e], __fmul_rn(lo, s.e[e])));
          } else {
            x2.e[e] = from_f32<Tc>(lo);
            if (two) y2.e[e] = from_f32<Tc>(to_f32(y[u].e[e]));
          }
        }
        x2.store(dst + at);
        if (two) y2.store(dst + at2);
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
  const int rest = a.kv.dh - a.rot;
  const bool halves = rest / 2 % V == 0 && rest % 2 == 0;
  const int items = a.rot / 2 / V + (halves ? rest / 2 / V : rest / V);
  int nx = 1;
  while (nx < items && nx < 32) nx *= 2;
  // Few tokens: one per block, the heads spread over its threads.  Many: eight,
  // so that a thread has several heads for its table values and loads.
  const int tb = a.T >= a.num_sms * 8 * kMaxTokens ? kMaxTokens : 1;
  return launch_pdl(kv_append_kernel<Tin, Tc, V>, dim3((a.T - 1) / tb + 1), dim3(kThreads), 0, s, a,
                    tb, nx);
}

template <typename Tin, typename Tc>
cudaError_t dispatch(const KvAppendArgs& a, cudaStream_t s) {
  const int is = sizeof(Tin), cs = sizeof(Tc);
  if constexpr (sizeof(Tin) == 2) {
    if (fits<8>(a, is, cs)) return launch<Tin, Tc, 8>(a, s);
  }
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
