// Attention of one query token per sequence over a paged K/V cache:
//   o = sum_t p_t v_t / sum_t p_t,  p_t = 2^(c q.k_t - max),  c = scale log2 e,
// over the last `window` (or all) keys of the sequence; query head h reads
// key/value head h / (q_heads / kv_heads).
//
// Bound by HBM: each seen K and V row is read once per tile of up to 16 query
// heads that share it.  The products run on the tensor cores (mma.sync; a
// query tile has 8 or 16 rows, far too few for a tcgen05 tile of 128), so that
// grouped heads cost no more issue slots than one head.
//
// A warp takes 16 keys at a time and keeps its own running maximum, sum and
// output; nothing is shared between warps until the end.  The transposed
// products S^T = K Q^T and O^T = V^T P^T put the keys (and then the head
// elements) on the 16-row side of the MMA and the query heads on its 8-column
// side, so 8 heads fill a tile.  The order of a dot product's terms is free,
// so a lane's fragments of K are 16-byte pieces of a row as they lie in
// memory: each lane copies its own pieces (cp.async) into shared memory and
// reads the same bytes back -- a FIFO per lane, without bank conflicts, swizzle
// or barriers, several tiles deep to cover the latency of HBM.
//
// Types: 16-bit caches use the m16n8k16 products, exact in the cache's type;
// the probabilities go in as two 16-bit parts (value and remainder, together
// 16 bits or more), because one rounding to bfloat16 would be as large as the
// output's own.  float32 uses 3xTF32: x = hi + lo, hi the nearest tf32 value,
// and hi hi + hi lo + lo hi; the tensor cores truncate their sums, so the
// large products of S have accumulators apart from the small ones and every
// tile's O^T is added to the running one outside.
//
// Work: the tiles of all (sequence, kv head, head tile) items, sequence after
// sequence, form one line that is cut into equal pieces, one per resident
// block, whatever the lengths are.  An item inside one piece is finished
// there; one that is cut leaves partial (max, sum, output) triples in the
// workspace, two per block at most, and a second kernel joins them.  Both
// kernels derive the line from the lengths on the device.
#include "common.cuh"
#include "dtype.cuh"
#include "kernels.cuh"
#include "paged.h"

namespace esmb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T, int D, int NT>
struct Cfg {
  static constexpr bool kF32Cache = sizeof(T) == 4;
  static constexpr int kSize = static_cast<int>(sizeof(T));
  static constexpr int kChunk = 16 / kSize;               // elements of a 16-byte piece
  static constexpr int kKPieces = D * kSize / 64;         // a lane's pieces of one K row: 4 lanes a row
  static constexpr int kVPieces = D * kSize / 128 > 0 ? D * kSize / 128 : 1;  // of V: 8 lanes a row
  static constexpr int kStage = (2 * kKPieces + 4 * kVPieces) * 512;  // bytes per warp and tile
  static constexpr int kWarps = kStage > 16384 ? 2 : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kTile = 16 * kWarps;  // keys per block and step
  // Two blocks per SM where three tiles per warp fit 96 KB, else one.
  static constexpr int kCtas = kWarps * kStage * 3 <= 98304 ? 2 : 1;
  static constexpr int kFit = (kCtas == 2 ? 98304 : 196608) / (kWarps * kStage);
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kSmem = kWarps * kStage * kStages;
  static constexpr int kMTiles = kVPieces * (kF32Cache ? 2 : 4);  // 16-row tiles of O^T
  static constexpr int kHeads = 8 * NT;
  static constexpr int kPad = D + 1;  // row of a warp's output in shared memory
  static constexpr int kSlot = kHeads * (D + 2);  // floats of one partial: O, max, sum
  static_assert(kStages >= 3, "pipeline");
  static_assert(kHeads * kPad * 4 <= kStage * kStages, "a warp's output fits its FIFO");
};

// The line of tiles.  An item is (sequence, kv head, head tile).
struct Line {
  const int* lens;
  int B, max_pages, page_size, window;
  int per_seq;  // items per sequence
  int tile;     // keys per tile

  __device__ __forceinline__ KeyRange range(int b) const {
    return key_range(__ldcg(lens + b), max_pages, page_size, window);
  }
  // Tiles start at multiples of 16 keys, so that one never straddles a page
  // whose size is a multiple of 16.
  __device__ __forceinline__ int tiles(int b) const {
    const KeyRange r = range(b);
    return r.end > r.first ? (r.end - (r.first & ~15) + tile - 1) / tile : 0;
  }
  // Whole-warp: tiles of all sequences, times per_seq.
  __device__ __forceinline__ long total() const {
    long n = 0;
    for (int b = threadIdx.x & 31; b < B; b += 32) n += tiles(b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n * per_seq;
  }
  // Whole-warp: the sequence that holds place x of the line (0 <= x <
  // total()) and the place of its first tile.
  __device__ __forceinline__ int find(long x, long& start) const {
    const int lane = threadIdx.x & 31;
    long base = 0;
    for (int b0 = 0; b0 < B; b0 += 32) {
      const long n = b0 + lane < B ? static_cast<long>(tiles(b0 + lane)) * per_seq : 0;
      long sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const uint32_t over = __ballot_sync(0xffffffffu, base + sum > x);
      if (over != 0) {
        const int first = __ffs(over) - 1;
        start = base + __shfl_sync(0xffffffffu, sum - n, first);
        return b0 + first;
      }
      base += __shfl_sync(0xffffffffu, sum, 31);
    }
    start = base;
    return B;
  }
};

// Place where block c's piece of the line begins.
__device__ __forceinline__ long piece(long total, long c, long blocks) { return c * total / blocks; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                      __half) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                      __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo, hi the nearest tf32 value.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  lo = __float_as_uint(__fsub_rn(x, __uint_as_float(hi)));
}
// The transpose of an 8 x 8 matrix of 16-bit values spread over a warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Two values packed in the 16-bit type, and their remainders.
__device__ __forceinline__ void pack2(float x, float y, uint32_t& hi, uint32_t& lo, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const __nv_bfloat162 l = __floats2bfloat162_rn(__fsub_rn(x, __low2float(h)), __fsub_rn(y, __high2float(h)));
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void pack2(float x, float y, uint32_t& hi, uint32_t& lo, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  const __half2 l = __floats2half2_rn(__fsub_rn(x, __low2float(h)), __fsub_rn(y, __high2float(h)));
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.0f : m; }

// The probabilities of float16 caches are scaled by 2^10: their parts reach
// down to 2^-34 of the largest before float16's spacing ends, and long sums of
// small ones keep their share.
template <typename T>
constexpr float kShift = 0.0f;
template <>
constexpr float kShift<__half> = 10.0f;

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Cfg<T, D, NT>::kThreads, Cfg<T, D, NT>::kCtas)
    attention_decode_kernel(AttentionDecodeArgs a, int group, int head_tiles, int tile_heads, int q_on_16) {
  using C = Cfg<T, D, NT>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float s_m[C::kWarps][C::kHeads], s_l[C::kWarps][C::kHeads];
  pdl_wait();
  pdl_trigger();
  const PagedKV& kv = a.kv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const float c = __fmul_rn(a.scale, kLog2e);
  const Line line{a.lens, a.B, kv.max_pages, kv.page_size, a.window, kv.heads * head_tiles, C::kTile};
  const uint32_t fifo = smem_u32(smem) + warp * C::kStage * C::kStages + lane * 16;
  float* const own_o = reinterpret_cast<float*>(smem + warp * C::kStage * C::kStages);
  const T* const kbase = static_cast<const T*>(kv.k);
  const T* const vbase = static_cast<const T*>(kv.v);

  // Sequences without keys are on no block's piece.
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    const KeyRange r = line.range(b);
    if (r.bad && threadIdx.x == 0) atomicOr(a.status, kStatusBadIndex);
    if (r.end > r.first) continue;
    const long n = static_cast<long>(a.q_heads) * kv.dh;
    for (long i = threadIdx.x; i < n; i += C::kThreads) static_cast<T*>(a.out)[b * n + i] = from_f32<T>(0.0f);
    if (a.lse != nullptr)
      for (int h = threadIdx.x; h < a.q_heads; h += C::kThreads)
        a.lse[static_cast<long>(b) * a.q_heads + h] = -INFINITY;
  }

  const long total = line.total();
  long x = piece(total, blockIdx.x, gridDim.x);
  const long x_end = piece(total, blockIdx.x + 1, gridDim.x);
  if (x >= x_end) return;
  long start;
  int b = line.find(x, start);
  int nt = line.tiles(b);
  int item = static_cast<int>((x - start) / nt);
  int tile = static_cast<int>((x - start) - static_cast<long>(item) * nt);
  bool bad = false;

  while (true) {
    const int n = static_cast<int>(min(static_cast<long>(nt - tile), x_end - x));
    const int hk = item / head_tiles, ht = item - hk * head_tiles;
    const int h0 = hk * group + ht * tile_heads;  // first query head of the tile
    const int heads = min(tile_heads, group - ht * tile_heads);
    const KeyRange r = line.range(b);
    const int key0 = (r.first & ~15) + tile * C::kTile + 16 * warp;
    const int* const table = kv.table + b * kv.table_stride;

    // Q^T fragments: columns are the heads g (and g + 8), rows the head
    // elements in the order of the K pieces.
    uint32_t q[NT][C::kKPieces][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int h = g + 8 * j;
      const T* qr = static_cast<const T*>(a.q) + b * a.q_seq + (h0 + h) * a.q_head;
#pragma unroll
      for (int p = 0; p < C::kKPieces; ++p) {
        const int d = (p * 4 + t) * C::kChunk;
        Vec<T, C::kChunk> e;
        if (h < heads && d < kv.dh) {
          if (q_on_16) {
            e.load(qr + d);
          } else {
#pragma unroll
            for (int i = 0; i < C::kChunk; ++i) e.e[i] = qr[d + i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < C::kChunk; ++i) e.e[i] = from_f32<T>(0.0f);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) q[j][p][i] = reinterpret_cast<const uint32_t*>(e.e)[i];
      }
    }
    float m[NT][2], l[NT][2], o[NT][C::kMTiles][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      m[j][0] = m[j][1] = -INFINITY;
      l[j][0] = l[j][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < C::kMTiles; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][i][e] = 0.0f;
    }

    // Page of key `lane & 15` of the warp's tile i, -1 outside the range.
    auto page_of = [&](int i) -> int {
      const int key = key0 + i * C::kTile + (lane & 15);
      return i < n && key >= r.first && key < r.end ? table[key / kv.page_size] : -1;
    };
    // Starts the copies of tile i; returns the mask of its keys.
    auto issue = [&](int i, int page) -> uint32_t {
      const int key = key0 + i * C::kTile + (lane & 15);
      const bool in = i < n && key >= r.first && key < r.end;
      const bool on = in && page >= 0 && page < kv.num_pages;
      bad |= in && !on;
      const long slot = key % kv.page_size;
      const long ko = on ? page * kv.k_page + slot * kv.k_slot : 0;
      const long vo = on ? page * kv.v_page + slot * kv.v_slot : 0;
      const uint32_t mask = __ballot_sync(0xffffffffu, on) & 0xffffu;
      const uint32_t dst = fifo + (i % C::kStages) * C::kStage;
      if (mask != 0) {
#pragma unroll
        for (int row = 0; row < 2; ++row) {
          const int k = g + 8 * row;
          const T* src = kbase + __shfl_sync(0xffffffffu, ko, k) + hk * kv.k_head;
#pragma unroll
          for (int p = 0; p < C::kKPieces; ++p) {
            const int d = (p * 4 + t) * C::kChunk;
            const bool ok = ((mask >> k) & 1u) && d < kv.dh;
            cp_async16(dst + (row * C::kKPieces + p) * 512, ok ? src + d : kbase, ok);
          }
        }
#pragma unroll
        for (int row = 0; row < 4; ++row) {
          const int k = C::kF32Cache ? t + 4 * row : 2 * t + (row & 1) + 8 * (row >> 1);
          const T* src = vbase + __shfl_sync(0xffffffffu, vo, k) + hk * kv.v_head;
#pragma unroll
          for (int p = 0; p < C::kVPieces; ++p) {
            const int d = (p * 8 + g) * C::kChunk;
            const bool ok = ((mask >> k) & 1u) && d < kv.dh;
            cp_async16(dst + (2 * C::kKPieces + row * C::kVPieces + p) * 512, ok ? src + d : vbase, ok);
          }
        }
      }
      cp_commit();
      return mask;
    };

    uint32_t mask[C::kStages];
    int page = page_of(0);
#pragma unroll
    for (int i = 0; i < C::kStages - 1; ++i) {
      const int next = page_of(i + 1);
      mask[i] = issue(i, page);
      page = next;
    }
    for (int i = 0; i < n; ++i) {
      const int next = page_of(i + C::kStages);
      mask[C::kStages - 1] = issue(i + C::kStages - 1, page);
      page = next;
      cp_wait<C::kStages - 1>();
      const uint32_t keys = mask[0];
#pragma unroll
      for (int j = 0; j + 1 < C::kStages; ++j) mask[j] = mask[j + 1];
      if (keys == 0) continue;
      const uint32_t src = fifo + (i % C::kStages) * C::kStage;

      // S^T: rows are the keys g and g + 8, columns the heads 2t and 2t + 1.
      float s[NT][4], s_lo[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = s_lo[j][e] = 0.0f;
#pragma unroll
      for (int p = 0; p < C::kKPieces; ++p) {
        const uint4 k0 = lds16(src + p * 512), k1 = lds16(src + (C::kKPieces + p) * 512);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const uint32_t f[4] = {w0[e], w1[e], w0[e + 1], w1[e + 1]};
          if constexpr (C::kF32Cache) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) split_tf32(__uint_as_float(f[u]), hi[u], lo[u]);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              uint32_t qh[2], ql[2];
              split_tf32(__uint_as_float(q[j][p][e]), qh[0], ql[0]);
              split_tf32(__uint_as_float(q[j][p][e + 1]), qh[1], ql[1]);
              mma8(s[j], hi, qh[0], qh[1]);
              mma8(s_lo[j], hi, ql[0], ql[1]);
              mma8(s_lo[j], lo, qh[0], qh[1]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) mma16(s[j], f, q[j][p][e], q[j][p][e + 1], T());
          }
        }
      }

      // Scores in powers of two, the running maximum, the probabilities.
      const bool k_lo = (keys >> g) & 1u, k_hi = (keys >> (g + 8)) & 1u;
      float top[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = C::kF32Cache ? __fadd_rn(s[j][e], s_lo[j][e]) : s[j][e];
          s[j][e] = (e < 2 ? k_lo : k_hi) ? __fmul_rn(v, c) : -INFINITY;
        }
        top[j][0] = fmaxf(s[j][0], s[j][2]);
        top[j][1] = fmaxf(s[j][1], s[j][3]);
      }
#pragma unroll
      for (int d = 4; d < 32; d <<= 1)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) top[j][e] = fmaxf(top[j][e], __shfl_xor_sync(0xffffffffu, top[j][e], d));
      float alpha[NT][2];
      bool moved = false;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float next_m = fmaxf(m[j][e], top[j][e]), ref = finite_ref(next_m);
          moved |= next_m != m[j][e];
          alpha[j][e] = ex2_ftz(__fsub_rn(m[j][e], ref));
          m[j][e] = next_m;
#pragma unroll
          for (int half = 0; half < 2; ++half)
            s[j][e + 2 * half] = ex2_ftz(__fadd_rn(__fsub_rn(s[j][e + 2 * half], ref), kShift<T>));
          l[j][e] = __fmaf_rn(l[j][e], alpha[j][e], __fadd_rn(s[j][e], s[j][e + 2]));
        }
      if (!C::kF32Cache && __any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i2 = 0; i2 < C::kMTiles; ++i2)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][i2][e] = __fmul_rn(o[j][i2][e], alpha[j][e & 1]);
      }

      // O^T += V^T P^T: rows are head elements, columns the heads.
      if constexpr (C::kF32Cache) {
        // b[j][h][i]: P of key t + 4 i + 8 h, head g.
        uint32_t bh[NT][2][2], bl[NT][2][2];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
              const int from = (t + 4 * i2) * 4 + (g >> 1);
              const float p0 = __shfl_sync(0xffffffffu, s[j][2 * h], from);
              const float p1 = __shfl_sync(0xffffffffu, s[j][2 * h + 1], from);
              split_tf32((g & 1) ? p1 : p0, bh[j][h][i2], bl[j][h][i2]);
            }
#pragma unroll
        for (int p = 0; p < C::kVPieces; ++p) {
          uint32_t v[4][4];
#pragma unroll
          for (int row = 0; row < 4; ++row) {
            const uint4 w = lds16(src + (2 * C::kKPieces + row * C::kVPieces + p) * 512);
            v[row][0] = w.x;
            v[row][1] = w.y;
            v[row][2] = w.z;
            v[row][3] = w.w;
          }
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            float acc[NT][4], acc_lo[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[j][e] = acc_lo[j][e] = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int u = 0; u < 4; ++u)
                split_tf32(__uint_as_float(v[2 * h + (u >> 1)][2 * i2 + (u & 1)]), hi[u], lo[u]);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                mma8(acc[j], hi, bh[j][h][0], bh[j][h][1]);
                mma8(acc_lo[j], hi, bl[j][h][0], bl[j][h][1]);
                mma8(acc_lo[j], lo, bh[j][h][0], bh[j][h][1]);
              }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[j][2 * p + i2][e] = __fmaf_rn(o[j][2 * p + i2][e], alpha[j][e & 1],
                                                __fadd_rn(acc[j][e], acc_lo[j][e]));
          }
        }
      } else {
        uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t hi, lo;
            pack2(s[j][2 * h], s[j][2 * h + 1], hi, lo, T());
            bh[j][h] = transpose8(hi);
            bl[j][h] = transpose8(lo);
          }
#pragma unroll
        for (int p = 0; p < C::kVPieces; ++p) {
          uint32_t v[4][4];
#pragma unroll
          for (int row = 0; row < 4; ++row) {
            const uint4 w = lds16(src + (2 * C::kKPieces + row * C::kVPieces + p) * 512);
            v[row][0] = w.x;
            v[row][1] = w.y;
            v[row][2] = w.z;
            v[row][3] = w.w;
          }
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) {
            const uint32_t f[4] = {
                __byte_perm(v[0][i2], v[1][i2], 0x5410), __byte_perm(v[0][i2], v[1][i2], 0x7632),
                __byte_perm(v[2][i2], v[3][i2], 0x5410), __byte_perm(v[2][i2], v[3][i2], 0x7632)};
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              mma16(o[j][4 * p + i2], f, bh[j][0], bh[j][1], T());
              mma16(o[j][4 * p + i2], f, bl[j][0], bl[j][1], T());
            }
          }
        }
      }
    }
    cp_wait<0>();
    __syncwarp();

    // The warps' results meet in shared memory.  Row g of O^T tile i is head
    // element (piece 8-lane g, element 2 i'), row g + 8 the next one.
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], d);
        if (g == 0) {
          s_m[warp][8 * j + 2 * t + e] = m[j][e];
          s_l[warp][8 * j + 2 * t + e] = l[j][e];
        }
      }
      constexpr int kPer = C::kF32Cache ? 2 : 4;
#pragma unroll
      for (int i = 0; i < C::kMTiles; ++i) {
        const int d = (i / kPer * 8 + g) * C::kChunk + 2 * (i % kPer);
        if (d < D) {
#pragma unroll
          for (int e = 0; e < 4; ++e) own_o[(8 * j + 2 * t + (e & 1)) * C::kPad + d + (e >> 1)] = o[j][i][e];
        }
      }
    }
    __syncthreads();
    const bool whole = n == nt;
    float* const slot = static_cast<float*>(a.workspace) +
                        (2 * static_cast<long>(blockIdx.x) + (tile > 0 ? 0 : 1)) * C::kSlot;
    for (int i = threadIdx.x; i < heads * D; i += C::kThreads) {
      const int h = i / D, d = i % D;
      float top = s_m[0][h];
#pragma unroll
      for (int w = 1; w < C::kWarps; ++w) top = fmaxf(top, s_m[w][h]);
      const float ref = finite_ref(top);
      float sum = 0.0f, out = 0.0f;
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w) {
        const float f = ex2_ftz(__fsub_rn(s_m[w][h], ref));
        const float ow = reinterpret_cast<const float*>(smem + w * C::kStage * C::kStages)[h * C::kPad + d];
        sum = __fmaf_rn(s_l[w][h], f, sum);
        out = __fmaf_rn(ow, f, out);
      }
      if (whole) {
        const long row = static_cast<long>(b) * a.q_heads + h0 + h;
        if (d < kv.dh)
          static_cast<T*>(a.out)[row * kv.dh + d] = from_f32<T>(sum == 0.0f ? 0.0f : __fdiv_rn(out, sum));
        if (d == 0 && a.lse != nullptr)
          a.lse[row] = sum == 0.0f ? -INFINITY : __fmul_rn(__fadd_rn(top, __fsub_rn(log2f(sum), kShift<T>)), kLn2);
      } else {
        slot[i] = out;
        if (d == 0) {
          slot[C::kHeads * D + h] = top;
          slot[C::kHeads * (D + 1) + h] = sum;
        }
      }
    }
    __syncthreads();

    x += n;
    if (x >= x_end) break;
    tile = 0;
    if (++item == line.per_seq) {
      item = 0;
      do nt = line.tiles(++b);
      while (nt == 0);
    }
  }
  if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(a.status, kStatusBadIndex);
}

// Joins the pieces of a cut item.  Block (i, h): the item that the beginning
// of piece i + 1 cuts, if it is the first to cut it, head h of its tile.  Warp
// w takes the pieces i + w, i + w + 4, ...
template <typename T, int D, int NT>
__global__ void __launch_bounds__(128)
    attention_join_kernel(AttentionDecodeArgs a, int group, int head_tiles, int tile_heads, int pieces) {
  using C = Cfg<T, D, NT>;
  constexpr int kPer = (D + 31) / 32;
  __shared__ float s_m[4], s_l[4], s_o[4][D];
  const PagedKV& kv = a.kv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y;
  const Line line{a.lens, a.B, kv.max_pages, kv.page_size, a.window, kv.heads * head_tiles, C::kTile};
  // The lengths were complete before the attention kernel began, and this
  // kernel begins after all of that kernel's blocks have; only the partial
  // results have to be waited for.
  const long total = line.total();
  const long before = piece(total, blockIdx.x, pieces), cut = piece(total, blockIdx.x + 1, pieces);
  bool mine = cut > before && cut < total;
  long start = 0;
  int b = 0, nt = 1, item = 0;
  if (mine) {
    b = line.find(cut, start);
    nt = line.tiles(b);
    item = static_cast<int>((cut - start) / nt);
    start += static_cast<long>(item) * nt;
    mine = start < cut && start >= before;
  }
  const int hk = item / head_tiles, ht = item - hk * head_tiles;
  mine = mine && h < min(tile_heads, group - ht * tile_heads);
  pdl_wait();
  pdl_trigger();
  if (!mine) return;
  const long end = start + nt;
  float m = -INFINITY, l = 0.0f, o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) o[i] = 0.0f;
  for (long k = blockIdx.x + warp; k < pieces && piece(total, k, pieces) < end; k += 4) {
    if (piece(total, k + 1, pieces) == piece(total, k, pieces)) continue;  // an empty piece
    const float* slot = static_cast<const float*>(a.workspace) + (2 * k + (k == blockIdx.x ? 1 : 0)) * C::kSlot;
    const float mk = slot[C::kHeads * D + h], lk = slot[C::kHeads * (D + 1) + h];
    const float top = fmaxf(m, mk), ref = finite_ref(top);
    const float f0 = ex2_ftz(__fsub_rn(m, ref)), f1 = ex2_ftz(__fsub_rn(mk, ref));
    l = __fmaf_rn(l, f0, __fmul_rn(lk, f1));
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = __fmaf_rn(o[i], f0, __fmul_rn(slot[h * D + 32 * i + lane], f1));
    m = top;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) s_o[warp][32 * i + lane] = o[i];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3])), ref = finite_ref(top);
  float f[4], sum = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = ex2_ftz(__fsub_rn(s_m[w], ref));
    sum = __fmaf_rn(s_l[w], f[w], sum);
  }
  const long row = static_cast<long>(b) * a.q_heads + hk * group + ht * tile_heads + h;
  for (int d = threadIdx.x; d < kv.dh; d += 128) {
    float out = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) out = __fmaf_rn(s_o[w][d], f[w], out);
    static_cast<T*>(a.out)[row * kv.dh + d] = from_f32<T>(sum == 0.0f ? 0.0f : __fdiv_rn(out, sum));
  }
  if (threadIdx.x == 0 && a.lse != nullptr)
    a.lse[row] = sum == 0.0f ? -INFINITY : __fmul_rn(__fadd_rn(top, __fsub_rn(log2f(sum), kShift<T>)), kLn2);
}

template <typename T, int D, int NT>
cudaError_t launch(const AttentionDecodeArgs& a, cudaStream_t s) {
  using C = Cfg<T, D, NT>;
  const int group = a.q_heads / a.kv.heads;
  const int head_tiles = (group + C::kHeads - 1) / C::kHeads;
  const int tile_heads = (group + head_tiles - 1) / head_tiles;
  const int blocks = a.num_sms * C::kCtas;
  const bool q_on_16 = ((reinterpret_cast<uintptr_t>(a.q) | static_cast<uintptr_t>(a.q_seq * C::kSize) |
                         static_cast<uintptr_t>(a.q_head * C::kSize)) & 15) == 0;
  auto kernel = attention_decode_kernel<T, D, NT>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kernel, dim3(blocks), dim3(C::kThreads), C::kSmem, s, a, group, head_tiles, tile_heads,
                 q_on_16 ? 1 : 0);
  if (e != cudaSuccess) return e;
  return launch_pdl(attention_join_kernel<T, D, NT>, dim3(blocks - 1, tile_heads), dim3(128), 0, s, a, group,
                    head_tiles, tile_heads, blocks);
}

template <typename T, int D, int NT>
size_t workspace(int num_sms) {
  using C = Cfg<T, D, NT>;
  return static_cast<size_t>(2) * num_sms * C::kCtas * C::kSlot * sizeof(float);
}

// Calls f with the kernel's parameters as types: D the smallest of 32, 64, 128
// and 256 that holds a head, one tile of 8 heads up to a group of 8 and two
// beyond.
template <int V>
struct Int {
  static constexpr int value = V;
};
template <typename T, typename F>
auto with_shape(int dh, int group, F f) {
  auto with_d = [&](auto d) { return group <= 8 ? f(T(), d, Int<1>()) : f(T(), d, Int<2>()); };
  if (dh <= 32) return with_d(Int<32>());
  if (dh <= 64) return with_d(Int<64>());
  if (dh <= 128) return with_d(Int<128>());
  return with_d(Int<256>());
}
template <typename F>
auto with_cfg(int type, int dh, int group, F f) {
  if (type == kF32) return with_shape<float>(dh, group, f);
  if (type == kF16) return with_shape<__half>(dh, group, f);
  return with_shape<__nv_bfloat16>(dh, group, f);
}

}  // namespace

size_t attention_decode_workspace(int type, int q_heads, int kv_heads, int dh, int num_sms) {
  return with_cfg(type, dh, q_heads / kv_heads, [&](auto t, auto d, auto n) {
    return workspace<decltype(t), decltype(d)::value, decltype(n)::value>(num_sms);
  });
}

cudaError_t launch_attention_decode(const AttentionDecodeArgs& a, cudaStream_t s) {
  if (a.B <= 0) return cudaSuccess;
  return with_cfg(a.kv.type, a.kv.dh, a.q_heads / a.kv.heads, [&](auto t, auto d, auto n) {
    return launch<decltype(t), decltype(d)::value, decltype(n)::value>(a, s);
  });
}

}  // namespace esmb200
