// A Linear with 4-bit weights and group scales for few activation rows:
//   out[m, n] = sum_k x[m, k] * (q[n, k] - z[n, k / G]) * s[n, k / G] + bias[n]
//
// Bound by HBM: the packed weights are read once (N K / 2 bytes) and x is
// small.  At 0.5 bytes a weight the issue slots are the next limit (a B200
// reads about 90 weights per SM and clock against 128 lanes), so the products
// run on the tensor cores, mma.sync m16n8k16 in half precision with float32
// sums: 16 weight rows on the M side, the activation rows as its 8 columns.
//
// Weights: a nibble in bits 0-3 of a half is the subnormal number q 2^-24, in
// bits 4-7 it is q 2^-20, both exact operands, so unpacking eight weights is a
// shift and four masks.  The columns of x that meet the second kind, the odd
// ones, are divided by 16 beforehand.  The group's zero point and scale come in
// in float32,
//   s 2^24 (sum - z X),  X = 2^-24 sum of the group's x,
// where X is formed once per block.  (Integers q - z in bfloat16, made by
// setting a nibble into a mantissa and taking the offset off, were exact
// without X but took 11 operations per eight weights: 43 us for 28672 x 8192.)
//
// Activations enter as half, after a power of two that brings the largest of
// each 256 columns to 2^14..2^15.  float16 and bfloat16 keep their bits in one
// column.  float32 becomes three in columns that would be empty for few rows, of
// 11 bits each and in fixed point: multiples of 2^4, of 2^-8 and of 2^-20.  A
// group's products and its X are then whole numbers of one unit, below 2^24 of
// them, so the tensor cores, which cut the products of one instruction off some 24
// bits below the largest, and the difference sum - z X are exact; bits below 2^-35
// of those 256 columns' largest value are rounded off.  (With three parts of 8 bits
// in floating point, one x 2000 times the others in a column whose weight is 0 cost
// the rest of its row an error of 3.5e-4, ordinary rows 3.4e-7.)  In one column of
// float16 or bfloat16 the cut remains: 2000 times the others does not show in the
// outputs' own rounding, 60000 times costs 1.5e-2 where its weight is 0.
//
// Layout: the order of a sum over k is free.  A warp takes steps of 16 rows x
// 256 columns (128 bytes a row), copied by cp.async into its own ring of
// kStages slots; ldmatrix hands lane (g, t) word t of each 16-byte piece of
// row g, eight consecutive columns, of which the halves of a register are
// (0,4) (1,5) (2,6) (3,7).  x is laid out in shared memory in that order when
// it is staged, once per block.  A piece of 16 bytes is 32 columns, so groups
// of 32, 64 and 128 end after 1, 2 or 4 pieces.
//
// Work: a block takes an equal, consecutive share of the 16-row tiles, and its
// warps equal, consecutive shares of their steps, so that each streams one run
// of memory and nothing waits in between.  A tile inside one warp's share is
// finished there; one that is cut leaves partial sums in shared memory, two per
// warp at most, joined when all warps are done.  Where x does not fit beside
// the rings, or the tiles are too few to share out evenly, a cluster of 2, 4 or
// 8 blocks takes a share of the tiles together, each block a range of K (and
// that part of x alone), and adds its sums up through distributed shared memory
// in the order of the blocks.
//
// Measured on a B200: 28672 x 8192 (121 MB), one bf16 row 27 us, 4.5 TB/s, of
// which 6.5 us are the launch, x and the last tiles (5.7 TB/s beyond); eight
// rows 34 us, 16 rows 57 us; 4096 x 4096, one row 6.6 us; 1280 x 1280 4.1 us.
#pragma once

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "dtype.cuh"
#include "kernels.cuh"
#include "per_device.h"

namespace esmb200 {
namespace w4 {

constexpr int kMaxSmem = 224 * 1024;
constexpr int kStep = 256;       // columns
constexpr int kBytes = kStep / 2;  // of a row
constexpr float kLargest = 3.402823466e38f;  // of float32's finite values
constexpr int kColumn = kStep * 2 + 64;  // bytes of a step's column of x in shared memory
// W warps per block: 16 for one column tile (128 registers a thread are enough;
// most loads in flight for one copy of x), else 8, whose 255 registers hold two
// tiles' sums without spills (28672 x 8192, 16 bf16 rows: 59 against 73 us).
// Small calls take 8 too: their blocks leave room for the next kernel's to
// start beside them (1280 x 1280: 4.2 against 5.7 us).
// A: rows on 16-byte boundaries; else the nine 16-byte blocks that cover a
// row's 128 bytes are copied.
template <int NT, bool A, int W, int G>
struct Shape {
  static constexpr int kThreads = 32 * W;
  static constexpr int kStages = W == 16 ? 3 : 4;
  static constexpr int kPitch = A ? 128 : 144;
  static constexpr int kSlot = 16 * kPitch;
  static constexpr int kRing = W * kStages * kSlot;
  // A step's scales and zero points: (s 2^24, -z) of [kStep / G groups][16 rows],
  // the groups apart so that lanes of neighbouring groups write to other banks.
  static constexpr int kScaleGroup = 128 + 128 / (kStep / G);
  static constexpr int kScales = (kStep / G) * kScaleGroup;
  static constexpr int kScaleRing = W * (kStages - 1) * kScales;
  // The warps' partial sums: two of 16 rows x 8 NT columns each, in rows whose
  // pitch spreads a column over the banks.
  static constexpr int kRow = 8 * NT + 2;
  static constexpr int kPartial = 16 * kRow;  // floats
  static constexpr int kPartials = W * 2 * kPartial * 4;
  static constexpr int kRest = kRing + kScaleRing + kPartials;  // of shared memory, beside x and a cluster's sums
};
// Rows of x times steps, for each warp of a block, up to which the blocks make
// x's records themselves; beyond, a kernel before this one makes them once.
// (10240 x 2560, 4 float32 rows: five for each warp take 13.0 us, the kernel
// 11.2.)
constexpr int kMakeSelf = 3;
// Steps per SM from which a call runs with 16 warps per block.
constexpr int kLargeSteps = 32;

struct Plan {
  int tiles;     // 16-row tiles, shared out evenly over the clusters
  int at_once;   // tiles that a cluster takes before it adds up its sums
  int steps;     // of 256 columns
  int cluster;   // blocks that share a row's steps
  int cols;      // columns in use: rows of x, times 3 for float32
  int x_bytes;   // of shared memory for x's records
  int m0, rows;  // the rows of x of this launch
  int x_on_16;
  int prepared;  // x's records lie in the workspace
};

template <typename XT>
constexpr int kSplit = sizeof(XT) == 4 ? 3 : 1;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// Global -> shared copy of `bytes` (a multiple of 16), counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ float2 lds8(uint32_t a) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long lds8_pair(uint32_t a) {
  unsigned long long v;
  asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts8(uint32_t a, float x, float y) {
  asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(x), "f"(y) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same without sums to add to.
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// x as the products read it: one record per step of `cols` columns,
//   columns  each kColumn bytes: eight pieces of 64 bytes, 16 for each lane t,
//            and 64 bytes that move the next column to other banks
//   sums     float [group][cols8]: X of the group (cols8: whole tiles of 8)
//   factors  float [cols8]: the power of two that was taken out
struct Record {
  int sums, factors, bytes;
  __host__ __device__ constexpr Record(int cols, int cols8, int groups_per_step)
      : sums(cols * kColumn), factors(sums + groups_per_step * cols8 * 4), bytes(factors + cols8 * 4) {}
};

// Eight columns of x from k on, zeros behind K.
template <typename XT>
__device__ __forceinline__ void load_x(const LinearW4Args& a, const Plan& p, int m, int step, Vec<XT, 8>& v) {
  const long k = static_cast<long>(step) * kStep + (threadIdx.x & 31) * 8;
  const XT* src = static_cast<const XT*>(a.x) + static_cast<long>(p.m0 + m) * a.ldx + k;
  if (p.x_on_16 && k + 8 <= a.K) {
    v.load(src);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v.e[e] = k + e < a.K ? src[e] : from_f32<XT>(0.0f);
  }
}

// Row m's part of a step's record, by one warp, eight columns of x per lane.
template <typename XT, int G>
__device__ __forceinline__ void write_x(const Vec<XT, 8>& v, int m, int cols8, const Record& rec, unsigned char* record) {
  const int lane = threadIdx.x & 31;
  float* const sums = reinterpret_cast<float*>(record + rec.sums);
  float* const factors = reinterpret_cast<float*>(record + rec.factors);
  {
    __half h[kSplit<XT>][8];
    float out = 1.0f;
    {
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t bits = __float_as_uint(to_f32(v.e[e])) & 0x7FFFFFFFu;
        top = max(top, bits < 0x7F800000u ? bits : 0u);
      }
      top = __reduce_max_sync(0xffffffffu, top);
      // 2^(exponent) of the largest finite value, kept where both the factor
      // and its inverse are normal numbers.
      const uint32_t ex = max(top >> 23, 15u);
      const float in = __uint_as_float((268u - ex) << 23);  // 2^(14 - exponent)
      out = __uint_as_float((ex - 14u) << 23);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __fmul_rn(to_f32(v.e[e]), in), down = e & 1 ? 0.0625f : 1.0f;
        if constexpr (kSplit<XT> == 1) {
          h[0][e] = __float2half_rn(__fmul_rn(y, down));
        } else {
          // An infinity or NaN goes whole into the first column.
          const bool finite = fabsf(y) <= 65504.0f;
          float rest = finite ? y : 0.0f;
#pragma unroll
          for (int sp = 0; sp < 2; ++sp) {
            // To the nearest multiple of 2^4 or 2^-8: the last place of a sum with
            // 1.5 times 2^27 or 2^15.
            const float unit = sp == 0 ? 0x1.8p27f : 0x1.8p15f, part = __fsub_rn(__fadd_rn(rest, unit), unit);
            h[sp][e] = __float2half_rn(finite || sp > 0 ? __fmul_rn(part, down) : y);
            rest = __fsub_rn(rest, part);
          }
          rest = __fsub_rn(__fadd_rn(rest, 0x1.8p3f), 0x1.8p3f);  // of 2^-20
          h[2][e] = __float2half_rn(__fmul_rn(rest, down));
        }
      }
    }
#pragma unroll
    for (int sp = 0; sp < kSplit<XT>; ++sp) {
      const int col = m * kSplit<XT> + sp;
      auto pair = [&](int e) {
        return static_cast<uint32_t>(__half_as_ushort(h[sp][e])) |
               (static_cast<uint32_t>(__half_as_ushort(h[sp][e + 4])) << 16);
      };
      *reinterpret_cast<uint4*>(record + col * kColumn + lane * 16) =
          make_uint4(pair(0), pair(2), pair(1), pair(3));
      float x = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) x = __fmaf_rn(__half2float(h[sp][e]), e & 1 ? 16.0f : 1.0f, x);
#pragma unroll
      for (int d = 1; d < G / 8; d <<= 1) x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, d));
      if (lane % (G / 8) == 0) sums[lane / (G / 8) * cols8 + col] = __fmul_rn(x, 0x1p-24f);
      if (lane == 0) factors[col] = out;
    }
  }
}

// Out of the way of the products: sums that came out infinite or NaN are taken
// again as the definition reads, sum_k x[m, k] ((q[n, k] - z) s), where the row of
// x holds no NaN.  An infinite x is one reason, whose products with a nibble of 0
// or with the zero point are not its own; a scale whose 2^24-fold is beyond
// float32 another.  The block's warps take an output each, of those that the block
// wrote: tiles [tile0, tile1), in a cluster every p.cluster-th run of its threads'
// number.  known: RowOfX of the launch's rows, in shared memory.  (28672 x 8192,
// bf16: a row with a NaN adds 9 us to 40, 16 of them 0.4 ms; an infinite one 0.5 ms.
// The check costs calls without either 0.1 us.)
enum RowOfX : int { kUnknown = 0, kHasNaN = 1, kNoNaN = 2 };
template <typename XT>
__device__ __noinline__ void take_again(const LinearW4Args& a, const Plan& p, int tile0, int tile1, int rank,
                                        volatile int* known) {
  const int lane = threadIdx.x & 31, warps = blockDim.x / 32;
  for (int first = tile0; first < tile1; first += p.at_once) {
    const int outputs = min(p.at_once, tile1 - first) * 16 * p.rows;
    for (int i = threadIdx.x >> 5; i < outputs; i += warps) {
      if (i / blockDim.x % p.cluster != rank) continue;
      const int m = i % p.rows;
      const long n = static_cast<long>(first) * 16 + i / p.rows;
      if (n >= a.N) continue;
      XT* const out = static_cast<XT*>(a.out) + static_cast<long>(p.m0 + m) * a.ldo + n;
      if (!isnan(to_f32(*out))) continue;
      const XT* const x = static_cast<const XT*>(a.x) + static_cast<long>(p.m0 + m) * a.ldx;
      int row = __shfl_sync(0xffffffffu, known[m], 0);
      if (row == kUnknown) {
        bool nan = false;
        for (int k = lane; k < a.K; k += 32) nan |= isnan(to_f32(x[k]));
        row = __any_sync(0xffffffffu, nan) ? kHasNaN : kNoNaN;
        known[m] = row;
      }
      if (row == kHasNaN) continue;
      const uint8_t* const w = a.W + n * a.ldw;
      const int log = 31 - __clz(a.group);
      float sum = 0.0f;
#pragma unroll 8
      for (int k = 2 * lane; k < a.K; k += 64) {
        const bool two = k + 1 < a.K;
        const int g = k >> log, q2 = w[k >> 1], z = a.zeros != nullptr ? a.zeros[n * a.ldz + g] : 8;
        const float s = load_typed(a.scales, n * a.lds + g, a.scale_type);
        const float x0 = to_f32(x[k]), x1 = two ? to_f32(x[k + 1]) : 0.0f;
        sum = __fmaf_rn(x0, __fmul_rn(static_cast<float>((q2 & 15) - z), s), sum);
        if (two) sum = __fmaf_rn(x1, __fmul_rn(static_cast<float>((q2 >> 4) - z), s), sum);
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, d));
      if (a.bias != nullptr) sum = __fadd_rn(sum, a.bias[n]);
      if (lane == 0) *out = from_f32<XT>(sum);
    }
  }
}

constexpr int kPrepareWarps = 8;

// The records of all steps, once, for launches whose blocks would spend longer
// on making them than on copying them: one warp per row and step.
template <typename XT, int G>
__global__ void __launch_bounds__(32 * kPrepareWarps) prepare_x_kernel(LinearW4Args a, Plan p, int cols8) {
  pdl_wait();
  pdl_trigger();
  const Record rec(p.cols, cols8, kStep / G);
  const int i = blockIdx.x * kPrepareWarps + (threadIdx.x >> 5);
  if (i >= p.rows * p.steps) return;
  Vec<XT, 8> v;
  load_x(a, p, i / p.steps, i % p.steps, v);
  write_x<XT, G>(v, i / p.steps, cols8, rec,
                 static_cast<unsigned char*>(a.workspace) + static_cast<long>(i % p.steps) * rec.bytes);
}

__device__ __forceinline__ float lds_cluster(uint32_t a, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(a, rank)) : "memory");
  return v;
}

// G: columns of a group.
template <typename XT, int G, int NT, bool A, int W>
__global__ void __launch_bounds__(32 * W, 1) linear_w4_kernel(const __grid_constant__ LinearW4Args a, const __grid_constant__ Plan p) {
  using R = Shape<NT, A, W, G>;
  constexpr int kWarps = W, kThreads = R::kThreads, kStages = R::kStages;
  constexpr int kGroups = kStep / G;  // of a step: 2, 4 or 8
  constexpr int kHeld = 16 * kGroups / 32;  // scales of a step that one lane loads
  // One column tile: two chains of products, which halve the wait for one another;
  // more tiles have chains enough, and one sum takes fewer registers.
  constexpr bool kTwoChains = NT == 1;
  extern __shared__ __align__(128) unsigned char smem[];
  float* const part = reinterpret_cast<float*>(smem + p.x_bytes + R::kRing + R::kScaleRing);  // [warp][2][16][kRow]
  float* const sums = reinterpret_cast<float*>(smem + p.x_bytes + R::kRest);  // cluster: [tile][16][rows]
  const Record rec(p.cols, 8 * NT, kGroups);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + p.x_bytes + warp * kStages * R::kSlot;
  const uint32_t scale_ring = smem_u32(smem) + p.x_bytes + R::kRing + warp * (kStages - 1) * R::kScales;
  const int rank = p.cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int share = blockIdx.x / p.cluster, shares = gridDim.x / p.cluster;
  const int tile0 = static_cast<int>(static_cast<long>(share) * p.tiles / shares);
  const int tile1 = static_cast<int>((static_cast<long>(share) + 1) * p.tiles / shares);
  const int step0 = rank * p.steps / p.cluster, steps = (rank + 1) * p.steps / p.cluster - step0;
  const int row_bytes = static_cast<int>((static_cast<long>(a.K) + 1) / 2);
  __shared__ uint64_t s_x;  // x's records have arrived
  __shared__ int s_again, s_known[8 * NT];  // an output is not finite; RowOfX of the launch's rows
  __shared__ int2 s_cut[kWarps];  // the tile that the end of a warp's share is the first to cut (or -1), its last warp
  if (threadIdx.x < 8 * NT) s_known[threadIdx.x] = kUnknown;
  if (threadIdx.x == 0) s_again = 0;
  if (p.prepared && threadIdx.x == 0) {
    mbar_init(&s_x, 1);
    fence_barrier_init();
  }
  // Behind prepare_x_kernel only x has to be waited for: that kernel began when
  // everything before it was complete, and this one begins after all its blocks
  // have.
  if (!p.prepared) {
    pdl_wait();
    pdl_trigger();
  }
  // The block makes its steps of x itself: a warp takes 256 columns of one row
  // at a time, all of them loaded now, before the weights' copies are set up.
  Vec<XT, 8> mine[kMakeSelf];
  if (!p.prepared) {
#pragma unroll
    for (int u = 0; u < kMakeSelf; ++u) {
      const int i = warp + u * kWarps;
      if (i < p.rows * steps) load_x(a, p, i / steps, step0 + i % steps, mine[u]);
    }
  }

  // A place in the warp's share of the work: steps [at, end) of the tiles
  // [first, first + p.at_once), counted tile after tile.
  struct Place {
    int first, at, end, tile, step;  // step: within the block's
  };
  auto enter = [&](Place& c) {
    const int all = min(p.at_once, tile1 - c.first) * steps;
    c.at = warp * all / kWarps;
    c.end = (warp + 1) * all / kWarps;
    c.tile = steps > 0 ? c.at / steps : 0;
    c.step = c.at - c.tile * steps;
    c.tile += c.first;
  };
  // On to where the warp has a step to do; false if there is none left.
  auto skip_empty = [&](Place& c) -> bool {
    while (c.at >= c.end) {
      c.first += p.at_once;
      if (c.first >= tile1) return false;
      enter(c);
    }
    return true;
  };

  // What a warp reads ahead of its products, step after step of its share: the
  // weights' copies into its ring, and the scales and zero points.  Of these a
  // lane loads kHeld, of one group and as many rows (neighbouring lanes take a
  // row's groups: a load touches the fewest lines), keeps them as they are until the next step's copies are started -- a conversion at once would make
  // the warp wait -- and then puts them, converted, into a ring of their own.
  // Rows behind N read the last row's: they are not written.
  constexpr int kCopies = A ? 4 : 5;
  const uint8_t* src[kCopies];
  uint32_t src_dst[kCopies];
  int src_row[kCopies], src_from[kCopies];  // first byte within the step's 128 bytes of the row
  int src_first[kCopies];  // the same, rows off 16-byte boundaries taken into account
#pragma unroll
  for (int h = 0; h < kCopies; ++h) {
    const int id = lane + 32 * h;
    const int row = A ? id >> 3 : id / 9, piece = A ? id & 7 : id - row * 9;
    src_row[h] = row < 16 ? row : -1;
    src_from[h] = piece * 16;
    src_dst[h] = ring + (A ? row * 128 + ((piece ^ (row & 7)) << 4) : row * R::kPitch + piece * 16);
  }
  // Where the pieces of a row start in a 16-byte block, for rows that are not
  // on such boundaries.
  auto shift_of = [&](long n) {
    return A ? 0u : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a.W) + n * a.ldw) & 15u;
  };
  const uint8_t* const nowhere = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(a.W) & ~uintptr_t(15));
  const int groups = static_cast<int>((static_cast<long>(a.K) + G - 1) / G);
  const bool f32_scales = a.scale_type == kF32;
  constexpr int kRowsAtOnce = 32 / kGroups;
  const int s_lane = lane / kGroups, s_grp = lane % kGroups;  // the lane's first row, and its group
  const char* s_row[kHeld];
  const uint8_t* z_row[kHeld];
  struct Raw {
    uint32_t s[kHeld];
    int z[kHeld];
  };
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    s_row[u] = nullptr;
    z_row[u] = nullptr;
  }
  uint32_t s_put = scale_ring, s_get = scale_ring;
  auto put_scales = [&](const Raw& raw) {
    const uint32_t at = s_put + s_grp * R::kScaleGroup + s_lane * 8;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      float v;
      if (f32_scales) v = __uint_as_float(raw.s[u]);
      else if (a.scale_type == kF16) v = __half2float(__ushort_as_half(static_cast<uint16_t>(raw.s[u])));
      else v = __uint_as_float(raw.s[u] << 16);
      sts8(at + u * kRowsAtOnce * 8, __fmul_rn(v, 0x1p24f), static_cast<float>(-raw.z[u]));
    }
    s_put = s_put + R::kScales == scale_ring + (kStages - 1) * R::kScales ? scale_ring : s_put + R::kScales;
  };
  uint32_t put = 0;
  int left = 0, run = 0, grp0 = 0;  // bytes of the row from the step on; steps until the next tile; the lane's group
  Place ahead;
  ahead.first = tile0;
  enter(ahead);
  // To the first step of the warp's share, or on from the end of a run of steps
  // in one tile.
  auto next_run = [&](int done) {
    ahead.at += done;
    if (done > 0) {
      ahead.step = 0;
      ++ahead.tile;
    }
    if (!skip_empty(ahead)) {
      run = -1;
      return;
    }
    run = min(steps - ahead.step, ahead.end - ahead.at);
    const int step = step0 + ahead.step;
    left = row_bytes - step * kBytes;
    grp0 = step * kGroups + s_grp;
#pragma unroll
    for (int h = 0; h < kCopies; ++h) {
      const long n = min(static_cast<long>(ahead.tile) * 16 + max(src_row[h], 0), static_cast<long>(a.N) - 1);
      src_first[h] = src_from[h] - static_cast<int>(shift_of(n));
      src[h] = a.W + n * a.ldw + step * static_cast<long>(kBytes) + src_first[h];
    }
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const long n = min(static_cast<long>(ahead.tile) * 16 + s_lane + u * kRowsAtOnce, static_cast<long>(a.N) - 1);
      s_row[u] = static_cast<const char*>(a.scales) + n * a.lds * (f32_scales ? 4 : 2);
      if (a.zeros != nullptr) z_row[u] = a.zeros + n * a.ldz;
    }
  };
  next_run(0);
  int run_len = run;
  auto issue = [&](Raw& raw) {
    if (run > 0) {
      if (A && left >= kBytes) {
#pragma unroll
        for (int h = 0; h < kCopies; ++h) cp_async16(src_dst[h] + put, src[h], 16);
      } else {
        // The end of a row: nothing behind it is read, except that unaligned
        // blocks holding a byte of the row are copied whole (they never leave
        // the 16 bytes that some byte of W lies in).
#pragma unroll
        for (int h = 0; h < kCopies; ++h) {
          if constexpr (A) {
            const int bytes = min(max(left - src_from[h], 0), 16);
            cp_async16(src_dst[h] + put, bytes > 0 ? src[h] : nowhere, bytes);
          } else if (src_row[h] >= 0) {
            const bool on = src_first[h] < min(left, kBytes);
            cp_async16(src_dst[h] + put, on ? src[h] : nowhere, on ? 16 : 0);
          }
        }
      }
      // Groups behind K read the last one's: there x is 0.
      const uint32_t at = static_cast<uint32_t>(min(grp0, groups - 1));
#pragma unroll
      for (int u = 0; u < kHeld; ++u) {
        raw.s[u] = f32_scales ? __ldg(reinterpret_cast<const uint32_t*>(s_row[u]) + at)
                              : __ldg(reinterpret_cast<const uint16_t*>(s_row[u]) + at);
        if (a.zeros != nullptr) raw.z[u] = __ldg(z_row[u] + at);
      }
#pragma unroll
      for (int h = 0; h < kCopies; ++h) src[h] += kBytes;
      left -= kBytes;
      grp0 += kGroups;
      if (--run == 0) {
        next_run(run_len);
        run_len = run;
      }
    }
    put = put + R::kSlot == kStages * R::kSlot ? 0 : put + R::kSlot;
    cp_commit();
  };
  // With few warps, whose latency counts, the first steps' scales are all on
  // their way before any is converted (1280 x 1280: 4.05 against 4.45 us); with
  // many, one step after the other spreads the first burst (28672 x 8192: 27.7
  // against 28.2).
  constexpr bool kInTurn = W == 16;
  Raw raw;  // of the last step that was started
  {
    Raw first[kStages - 1];
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
#pragma unroll
      for (int u = 0; u < kHeld; ++u) {
        first[i].s[u] = 0u;
        first[i].z[u] = 8;
      }
      issue(first[i]);
      if (kInTurn && i + 2 < kStages) put_scales(first[i]);
    }
#pragma unroll
    for (int i = 0; i < kStages - 2; ++i)
      if (!kInTurn) put_scales(first[i]);
    raw = first[kStages - 2];
  }

  if (p.prepared) {
    pdl_wait();
    pdl_trigger();
  }

  // The lane's place in the columns' tiles; lanes of columns that no row of x
  // has read the last one's, whose products nobody reads.
  uint32_t x_lane[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) x_lane[j] = smem_u32(smem) + min(8 * j + g, p.cols - 1) * kColumn + t * 16;
  uint32_t get = 0;

  bool late = false;
  const int per_turn = kThreads / (16 * p.rows), turn_rest = kThreads % (16 * p.rows);
  __syncthreads();
  if (!p.prepared) {
#pragma unroll
    for (int u = 0; u < kMakeSelf; ++u) {
      const int i = warp + u * kWarps;
      if (i < p.rows * steps) write_x<XT, G>(mine[u], i / steps, 8 * NT, rec, smem + i % steps * rec.bytes);
    }
  } else if (steps > 0) {
    if (threadIdx.x == 0) {
      const uint32_t bytes = static_cast<uint32_t>(steps) * rec.bytes;
      mbar_arrive_expect_tx(&s_x, bytes);
      bulk_load(smem_u32(smem), static_cast<const unsigned char*>(a.workspace) + static_cast<long>(step0) * rec.bytes,
                bytes, &s_x);
    }
    late = !mbar_wait(&s_x, 0, a.status);
    if (late) mbar_wait(&s_x, 0, a.status);  // the copy's time to end, before the shared memory goes
  }
  // Without x (the status word says so) the block only keeps its cluster going.
  late = __syncthreads_or(late);

  Place c;
  for (c.first = tile0; c.first < tile1; c.first += p.at_once) {
    enter(c);
    if (late) c.at = c.end;
    const int here = min(p.at_once, tile1 - c.first);
    {
      auto finish = [&](int tile, int row, int m, float y) {
        const long n = static_cast<long>(tile) * 16 + row;
        if (n >= a.N) return;
        if (!(fabsf(y) <= kLargest)) {  // NaN marks it for take_again
          s_again = 1;
          y = __int_as_float(0x7FFFFFFF);
        }
        if (a.bias != nullptr) y = __fadd_rn(y, __ldg(a.bias + n));
        static_cast<XT*>(a.out)[static_cast<long>(p.m0 + m) * a.ldo + n] = from_f32<XT>(y);
      };
      // The block's sum of a tile's row.
      auto put_sum = [&](int tile, int row, int m, float y) {
        if (p.cluster > 1) sums[((tile - c.first) * 16 + row) * p.rows + m] = y;
        else finish(tile, row, m, y);
      };

      while (c.at < c.end) {
        const int n = min(steps - c.step, c.end - c.at), from = c.step;
        // Rows off 16-byte boundaries: the word of rows g and g + 8 that the lane
        // starts from, and by how many bits the next one is shifted in.
        uint32_t word[2], bits[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t sh = shift_of(min(static_cast<long>(c.tile) * 16 + g + 8 * h, static_cast<long>(a.N) - 1));
          word[h] = ring + (8 * h + g) * R::kPitch + (sh & ~3u) + 4 * t;
          bits[h] = 8 * (sh & 3u);
        }
        unsigned long long sum[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) sum[j][0] = sum[j][1] = 0ull;
        uint32_t xc = static_cast<uint32_t>(c.step) * rec.bytes;
        uint32_t x_sums = smem_u32(smem) + xc + rec.sums + 8 * t;
        for (int i0 = 0; i0 < n; ++i0) {
          cp_wait<kStages - 2>();
          __syncwarp();
          put_scales(raw);
          issue(raw);
          const uint32_t sc = s_get + g * 8;
          s_get = s_get + R::kScales == scale_ring + (kStages - 1) * R::kScales ? scale_ring : s_get + R::kScales;
          const uint32_t slot = ring + get;
          get = get + R::kSlot == kStages * R::kSlot ? 0 : get + R::kSlot;
          float lo[NT][4], hi[kTwoChains ? NT : 1][4];
          unsigned long long y[NT][2];  // rows g, g + 8: columns 2t, 2t + 1
#pragma unroll
          for (int j = 0; j < NT; ++j) y[j][0] = y[j][1] = 0ull;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t w[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if constexpr (A) {
                const int r = lane & 7, piece = 4 * half + (lane >> 3);
                ldmatrix4(w[h], slot + (8 * h + r) * 128 + ((piece ^ r) << 4));
              } else {
                const uint32_t row = word[h] + (slot - ring) + half * 64;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  // The second word of the last piece may lie behind the row's
                  // blocks; it is only shifted in when the row starts inside a
                  // word, and then it does not.
                  const uint32_t w0 = lds4(row + 16 * i), w1 = bits[h] != 0 ? lds4(row + 16 * i + 4) : 0u;
                  w[h][i] = __funnelshift_r(w0, w1, bits[h]);
                }
              }
            }
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) {
              const int i = 4 * half + i2;  // the piece; 32 columns
              const int grp = half * (128 / G) + i2 * 32 / G;
              const bool first = i2 * 32 % G == 0, last = (i2 + 1) * 32 % G == 0;
              uint32_t q[2][4];  // pairs (0,4) (2,6) times 2^-24 and (1,5) (3,7) times 2^-20
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t v = w[h][i2] >> 8;
                q[h][0] = w[h][i2] & 0x000F000Fu;
                q[h][1] = v & 0x000F000Fu;
                q[h][2] = w[h][i2] & 0x00F000F0u;
                q[h][3] = v & 0x00F000F0u;
              }
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                if (j == 0 || 8 * j < p.cols) {
                  const uint4 b = lds16(x_lane[j] + xc + i * 64);
                  if (first) {
                    mma_first(lo[j], q[0][0], q[1][0], q[0][1], q[1][1], b.x, b.y);
                    if constexpr (kTwoChains) mma_first(hi[j], q[0][2], q[1][2], q[0][3], q[1][3], b.z, b.w);
                    else mma(lo[j], q[0][2], q[1][2], q[0][3], q[1][3], b.z, b.w);
                  } else {
                    mma(lo[j], q[0][0], q[1][0], q[0][1], q[1][1], b.x, b.y);
                    mma(kTwoChains ? hi[j] : lo[j], q[0][2], q[1][2], q[0][3], q[1][3], b.z, b.w);
                  }
                }
              }
              if (last) {
                // Rows g and g + 8: (s 2^24, -z).
                const float2 r0 = lds8(sc + grp * R::kScaleGroup), r1 = lds8(sc + grp * R::kScaleGroup + 64);
                const unsigned long long s2[2] = {f2_pack(r0.x, r0.x), f2_pack(r1.x, r1.x)};
                const unsigned long long z2[2] = {f2_pack(r0.y, r0.y), f2_pack(r1.y, r1.y)};
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                  if (j == 0 || 8 * j < p.cols) {
                    const unsigned long long x = lds8_pair(x_sums + (grp * 8 * NT + 8 * j) * 4);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                      unsigned long long all = f2_pack(lo[j][2 * h], lo[j][2 * h + 1]);
                      if constexpr (kTwoChains) all = f2_add(all, f2_pack(hi[j][2 * h], hi[j][2 * h + 1]));
                      y[j][h] = f2_fma(f2_fma(z2[h], x, all), s2[h], y[j][h]);
                    }
                  }
                }
              }
            }
          }
          // The power of two that was taken out of these 256 columns.
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if (j == 0 || 8 * j < p.cols) {
              const unsigned long long f = lds8_pair(x_sums + (kGroups * 8 * NT + 8 * j) * 4);
#pragma unroll
              for (int h = 0; h < 2; ++h) sum[j][h] = f2_fma(y[j][h], f, sum[j][h]);
            }
          }
          xc += rec.bytes;
          x_sums += rec.bytes;
        }

        // The segment's sums, [row][column], as a partial: the first place for
        // a tile that began before this warp's share, the second for one that
        // ends behind it, and in passing for a whole one.
        float* const to = part + (warp * 2 + (from > 0 ? 0 : 1)) * R::kPartial;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float* at = to + g * R::kRow + 8 * j + 2 * t;
          *reinterpret_cast<unsigned long long*>(at) = sum[j][0];
          *reinterpret_cast<unsigned long long*>(at + 8 * R::kRow) = sum[j][1];
        }
        if (n == steps) {
          __syncwarp();
          for (int i = lane; i < 16 * p.rows; i += 32) {
            const int row = i & 15, m = i >> 4;
            float y = 0.0f;
#pragma unroll
            for (int sp = 0; sp < kSplit<XT>; ++sp) y = __fadd_rn(y, to[row * R::kRow + m * kSplit<XT> + sp]);
            put_sum(c.tile, row, m, y);
          }
          __syncwarp();
        }
        c.at += n;
        c.step = 0;
        ++c.tile;
      }
      // Joins the tiles that the warps' shares cut, each at the end of the share
      // that is the first to cut it; the sums of all of them are spread over
      // the threads.
      const int all = late ? 0 : here * steps, each = 16 * p.rows;
      if (threadIdx.x < kWarps) {
        const int w = threadIdx.x, begin = w * all / kWarps, cut = (w + 1) * all / kWarps;
        const int tile = steps > 0 ? cut / steps : 0, start = tile * steps;
        int last = w;
        while (last + 1 < kWarps && (last + 1) * all / kWarps < start + steps) ++last;
        s_cut[w] = make_int2(w + 1 < kWarps && start < cut && start >= begin ? tile : -1, last);
      }
      __syncthreads();
      for (int w = threadIdx.x / each, i = threadIdx.x % each; w + 1 < kWarps;) {
        const int2 cut = s_cut[w];
        if (cut.x >= 0) {
          const int row = i & 15, m = i >> 4;
          const float* from = part + row * R::kRow + m * kSplit<XT>;
          float y = 0.0f;
          for (int u = w; u <= cut.y; ++u) {
            if (u > w && u * all / kWarps == (u + 1) * all / kWarps) continue;  // an empty share
#pragma unroll
            for (int sp = 0; sp < kSplit<XT>; ++sp) y = __fadd_rn(y, from[(u * 2 + (u == w ? 1 : 0)) * R::kPartial + sp]);
          }
          put_sum(c.first + cut.x, row, m, y);
        }
        w += per_turn;
        i += turn_rest;
        if (i >= each) {
          i -= each;
          ++w;
        }
      }
      if (p.cluster > 1) {
        cluster_sync();
#pragma unroll 1
        for (int i = rank * kThreads + threadIdx.x; i < here * 16 * p.rows; i += p.cluster * kThreads) {
          float of[8];  // the blocks' sums, read together, added up in their order
#pragma unroll
          for (int r = 0; r < 8; ++r) of[r] = r < p.cluster ? lds_cluster(smem_u32(sums + i), r) : 0.0f;
          float y = of[0];
#pragma unroll
          for (int r = 1; r < 8; ++r) y = __fadd_rn(y, of[r]);
          const int m = i % p.rows, row = i / p.rows;
          finish(c.first + (row >> 4), row & 15, m, y);
        }
        cluster_sync();
      } else if (p.steps == 0) {  // K = 0: the bias alone
        for (int i = threadIdx.x; i < here * 16 * p.rows; i += kThreads)
          finish(c.first + i / (16 * p.rows), i & 15, (i >> 4) % p.rows, 0.0f);
      }
    }
  }
  cp_wait<0>();
  __syncthreads();
  if (s_again != 0) take_again<XT>(a, p, tile0, tile1, rank, s_known);
}

template <typename XT, int G, int NT, bool A, int W>
cudaError_t launch(const LinearW4Args& a, const Plan& p, int smem, int shares, cudaStream_t s) {
  auto kernel = linear_w4_kernel<XT, G, NT, A, W>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(kernel, kMaxSmem, allowed);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(shares * p.cluster);
  cfg.blockDim = dim3(32 * W);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2] = {pdl_attribute()};
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, p);
}

// Clusters of 2^log blocks of the kernel that fit the device at once (one block
// per SM), 0 if the device cannot say.
template <typename XT, int G, int NT, bool A, int W>
int clusters_at_once(int log) {
  static PerDevice known[4];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return 0;
  return known[log].get(device, [&] {
    int n = 0;
    auto kernel = linear_w4_kernel<XT, G, NT, A, W>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1 << log);
    cfg.blockDim = dim3(32 * W);
    cfg.dynamicSmemBytes = kMaxSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1 << log;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    return n;
  });
}

// One pass over the weights for rows [m0, m0 + rows) of x.  The cluster's size:
// the fewest rounds of steps that a warp has to go through, adding up a
// cluster's sums counted as two.
template <typename XT, int G, int NT, bool A, int W>
cudaError_t pass_of(const LinearW4Args& a, Plan p, cudaStream_t s) {
  using R = Shape<NT, A, W, G>;
  const Record rec(p.cols, 8 * NT, kStep / G);
  int best = -1, best_rounds = 0, best_shares = 0;
  for (int log = 0; log < 4 && (log == 0 || 1 << log <= p.steps); ++log) {
    const int steps = (p.steps + (1 << log) - 1) >> log;
    const long smem = R::kRest + static_cast<long>(steps) * rec.bytes + (log > 0 ? 64 * p.rows : 0);
    if (smem > kMaxSmem) continue;
    const int most = log == 0 ? a.num_sms : clusters_at_once<XT, G, NT, A, W>(log);
    if (most <= 0) continue;
    const int shares = p.tiles < most ? p.tiles : most;
    const int mine = (p.tiles + shares - 1) / shares;
    // Tiles between two cluster sums: as many as memory is left for.
    const int fit = log == 0 ? mine : static_cast<int>(std::min<long>(mine, (kMaxSmem - (smem - 64 * p.rows)) / (64 * p.rows)));
    const int rounds = (mine + fit - 1) / fit * (static_cast<int>((static_cast<long>(fit) * steps + W - 1) / W) + (log > 0 ? 2 : 0));
    if (best < 0 || rounds < best_rounds) {
      best = log;
      best_rounds = rounds;
      best_shares = shares;
    }
    if (log == 0 && rounds <= 3) break;  // nothing to gain
  }
  if (best < 0) return cudaErrorInvalidValue;
  p.cluster = 1 << best;
  p.x_bytes = ((p.steps + p.cluster - 1) / p.cluster) * rec.bytes;
  int smem = R::kRest + p.x_bytes;
  p.at_once = (p.tiles + best_shares - 1) / best_shares;
  if (best > 0) {
    const int fit = (kMaxSmem - smem) / (64 * p.rows);
    if (p.at_once > fit) p.at_once = fit;
    smem += p.at_once * 64 * p.rows;
  }
  return launch<XT, G, NT, A, W>(a, p, smem, best_shares, s);
}

// Whether a cluster of 8 blocks (or of as many as there are steps) holds x.
template <typename R>
constexpr bool holds(int steps, int rows, int cols, int cols8, int group) {
  int blocks = 8;
  while (blocks > 1 && blocks > steps) blocks /= 2;
  const long each = (steps + blocks - 1) / blocks;
  return R::kRest + each * Record(cols, cols8, kStep / group).bytes + 64 * rows <= kMaxSmem;
}

template <typename XT, int G, int NT, bool A>
cudaError_t pass(const LinearW4Args& a, int m0, int rows, cudaStream_t s) {
  Plan p = {};
  p.m0 = m0;
  p.rows = rows;
  p.cols = rows * kSplit<XT>;
  p.tiles = static_cast<int>((static_cast<long>(a.N) + 15) / 16);
  p.steps = static_cast<int>((static_cast<long>(a.K) + kStep - 1) / kStep);
  p.x_on_16 = ((reinterpret_cast<uintptr_t>(a.x) | static_cast<uintptr_t>(a.ldx * static_cast<long>(sizeof(XT)))) & 15) == 0;
  bool wide = false;
  if constexpr (NT <= 1)
    wide = static_cast<long>(p.tiles) * p.steps >= static_cast<long>(a.num_sms) * kLargeSteps &&
           holds<Shape<NT, A, 16, G>>(p.steps, rows, p.cols, 8 * NT, G);
  p.prepared = static_cast<long>(rows) * p.steps > kMakeSelf * (wide ? 16 : 8);
  if (p.prepared) {
    const cudaError_t e = launch_pdl(prepare_x_kernel<XT, G>, dim3((rows * p.steps + kPrepareWarps - 1) / kPrepareWarps),
                                     dim3(32 * kPrepareWarps), 0, s, a, p, 8 * NT);
    if (e != cudaSuccess) return e;
  }
  if constexpr (NT <= 1) {
    if (wide) return pass_of<XT, G, NT, A, 16>(a, p, s);
  }
  // One row of the longest K always fits: where not beside the rings of eight
  // warps (float32 in groups of 32, three columns and eight sums a step, beyond
  // 118784 columns), then beside those of six.
  if constexpr (NT == 1) {
    constexpr int kMost = kLinearW4MaxK / kStep;
    if constexpr (!holds<Shape<NT, A, 8, G>>(kMost, 1, kSplit<XT>, 8, G)) {
      static_assert(holds<Shape<NT, A, 6, G>>(kMost, 1, kSplit<XT>, 8, G), "one row of the longest K");
      if (!holds<Shape<NT, A, 8, G>>(p.steps, rows, p.cols, 8, G)) return pass_of<XT, G, NT, A, 6>(a, p, s);
    }
  }
  return pass_of<XT, G, NT, A, 8>(a, p, s);
}

// Rows of x that one pass can take: `tiles` column tiles, and no more than a
// cluster of 8 blocks can hold.
template <typename XT>
int rows_at_once(int K, int group, int tiles) {
  const int steps = static_cast<int>((static_cast<long>(K) + kStep - 1) / kStep);
  for (int nt = tiles; nt > 1; nt /= 2) {
    const int rows = 8 * nt / kSplit<XT>, cols = rows * kSplit<XT>;
    if (nt == 8   ? holds<Shape<8, false, 8, 32>>(steps, rows, cols, 64, group)
        : nt == 4 ? holds<Shape<4, false, 8, 32>>(steps, rows, cols, 32, group)
                  : holds<Shape<2, false, 8, 32>>(steps, rows, cols, 16, group))
      return rows;
  }
  int rows = 8 / kSplit<XT>;
  while (rows > 1 && !holds<Shape<1, false, 8, 32>>(steps, rows, rows * kSplit<XT>, 8, group)) --rows;
  return rows;
}

// Rows of each pass when one takes `most`: equal ones, so that 65 run as 33 + 32
// rather than 64 + 1.
inline int rows_each(int M, int most) {
  const int passes = (M - 1) / most + 1;
  return (M - 1) / passes + 1;
}

template <typename XT, int G, bool A>
cudaError_t all_rows(const LinearW4Args& a, cudaStream_t s) {
  // Many rows: eight column tiles in one pass where a call's latency counts; in
  // large calls two at a time, which reads the weights more often but keeps the
  // sums of a pass in fewer registers and x in one block (28672 x 8192, 32 bf16
  // rows: 118 against 144 us; 4096 x 4096: 21 against 16).
  const long steps = (static_cast<long>(a.K) + kStep - 1) / kStep;
  const bool large = (static_cast<long>(a.N) + 15) / 16 * steps >= static_cast<long>(a.num_sms) * 64;
  const int most = rows_at_once<XT>(a.K, G, large ? 2 : 8);
  const int each = rows_each(a.M, most);
  // The passes share the workspace: each one's kernels wait for the last's.
  for (int m0 = 0, rows = 0; m0 < a.M; m0 += rows) {
    rows = a.M - m0 < each ? a.M - m0 : each;
    const int cols = rows * kSplit<XT>;
    const cudaError_t e = cols <= 8    ? pass<XT, G, 1, A>(a, m0, rows, s)
                          : cols <= 16 ? pass<XT, G, 2, A>(a, m0, rows, s)
                          : cols <= 32 ? pass<XT, G, 4, A>(a, m0, rows, s)
                                       : pass<XT, G, 8, A>(a, m0, rows, s);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename XT, bool A>
cudaError_t by_group(const LinearW4Args& a, cudaStream_t s) {
  if (a.group == 128) return all_rows<XT, 128, A>(a, s);
  if (a.group == 64) return all_rows<XT, 64, A>(a, s);
  return all_rows<XT, 32, A>(a, s);
}

// Bytes of workspace for a call.
template <typename XT>
size_t workspace(int M, int K, int group) {
  if (M <= 0 || K <= 0) return 0;
  const int most = rows_at_once<XT>(K, group, 8);  // small calls' passes: the larger ones
  const int rows = rows_each(M, most), cols = rows * kSplit<XT>;
  const long steps = (static_cast<long>(K) + kStep - 1) / kStep;
  if (rows * steps <= kMakeSelf * 8) return 0;
  const int cols8 = cols <= 8 ? 8 : cols <= 16 ? 16 : cols <= 32 ? 32 : 64;
  return static_cast<size_t>(steps) * Record(cols, cols8, kStep / group).bytes;
}

// The kernels of one activation type (one translation unit each).
template <typename XT>
cudaError_t linear(const LinearW4Args& a, cudaStream_t s) {
  const bool on_16 = ((reinterpret_cast<uintptr_t>(a.W) | static_cast<uintptr_t>(a.ldw)) & 15) == 0;
  return on_16 ? by_group<XT, true>(a, s) : by_group<XT, false>(a, s);
}

}  // namespace w4
}  // namespace esmb200
