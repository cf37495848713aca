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
// side, so 8 heads fill a tile.  The order of a dot product's terms is free, so
// a lane's fragments of K are 16-byte pieces of a row as they lie in memory.
//
// Each warp has its own ring of tiles in shared memory, filled ahead by TMA to
// cover the latency of HBM: the cache is a tensor (element, head, slot, page),
// a box as many slots as divide a page and the 16 keys of a tile, 128 bytes of
// a row wide, in the 128-byte swizzle.  Completion is counted on an mbarrier
// per tile; the loading warp is the reading one, so nothing else waits.  Rows
// are read in an order that the swizzle spreads over all banks.  (Measured on
// the way here: 16-byte cp.async copies of the same ring, 16 per lane and tile,
// and one row-sized bulk copy per lane, which is issued lane by lane, both
// cost more issue slots than the products.)
//
// Types: 16-bit caches use the m16n8k16 products, exact in the cache's type;
// the probabilities go in as two 16-bit parts (value and remainder, together
// 16 bits or more), because one rounding to bfloat16 would be as large as the
// output's own.  float32 uses 3xTF32: x = hi + lo, hi a tf32 value, and hi hi +
// hi lo + lo hi.  The tensor cores truncate their sums, which over many tiles of
// one sign is a loss that grows with their number (2^31 keys of float16 values
// in [1, 2): 1.2%): in every type a tile's O^T is added to the running one
// outside, rounded to nearest, and the large products of float32's S have
// accumulators apart from the small ones.  (The additions cost 16-bit heads of
// 32 3%, of 64 and 128 under 2%, of 256 with two head tiles 10%, where they
// spill.)
//
// Work: the 16-key tiles of all (sequence, kv head, head tile) items, sequence
// after sequence, form one line that is cut into equal pieces, one per resident
// warp, whatever the lengths are.  A warp's copies run ahead across its items.
// An item inside one piece is finished there; one that is cut leaves partial
// (max, sum, output) triples in the workspace, two per warp at most, and a
// second kernel joins them.  Both kernels derive the line from the lengths on
// the device.  Few items of short caches go without (item_per_block).
//
// Measured on a B200: 131071 keys of one sequence (32/8 heads of 128, bf16, 537
// MB) 93 us, 5.8 TB/s, 88% of the copy rate; 64 sequences of 1 to 4099 keys 101
// us, 84%; 48 sequences of 122 to 1026 keys (20 heads of 64, float32) 50 us,
// 77%, where the splits into tf32 parts cost as much as the memory; 130 keys of
// one sequence 6.8 us, a chain of latencies (behind a page table with room for
// thousands 8.6: the second kernel).
#include <cudaTypedefs.h>

#include <atomic>
#include <type_traits>

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
  static constexpr int kRow = 128;  // bytes of a row in a box; elements behind dh arrive as zeros
  static constexpr int kBoxes = D * kSize > kRow ? D * kSize / kRow : 1;  // across a row
  static constexpr int kPart = 16 * kRow * kBoxes;                        // bytes of a tile's K (or V)
  static constexpr int kStage = 2 * kPart;                        // bytes per warp and tile
  static constexpr int kWarps = kStage > 16384 ? 2 : 4;
  static constexpr int kThreads = kWarps * 32;
  // Two blocks per SM where three tiles per warp fit half of its shared memory.
  static constexpr int kHalf = 112 * 1024, kWhole = 225 * 1024;
  static constexpr int kCtas = kWarps * kStage * 3 <= kHalf ? 2 : 1;
  static constexpr int kFit = (kCtas == 2 ? kHalf : kWhole) / (kWarps * kStage);
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kSmem = kWarps * kStage * kStages + 1024;  // the swizzle's alignment
  static_assert(kVPieces == kBoxes, "a box is the width of a V piece of 8 lanes");
  static constexpr int kMTiles = kVPieces * (kF32Cache ? 2 : 4);  // 16-row tiles of O^T
  static constexpr int kHeads = 8 * NT;
  static constexpr int kSlot = kHeads * (D + 2);  // floats of one partial: O, max, sum
  static_assert(kStages >= 3, "pipeline");
};

constexpr int kTile = 16;  // keys per tile (tiles_of)

// The line of tiles.  An item is (sequence, kv head, head tile).
struct Line {
  const int* lens;
  int B, max_pages, page_size, window;
  int per_seq;  // items per sequence

  __device__ __forceinline__ KeyRange range(int b) const {
    return key_range(__ldcg(lens + b), max_pages, page_size, window);
  }
  __device__ __forceinline__ int tiles(int b) const {
    return tiles_of(range(b));
  }
  // Whole-warp: the tiles of sequence `lane`, for batches of up to 32, whose
  // lengths are then read once for everything below.
  __device__ __forceinline__ int own() const {
    const int lane = threadIdx.x & 31;
    return B <= 32 && lane < B ? tiles(lane) : 0;
  }
  // Whole-warp: tiles of all sequences, times per_seq.
  __device__ __forceinline__ long total(int mine) const {
    long n = mine;
    if (B > 32)
      for (int b = threadIdx.x & 31; b < B; b += 32) n += tiles(b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n * per_seq;
  }
  // Whole-warp: the sequence that holds place x of the line (0 <= x <
  // total()), its tiles, and the place of its first one.
  __device__ __forceinline__ int find(long x, int mine, long& start, int& nt) const {
    const int lane = threadIdx.x & 31;
    long base = 0;
    for (int b0 = 0; b0 < B; b0 += 32) {
      const int count = B <= 32 ? mine : b0 + lane < B ? tiles(b0 + lane) : 0;
      const long n = static_cast<long>(count) * per_seq;
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
        nt = __shfl_sync(0xffffffffu, count, first);
        return b0 + first;
      }
      base += __shfl_sync(0xffffffffu, sum, 31);
    }
    start = base;
    nt = 1;
    return B;
  }
};

// n / d for 0 <= n < 2^31 and a divisor fixed at launch: with L = ceil(log2 d)
// and m = ceil(2^(31 + L) / d), n m = n 2^(31 + L) / d + n e / d, e < d <= 2^L,
// and n e < 2^(31 + L), so the floor is right.
struct Divisor {
  uint32_t d, m, shift;  // m = 0: d is 1
  explicit Divisor(int value) : d(static_cast<uint32_t>(value)), m(0), shift(0) {
    if (d == 1) return;
    uint32_t l = 1;
    while ((1ull << l) < d) ++l;
    m = static_cast<uint32_t>(((1ull << (31 + l)) + d - 1) / d);
    shift = l - 1;
  }
  __device__ __forceinline__ int of(int n) const {
    return m == 0 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), m) >> shift);
  }
};

// The line's pieces: one per warp, or one per tile of a short line (up to two per
// SM), where the tiles' latency counts (1 sequence of 130 keys: 9 us, with four
// tiles a piece 12), or per two tiles in between, where the joining does.
__host__ __device__ __forceinline__ int pieces_of(long total, int warps, int num_sms) {
  const long few = 2 * num_sms;
  const long n = total <= few ? total : (total + 1) / 2 > few ? (total + 1) / 2 : few;
  return n < warps ? static_cast<int>(n) : warps;
}
// Items that fit the device a block each, in caches whose page tables hold only
// short sequences, take a block each: its warps join their parts in shared
// memory, and there is no second kernel (one sequence of 130 keys, 20 heads of
// 64, float32: 6.8 against 8.4 us; 32 of up to 250, 32/8 heads of 128, bf16: 9.8
// against 15.9).  Short: 4 tiles a warp, 8 where the items fill half the device
// (32 of 500: 15.5 against 21.5; but one of 500: 10.1 against 8.5).  Products of
// wide heads in two tiles or in float32 take longer than the second kernel (16
// heads of 256 over one, bf16: 13.5 against 12.5).
template <typename C>
constexpr bool kBlocksPay = C::kBoxes * C::kHeads <= 32;
__host__ __forceinline__ bool item_per_block(long items, long capacity, int blocks, int warps) {
  return items <= blocks && capacity <= static_cast<long>(items * 2 >= blocks ? 8 : 4) * kTile * warps;
}
// Place where piece c begins.
__device__ __forceinline__ long piece(long total, long c, long pieces) { return c * total / pieces; }

// Box of the cache's tensor at (element, head, slot, page) -> shared memory.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int element, int head,
                                        int slot, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(element), "r"(head), "r"(slot), "r"(page), "r"(smem_u32(bar))
      : "memory");
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
// The same without sums to add to.
__device__ __forceinline__ void mma16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                            __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// x = hi + lo, hi the leading 11 bits: two operations for the many values of K
// and V.  (The tensor core reads 11 of lo's 13 bits: 2^-21 of x at most.)
__device__ __forceinline__ void cut_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xFFFFE000u;
  lo = __float_as_uint(__fsub_rn(x, __uint_as_float(hi)));
}
// x = hi + lo, hi the nearest tf32 value, which leaves lo one bit less: for the
// few values of Q and P.
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

// q . k of one float32 query row and key `row` of a tile, in whole float32
// values: for scores that the products of parts cannot give (an infinite
// element, or one that rounds up to infinity in tf32).
__device__ __noinline__ float whole_score(const float* q, uint32_t tile, int row, int dh) {
  float sum = 0.0f;
  for (int d0 = 0; d0 < dh; d0 += 16) {  // by sixteens: no chain is longer than the products' own
    float part = 0.0f;
    for (int d = d0; d < d0 + 16 && d < dh; d += 4) {
      const int piece = d / 4;
      const uint4 w = lds16(tile + ((piece >> 3) * 16 + row) * 128 + (((piece ^ row) & 7) << 4));
      const uint32_t k[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) part = __fmaf_rn(q[d + i], __uint_as_float(k[i]), part);
    }
    sum = __fadd_rn(sum, part);
  }
  return sum;
}

__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.0f : m; }

// A score may pass its head's reference by this much (in powers of two) before
// the reference moves: probabilities are at most 2^8 instead of 1, and almost
// no tile has to find its maximum or rescale anything.  (The difference is what
// is compared and shifted: beside a reference of 2^24 or more a sum with the
// slack or the shift would round away.)
constexpr float kSlack = 8.0f;
// The probabilities of float16 caches are scaled by 2^7 (with the slack still
// below float16's largest value): their two parts reach down to 2^-31 before
// float16's spacing ends, so that long sums of small ones keep their share.
template <typename T>
constexpr float kShift = 0.0f;
template <>
constexpr float kShift<__half> = 7.0f;

// The lane's eight (float32: four) consecutive elements of heads 2t and 2t + 1
// in piece p of O^T.
template <typename C, int NT>
__device__ __forceinline__ void row_of(const float (&o)[NT][C::kMTiles][4], int j, int p, int e, float (&v)[C::kChunk]) {
#pragma unroll
  for (int i = 0; i < C::kChunk / 2; ++i) {
    v[2 * i] = o[j][C::kChunk / 2 * p + i][e];
    v[2 * i + 1] = o[j][C::kChunk / 2 * p + i][e + 2];
  }
}

// log(sum_t exp(scale q.k_t)) from the reference and the sum of powers of two.
template <typename T>
__device__ __forceinline__ float log_sum(float m, float sum) {
  return sum == 0.0f ? -INFINITY : __fmul_rn(__fadd_rn(m, __fsub_rn(log2f(sum), kShift<T>)), kLn2);
}

// A softmax sum in parts: the lane's elements 32 i + lane.
template <int kPer>
struct Joined {
  float m = -INFINITY, l = 0.0f, o[kPer] = {};

  __device__ __forceinline__ void add(float mk, float lk, const float (&ok)[kPer]) {
    const float top = fmaxf(m, mk), ref = finite_ref(top);
    const float f0 = ex2_ftz(__fsub_rn(m, ref)), f1 = ex2_ftz(__fsub_rn(mk, ref));
    l = __fmaf_rn(l, f0, __fmul_rn(lk, f1));
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = __fmaf_rn(o[i], f0, __fmul_rn(ok[i], f1));
    m = top;
  }
  // Row `row` of out and lse.
  template <typename T>
  __device__ __forceinline__ void finish(const AttentionDecodeArgs& a, long row) const {
    const int lane = threadIdx.x & 31, dh = a.kv.dh;
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (32 * i + lane < dh) static_cast<T*>(a.out)[row * dh + 32 * i + lane] = from_f32<T>(__fmul_rn(o[i], inv));
    if (lane == 0 && a.lse != nullptr) a.lse[row] = log_sum<T>(m, l);
  }
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Cfg<T, D, NT>::kThreads, Cfg<T, D, NT>::kCtas)
    attention_decode_kernel(AttentionDecodeArgs a, const __grid_constant__ CUtensorMap kmap,
                            const __grid_constant__ CUtensorMap vmap, int box_rows, int group, int head_tiles,
                            int tile_heads, int q_on_16, Divisor page_size, int by_block) {
  using C = Cfg<T, D, NT>;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ uint64_t s_full[C::kWarps][C::kStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (lane < C::kStages) mbar_init(&s_full[warp][lane], 1);
  if (lane == 0) {
    prefetch_tmap(&kmap);
    prefetch_tmap(&vmap);
  }
  fence_barrier_init();
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  const PagedKV& kv = a.kv;
  const float c = __fmul_rn(a.scale, kLog2e);
  const Line line{a.lens, a.B, kv.max_pages, kv.page_size, a.window, kv.heads * head_tiles};
  const uint32_t rings = (smem_u32(smem) + 1023u) & ~1023u;
  const uint32_t ring = rings + warp * C::kStage * C::kStages;
  // MMA row g is key `krow` of the tile's first or second eight, and a lane
  // reads V pieces `vcol` of keys t, t + 4, t + 8 and t + 12: so the lanes that
  // shared memory serves together read 16-byte columns that the swizzle (column
  // XOR row) puts into different banks.
  const int krow = ((g & 1) << 2) | (g >> 1), vcol = krow;
  const uint32_t k_lane = krow * C::kRow + ((t ^ krow) << 4);
  const uint32_t v_lane = C::kPart + t * C::kRow + ((vcol ^ t) << 4);

  // Sequences without keys are on no warp's piece: the blocks see to them when
  // they are done.
  auto fill_empty = [&]() {
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
  };

  // The warp's piece of the line, from tile `tile` of item `item` of sequence b.
  const int own = warp * gridDim.x + blockIdx.x;
  long x, x_end;
  int b, item, tile, nt;
  if (by_block) {
    // The block's item, its tiles shared out among the warps.
    b = blockIdx.x / line.per_seq;
    item = blockIdx.x - b * line.per_seq;
    nt = line.tiles(b);
    if (nt == 0) {
      fill_empty();
      return;
    }
    tile = warp * nt / C::kWarps;
    x = tile;
    x_end = (warp + 1) * nt / C::kWarps;
  } else {
    // Neighbouring pieces go to different SMs.
    const int mine = line.own();
    const long total = line.total(mine);
    const int pieces = pieces_of(total, gridDim.x * C::kWarps, a.num_sms);
    if (own >= pieces) {
      fill_empty();
      return;
    }
    x = piece(total, own, pieces);
    x_end = piece(total, own + 1, pieces);
    long start;
    b = line.find(x, mine, start, nt);
    item = static_cast<int>((x - start) / nt);
    tile = static_cast<int>((x - start) - static_cast<long>(item) * nt);
  }
  bool bad = false, alive = true;

  // The tile whose copies start next, ahead of the one in use; its pages are
  // looked up one step earlier still.
  struct Ahead {
    int b, item, tile, nt, left;
    KeyRange r;
    const int* table;
    int page, slot, in;  // of key `lane & 15`
  } ahead;
  ahead.b = b;
  ahead.item = item;
  ahead.tile = tile;
  ahead.nt = nt;
  ahead.left = static_cast<int>(x_end - x);
  auto ahead_sequence = [&]() {
    ahead.r = line.range(ahead.b);
    ahead.table = kv.table + ahead.b * kv.table_stride;
  };
  // Page and slot of key `lane & 15` of the tile ahead.
  auto look_up = [&]() {
    const int key = (ahead.r.first & ~15) + ahead.tile * kTile + (lane & 15);
    ahead.page = -1;
    ahead.slot = 0;
    ahead.in = 0;
    if (ahead.left > 0 && key < ahead.r.end) {
      const int entry = page_size.of(key);
      ahead.slot = key - entry * static_cast<int>(page_size.d);
      ahead.page = ahead.table[entry];
      ahead.in = key >= ahead.r.first;
    }
  };
  uint32_t put = 0, get = 0;  // ring places, in bytes
  int put_bar = 0, get_bar = 0;
  uint32_t parity = 0;  // of the barrier phase that `get_bar` waits for
  // Starts the copies of the tile ahead, moves on and looks up the next one;
  // returns the mask of the tile's keys.
  auto issue = [&]() -> uint32_t {
    const int page = ahead.page, slot = ahead.slot, hk = head_tiles == 1 ? ahead.item : ahead.item / head_tiles;
    const bool on = ahead.in && page >= 0 && page < kv.num_pages;
    bad |= ahead.in && !on;
    const uint32_t mask = __ballot_sync(0xffffffffu, on) & 0xffffu;
    const uint32_t dst = ring + put;
    uint64_t* const bar = &s_full[warp][put_bar];
    put = put + C::kStage == C::kStage * C::kStages ? 0 : put + C::kStage;
    put_bar = put_bar + 1 == C::kStages ? 0 : put_bar + 1;
    if (--ahead.left > 0 && ++ahead.tile == ahead.nt) {
      ahead.tile = 0;
      if (++ahead.item == line.per_seq) {
        ahead.item = 0;
        do ahead.nt = line.tiles(++ahead.b);
        while (ahead.nt == 0);
        ahead_sequence();
      }
    }
    look_up();
    // The warp has read what this place of the ring held.
    __syncwarp();
    if (box_rows == 16) {
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, mask != 0 ? C::kStage : 0);
        if (mask != 0) {
          // The page of key 0 is the tile's, unless key 0 lies before the
          // window: it was looked up all the same.
#pragma unroll
          for (int i = 0; i < C::kBoxes; ++i) {
            tma_box(dst + i * 16 * C::kRow, &kmap, bar, i * C::kRow / C::kSize, hk, slot, page);
            tma_box(dst + C::kPart + i * 16 * C::kRow, &vmap, bar, i * C::kRow / C::kSize, hk, slot, page);
          }
        }
      }
    } else {
      const uint32_t box = (1u << box_rows) - 1u;
      int boxes = 0;
      for (int j = 0; j < 16; j += box_rows) boxes += ((mask >> j) & box) != 0;
      if (lane == 0) mbar_arrive_expect_tx(bar, boxes * box_rows * 2 * C::kPart / 16);
      for (int j = 0; j < 16; j += box_rows) {
        const int page_j = __shfl_sync(0xffffffffu, page, j), slot_j = __shfl_sync(0xffffffffu, slot, j);
        if (lane == 0 && ((mask >> j) & box) != 0) {
#pragma unroll
          for (int i = 0; i < C::kBoxes; ++i) {
            tma_box(dst + (i * 16 + j) * C::kRow, &kmap, bar, i * C::kRow / C::kSize, hk, slot_j, page_j);
            tma_box(dst + C::kPart + (i * 16 + j) * C::kRow, &vmap, bar, i * C::kRow / C::kSize, hk, slot_j, page_j);
          }
        }
      }
    }
    return mask;
  };

  // A warp's partial of the block's item: where its ring was, when its last tile
  // has been read.
  auto block_part = [&](int w) {
    return reinterpret_cast<float*>(smem + (rings - smem_u32(smem)) + w * C::kStage * C::kStages);
  };
  static_assert(C::kSlot * 4 <= C::kStage * C::kStages, "partial");

  uint32_t mask[C::kStages];
  ahead_sequence();
  look_up();
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) mask[i] = issue();

  while (true) {
    const int n = static_cast<int>(min(static_cast<long>(nt - tile), x_end - x));
    const int hk = item / head_tiles, ht = item - hk * head_tiles;
    const int h0 = hk * group + ht * tile_heads;  // first query head of the tile
    const int heads = min(tile_heads, group - ht * tile_heads);

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
    // float32: q's small parts, kept beside the large ones where registers are
    // left, else split off again in every tile.
    constexpr bool kKeepLo = C::kF32Cache && D <= 64 && NT == 1;
    uint32_t q_lo[kKeepLo ? NT : 1][kKeepLo ? C::kKPieces : 1][4];
    if constexpr (kKeepLo) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int p = 0; p < C::kKPieces; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) split_tf32(__uint_as_float(q[j][p][i]), q[j][p][i], q_lo[j][p][i]);
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

    for (int i = 0; i < n; ++i) {
      mask[C::kStages - 1] = issue();
      if (!__all_sync(0xffffffffu, mbar_wait(&s_full[warp][get_bar], parity, a.status))) {
        alive = false;
        break;
      }
      if (++get_bar == C::kStages) {
        get_bar = 0;
        parity ^= 1u;
      }
      const uint32_t keys = mask[0];
#pragma unroll
      for (int j = 0; j + 1 < C::kStages; ++j) mask[j] = mask[j + 1];
      const uint32_t src = ring + get;
      get = get + C::kStage == C::kStage * C::kStages ? 0 : get + C::kStage;
      if (keys == 0) continue;
      if (keys != 0xffffu) {
        // V of keys that are not seen: whatever lies there times a probability
        // of 0 must be 0.
        if (!((keys >> (lane & 15)) & 1u))
          for (int i = lane >> 4; i < C::kBoxes * 8; i += 2)
            sts128(src + C::kPart + ((i >> 3) * 16 + (lane & 15)) * C::kRow + (i & 7) * 16,
                   make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        fence_proxy_async_smem();
        __syncwarp();
      }

      // The lane's 16-byte pieces of K rows krow and krow + 8 and of V rows
      // t + 4 (row % 2) + 8 (row / 2).
      auto k_piece = [&](int row, int p) {
        return lds16(src + (k_lane ^ ((p & 1) << 6)) + (p >> 1) * 16 * C::kRow + row * 8 * C::kRow);
      };
      auto v_piece = [&](int row, int p) {
        return lds16(src + (v_lane ^ ((row & 1) << 6)) + ((row & 1) * 4 + (row >> 1) * 8 + p * 16) * C::kRow);
      };
      // S^T: rows are the keys krow and krow + 8, columns the heads 2t and 2t + 1.
      // Two chains of sums: float32 keeps its small products apart, the others
      // halve the wait for one another.
      float s[NT][4], s_lo[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = s_lo[j][e] = 0.0f;
      constexpr int kAtOnce = C::kKPieces < 4 ? C::kKPieces : 4;  // pieces loaded before the first product
#pragma unroll
      for (int p0 = 0; p0 < C::kKPieces; p0 += kAtOnce) {
        uint4 k0[kAtOnce], k1[kAtOnce];
#pragma unroll
        for (int p = 0; p < kAtOnce; ++p) {
          k0[p] = k_piece(0, p0 + p);
          k1[p] = k_piece(1, p0 + p);
        }
#pragma unroll
        for (int p1 = 0; p1 < kAtOnce; ++p1) {
          const int p = p0 + p1;
          const uint32_t w0[4] = {k0[p1].x, k0[p1].y, k0[p1].z, k0[p1].w};
          const uint32_t w1[4] = {k1[p1].x, k1[p1].y, k1[p1].z, k1[p1].w};
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const uint32_t f[4] = {w0[e], w1[e], w0[e + 1], w1[e + 1]};
            if constexpr (C::kF32Cache) {
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int u = 0; u < 4; ++u) cut_tf32(__uint_as_float(f[u]), hi[u], lo[u]);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                uint32_t qh[2], ql[2];
                if constexpr (kKeepLo) {
                  qh[0] = q[j][p][e];
                  qh[1] = q[j][p][e + 1];
                  ql[0] = q_lo[j][p][e];
                  ql[1] = q_lo[j][p][e + 1];
                } else {
                  split_tf32(__uint_as_float(q[j][p][e]), qh[0], ql[0]);
                  split_tf32(__uint_as_float(q[j][p][e + 1]), qh[1], ql[1]);
                }
                mma8(s[j], hi, qh[0], qh[1]);
                mma8(s_lo[j], hi, ql[0], ql[1]);
                mma8(s_lo[j], lo, qh[0], qh[1]);
              }
            } else {
#pragma unroll
              for (int j = 0; j < NT; ++j) mma16(e == 0 ? s[j] : s_lo[j], f, q[j][p][e], q[j][p][e + 1], T());
            }
          }
        }
      }
      // V is on its way while the scores are turned into probabilities.
      constexpr bool kEarlyV = C::kVPieces <= 2;
      uint4 v_early[kEarlyV ? C::kVPieces : 1][4];
      if constexpr (kEarlyV) {
#pragma unroll
        for (int p = 0; p < C::kVPieces; ++p)
#pragma unroll
          for (int row = 0; row < 4; ++row) v_early[p][row] = v_piece(row, p);
      }

      // Scores in powers of two, the running maximum, the probabilities.
      const bool k_lo = (keys >> krow) & 1u, k_hi = (keys >> (krow + 8)) & 1u;
      bool over = false;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = __fadd_rn(s[j][e], s_lo[j][e]);
          s[j][e] = (e < 2 ? k_lo : k_hi) ? __fmul_rn(v, c) : -INFINITY;
          const float above = __fsub_rn(s[j][e], m[j][e & 1]);
          over |= C::kF32Cache ? !(above <= kSlack) : above > kSlack;  // float32: NaN too
        }
      // The reference m of a head moves only when a score passes it by 2^8:
      // then to the maximum so far, everything summed up being rescaled.
      if (__any_sync(0xffffffffu, over)) {
        if constexpr (C::kF32Cache) {
          // The parts of an infinity are NaN, and so is then the score.  (Nothing
          // to find any more where the head's sum is NaN already: with NaN in q a call
          // of 131071 keys, heads of 128, takes 248 us, others 222; without this 1090.)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int h = 8 * j + 2 * t + (e & 1);
              if (isnan(s[j][e]) && h < heads && !isnan(l[j][e & 1]))
                s[j][e] = __fmul_rn(c, whole_score(static_cast<const float*>(a.q) + b * a.q_seq + (h0 + h) * a.q_head, src,
                                                   krow + 4 * (e & 2), kv.dh));
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(s[j][e], s[j][e + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            top = fmaxf(m[j][e], top);
            const float alpha = ex2_ftz(__fsub_rn(m[j][e], finite_ref(top)));
            m[j][e] = top;
            l[j][e] = __fmul_rn(l[j][e], alpha);
#pragma unroll
            for (int i2 = 0; i2 < C::kMTiles; ++i2) {
              o[j][i2][e] = __fmul_rn(o[j][i2][e], alpha);
              o[j][i2][e + 2] = __fmul_rn(o[j][i2][e + 2], alpha);
            }
          }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float ref = finite_ref(m[j][e]);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float d = __fsub_rn(s[j][e + 2 * half], ref);
            s[j][e + 2 * half] = ex2_ftz(kShift<T> == 0.0f ? d : __fadd_rn(d, kShift<T>));
          }
          l[j][e] = __fadd_rn(l[j][e], __fadd_rn(s[j][e], s[j][e + 2]));
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
              const int from = (2 * t + i2) * 4 + (g >> 1);
              const float p0 = __shfl_sync(0xffffffffu, s[j][2 * h], from);
              const float p1 = __shfl_sync(0xffffffffu, s[j][2 * h + 1], from);
              split_tf32((g & 1) ? p1 : p0, bh[j][h][i2], bl[j][h][i2]);
            }
#pragma unroll
        for (int p = 0; p < C::kVPieces; ++p) {
          uint32_t v[4][4];
#pragma unroll
          for (int row = 0; row < 4; ++row) {
            uint4 w;
            if constexpr (kEarlyV) w = v_early[p][row];
            else w = v_piece(row, p);
            v[row][0] = w.x;
            v[row][1] = w.y;
            v[row][2] = w.z;
            v[row][3] = w.w;
          }
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            float acc[NT][4], acc_lo[NT][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int u = 0; u < 4; ++u)
                cut_tf32(__uint_as_float(v[2 * h + (u >> 1)][2 * i2 + (u & 1)]), hi[u], lo[u]);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                if (h == 0) {
                  mma8_first(acc[j], hi, bh[j][h][0], bh[j][h][1]);
                  mma8_first(acc_lo[j], hi, bl[j][h][0], bl[j][h][1]);
                } else {
                  mma8(acc[j], hi, bh[j][h][0], bh[j][h][1]);
                  mma8(acc_lo[j], hi, bl[j][h][0], bl[j][h][1]);
                }
                mma8(acc_lo[j], lo, bh[j][h][0], bh[j][h][1]);
              }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                o[j][2 * p + i2][e] = __fadd_rn(o[j][2 * p + i2][e], __fadd_rn(acc[j][e], acc_lo[j][e]));
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
            uint4 w;
            if constexpr (kEarlyV) w = v_early[p][row];
            else w = v_piece(row, p);
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
              float acc[4];
              mma16_first(acc, f, bh[j][0], bh[j][1], T());
              mma16(acc, f, bl[j][0], bl[j][1], T());
#pragma unroll
              for (int e = 0; e < 4; ++e) o[j][4 * p + i2][e] = __fadd_rn(o[j][4 * p + i2][e], acc[e]);
            }
          }
        }
      }
    }
    if (!alive) break;

    // The item's part: finished, or one of the warp's two partials.
    const bool whole = n == nt;
    float* const part = by_block ? block_part(warp)
                                 : static_cast<float*>(a.workspace) +
                                       (2 * static_cast<long>(own) + (tile > 0 ? 0 : 1)) * C::kSlot;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int h = 8 * j + 2 * t + e;
        float sum = l[j][e];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (h >= heads) continue;
        const long row = static_cast<long>(b) * a.q_heads + h0 + h;
        const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
        if (g == 0) {
          if (!whole) {
            part[C::kHeads * D + h] = m[j][e];
            part[C::kHeads * (D + 1) + h] = sum;
          } else if (a.lse != nullptr) {
            a.lse[row] = log_sum<T>(m[j][e], sum);
          }
        }
#pragma unroll
        for (int p = 0; p < C::kVPieces; ++p) {
          const int d = (p * 8 + vcol) * C::kChunk;
          if (d >= kv.dh) continue;
          float v[C::kChunk];
          row_of<C, NT>(o, j, p, e, v);
          if (whole) {
            Vec<T, C::kChunk> y;
#pragma unroll
            for (int i = 0; i < C::kChunk; ++i) y.e[i] = from_f32<T>(__fmul_rn(v[i], inv));
            y.store(static_cast<T*>(a.out) + row * kv.dh + d);
          } else {
            Vec<float, C::kChunk> y;
#pragma unroll
            for (int i = 0; i < C::kChunk; ++i) y.e[i] = v[i];
            y.store(part + h * D + d);
          }
        }
      }
    }

    x += n;
    if (x >= x_end) break;
    tile = 0;
    if (++item == line.per_seq) {
      item = 0;
      do nt = line.tiles(++b);
      while (nt == 0);
    }
  }
  // Every copy has been waited for, unless a wait ran out: then give the others
  // their time before the shared memory goes.
  if (!alive)
    for (int i = 1; i < C::kStages; ++i) {
      if (++get_bar == C::kStages) {
        get_bar = 0;
        parity ^= 1u;
      }
      mbar_wait(&s_full[warp][get_bar], parity, a.status);
    }
  if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(a.status, kStatusBadIndex);
  if (by_block && nt > 1) {
    __syncthreads();
    const int hk = item / head_tiles, ht = item - hk * head_tiles;
    const int heads = min(tile_heads, group - ht * tile_heads);
    constexpr int kPer = D / 32;
    for (int h = warp; h < heads; h += C::kWarps) {
      Joined<kPer> sum;
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w) {
        const float* const part = block_part(w);
        float o[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) o[i] = 32 * i + lane < kv.dh ? part[h * D + 32 * i + lane] : 0.0f;
        sum.add(part[C::kHeads * D + h], part[C::kHeads * (D + 1) + h], o);
      }
      sum.template finish<T>(a, static_cast<long>(b) * a.q_heads + hk * group + ht * tile_heads + h);
    }
  }
  fill_empty();
}

// Joins the partials of the cut items, for head blockIdx.y of their tiles.
// Every warp looks at one beginning of a piece, i + 1: if it is the first to
// cut its item, the item is this warp's.  A few partials the warp joins alone;
// an item of many (a long sequence) is left to all warps of the block.
constexpr int kJoinWarps = 8;
constexpr int kAlone = 12;  // partials that a warp joins alone

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * kJoinWarps)
    attention_join_kernel(AttentionDecodeArgs a, int group, int head_tiles, int tile_heads, int warps) {
  using C = Cfg<T, D, NT>;
  constexpr int kPer = D / 32;
  struct Item {
    long row;         // of out
    int first, last;  // its pieces; first > last: none
  };
  __shared__ Item s_item[kJoinWarps];
  __shared__ float s_m[kJoinWarps], s_l[kJoinWarps], s_o[kJoinWarps][D];
  const PagedKV& kv = a.kv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y;
  const Line line{a.lens, a.B, kv.max_pages, kv.page_size, a.window, kv.heads * head_tiles};
  // The lengths were complete before the attention kernel began, and this
  // kernel begins after all of that kernel's blocks have; only the partial
  // results have to be waited for.
  const int own = line.own();
  const long total = line.total(own);
  const int pieces = pieces_of(total, warps, a.num_sms);
  // Joins the partials first + from, first + from + step, ... of an item.
  auto join = [&](const Item& it, int from, int step, Joined<kPer>& sum) {
    constexpr int kBatch = 4;  // partials in flight
    for (int k0 = it.first + from; k0 <= it.last; k0 += kBatch * step) {
      float mk[kBatch], lk[kBatch], ok[kBatch][kPer];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int k = k0 + u * step;
        const float* part = static_cast<const float*>(a.workspace) +
                            (2 * static_cast<long>(k) + (k == it.first ? 1 : 0)) * C::kSlot;
        const bool on = k <= it.last;
        mk[u] = on ? part[C::kHeads * D + h] : -INFINITY;
        lk[u] = on ? part[C::kHeads * (D + 1) + h] : 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) ok[u][i] = on && 32 * i + lane < kv.dh ? part[h * D + 32 * i + lane] : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) sum.add(mk[u], lk[u], ok[u]);
    }
  };
  bool waited = false;
  for (int i0 = 0; i0 + 1 < pieces || !waited; i0 += gridDim.x * kJoinWarps) {
    const int i = i0 + blockIdx.x * kJoinWarps + warp;
    Item it = {0, 0, -1};
    if (i + 1 < pieces) {
      const long before = piece(total, i, pieces), cut = piece(total, i + 1, pieces);
      long start;
      int nt;
      const int b = line.find(cut, own, start, nt), item = static_cast<int>((cut - start) / nt);
      const int hk = item / head_tiles, ht = item - hk * head_tiles;
      start += static_cast<long>(item) * nt;
      if (start < cut && start >= before && h < min(tile_heads, group - ht * tile_heads)) {
        it.row = static_cast<long>(b) * a.q_heads + hk * group + ht * tile_heads + h;
        it.first = i;
        // The last k with piece(k) < start + nt.
        it.last = static_cast<int>(min(((start + nt) * pieces + total - 1) / total, static_cast<long>(pieces)) - 1);
      }
    }
    if (!waited) {
      pdl_wait();
      pdl_trigger();
      waited = true;
    }
    const bool alone = it.last - it.first < kAlone;
    if (alone && it.last >= it.first) {
      Joined<kPer> sum;
      join(it, 0, 1, sum);
      sum.template finish<T>(a, it.row);
    }
    if (lane == 0) {
      s_item[warp] = it;
      if (alone) s_item[warp].last = it.first - 1;
    }
    __syncthreads();
    for (int w = 0; w < kJoinWarps; ++w) {
      const Item many = s_item[w];
      if (many.last < many.first) continue;
      Joined<kPer> sum;
      join(many, warp, kJoinWarps, sum);
#pragma unroll
      for (int j = 0; j < kPer; ++j) s_o[warp][32 * j + lane] = sum.o[j];
      if (lane == 0) {
        s_m[warp] = sum.m;
        s_l[warp] = sum.l;
      }
      __syncthreads();
      if (warp == 0) {
        Joined<kPer> all;
#pragma unroll
        for (int u = 0; u < kJoinWarps; ++u) {
          float ok[kPer];
#pragma unroll
          for (int j = 0; j < kPer; ++j) ok[j] = s_o[u][32 * j + lane];
          all.add(s_m[u], s_l[u], ok);
        }
        all.template finish<T>(a, many.row);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::atomic<void*> fn{nullptr};
  void* p = fn.load(std::memory_order_acquire);
  if (p == nullptr) {
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    fn.store(p, std::memory_order_release);
  }
  return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
}

// The cache as a tensor (element, head, slot, page) with boxes of box_rows
// slots and 128 bytes of one head, in the 128-byte swizzle.  Elements behind dh
// read as zero.
template <typename T>
bool cache_map(CUtensorMap* map, const PagedKV& kv, const void* base, long page, long slot, long head, int box_rows) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  constexpr cuuint64_t size = sizeof(T);
  // A dimension of one entry takes no steps, but its stride has to be valid.
  auto step = [](long stride, int n) { return n > 1 ? static_cast<cuuint64_t>(stride) * size : cuuint64_t(16); };
  const int pages = kv.num_pages > 0 ? kv.num_pages : 1;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(kv.dh), static_cast<cuuint64_t>(kv.heads),
                        static_cast<cuuint64_t>(kv.page_size), static_cast<cuuint64_t>(pages)};
  cuuint64_t strides[3] = {step(head, kv.heads), step(slot, kv.page_size), step(page, pages)};
  cuuint32_t box[4] = {static_cast<cuuint32_t>(128 / size), 1, static_cast<cuuint32_t>(box_rows), 1};
  cuuint32_t one[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = sizeof(T) == 4                    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return fn(map, type, 4, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
  int box_rows = 16;
  while (a.kv.page_size % box_rows != 0) box_rows /= 2;
  // Without pages there is no cache to describe and no key is ever copied; any
  // device address makes a valid map.
  const void* const k = a.kv.num_pages > 0 ? a.kv.k : a.out;
  const void* const v = a.kv.num_pages > 0 ? a.kv.v : a.out;
  CUtensorMap kmap, vmap;
  if (!cache_map<T>(&kmap, a.kv, k, a.kv.k_page, a.kv.k_slot, a.kv.k_head, box_rows) ||
      !cache_map<T>(&vmap, a.kv, v, a.kv.v_page, a.kv.v_slot, a.kv.v_head, box_rows))
    return cudaErrorInvalidValue;
  auto kernel = attention_decode_kernel<T, D, NT>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(kernel, C::kSmem, allowed);
  if (e != cudaSuccess) return e;
  const long items = static_cast<long>(a.B) * a.kv.heads * head_tiles;
  const bool by_block = kBlocksPay<C> && item_per_block(items, static_cast<long>(a.kv.max_pages) * a.kv.page_size, blocks,
                                                        C::kWarps);
  e = launch_pdl(kernel, dim3(by_block ? static_cast<int>(items) : blocks), dim3(C::kThreads), C::kSmem, s, a, kmap,
                 vmap, box_rows, group, head_tiles, tile_heads, q_on_16 ? 1 : 0, Divisor(a.kv.page_size),
                 by_block ? 1 : 0);
  if (e != cudaSuccess || by_block) return e;
  // As many blocks as the longest line of this cache can have pieces for.
  const long most = items * ((static_cast<long>(a.kv.max_pages) * a.kv.page_size + kTile - 1) / kTile);
  const int joins = (pieces_of(most, blocks * C::kWarps, a.num_sms) + kJoinWarps - 1) / kJoinWarps;
  return launch_pdl(attention_join_kernel<T, D, NT>, dim3(joins > 0 ? joins : 1, tile_heads), dim3(32 * kJoinWarps), 0, s, a, group,
                    head_tiles, tile_heads, blocks * C::kWarps);
}

template <typename T, int D, int NT>
size_t workspace(int num_sms) {
  using C = Cfg<T, D, NT>;
  return static_cast<size_t>(2) * num_sms * C::kCtas * C::kWarps * C::kSlot * sizeof(float);
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
