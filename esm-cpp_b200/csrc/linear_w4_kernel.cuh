// A Linear with 4-bit weights and group scales for few activation rows:
//   out[m, n] = sum_k x[m, k] * (q[n, k] - z[n, k / G]) * s[n, k / G] + bias[n]
//
// Bound by HBM: the packed weights are read once (N K / 2 bytes) and x is
// small.  At 0.5 bytes a weight the issue slots are the next limit (a B200
// reads about 90 weights per SM and clock against 128 lanes), so the products
// run on the tensor cores: mma.sync m16n8k16 with 16 weight rows on the M side
// and the activation rows as its 8 columns.  The weights become the integers
// q - z, exact in half or bfloat16: their nibbles are set into the mantissa of
// 1024 (128 for bfloat16) by one logic operation per pair and the offset and
// zero point come off in one packed add.  A group's sum is an exact-product
// float32 accumulation that meets its scale once, in float32.
//
// float32 activations enter as three bfloat16 columns, x = hi + mid + lo, each
// the leading 8 bits of what is left (truncated, so that nothing overflows):
// all 24 bits, in columns that would be empty for few rows.  The weights carry
// 2^-11 on the bfloat16 path, taken off again in the scale, so that sums of
// 128 products near the type's largest value stay finite.
//
// Layout: the order of a sum over k is free.  A warp takes steps of 16 rows x
// 256 columns (128 bytes a row), copied by cp.async into its own ring of
// kStages slots; ldmatrix hands lane (g, t) word t of each 16-byte piece of
// row g, eight consecutive columns whose nibbles pair up as (0,4) (1,5) (2,6)
// (3,7).  x is laid out in shared memory in that order when it is staged, once
// per block.  A piece of 16 bytes is 32 columns, so groups of 32, 64 and 128
// end after 1, 2 or 4 pieces.
//
// Work: a block takes an equal, consecutive share of the 16-row tiles, and its
// 8 warps equal, consecutive shares of their steps, so that each streams one
// run of memory and nothing waits in between.  A tile inside one warp's share
// is finished there; one that is cut leaves partial sums in shared memory, two
// per warp at most, joined when all warps are done.  Where x does not fit
// beside the rings it is staged in phases of K, the tiles' sums being kept in
// shared memory from phase to phase.
#pragma once

#include "common.cuh"
#include "dtype.cuh"
#include "kernels.cuh"

namespace esmb200 {
namespace w4 {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxSmem = 224 * 1024;
constexpr int kStep = 256;       // columns
constexpr int kBytes = kStep / 2;  // of a row
constexpr int kStages = 4;
constexpr int kMaxAcc = 32 * 1024;  // bytes of the sums that are kept from phase to phase

// A: rows on 16-byte boundaries; else the nine 16-byte blocks that cover a
// row's 128 bytes are copied.
template <bool A>
struct Ring {
  static constexpr int kPitch = A ? 128 : 144;
  static constexpr int kSlot = 16 * kPitch;
  static constexpr int kAll = kWarps * kStages * kSlot;
};
// Bytes of the warps' partial sums: two of 16 rows x 8 NT columns each.
__host__ __device__ constexpr int partial_bytes(int nt) { return kWarps * 2 * 16 * 8 * nt * 4; }

struct Plan {
  int tiles;     // 16-row tiles, shared out evenly over the blocks
  int at_once;   // tiles that a block takes through all phases together
  int steps;     // of 256 columns
  int phase;     // steps staged at a time
  int cols;      // columns in use: rows of x, times 3 for float32
  int x_bytes;   // of shared memory for x
  int m0, rows;  // the rows of x of this launch
  int x_on_16;
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

// lds16 for the lanes with `on`; the others keep what they have.
__device__ __forceinline__ void lds16_if(uint4& v, uint32_t a, bool on) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "@p ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
      : "r"(a), "r"(static_cast<int>(on))
      : "memory");
}

// (a & b) | c in one operation: the compiler makes two of it when b and c are
// both constants.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// The operations that depend on the MMA's type: half for half activations,
// bfloat16 for the others.
template <typename XT>
struct Mma {  // bfloat16
  // -(128 + z) 2^-11, twice.
  static __device__ __forceinline__ uint32_t offset(int z) { return 0xBD80BD80u | (static_cast<uint32_t>(z) * 0x10001u); }
  // The eight columns of a word as q - z (times 2^-11), in pairs (0,4) (1,5) (2,6) (3,7).
  static __device__ __forceinline__ void weights(uint32_t w, uint32_t off, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = and_or(w >> (4 * i), 0x000F000Fu, 0x43004300u);  // 128 + q
      asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(p[i]) : "r"(b), "r"(0x3A003A00u), "r"(off));
    }
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static constexpr float kScale = 2048.0f;
};
template <>
struct Mma<__half> {
  // -(1024 + z), twice.
  static __device__ __forceinline__ uint32_t offset(int z) { return 0xE400E400u | (static_cast<uint32_t>(z) * 0x10001u); }
  // Nibbles in bits 4-7 become 1024 + 16 q, and (1024 + 16 q) / 16 - (64 + z) is
  // exact too, so that one shift serves four pairs.
  static __device__ __forceinline__ void weights(uint32_t w, uint32_t off, uint32_t (&p)[4]) {
    const uint32_t off16 = 0xD400D400u | ((off & 0x000F000Fu) << 4);  // -(64 + z)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = w >> (8 * i);
      const uint32_t lo = and_or(v, 0x000F000Fu, 0x64006400u), hi = and_or(v, 0x00F000F0u, 0x64006400u);
      asm("add.rn.f16x2 %0, %1, %2;" : "=r"(p[2 * i]) : "r"(lo), "r"(off));
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(p[2 * i + 1]) : "r"(hi), "r"(0x2C002C00u), "r"(off16));
    }
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static constexpr float kScale = 1.0f;
};

// 16 bits of each of the eight elements, as pairs (0,4) (1,5) (2,6) (3,7).
__device__ __forceinline__ uint4 interleave(const uint16_t (&e)[8]) {
  auto pair = [&](int i) { return static_cast<uint32_t>(e[i]) | (static_cast<uint32_t>(e[i + 4]) << 16); };
  return make_uint4(pair(0), pair(1), pair(2), pair(3));
}

// Stages steps [c0, c0 + n) of x: eight columns k8 of row m at
// xs[((k8 / 4) * cols + column) * 4 + k8 % 4] (16-byte units), k8 counted from
// step c0.
template <typename XT>
__device__ __forceinline__ void stage_x(const LinearW4Args& a, const Plan& p, uint4* xs, int c0, int n) {
  const int n8 = n * (kStep / 8);
  for (int i = threadIdx.x; i < p.rows * n8; i += kThreads) {
    const int m = i / n8, k8 = i - m * n8;
    const int k = c0 * kStep + k8 * 8;
    const XT* src = static_cast<const XT*>(a.x) + static_cast<long>(p.m0 + m) * a.ldx + k;
    Vec<XT, 8> v;
    if (p.x_on_16 && k + 8 <= a.K) {
      v.load(src);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v.e[e] = k + e < a.K ? src[e] : from_f32<XT>(0.0f);
    }
    uint4* dst = xs + (static_cast<long>(k8 >> 2) * p.cols + m * kSplit<XT>) * 4 + (k8 & 3);
    if constexpr (kSplit<XT> == 1) {
      uint16_t e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = *reinterpret_cast<const uint16_t*>(&v.e[j]);
      *dst = interleave(e);
    } else {
      uint16_t e[3][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float rest = v.e[j];
        const bool finite = fabsf(rest) <= 3.402823466e38f;
        // An infinity or NaN goes whole into the first column (a NaN's payload
        // may lie in the bits that are cut off).
        if (!finite && rest != rest) rest = __uint_as_float(0x7FC00000u);
#pragma unroll
        for (int sp = 0; sp < 3; ++sp) {
          const uint32_t top = __float_as_uint(rest) & 0xFFFF0000u;
          e[sp][j] = static_cast<uint16_t>(top >> 16);
          rest = finite ? __fsub_rn(rest, __uint_as_float(top)) : 0.0f;
        }
      }
#pragma unroll
      for (int sp = 0; sp < 3; ++sp) dst[sp * 4] = interleave(e[sp]);
    }
  }
}

static_assert(64 * kStep * 2 + Ring<false>::kAll + partial_bytes(8) + kMaxAcc <= kMaxSmem,
              "the shortest phase of 64 columns fits");

// G: columns of a group.
template <typename XT, int G, int NT, bool A>
__global__ void __launch_bounds__(kThreads, NT <= 4 ? 2 : 1) linear_w4_kernel(LinearW4Args a, Plan p) {
  using R = Ring<A>;
  using M = Mma<XT>;
  constexpr int kGroups = kStep / G;  // of a step: 2, 4 or 8
  constexpr int kHeld = kGroups > 4 ? kGroups / 4 : 1;  // of a row's that one lane holds
  extern __shared__ __align__(128) unsigned char smem[];
  uint4* const xs = reinterpret_cast<uint4*>(smem);
  float* const part = reinterpret_cast<float*>(smem + p.x_bytes + R::kAll);  // [warp][2][16][8 NT]
  float* const acc_keep = reinterpret_cast<float*>(smem + p.x_bytes + R::kAll + partial_bytes(NT));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + p.x_bytes + warp * kStages * R::kSlot;
  const int tile0 = static_cast<int>(static_cast<long>(blockIdx.x) * p.tiles / gridDim.x);
  const int tile1 = static_cast<int>((static_cast<long>(blockIdx.x) + 1) * p.tiles / gridDim.x);
  const int row_bytes = static_cast<int>((static_cast<long>(a.K) + 1) / 2);
  pdl_wait();
  pdl_trigger();

  // A place in the warp's share of the work: steps [at, end) of the tiles
  // [first, first + p.at_once) in one phase, counted tile after tile.
  struct Place {
    int first, phase0;       // phase0: the phase's first step
    int at, end;
    int tile, step, steps;  // of the phase
  };
  auto enter = [&](Place& c) {
    const int n = min(p.at_once, tile1 - c.first);
    c.steps = min(p.phase, p.steps - c.phase0);
    const int all = n > 0 ? n * c.steps : 0;
    c.at = warp * all / kWarps;
    c.end = (warp + 1) * all / kWarps;
    c.tile = c.steps > 0 ? c.at / c.steps : 0;
    c.step = c.at - c.tile * c.steps;
    c.tile += c.first;
  };
  // On to the next step; false behind the last one.
  auto skip_empty = [&](Place& c) -> bool {
    while (c.at >= c.end) {
      if (c.first >= tile1) return false;
      c.phase0 += p.phase;
      if (c.phase0 >= p.steps) {
        c.phase0 = 0;
        c.first += p.at_once;
        if (c.first >= tile1) return false;
      }
      enter(c);
    }
    return true;
  };

  // Copies.  A lane copies the same places of every tile; within a tile its
  // addresses move by 128 bytes a step.
  constexpr int kCopies = A ? 4 : 5;
  const uint8_t* src[kCopies];
  uint32_t src_dst[kCopies];
  int src_row[kCopies];  // -1: nothing to copy
  int src_from[kCopies];  // first byte within the step's 128 bytes of the row
#pragma unroll
  for (int h = 0; h < kCopies; ++h) {
    const int id = lane + 32 * h;
    const int row = A ? id >> 3 : id / 9, piece = A ? id & 7 : id - row * 9;
    // Where an unaligned row's pieces start in a 16-byte block: the same in
    // every tile, 16 rows being a multiple of 16 bytes whatever ldw is.
    const int sh = A ? 0 : static_cast<int>((reinterpret_cast<uintptr_t>(a.W) + row * a.ldw) & 15);
    src_row[h] = row < 16 ? row : -1;
    src_from[h] = piece * 16 - sh;
    src_dst[h] = ring + (A ? row * 128 + ((piece ^ (row & 7)) << 4) : row * R::kPitch + piece * 16);
  }
  // Rows behind N and blocks behind a row's end are filled with zeros; their
  // copies read nothing, from W's first block.
  const uint8_t* const nowhere = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(a.W) & ~uintptr_t(15));
  uint32_t put = 0;
  Place ahead;
  ahead.first = tile0;
  ahead.phase0 = 0;
  enter(ahead);
  bool more = skip_empty(ahead), moved = true;
  // Starts the copies of the warp's next step.
  auto issue = [&]() {
    if (more) {
      const int left = row_bytes - (ahead.phase0 + ahead.step) * kBytes;
      if (moved) {
#pragma unroll
        for (int h = 0; h < kCopies; ++h) {
          const long n = static_cast<long>(ahead.tile) * 16 + src_row[h];
          src[h] = src_row[h] >= 0 && n < a.N
                       ? a.W + n * a.ldw + (ahead.phase0 + ahead.step) * static_cast<long>(kBytes) + src_from[h]
                       : nullptr;
        }
        moved = false;
      }
      if (A && left >= kBytes && ahead.tile * 16 + 16 <= a.N) {
#pragma unroll
        for (int h = 0; h < kCopies; ++h) cp_async16(src_dst[h] + put, src[h], 16);
      } else {
#pragma unroll
        for (int h = 0; h < kCopies; ++h) {
          // Unaligned: a block that holds a byte of the row's piece is copied
          // whole; it never leaves the 16 bytes that some byte of W lies in.
          int bytes = A ? min(max(left - src_from[h], 0), 16) : src_from[h] < min(left, kBytes) ? 16 : 0;
          if (src[h] == nullptr) bytes = 0;
          if (A || src_row[h] >= 0) cp_async16(src_dst[h] + put, bytes > 0 ? src[h] : nowhere, bytes);
        }
      }
#pragma unroll
      for (int h = 0; h < kCopies; ++h)
        if (src[h] != nullptr) src[h] += kBytes;
      ++ahead.at;
      if (++ahead.step == ahead.steps) {
        ahead.step = 0;
        ++ahead.tile;
        moved = true;
      }
      if (ahead.at == ahead.end) {
        more = skip_empty(ahead);
        moved = true;
      }
    }
    put = put + R::kSlot == kStages * R::kSlot ? 0 : put + R::kSlot;
    cp_commit();
  };

  // Scales and zero points of rows g and g + 8 for a step: lane t holds those
  // of groups t and t + 4 (t % 2 where a step has two).  They are loaded two
  // steps ahead and kept as they are until used: a conversion here would make
  // the warp wait for the load.  Rows behind N and groups behind K read the
  // last row's and the last group's: those rows are not written, and there x
  // is 0.
  struct Scales {
    uint32_t s[2][kHeld];
    int z[2][kHeld];
  };
  const int groups = static_cast<int>((static_cast<long>(a.K) + G - 1) / G);
  const bool f32_scales = a.scale_type == kF32;
  const char* s_row[2];
  const uint8_t* z_row[2];
  Place scaled = ahead;
  bool s_more = more, s_moved = true;
  auto load_scales = [&](Scales& v) {
    if (!s_more) return;
    if (s_moved) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long n = min(static_cast<long>(scaled.tile) * 16 + g + 8 * h, static_cast<long>(a.N) - 1);
        s_row[h] = static_cast<const char*>(a.scales) + n * a.lds * (f32_scales ? 4 : 2);
        if (a.zeros != nullptr) z_row[h] = a.zeros + n * a.ldz;
      }
      s_moved = false;
    }
    const int grp0 = (scaled.phase0 + scaled.step) * kGroups + (t & (kGroups - 1));
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const uint32_t at = static_cast<uint32_t>(min(grp0 + 4 * u, groups - 1));
      if (f32_scales) {
#pragma unroll
        for (int h = 0; h < 2; ++h) v.s[h][u] = __ldg(reinterpret_cast<const uint32_t*>(s_row[h]) + at);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) v.s[h][u] = __ldg(reinterpret_cast<const uint16_t*>(s_row[h]) + at);
      }
      if (a.zeros != nullptr) {
#pragma unroll
        for (int h = 0; h < 2; ++h) v.z[h][u] = __ldg(z_row[h] + at);
      }
    }
    ++scaled.at;
    if (++scaled.step == scaled.steps) {
      scaled.step = 0;
      ++scaled.tile;
      s_moved = true;
    }
    if (scaled.at == scaled.end) {
      s_more = skip_empty(scaled);
      s_moved = true;
    }
  };
  auto scale_of = [&](uint32_t bits) {
    const float v = f32_scales               ? __uint_as_float(bits)
                    : a.scale_type == kF16 ? __half2float(__ushort_as_half(static_cast<uint16_t>(bits)))
                                           : __uint_as_float(bits << 16);
    return __fmul_rn(v, M::kScale);
  };
  // The value of the step's group grp, held by lane grp % 4 (% 2) of the row.
  auto of_group = [&](auto v, int grp) { return __shfl_sync(0xffffffffu, v, (lane & ~3) | (grp & 3)); };

#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue();
  Scales now, next;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      now.s[h][u] = next.s[h][u] = 0u;
      now.z[h][u] = next.z[h][u] = 8;
    }
  load_scales(now);
  load_scales(next);

  const uint32_t x_lane = smem_u32(smem) + (g * 4 + t) * 16;
  const uint32_t x_col = static_cast<uint32_t>(p.cols) * 64;  // bytes from one 16-byte piece's columns to the next
  uint32_t get = 0;
  // The B fragments of the columns; lanes of columns that no row of x has keep
  // zeros.  Several sets where they fit, so that a piece's loads do not wait
  // for the products of the one before.
  constexpr int kSets = NT <= 2 ? 4 : 1;
  uint4 xb[kSets][NT];
#pragma unroll
  for (int i = 0; i < kSets; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) xb[i][j] = make_uint4(0u, 0u, 0u, 0u);

  Place c;
  c.first = tile0;
  c.phase0 = 0;
  bool begun = false;
  for (; c.first < tile1; c.first += p.at_once) {
    for (c.phase0 = 0; c.phase0 < p.steps || c.phase0 == 0; c.phase0 += p.phase) {
      enter(c);
      if (!begun || p.phase < p.steps) {
        if (begun) __syncthreads();
        stage_x<XT>(a, p, xs, c.phase0, c.steps);
      }
      __syncthreads();
      begun = true;
      const bool final_phase = c.phase0 + p.phase >= p.steps;
      // Sum y of a tile's row over the phase: into the output, or kept.
      auto put_sum = [&](int tile, int row, int m, float y) {
        float* const keep = acc_keep + ((tile - c.first) * 16 + row) * p.rows + m;
        if (c.phase0 > 0) y = __fadd_rn(*keep, y);
        if (!final_phase) {
          *keep = y;
          return;
        }
        const long n = static_cast<long>(tile) * 16 + row;
        if (n >= a.N) return;
        if (a.bias != nullptr) y = __fadd_rn(y, __ldg(a.bias + n));
        static_cast<XT*>(a.out)[static_cast<long>(p.m0 + m) * a.ldo + n] = from_f32<XT>(y);
      };

      while (c.at < c.end) {
        const int n = min(c.steps - c.step, c.end - c.at), from = c.step;
        float sum[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[j][e] = 0.0f;
        uint32_t xc = x_lane + static_cast<uint32_t>(c.step) * 8 * x_col;
        for (int i0 = 0; i0 < n; ++i0) {
          cp_wait<kStages - 2>();
          __syncwarp();
          issue();
          const uint32_t slot = ring + get;
          get = get + R::kSlot == kStages * R::kSlot ? 0 : get + R::kSlot;
          float acc[NT][4];
          uint32_t off[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t w[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if constexpr (A) {
                const int r = lane & 7, piece = 4 * half + (lane >> 3);
                ldmatrix4(w[h], slot + (8 * h + r) * 128 + ((piece ^ r) << 4));
              } else {
                const uint32_t sh = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a.W) + (g + 8 * h) * a.ldw) & 15u;
                const uint32_t row = slot + (8 * h + g) * R::kPitch + half * 64 + (sh & ~3u) + 4 * t;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  // The second word of the last piece may lie behind the row's
                  // blocks; it is only shifted in when sh % 4 is not 0, and
                  // then it does not.
                  const uint32_t lo = lds4(row + 16 * i), hi = (sh & 3u) ? lds4(row + 16 * i + 4) : 0u;
                  w[h][i] = __funnelshift_r(lo, hi, 8 * (sh & 3u));
                }
              }
            }
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) {
              const int i = 4 * half + i2;  // the piece; 32 columns
              const int grp = i * 32 / G;
              const bool first = i * 32 % G == 0, last = (i + 1) * 32 % G == 0;
              if (first) {
#pragma unroll
                for (int h = 0; h < 2; ++h) off[h] = M::offset(of_group(now.z[h][grp / 4], grp));
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                  for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
              }
              uint32_t q[2][4];
#pragma unroll
              for (int h = 0; h < 2; ++h) M::weights(w[h][i2], off[h], q[h]);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                if (j == 0 || 8 * j < p.cols) {
                  uint4& b = xb[i % kSets][j];
                  lds16_if(b, xc + i * x_col + j * 512, 8 * j + g < p.cols);
                  M::mma(acc[j], q[0][0], q[1][0], q[0][1], q[1][1], b.x, b.y);
                  M::mma(acc[j], q[0][2], q[1][2], q[0][3], q[1][3], b.z, b.w);
                }
              }
              if (last) {
                const float s0 = scale_of(of_group(now.s[0][grp / 4], grp));
                const float s1 = scale_of(of_group(now.s[1][grp / 4], grp));
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                  for (int e = 0; e < 4; ++e) sum[j][e] = __fmaf_rn(acc[j][e], e < 2 ? s0 : s1, sum[j][e]);
              }
            }
          }
          xc += 8 * x_col;
          now = next;
          load_scales(next);
        }

        // The segment's sums, [row][column], as a partial: the first place for
        // a tile that began before this warp's share, the second for one that
        // ends behind it, and in passing for a whole one.
        float* const to = part + (warp * 2 + (from > 0 ? 0 : 1)) * 16 * 8 * NT;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float* at = to + g * 8 * NT + 8 * j + 2 * t;
          *reinterpret_cast<float2*>(at) = make_float2(sum[j][0], sum[j][1]);
          *reinterpret_cast<float2*>(at + 8 * 8 * NT) = make_float2(sum[j][2], sum[j][3]);
        }
        if (n == c.steps) {
          __syncwarp();
          for (int i = lane; i < 16 * p.rows; i += 32) {
            const int row = i & 15, m = i >> 4;
            float y = 0.0f;
#pragma unroll
            for (int sp = 0; sp < kSplit<XT>; ++sp) y = __fadd_rn(y, to[row * 8 * NT + m * kSplit<XT> + sp]);
            put_sum(c.tile, row, m, y);
          }
          __syncwarp();
        }
        c.at += n;
        c.step = 0;
        ++c.tile;
      }
      __syncthreads();
      // Joins the tiles that the warps' shares cut: warp w the one that the end
      // of its share is the first to cut.
      const int all = min(p.at_once, tile1 - c.first) * c.steps;
      const int begin = warp * all / kWarps, cut = (warp + 1) * all / kWarps;
      const int tile = c.steps > 0 ? cut / c.steps : 0, start = tile * c.steps;
      if (warp + 1 < kWarps && start < cut && start >= begin) {
        int last = warp + 1;
        while (last + 1 < kWarps && (last + 1) * all / kWarps < start + c.steps) ++last;
        for (int i = lane; i < 16 * p.rows; i += 32) {
          const int row = i & 15, m = i >> 4;
          float y = 0.0f;
          for (int w = warp; w <= last; ++w) {
            if (w > warp && w * all / kWarps == (w + 1) * all / kWarps) continue;  // an empty share
            const float* from = part + (w * 2 + (w == warp ? 1 : 0)) * 16 * 8 * NT + row * 8 * NT + m * kSplit<XT>;
#pragma unroll
            for (int sp = 0; sp < kSplit<XT>; ++sp) y = __fadd_rn(y, from[sp]);
          }
          put_sum(c.first + tile, row, m, y);
        }
      }
      if (p.steps == 0) {  // K = 0: the bias alone
        for (int i = threadIdx.x; i < (min(p.at_once, tile1 - c.first)) * 16 * p.rows; i += kThreads)
          put_sum(c.first + i / (16 * p.rows), i % 16, i / 16 % p.rows, 0.0f);
      }
    }
    if (c.first + p.at_once < tile1) __syncthreads();  // the partials are free again
  }
}

template <typename XT, int G, int NT, bool A>
cudaError_t launch(const LinearW4Args& a, const Plan& p, int smem, int ctas_per_sm, cudaStream_t s) {
  const int most = a.num_sms * ctas_per_sm;
  auto kernel = linear_w4_kernel<XT, G, NT, A>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(p.tiles < most ? p.tiles : most), dim3(kThreads), smem, s, a, p);
}

// One pass over the weights for rows [m0, m0 + rows) of x.
template <typename XT, int G, int NT, bool A>
cudaError_t pass(const LinearW4Args& a, int m0, int rows, cudaStream_t s) {
  Plan p = {};
  p.m0 = m0;
  p.rows = rows;
  p.cols = rows * kSplit<XT>;
  p.tiles = static_cast<int>((static_cast<long>(a.N) + 15) / 16);
  p.steps = static_cast<int>((static_cast<long>(a.K) + kStep - 1) / kStep);
  p.x_on_16 = ((reinterpret_cast<uintptr_t>(a.x) | static_cast<uintptr_t>(a.ldx * static_cast<long>(sizeof(XT)))) & 15) == 0;
  const long per_step = static_cast<long>(p.cols) * kStep * 2;  // bytes of x in shared memory
  const int rest = Ring<A>::kAll + partial_bytes(NT);
  const long all = p.steps * per_step;
  if (all + rest <= kMaxSmem) {
    p.phase = p.steps > 0 ? p.steps : 1;
    p.at_once = p.tiles;
    p.x_bytes = static_cast<int>(all);
    const int smem = p.x_bytes + rest;
    return launch<XT, G, NT, A>(a, p, smem, NT <= 4 && 2 * (smem + 1024) <= 227 * 1024 ? 2 : 1, s);
  }
  p.phase = static_cast<int>((kMaxSmem - rest - kMaxAcc) / per_step);
  p.at_once = kMaxAcc / (64 * rows);
  p.x_bytes = static_cast<int>(p.phase * per_step);
  return launch<XT, G, NT, A>(a, p, p.x_bytes + rest + kMaxAcc, 1, s);
}

template <typename XT, int G, bool A>
cudaError_t all_rows(const LinearW4Args& a, cudaStream_t s) {
  constexpr int most = 64 / kSplit<XT>;  // rows that fill the 8 column tiles of a pass
  // Equal passes: M = 65 runs as 33 + 32 rather than 64 + 1.
  const int passes = (a.M + most - 1) / most, each = (a.M + passes - 1) / passes;
  for (int m0 = 0; m0 < a.M; m0 += each) {
    const int rows = a.M - m0 < each ? a.M - m0 : each, cols = rows * kSplit<XT>;
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

// The kernels of one activation type (one translation unit each).
template <typename XT>
cudaError_t linear(const LinearW4Args& a, cudaStream_t s) {
  const bool on_16 = ((reinterpret_cast<uintptr_t>(a.W) | static_cast<uintptr_t>(a.ldw)) & 15) == 0;
  return on_16 ? by_group<XT, true>(a, s) : by_group<XT, false>(a, s);
}

}  // namespace w4
}  // namespace esmb200
