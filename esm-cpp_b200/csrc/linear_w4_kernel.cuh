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
// Layout: the order of a sum over k is free.  A warp takes chunks of 16 rows x
// 128 columns (64 bytes a row), copied by cp.async into its own ring of
// kStages slots; ldmatrix hands lane (g, t) word t of each 16-byte piece of
// row g, eight consecutive columns whose nibbles pair up as (0,4) (1,5) (2,6)
// (3,7).  x is laid out in shared memory in that order when it is staged, once
// per block.  A piece of 16 bytes is 32 columns, so groups of 32, 64 and 128
// end after 1, 2 or 4 pieces.
//
// The 8 warps of a block split K by chunks and meet in shared memory once per
// 16 rows; a block takes an equal, consecutive share of all rows and its rings
// run on across row tiles.  Where x does not fit beside the rings it is staged
// in phases, and a block takes 32 rows at a time to share the staging.
#pragma once

#include "common.cuh"
#include "dtype.cuh"
#include "kernels.cuh"

namespace esmb200 {
namespace w4 {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxSmem = 224 * 1024;

// RT: 16-row tiles a block takes at a time (2 where x comes in phases).  A:
// rows on 16-byte boundaries.
template <int RT, bool A>
struct Ring {
  static constexpr int kRow = A ? 64 : 80;  // unaligned rows: five 16-byte blocks that cover the 64 bytes
  static constexpr int kTile = 16 * kRow;
  static constexpr int kSlot = RT * kTile;
  static constexpr int kStages = RT == 1 ? 8 : A ? 4 : 3;
  static constexpr int kBytes = kWarps * kStages * kSlot;
};

struct Plan {
  int tiles;       // row blocks of 16 RT rows, shared out evenly
  int chunks;      // of 128 columns
  int phase;       // chunks staged at a time, a multiple of kWarps
  int cols;        // columns in use: rows of x, times 3 for float32
  int x_bytes;     // of shared memory for x
  int m0, rows;    // the rows of x of this launch
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
      const uint32_t b = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;  // 128 + q
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
  static __device__ __forceinline__ uint32_t offset(int z) { return 0xE400E400u | (static_cast<uint32_t>(z) * 0x10001u); }
  static __device__ __forceinline__ void weights(uint32_t w, uint32_t off, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = ((w >> (4 * i)) & 0x000F000Fu) | 0x64006400u;  // 1024 + q
      asm("add.rn.f16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(b), "r"(off));
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

// Stages chunks [c0, c0 + n) of x: eight columns k8 of row m at
// xs[((k8 / 4) * cols + column) * 4 + k8 % 4] (16-byte units), k8 counted from
// chunk c0.
template <typename XT>
__device__ __forceinline__ void stage_x(const LinearW4Args& a, const Plan& p, uint4* xs, int c0, int n) {
  const int n8 = n * 16;
  for (int i = threadIdx.x; i < p.rows * n8; i += kThreads) {
    const int m = i / n8, k8 = i - m * n8;
    const int k = c0 * 128 + k8 * 8;
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

static_assert(kWarps * 64 * 256 + Ring<2, false>::kBytes + kWarps * 16 * 64 * 4 <= kMaxSmem &&
                  kWarps * 64 * 256 + Ring<2, true>::kBytes + kWarps * 16 * 64 * 4 <= kMaxSmem,
              "the shortest phase of 64 columns fits");

template <typename XT, int kSubs, int NT, int RT, bool A>
__global__ void __launch_bounds__(kThreads, RT == 1 && NT <= 4 ? 2 : 1) linear_w4_kernel(LinearW4Args a, Plan p) {
  using R = Ring<RT, A>;
  using M = Mma<XT>;
  extern __shared__ __align__(128) unsigned char smem[];
  uint4* const xs = reinterpret_cast<uint4*>(smem);
  float* const red = reinterpret_cast<float*>(smem + p.x_bytes + R::kBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + p.x_bytes + warp * R::kStages * R::kSlot;
  const int tile0 = static_cast<int>(static_cast<long>(blockIdx.x) * p.tiles / gridDim.x);
  const int tiles = static_cast<int>((static_cast<long>(blockIdx.x) + 1) * p.tiles / gridDim.x) - tile0;
  const int own = p.chunks > warp ? (p.chunks - warp + kWarps - 1) / kWarps : 0;  // this warp's chunks of a tile
  const int row_bytes = static_cast<int>((static_cast<long>(a.K) + 1) / 2);
  pdl_wait();
  pdl_trigger();

  // Copies.  A lane copies the same places of every 16-row tile; within a tile
  // its addresses move by 64 kWarps bytes a chunk.
  constexpr int kCopies = A ? 2 : 3;
  int i_tile = -1, i_chunk = own - 1;
  uint32_t i_dst = 0;
  int i_left = 0;                   // bytes of a row from the chunk's first on
  const uint8_t* src[RT][kCopies];  // the chunk's
  int src_from[kCopies];            // first byte of the copy within the chunk's 64 bytes of the row
  bool src_on[RT][kCopies];
  uint32_t src_dst[kCopies];
  int src_row[kCopies];
#pragma unroll
  for (int h = 0; h < kCopies; ++h) {
    const int id = lane + 32 * h;
    const int row = A ? id >> 2 : id / 5, part = A ? id & 3 : id - row * 5;
    // Unaligned rows: the 16-byte blocks that hold a byte of the row's piece;
    // where a row's pieces start in a block (the same in every tile, 16 rows
    // being a multiple of 16 bytes whatever ldw is).
    const int sh = A ? 0 : static_cast<int>((reinterpret_cast<uintptr_t>(a.W) + row * a.ldw) & 15);
    src_row[h] = row < 16 ? row : -1;
    src_from[h] = part * 16 - sh;
    src_dst[h] = ring + (A ? row * 64 + ((part ^ ((row >> 1) & 3)) << 4) : row * 80 + part * 16);
  }
  // Rows behind N and blocks behind a row's end are filled with zeros; their
  // copies read nothing, from W's first block.
  const uint8_t* const nowhere = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(a.W) & ~uintptr_t(15));
  // Starts the copies of the warp's next (tile, chunk).
  auto issue = [&]() {
    if (++i_chunk == own) {
      i_chunk = 0;
      ++i_tile;
      i_left = row_bytes - warp * 64;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < kCopies; ++h) {
          const long n = (static_cast<long>(tile0 + i_tile) * RT + rt) * 16 + src_row[h];
          src_on[rt][h] = src_row[h] >= 0 && i_tile < tiles && n < a.N;
          src[rt][h] = src_on[rt][h] ? a.W + n * a.ldw + warp * 64 + src_from[h] : nowhere;
        }
    }
    if (i_tile < tiles && own > 0) {
      if (A && i_left >= 64) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int h = 0; h < kCopies; ++h)
            cp_async16(src_dst[h] + i_dst + rt * R::kTile, src[rt][h], src_on[rt][h] ? 16 : 0);
      } else {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int h = 0; h < kCopies; ++h) {
            const int left = i_left - src_from[h];
            int bytes = A ? min(max(left, 0), 16) : src_from[h] < min(i_left, 64) ? 16 : 0;
            if (!src_on[rt][h]) bytes = 0;
            if (A || src_row[h] >= 0)
              cp_async16(src_dst[h] + i_dst + rt * R::kTile, bytes > 0 ? src[rt][h] : nowhere, bytes);
          }
      }
      i_left -= 64 * kWarps;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < kCopies; ++h)
          if (src_on[rt][h]) src[rt][h] += 64 * kWarps;
    }
    i_dst = i_dst + R::kSlot == R::kStages * R::kSlot ? 0 : i_dst + R::kSlot;
    cp_commit();
  };
  // Scales and zero points of rows g and g + 8 of a (tile, chunk): lane t
  // holds those of group t % kSubs of the chunk.  They are loaded two steps
  // ahead and kept as they are until used: a conversion here would make the
  // warp wait for the load.
  struct Scales {
    uint32_t s[RT][2];
    int z[RT][2];
  };
  const int groups = static_cast<int>((static_cast<long>(a.K) + a.group - 1) / a.group);
  const bool f32_scales = a.scale_type == kF32;
  int s_tile = -1, s_chunk = own - 1, s_grp = 0;
  const char* s_at[RT][2];
  const uint8_t* z_at[RT][2];
  bool s_on[RT][2];
  auto load_scales = [&](Scales& v) {
    if (++s_chunk == own) {
      s_chunk = 0;
      ++s_tile;
      s_grp = warp * kSubs + (t & (kSubs - 1));
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const long n = (static_cast<long>(tile0 + s_tile) * RT + rt) * 16 + g + 8 * h;
          s_on[rt][h] = s_tile < tiles && own > 0 && n < a.N;
          s_at[rt][h] = static_cast<const char*>(a.scales) + (n * a.lds + s_grp) * (f32_scales ? 4 : 2);
          z_at[rt][h] = a.zeros + n * a.ldz + s_grp;
        }
    }
    const bool in = s_grp < groups;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v.s[rt][h] = 0u;
        v.z[rt][h] = 8;
        if (in && s_on[rt][h]) {
          v.s[rt][h] = f32_scales ? __ldg(reinterpret_cast<const uint32_t*>(s_at[rt][h]))
                                  : __ldg(reinterpret_cast<const uint16_t*>(s_at[rt][h]));
          if (a.zeros != nullptr) v.z[rt][h] = __ldg(z_at[rt][h]);
        }
        s_at[rt][h] += kWarps * kSubs * (f32_scales ? 4 : 2);
        z_at[rt][h] += kWarps * kSubs;
      }
    s_grp += kWarps * kSubs;
  };
  auto scale_of = [&](uint32_t bits) {
    const float v = f32_scales               ? __uint_as_float(bits)
                    : a.scale_type == kF16 ? __half2float(__ushort_as_half(static_cast<uint16_t>(bits)))
                                           : __uint_as_float(bits << 16);
    return __fmul_rn(v, M::kScale);
  };
  // Lane t's value of group grp of its row.
  auto of_group = [&](auto v, int grp) { return kSubs == 1 ? v : __shfl_sync(0xffffffffu, v, (lane & ~3) | grp); };

#pragma unroll
  for (int i = 0; i < R::kStages - 1; ++i) issue();
  Scales now, next;
  load_scales(now);
  load_scales(next);

  const uint32_t x_lane = smem_u32(smem) + (g * 4 + t) * 16;
  const uint32_t x_col = static_cast<uint32_t>(p.cols) * 64;  // bytes from one 16-byte piece's columns to the next
  uint32_t get = ring;
  for (int tile = 0; tile < tiles; ++tile) {
    float sum[RT][NT][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[rt][j][e] = 0.0f;
    for (int c0 = 0; c0 < p.chunks; c0 += p.phase) {
      if (tile == 0 || p.phase < p.chunks) {
        if (tile > 0 || c0 > 0) __syncthreads();
        stage_x<XT>(a, p, xs, c0, min(p.phase, p.chunks - c0));
        __syncthreads();
      }
      const int c_end = min(p.chunks, c0 + p.phase) - c0;
      uint32_t xc = x_lane + static_cast<uint32_t>(warp) * 4 * x_col;
      for (int c = warp; c < c_end; c += kWarps) {
        cp_wait<R::kStages - 2>();
        __syncwarp();
        issue();
        uint32_t w[RT][2][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if constexpr (A) {
              const int r = lane & 7, pc = lane >> 3;
              ldmatrix4(w[rt][h], get + rt * R::kTile + (8 * h + r) * 64 + ((pc ^ ((r >> 1) & 3)) << 4));
            } else {
              const uint32_t sh = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(a.W) + (g + 8 * h) * a.ldw) & 15u;
              const uint32_t row = get + rt * R::kTile + (8 * h + g) * 80 + (sh & ~3u) + 4 * t;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                // The second word of the last piece may lie behind the row's
                // five blocks; it is only shifted in when sh % 4 is not 0, and
                // then it does not.
                const uint32_t lo = lds4(row + 16 * i), hi = (sh & 3u) ? lds4(row + 16 * i + 4) : 0u;
                w[rt][h][i] = __funnelshift_r(lo, hi, 8 * (sh & 3u));
              }
            }
          }
        get = get + R::kSlot == ring + R::kStages * R::kSlot ? ring : get + R::kSlot;
        float acc[RT][NT][4];
        uint32_t off[RT][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // Group of piece i within the chunk, and whether it starts or ends
          // with this piece.
          const int grp = (i * kSubs) >> 2;
          const bool first = i == 0 || ((i - 1) * kSubs) >> 2 != grp;
          const bool last = i == 3 || ((i + 1) * kSubs) >> 2 != grp;
          if (first) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int h = 0; h < 2; ++h) off[rt][h] = M::offset(of_group(now.z[rt][h], grp));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[rt][j][e] = 0.0f;
          }
          uint32_t q[RT][2][4];
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int h = 0; h < 2; ++h) M::weights(w[rt][h][i], off[rt][h], q[rt][h]);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if (j == 0 || 8 * j < p.cols) {
              uint4 b = make_uint4(0u, 0u, 0u, 0u);
              if (8 * j + g < p.cols) b = lds16(xc + i * x_col + j * 512);
#pragma unroll
              for (int rt = 0; rt < RT; ++rt) {
                M::mma(acc[rt][j], q[rt][0][0], q[rt][1][0], q[rt][0][1], q[rt][1][1], b.x, b.y);
                M::mma(acc[rt][j], q[rt][0][2], q[rt][1][2], q[rt][0][3], q[rt][1][3], b.z, b.w);
              }
            }
          }
          if (last) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              const float s0 = scale_of(of_group(now.s[rt][0], grp)), s1 = scale_of(of_group(now.s[rt][1], grp));
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  sum[rt][j][e] = __fmaf_rn(acc[rt][j][e], e < 2 ? s0 : s1, sum[rt][j][e]);
            }
          }
        }
        xc += kWarps * 4 * x_col;
        now = next;
        load_scales(next);
      }
    }

    // The warps' sums meet: red[warp][row][column].
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const long n0 = (static_cast<long>(tile0 + tile) * RT + rt) * 16;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float* to = red + (warp * 16 + g) * (8 * NT) + 8 * j + 2 * t;
        *reinterpret_cast<float2*>(to) = make_float2(sum[rt][j][0], sum[rt][j][1]);
        *reinterpret_cast<float2*>(to + 8 * 8 * NT) = make_float2(sum[rt][j][2], sum[rt][j][3]);
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 16 * p.rows; i += kThreads) {
        const int row = i & 15, m = i >> 4;
        if (n0 + row >= a.N) continue;
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
#pragma unroll
          for (int sp = 0; sp < kSplit<XT>; ++sp)
            y = __fadd_rn(y, red[(w * 16 + row) * (8 * NT) + m * kSplit<XT> + sp]);
        if (a.bias != nullptr) y = __fadd_rn(y, __ldg(a.bias + n0 + row));
        static_cast<XT*>(a.out)[static_cast<long>(p.m0 + m) * a.ldo + n0 + row] = from_f32<XT>(y);
      }
    }
  }
}

template <typename XT, int kSubs, int NT, int RT, bool A>
cudaError_t launch(const LinearW4Args& a, Plan p, int ctas_per_sm, cudaStream_t s) {
  using R = Ring<RT, A>;
  p.tiles = (a.N + 16 * RT - 1) / (16 * RT);
  const int most = a.num_sms * ctas_per_sm;
  const int smem = p.x_bytes + R::kBytes + kWarps * 16 * 8 * NT * 4;
  auto kernel = linear_w4_kernel<XT, kSubs, NT, RT, A>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(p.tiles < most ? p.tiles : most), dim3(kThreads), smem, s, a, p);
}

// One pass over the weights for rows [m0, m0 + rows) of x.
template <typename XT, int kSubs, int NT, bool A>
cudaError_t pass(const LinearW4Args& a, int m0, int rows, cudaStream_t s) {
  Plan p = {};
  p.m0 = m0;
  p.rows = rows;
  p.cols = rows * kSplit<XT>;
  p.chunks = static_cast<int>((static_cast<long>(a.K) + 127) / 128);
  p.x_on_16 = ((reinterpret_cast<uintptr_t>(a.x) | static_cast<uintptr_t>(a.ldx * static_cast<long>(sizeof(XT)))) & 15) == 0;
  const long per_chunk = static_cast<long>(p.cols) * 256;  // bytes of x in shared memory
  const int red = kWarps * 16 * 8 * NT * 4;
  const long all = p.chunks * per_chunk;
  const int ring1 = Ring<1, A>::kBytes, ring2 = Ring<2, A>::kBytes;
  // x whole beside the rings of one-tile blocks, two blocks per SM if they fit;
  // else phases of it and two tiles at a time.
  if (all + ring1 + red <= kMaxSmem) {
    p.phase = (p.chunks + kWarps - 1) / kWarps * kWarps;
    if (p.phase == 0) p.phase = kWarps;
    p.x_bytes = static_cast<int>(all);
    const bool two = NT <= 4 && 2 * (all + ring1 + red + 1024) <= 227 * 1024;
    return launch<XT, kSubs, NT, 1, A>(a, p, two ? 2 : 1, s);
  }
  const long room = (kMaxSmem - ring2 - red) / (per_chunk * kWarps);
  p.phase = static_cast<int>(room < 1 ? 1 : room) * kWarps;
  p.x_bytes = static_cast<int>(p.phase * per_chunk);
  return launch<XT, kSubs, NT, 2, A>(a, p, 1, s);
}

template <typename XT, int kSubs, bool A>
cudaError_t all_rows(const LinearW4Args& a, cudaStream_t s) {
  constexpr int most = 64 / kSplit<XT>;  // rows that fill the 8 column tiles of a pass
  // Equal passes: M = 65 runs as 33 + 32 rather than 64 + 1.
  const int passes = (a.M + most - 1) / most, each = (a.M + passes - 1) / passes;
  for (int m0 = 0; m0 < a.M; m0 += each) {
    const int rows = a.M - m0 < each ? a.M - m0 : each, cols = rows * kSplit<XT>;
    const cudaError_t e = cols <= 8    ? pass<XT, kSubs, 1, A>(a, m0, rows, s)
                          : cols <= 16 ? pass<XT, kSubs, 2, A>(a, m0, rows, s)
                          : cols <= 32 ? pass<XT, kSubs, 4, A>(a, m0, rows, s)
                                       : pass<XT, kSubs, 8, A>(a, m0, rows, s);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename XT, bool A>
cudaError_t by_group(const LinearW4Args& a, cudaStream_t s) {
  if (a.group == 128) return all_rows<XT, 1, A>(a, s);
  if (a.group == 64) return all_rows<XT, 2, A>(a, s);
  return all_rows<XT, 4, A>(a, s);
}

// The kernels of one activation type (one translation unit each).
template <typename XT>
cudaError_t linear(const LinearW4Args& a, cudaStream_t s) {
  const bool on_16 = ((reinterpret_cast<uintptr_t>(a.W) | static_cast<uintptr_t>(a.ldw)) & 15) == 0;
  return on_16 ? by_group<XT, true>(a, s) : by_group<XT, false>(a, s);
}

}  // namespace w4
}  // namespace esmb200
