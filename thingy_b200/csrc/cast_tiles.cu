// Casts of a bf16 matrix to e4m3 in both orientations, one read of the matrix:
//
//   s = max(RN(amax / 448), 1e-4)  [2^ceil(log2 s) on request],  q = e4m3(RN(x / s))
//
// with amax over 128 x 128 blocks (weights: x's codes and its transpose's share
// the scale) or over 1 x 128 groups of the rows and, for the transposed codes,
// 128 x 1 groups of the columns (activations and gradients: the products of a
// training step contract over either axis). Gradients (tile_scale): a group
// with amax < 1e-4 has s = max(RN(amax / 448), 2^-92).
//
// One CTA casts one 128 x 128 tile, 256 threads, four CTAs an SM: thread (rg, v)
// holds rows 8 rg .. 8 rg + 7, columns 8 v .. 8 v + 7, eight 16-byte loads, a
// warp two whole 256-byte row pieces a load. The tile stays in registers. The
// codes of the transpose go through a 16 KB shared tile, its 8-byte pieces
// permuted by the column's piece number (a warp's stores then cover every bank
// once instead of one), so that they too leave as whole 128-byte row pieces.
//
// Bound: memory, 2 bytes read and 2 written an element (1 without the
// transpose); next to it the instruction issue, so the block kind converts an
// element once and transposes the bytes, and the two-way kind makes a row's
// scale in two of the 16 lanes that share it. (A persistent form that read the
// tiles by TMA two ahead, two CTAs an SM, was slower: 113 against 105 us at
// 16384 x 7168.)
#include "cutie.h"
#include "launch.cuh"

namespace cutie {
namespace {

constexpr int kTile = 128, kThreads = 256;

// The scale of a group's maximum. An infinite maximum stays infinite (the
// division's remainder would turn it into a NaN, and that into the floor).
// The activation quantizer's floor of 1e-4 loses a group whose maximum is far
// below it: every |x| < 9.8e-8 has the code zero, and gradients are often that
// small. While amax >= 1e-4 the floor costs an element at most 2^-10 of amax
// (half the least code's step), 2^-10 sqrt(128 / 3) = 0.6% of the group's norm
// in the mean square; below, a gradient's group goes without it.
__device__ __forceinline__ float tile_scale(float amax, const CastArgs& a) {
  const float least = a.gradient && amax < kMinScale ? kMinGradientScale : kMinScale;
  return amax <= 3.4e38f ? make_scale(amax, a.pow2, least) : amax;
}
// RN(1 / s): the negated exponent for a power of two, else rcp_scale; NaN for
// an infinite scale, so that every code of its group is NaN.
__device__ __forceinline__ float rcp_of(float s, bool pow2) {
  const float r = pow2 ? __uint_as_float(0x7f000000u - __float_as_uint(s)) : rcp_scale(s);
  return s <= 3.4e38f ? r : __uint_as_float(0x7fffffffu);
}

// Codes of 8 bf16 values (four pairs) over one scale; rc = RN(1 / s).
__device__ __forceinline__ uint2 codes_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d, float s,
                                          float rc) {
  const float2 ns = make_float2(-s, -s), r2 = make_float2(rc, rc);
  return make_uint2(f4_to_e4m3x4(div2_rn(bf2_to_f2(a), ns, r2), div2_rn(bf2_to_f2(b), ns, r2)),
                    f4_to_e4m3x4(div2_rn(bf2_to_f2(c), ns, r2), div2_rn(bf2_to_f2(d), ns, r2)));
}

// Four rows of four bytes -> four columns.
__device__ __forceinline__ void transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d,
                                           uint32_t (&t)[4]) {
  const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362);
  const uint32_t cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
  t[0] = __byte_perm(ab0, cd0, 0x5410), t[1] = __byte_perm(ab0, cd0, 0x7632);
  t[2] = __byte_perm(ab1, cd1, 0x5410), t[3] = __byte_perm(ab1, cd1, 0x7632);
}

__device__ __forceinline__ uint32_t pair_to_bf2(uint32_t a, uint32_t b) {
  return f2_to_bf2(make_float2(__uint_as_float(a), __uint_as_float(b)));
}

// SORTED: rows sorted by expert (two-way kind). Padding rows are zeros whatever
// x holds there, so that they change no column group. Tiles that are all padding
// are written too: where experts begin at multiples of 256 or more they lie within
// one, and the weight gradient goes over all of its columns.
template <bool BLOCK, bool TRANSPOSED, bool SORTED = false, bool F32 = false>
__global__ void __launch_bounds__(kThreads, 4)
    cast_tiles_kernel(CastArgs a) {
  __shared__ __align__(16) uint8_t t_codes[TRANSPOSED ? kTile * kTile : 16];
  __shared__ __align__(16) uint32_t part[8][64];  // a warp's column maxima (bf16 pairs)
  __shared__ float2 col_scale[8][16];             // (scale, reciprocal) of column 8 v + j at [j][v]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rg = tid >> 4, v = tid & 15;
  const int tiles_c = (a.H + kTile - 1) / kTile;
  const int64_t tr = blockIdx.x / tiles_c;  // tile row
  const int tc = blockIdx.x % tiles_c;      // tile column
  const int64_t r0 = tr * kTile + rg * 8;
  const int c0 = tc * kTile + v * 8;
  const bool col_ok = c0 < a.H;  // H is a multiple of 8: a vector is whole or absent
  griddep_wait();
  griddep_launch_dependents();

  // SORTED: the sources of the warp's 16 rows; read beside the rows, not before them
  // (M is a multiple of 128)
  const int source = SORTED && lane < 16 ? a.sources[tr * kTile + 16 * warp + lane] : 0;
  uint32_t x[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint4 w = make_uint4(0, 0, 0, 0);
    if (col_ok && r0 + i < a.M) {
      if (F32) {
        const float* f = static_cast<const float*>(a.x) + (r0 + i) * a.ldx + c0;
        const uint4 lo = ld_stream(f), hi = ld_stream(f + 4);
        w = make_uint4(pair_to_bf2(lo.x, lo.y), pair_to_bf2(lo.z, lo.w), pair_to_bf2(hi.x, hi.y),
                       pair_to_bf2(hi.z, hi.w));
      } else {
        w = ld_stream(static_cast<const uint16_t*>(a.x) + (r0 + i) * a.ldx + c0);
      }
    }
    x[i][0] = w.x, x[i][1] = w.y, x[i][2] = w.z, x[i][3] = w.w;
  }
  if (SORTED) {
    const uint32_t none = __ballot_sync(0xffffffffu, source < 0);
    const uint32_t mine = none >> (rg & 1) * 8 & 0xffu;
    if (mine != 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (mine >> i & 1u) x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0u;
    }
  }
  const uint32_t all = 0xffffffffu;
  uint2 codes[BLOCK ? 8 : 1];  // block kind: the rows' codes, which its transpose shares
  if (BLOCK) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      m = absmax_bf2(m, absmax_bf2(absmax_bf2(x[i][0], x[i][1]), absmax_bf2(x[i][2], x[i][3])));
    m &= 0x7fff7fffu;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_bf2(m, __shfl_xor_sync(all, m, o));
    if (lane == 0) part[warp][0] = m;
    __syncthreads();
    m = part[0][0];
#pragma unroll
    for (int w = 1; w < 8; ++w) m = max_bf2(m, part[w][0]);
    const float2 f = bf2_to_f2(m);
    const float s = tile_scale(fmaxf(f.x, f.y), a);
    if (tid == 0) {
      a.s[tr * a.lds + tc] = s;
      if (TRANSPOSED) a.st[(int64_t)tc * a.ldst + tr] = s;
    }
    const float rc = rcp_of(s, a.pow2);
#pragma unroll
    for (int i = 0; i < 8; ++i) codes[i] = codes_of(x[i][0], x[i][1], x[i][2], x[i][3], s, rc);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col_ok && r0 + i < a.M) st_stream2(a.q + (r0 + i) * a.ldq + c0, codes[i].x, codes[i].y);
  } else {
    // column maxima over the thread's 8 rows, the warp's two row groups, the warps
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t m = x[0][j];
#pragma unroll
      for (int i = 1; i < 8; ++i) m = absmax_bf2(m, x[i][j]);
      m &= 0x7fff7fffu;
      m = max_bf2(m, __shfl_xor_sync(all, m, 16));
      if (lane < 16) part[warp][v * 4 + j] = m;
    }
    // row maxima over the 16 lanes of a row group, folded so that lanes 2 i and
    // 2 i + 1 end with row i's: each lane then makes one scale, not eight
    uint32_t m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      m[i] = absmax_bf2(absmax_bf2(x[i][0], x[i][1]), absmax_bf2(x[i][2], x[i][3])) & 0x7fff7fffu;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      const bool up = (v & (2 * o)) != 0;
#pragma unroll
      for (int i = 0; i < o; ++i) {
        const uint32_t keep = up ? m[i + o] : m[i], send = up ? m[i] : m[i + o];
        m[i] = max_bf2(keep, __shfl_xor_sync(all, send, 2 * o));
      }
    }
    const float2 f = bf2_to_f2(max_bf2(m[0], __shfl_xor_sync(all, m[0], 1)));
    const float my_s = tile_scale(fmaxf(f.x, f.y), a), my_rc = rcp_of(my_s, a.pow2);
    if ((v & 1) == 0 && r0 + (v >> 1) < a.M) a.s[(int64_t)tc * a.lds + r0 + (v >> 1)] = my_s;
    __syncthreads();
    if (tid < 64) {  // columns 2 tid and 2 tid + 1, kept so that a warp's 16 reads below are in a row
      uint32_t c = part[0][tid];
#pragma unroll
      for (int w = 1; w < 8; ++w) c = max_bf2(c, part[w][tid]);
      const float2 g = bf2_to_f2(c);
      const float s0 = tile_scale(g.x, a), s1 = tile_scale(g.y, a);
      col_scale[2 * (tid & 3)][tid >> 2] = make_float2(s0, rcp_of(s0, a.pow2));
      col_scale[2 * (tid & 3) + 1][tid >> 2] = make_float2(s1, rcp_of(s1, a.pow2));
      const int at = tc * kTile + 2 * tid;
      if (at < a.H) {  // H is even
        a.st[tr * a.ldst + at] = s0;
        a.st[tr * a.ldst + at + 1] = s1;
      }
    }
    // codes along the rows: 8 a thread, 128 contiguous bytes a row of the tile
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = __shfl_sync(all, my_s, 2 * i, 16), rc = __shfl_sync(all, my_rc, 2 * i, 16);
      const uint2 w = codes_of(x[i][0], x[i][1], x[i][2], x[i][3], s, rc);
      if (col_ok && r0 + i < a.M) st_stream2(a.q + (r0 + i) * a.ldq + c0, w.x, w.y);
    }
  }
  if (!TRANSPOSED) return;
  // codes along the columns: a column's 8 rows of this thread are 8 bytes, piece
  // rg of its column, permuted by c / 8 = v
  if (BLOCK) {
    // the 8 x 8 bytes transposed in registers: 4 x 4 blocks
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t top[4], low[4];
      transpose4(q ? codes[0].y : codes[0].x, q ? codes[1].y : codes[1].x, q ? codes[2].y : codes[2].x,
                 q ? codes[3].y : codes[3].x, top);
      transpose4(q ? codes[4].y : codes[4].x, q ? codes[5].y : codes[5].x, q ? codes[6].y : codes[6].x,
                 q ? codes[7].y : codes[7].x, low);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint2*>(t_codes + (v * 8 + 4 * q + c) * kTile + ((rg ^ v) << 3)) =
            make_uint2(top[c], low[c]);
    }
  } else {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 sc = col_scale[2 * j + h][v];
        // rows 2 i and 2 i + 1 of the column as a pair
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __byte_perm(x[2 * i][j], x[2 * i + 1][j], h ? 0x7632 : 0x5410);
        *reinterpret_cast<uint2*>(t_codes + (v * 8 + 2 * j + h) * kTile + ((rg ^ v) << 3)) =
            codes_of(w[0], w[1], w[2], w[3], sc.x, sc.y);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = i * 16 + rg;  // the tile's column, 16 lanes a column
    const int col = tc * kTile + c;
    const int64_t row = tr * kTile + v * 8;
    const uint2 w = *reinterpret_cast<const uint2*>(t_codes + c * kTile + ((v ^ (c >> 3)) << 3));
    if (col >= a.H) continue;
    uint8_t* p = a.qt + (int64_t)col * a.ldqt + row;
    if (row + 8 <= a.M) {
      st_stream2(p, w.x, w.y);
    } else {
      for (int b = 0; b < 8 && row + b < a.M; ++b)
        p[b] = (uint8_t)((b < 4 ? w.x >> (8 * b) : w.y >> (8 * (b - 4))) & 0xffu);
    }
  }
}

}  // namespace

cudaError_t launch_cast_tiles(const CastArgs& a, bool block, cudaStream_t stream) {
  const int64_t tiles = ((a.M + kTile - 1) / kTile) * ((a.H + kTile - 1) / kTile);
  auto kernel = block && a.x_f32 ? (a.qt != nullptr ? cast_tiles_kernel<true, true, false, true>
                                                    : cast_tiles_kernel<true, false, false, true>)
                : block ? (a.qt != nullptr ? cast_tiles_kernel<true, true> : cast_tiles_kernel<true, false>)
                      : a.sources != nullptr ? cast_tiles_kernel<false, true, true>
                                             : cast_tiles_kernel<false, true>;
  return launch_pdl(kernel, (unsigned)tiles, kThreads, 0, stream, a);
}

}  // namespace cutie
