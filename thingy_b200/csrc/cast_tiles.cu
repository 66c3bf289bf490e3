// Casts of a bf16 matrix to e4m3 in both orientations, one read of the matrix:
//
//   s = max(RN(amax / 448), 1e-4)  [2^ceil(log2 s) on request],  q = e4m3(RN(x / s))
//
// with amax over 128 x 128 blocks (weights: x's codes and its transpose's share
// the scale) or over 1 x 128 groups of the rows and, for the transposed codes,
// 128 x 1 groups of the columns (activations and gradients: the products of a
// training step contract over either axis).
//
// One CTA casts one 128 x 128 tile, 256 threads: thread (rg, v) holds rows
// 8 rg .. 8 rg + 7, columns 8 v .. 8 v + 7, eight 16-byte loads, a warp two
// whole 256-byte row pieces a load. The tile stays in registers: a row's
// maximum is a butterfly over the 16 lanes that share it, a column's a step
// over the warp's two row groups and one over the 8 warps through shared
// memory. The codes of the transpose go through a 16 KB shared tile, its
// 8-byte pieces permuted by the column's piece number (a warp's stores then
// cover every bank once instead of one), so that they too leave as whole
// 128-byte row pieces.
//
// Bound: memory, 2 bytes read and 2 written an element (1 without the
// transpose).
#include "cutie.h"
#include "launch.cuh"

namespace cutie {
namespace {

constexpr int kTile = 128, kThreads = 256;

// The scale of a group's maximum. An infinite maximum stays infinite (the
// division's remainder would turn it into a NaN, and that into the floor).
__device__ __forceinline__ float tile_scale(float amax, bool pow2) {
  return amax <= 3.4e38f ? make_scale(amax, pow2) : amax;
}
// RN(1 / s): the negated exponent for a power of two, else rcp_scale; NaN for
// an infinite scale, so that every code of its group is NaN.
__device__ __forceinline__ float rcp_of(float s, bool pow2) {
  const float r = pow2 ? __uint_as_float(0x7f000000u - __float_as_uint(s)) : rcp_scale(s);
  return s <= 3.4e38f ? r : __uint_as_float(0x7fffffffu);
}

template <bool BLOCK, bool TRANSPOSED>
__global__ void __launch_bounds__(kThreads, 4)
    cast_tiles_kernel(CastArgs a) {
  __shared__ __align__(16) uint8_t t_codes[TRANSPOSED ? kTile * kTile : 16];
  __shared__ __align__(16) uint32_t part[8][64];  // a warp's column maxima (bf16 pairs)
  __shared__ float2 col_scale[kTile];             // (scale, reciprocal) of a column
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

  uint32_t x[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint4 w = make_uint4(0, 0, 0, 0);
    if (col_ok && r0 + i < a.M) w = ld_stream(a.x + (r0 + i) * a.ldx + c0);
    x[i][0] = w.x, x[i][1] = w.y, x[i][2] = w.z, x[i][3] = w.w;
  }
  // magnitudes: a row's over 8 columns, a column pair's over 8 rows
  uint32_t rmax[8], cmax[4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    rmax[i] = absmax_bf2(absmax_bf2(x[i][0], x[i][1]), absmax_bf2(x[i][2], x[i][3])) & 0x7fff7fffu;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t m = x[0][j];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = absmax_bf2(m, x[i][j]);
    cmax[j] = m & 0x7fff7fffu;
  }
  float row_s[8];
  if (BLOCK) {
    uint32_t m = max_bf2(max_bf2(cmax[0], cmax[1]), max_bf2(cmax[2], cmax[3]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_bf2(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) part[warp][0] = m;
    __syncthreads();
    m = part[0][0];
#pragma unroll
    for (int w = 1; w < 8; ++w) m = max_bf2(m, part[w][0]);
    const float2 f = bf2_to_f2(m);
    const float s = tile_scale(fmaxf(f.x, f.y), a.pow2);
#pragma unroll
    for (int i = 0; i < 8; ++i) row_s[i] = s;
    if (tid == 0) {
      a.s[tr * a.lds + tc] = s;
      if (TRANSPOSED) a.st[(int64_t)tc * a.ldst + tr] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t m = rmax[i];
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = max_bf2(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float2 f = bf2_to_f2(m);
      row_s[i] = tile_scale(fmaxf(f.x, f.y), a.pow2);
      if (v == i && r0 + i < a.M) a.s[(int64_t)tc * a.lds + r0 + i] = row_s[i];
    }
    if (TRANSPOSED) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        cmax[j] = max_bf2(cmax[j], __shfl_xor_sync(0xffffffffu, cmax[j], 16));
        if (lane < 16) part[warp][v * 4 + j] = cmax[j];
      }
      __syncthreads();
      if (tid < 64) {
        uint32_t m = part[0][tid];
#pragma unroll
        for (int w = 1; w < 8; ++w) m = max_bf2(m, part[w][tid]);
        const float2 f = bf2_to_f2(m);
        const float s0 = tile_scale(f.x, a.pow2), s1 = tile_scale(f.y, a.pow2);
        col_scale[2 * tid] = make_float2(s0, rcp_of(s0, a.pow2));
        col_scale[2 * tid + 1] = make_float2(s1, rcp_of(s1, a.pow2));
        const int c = tc * kTile + 2 * tid;
        if (c < a.H) a.st[tr * a.ldst + c] = s0;
        if (c + 1 < a.H) a.st[tr * a.ldst + c + 1] = s1;
      }
    }
  }
  // codes along the rows: 8 a thread, 128 contiguous bytes a row of the tile
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float s = row_s[i], rc = rcp_of(s, a.pow2);
    const float2 ns = make_float2(-s, -s), r2 = make_float2(rc, rc);
    float2 y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = div2_rn(bf2_to_f2(x[i][j]), ns, r2);
    const uint32_t lo = f4_to_e4m3x4(y[0], y[1]), hi = f4_to_e4m3x4(y[2], y[3]);
    if (col_ok && r0 + i < a.M) st_stream2(a.q + (r0 + i) * a.ldq + c0, lo, hi);
  }
  if (!TRANSPOSED) return;
  // codes along the columns: a column's 8 rows of this thread are 8 bytes
  if (!BLOCK) __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = v * 8 + 2 * j + h;
      const float2 sc = BLOCK ? make_float2(row_s[0], rcp_of(row_s[0], a.pow2)) : col_scale[c];
      const float2 ns = make_float2(-sc.x, -sc.x), r2 = make_float2(sc.y, sc.y);
      float2 y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = bf2_to_f2(x[2 * i][j]), q = bf2_to_f2(x[2 * i + 1][j]);
        y[i] = div2_rn(h ? make_float2(p.y, q.y) : make_float2(p.x, q.x), ns, r2);
      }
      // piece rg of column c, permuted by c / 8 = v
      *reinterpret_cast<uint2*>(t_codes + c * kTile + ((rg ^ v) << 3)) =
          make_uint2(f4_to_e4m3x4(y[0], y[1]), f4_to_e4m3x4(y[2], y[3]));
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
  auto kernel = block ? (a.qt != nullptr ? cast_tiles_kernel<true, true> : cast_tiles_kernel<true, false>)
                      : cast_tiles_kernel<false, true>;
  return launch_pdl(kernel, (unsigned)tiles, kThreads, 0, stream, a);
}

}  // namespace cutie
