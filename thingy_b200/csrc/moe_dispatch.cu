// Tokens sorted by expert and back (sm_100a). A plan holds, for T tokens with
// k choices each:
//   sources[r]      = t k + j, the choice of sorted row r, or -1 in padding
//   positions[t, j] = r, or -1 where the choice is absent
//   offsets[e]      = where expert e's rows begin, a multiple of `align`
//   counts[e]       = how many rows it has before its padding
// and the rows move by it:
//   permute:  out[r] = x[sources[r] / k], 0 in padding
//   combine:  y[t] = sum_j w[t, j] ys[positions[t, j]]  (w = 1: permute's gradient)
//   backward: dys[r] = w[t, j] dy[t], 0 in padding;  dw[t, j] = <dy[t], ys[r]>
// Sums run in fp32 in the order of j; no atomics, so results repeat. Entries of
// a plan out of range count as absent: nothing is read or written there.
#include <cuda_fp16.h>

#include "cutie.h"
#include "launch.cuh"

namespace cutie {
namespace {

// ------------------------------------------------------------------ sort
//
// A stable counting sort. A CTA takes a chunk of consecutive choices, a warp a
// consecutive part of it. Choices of one expert within 32 are found by a match
// among the lanes, so a warp's counters in shared memory need no atomics and
// ranks follow the choices' order. Up to kSortOne choices one CTA does all;
// above, a first launch counts each chunk and in the second every CTA adds up
// the chunks before its own, of which there are no more than run at once (1M ids of
// 512 experts: 128 chunks 32 us, 512 chunks 103; 262144 of 256: 128 chunks 12.4 us, 64
// chunks 15). Latency bounds both: the ids and the plan are a few MB at most.
constexpr size_t kSortStatic = (4 * kMoeMaxExperts + 32) * sizeof(int);  // shared memory of its own, at most
constexpr int kSortThreads = 1024, kSortOne = 4096, kSortChunk = 2048, kSortMaxChunks = 128;

struct SortArgs {
  const void* ids;
  bool wide;  // int64 ids, else int32
  int n, E, align, R;
  int *sources, *positions, *offsets, *counts;
  int* chunk_counts;  // [chunks, E], of the first launch
  int chunk;          // choices a CTA
};

// Choice i's expert; E where it is absent.
__device__ __forceinline__ int expert_of(const SortArgs& a, int i) {
  if (a.wide) {
    const int64_t e = static_cast<const int64_t*>(a.ids)[i];
    return e >= 0 && e < a.E ? (int)e : a.E;
  }
  const int e = static_cast<const int*>(a.ids)[i];
  return e >= 0 && e < a.E ? e : a.E;
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(const SortArgs a) {
  __shared__ int count[kMoeMaxExperts + 1];
  for (int e = threadIdx.x; e <= a.E; e += kSortThreads) count[e] = 0;
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  const int begin = (int)blockIdx.x * a.chunk, end = min(a.n - begin, a.chunk) + begin;
  for (int i = begin + (int)threadIdx.x; i < end; i += kSortThreads) atomicAdd(&count[expert_of(a, i)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += kSortThreads) a.chunk_counts[(int64_t)blockIdx.x * a.E + e] = count[e];
}

__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(const SortArgs a) {
  extern __shared__ int warp_next[];  // [warps][E + 1]: a warp's counts, then its next row of each expert
  __shared__ int before[kMoeMaxExperts], total[kMoeMaxExperts], first[kMoeMaxExperts + 1];
  __shared__ int warp_sum[kMoeMaxExperts / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = kSortThreads / 32;
  const int ld = a.E + 1;
  for (int i = tid; i < warps * ld; i += kSortThreads) warp_next[i] = 0;
  for (int e = tid; e < a.E; e += kSortThreads) before[e] = total[e] = 0;
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  const int begin = (int)blockIdx.x * a.chunk, end = min(a.n - begin, a.chunk) + begin;
  const int part = (a.chunk / 32 + warps - 1) / warps * 32;
  const int w0 = min(begin + warp * part, end), w1 = min(w0 + part, end);
  int* next = warp_next + warp * ld;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int i = i0 + lane, e = i < w1 ? expert_of(a, i) : a.E;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (lane == __ffs(same) - 1) next[e] += __popc(same);
    __syncwarp();
  }
  if (a.chunk_counts != nullptr) {
    // groups of threads, one a power of two >= E, each with a share of the chunks
    int width = 32;
    while (width < a.E) width *= 2;
    const int e = tid & (width - 1), groups = kSortThreads / width;
    if (e < a.E) {
      int b = 0, t = 0;
#pragma unroll 8
      for (int c = tid / width; c < (int)gridDim.x; c += groups) {
        const int v = a.chunk_counts[(int64_t)c * a.E + e];
        t += v;
        if (c < (int)blockIdx.x) b += v;
      }
      atomicAdd(&before[e], b);
      atomicAdd(&total[e], t);
    }
  }
  __syncthreads();
  // padded counts summed over the experts
  int mine = 0, up = 0;
  if (tid < kMoeMaxExperts) {
    if (tid < a.E) {
      if (a.chunk_counts == nullptr) {
        int t = 0;
        for (int w = 0; w < warps; ++w) t += warp_next[w * ld + tid];
        total[tid] = t;
      }
      mine = (total[tid] + a.align - 1) / a.align * a.align;
    }
    up = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += v;
    }
    if (lane == 31) warp_sum[warp] = up;
  }
  __syncthreads();
  if (tid < a.E) {
    int sum = up - mine;
    for (int w = 0; w < warp; ++w) sum += warp_sum[w];
    first[tid] = sum;
    if (tid == a.E - 1) first[a.E] = sum + mine;
    int row = sum + before[tid];
    for (int w = 0; w < warps; ++w) {
      const int c = warp_next[w * ld + tid];
      warp_next[w * ld + tid] = row;
      row += c;
    }
    if (blockIdx.x == 0) {
      a.offsets[tid] = sum;
      a.counts[tid] = total[tid];
      if (tid == a.E - 1) a.offsets[a.E] = sum + mine;
    }
  }
  __syncthreads();
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int i = i0 + lane, e = i < w1 ? expert_of(a, i) : a.E;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int row = e < a.E ? next[e] + __popc(same & ((1u << lane) - 1u)) : -1;
    __syncwarp();
    if (lane == __ffs(same) - 1) next[e] += __popc(same);
    __syncwarp();
    if (i < w1) {
      a.positions[i] = row;
      if (row >= 0) a.sources[row] = i;
    }
  }
  // padding: an expert a warp, then what is behind the last
  for (int e = (int)blockIdx.x * warps + warp; e < a.E; e += (int)gridDim.x * warps)
    for (int r = first[e] + total[e] + lane; r < first[e + 1]; r += 32) a.sources[r] = -1;
  for (int64_t r = (int64_t)first[a.E] + (int)blockIdx.x * kSortThreads + tid; r < a.R;
       r += (int64_t)gridDim.x * kSortThreads)
    a.sources[r] = -1;
}

// ------------------------------------------------------------------ rows
//
// Bound by memory. A thread moves vectors of 16 bytes (4, 2 or 1 where rows do
// not start on 16-byte boundaries or are not whole vectors). Permute goes by
// token: a row of x is read once and stored k times (by sorted row it would be
// read k times, past the L2 for a full batch). Rows in padding are zeroed by
// CTAs of their own behind those that copy.
constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32, kUnroll = 2, kAtOnce = 8;

template <int VB>
struct Raw;
template <>
struct Raw<16> {
  using T = uint4;
};
template <>
struct Raw<4> {
  using T = uint32_t;
};
template <>
struct Raw<2> {
  using T = uint16_t;
};
template <>
struct Raw<1> {
  using T = uint8_t;
};

// VB bytes of elements of type DT as floats, and back with one rounding.
template <int DT, int VB>
struct Elements {
  static constexpr int kSize = DT == CUTIE_DTYPE_F32 ? 4 : 2, N = VB / kSize;
  static __device__ __forceinline__ void get(const typename Raw<VB>::T& v, float (&f)[N]) {
    if constexpr (DT == CUTIE_DTYPE_F32) {
      const float* p = reinterpret_cast<const float*>(&v);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = p[i];
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(&v);
#pragma unroll
      for (int i = 0; i < N; ++i)
        f[i] = DT == CUTIE_DTYPE_BF16 ? __uint_as_float((uint32_t)p[i] << 16)
                                      : __half2float(__ushort_as_half(p[i]));
    }
  }
  static __device__ __forceinline__ typename Raw<VB>::T put(const float (&f)[N]) {
    typename Raw<VB>::T v;
    if constexpr (DT == CUTIE_DTYPE_F32) {
      float* p = reinterpret_cast<float*>(&v);
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = f[i];
    } else if constexpr (N == 1) {
      v = DT == CUTIE_DTYPE_BF16 ? (uint16_t)(f2_to_bf2(make_float2(f[0], 0.f)) & 0xffffu)
                                 : __half_as_ushort(__float2half_rn(f[0]));
    } else {
      uint32_t* p = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        if (DT == CUTIE_DTYPE_BF16) {
          p[i / 2] = f2_to_bf2(make_float2(f[i], f[i + 1]));
        } else {
          const __half2 h = __floats2half2_rn(f[i], f[i + 1]);
          p[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
    }
    return v;
  }
};

struct RowArgs {
  const char* x;  // rows that are read; strides in bytes
  int64_t ldx;
  const char* dy;  // backward: [T] rows
  int64_t lddy;
  char* out;
  int64_t ldo;
  const float* w;  // [T, k] or null
  float* dw;       // [T, k] or null
  const int *positions, *sources;
  int T, k, R, V;       // V: vectors a row
  unsigned work_blocks;  // CTAs that copy or sum; the others zero padding
  int zero_rows;         // sorted rows a warp looks at, at most 32
};

// Rows of `out` whose source is absent are zeroed.
template <int VB>
__device__ __forceinline__ void zero_padding(const RowArgs& a) {
  const int lane = threadIdx.x & 31;
  const int64_t r0 = ((int64_t)(blockIdx.x - a.work_blocks) * kRowWarps + (threadIdx.x >> 5)) * a.zero_rows;
  const int64_t r = r0 + lane;
  unsigned todo = __ballot_sync(0xffffffffu, lane < a.zero_rows && r < a.R && a.sources[r] < 0);
  for (; todo != 0; todo &= todo - 1) {
    typename Raw<VB>::T* row = reinterpret_cast<typename Raw<VB>::T*>(a.out + (r0 + __ffs(todo) - 1) * a.ldo);
    for (int v = lane; v < a.V; v += 32) row[v] = typename Raw<VB>::T{};
  }
}

template <int VB>
__global__ void __launch_bounds__(kRowThreads) permute_kernel(const RowArgs a) {
  using W = typename Raw<VB>::T;
  griddep_wait();
  griddep_launch_dependents();
  if (blockIdx.x >= a.work_blocks) {
    zero_padding<VB>(a);
    return;
  }
  const int64_t base = (int64_t)blockIdx.x * (kRowThreads * kUnroll);
  const int64_t t0 = base / a.V;
  const int v0 = (int)(base - t0 * a.V);
  W val[kUnroll];
  int64_t t[kUnroll];
  int v[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int at = v0 + u * kRowThreads + (int)threadIdx.x;
    t[u] = t0 + at / a.V;
    v[u] = at % a.V;
    if (t[u] < a.T) val[u] = reinterpret_cast<const W*>(a.x + t[u] * a.ldx)[v[u]];
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (t[u] >= a.T) break;
    const int* p = a.positions + t[u] * a.k;
#pragma unroll 4
    for (int j = 0; j < a.k; ++j) {
      const int r = p[j];
      if ((unsigned)r < (unsigned)a.R) reinterpret_cast<W*>(a.out + r * a.ldo)[v[u]] = val[u];
    }
  }
}

template <int DT, int VB, bool WEIGHTED>
__global__ void __launch_bounds__(kRowThreads) combine_kernel(const RowArgs a) {
  using W = typename Raw<VB>::T;
  using El = Elements<DT, VB>;
  griddep_wait();
  griddep_launch_dependents();
  const int64_t base = (int64_t)blockIdx.x * kRowThreads;
  const int64_t t0 = base / a.V;
  const int at = (int)(base - t0 * a.V) + (int)threadIdx.x;
  const int64_t t = t0 + at / a.V;
  const int v = at % a.V;
  if (t >= a.T) return;
  float acc[El::N];
#pragma unroll
  for (int i = 0; i < El::N; ++i) acc[i] = 0.f;
  for (int j0 = 0; j0 < a.k; j0 += kAtOnce) {
    W val[kAtOnce];
    int row[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) row[j] = j0 + j < a.k ? a.positions[t * a.k + j0 + j] : -1;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if ((unsigned)row[j] < (unsigned)a.R) val[j] = reinterpret_cast<const W*>(a.x + row[j] * a.ldx)[v];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if ((unsigned)row[j] >= (unsigned)a.R) continue;
      float f[El::N];
      El::get(val[j], f);
      const float w = WEIGHTED ? a.w[t * a.k + j0 + j] : 1.f;
#pragma unroll
      for (int i = 0; i < El::N; ++i) acc[i] = WEIGHTED ? fmaf(w, f[i], acc[i]) : acc[i] + f[i];
    }
  }
  reinterpret_cast<W*>(a.out + t * a.ldo)[v] = El::put(acc);
}

// P warps a token: 1, or all of the CTA's where tokens are few. The k dot
// products of a token are kept in registers, kAtOnce at a time, and added over
// the lanes once a row.
template <int DT, int VB, int P>
__global__ void __launch_bounds__(kRowThreads) combine_backward_kernel(const RowArgs a) {
  using W = typename Raw<VB>::T;
  using El = Elements<DT, VB>;
  __shared__ float part[P == 1 ? 1 : kRowWarps][kAtOnce];
  griddep_wait();
  griddep_launch_dependents();
  if (blockIdx.x >= a.work_blocks) {
    zero_padding<VB>(a);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = P == 1 ? (int64_t)blockIdx.x * kRowWarps + warp : blockIdx.x;
  if (t >= a.T) return;
  const W* dy = reinterpret_cast<const W*>(a.dy + t * a.lddy);
  for (int j0 = 0; j0 < a.k; j0 += kAtOnce) {
    int row[kAtOnce];
    float w[kAtOnce], dot[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const bool some = j0 + j < a.k;
      row[j] = some ? a.positions[t * a.k + j0 + j] : -1;
      w[j] = some ? a.w[t * a.k + j0 + j] : 0.f;
      dot[j] = 0.f;
    }
    for (int v = (P == 1 ? 0 : warp * 32) + lane; v < a.V; v += 32 * P) {
      W val[kAtOnce];
      if (a.dw != nullptr) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
          if ((unsigned)row[j] < (unsigned)a.R) val[j] = reinterpret_cast<const W*>(a.x + row[j] * a.ldx)[v];
      }
      float g[El::N];
      El::get(dy[v], g);
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if ((unsigned)row[j] >= (unsigned)a.R) continue;
        float f[El::N];
        if (a.dw != nullptr) {
          El::get(val[j], f);
#pragma unroll
          for (int i = 0; i < El::N; ++i) dot[j] = fmaf(g[i], f[i], dot[j]);
        }
        if (a.out != nullptr) {
#pragma unroll
          for (int i = 0; i < El::N; ++i) f[i] = w[j] * g[i];
          reinterpret_cast<W*>(a.out + row[j] * a.ldo)[v] = El::put(f);
        }
      }
    }
    if (a.dw == nullptr) continue;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) dot[j] = warp_reduce<false>(dot[j]);
    if (P == 1) {
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (lane == j && j0 + j < a.k) a.dw[t * a.k + j0 + j] = dot[j];
    } else {
      __syncthreads();  // the round before has been read
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (lane == j) part[warp][j] = dot[j];
      __syncthreads();
      if (threadIdx.x < kAtOnce && j0 + (int)threadIdx.x < a.k) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < P; ++q) s += part[q][threadIdx.x];
        a.dw[t * a.k + j0 + threadIdx.x] = s;
      }
    }
  }
}

// The widest vector that all of `bits` (addresses, strides, a row's bytes) are multiples of.
int vector_bytes(uint64_t bits, int element) {
  for (int vb : {16, 4, 2})
    if (bits % vb == 0 && vb >= element) return vb;
  return element;
}

// Rows a warp looks at for padding: few while that leaves warps for every SM.
int zero_rows(int64_t R) {
  int g = 32;
  while (g > 1 && R / g < 8 * kRowWarps * device_sm_count()) g /= 2;
  return g;
}

}  // namespace

size_t moe_sort_workspace(int64_t n, int64_t E) {
  if (n <= kSortOne) return 0;
  const int64_t chunks = (n + kSortChunk - 1) / kSortChunk;
  return (size_t)((chunks < kSortMaxChunks ? chunks : kSortMaxChunks) * E * 4);
}

cudaError_t moe_sort(const void* ids, bool wide, int n, int E, int align, int* sources, int R, int* positions,
                     int* offsets, int* counts, void* workspace, cudaStream_t stream) {
  SortArgs a{ids, wide, n, E, align, R, sources, positions, offsets, counts, nullptr, 0};
  int64_t chunk = n;
  if (n > kSortOne) {
    a.chunk_counts = static_cast<int*>(workspace);
    chunk = ((int64_t)n + kSortMaxChunks - 1) / kSortMaxChunks;
    if (chunk < kSortChunk) chunk = kSortChunk;
  }
  a.chunk = (int)((chunk + kSortThreads - 1) / kSortThreads * kSortThreads);
  const unsigned grid = n > kSortOne ? (unsigned)(((int64_t)n + a.chunk - 1) / a.chunk) : 1u;
  if (grid > 1) {
    const cudaError_t e = launch_pdl(sort_count_kernel, grid, kSortThreads, 0, stream, a);
    if (e != cudaSuccess) return e;
  } else {
    a.chunk_counts = nullptr;
  }
  const size_t smem = (size_t)(kSortThreads / 32) * (E + 1) * sizeof(int);
  if (smem + kSortStatic > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(sort_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (kSortThreads / 32) * (kMoeMaxExperts + 1) * (int)sizeof(int));
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(sort_place_kernel, grid, kSortThreads, smem, stream, a);
}

namespace {

RowArgs row_args(const MoeRows& p, int vb) {
  RowArgs a{};
  a.x = static_cast<const char*>(p.x), a.ldx = p.ldx;
  a.dy = static_cast<const char*>(p.dy), a.lddy = p.lddy;
  a.out = static_cast<char*>(p.out), a.ldo = p.ldo;
  a.w = p.w, a.dw = p.dw;
  a.positions = p.positions, a.sources = p.sources;
  a.T = p.T, a.k = p.k, a.R = p.R;
  a.V = (int)(p.row_bytes / vb);
  return a;
}

// CTAs behind `work` that look for padding, or an error where the launch would have too many.
cudaError_t row_grid(RowArgs* a, int64_t work, bool zero, unsigned* grid) {
  a->zero_rows = zero ? zero_rows(a->R) : 1;
  const int64_t per = (int64_t)kRowWarps * a->zero_rows, zeros = zero ? (a->R + per - 1) / per : 0;
  if (work + zeros > INT32_MAX) return cudaErrorInvalidConfiguration;
  a->work_blocks = (unsigned)work;
  *grid = (unsigned)(work + zeros);
  return cudaSuccess;
}

uint64_t bits_of(const void* p, int64_t ld) { return reinterpret_cast<uint64_t>(p) | (uint64_t)ld; }

template <int VB>
cudaError_t launch_permute(const MoeRows& p, cudaStream_t stream) {
  RowArgs a = row_args(p, VB);
  unsigned grid;
  const int64_t per = kRowThreads * kUnroll;
  const cudaError_t e = row_grid(&a, ((int64_t)a.T * a.V + per - 1) / per, true, &grid);
  return e != cudaSuccess ? e : launch_pdl(permute_kernel<VB>, grid, kRowThreads, 0, stream, a);
}

template <int DT, int VB>
cudaError_t launch_combine(const MoeRows& p, cudaStream_t stream) {
  RowArgs a = row_args(p, VB);
  unsigned grid;
  const cudaError_t e = row_grid(&a, ((int64_t)a.T * a.V + kRowThreads - 1) / kRowThreads, false, &grid);
  if (e != cudaSuccess) return e;
  return a.w != nullptr ? launch_pdl(combine_kernel<DT, VB, true>, grid, kRowThreads, 0, stream, a)
                        : launch_pdl(combine_kernel<DT, VB, false>, grid, kRowThreads, 0, stream, a);
}

template <int DT, int VB>
cudaError_t launch_backward_rows(const MoeRows& p, cudaStream_t stream) {
  RowArgs a = row_args(p, VB);
  // a warp a token once that gives every SM two CTAs
  const bool few = a.T < 2 * kRowWarps * device_sm_count();
  unsigned grid;
  const cudaError_t e = row_grid(&a, few ? a.T : ((int64_t)a.T + kRowWarps - 1) / kRowWarps, a.out != nullptr, &grid);
  if (e != cudaSuccess) return e;
  return few ? launch_pdl(combine_backward_kernel<DT, VB, kRowWarps>, grid, kRowThreads, 0, stream, a)
             : launch_pdl(combine_backward_kernel<DT, VB, 1>, grid, kRowThreads, 0, stream, a);
}

template <int DT, int VB>
cudaError_t launch_rows(const MoeRows& p, bool backward, cudaStream_t stream) {
  return backward ? launch_backward_rows<DT, VB>(p, stream) : launch_combine<DT, VB>(p, stream);
}

}  // namespace

cudaError_t moe_permute(const MoeRows& p, cudaStream_t stream) {
  switch (vector_bytes(bits_of(p.x, p.ldx) | bits_of(p.out, p.ldo) | (uint64_t)p.row_bytes, 1)) {
    case 16: return launch_permute<16>(p, stream);
    case 4: return launch_permute<4>(p, stream);
    case 2: return launch_permute<2>(p, stream);
    default: return launch_permute<1>(p, stream);
  }
}

cudaError_t moe_combine(const MoeRows& p, int dtype, bool backward, cudaStream_t stream) {
  const uint64_t bits = bits_of(p.x, p.ldx) | bits_of(p.out, p.ldo) | bits_of(p.dy, p.lddy) | (uint64_t)p.row_bytes;
  const int vb = vector_bytes(bits, dtype == CUTIE_DTYPE_F32 ? 4 : 2);
  if (dtype == CUTIE_DTYPE_F32)
    return vb == 16 ? launch_rows<CUTIE_DTYPE_F32, 16>(p, backward, stream)
                    : launch_rows<CUTIE_DTYPE_F32, 4>(p, backward, stream);
  if (dtype == CUTIE_DTYPE_BF16)
    return vb == 16  ? launch_rows<CUTIE_DTYPE_BF16, 16>(p, backward, stream)
           : vb == 4 ? launch_rows<CUTIE_DTYPE_BF16, 4>(p, backward, stream)
                     : launch_rows<CUTIE_DTYPE_BF16, 2>(p, backward, stream);
  return vb == 16  ? launch_rows<CUTIE_DTYPE_F16, 16>(p, backward, stream)
         : vb == 4 ? launch_rows<CUTIE_DTYPE_F16, 4>(p, backward, stream)
                   : launch_rows<CUTIE_DTYPE_F16, 2>(p, backward, stream);
}

}  // namespace cutie
