// FP8 product with a scale for each block of 128 (sm_100a):
//
//   D[m, n] = sum_kb sA[m, kb] sB[n, kb] * sum_{k in block kb} a[m, k] b[n, k]
//
// a: e4m3 [M, K] with fp32 scales of 1 x 128 groups; b: e4m3 [N, K] with fp32
// scales of 128 x 128 blocks (a weight) or of 1 x 128 groups (the other
// operand of a weight gradient). fp32 scales are not powers of two, so the
// tensor cores' own block scaling cannot apply them: the inner sum of every
// 128-wide K block is made by tcgen05.mma (kind::f8f6f4, fp32 accumulators in
// tensor memory, overwritten by each block) and the outer sum by the epilogue
// warps in fp32 registers, one FMA an element and block.
#include <atomic>

#include "cutie.h"
#include "launch.cuh"
#include "tcgen05.cuh"

namespace cutie {

static __device__ int g_block_gemm_device_error = 0;

namespace {

constexpr int kBM = 128, kBK = 128;
constexpr uint32_t kBoxBytes = kBM * kBK;  // one 128-row operand box: 16 KB
constexpr int kMaxRanks = 8;               // of a K split: a portable cluster

// Clusters of S CTAs (along z; pairs along x) that run at once on the current device, remembered.
int max_clusters(const void* kernel, int threads, size_t smem, dim3 cluster,
                 std::atomic<int> (&cache)[64][kMaxRanks + 1]) {
  int dev = 0;
  const unsigned S = cluster.x * cluster.z;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64 && cache[dev][S].load(std::memory_order_relaxed) > 0) return cache[dev][S].load();
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = cluster;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster.x;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = cluster.z;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) return 0;
  if (dev < 64) cache[dev][S].store(n);
  return n;
}

// Launch with clusters of `pair` CTAs along x, grid.z along z, and programmatic stream serialization.
template <class K, class... A>
cudaError_t launch_cluster(K kernel, dim3 grid, unsigned pair, int threads, size_t smem, cudaStream_t stream,
                           const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = pair;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = grid.z;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ------------------------------------------------------------------ tiled
//
// Persistent CTAs of 12 warps (the last one idle), one an SM, each walking tiles of 128 x BN:
//  * warp 8, one thread: TMA of the A box and the BN / 128 B boxes of a K
//    block into a ring of stages (128-byte swizzled rows; rows and columns
//    past the matrices are zero-filled, so M, N and K may be any).
//  * warp 9, one thread: four MMAs of 128 x BN x 32 a K block into one of two
//    accumulator buffers in tensor memory; a commit hands the buffer to the
//    epilogue, a second frees the stage.
//  * warps 0-7: the outer sum. Warp group g = warp / 4 keeps columns
//    g BN/2 .. of the tile for its 128 rows, a row a thread, in BN / 2 fp32
//    registers, and adds scale * buffer to them while the MMAs of the next K
//    block fill the other buffer.
//  * warp 10: the scales, copied to a ring in shared memory up to two slots of
//    kScaleBlocks K blocks ahead, so that the sums spend hardly an instruction
//    on them (one wait in kScaleBlocks blocks).
// Tiles are walked in bands of kBand rows of tiles, so that the CTAs of a
// wave share their operands in L2.
//
// Pairs (cta_group::2): two CTAs of a cluster make a tile of 256 x 256, 128 rows
// each. Each loads its rows of A and half of the rows of B; rank 0's MMAs (256 x
// 256 x 32) read both, so a K block brings 32 KB instead of 48 KB into an SM's
// shared memory and the ring holds six. Rank 0 waits for the loads and the
// buffers of both, its commits go to both, and every CTA sums its own 128 rows.
//
// Bound: the tensor cores' 512 cycles a K block of 256 columns, the sums' about
// 700 and the hand-overs between them (a buffer is free once its last piece is in
// registers, then a signal, the next MMAs and a signal back) make 870 cycles;
// over seconds it is power, at 1.5 GHz. Tried without gain: accumulators handed
// over in halves (MMAs of 128 columns read A twice), 16 summing warps, spinning
// waits, deeper scale rings. A release at cluster scope on the arrival that frees
// a buffer cost 1000 cycles; it orders tensor memory only, which the fences do.
constexpr int kThreads = 384, kEpiWarps = 8, kBand = 16;
// registers a thread: 256 x 216 + 128 x 64 = 63488 of the 384 x 168 = 64512 at launch
constexpr int kEpiRegs = 216, kIssueRegs = 64;
constexpr int kScaleBlocks = 4;  // K blocks a slot of the scale ring
constexpr int kSplitBlocks = 16, kCutBlocks = 32;  // see split_ranks, launch_large

constexpr int kStageRow = 9;  // see store_rows

template <int BN, bool SB_ROWS, bool VEC, bool PAIR = false>
struct TilePlan {
  static constexpr int kNB = PAIR ? 1 : BN / 128;  // boxes of B that a CTA loads
  static constexpr uint32_t kStageBytes = (1 + kNB) * kBoxBytes;
  static constexpr int kStages = kNB == 2 ? 4 : 6;
  static constexpr size_t kSmemBytes = kStages * kStageBytes + 1024;
  static constexpr uint32_t kTmemCols = 2 * BN;
  static constexpr int kCols = BN / 2;  // columns of a warp group
  // scales of a K block: 128 rows', then the columns' (a scale each, or a block's)
  static constexpr int kScales = 128 + (SB_ROWS ? BN : 4);
  static constexpr int kScaleSlots = SB_ROWS ? 2 : 4;
  static_assert(kSmemBytes + kScaleSlots * kScaleBlocks * kScales * 4 + kEpiWarps * 32 * kStageRow * 4 * (VEC ? 0 : 1) + 512 <=
                    227 * 1024,
                "shared memory");
};

// Split form: a partial tile of 128 x 128 in shared memory, rows 4 floats apart
// from 128 (16-byte stores of 32 rows then fall into different banks).
constexpr int kPartRow = 132;
constexpr uint32_t kPartRowBytes = kPartRow * 4, kPartBytes = kBM * kPartRowBytes;
static_assert(kPartBytes + (kBM + kMaxRanks) * kPartRowBytes <= 6 * 2 * kBoxBytes, "parts fit the ring");

struct TileArgs {
  const float* sa;
  int64_t sa_row, sa_kb;
  const float* sb;
  int64_t sb_row, sb_kb;
  void* d;
  int64_t ldd;
  int M, N, KB, tiles_m, tiles_n;
  int tiles;  // to walk
  int band;   // rows of tiles that are walked together
  int tail;   // 128-wide form: >= 0: the parts of the larger tiles from this one on,
  int parts;  // 2 (columns) or 4 (columns and rows) each
  bool d_f32, accumulate;
  long long wait_limit;  // SM cycles a wait may block before it gives up (< 0: never blocks)
};

// Tile t of the banded walk.
__device__ __forceinline__ void tile_at(const TileArgs& g, int t, int* tm, int* tn) {
  const int band = t / (g.band * g.tiles_n), first = band * g.band;
  const int rows = g.tiles_m - first < g.band ? g.tiles_m - first : g.band;
  const int in = t - band * g.band * g.tiles_n;
  *tm = first + in % rows;
  *tn = in / rows;
}

template <int BN>
__device__ __forceinline__ void tile_of(const TileArgs& g, int t, int* tm, int* tn) {
  if (BN == 128 && g.tail >= 0) {
    tile_at(g, g.tail + t / g.parts, tm, tn);
    *tn = 2 * *tn + (t & 1);
    if (g.parts == 4) *tm = 2 * *tm + ((t >> 1) & 1);
  } else {
    tile_at(g, t, tm, tn);
  }
}

// A warp's 32 rows of NC columns. VEC: the rows of D start on 32-byte
// boundaries and hold whole 32-byte sectors, which the threads store that have
// them. Otherwise 8 columns at a time go through the warp's 32 x 9 floats of
// shared memory and leave as 8 consecutive elements of four rows an instruction
// (stored an element a thread they cost 30 us instead of 10 at 1001 x 1544).
// A template, not a branch: the mere presence of the second form cost the main
// loop of the first 6%.
template <int NC, bool VEC>
__device__ __forceinline__ void store_rows(const TileArgs& g, const float2 (&acc)[NC / 2], int row0,
                                           int col, int lane, float* stage) {
  if (VEC) {
    const int row = row0 + lane;
    if (row >= g.M) return;
    const int64_t at = (int64_t)row * g.ldd + col;
    if (!g.d_f32) {
      uint16_t* p = static_cast<uint16_t*>(g.d) + at;
#pragma unroll
      for (int c = 0; c < NC; c += 16) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = f2_to_bf2(acc[c / 2 + i]);
        if (col + c < g.N) st_stream8(p + c, w);
      }
    } else {
      float* p = static_cast<float*>(g.d) + at;
#pragma unroll
      for (int c = 0; c < NC; c += 8) {
        if (col + c >= g.N) break;
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = acc[c / 2 + i].x, v[2 * i + 1] = acc[c / 2 + i].y;
        if (g.accumulate) {
          const float4 o0 = *reinterpret_cast<const float4*>(p + c);
          const float4 o1 = *reinterpret_cast<const float4*>(p + c + 4);
          v[0] += o0.x, v[1] += o0.y, v[2] += o0.z, v[3] += o0.w;
          v[4] += o1.x, v[5] += o1.y, v[6] += o1.z, v[7] += o1.w;
        }
        st_stream8(p + c, reinterpret_cast<const uint32_t*>(v));
      }
    }
  } else {
    const int r4 = lane >> 3, c8 = lane & 7;
#pragma unroll
    for (int c = 0; c < NC; c += 8) {
      if (col + c >= g.N) break;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        stage[lane * kStageRow + 2 * i] = acc[c / 2 + i].x;
        stage[lane * kStageRow + 2 * i + 1] = acc[c / 2 + i].y;
      }
      __syncwarp();
      const int cc = col + c + c8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = row0 + 4 * i + r4;
        if (r >= g.M || cc >= g.N) break;
        const float v = stage[(4 * i + r4) * kStageRow + c8];
        const int64_t to = (int64_t)r * g.ldd + cc;
        if (g.d_f32) {
          float* p = static_cast<float*>(g.d) + to;
          *p = g.accumulate ? *p + v : v;
        } else {
          static_cast<uint16_t*>(g.d)[to] = (uint16_t)(f2_to_bf2(make_float2(v, 0.f)) & 0xffffu);
        }
      }
    }
  }
}

// Four columns of a row. VEC: they are aligned in D and all or none in it.
template <bool VEC>
__device__ __forceinline__ void store_four(const TileArgs& g, int row, int col, float4 v) {
  const int64_t at = (int64_t)row * g.ldd + col;
  const float f[4] = {v.x, v.y, v.z, v.w};
  if (g.d_f32) {
    float* p = static_cast<float*>(g.d) + at;
    if (VEC) {
      if (g.accumulate) {
        const float4 o = *reinterpret_cast<const float4*>(p);
        v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
      }
      *reinterpret_cast<float4*>(p) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col + i < g.N) p[i] = g.accumulate ? p[i] + f[i] : f[i];
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(g.d) + at;
    const uint32_t lo = f2_to_bf2(make_float2(v.x, v.y)), hi = f2_to_bf2(make_float2(v.z, v.w));
    if (VEC) {
      *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (col + i < g.N) p[i] = (uint16_t)((i < 2 ? lo : hi) >> (16 * (i & 1)));
    }
  }
}

template <int BN, bool SB_ROWS, bool VEC, bool SPLIT, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    block_gemm_kernel(const __grid_constant__ CUtensorMap map_a,
                      const __grid_constant__ CUtensorMap map_b, const TileArgs g) {
  using P = TilePlan<BN, SB_ROWS, VEC, PAIR>;
  static_assert(!PAIR || (BN == 256 && !SPLIT), "pairs make 256 x 256 tiles");
  constexpr int NC = P::kCols;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[P::kStages];
  __shared__ __align__(8) uint64_t empty_bar[P::kStages];
  __shared__ __align__(8) uint64_t acc_full[2];
  __shared__ __align__(8) uint64_t acc_empty[2];
  __shared__ __align__(8) uint64_t scale_full[P::kScaleSlots];
  __shared__ __align__(8) uint64_t scale_empty[P::kScaleSlots];
  __shared__ __align__(16) float scales[P::kScaleSlots][kScaleBlocks][P::kScales];
  __shared__ float stage[VEC || SPLIT ? 1 : kEpiWarps][32 * kStageRow];
  __shared__ __align__(8) uint64_t recv_bar;
  __shared__ uint32_t tmem_base_slot;
  __shared__ uint32_t abort_flag;
  __shared__ uint32_t issued;     // K blocks whose copies were issued
  __shared__ uint32_t committed;  // K blocks whose MMAs were committed

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  // tiles begin, begin + step, ... are this CTA's, or its pair's
  const int tiles = g.tiles, begin = PAIR ? blockIdx.x / 2 : blockIdx.x, step = PAIR ? gridDim.x / 2 : gridDim.x;
  // K blocks of this CTA: all, or the rank's of its cluster
  const int S = SPLIT ? (int)gridDim.z : 1, rank = SPLIT || PAIR ? (int)tc::cluster_ctarank() : 0;
  const int kb0 = SPLIT ? (int)((int64_t)g.KB * rank / S) : 0;
  const int nkb = SPLIT ? (int)((int64_t)g.KB * (rank + 1) / S) - kb0 : g.KB;
  // and the tile's rows that it adds up
  const int share = (kBM + S - 1) / S, own_lo = min(rank * share, kBM), own_n = min(share, kBM - own_lo);
  volatile uint32_t* abortp = &abort_flag;

  if (threadIdx.x == 0) {
    tc::prefetch_map(&map_a);
    tc::prefetch_map(&map_b);
    for (int s = 0; s < P::kStages; ++s) {
      mbar_init(smem_addr(&full_bar[s]), 1);
      mbar_init(smem_addr(&empty_bar[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_addr(&acc_full[b]), 1);
      mbar_init(smem_addr(&acc_empty[b]), (PAIR ? 2 : 1) * kEpiWarps);
    }
    for (int s = 0; s < P::kScaleSlots; ++s) {
      mbar_init(smem_addr(&scale_full[s]), 32);
      mbar_init(smem_addr(&scale_empty[s]), kEpiWarps);
    }
    if (SPLIT) mbar_init(smem_addr(&recv_bar), 1);
    abort_flag = 0;
    issued = committed = 0;
    mbar_init_fence();
    if (SPLIT) mbar_arrive_expect_tx(smem_addr(&recv_bar), (uint32_t)((S - 1) * own_n) * kPartRowBytes);
  }
  if (warp == kEpiWarps) {
    if (PAIR) tc::tmem_alloc_pair(smem_addr(&tmem_base_slot), P::kTmemCols);
    else tc::tmem_alloc(smem_addr(&tmem_base_slot), P::kTmemCols);
  }
  tc::fence_before();
  __syncthreads();
  if (PAIR) tc::cluster_sync();  // both CTAs' barriers and tensor memory are ready
  tc::fence_after();
  const uint32_t tmem = tmem_base_slot;
  griddep_wait();
  griddep_launch_dependents();

  if (warp >= kEpiWarps) {
    tc::regs_down<kIssueRegs>();
  if (warp == kEpiWarps) {
    // ---- operands
    const bool leader = tc::elect_one();
    uint32_t s = 0, parity = 1;  // a fresh barrier passes a wait for the phase before its first
    bool ok = true;
    for (int t = begin; t < tiles && ok; t += step) {
      int tm, tn;
      tile_of<BN>(g, t, &tm, &tn);
      for (int kb = 0; kb < nkb; ++kb) {
        ok = tc::wait_or_abort(smem_addr(&empty_bar[s]), parity, abortp, g.wait_limit);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        if (leader) {
          const uint32_t st = base + s * P::kStageBytes, bar = smem_addr(&full_bar[s]);
          if constexpr (PAIR) {
            // both CTAs' loads are counted on rank 0's barrier
            if (rank == 0) mbar_arrive_expect_tx(bar, 2 * P::kStageBytes);
            const uint32_t to = tc::mapa(bar, 0);
            tc::tma_load_2d_pair(st, &map_a, kb * kBK, (2 * tm + rank) * kBM, to);
            tc::tma_load_2d_pair(st + kBoxBytes, &map_b, kb * kBK, tn * BN + 128 * rank, to);
          } else {
            mbar_arrive_expect_tx(bar, P::kStageBytes);
            tc::tma_load_2d(st, &map_a, (kb0 + kb) * kBK, tm * kBM, bar);
#pragma unroll
            for (int h = 0; h < P::kNB; ++h)
              tc::tma_load_2d(st + (1 + h) * kBoxBytes, &map_b, (kb0 + kb) * kBK, tn * BN + 128 * h, bar);
          }
          ++issued;
        }
        if (++s == P::kStages) s = 0, parity ^= 1;
      }
    }
    if (PAIR)  // rank 0's commits arrive here: all before this CTA's memory goes
      for (int i = 0; i < P::kStages && ok; ++i) {
        ok = __all_sync(0xffffffffu, tc::wait_or_abort(smem_addr(&empty_bar[s]), parity, abortp, g.wait_limit));
        if (++s == P::kStages) s = 0, parity ^= 1;
      }
  } else if (warp == kEpiWarps + 1) {
    // ---- MMAs
    const bool leader = tc::elect_one();
    constexpr uint32_t idesc = tc::f8_idesc(PAIR ? 2 * kBM : kBM, BN);
    const uint32_t lo0 = tc::sw128_lo(base), hi = tc::sw128_hi();
    uint32_t s = 0, parity = 0, buf = 0, buf_parity = 1;
    bool ok = !PAIR || rank == 0;  // rank 0 issues for both
    for (int t = begin; t < tiles && ok; t += step) {
      for (int kb = 0; kb < nkb; ++kb) {
        ok = tc::wait_or_abort(smem_addr(&full_bar[s]), parity, abortp, g.wait_limit) &&
             tc::wait_or_abort(smem_addr(&acc_empty[buf]), buf_parity, abortp, g.wait_limit);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc::fence_after();
        if (leader) {
          const uint32_t lo = lo0 + s * (P::kStageBytes >> 4);
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            if (PAIR)
              tc::mma_f8_pair(tmem + buf * BN, lo + 2 * kk, lo + (kBoxBytes >> 4) + 2 * kk, hi, idesc,
                              kk != 0);
            else
              tc::mma_f8(tmem + buf * BN, lo + 2 * kk, lo + (kBoxBytes >> 4) + 2 * kk, hi, idesc,
                         kk != 0);
          if (PAIR) {
            tc::commit_pair(smem_addr(&acc_full[buf]));
            tc::commit_pair(smem_addr(&empty_bar[s]));
          } else {
            tc::commit(smem_addr(&acc_full[buf]));
            tc::commit(smem_addr(&empty_bar[s]));
          }
          ++committed;
        }
        __syncwarp();
        if (++s == P::kStages) s = 0, parity ^= 1;
        buf ^= 1;
        buf_parity ^= buf == 0;
      }
    }
  } else if (warp == kEpiWarps + 2) {
    // ---- scales; those of rows and columns past the matrices are left as they are
    uint32_t s = 0, parity = 1;
    bool ok = true;
    constexpr int kNS = SB_ROWS ? BN / 32 : 1;
    for (int t = begin; t < tiles && ok; t += step) {
      int tm, tn;
      tile_of<BN>(g, t, &tm, &tn);
      const float *pa[4], *pb[kNS];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = (PAIR ? 2 * tm + rank : tm) * kBM + lane + 32 * i;
        pa[i] = row < g.M ? g.sa + (int64_t)row * g.sa_row + kb0 * g.sa_kb : nullptr;
      }
#pragma unroll
      for (int i = 0; i < kNS; ++i) {
        const int col = tn * BN + (SB_ROWS ? lane + 32 * i : 128 * lane);
        const bool some = col < g.N && (SB_ROWS || lane < BN / 128);
        pb[i] = some ? g.sb + (int64_t)(SB_ROWS ? col : col / 128) * g.sb_row + kb0 * g.sb_kb : nullptr;
      }
      for (int kb = 0; kb < nkb; ++kb) {
        const int j = kb % kScaleBlocks;
        if (j == 0) {
          ok = __all_sync(0xffffffffu,
                          tc::wait_or_abort(smem_addr(&scale_empty[s]), parity, abortp, g.wait_limit));
          if (!ok) break;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (pa[i] != nullptr) {
            tc::cp_async_4(smem_addr(&scales[s][j][lane + 32 * i]), pa[i]);
            pa[i] += g.sa_kb;
          }
#pragma unroll
        for (int i = 0; i < kNS; ++i)
          if (pb[i] != nullptr) {
            tc::cp_async_4(smem_addr(&scales[s][j][128 + lane + 32 * i]), pb[i]);
            pb[i] += g.sb_kb;
          }
        if (j == kScaleBlocks - 1 || kb == nkb - 1) {
          tc::cp_async_arrive(smem_addr(&scale_full[s]));
          if (++s == P::kScaleSlots) s = 0, parity ^= 1;
        }
      }
    }
    tc::cp_async_wait_all();
  }
  } else {
    // ---- the outer sum
    tc::regs_up<kEpiRegs>();
    const int wg = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t tm_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(wg * NC);
    // The buffer is read in pieces of CH columns, each load issued before the
    // sums of the piece before it, the first of the next K block before those
    // of the last of this one: no sum waits for its own load's latency. `lo`
    // and `hi` take turns. With a scale a column the pieces are half as wide and
    // the piece's scales are in registers before its load is waited for. After
    // an abort the waits return at once and the loads go on (tensor memory is
    // still this CTA's).
    constexpr int CH = SB_ROWS ? 16 : 32;
    uint32_t lo[CH], hi[CH];
    uint32_t buf = 0, buf_parity = 0, slot = 0, slot_parity = 0;
    float sc = 0.f;  // the row's scale of the block, times the column block's
    const float* sb = nullptr;  // the columns' scales of the block
    const bool first = lane == 0;
    // K block kb of a tile: its first load, and its scales
    auto begin_block = [&](int kb) {
      const int j = kb % kScaleBlocks;
      if (j == 0) tc::wait_or_abort(smem_addr(&scale_full[slot]), slot_parity, abortp, g.wait_limit);
      sc = scales[slot][j][r];
      sb = &scales[slot][j][128 + (SB_ROWS ? wg * NC : wg * NC / 128)];
      if (!SB_ROWS) sc *= *sb;
      tc::wait_or_abort(smem_addr(&acc_full[buf]), buf_parity, abortp, g.wait_limit);
      __syncwarp();
      tc::fence_after();
      tc::tmem_ld_async(tm_lane + buf * BN, lo);
    };
    if (begin < tiles) begin_block(0);
    for (int t = begin; t < tiles; t += step) {
      float2 acc[NC / 2];
#pragma unroll
      for (int i = 0; i < NC / 2; ++i) acc[i] = make_float2(0.f, 0.f);
      for (int kb = 0; kb < nkb; ++kb) {
        const bool last = kb == nkb - 1;
        const float s = sc;
        const float* col = sb;
        const uint32_t tm = tm_lane + buf * BN;
        float4 f[SB_ROWS ? CH / 4 : 1];
        auto column_scales = [&](int c) {  // of piece c, before its load is waited for
          if (SB_ROWS) {
#pragma unroll
            for (int i = 0; i < CH / 4; ++i) f[i] = *reinterpret_cast<const float4*>(col + c + 4 * i);
          }
        };
        auto add = [&](int c, const uint32_t(&v)[CH]) {
          const float2 s2 = make_float2(s, s);
#pragma unroll
          for (int i = 0; i < CH / 4; ++i) {
            float2 d0 = make_float2(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]));
            float2 d1 = make_float2(__uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
            if (SB_ROWS) {
              d0 = __fmul2_rn(d0, make_float2(f[i].x, f[i].y));
              d1 = __fmul2_rn(d1, make_float2(f[i].z, f[i].w));
            }
            acc[c / 2 + 2 * i] = __ffma2_rn(d0, s2, acc[c / 2 + 2 * i]);
            acc[c / 2 + 2 * i + 1] = __ffma2_rn(d1, s2, acc[c / 2 + 2 * i + 1]);
          }
        };
        const bool slot_done = last || kb % kScaleBlocks == kScaleBlocks - 1;
        const uint32_t done = smem_addr(&scale_empty[slot]);
#pragma unroll
        for (int c = 0; c < NC; c += 2 * CH) {
          column_scales(c);
          tc::tmem_ld_wait(lo);
          tc::tmem_ld_async(tm + (uint32_t)(c + CH), hi);
          add(c, lo);
          column_scales(c + CH);
          tc::tmem_ld_wait(hi);
          if (c + 2 * CH < NC) {
            tc::tmem_ld_async(tm + (uint32_t)(c + 2 * CH), lo);
          } else {  // all of the buffer is in registers
            tc::fence_before();
            __syncwarp();
            if (PAIR) tc::arrive_cluster_if(first, tc::mapa(smem_addr(&acc_empty[buf]), 0));
            else tc::arrive_if(first, smem_addr(&acc_empty[buf]));
            buf ^= 1;
            buf_parity ^= buf == 0;
            if (slot_done && ++slot == P::kScaleSlots) slot = 0, slot_parity ^= 1;
            if (!last || t + step < tiles) begin_block(last ? 0 : kb + 1);
          }
          add(c + CH, hi);
        }
        if (slot_done) {
          __syncwarp();
          tc::arrive_if(first, done);
        }
      }
      int tm_i, tn_i;
      tile_of<BN>(g, t, &tm_i, &tn_i);
      if constexpr (!SPLIT) {
        if (*abortp == 0u)
          store_rows<NC, VEC>(g, acc, (PAIR ? 2 * tm_i + rank : tm_i) * kBM + (warp & 3) * 32, tn_i * BN + wg * NC, lane,
                              stage[VEC ? 0 : warp]);
      } else {
        // the last accumulator was complete, so this CTA's ring is idle, and so
        // are the others' once they have arrived too: the partial tile to the
        // ring, every rank's share of its rows to that rank, and what came from
        // the others added in rank order
        float* part = reinterpret_cast<float*>(smem_raw + (base - smem_addr(smem_raw)));
        asm volatile("barrier.cta.sync 1, 256;" ::: "memory");  // all warps are past the ring
#pragma unroll
        for (int c = 0; c < NC; c += 4)
          *reinterpret_cast<float4*>(part + r * kPartRow + wg * NC + c) =
              make_float4(acc[c / 2].x, acc[c / 2].y, acc[c / 2 + 1].x, acc[c / 2 + 1].y);
        tc::fence_async_smem();
        asm volatile("barrier.cta.sync 1, 256;" ::: "memory");
        tc::cluster_arrive();
        tc::cluster_wait();
        // also after an abort, so that every copy between the ranks is counted
        // and over before one of them ends
        if (threadIdx.x == 0) {
          for (int q = 0; q < S; ++q) {
            const int lo_q = min(q * share, kBM), n = min(share, kBM - lo_q);
            if (q == rank || n == 0) continue;
            tc::bulk_s2c(tc::mapa(base + kPartBytes + (uint32_t)(rank * share) * kPartRowBytes, (uint32_t)q),
                         smem_addr(part + lo_q * kPartRow), (uint32_t)n * kPartRowBytes,
                         tc::mapa(smem_addr(&recv_bar), (uint32_t)q));
          }
        }
        const bool got = __all_sync(
            0xffffffffu, tc::wait_or_abort(smem_addr(&recv_bar), 0u, abortp, g.wait_limit));
        if (!got) mbar_wait_bounded(smem_addr(&recv_bar), 0u, kDrainLimitCycles);
        __syncwarp();
        tc::cluster_arrive();  // what the others sent has arrived
        if (got && *abortp == 0u) {
          const float* in = part + kPartBytes / 4;
          const int col = tn_i * BN + lane * 4;
          for (int i = warp; i < own_n; i += kEpiWarps) {
            const int row = tm_i * kBM + own_lo + i;
            if (row >= g.M || col >= g.N) continue;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int q = 0; q < kMaxRanks; ++q)
              if (q < S) {
                const float4 o = *reinterpret_cast<const float4*>(
                    (q == rank ? part + (own_lo + i) * kPartRow : in + (q * share + i) * kPartRow) + lane * 4);
                v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
              }
            store_four<VEC>(g, row, col, v);
          }
        }
      }
    }
  }
  __syncwarp();
  if (SPLIT) {
    if (warp >= kEpiWarps) {
      tc::cluster_arrive();
      tc::cluster_wait();
      tc::cluster_arrive();
    }
    tc::cluster_wait();  // what this CTA sent has arrived: its memory may go
  }
  tc::fence_before();
  __syncthreads();
  if (*abortp) {
    // let copies and MMAs in flight finish before their memory goes away
    if (threadIdx.x == 0) {
      atomicCAS(&g_block_gemm_device_error, kDevErrNone, kDevErrBulkWaitTimeout);
      const uint32_t n = issued, m = committed;
      for (uint32_t k = n > P::kStages ? n - P::kStages : 0; k < n && (!PAIR || rank == 0); ++k)
        mbar_wait_bounded(smem_addr(&full_bar[k % P::kStages]), (k / P::kStages) & 1u,
                          kDrainLimitCycles);
      if (m > 0)
        mbar_wait_bounded(smem_addr(&acc_full[(m - 1) & 1u]), ((m - 1) >> 1) & 1u,
                          kDrainLimitCycles);
      // and what nothing counts now: a pair's loads on their way here, or parts of
      // a rank that gave up later than this one
      for (const long long t0 = clock64(); (SPLIT || PAIR) && clock64() - t0 < kDrainLimitCycles / 100;) {
      }
    }
    __syncthreads();
  }
  if (PAIR) {
    tc::cluster_arrive();
    tc::cluster_wait();
  }
  if (warp == kEpiWarps) {
    if (PAIR) tc::tmem_dealloc_pair(tmem, P::kTmemCols);
    else tc::tmem_dealloc(tmem, P::kTmemCols);
  }
}

template <int BN, bool SB_ROWS, bool VEC>
cudaError_t launch_tiled(const BlockGemmArgs& p, TileArgs g, cudaStream_t stream) {
  using P = TilePlan<BN, SB_ROWS, VEC>;
  auto kernel = block_gemm_kernel<BN, SB_ROWS, VEC, false, false>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::kSmemBytes);
  if (e != cudaSuccess) return e;
  CUtensorMap map_a, map_b;
  if (!tc::encode_e4m3_operand(&map_a, p.a, p.M, p.K, p.lda, kBM) ||
      !tc::encode_e4m3_operand(&map_b, p.b, p.N, p.K, p.ldb, kBM))
    return cudaErrorInvalidValue;
  const int sms = device_sm_count();
  return launch_pdl(kernel, (unsigned)(g.tiles < sms ? g.tiles : sms), kThreads, P::kSmemBytes, stream,
                    map_a, map_b, g);
}

// 256 x 256 tiles by pairs of CTAs; how many pairs run at once.
template <bool SB_ROWS, bool VEC>
int pair_clusters() {
  static std::atomic<int> cache[64][kMaxRanks + 1];
  return max_clusters(reinterpret_cast<const void*>(block_gemm_kernel<256, SB_ROWS, VEC, false, true>),
                      kThreads, TilePlan<256, SB_ROWS, VEC, true>::kSmemBytes, dim3(2, 1, 1), cache);
}

template <bool SB_ROWS, bool VEC>
cudaError_t launch_pairs(const BlockGemmArgs& p, TileArgs g, int pairs, cudaStream_t stream) {
  using P = TilePlan<256, SB_ROWS, VEC, true>;
  auto kernel = block_gemm_kernel<256, SB_ROWS, VEC, false, true>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::kSmemBytes);
  if (e != cudaSuccess) return e;
  CUtensorMap map_a, map_b;
  if (!tc::encode_e4m3_operand(&map_a, p.a, p.M, p.K, p.lda, kBM) ||
      !tc::encode_e4m3_operand(&map_b, p.b, p.N, p.K, p.ldb, kBM))
    return cudaErrorInvalidValue;
  return launch_cluster(kernel, dim3(2u * (unsigned)(g.tiles < pairs ? g.tiles : pairs)), 2, kThreads,
                        P::kSmemBytes, stream, map_a, map_b, g);
}

// The split form: tiles of 128 x 128 that leave SMs idle, K split over a cluster.
template <bool SB_ROWS, bool VEC>
int split_clusters(int S) {
  static std::atomic<int> cache[64][kMaxRanks + 1];
  return max_clusters(reinterpret_cast<const void*>(block_gemm_kernel<128, SB_ROWS, VEC, true, false>), kThreads,
                      TilePlan<128, SB_ROWS, true>::kSmemBytes, dim3(1, 1, (unsigned)S), cache);
}

// Ranks: the most with which all tiles still run at once; 1, not split, where that
// leaves out fewer than kSplitBlocks K blocks of a CTA's time: adding the parts
// costs 2 to 3 us (cold L2, unsplit against split: 512 x 2048 x 2048, 8 blocks
// left out, 14 against 16 us; 512 x 2048 x 4096, 16 left out, 22 against 20;
// 128 x 2048 x 7168, 28 to 49 left out, 27 against 22 to 18).
template <bool SB_ROWS, bool VEC>
int split_ranks(const TileArgs& g) {
  const int tiles = g.tiles;
  int S = kMaxRanks;
  while (S > 1 && (S > g.KB || split_clusters<SB_ROWS, VEC>(S) < tiles)) --S;
  return g.KB - (g.KB + S - 1) / S >= kSplitBlocks ? S : 1;
}

template <bool SB_ROWS, bool VEC>
cudaError_t launch_split(const BlockGemmArgs& p, TileArgs g, int S, cudaStream_t stream) {
  using P = TilePlan<128, SB_ROWS, true>;
  auto kernel = block_gemm_kernel<128, SB_ROWS, VEC, true, false>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P::kSmemBytes);
  if (e != cudaSuccess) return e;
  CUtensorMap map_a, map_b;
  if (!tc::encode_e4m3_operand(&map_a, p.a, p.M, p.K, p.lda, kBM) ||
      !tc::encode_e4m3_operand(&map_b, p.b, p.N, p.K, p.ldb, kBM))
    return cudaErrorInvalidValue;
  return launch_cluster(kernel, dim3((unsigned)g.tiles, 1, (unsigned)S), 1, kThreads,
                        P::kSmemBytes, stream, map_a, map_b, g);
}

// ------------------------------------------------------------------ few rows
//
// At most 64 rows of A: bound by reading the weight once. The weight is the
// 128-row side of the MMA and the batch its N side (BR = 16, 32 or 64 columns,
// the smallest that holds the batch; rows past M are zero-filled), so a K block
// costs 16 KB of weight and a batch box of BR rows. N / 128 tiles do
// not fill the GPU, so K is split over a cluster of S CTAs, with two CTAs an SM
// (one for BR = 64): every SM then has its share of the weight on the way at
// once. Two K blocks share a ring stage and its barriers: the hand-over
// between the warps, not the bytes, set the time of one-block stages.
// The ranks' partial tiles are reduce-scattered: each rank owns a share of the
// batch rows, the others send it theirs (bulk copies between shared memories,
// no multicast), and it adds all in rank order, so the result does not depend
// on timing.
// Warps 0-3 sum (a weight row a thread), 4 issues TMA, 5 MMAs, 6 copies scales.
// Rows up to which this form is taken, and rows from which it is only while K is
// split (N leaves SMs idle). Against the tiled form, cold L2: 33 x 5120 x 5120
// 18 against 22 us, 64 x 7168 x 7168 27 against 29; 64 x 16384 x 4096 (no split)
// 28 against 24; a 128-column plan lost from 128 x 5120 x 5120 (27 against 23) on.
constexpr int kFewRows = 64, kFewSplitRows = 32;
constexpr int kFewThreads = 224, kFewScaleSlots = 3, kFewStep = 2;

template <int BR>
struct FewPlan {
  static constexpr int kCtas = BR <= 32 ? 2 : 1;  // an SM
  static constexpr uint32_t kBlockBytes = kBoxBytes + BR * kBK;
  static constexpr uint32_t kStageBytes = kFewStep * kBlockBytes;
  static constexpr int kStages = BR == 64 ? 3 : 2;
  // partial sums: batch row m, weight row r at m * 128 + r; this rank's in the
  // ring once that is idle, the others' in a place of their own
  static constexpr uint32_t kRowBytes = kBM * 4;
  static constexpr uint32_t kOffRecv = kStages * kStageBytes;
  static constexpr size_t kSmemBytes = kOffRecv + (BR + kMaxRanks) * kRowBytes + 1024;
  static constexpr int kBufs = 2;  // of kFewStep x BR columns
  static constexpr uint32_t kTmemCols = kBufs * kFewStep * BR;
  static constexpr int kScales = BR + 4;  // the batch's, then the weight block's
  static_assert(kCtas * kTmemCols <= 512, "tensor memory columns");
  static_assert(kCtas * (kSmemBytes + kFewScaleSlots * kScaleBlocks * kScales * 4 + 1536) <= 227 * 1024,
                "shared memory");
  static_assert(BR * kRowBytes <= kOffRecv, "the partial tile fits the ring");
};
static_assert(kScaleBlocks % kFewStep == 0, "a stage's scales share a slot");

template <int BR>
__global__ void __launch_bounds__(kFewThreads, FewPlan<BR>::kCtas)
    block_gemm_few_kernel(const __grid_constant__ CUtensorMap map_a,
                          const __grid_constant__ CUtensorMap map_b, const TileArgs g) {
  using P = FewPlan<BR>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[P::kStages];
  __shared__ __align__(8) uint64_t empty_bar[P::kStages];
  __shared__ __align__(8) uint64_t acc_full[P::kBufs];
  __shared__ __align__(8) uint64_t acc_empty[P::kBufs];
  __shared__ __align__(8) uint64_t scale_full[kFewScaleSlots];
  __shared__ __align__(8) uint64_t scale_empty[kFewScaleSlots];
  __shared__ __align__(8) uint64_t recv_bar;
  __shared__ __align__(16) float scales[kFewScaleSlots][kScaleBlocks][P::kScales];
  __shared__ uint32_t tmem_base_slot;
  __shared__ uint32_t abort_flag;
  __shared__ uint32_t issued, committed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  const int n0 = blockIdx.x * kBM, S = (int)gridDim.z;
  const int rank = (int)tc::cluster_ctarank();  // = blockIdx.z: the cluster spans z
  const int kb0 = (int)((int64_t)g.KB * rank / S), kb1 = (int)((int64_t)g.KB * (rank + 1) / S);
  const int steps = (kb1 - kb0 + kFewStep - 1) / kFewStep;
  // this rank's share of the batch rows
  const int share = (g.M + S - 1) / S;
  const int m_lo = min(rank * share, g.M), m_hi = min(m_lo + share, g.M);
  volatile uint32_t* abortp = &abort_flag;

  if (threadIdx.x == 0) {
    tc::prefetch_map(&map_a);
    tc::prefetch_map(&map_b);
    for (int s = 0; s < P::kStages; ++s) {
      mbar_init(smem_addr(&full_bar[s]), 1);
      mbar_init(smem_addr(&empty_bar[s]), 1);
    }
    for (int b = 0; b < P::kBufs; ++b) {
      mbar_init(smem_addr(&acc_full[b]), 1);
      mbar_init(smem_addr(&acc_empty[b]), 4);
    }
    for (int s = 0; s < kFewScaleSlots; ++s) {
      mbar_init(smem_addr(&scale_full[s]), 32);
      mbar_init(smem_addr(&scale_empty[s]), 4);
    }
    mbar_init(smem_addr(&recv_bar), 1);
    abort_flag = 0;
    issued = committed = 0;
    mbar_init_fence();
    mbar_arrive_expect_tx(smem_addr(&recv_bar), (uint32_t)((S - 1) * (m_hi - m_lo)) * P::kRowBytes);
  }
  if (warp == 5) tc::tmem_alloc(smem_addr(&tmem_base_slot), P::kTmemCols);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (S > 1) tc::cluster_arrive();  // this CTA's barriers are ready for the others' copies
  const uint32_t tmem = tmem_base_slot;
  griddep_wait();
  griddep_launch_dependents();

  if (warp == 4) {
    const bool leader = tc::elect_one();
    uint32_t s = 0, parity = 1;
    for (int i = 0; i < steps; ++i) {
      const bool ok = tc::wait_or_abort(smem_addr(&empty_bar[s]), parity, abortp, g.wait_limit);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (leader) {
        const int kb = kb0 + i * kFewStep, n = min(kFewStep, kb1 - kb);
        uint32_t st = base + s * P::kStageBytes;
        const uint32_t bar = smem_addr(&full_bar[s]);
        mbar_arrive_expect_tx(bar, (uint32_t)n * P::kBlockBytes);
        for (int j = 0; j < n; ++j, st += P::kBlockBytes) {
          tc::tma_load_2d(st, &map_b, (kb + j) * kBK, n0, bar);
          tc::tma_load_2d(st + kBoxBytes, &map_a, (kb + j) * kBK, 0, bar);
        }
        ++issued;
      }
      if (++s == P::kStages) s = 0, parity ^= 1;
    }
  } else if (warp == 5) {
    const bool leader = tc::elect_one();
    constexpr uint32_t idesc = tc::f8_idesc(kBM, BR);
    const uint32_t lo0 = tc::sw128_lo(base), hi = tc::sw128_hi();
    uint32_t s = 0, parity = 0, buf = 0, buf_parity = 1;
    for (int i = 0; i < steps; ++i) {
      const bool ok = tc::wait_or_abort(smem_addr(&full_bar[s]), parity, abortp, g.wait_limit) &&
                      tc::wait_or_abort(smem_addr(&acc_empty[buf]), buf_parity, abortp, g.wait_limit);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc::fence_after();
      if (leader) {
        uint32_t lo = lo0 + s * (P::kStageBytes >> 4), d = tmem + buf * kFewStep * BR;
        const int n = min(kFewStep, kb1 - kb0 - i * kFewStep);
        for (int j = 0; j < n; ++j, lo += P::kBlockBytes >> 4, d += BR) {
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            tc::mma_f8(d, lo + 2 * kk, lo + (kBoxBytes >> 4) + 2 * kk, hi, idesc, kk != 0);
        }
        tc::commit(smem_addr(&empty_bar[s]));
        tc::commit(smem_addr(&acc_full[buf]));
        ++committed;
      }
      __syncwarp();
      if (++s == P::kStages) s = 0, parity ^= 1;
      if (++buf == P::kBufs) buf = 0, buf_parity ^= 1;
    }
  } else if (warp == 6) {
    uint32_t s = 0, parity = 1;
    constexpr int kNA = (BR + 31) / 32;
    const float *pa[kNA], *pb = nullptr;
#pragma unroll
    for (int i = 0; i < kNA; ++i) {
      const int row = lane + 32 * i;
      pa[i] = row < g.M && row < BR ? g.sa + (int64_t)row * g.sa_row + kb0 * g.sa_kb : nullptr;
    }
    if (lane == 0) pb = g.sb + (int64_t)blockIdx.x * g.sb_row + kb0 * g.sb_kb;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int j = (kb - kb0) % kScaleBlocks;
      if (j == 0) {
        const bool ok = tc::wait_or_abort(smem_addr(&scale_empty[s]), parity, abortp, g.wait_limit);
        if (!__all_sync(0xffffffffu, ok)) break;
      }
#pragma unroll
      for (int i = 0; i < kNA; ++i)
        if (pa[i] != nullptr) {
          tc::cp_async_4(smem_addr(&scales[s][j][lane + 32 * i]), pa[i]);
          pa[i] += g.sa_kb;
        }
      if (pb != nullptr) {
        tc::cp_async_4(smem_addr(&scales[s][j][BR]), pb);
        pb += g.sb_kb;
      }
      if (j == kScaleBlocks - 1 || kb == kb1 - 1) {
        tc::cp_async_arrive(smem_addr(&scale_full[s]));
        if (++s == kFewScaleSlots) s = 0, parity ^= 1;
      }
    }
    tc::cp_async_wait_all();
  } else {
    const int row = warp * 32 + lane;
    const uint32_t tm_lane = tmem + ((uint32_t)(warp * 32) << 16);
    uint32_t buf = 0, buf_parity = 0, slot = 0, slot_parity = 0;
    float2 acc[BR / 2];
#pragma unroll
    for (int c = 0; c < BR / 2; ++c) acc[c] = make_float2(0.f, 0.f);
    bool ok = true;
    for (int kb = kb0; kb < kb1; kb += kFewStep) {
      const int j0 = (kb - kb0) % kScaleBlocks;
      ok = (j0 != 0 || tc::wait_or_abort(smem_addr(&scale_full[slot]), slot_parity, abortp, g.wait_limit)) &&
           tc::wait_or_abort(smem_addr(&acc_full[buf]), buf_parity, abortp, g.wait_limit);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc::fence_after();
#pragma unroll
      for (int j = 0; j < kFewStep; ++j) {
        if (kb + j >= kb1) break;
        const float* sc = scales[slot][j0 + j];
        const float2 sw = make_float2(sc[BR], sc[BR]);
#pragma unroll
        for (int c = 0; c < BR; c += 16) {
          if (c >= g.M) break;
          uint32_t v[16];
          tc::tmem_ld_async(tm_lane + (buf * kFewStep + j) * BR + (uint32_t)c, v);
          float2 f[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 q = *reinterpret_cast<const float4*>(sc + c + 4 * i);
            f[2 * i] = __fmul2_rn(make_float2(q.x, q.y), sw);
            f[2 * i + 1] = __fmul2_rn(make_float2(q.z, q.w), sw);
          }
          tc::tmem_ld_wait(v);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            acc[c / 2 + i] = __ffma2_rn(
                make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), f[i],
                acc[c / 2 + i]);
        }
      }
      tc::fence_before();
      __syncwarp();
      tc::arrive_if(lane == 0, smem_addr(&acc_empty[buf]));
      if (++buf == P::kBufs) buf = 0, buf_parity ^= 1;
      if (j0 + kFewStep == kScaleBlocks) {
        tc::arrive_if(lane == 0, smem_addr(&scale_empty[slot]));
        if (++slot == kFewScaleSlots) slot = 0, slot_parity ^= 1;
      }
    }
    auto store = [&](int m, float v) {
      if (n0 + row >= g.N) return;
      const int64_t at = (int64_t)m * g.ldd + n0 + row;
      if (g.d_f32) {
        float* p = static_cast<float*>(g.d) + at;
        *p = g.accumulate ? *p + v : v;
      } else {
        static_cast<uint16_t*>(g.d)[at] = (uint16_t)(f2_to_bf2(make_float2(v, 0.f)) & 0xffffu);
      }
    };
    if (S == 1) {
      if (ok) {
#pragma unroll
        for (int c = 0; c < BR; ++c)
          if (c < g.M) store(c, c & 1 ? acc[c / 2].y : acc[c / 2].x);
      }
    } else {
      // the last accumulator was complete, so every copy and MMA of the ring is done
      float* part = reinterpret_cast<float*>(smem_raw + (base - smem_addr(smem_raw)));
      asm volatile("barrier.cta.sync 1, 128;" ::: "memory");  // all four warps are past the ring
#pragma unroll
      for (int c = 0; c < BR; ++c)
        if (c < g.M) part[c * kBM + row] = c & 1 ? acc[c / 2].y : acc[c / 2].x;
      tc::fence_async_smem();
      asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
      tc::cluster_wait();  // every CTA's barriers exist
      const uint32_t recv = base + P::kOffRecv;
      // also after an abort, so that every copy between the ranks is counted and
      // over before one of them ends
      if (threadIdx.x == 0) {
        for (int q = 0; q < S; ++q) {
          const int lo = min(q * share, g.M), n = min(lo + share, g.M) - lo;
          if (q == rank || n == 0) continue;
          tc::bulk_s2c(tc::mapa(recv + (uint32_t)(rank * share) * P::kRowBytes, (uint32_t)q),
                       smem_addr(part + lo * kBM), (uint32_t)n * P::kRowBytes,
                       tc::mapa(smem_addr(&recv_bar), (uint32_t)q));
        }
      }
      ok = __all_sync(0xffffffffu, tc::wait_or_abort(smem_addr(&recv_bar), 0u, abortp, g.wait_limit)) && ok;
      if (!ok) mbar_wait_bounded(smem_addr(&recv_bar), 0u, kDrainLimitCycles);
      __syncwarp();
      tc::cluster_arrive();  // what the others sent has arrived
      if (ok) {
        const float* in = reinterpret_cast<const float*>(smem_raw + (recv - smem_addr(smem_raw)));
        for (int m = m_lo; m < m_hi; ++m) {
          float v = 0.f;
#pragma unroll
          for (int q = 0; q < kMaxRanks; ++q)
            if (q < S)
              v += q == rank ? part[m * kBM + row] : in[(q * share + m - m_lo) * kBM + row];
          store(m, v);
        }
      }
    }
  }
  __syncwarp();
  if (S > 1) {
    if (warp >= 4) {
      tc::cluster_wait();
      tc::cluster_arrive();
    }
    tc::cluster_wait();  // what this CTA sent has arrived: its memory may go
  }
  tc::fence_before();
  __syncthreads();
  if (*abortp) {
    if (threadIdx.x == 0) {
      atomicCAS(&g_block_gemm_device_error, kDevErrNone, kDevErrBulkWaitTimeout);
      const uint32_t n = issued, m = committed;  // copies and MMAs in flight finish first
      for (uint32_t k = n > P::kStages ? n - P::kStages : 0; k < n; ++k)
        mbar_wait_bounded(smem_addr(&full_bar[k % P::kStages]), (k / P::kStages) & 1u,
                          kDrainLimitCycles);
      if (m > 0)
        mbar_wait_bounded(smem_addr(&acc_full[(m - 1) % P::kBufs]), ((m - 1) / P::kBufs) & 1u,
                          kDrainLimitCycles);
      // and parts of a rank that gave up later than this one: nothing counts them now
      for (const long long t0 = clock64(); clock64() - t0 < kDrainLimitCycles / 100;) {
      }
    }
    __syncthreads();
  }
  if (warp == 5) tc::tmem_dealloc(tmem, P::kTmemCols);
}

// Ranks of the split: the most with which all tiles still run at once, a full
// stage a rank at least. One cluster more than fit doubles the time (1 x 5120 x
// 5120: 6 ranks 16 us, 7 ranks 20 us).
template <int BR>
int few_ranks(int64_t N, int64_t KB) {
  static std::atomic<int> cache[64][kMaxRanks + 1];
  const int64_t tiles = (N + kBM - 1) / kBM;
  // the occupancy query counts one CTA an SM for a kernel that allocates tensor
  // memory; kCtas of them do run together
  auto fit = [&](int S) {
    return FewPlan<BR>::kCtas *
           max_clusters(reinterpret_cast<const void*>(block_gemm_few_kernel<BR>), kFewThreads,
                        FewPlan<BR>::kSmemBytes, dim3(1, 1, (unsigned)S), cache);
  };
  int S = kMaxRanks;
  while (S > 1 && (S * kFewStep > KB || fit(S) < tiles)) --S;
  return S;
}

template <int BR>
cudaError_t launch_few(const BlockGemmArgs& p, const TileArgs& g, int S, cudaStream_t stream) {
  const cudaError_t e = cudaFuncSetAttribute(block_gemm_few_kernel<BR>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)FewPlan<BR>::kSmemBytes);
  if (e != cudaSuccess) return e;
  CUtensorMap map_a, map_b;
  if (!tc::encode_e4m3_operand(&map_a, p.a, p.M, p.K, p.lda, BR) ||
      !tc::encode_e4m3_operand(&map_b, p.b, p.N, p.K, p.ldb, kBM))
    return cudaErrorInvalidValue;
  return launch_cluster(block_gemm_few_kernel<BR>,
                        dim3((unsigned)((p.N + kBM - 1) / kBM), 1, (unsigned)S), 1, kFewThreads,
                        FewPlan<BR>::kSmemBytes, stream, map_a, map_b, g);
}

// The 128-wide tiles of `g`, with K split where they leave SMs idle.
template <bool SB_ROWS, bool VEC>
cudaError_t launch_narrow(const BlockGemmArgs& p, const TileArgs& g, cudaStream_t stream) {
  const int S = split_ranks<SB_ROWS, VEC>(g);
  return S > 1 ? launch_split<SB_ROWS, VEC>(p, g, S, stream) : launch_tiled<128, SB_ROWS, VEC>(p, g, stream);
}

// Tiles of rows x 256 columns over `units` CTAs or pairs: `last` of them in a round
// that is not full. Where those are at most half a round, they become a launch of
// their own of 128 x 128 tiles, which takes half as long or (split) less, from
// kCutBlocks K blocks on: 5120 x 4096 x 8192 with a scale a row (4.3 rounds) 309 ->
// 292 us, 5000 x 1024 x 4096 (1.1 rounds) 47 -> 42; 2048 x 2816 x 2048 28.6 -> 29.6.
struct Rounds {
  int tiles_m, tiles, last, halves;  // halves: the time, in half rounds
  bool cut;
  Rounds(const TileArgs& g, int rows, int units)
      : tiles_m((g.M + rows - 1) / rows), tiles(tiles_m * ((g.N + 255) / 256)), last(tiles % units),
        cut(last > 0 && 2 * last <= units && g.KB >= kCutBlocks) {
    halves = 2 * (tiles / units) + (last == 0 ? 0 : cut ? 1 : 2);
  }
};

// 256-wide tiles while every SM gets one, else 128-wide ones. Pairs unless their
// taller tiles need more rounds (a round takes either the same). A pair moves two
// thirds of the bytes through shared memory; the SM's clock under the power cap
// gains more by it than a short run shows, us of single CTAs against pairs over
// seconds: 16384 x 7168 x 7168 889 -> 849, 4096 x 4096 x 4096 86 -> 80, 5120 x 4096 x
// 8208 with a scale a row 316 -> 297; in short runs 5120 x 5120 x 8192 300 -> 292.
template <bool SB_ROWS, bool VEC>
cudaError_t launch_large(const BlockGemmArgs& p, TileArgs g, cudaStream_t stream) {
  const int sms = device_sm_count(), pairs = pair_clusters<SB_ROWS, VEC>();
  const Rounds one(g, kBM, sms), two(g, 2 * kBM, pairs > 0 ? pairs : 1);
  g.band = kBand, g.tail = -1;
  if (one.tiles < sms) {
    g.tiles_m = one.tiles_m, g.tiles_n = (g.N + 127) / 128;
    g.tiles = g.tiles_m * g.tiles_n;
    return launch_narrow<SB_ROWS, VEC>(p, g, stream);
  }
  const bool pair = pairs > 0 && two.halves <= one.halves;
  const Rounds& r = pair ? two : one;
  g.tiles_m = r.tiles_m, g.tiles_n = (g.N + 255) / 256;
  g.tiles = r.cut ? r.tiles - r.last : r.tiles;
  if (pair) g.band = kBand / 2;
  const cudaError_t e = pair ? launch_pairs<SB_ROWS, VEC>(p, g, pairs, stream)
                             : launch_tiled<256, SB_ROWS, VEC>(p, g, stream);
  if (e != cudaSuccess || !r.cut) return e;
  g.parts = pair ? 4 : 2;
  g.tail = g.tiles, g.tiles = g.parts * r.last;
  return launch_narrow<SB_ROWS, VEC>(p, g, stream);
}

}  // namespace

cudaError_t device_error_block_gemm(int* out, bool clear) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_block_gemm_device_error, sizeof(int));
  if (e != cudaSuccess) return e;
  if (clear && v != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_block_gemm_device_error, &zero, sizeof(int));
  }
  *out = v;
  return e;
}

int block_gemm(const BlockGemmArgs& p, cudaStream_t stream, const char** why) {
  TileArgs g{};
  g.sa = p.sa, g.sa_row = p.sa_row, g.sa_kb = p.sa_kb;
  g.sb = p.sb, g.sb_row = p.sb_row, g.sb_kb = p.sb_kb;
  g.d = p.d, g.ldd = p.ldd;
  g.M = (int)p.M, g.N = (int)p.N, g.KB = (int)((p.K + kBK - 1) / kBK);
  g.d_f32 = p.d_f32, g.accumulate = p.accumulate;
  g.wait_limit = p.wait_limit;
  const int columns = p.M <= 16 ? 16 : p.M <= 32 ? 32 : 64;
  const int ranks = p.b_rows || p.M > kFewRows ? 0
                    : columns == 16            ? few_ranks<16>(p.N, g.KB)
                    : columns == 32            ? few_ranks<32>(p.N, g.KB)
                                               : few_ranks<64>(p.N, g.KB);
  cudaError_t e;
  if (ranks > (p.M <= kFewSplitRows ? 0 : 1)) {
    e = columns == 16   ? launch_few<16>(p, g, ranks, stream)
        : columns == 32 ? launch_few<32>(p, g, ranks, stream)
                        : launch_few<64>(p, g, ranks, stream);
  } else {
    const bool vec = aligned_rows_host(p.d, p.ldd * (p.d_f32 ? 4 : 2), 32) && p.N % (p.d_f32 ? 8 : 16) == 0;
    e = p.b_rows ? (vec ? launch_large<true, true>(p, g, stream) : launch_large<true, false>(p, g, stream))
                 : (vec ? launch_large<false, true>(p, g, stream) : launch_large<false, false>(p, g, stream));
  }
  if (e != cudaSuccess) {
    *why = cudaGetErrorString(e);
    return CUTIE_ERR_CUDA;
  }
  return CUTIE_OK;
}

}  // namespace cutie
