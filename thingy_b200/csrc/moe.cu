// A whole mixture-of-experts layer for at most 64 tokens in one kernel (sm_100a):
//
//   logits = x R^T;  the top k of E experts a token, weights w (softmax or sigmoid, renormalized)
//   g, u = dequant(q) dequant(w13[e])^T;  h = silu(g) u;  (qh, sh) = 1 x 128 cast of h
//   out[t] = sum_j w[t, j] dequant(qh) dequant(w2[e_j])^T
//
// Everything is e4m3 with fp32 scales as in the block-scaled product
// (block_gemm.cu): 1 x 128 groups of the activations, 128 x 128 blocks of the
// weights, the sum of each 128-wide K block on the tensor cores and the sum
// over blocks in fp32 registers.
//
// Bound: memory; the weights of the experts that some token chose are read
// once, and a token's share of the arithmetic is small. So the weights are
// the 128-row side of the MMA and the expert's tokens its N side (a multiple
// of 16), and the kernel is organised around one stream of weight tiles a SM:
// a persistent cooperative grid, one CTA an SM, walks a list of equal units
// (item, K block) of 32 KB of weights. An item is 128 gate rows with their
// 128 up rows, or 256 rows of the down weight, of one expert; units are dealt
// to the CTAs in contiguous runs, so an item may be split over K between
// neighbours. A split item's partial sums go to the workspace, and the CTA
// that arrives last adds them in the order of K (the result does not depend
// on who that is) and finishes the item.
//
// Three grid barriers: logits complete (and, for many tokens, the choices),
// hidden rows complete, down products complete. The weight stream does not
// stop at the second: its TMA thread needs only the choices, and fills the
// ring with down tiles while the last hidden rows are finished.
//
// Warps: 0-7 the outer sums (warps 0-3 the first 128 rows of an item, 4-7 the
// second, a row a thread) and the epilogues; 8 the weight tiles (TMA); 9 the
// tokens' rows (TMA gather of 4 rows for the first product, boxes of 16 hidden
// rows for the second); 10 the MMAs; 11 the products of the scales.
#include "cutie.h"
#include "launch.cuh"
#include "tcgen05.cuh"

namespace cutie {

static __device__ int g_moe_device_error = 0;

namespace {

using tc::kLayoutSw128;
using tc::smem_desc;

constexpr int kMoeThreads = 384, kMoeWarps = 12, kEpiThreads = 256;
constexpr uint32_t kBox = 128 * 128;  // a 128-row weight tile of one K block
constexpr int kBufs = 4;              // accumulator buffers in tensor memory
constexpr int kXStride = 132;         // floats between columns of the exchange
constexpr int kMaxE = kMoeMaxExperts, kMaxK = kMoeMaxTopK;

template <int NMAX>
struct MoePlan {
  static constexpr uint32_t kStageBytes = 2 * kBox + NMAX * 128;
  static constexpr int kStages = NMAX == 16 ? 6 : NMAX == 32 ? 5 : 4;
  static constexpr uint32_t kXBytes = NMAX * kXStride * 4;
  static constexpr size_t kSmemBytes = kStages * kStageBytes + kXBytes + 1024;
  static constexpr uint32_t kTmemCols = kBufs * 2 * NMAX;
  static constexpr int kPairs = NMAX * kMaxK;
  static_assert(kStageBytes % 1024 == 0, "swizzled tiles start on 1 KB");
};

// Units of a phase dealt in runs of `per`; KB units an item.
struct Deal {
  int per, units, KB;
  __device__ Deal(int items, int kb) : units(items * kb), KB(kb) {
    per = (units + (int)gridDim.x - 1) / (int)gridDim.x;
  }
  __device__ int begin() const { return min(per * (int)blockIdx.x, units); }
  __device__ int end() const { return min(per * ((int)blockIdx.x + 1), units); }
};

template <int NMAX>
struct MoeShared {
  uint64_t full[8], empty[8], acc_full[kBufs], acc_empty[kBufs], scale_full[kBufs];
  float scales[kBufs][2][NMAX];
  uint64_t mask[kMaxE];       // tokens of an expert
  float weight[MoePlan<NMAX>::kPairs];
  uint16_t ids[MoePlan<NMAX>::kPairs];     // expert of (token, slot)
  uint16_t row_of[MoePlan<NMAX>::kPairs];  // its hidden row: experts in order, tokens in order
  uint8_t token_at[MoePlan<NMAX>::kPairs]; // token of a hidden row
  uint16_t first_row[kMaxE];
  uint16_t active[kMaxE < MoePlan<NMAX>::kPairs ? kMaxE : MoePlan<NMAX>::kPairs];
  int n_active;
  uint32_t tmem_base, abort_flag, last, issued_w, issued_a, committed;
  uint64_t target;  // the grid barrier's count at the next barrier
};

__device__ __forceinline__ bool wait_or_abort(uint32_t bar, uint32_t parity,
                                              volatile uint32_t* abort_flag) {
  if (mbar_test(bar, parity)) return true;
  const long long t0 = clock64();
  while (!*abort_flag && clock64() - t0 <= kWaitLimitCycles)
    if (mbar_try_wait(bar, parity)) return true;
  *abort_flag = 1u;
  return false;
}

// ------------------------------------------------------------------ grid barrier
//
// A 64-bit count in the workspace, zero before its first use. Every CTA adds
// one a barrier, every launch passes the same number of barriers, so the
// count is a multiple of the grid's size between launches and needs no reset.

__device__ __forceinline__ uint64_t barrier_arrive(uint64_t* count) {
  __threadfence();
  asm volatile("fence.proxy.async;" ::: "memory");  // hidden rows are read by TMA
  return atomicAdd(reinterpret_cast<unsigned long long*>(count), 1ull);
}

__device__ __forceinline__ bool barrier_wait(const uint64_t* count, uint64_t target,
                                             volatile uint32_t* abort_flag) {
  const long long t0 = clock64();
  for (;;) {
    uint64_t v;
    asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(count) : "memory");
    if (v >= target) break;
    if (clock64() - t0 > kWaitLimitCycles) {
      *abort_flag = 1u;
      return false;
    }
  }
  asm volatile("fence.proxy.async;" ::: "memory");
  return true;
}

// Loads of what other CTAs wrote in this launch: from L2, and never moved
// across the waits that order them (the plain intrinsics may be).
__device__ __forceinline__ float ld_l2(const float* p) {
  float v;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ int ld_l2(const int* p) {
  int v;
  asm volatile("ld.global.cg.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_l2(const float4* p) {
  float4 v;
  asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// ------------------------------------------------------------------ router

// Partial logits of 4 experts x 8 tokens over one share of the columns, a warp
// a job; the lanes split the columns, so a job ends with 32 sums over 32
// lanes, folded so that lane l keeps sum l.
__device__ __forceinline__ void router_job(const MoeArgs& g, int job, int lane) {
  const int eg = (g.E + 3) / 4, tg = (g.T + 7) / 8, chunks = (g.H + 255) / 256;
  const int e0 = 4 * (job % eg), t0 = 8 * ((job / eg) % tg), s = job / (eg * tg);
  const int ne = min(4, g.E - e0), nt = min(8, g.T - t0);
  const int c0 = chunks * s / g.splits, c1 = chunks * (s + 1) / g.splits;
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = 0.f;
  for (int c = c0; c < c1; ++c) {
    const int col = c * 256 + lane * 8;
    if (col >= g.H) continue;
    float2 w[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 u = i < ne ? ld_keep(g.router + (int64_t)(e0 + i) * g.H + col) : make_uint4(0, 0, 0, 0);
      w[i][0] = bf2_to_f2(u.x), w[i][1] = bf2_to_f2(u.y), w[i][2] = bf2_to_f2(u.z), w[i][3] = bf2_to_f2(u.w);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j >= nt) break;
      const uint4 u = ld_keep(g.x + (int64_t)(t0 + j) * g.ldx + col);
      const float2 x[4] = {bf2_to_f2(u.x), bf2_to_f2(u.y), bf2_to_f2(u.z), bf2_to_f2(u.w)};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a = v[i * 8 + j];
#pragma unroll
        for (int q = 0; q < 4; ++q) a = __fmaf_rn(w[i][q].x, x[q].x, a), a = __fmaf_rn(w[i][q].y, x[q].y, a);
        v[i * 8 + j] = a;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = up ? v[i + o] : v[i], send = up ? v[i] : v[i + o];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  const int i = lane >> 3, j = lane & 7;
  if (i < ne && j < nt) g.logits[((int64_t)s * g.T + t0 + j) * g.E + e0 + i] = v[0];
}

// Order of floats as unsigned; NaN lowest but one, 0 is "none".
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __float_as_uint(f);
  return f != f ? 1u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// One token's choice by one warp: k rounds of a warp maximum, ties to the
// lowest expert. Lane j < k returns with (*id, *w) of slot j.
__device__ __forceinline__ void choose(const MoeArgs& g, int t, int lane, int* id, float* w) {
  constexpr int NQ = kMaxE / 32;
  float l[NQ];
  uint32_t key[NQ];
  float m = -INFINITY;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int e = q * 32 + lane;
    l[q] = 0.f;
    if (e < g.E) {
      for (int s = 0; s < g.splits; ++s) l[q] += ld_l2(g.logits + ((int64_t)s * g.T + t) * g.E + e);
      m = fmaxf(m, l[q]);
    }
  }
  float z = 1.f;
  const bool softmax = g.scoring == 0;
  if (softmax) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    z = 0.f;
#pragma unroll
    for (int q = 0; q < NQ; ++q)
      if (q * 32 + lane < g.E) z += expf(l[q] - m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
  }
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int e = q * 32 + lane;
    key[q] = 0;
    if (e < g.E) {
      // without a bias the choice goes by the logits, which the scores grow
      // with (and saturate against); with one by the biased scores
      float sel = l[q];
      if (g.bias != nullptr)
        sel = (softmax ? expf(l[q] - m) / z : 1.f / (1.f + expf(-l[q]))) + g.bias[e];
      key[q] = ordered(sel);
    }
  }
  int my_id = 0;
  float my_l = 0.f;
  for (int j = 0; j < g.k; ++j) {
    uint32_t best = 0, at = 0xffffffffu;
    float bl = 0.f;
#pragma unroll
    for (int q = 0; q < NQ; ++q)
      if (key[q] > best) best = key[q], at = (uint32_t)(q * 32 + lane), bl = l[q];
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const uint32_t e = __reduce_min_sync(0xffffffffu, best == top ? at : 0xffffffffu);
    const float le = __shfl_sync(0xffffffffu, bl, (int)(e & 31u));
#pragma unroll
    for (int q = 0; q < NQ; ++q)
      if ((uint32_t)(q * 32 + lane) == e) key[q] = 0;
    if (lane == j) my_id = (int)e, my_l = le;
  }
  float p = 0.f;
  if (lane < g.k) p = softmax ? expf(my_l - m) : 1.f / (1.f + expf(-my_l));
  float den = softmax ? z : 1.f;
  if (g.renormalize) {
    den = p;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
  }
  *id = my_id;
  *w = p / den * g.routed_scale;
}

// ------------------------------------------------------------------ epilogues

__device__ __forceinline__ void epi_sync() { asm volatile("barrier.cta.sync 1, 256;" ::: "memory"); }

// Sums of a split item: this CTA's partial to the workspace; true in the CTA
// that arrives last, with the whole sums in acc. n columns, thread = row.
template <int NMAX>
__device__ __forceinline__ bool join(const MoeArgs& g, MoeShared<NMAX>& sh, const Deal& deal, int item,
                                     int* counters, int n, float (&acc)[NMAX]) {
  const int tid = threadIdx.x;
  const int first = item * deal.KB, c0 = first / deal.per, c1 = (first + deal.KB - 1) / deal.per;
  // a run that begins inside the item keeps its part in slot 0, one that ends in it in slot 1
  const int mine = first < deal.per * (int)blockIdx.x ? 0 : 1;
  float* p = g.partial + (int64_t)(blockIdx.x * 2 + mine) * NMAX * 256 + tid;
#pragma unroll
  for (int c = 0; c < NMAX; ++c)
    if (c < n) __stcg(p + c * 256, acc[c]);
  __threadfence();
  epi_sync();
  if (tid == 0) {
    const int old = atomicAdd(counters + item, 1);
    __threadfence();
    sh.last = old == c1 - c0;
  }
  epi_sync();
  if (!sh.last) return false;
#pragma unroll
  for (int c = 0; c < NMAX; ++c) acc[c] = 0.f;
  for (int b = c0; b <= c1; ++b) {
    const float* o = g.partial + (int64_t)(b * 2 + (first < deal.per * b ? 0 : 1)) * NMAX * 256 + tid;
#pragma unroll
    for (int c = 0; c < NMAX; ++c)
      if (c < n) acc[c] += ld_l2(o + c * 256);
  }
  return true;
}

// The outer sums of this CTA's run of one phase; finish(item, n, row0, acc) at
// each item that is complete here.
template <int NMAX, class F>
__device__ __forceinline__ void sum_phase(const MoeArgs& g, MoeShared<NMAX>& sh, const Deal& deal,
                                          int groups, int* counters, uint32_t tmem, uint32_t& it,
                                          volatile uint32_t* abortp, F finish) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2;
  const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(half * NMAX);
  float acc[NMAX];
  int item = -1, n = 0, row0 = 0, begun = 0;
  const int u1 = deal.end();
  for (int u = deal.begin(); u < u1; ++u, ++it) {
    const int kb = u % deal.KB;
    if (item < 0) {
      item = u / deal.KB, begun = kb;
      const int e = sh.active[item / groups];
      n = __popcll(sh.mask[e]), row0 = sh.first_row[e];
#pragma unroll
      for (int c = 0; c < NMAX; ++c) acc[c] = 0.f;
    }
    const uint32_t buf = it % kBufs, use = it / kBufs;
    const bool ok = wait_or_abort(smem_addr(&sh.acc_full[buf]), use & 1u, abortp) &&
                    wait_or_abort(smem_addr(&sh.scale_full[buf]), use & 1u, abortp);
    if (__all_sync(0xffffffffu, ok)) {
      tc::fence_after();
#pragma unroll
      for (int c = 0; c < NMAX; c += 16) {
        if (c >= n) break;
        uint32_t v[16];
        tc::tmem_ld16_async(lane_base + buf * 2 * NMAX + (uint32_t)c, v);
        const float4* sc = reinterpret_cast<const float4*>(&sh.scales[buf][half][c]);
        const float4 f[4] = {sc[0], sc[1], sc[2], sc[3]};
        tc::tmem_ld_wait(v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[c + 4 * i] = __fmaf_rn(__uint_as_float(v[4 * i]), f[i].x, acc[c + 4 * i]);
          acc[c + 4 * i + 1] = __fmaf_rn(__uint_as_float(v[4 * i + 1]), f[i].y, acc[c + 4 * i + 1]);
          acc[c + 4 * i + 2] = __fmaf_rn(__uint_as_float(v[4 * i + 2]), f[i].z, acc[c + 4 * i + 2]);
          acc[c + 4 * i + 3] = __fmaf_rn(__uint_as_float(v[4 * i + 3]), f[i].w, acc[c + 4 * i + 3]);
        }
      }
      tc::fence_before();
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_addr(&sh.acc_empty[buf]));
    if (kb == deal.KB - 1 || u == u1 - 1) {
      const bool whole = begun == 0 && kb == deal.KB - 1;
      if (whole || join<NMAX>(g, sh, deal, item, counters, n, acc)) finish(item, n, row0, acc);
      item = -1;
    }
  }
}

// ------------------------------------------------------------------ kernel

template <int NMAX>
__global__ void __launch_bounds__(kMoeThreads, 1)
    moe_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_w13,
               const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w2,
               const MoeArgs g) {
  using P = MoePlan<NMAX>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(16) MoeShared<NMAX> sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
  float* exchange = reinterpret_cast<float*>(smem_raw + (base - smem_addr(smem_raw)) +
                                             P::kStages * P::kStageBytes);
  volatile uint32_t* abortp = &sh.abort_flag;
  const int IG = g.I / 128, KB1 = g.H / 128, HB = (g.H + 255) / 256, KB2 = IG;

  if (tid == 0) {
    tc::prefetch_map(&map_q);
    tc::prefetch_map(&map_w13);
    tc::prefetch_map(&map_h);
    tc::prefetch_map(&map_w2);
    for (int s = 0; s < P::kStages; ++s) {
      mbar_init(smem_addr(&sh.full[s]), 2);
      mbar_init(smem_addr(&sh.empty[s]), 1);
    }
    for (int b = 0; b < kBufs; ++b) {
      mbar_init(smem_addr(&sh.acc_full[b]), 1);
      mbar_init(smem_addr(&sh.acc_empty[b]), 8);
      mbar_init(smem_addr(&sh.scale_full[b]), 1);
    }
    sh.abort_flag = 0;
    sh.issued_w = sh.issued_a = sh.committed = 0;
    mbar_init_fence();
  }
  if (warp == 10) tc::tmem_alloc(smem_addr(&sh.tmem_base), P::kTmemCols);
  for (int e = tid; e < g.E; e += kMoeThreads) sh.mask[e] = 0;

  // ---- router: partial logits, and the counters of split items to zero
  for (int i = blockIdx.x * kMoeThreads + tid; i < g.n_counters; i += gridDim.x * kMoeThreads)
    g.counters[i] = 0;
  const int jobs = ((g.E + 3) / 4) * ((g.T + 7) / 8) * g.splits;
  for (int j = warp * gridDim.x + blockIdx.x; j < jobs; j += gridDim.x * kMoeWarps)
    router_job(g, j, lane);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (tid == 0) {
    const uint64_t old = barrier_arrive(g.barrier);
    sh.target = (old / gridDim.x + 1) * gridDim.x;
    barrier_wait(g.barrier, sh.target, abortp);
  }
  __syncthreads();
  uint64_t target = sh.target;

  // ---- choices: every CTA makes them all for few tokens; for more, each
  // token's is made once and read by all after another barrier
  const int pairs = g.T * g.k;
  const bool deal_tokens = g.deal_tokens;
  for (int t = deal_tokens ? warp * gridDim.x + blockIdx.x : warp; t < g.T;
       t += deal_tokens ? kMoeWarps * gridDim.x : kMoeWarps) {
    int id;
    float w;
    choose(g, t, lane, &id, &w);
    if (lane < g.k) {
      const int p = t * g.k + lane;
      if (deal_tokens || blockIdx.x == 0) g.ids[p] = id, g.weights[p] = w;
      if (!deal_tokens) sh.ids[p] = (uint16_t)id, sh.weight[p] = w;
    }
  }
  if (deal_tokens) {
    __syncthreads();
    target += gridDim.x;
    if (tid == 0) {
      barrier_arrive(g.barrier);
      barrier_wait(g.barrier, target, abortp);
    }
    __syncthreads();
    for (int p = tid; p < pairs; p += kMoeThreads) {
      sh.ids[p] = (uint16_t)ld_l2(g.ids + p);
      sh.weight[p] = ld_l2(g.weights + p);
    }
  }
  __syncthreads();
  for (int p = tid; p < pairs; p += kMoeThreads)
    atomicOr(reinterpret_cast<unsigned long long*>(&sh.mask[sh.ids[p] < g.E ? sh.ids[p] : 0]),
             1ull << (p / g.k));
  __syncthreads();
  if (warp == 0) {  // experts that some token chose, and where their rows begin
    int rows = 0, n = 0;
    for (int e0 = 0; e0 < g.E; e0 += 32) {
      const int e = e0 + lane, c = e < g.E ? __popcll(sh.mask[e]) : 0;
      int at = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += up;
      }
      const uint32_t some = __ballot_sync(0xffffffffu, c > 0);
      if (e < g.E) sh.first_row[e] = (uint16_t)(rows + at - c);
      if (c > 0) sh.active[n + __popc(some & ((1u << lane) - 1u))] = (uint16_t)e;
      rows += __shfl_sync(0xffffffffu, at, 31);
      n += __popc(some);
    }
    if (lane == 0) sh.n_active = n;
  }
  __syncthreads();
  for (int p = tid; p < pairs; p += kMoeThreads) {
    const int t = p / g.k, e = sh.ids[p] < g.E ? sh.ids[p] : 0;
    const int row = sh.first_row[e] + __popcll(sh.mask[e] & ((1ull << t) - 1ull));
    sh.row_of[p] = (uint16_t)row;
    sh.token_at[row] = (uint8_t)t;
  }
  __syncthreads();

  const uint32_t tmem = sh.tmem_base;
  const Deal d1(sh.n_active * IG, KB1), d2(sh.n_active * HB, KB2);
  const uint64_t hidden_target = target + gridDim.x, down_target = target + 2 * (uint64_t)gridDim.x;

  if (warp == 8) {
    // ---- weight tiles of both phases, without a stop between them
    if (lane == 0) {
      uint32_t it = 0;
      for (int phase = 0; phase < 2 && !*abortp; ++phase) {
        const Deal& d = phase == 0 ? d1 : d2;
        const int groups = phase == 0 ? IG : HB;
        for (int u = d.begin(); u < d.end(); ++u, ++it) {
          const int item = u / d.KB, kb = u - item * d.KB;
          const int e = sh.active[item / groups], grp = item % groups;
          const uint32_t s = it % P::kStages, use = it / P::kStages;
          if (use > 0 && !wait_or_abort(smem_addr(&sh.empty[s]), (use - 1u) & 1u, abortp)) break;
          const uint32_t st = base + s * P::kStageBytes, bar = smem_addr(&sh.full[s]);
          mbar_arrive_expect_tx(bar, 2 * kBox);
          if (phase == 0) {
            const int r = e * 2 * g.I + grp * 128;
            tc::tma_load_2d(st, &map_w13, kb * 128, r, bar);
            tc::tma_load_2d(st + kBox, &map_w13, kb * 128, r + g.I, bar);
          } else {
            const int r = e * g.H + grp * 256;
            tc::tma_load_2d(st, &map_w2, kb * 128, r, bar);
            tc::tma_load_2d(st + kBox, &map_w2, kb * 128, r + 128, bar);
          }
          sh.issued_w = it + 1;
        }
      }
    }
  } else if (warp == 9) {
    // ---- the tokens' rows
    if (lane == 0) {
      uint32_t it = 0;
      for (int phase = 0; phase < 2 && !*abortp; ++phase) {
        const Deal& d = phase == 0 ? d1 : d2;
        const int groups = phase == 0 ? IG : HB;
        if (phase == 1 && d.begin() < d.end() && !barrier_wait(g.barrier, hidden_target, abortp)) break;
        for (int u = d.begin(); u < d.end(); ++u, ++it) {
          const int item = u / d.KB, kb = u - item * d.KB;
          const int e = sh.active[item / groups];
          const int n = __popcll(sh.mask[e]), row0 = sh.first_row[e];
          const uint32_t s = it % P::kStages, use = it / P::kStages;
          if (use > 0 && !wait_or_abort(smem_addr(&sh.empty[s]), (use - 1u) & 1u, abortp)) break;
          const uint32_t st = base + s * P::kStageBytes + 2 * kBox, bar = smem_addr(&sh.full[s]);
          const int np = (n + 15) & ~15;
          mbar_arrive_expect_tx(bar, (uint32_t)np * 128u);
          if (phase == 0) {
            for (int c = 0; c < np; c += 4) {
              // columns past the expert's tokens repeat its last one and are not used
              const int last = row0 + n - 1;
              tc::tma_gather4(st + (uint32_t)c * 128u, &map_q, kb * 128,
                              sh.token_at[min(row0 + c, last)], sh.token_at[min(row0 + c + 1, last)],
                              sh.token_at[min(row0 + c + 2, last)],
                              sh.token_at[min(row0 + c + 3, last)], bar);
            }
          } else {
            for (int c = 0; c < np; c += 16)
              tc::tma_load_2d(st + (uint32_t)c * 128u, &map_h, kb * 128, row0 + c, bar);
          }
          sh.issued_a = it + 1;
        }
      }
    }
  } else if (warp == 10) {
    // ---- MMAs
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int phase = 0; phase < 2 && ok; ++phase) {
        const Deal& d = phase == 0 ? d1 : d2;
        const int groups = phase == 0 ? IG : HB;
        for (int u = d.begin(); u < d.end(); ++u, ++it) {
          const int e = sh.active[u / d.KB / groups];
          const int np = (__popcll(sh.mask[e]) + 15) & ~15;
          const uint32_t s = it % P::kStages, buf = it % kBufs;
          ok = wait_or_abort(smem_addr(&sh.full[s]), (it / P::kStages) & 1u, abortp) &&
               (it < kBufs ||
                wait_or_abort(smem_addr(&sh.acc_empty[buf]), (it / kBufs - 1u) & 1u, abortp));
          if (!ok) break;
          tc::fence_after();
          const uint32_t st = base + s * P::kStageBytes, idesc = tc::f8_idesc(128, np);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc::mma_f8(tmem + buf * 2 * NMAX + h * NMAX,
                         smem_desc(st + h * kBox + 32u * kk, 16, 1024, kLayoutSw128),
                         smem_desc(st + 2 * kBox + 32u * kk, 16, 1024, kLayoutSw128), idesc, kk != 0);
          tc::commit(smem_addr(&sh.empty[s]));
          tc::commit(smem_addr(&sh.acc_full[buf]));
          sh.committed = it + 1;
        }
      }
    }
  } else if (warp == 11) {
    // ---- scale products: a token's (or hidden row's) scale of the K block
    // times each 128-row tile's, loaded two units ahead
    uint32_t it = 0;
    bool ok = true;
    constexpr int NL = (NMAX + 31) / 32;
    struct Vals {
      float a[NL], w0, w1;
    };
    for (int phase = 0; phase < 2 && ok; ++phase) {
      const Deal& d = phase == 0 ? d1 : d2;
      const int groups = phase == 0 ? IG : HB, u1 = d.end();
      if (phase == 1 && d.begin() < u1) {
        int pass = 1;
        if (lane == 0) pass = barrier_wait(g.barrier, hidden_target, abortp);
        if (!__shfl_sync(0xffffffffu, pass, 0)) break;
      }
      auto fetch = [&](int u) {
        Vals v;
#pragma unroll
        for (int i = 0; i < NL; ++i) v.a[i] = 0.f;
        v.w0 = v.w1 = 0.f;
        if (u >= u1) return v;
        const int item = u / d.KB, kb = u - item * d.KB, grp = item % groups;
        const int e = sh.active[item / groups];
        const int n = __popcll(sh.mask[e]), row0 = sh.first_row[e];
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int c = lane + 32 * i;
          if (c < n)
            v.a[i] = phase == 0 ? __ldg(g.q_scale + sh.token_at[row0 + c] * g.sq_row + kb * g.sq_kb)
                                : ld_l2(g.h_scale + (int64_t)(row0 + c) * IG + kb);
        }
        if (phase == 0) {
          const float* p = g.w13_scale + ((int64_t)e * 2 * IG + grp) * KB1 + kb;
          v.w0 = __ldg(p), v.w1 = __ldg(p + (int64_t)IG * KB1);
        } else {
          const float* p = g.w2_scale + ((int64_t)e * (g.H / 128) + grp * 2) * KB2 + kb;
          v.w0 = __ldg(p);
          v.w1 = grp * 2 + 1 < g.H / 128 ? __ldg(p + KB2) : 0.f;
        }
        return v;
      };
      Vals v0 = fetch(d.begin()), v1 = fetch(d.begin() + 1);
      for (int u = d.begin(); u < u1; ++u, ++it) {
        const Vals v2 = fetch(u + 2);
        const uint32_t buf = it % kBufs;
        ok = it < kBufs || __all_sync(0xffffffffu, wait_or_abort(smem_addr(&sh.acc_empty[buf]),
                                                                 (it / kBufs - 1u) & 1u, abortp));
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < NL; ++i)
          if (lane + 32 * i < NMAX) {
            sh.scales[buf][0][lane + 32 * i] = v0.a[i] * v0.w0;
            sh.scales[buf][1][lane + 32 * i] = v0.a[i] * v0.w1;
          }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&sh.scale_full[buf]));
        v0 = v1;
        v1 = v2;
      }
    }
  } else {
    // ---- outer sums and epilogues
    uint32_t it = 0;
    const int half = warp >> 2, r = tid & 127;
    sum_phase<NMAX>(g, sh, d1, IG, g.counters, tmem, it, abortp,
                    [&](int item, int n, int row0, float (&acc)[NMAX]) {
                      const int grp = item % IG;
                      if (half == 1) {
#pragma unroll
                        for (int c = 0; c < NMAX; ++c)
                          if (c < n) exchange[c * kXStride + r] = acc[c];
                      }
                      epi_sync();
                      if (half == 0) {
#pragma unroll
                        for (int c = 0; c < NMAX; ++c)
                          if (c < n) {
                            const float gate = acc[c], up = exchange[c * kXStride + r];
                            exchange[c * kXStride + r] = gate / (1.f + expf(-gate)) * up;
                          }
                      }
                      epi_sync();
                      for (int c = warp; c < n; c += 8) {  // a row's group of 128, a warp
                        const float4 h = *reinterpret_cast<const float4*>(exchange + c * kXStride + 4 * lane);
                        float m = fmaxf(fmaxf(fabsf(h.x), fabsf(h.y)), fmaxf(fabsf(h.z), fabsf(h.w)));
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                        // h is not bf16: the quantizer's short reciprocal does not
                        // apply, the divisions are the compiler's
                        const float s = fmaxf(__fdiv_rn(m, kE4m3Max), kMinScale);
                        const uint32_t code = f4_to_e4m3x4(
                            make_float2(__fdiv_rn(h.x, s), __fdiv_rn(h.y, s)),
                            make_float2(__fdiv_rn(h.z, s), __fdiv_rn(h.w, s)));
                        *reinterpret_cast<uint32_t*>(g.hidden + (int64_t)(row0 + c) * g.I + grp * 128 +
                                                     4 * lane) = code;
                        if (lane == 0) g.h_scale[(int64_t)(row0 + c) * IG + grp] = s;
                      }
                      epi_sync();
                    });
    __threadfence();
    asm volatile("fence.proxy.async;" ::: "memory");
    epi_sync();
    if (tid == 0) barrier_arrive(g.barrier);
    sum_phase<NMAX>(g, sh, d2, HB, g.counters + g.n_counters1, tmem, it, abortp,
                    [&](int item, int n, int row0, float (&acc)[NMAX]) {
                      const int col = (item % HB) * 256 + half * 128 + r;
                      if (col < g.H) {
#pragma unroll
                        for (int c = 0; c < NMAX; ++c)
                          if (c < n) __stcg(g.down + (int64_t)(row0 + c) * g.H + col, acc[c]);
                      }
                    });
    __threadfence();
    epi_sync();
    if (tid == 0) {
      // one count serves all barriers: nobody arrives at one before the last is
      // complete (a CTA without a run in the second phase has not waited for it)
      barrier_wait(g.barrier, hidden_target, abortp);
      barrier_arrive(g.barrier);
      barrier_wait(g.barrier, down_target, abortp);
    }
    epi_sync();
    // ---- the weighted sum over a token's experts, four columns a thread
    const int vec = g.H / 4;
    for (int i = blockIdx.x * kEpiThreads + tid; i < g.T * vec; i += gridDim.x * kEpiThreads) {
      const int t = i / vec, col = (i - t * vec) * 4;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int j = 0; j < g.k; ++j) {
        const float w = sh.weight[t * g.k + j];
        const float4 v = ld_l2(reinterpret_cast<const float4*>(
            g.down + (int64_t)sh.row_of[t * g.k + j] * g.H + col));
        y.x = __fmaf_rn(w, v.x, y.x), y.y = __fmaf_rn(w, v.y, y.y);
        y.z = __fmaf_rn(w, v.z, y.z), y.w = __fmaf_rn(w, v.w, y.w);
      }
      *reinterpret_cast<uint2*>(g.out + (int64_t)t * g.ldo + col) =
          make_uint2(f2_to_bf2(make_float2(y.x, y.y)), f2_to_bf2(make_float2(y.z, y.w)));
    }
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (*abortp) {
    // let copies and MMAs in flight finish before their memory goes away
    if (tid == 0) {
      atomicCAS(&g_moe_device_error, kDevErrNone, kDevErrBulkWaitTimeout);
      const uint32_t both = min(sh.issued_w, sh.issued_a), any = max(sh.issued_w, sh.issued_a);
      for (uint32_t k = both > (uint32_t)P::kStages ? both - P::kStages : 0; k < both; ++k)
        mbar_wait_bounded(smem_addr(&sh.full[k % P::kStages]), (k / P::kStages) & 1u, kDrainLimitCycles);
      // a stage with only one of its two loads never completes its phase: complete it by hand
      for (uint32_t k = both; k < any; ++k) {
        mbar_arrive(smem_addr(&sh.full[k % P::kStages]));
        mbar_wait_bounded(smem_addr(&sh.full[k % P::kStages]), (k / P::kStages) & 1u, kDrainLimitCycles);
      }
      if (sh.committed > 0)
        mbar_wait_bounded(smem_addr(&sh.acc_full[(sh.committed - 1) % kBufs]),
                          ((sh.committed - 1) / kBufs) & 1u, kDrainLimitCycles);
    }
    __syncthreads();
  }
  if (warp == 10) tc::tmem_dealloc(tmem, P::kTmemCols);
}

// ------------------------------------------------------------------ host

// Shares of the router's columns: enough jobs of 4 experts x 8 tokens for
// every warp of the grid, at most one chunk of 256 columns a job.
int router_splits(int64_t T, int64_t E, int64_t H, int sms) {
  const int64_t jobs = ((E + 3) / 4) * ((T + 7) / 8), chunks = (H + 255) / 256;
  int64_t s = (int64_t)sms * kMoeWarps / jobs;
  return (int)(s < 1 ? 1 : s > chunks ? chunks : s);
}

int moe_columns(int64_t T) { return T <= 16 ? 16 : T <= 32 ? 32 : 64; }

template <int NMAX>
cudaError_t launch_moe(const CUtensorMap& mq, const CUtensorMap& m13, const CUtensorMap& mh,
                       const CUtensorMap& m2, const MoeArgs& g, int sms, cudaStream_t stream) {
  auto kernel = moe_kernel<NMAX>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)MoePlan<NMAX>::kSmemBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)sms);
  cfg.blockDim = dim3(kMoeThreads);
  cfg.dynamicSmemBytes = MoePlan<NMAX>::kSmemBytes;
  cfg.stream = stream;
  // the CTAs wait for one another: a cooperative launch, so that all are resident
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, mq, m13, mh, m2, g);
}

}  // namespace

cudaError_t device_error_moe(int* out, bool clear) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_moe_device_error, sizeof(int));
  if (e != cudaSuccess) return e;
  if (clear && v != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_moe_device_error, &zero, sizeof(int));
  }
  *out = v;
  return e;
}

size_t moe_workspace(MoeArgs* g, void* base) {
  const int sms = device_sm_count();
  const int64_t pairs = (int64_t)g->T * g->k, experts = pairs < g->E ? pairs : g->E;
  g->splits = router_splits(g->T, g->E, g->H, sms);
  g->n_counters1 = (int)(experts * (g->I / 128));
  g->n_counters = g->n_counters1 + (int)(experts * ((g->H + 255) / 256));
  size_t at = 0;
  uint8_t* p = static_cast<uint8_t*>(base);
  auto take = [&](size_t bytes) {
    uint8_t* r = p == nullptr ? nullptr : p + at;
    at += (bytes + 255) & ~(size_t)255;
    return r;
  };
  g->barrier = reinterpret_cast<uint64_t*>(take(8));
  g->counters = reinterpret_cast<int*>(take((size_t)g->n_counters * 4));
  g->logits = reinterpret_cast<float*>(take((size_t)g->splits * g->T * g->E * 4));
  int* ids = reinterpret_cast<int*>(take((size_t)pairs * 4));
  float* weights = reinterpret_cast<float*>(take((size_t)pairs * 4));
  if (g->ids == nullptr) g->ids = ids;
  if (g->weights == nullptr) g->weights = weights;
  g->hidden = take((size_t)pairs * g->I);
  g->h_scale = reinterpret_cast<float*>(take((size_t)pairs * (g->I / 128) * 4));
  g->down = reinterpret_cast<float*>(take((size_t)pairs * g->H * 4));
  g->partial = reinterpret_cast<float*>(take((size_t)sms * 2 * moe_columns(g->T) * 256 * 4));
  return at;
}

int moe_fp8(MoeArgs g, const void* q, int64_t ldq, const void* w13, const void* w2,
            cudaStream_t stream, const char** why) {
  const int sms = device_sm_count();
  const int64_t pairs = (int64_t)g.T * g.k;
  g.deal_tokens = g.T > 8;
  CUtensorMap mq, m13, mh, m2;
  if (!tc::encode_e4m3_operand(&mq, q, g.T, g.H, ldq, 1) ||
      !tc::encode_e4m3_operand(&m13, w13, (int64_t)g.E * 2 * g.I, g.H, g.H) ||
      !tc::encode_e4m3_operand(&mh, g.hidden, pairs, g.I, g.I, 16) ||
      !tc::encode_e4m3_operand(&m2, w2, (int64_t)g.E * g.H, g.I, g.I)) {
    *why = "cuTensorMapEncodeTiled failed for an operand";
    return CUTIE_ERR_CUDA;
  }
  const int n = moe_columns(g.T);
  const cudaError_t e = n == 16   ? launch_moe<16>(mq, m13, mh, m2, g, sms, stream)
                        : n == 32 ? launch_moe<32>(mq, m13, mh, m2, g, sms, stream)
                                  : launch_moe<64>(mq, m13, mh, m2, g, sms, stream);
  if (e != cudaSuccess) {
    *why = cudaGetErrorString(e);
    return CUTIE_ERR_CUDA;
  }
  return CUTIE_OK;
}

}  // namespace cutie
