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
// neighbours: the CTA whose run begins it owns it, the others send their part
// (the first thing in their run) through the workspace, and the owner (whose
// run ends with it) adds them in the order of K. The result does not depend on
// timing.
//
// Between CTAs: a grid barrier when the logits are complete (for many tokens
// another when the choices are), a count a hidden row group of each expert that
// its down products wait for, and a grid barrier before the weighted sum. The
// weight stream does not stop for the hidden rows: its TMA thread needs only
// the choices, and fills the ring with down tiles in the meantime.
//
// Warps: 0-7 the outer sums (warps 0-3 the first 128 rows of an item, 4-7 the
// second, a row a thread) and the epilogues; 8 the weight tiles (TMA); 9 the
// tokens' rows (TMA gather of 4 rows for the first product, boxes of 16 hidden
// rows for the second); 10 the MMAs; 11 the scales.
#include "cutie.h"
#include "launch.cuh"
#include "tcgen05.cuh"

namespace cutie {

static __device__ int g_moe_device_error = 0;

namespace {

constexpr int kMoeThreads = 384, kMoeWarps = 12, kEpiThreads = 256;
constexpr uint32_t kBox = 128 * 128;  // a 128-row weight tile of one K block
constexpr int kBufs = 4;              // accumulator buffers in tensor memory
constexpr int kScaleSlots = 8;        // units whose scales are on their way or in use
constexpr int kXStride = 132;         // floats between columns of the exchange
constexpr int kMaxE = kMoeMaxExperts, kMaxK = kMoeMaxTopK;
constexpr int kTaggedTokens = 8;  // tokens up to which parts carry tags
constexpr int kChooseTokens = 8;  // tokens up to which every CTA makes all choices

template <int NMAX>
struct MoePlan {
  static constexpr uint32_t kStageBytes = 2 * kBox + NMAX * 128;
  static constexpr int kStages = NMAX == 16 ? 6 : NMAX == 32 ? 5 : 4;
  static constexpr int kXCols = NMAX == 16 ? 8 : NMAX == 32 ? 16 : 32;  // columns an exchange pass
  static constexpr uint32_t kXBytes = 2 * kXCols * kXStride * 4;
  static constexpr size_t kSmemBytes = kStages * kStageBytes + kXBytes + 1024;
  static constexpr uint32_t kTmemCols = kBufs * 2 * NMAX;
  static constexpr int kPairs = NMAX * kMaxK;
  static_assert(NMAX != 16 || kTaggedTokens * 8 <= NMAX * 4, "tagged parts fit the parts' place");
  static_assert(kStageBytes % 1024 == 0, "swizzled tiles start on 1 KB");
  static_assert(2 * kChooseTokens * kMaxE * 4 <= kStages * kStageBytes, "logits and keys fit the idle ring");
};

// Units of a phase dealt in runs of `per`; KB units an item, `groups` items an expert.
struct Deal {
  int per, units, KB, groups;
  __device__ __forceinline__ void set(int experts, int groups_, int kb) {
    KB = kb, groups = groups_, units = experts * groups_ * kb;
    per = (units + (int)gridDim.x - 1) / (int)gridDim.x;
  }
};

// A walk over this CTA's run: unit u is K block kb of item grp of the a-th active expert.
struct Walk {
  int u, end, kb, KB, grp, groups, a;
  __device__ __forceinline__ void set(const Deal& d) {
    u = min(d.per * (int)blockIdx.x, d.units), end = min(u + d.per, d.units);
    const int item = u / d.KB;
    KB = d.KB, groups = d.groups;
    kb = u - item * KB, a = item / groups, grp = item - a * groups;
  }
  __device__ __forceinline__ bool more() const { return u < end; }
  __device__ __forceinline__ void next() {
    ++u;
    if (++kb == KB) {
      kb = 0;
      if (++grp == groups) grp = 0, ++a;
    }
  }
};

template <int NMAX>
struct MoeShared {
  uint64_t full[8], empty[8], acc_full[kBufs], acc_empty[kBufs];
  uint64_t scale_full[kScaleSlots], scale_empty[kScaleSlots];
  float scales[kScaleSlots][NMAX + 4];  // the tokens', then the two weight tiles'
  uint64_t mask[kMaxE];       // tokens of an expert
  float weight[MoePlan<NMAX>::kPairs];
  uint16_t ids[MoePlan<NMAX>::kPairs];     // expert of (token, slot)
  uint16_t row_of[MoePlan<NMAX>::kPairs];  // its hidden row: experts in order, tokens in order
  uint8_t token_at[MoePlan<NMAX>::kPairs]; // token of a hidden row
  uint16_t first_row[kMaxE];
  uint16_t active[kMaxE < MoePlan<NMAX>::kPairs ? kMaxE : MoePlan<NMAX>::kPairs];
  Deal deal[2];
  Walk walk[2];
  uint32_t tmem_base, abort_flag, issued_w, issued_a, committed;
  uint64_t target;  // the grid barrier's count at the next barrier
};

// ------------------------------------------------------------------ grid barrier
//
// A 64-bit count in the workspace, zero before its first use. Every CTA adds
// one a barrier, every launch passes the same number of barriers, so the
// count is a multiple of the grid's size between launches and needs no reset.

__device__ __forceinline__ uint64_t barrier_arrive(uint64_t* count) {
  uint64_t old;  // the release covers the CTA's writes, which a barrier of its threads ordered before
  asm volatile("atom.release.gpu.global.add.u64 %0, [%1], 1;" : "=l"(old) : "l"(count) : "memory");
  return old;
}

__device__ __forceinline__ bool barrier_wait(const uint64_t* count, uint64_t target,
                                             volatile uint32_t* abort_flag, long long limit) {
  const long long t0 = clock64();
  for (;;) {
    uint64_t v;
    asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(count) : "memory");
    if (v >= target) break;
    if (clock64() - t0 > limit) {
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
// Zero where `ok` is false; no branch, so that nothing waits for the load.
__device__ __forceinline__ float ld_l2_if(bool ok, const float* p) {
  float v;
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.u32 q, %2, 0;\n mov.f32 %0, 0f00000000;\n"
      " @q ld.global.cg.f32 %0, [%1];\n}"
      : "=&f"(v)
      : "l"(p), "r"((uint32_t)ok)
      : "memory");
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

// Counts between CTAs of one launch: add one, ordered after the CTA's writes
// that a barrier of its threads ordered before; wait for a number of them.
__device__ __forceinline__ void release_add(int* count) {
  asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(count) : "memory");
}
__device__ __forceinline__ bool wait_count(const int* count, int target, volatile uint32_t* abort_flag,
                                           long long limit) {
  const long long t0 = clock64();
  for (;;) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(count) : "memory");
    if (v >= target) return true;
    if (*abort_flag || clock64() - t0 > limit) {
      *abort_flag = 1u;
      return false;
    }
  }
}
// The same before TMA reads what was waited for.
__device__ __forceinline__ bool wait_count_tma(const int* count, int target, volatile uint32_t* abort_flag,
                                               long long limit) {
  const bool ok = wait_count(count, target, abort_flag, limit);
  asm volatile("fence.proxy.async;" ::: "memory");
  return ok;
}

// ------------------------------------------------------------------ router

// Logits of 4 experts x 8 tokens over one of `splits` shares of the columns, a
// CTA a job: the warps take chunks of 256 columns, the lanes 8 columns each, so
// a warp ends with 32 sums over 32 lanes, folded so that lane l keeps sum l;
// the warps' are added through shared memory.
__device__ __forceinline__ void router_job(const MoeArgs& g, int job, int warp, int lane,
                                           float (*red)[32]) {
  const int eg = (g.E + 3) / 4, tg = (g.T + 7) / 8, chunks = (g.H + 255) / 256;
  const int e0 = 4 * (job % eg), t0 = 8 * ((job / eg) % tg), s = job / (eg * tg);
  const int ne = min(4, g.E - e0), nt = min(8, g.T - t0);
  const int c1 = chunks * (s + 1) / g.splits;
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = 0.f;
  for (int c = chunks * s / g.splits + warp; c < c1; c += kMoeWarps) {
    const int col = c * 256 + lane * 8;
    if (col >= g.H) continue;
    uint4 w[4], x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = i < ne ? ld_keep(g.router + (int64_t)(e0 + i) * g.H + col) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = j < nt ? ld_keep(g.x + (int64_t)(t0 + j) * g.ldx + col) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float2 wf[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) wf[i] = bf2_to_f2(q == 0 ? w[i].x : q == 1 ? w[i].y : q == 2 ? w[i].z : w[i].w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 xf = bf2_to_f2(q == 0 ? x[j].x : q == 1 ? x[j].y : q == 2 ? x[j].z : x[j].w);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i * 8 + j] = __fmaf_rn(wf[i].y, xf.y, __fmaf_rn(wf[i].x, xf.x, v[i * 8 + j]));
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
  red[warp][lane] = v[0];
  __syncthreads();
  if (warp == 0) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kMoeWarps; ++i) sum += red[i][lane];
    const int i = lane >> 3, j = lane & 7;
    if (i < ne && j < nt) g.logits[((int64_t)s * g.T + t0 + j) * g.E + e0 + i] = sum;
  }
  __syncthreads();
}

// Order of floats as unsigned; NaN lowest but one, 0 is "none".
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __float_as_uint(f);
  return f != f ? 1u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// The larger one, or a NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float unordered(uint32_t key) {
  return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}

// Logits of `n` tokens from t0 on, [n][E] into shared memory: the sums of the
// router's shares, a thread a logit, eight loads in flight.
__device__ __forceinline__ void sum_logits(const MoeArgs& g, int t0, int n, float* to) {
  for (int i = threadIdx.x; i < n * g.E; i += kMoeThreads) {
    const float* p = g.logits + (int64_t)t0 * g.E + i;
    float sum = 0.f;
    for (int s = 0; s < g.splits; s += 8) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = ld_l2_if(s + j < g.splits, p + (int64_t)(s + j) * g.T * g.E);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[j];
    }
    to[i] = sum;
  }
}

// One token's choice by one warp from its logits in shared memory: k rounds of
// a warp maximum, ties to the lowest expert; `key` is E words of scratch. Lane
// j < k returns with (*id, *w) of slot j. A NaN logit is chosen last; under
// softmax it makes every weight of the token a NaN (m carries it), as the sum
// over all experts would. The loops stay rolled: every launch
// runs this once, and instructions fetched for the first time cost more than
// they compute (unrolled over 16 registers a lane this took 4 us, not 1.5).
__device__ __forceinline__ void choose(const MoeArgs& g, const float* logits, uint32_t* key, int lane,
                                       int* id, float* w) {
  const bool softmax = g.scoring == 0;
  float m = -INFINITY, z = 1.f;
  if (softmax) {  // the sum over all experts only where the weights need it
#pragma unroll 1
    for (int e = lane; e < g.E; e += 32) m = max_nan(m, logits[e]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!g.renormalize || g.bias != nullptr) {
      z = 0.f;
#pragma unroll 1
      for (int e = lane; e < g.E; e += 32) z += expf(logits[e] - m);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    }
  }
#pragma unroll 1
  for (int e = lane; e < g.E; e += 32) {
    // without a bias the choice goes by the logits, which the scores grow with
    // (and saturate against); with one by the biased scores
    float sel = logits[e];
    if (g.bias != nullptr) sel = (softmax ? expf(sel - m) / z : 1.f / (1.f + expf(-sel))) + g.bias[e];
    key[e] = ordered(sel);
  }
  int my_id = 0;
#pragma unroll 1
  for (int j = 0; j < g.k; ++j) {
    uint32_t best = 0, at = 0xffffffffu;
#pragma unroll 1
    for (int e = lane; e < g.E; e += 32)
      if (key[e] > best) best = key[e], at = (uint32_t)e;
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const uint32_t e = __reduce_min_sync(0xffffffffu, best == top ? at : 0xffffffffu);
    if ((e & 31u) == (uint32_t)lane) key[e] = 0;  // this lane's own entry: no other reads it
    if (lane == j) my_id = (int)e;
  }
  float p = 0.f;
  const float l = lane < g.k ? logits[my_id] : -INFINITY;
  // Renormalized weights are ratios: where the chosen scores are all below e^-64
  // (a bias chose them, or every sigmoid is that small) and might underflow, they
  // are taken relative to the largest of them instead.
  bool rescale = false;
  if (g.renormalize) {
    const float top = unordered(__reduce_max_sync(0xffffffffu, ordered(l)));
    rescale = softmax ? top < m - 64.f && m < INFINITY : top < -64.f;
    if (rescale) m = top;
  }
  if (lane < g.k) p = softmax || rescale ? expf(l - m) : 1.f / (1.f + expf(-l));
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

// A split item belongs to the CTA whose run begins it (and ends in it); the
// others' runs begin inside it, so their part is the first thing they finish.
// It goes through the workspace, n columns, thread = row.
//
// A flag after a part costs its sender a fence, whose acknowledgements queue
// behind the weights that the SM has asked for: 3 to 6 us, in which the sums and
// with them the stream stand still, and the owner waits as long. So for few
// tokens each value travels in 64 bits with a word that says it is there
// (cleared by its sender before the first grid barrier), stored and read whole:
// no fence and no flag. Of 8 experts of 4096 x 2048, top 2, a layer took 34.8 us
// for 1 token and 41 for 4 this way, 36.9 and 45.1 with flags; 59.4 for 12 either
// way. The clearing grows with the tokens while the stream gets longer, so above
// kTaggedTokens parts have one flag each.
__device__ __forceinline__ uint64_t* tagged_part(const MoeArgs& g, int phase, int b) {
  return reinterpret_cast<uint64_t*>(g.partial) + (int64_t)(phase * (int)gridDim.x + b) * g.T * 256;
}

// send_part: such a part to the workspace, and its flag or tags.
template <int NMAX>
__device__ __forceinline__ void send_part(const MoeArgs& g, int phase, int n, const float (&acc)[NMAX]) {
  if (NMAX == 16 && g.T <= kTaggedTokens) {
    uint64_t* p = tagged_part(g, phase, (int)blockIdx.x) + threadIdx.x;
#pragma unroll
    for (int c = 0; c < kTaggedTokens; ++c)
      if (c < n)
        asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(p + c * 256),
                     "l"((1ull << 32) | __float_as_uint(acc[c]))
                     : "memory");
    return;
  }
  float* p = g.partial + (int64_t)(phase * (int)gridDim.x + (int)blockIdx.x) * NMAX * 256 + threadIdx.x;
#pragma unroll
  for (int c = 0; c < NMAX; ++c)
    if (c < n) __stcg(p + c * 256, acc[c]);
  epi_sync();
  if (threadIdx.x == 0) release_add(g.part_flag + phase * gridDim.x + blockIdx.x);
}

// add_parts: the owner's sums plus the others' in the order of K.
template <int NMAX>
__device__ __forceinline__ void add_parts(const MoeArgs& g, const Deal& deal, int phase, int item, int n,
                                          float (&acc)[NMAX], volatile uint32_t* abortp) {
  const int last = ((item + 1) * deal.KB - 1) / deal.per;
  if (NMAX == 16 && g.T <= kTaggedTokens) {
#pragma unroll 1
    for (int b = (int)blockIdx.x + 1; b <= last; ++b) {
      const uint64_t* o = tagged_part(g, phase, b) + threadIdx.x;
      uint64_t v[kTaggedTokens];
      const long long t0 = clock64();
      for (;;) {
        bool here = true;
#pragma unroll
        for (int c = 0; c < kTaggedTokens; ++c) {
          asm volatile(
              "{\n .reg .pred q;\n setp.lt.s32 q, %2, %3;\n mov.b64 %0, 0x100000000;\n"
              " @q ld.relaxed.gpu.global.b64 %0, [%1];\n}"
              : "=&l"(v[c])
              : "l"(o + c * 256), "r"(c), "r"(n)
              : "memory");
        }
#pragma unroll
        for (int c = 0; c < kTaggedTokens; ++c) here &= (v[c] >> 32) != 0;
        if (here) break;
        if (*abortp || clock64() - t0 > g.wait_limit) {
          *abortp = 1u;
          break;
        }
      }
#pragma unroll
      for (int c = 0; c < kTaggedTokens; ++c) acc[c] += __uint_as_float((uint32_t)v[c]);
    }
    return;
  }
#pragma unroll 1
  for (int b = (int)blockIdx.x + 1; b <= last; ++b) {
    if ((threadIdx.x & 31) == 0) wait_count(g.part_flag + phase * gridDim.x + b, 1, abortp, g.wait_limit);
    __syncwarp();
    const float* o = g.partial + (int64_t)(phase * (int)gridDim.x + b) * NMAX * 256 + threadIdx.x;
#pragma unroll
    for (int c0 = 0; c0 < NMAX; c0 += 16) {
      if (c0 >= n) break;
      float v[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) v[c] = ld_l2_if(c0 + c < n, o + (c0 + c) * 256);
#pragma unroll
      for (int c = 0; c < 16; ++c) acc[c0 + c] += v[c];
    }
  }
}

// One group of 128 of a hidden row by one warp: silu(gate) * up, its scale and codes.
__device__ __noinline__ void hidden_group(const float* gate, const float* up, int lane, uint8_t* codes,
                                          float* scale) {
  float h[4], m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = gate[lane * 4 + i];
    h[i] = a / (1.f + expf(-a)) * up[lane * 4 + i];
    m = fmaxf(m, fabsf(h[i]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  // h is not bf16: the quantizer's short reciprocal does not apply
  const float s = fmaxf(__fdiv_rn(m, kE4m3Max), kMinScale);
  const uint32_t code = f4_to_e4m3x4(make_float2(__fdiv_rn(h[0], s), __fdiv_rn(h[1], s)),
                                     make_float2(__fdiv_rn(h[2], s), __fdiv_rn(h[3], s)));
  *reinterpret_cast<uint32_t*>(codes + 4 * lane) = code;
  if (lane == 0) *scale = s;
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
    }
    for (int s = 0; s < kScaleSlots; ++s) {
      mbar_init(smem_addr(&sh.scale_full[s]), 32);
      mbar_init(smem_addr(&sh.scale_empty[s]), 8);
    }
    sh.abort_flag = 0;
    sh.issued_w = sh.issued_a = sh.committed = 0;
    mbar_init_fence();
  }
  if (warp == 10) tc::tmem_alloc(smem_addr(&sh.tmem_base), P::kTmemCols);
  for (int e = tid; e < g.E; e += kMoeThreads) sh.mask[e] = 0;

  // ---- router: partial logits, and this launch's counts to zero
  for (int i = blockIdx.x * kMoeThreads + tid; i < g.n_counts; i += gridDim.x * kMoeThreads)
    g.part_flag[i] = 0;
  if (NMAX == 16 && g.T <= kTaggedTokens)
#pragma unroll
    for (int phase = 0; phase < 2; ++phase)
      for (int i = tid; i < g.T * 128; i += kMoeThreads)
        __stcg(reinterpret_cast<uint4*>(tagged_part(g, phase, (int)blockIdx.x)) + i, make_uint4(0, 0, 0, 0));
  const int jobs = ((g.E + 3) / 4) * ((g.T + 7) / 8) * g.splits;
  for (int j = blockIdx.x; j < jobs; j += gridDim.x)
    router_job(g, j, warp, lane, reinterpret_cast<float(*)[32]>(smem_raw));  // the ring is idle
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (tid == 0) {
    const uint64_t old = barrier_arrive(g.barrier);
    sh.target = (old / gridDim.x + 1) * gridDim.x;
    barrier_wait(g.barrier, sh.target, abortp, g.wait_limit);
  }
  __syncthreads();
  uint64_t target = sh.target;

  // ---- choices: every CTA makes them all for few tokens; for more, each
  // token's is made once and read by all after another barrier
  const int pairs = g.T * g.k;
  const bool deal_tokens = g.deal_tokens;
  float* logits = reinterpret_cast<float*>(smem_raw);  // the ring is idle: kChooseTokens x E at most
  for (int t0 = deal_tokens ? blockIdx.x : 0; t0 < g.T; t0 += deal_tokens ? gridDim.x : g.T) {
    const int n = deal_tokens ? 1 : g.T;
    sum_logits(g, t0, n, logits);
    __syncthreads();
    for (int t = warp; t < n; t += kMoeWarps) {
      int id;
      float w;
      choose(g, logits + t * g.E, reinterpret_cast<uint32_t*>(logits + (n + t) * g.E), lane, &id, &w);
      if (lane < g.k) {
        const int p = (t0 + t) * g.k + lane;
        if (deal_tokens || blockIdx.x == 0) g.ids[p] = id, g.weights[p] = w;
        if (!deal_tokens) sh.ids[p] = (uint16_t)id, sh.weight[p] = w;
      }
    }
    __syncthreads();
  }
  tc::fence_async_smem();  // the ring's TMA writes come after these accesses
  if (deal_tokens) {
    __syncthreads();
    target += gridDim.x;
    if (tid == 0) {
      barrier_arrive(g.barrier);
      barrier_wait(g.barrier, target, abortp, g.wait_limit);
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
    if (lane < 2) {
      sh.deal[lane].set(n, lane == 0 ? IG : HB, lane == 0 ? KB1 : KB2);
      sh.walk[lane].set(sh.deal[lane]);
    }
  }
  __syncthreads();
  // the weight stream needs no more than this; the others, the rows' tables
  if (warp != 8) {
    for (int p = tid < 256 ? tid : tid - 32; p < pairs; p += kMoeThreads - 32) {
      const int t = p / g.k, e = sh.ids[p] < g.E ? sh.ids[p] : 0;
      const int row = sh.first_row[e] + __popcll(sh.mask[e] & ((1ull << t) - 1ull));
      sh.row_of[p] = (uint16_t)row;
      sh.token_at[row] = (uint8_t)t;
    }
    asm volatile("barrier.cta.sync 2, 352;" ::: "memory");
  }

  const uint32_t tmem = sh.tmem_base;
  const uint64_t down_target = target + gridDim.x;

  if (warp == 8) {
    // ---- weight tiles of both phases, without a stop between them
    const bool leader = tc::elect_one();
    const uint64_t once = tc::evict_first_policy();
    uint32_t s = 0, parity = 1;  // a fresh barrier passes a wait for the phase before its first
    bool ok = true;
#pragma unroll 1
    for (int phase = 0; phase < 2 && ok; ++phase) {
      const CUtensorMap* map = phase == 0 ? &map_w13 : &map_w2;
      const int rows = phase == 0 ? 2 * g.I : g.H, step = phase == 0 ? 128 : 256;
      const int second = phase == 0 ? g.I : 128;
#pragma unroll 1
      for (Walk w = sh.walk[phase]; w.more(); w.next()) {
        ok = __all_sync(0xffffffffu, tc::wait_or_abort(smem_addr(&sh.empty[s]), parity, abortp, g.wait_limit));
        if (!ok) break;
        if (leader) {
          const uint32_t st = base + s * P::kStageBytes, bar = smem_addr(&sh.full[s]);
          const int r = sh.active[w.a] * rows + w.grp * step;
          mbar_arrive_expect_tx(bar, 2 * kBox);
          tc::tma_load_2d_hint(st, map, w.kb * 128, r, bar, once);
          tc::tma_load_2d_hint(st + kBox, map, w.kb * 128, r + second, bar, once);
          ++sh.issued_w;
        }
        if (++s == P::kStages) s = 0, parity ^= 1;
      }
    }
  } else if (warp == 9) {
    // ---- the tokens' rows
    const bool leader = tc::elect_one();
    uint32_t s = 0, parity = 1;
    bool ok = true;
#pragma unroll 1
    for (int phase = 0; phase < 2 && ok; ++phase) {
      int hidden_of = -1;  // the expert whose hidden rows are known to be complete
#pragma unroll 1
      for (Walk w = sh.walk[phase]; w.more(); w.next()) {
        if (phase == 1 && w.a != hidden_of) {
          hidden_of = w.a;
          if (leader) ok = wait_count_tma(g.ready + w.a, IG, abortp, g.wait_limit);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        ok = __all_sync(0xffffffffu, tc::wait_or_abort(smem_addr(&sh.empty[s]), parity, abortp, g.wait_limit));
        if (!ok) break;
        if (leader) {
          const int e = sh.active[w.a], n = __popcll(sh.mask[e]), row0 = sh.first_row[e];
          const uint32_t st = base + s * P::kStageBytes + 2 * kBox, bar = smem_addr(&sh.full[s]);
          const int np = (n + 15) & ~15, last = row0 + n - 1;
          mbar_arrive_expect_tx(bar, (uint32_t)np * 128u);
          if (phase == 0) {
            // columns past the expert's tokens repeat its last one and are not used
#pragma unroll 1
            for (int c = 0; c < np; c += 4)
              tc::tma_gather4(st + (uint32_t)c * 128u, &map_q, w.kb * 128,
                              sh.token_at[min(row0 + c, last)], sh.token_at[min(row0 + c + 1, last)],
                              sh.token_at[min(row0 + c + 2, last)],
                              sh.token_at[min(row0 + c + 3, last)], bar);
          } else {
#pragma unroll 1
            for (int c = 0; c < np; c += 16)
              tc::tma_load_2d(st + (uint32_t)c * 128u, &map_h, w.kb * 128, row0 + c, bar);
          }
          ++sh.issued_a;
        }
        if (++s == P::kStages) s = 0, parity ^= 1;
      }
    }
  } else if (warp == 10) {
    // ---- MMAs
    const bool leader = tc::elect_one();
    const uint32_t lo0 = tc::sw128_lo(base), hi = tc::sw128_hi();
    uint32_t s = 0, parity = 0, buf = 0, buf_parity = 1;
    bool ok = true;
#pragma unroll 1
    for (int phase = 0; phase < 2 && ok; ++phase) {
      uint32_t idesc = 0;
#pragma unroll 1
      for (Walk w = sh.walk[phase]; w.more(); w.next()) {
        if (idesc == 0 || w.kb == 0)
          idesc = tc::f8_idesc(128, (__popcll(sh.mask[sh.active[w.a]]) + 15) & ~15);
        ok = __all_sync(0xffffffffu,
                        tc::wait_or_abort(smem_addr(&sh.full[s]), parity, abortp, g.wait_limit) &&
                            tc::wait_or_abort(smem_addr(&sh.acc_empty[buf]), buf_parity, abortp, g.wait_limit));
        if (!ok) break;
        tc::fence_after();
        if (leader) {
          const uint32_t lo = lo0 + s * (P::kStageBytes >> 4);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc::mma_f8(tmem + buf * 2 * NMAX + h * NMAX, lo + h * (kBox >> 4) + 2 * kk,
                         lo + 2 * (kBox >> 4) + 2 * kk, hi, idesc, kk != 0);
          tc::commit(smem_addr(&sh.empty[s]));
          tc::commit(smem_addr(&sh.acc_full[buf]));
          ++sh.committed;
        }
        __syncwarp();
        if (++s == P::kStages) s = 0, parity ^= 1;
        if (++buf == kBufs) buf = 0, buf_parity ^= 1;
      }
    }
  } else if (warp == 11) {
    // ---- scales of a unit: each token's (or hidden row's) of the K block and the
    // two weight tiles', copied to a ring slot kScaleSlots units ahead of their
    // use (they come from HBM), a copy a lane
    constexpr int NL = (NMAX + 31) / 32;
    uint32_t s = 0, parity = 1;
    bool ok = true;
#pragma unroll 1
    for (int phase = 0; phase < 2 && ok; ++phase) {
      int hidden_of = -1;
      const int64_t step = phase == 0 ? g.sq_kb : 1;
      const float *pa[NL], *pw = nullptr;
      int n = 0;
#pragma unroll 1
      for (Walk w = sh.walk[phase]; w.more(); w.next()) {
        if (phase == 1 && w.a != hidden_of) {
          hidden_of = w.a;
          if (lane == 0) ok = wait_count(g.ready + w.a, IG, abortp, g.wait_limit);
          __syncwarp();  // orders the other lanes' copies of h_scale after lane 0's acquire; a vote does not
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        if (n == 0 || w.kb == 0) {  // addresses change at items only
          const int e = sh.active[w.a], row0 = sh.first_row[e];
          n = __popcll(sh.mask[e]);
#pragma unroll
          for (int i = 0; i < NL; ++i) {
            const int row = row0 + min(lane + 32 * i, n - 1);
            pa[i] = phase == 0 ? g.q_scale + sh.token_at[row] * g.sq_row : g.h_scale + (int64_t)row * IG;
          }
          // lane 0: the first tile's row of blocks, lane 1: the second's
          pw = phase == 0 ? g.w13_scale + ((int64_t)e * 2 * IG + w.grp + lane * IG) * KB1
                          : g.w2_scale + ((int64_t)e * (g.H / 128) + w.grp * 2 + lane) * KB2;
          if (lane >= (phase == 0 || w.grp * 2 + 1 < g.H / 128 ? 2 : 1)) pw = nullptr;
        }
        ok = __all_sync(0xffffffffu,
                        tc::wait_or_abort(smem_addr(&sh.scale_empty[s]), parity, abortp, g.wait_limit));
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < NL; ++i)
          if (lane + 32 * i < n)
            tc::cp_async_4(smem_addr(&sh.scales[s][lane + 32 * i]), pa[i] + w.kb * step);
        if (pw != nullptr) tc::cp_async_4(smem_addr(&sh.scales[s][NMAX + lane]), pw + w.kb);
        tc::cp_async_arrive(smem_addr(&sh.scale_full[s]));
        if (++s == kScaleSlots) s = 0, parity ^= 1;
      }
    }
    tc::cp_async_wait_all();
  } else {
    // ---- outer sums and epilogues
    uint32_t it = 0;
    const int half = warp >> 2, r = tid & 127;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(half * NMAX);
#pragma unroll 1
    for (int phase = 0; phase < 2; ++phase) {
      float acc[NMAX];
      int n = 0, row0 = 0;
      bool begun = false, from_start = false;
#pragma unroll 1
      for (Walk w = sh.walk[phase]; w.more(); w.next(), ++it) {
        if (!begun) {
          begun = true, from_start = w.kb == 0;
          const int e = sh.active[w.a];
          n = __popcll(sh.mask[e]), row0 = sh.first_row[e];
#pragma unroll
          for (int c = 0; c < NMAX; ++c) acc[c] = 0.f;
        }
        const uint32_t buf = it % kBufs, slot = it % kScaleSlots;
        const bool ok =
            tc::wait_or_abort(smem_addr(&sh.scale_full[slot]), (it / kScaleSlots) & 1u, abortp, g.wait_limit) &&
            tc::wait_or_abort(smem_addr(&sh.acc_full[buf]), (it / kBufs) & 1u, abortp, g.wait_limit);
        if (__all_sync(0xffffffffu, ok)) {
          tc::fence_after();
          const float ws = sh.scales[slot][NMAX + half];
#pragma unroll
          for (int c = 0; c < NMAX; c += 16) {
            if (c >= n) break;
            uint32_t v[16];
            tc::tmem_ld_async(lane_base + buf * 2 * NMAX + (uint32_t)c, v);
            const float4* sc = reinterpret_cast<const float4*>(&sh.scales[slot][c]);
            float4 f[4] = {sc[0], sc[1], sc[2], sc[3]};
            tc::tmem_ld_wait(v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              f[i].x *= ws, f[i].y *= ws, f[i].z *= ws, f[i].w *= ws;
              acc[c + 4 * i] = __fmaf_rn(__uint_as_float(v[4 * i]), f[i].x, acc[c + 4 * i]);
              acc[c + 4 * i + 1] = __fmaf_rn(__uint_as_float(v[4 * i + 1]), f[i].y, acc[c + 4 * i + 1]);
              acc[c + 4 * i + 2] = __fmaf_rn(__uint_as_float(v[4 * i + 2]), f[i].z, acc[c + 4 * i + 2]);
              acc[c + 4 * i + 3] = __fmaf_rn(__uint_as_float(v[4 * i + 3]), f[i].w, acc[c + 4 * i + 3]);
            }
          }
          tc::fence_before();
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_addr(&sh.acc_empty[buf]));
          mbar_arrive(smem_addr(&sh.scale_empty[slot]));
        }
        const bool to_end = w.kb == w.KB - 1;
        if (!to_end && w.u != w.end - 1) continue;
        // ---- the item, or this CTA's part of it, is complete
        begun = false;
        if (!from_start) {
          send_part<NMAX>(g, phase, n, acc);
          continue;
        }
        if (!to_end) add_parts<NMAX>(g, sh.deal[phase], phase, w.a * w.groups + w.grp, n, acc, abortp);
        if (phase == 0) {
          // hidden rows: both halves to shared memory, then a row's group of
          // 128 columns a warp
#pragma unroll
          for (int h0 = 0; h0 < NMAX; h0 += P::kXCols) {
            if (h0 >= n) break;
#pragma unroll
            for (int c = 0; c < P::kXCols; ++c)
              if (h0 + c < n) exchange[(half * P::kXCols + c) * kXStride + r] = acc[h0 + c];
            epi_sync();
#pragma unroll 1
            for (int c = warp; c < P::kXCols && h0 + c < n; c += 8)
              hidden_group(exchange + c * kXStride, exchange + (P::kXCols + c) * kXStride, lane,
                           g.hidden + (int64_t)(row0 + h0 + c) * g.I + w.grp * 128,
                           g.h_scale + (int64_t)(row0 + h0 + c) * IG + w.grp);
            asm volatile("fence.proxy.async;" ::: "memory");  // hidden rows are read by TMA
            epi_sync();
          }
          if (tid == 0) release_add(g.ready + w.a);
        } else {
          const int col = w.grp * 256 + half * 128 + r;
          if (col < g.H) {
#pragma unroll
            for (int c = 0; c < NMAX; ++c)
              if (c < n) __stcg(g.down + (int64_t)(row0 + c) * g.H + col, acc[c]);
          }
        }
      }
    }
    epi_sync();
    if (tid == 0) {
      barrier_arrive(g.barrier);
      barrier_wait(g.barrier, down_target, abortp, g.wait_limit);
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

// Shares of the router's columns: as many jobs of 4 experts x 8 tokens as CTAs,
// while each of a CTA's warps keeps at least one chunk of 256 columns.
int router_splits(int64_t T, int64_t E, int64_t H, int sms) {
  const int64_t jobs = ((E + 3) / 4) * ((T + 7) / 8), chunks = (H + 255) / 256;
  const int64_t most = (chunks + kMoeWarps - 1) / kMoeWarps, s = sms / jobs;
  return (int)(s < 1 ? 1 : s > most ? most : s);
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
  g->n_counts = 2 * sms + (int)experts;
  size_t at = 0;
  uint8_t* p = static_cast<uint8_t*>(base);
  auto take = [&](size_t bytes) {
    uint8_t* r = p == nullptr ? nullptr : p + at;
    at += (bytes + 255) & ~(size_t)255;
    return r;
  };
  g->barrier = reinterpret_cast<uint64_t*>(take(8));
  g->part_flag = reinterpret_cast<int*>(take((size_t)g->n_counts * 4));
  g->ready = g->part_flag + 2 * sms;
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
  g.deal_tokens = g.T > kChooseTokens;
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
