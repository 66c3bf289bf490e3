// AdamW over many tensors in one launch (sm_100a). For each element, in fp32:
//   g' = g c                           c: what clipping leaves of the gradients, or 1
//   m' = b1 m + (1 - b1) g'
//   v' = b2 v + (1 - b2) (g' g')
//   p' = p (1 - lr decay) - (lr / (1 - b1^t)) (m' / (sqrt(v') / sqrt(1 - b2^t) + eps))
// States in 32 bits are m and v. States in 8 bits are e4m3 codes of m and of
// r = sqrt(v) (the root halves the range of exponents that codes have to span)
// with a scale max(amax / 448, 2^-92) for each 128 elements of a tensor; m' and
// r' are rounded to one of the two neighbouring codes, the nearer one the
// likelier, by 16 bits each of a hash of (seed, step, tensor, element). Rounded
// to the nearest, r would stand still: a step changes it by (1 - b2) / 2 of
// itself, codes are 2^-3 apart. A positive r' never becomes zero, so no element
// is divided by eps alone because its code was lost.
//
// A CTA takes a run of neighbouring chunks of 4096 elements of one tensor; the
// tensor of its first is found by a search in the table that is the kernel's
// argument (no copy to the GPU, nothing to keep for a graph). Bound: memory, each
// value once, for states in 32 bits, whose kernel rounds every product and sum by
// itself. With codes (10 bytes an element of bf16) it is the issue of
// instructions: so that kernel multiplies in pairs (f32x2) and takes 16 elements a
// thread, whose group shares its maxima and scales over 8 lanes. What becomes codes
// has the same bits as in the other kernel (one code more or less would move the
// scale of its group in the next step); the update has a fused sum and an
// approximate reciprocal (2^-23). 134M elements in 311 to 319 us, 66% of the copy
// bandwidth, 64 thread instructions an element, against 412 and 89 in the other
// kernel's form. Tried: copies through shared memory a chunk ahead (9% more
// instructions, no gain), approximate roots and fused sums for the codes too (278).
#include <cuda_fp16.h>

#include "cutie.h"
#include "launch.cuh"

namespace cutie {
namespace {

constexpr int kThreads = 256, kEach = 8, kChunk = 4096, kGroup = 128;
constexpr int kCtas = 5, kCodesCtas = 3;  // an SM at once (codes: four spill, 318 against 312 us)
constexpr float kMinState = 0x1p-92f;

// Tensors a launch: its argument is the table, 32 KB at most. Short lists take
// a short one: an argument is copied at every launch.
constexpr int kFewTensors = 40, kManyTensors = 480;

template <int N>
struct Table {
  const void* g[N];
  void* p[N];
  void* m[N];
  void* v[N];
  float* ms[N];  // scales; null for states in 32 bits
  float* vs[N];
  int64_t n[N];
  uint32_t first[N + 1];  // chunks before the tensor's
  uint32_t ordinal[N];    // its place in the caller's list
  int8_t head[N];         // elements before the first that all of its arrays have on 16 bytes; -1: none
};
static_assert(sizeof(Table<kManyTensors>) + sizeof(AdamwStep) + 64 <= 32764, "a launch's argument");

__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x9E3779B9u;  // odd: leading bits of the golden ratio
  x ^= x >> 15;
  x *= 0x6A09E667u;  // odd: leading bits of the root of two
  return x ^ (x >> 16);
}

// Eight neighbouring values; the first `n` of them where the address is not the vector's.
template <class T>
__device__ __forceinline__ void load8(const T* p, bool vec, int n, float (&f)[kEach]);
template <>
__device__ __forceinline__ void load8(const float* p, bool vec, int n, float (&f)[kEach]) {
  if (vec) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) f[i] = i < n ? p[i] : 0.f;
  }
}
struct Bf16 {
  uint16_t bits;
};
struct F16 {
  uint16_t bits;
};
struct E4m3 {
  uint8_t bits;
};
__device__ __forceinline__ float to_float(Bf16 x) { return __uint_as_float((uint32_t)x.bits << 16); }
__device__ __forceinline__ float to_float(F16 x) { return __half2float(__ushort_as_half(x.bits)); }
template <class T>
__device__ __forceinline__ void load8_half(const T* p, bool vec, int n, float (&f)[kEach]) {
  T t[kEach];
  if (vec) {
    *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) t[i] = i < n ? p[i] : T{0};
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) f[i] = to_float(t[i]);
}
template <>
__device__ __forceinline__ void load8(const Bf16* p, bool vec, int n, float (&f)[kEach]) {
  load8_half(p, vec, n, f);
}
template <>
__device__ __forceinline__ void load8(const F16* p, bool vec, int n, float (&f)[kEach]) {
  load8_half(p, vec, n, f);
}
// e4m3 is the upper byte of a half, less the half's bias: exact
__device__ __forceinline__ void codes_to_float(const uint32_t (&w)[2], float (&f)[kEach]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint16_t two = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(two));
    const float2 f2 = __half22float2(*reinterpret_cast<const __half2*>(&h2));
    f[2 * i] = f2.x, f[2 * i + 1] = f2.y;
  }
}
template <>
__device__ __forceinline__ void load8(const E4m3* p, bool vec, int n, float (&f)[kEach]) {
  uint32_t w[2] = {0, 0};
  if (vec) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x, w[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (i < n) w[i / 4] |= (uint32_t)p[i].bits << (8 * (i & 3));
  }
  codes_to_float(w, f);
}

template <class T>
__device__ __forceinline__ void store8(T* p, bool vec, int n, const float (&f)[kEach]);
template <>
__device__ __forceinline__ void store8(float* p, bool vec, int n, const float (&f)[kEach]) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (i < n) p[i] = f[i];
  }
}
__device__ __forceinline__ void store8_half(void* p, bool vec, int n, const uint32_t (&w)[4]) {
  if (vec) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (i < n) static_cast<uint16_t*>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
  }
}
template <>
__device__ __forceinline__ void store8(Bf16* p, bool vec, int n, const float (&f)[kEach]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = f2_to_bf2(make_float2(f[2 * i], f[2 * i + 1]));
  store8_half(p, vec, n, w);
}
template <>
__device__ __forceinline__ void store8(F16* p, bool vec, int n, const float (&f)[kEach]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  store8_half(p, vec, n, w);
}

// Pairs of neighbouring values.
__device__ __forceinline__ float2 pair_of(const float (&f)[kEach], int i) { return make_float2(f[2 * i], f[2 * i + 1]); }

// The scale of a group of 128 values, 8 lanes with 16 each; NaN counts as nothing.
__device__ __forceinline__ float group_scale(const float2 (&x)[2][4]) {
  float amax = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) amax = fmaxf(fmaxf(amax, fabsf(x[h][i].x)), fabsf(x[h][i].y));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  return amax <= 3.4e38f ? make_scale(amax, false, kMinState) : amax;
}

// The code of y >= 0 in the upper byte; y: the value over its scale times 2^-120,
// bits: 16 random ones from bit 8 on. They are added below the three bits of
// mantissa that stay and the rest is cut off. All in integers: 2^-120 brings the
// least normal code, 2^-6, to fp32's least normal value, so that both have their
// subnormal codes at the same bits. The largest value is 448 (1 + 2^-23) and
// cannot carry past its code.
__device__ __forceinline__ uint32_t code_of(float y, uint32_t bits) {
  return (min(__float_as_uint(y), 0x07f00000u) << 4) + bits;  // NaN: code 0x7f
}
__device__ __forceinline__ uint32_t signed_code(float x, float rs, uint32_t bits) {
  const uint32_t v = code_of(__fmul_rn(__fmul_rn(fabsf(x), rs), 0x1p-120f), bits);
  return v | (__float_as_uint(x) & 0x80000000u);
}
// Of a root: two at a time, and never zero for one above zero.
__device__ __forceinline__ void root_codes(float2 x, float rs, uint32_t bits0, uint32_t bits1, uint32_t& v0,
                                           uint32_t& v1) {
  const float2 y = __fmul2_rn(__fmul2_rn(x, make_float2(rs, rs)), make_float2(0x1p-120f, 0x1p-120f));
  v0 = code_of(y.x, bits0), v1 = code_of(y.y, bits1);
  if (x.x > 0.f) v0 = max(v0, 0x01000000u);
  if (x.y > 0.f) v1 = max(v1, 0x01000000u);
}
__device__ __forceinline__ uint32_t upper_bytes(const uint32_t (&v)[kEach], int i) {
  return __byte_perm(__byte_perm(v[i], v[i + 1], 0x0073), __byte_perm(v[i + 2], v[i + 3], 0x0073), 0x5410);
}
__device__ __forceinline__ void store8(E4m3* p, bool vec, int n, const uint32_t (&v)[kEach]) {
  const uint2 w = make_uint2(upper_bytes(v, 0), upper_bytes(v, 4));
  if (vec) {
    *reinterpret_cast<uint2*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (i < n) p[i].bits = (uint8_t)(v[i] >> 24);
  }
}

// What a step's constants are, made by one thread; 1 - b^t in 64 bits: in 32 its
// first digits are gone while b^t is near one.
struct Factors {
  float keep, root, rate;  // of p, of sqrt(v'), of the update
  uint32_t key;
};
__device__ __forceinline__ void make_factors(const AdamwStep& a, Factors& f) {
  const double lr = a.lr_ptr != nullptr ? (double)*a.lr_ptr : a.lr;
  const int64_t step = a.step_ptr != nullptr ? *a.step_ptr : a.step;
  f.keep = (float)(1.0 - lr * a.decay);
  if (a.step_ptr != nullptr) {
    f.root = (float)rsqrt(1.0 - pow(a.beta2, (double)step));
    f.rate = (float)(lr / (1.0 - pow(a.beta1, (double)step)));
  } else {
    f.root = a.root;
    f.rate = (float)(lr / a.bias1);
  }
  f.key = mix(a.seed_key ^ (uint32_t)step);
}

// The last tensor whose chunks begin at `chunk` or before.
template <int N>
__device__ __forceinline__ int tensor_at(const Table<N>& t, int tensors, uint32_t chunk) {
  int lo = 0, hi = tensors;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A chunk of tensor i from element `begin` on, vectors where `vec`. WHOLE: all of its
// elements are there and on the vectors' boundaries, so that nothing in it branches.
// States in 32 bits: tensors inside of a buffer that begin between vectors have their
// first chunk behind `head` elements, which go one by one.
struct Chunk {
  int i, count;
  bool vec;
  int64_t begin;
};
template <int N>
__device__ __forceinline__ Chunk chunk_at(const Table<N>& t, int i, uint32_t chunk) {
  Chunk k;
  k.i = i;
  k.vec = t.head[k.i] >= 0;
  k.begin = (int64_t)(chunk - t.first[k.i]) * kChunk + max((int)t.head[k.i], 0);
  k.count = (int)min((int64_t)kChunk, t.n[k.i] - k.begin);
  return k;
}

// The first chunk of CTA `cta`.
__device__ __forceinline__ uint32_t run_begin(uint32_t chunks, uint32_t cta) {
  return (uint32_t)((uint64_t)chunks * cta / gridDim.x);
}

template <class P, class G, bool WHOLE, int N>
__device__ __forceinline__ void step_values(const Table<N>& t, const Chunk& k, const AdamwStep& a, const Factors& f,
                                            float c) {
  const G* g = static_cast<const G*>(t.g[k.i]) + k.begin;
  P* p = static_cast<P*>(t.p[k.i]) + k.begin;
  float *m = static_cast<float*>(t.m[k.i]) + k.begin, *v = static_cast<float*>(t.v[k.i]) + k.begin;
#pragma unroll
  for (int at = (int)threadIdx.x * kEach, step = 0; step < kChunk / (kThreads * kEach); ++step, at += kThreads * kEach) {
    const int n = WHOLE ? kEach : min(kEach, k.count - at);
    if (!WHOLE && n <= 0) break;
    const bool vec = WHOLE || (k.vec && n == kEach);
    float pf[kEach], gf[kEach], mf[kEach], vf[kEach];
    load8(g + at, vec, n, gf);
    load8(p + at, vec, n, pf);
    load8(m + at, vec, n, mf);
    load8(v + at, vec, n, vf);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const float gc = __fmul_rn(gf[i], c);
      mf[i] = __fadd_rn(__fmul_rn(a.b1, mf[i]), __fmul_rn(a.c1, gc));
      vf[i] = __fadd_rn(__fmul_rn(a.b2, vf[i]), __fmul_rn(a.c2, __fmul_rn(gc, gc)));
      const float d = __fadd_rn(__fmul_rn(__fsqrt_rn(vf[i]), f.root), a.eps);
      pf[i] = __fsub_rn(__fmul_rn(pf[i], f.keep), __fmul_rn(f.rate, __fdiv_rn(mf[i], d)));
    }
    store8(p + at, vec, n, pf);
    store8(m + at, vec, n, mf);
    store8(v + at, vec, n, vf);
  }
}

template <class P, class G, int N>
__global__ void __launch_bounds__(kThreads, kCtas)
    adamw_kernel(const __grid_constant__ Table<N> t, int tensors, const AdamwStep a) {
  __shared__ Factors shared;
  griddep_wait();
  griddep_launch_dependents();
  if (threadIdx.x == 0) make_factors(a, shared);
  __syncthreads();
  const Factors f = shared;
  const float c = a.clip != nullptr ? *a.clip : 1.f;
  for (uint32_t chunk = blockIdx.x; chunk < t.first[tensors]; chunk += gridDim.x) {
    Chunk k = chunk_at(t, tensor_at(t, tensors, chunk), chunk);
    if (k.vec && k.count == kChunk) step_values<P, G, true>(t, k, a, f, c);
    else step_values<P, G, false>(t, k, a, f, c);
    if (t.head[k.i] > 0 && chunk == t.first[k.i]) {
      k.begin = 0, k.count = (int)min((int64_t)t.head[k.i], t.n[k.i]), k.vec = false;
      step_values<P, G, false>(t, k, a, f, c);
    }
  }
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// Of zero or of at least 2^-75 (the root of fp32's least value) as it is used here.
__device__ __forceinline__ float fast_reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// RN(sqrt(a)) of zeros and of 2^-96 to 2^96 in pairs, by Markstein's iteration (P.
// Markstein, IBM J. Res. Dev. 34(1), 1990): from y = 1 / sqrt(a) within two ulps,
// g = a y and h = y / 2, r = 1/2 - g h, g1 = g + g r, h1 = h + h r, and g1 + (a - g1^2) h1
// is correctly rounded: tests/test_adamw_capi.py goes through every mantissa and
// start. Half the instructions of the general root. (Signs as they save negations.)
__device__ __forceinline__ float2 exact_roots(float2 a) {
  float2 y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(a.x));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(a.y));
  y = make_float2(fminf(y.x, 0x1p60f), fminf(y.y, 0x1p60f));  // of a zero: g = 0, and the rest of the steps too
  const float2 g = __fmul2_rn(a, y), nh = __fmul2_rn(y, both(-0.5f)), r = __ffma2_rn(g, nh, both(0.5f));
  const float2 g1 = __ffma2_rn(g, r, g), nh1 = __ffma2_rn(nh, r, nh);
  return __ffma2_rn(__ffma2_rn(g1, g1, __fmul2_rn(a, both(-1.f))), nh1, g1);
}
// Whether all of 8 values are zero or in that range.
__device__ __forceinline__ bool plain_range(const float2 (&a)[4]) {
  uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = __float_as_uint(a[i].x), y = __float_as_uint(a[i].y);
    lo = min(lo, min(x - 1u, y - 1u)), hi = max(hi, max(x, y));
  }
  return lo >= 0x0f800000u - 1u && hi <= 0x6f800000u;
}

template <class P, class G, bool WHOLE, int N>
__device__ __forceinline__ void step_codes(const Table<N>& t, const Chunk& k, const AdamwStep& a, const Factors& f,
                                           float c) {
  const float2 c2 = both(c), b1 = both(a.b1), b2 = both(a.b2), g_m = both(a.c1), g_v = both(a.c2);
  const float2 keep = both(f.keep), root = both(f.root), rate = both(-f.rate), eps = both(a.eps);
  const int at = ((int)threadIdx.x >> 3) * kGroup + ((int)threadIdx.x & 7) * kEach;
  const int64_t from = k.begin + at, group = k.begin / kGroup + ((int)threadIdx.x >> 3);
  const G* g = static_cast<const G*>(t.g[k.i]) + from;
  P* p = static_cast<P*>(t.p[k.i]) + from;
  E4m3 *m = static_cast<E4m3*>(t.m[k.i]) + from, *v = static_cast<E4m3*>(t.v[k.i]) + from;
  // whole warps go on: the lanes of a group exchange their maxima
  const int n[2] = {WHOLE ? kEach : max(0, min(kEach, k.count - at)), WHOLE ? kEach : max(0, min(kEach, k.count - at - 64))};
  const bool vec[2] = {WHOLE || (k.vec && n[0] == kEach), WHOLE || (k.vec && n[1] == kEach)};
  float ms = 0.f, rs = 0.f;
  float gf[2][kEach], pf[2][kEach], mf[2][kEach], rf[2][kEach];
  if (n[0] > 0) ms = t.ms[k.i][group], rs = t.vs[k.i][group];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    load8(g + 64 * h, vec[h], n[h], gf[h]);
    load8(p + 64 * h, vec[h], n[h], pf[h]);
    load8(m + 64 * h, vec[h], n[h], mf[h]);
    load8(v + 64 * h, vec[h], n[h], rf[h]);
  }
  float2 m2[2][4], r2[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float out[kEach];
    float2 v2[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // what becomes codes is rounded as written: products in pairs, sums one by one
      // (a sum in pairs would be fused with the product before it)
      const float2 gi = __fmul2_rn(pair_of(gf[h], i), c2), r = __fmul2_rn(pair_of(rf[h], i), both(rs));
      const float2 m = __fmul2_rn(b1, __fmul2_rn(pair_of(mf[h], i), both(ms))), mg = __fmul2_rn(g_m, gi);
      const float2 v = __fmul2_rn(b2, __fmul2_rn(r, r)), vg = __fmul2_rn(g_v, __fmul2_rn(gi, gi));
      m2[h][i] = make_float2(__fadd_rn(m.x, mg.x), __fadd_rn(m.y, mg.y));
      v2[i] = make_float2(__fadd_rn(v.x, vg.x), __fadd_rn(v.y, vg.y));
    }
    if (plain_range(v2)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) r2[h][i] = exact_roots(v2[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) r2[h][i] = make_float2(__fsqrt_rn(v2[i].x), __fsqrt_rn(v2[i].y));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 d = __ffma2_rn(r2[h][i], root, eps);
      const float2 u = __fmul2_rn(m2[h][i], make_float2(fast_reciprocal(d.x), fast_reciprocal(d.y)));
      const float2 q = __ffma2_rn(u, rate, __fmul2_rn(pair_of(pf[h], i), keep));
      out[2 * i] = q.x, out[2 * i + 1] = q.y;
    }
    store8(p + 64 * h, vec[h], n[h], out);
  }
  const float m_scale = group_scale(m2), r_scale = group_scale(r2);
  if ((threadIdx.x & 7) == 0 && n[0] > 0) t.ms[k.i][group] = m_scale, t.vs[k.i][group] = r_scale;
  const float m_rcp = __frcp_rn(m_scale), r_rcp = __frcp_rn(r_scale);
  const uint32_t key = mix(f.key ^ t.ordinal[k.i]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t mv[kEach], rv[kEach];
#pragma unroll
    for (int i = 0; i < kEach; i += 2) {
      const uint32_t b0 = mix((uint32_t)(from + 64 * h + i) * 0x9E3779B9u + key);
      const uint32_t b1 = mix((uint32_t)(from + 64 * h + i + 1) * 0x9E3779B9u + key);
      mv[i] = signed_code(m2[h][i / 2].x, m_rcp, __byte_perm(b0, 0, 0x4104));
      mv[i + 1] = signed_code(m2[h][i / 2].y, m_rcp, __byte_perm(b1, 0, 0x4104));
      root_codes(r2[h][i / 2], r_rcp, __byte_perm(b0, 0, 0x4324), __byte_perm(b1, 0, 0x4324), rv[i], rv[i + 1]);
    }
    store8(m + 64 * h, vec[h], n[h], mv);
    store8(v + 64 * h, vec[h], n[h], rv);
  }
}

// The chunk from element `at` on into the L2, while the one before it is computed.
template <class P, class G, int N>
__device__ __forceinline__ void fetch_next(const Table<N>& t, int i, int64_t at) {
  const uint32_t n = (uint32_t)min((int64_t)kChunk, t.n[i] - at) & ~15u;
  auto fetch = [](const void* p, uint32_t bytes) {
    if (bytes > 0 && reinterpret_cast<uint64_t>(p) % 16 == 0)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
  };
  fetch(static_cast<const P*>(t.p[i]) + at, n * (uint32_t)sizeof(P));
  fetch(static_cast<const G*>(t.g[i]) + at, n * (uint32_t)sizeof(G));
  fetch(static_cast<const E4m3*>(t.m[i]) + at, n);
  fetch(static_cast<const E4m3*>(t.v[i]) + at, n);
}

template <class P, class G, int N>
__global__ void __launch_bounds__(kThreads, kCodesCtas)
    adamw_codes_kernel(const __grid_constant__ Table<N> t, int tensors, const AdamwStep a) {
  __shared__ Factors shared;
  griddep_wait();
  griddep_launch_dependents();
  if (threadIdx.x == 0) make_factors(a, shared);
  __syncthreads();
  const Factors f = shared;
  const float c = a.clip != nullptr ? *a.clip : 1.f;
  const uint32_t end = run_begin(t.first[tensors], blockIdx.x + 1);
  uint32_t chunk = run_begin(t.first[tensors], blockIdx.x);
  for (int i = tensor_at(t, tensors, chunk); chunk < end; ++chunk) {
    while (t.first[i + 1] <= chunk) ++i;
    const Chunk k = chunk_at(t, i, chunk);
    if (threadIdx.x == 0 && chunk + 1 < end && chunk + 1 < t.first[i + 1] && k.vec)
      fetch_next<P, G>(t, i, k.begin + kChunk);
    if (k.vec && k.count == kChunk)
      step_codes<P, G, true>(t, k, a, f, c);
    else
      step_codes<P, G, false>(t, k, a, f, c);
  }
}

// The first element that starts a vector of 8 in each of the arrays (codes: element 0
// or none, a group of 128 is the tensor's own); -1 where there is none.
template <class P, class G, bool CODES>
int head_of(const void* p, const void* g, const void* m, const void* v) {
  auto bits = [](const void* x) { return reinterpret_cast<uint64_t>(x); };
  for (int h = 0; h < (CODES ? 1 : kEach); ++h) {
    const uint64_t wide = (bits(p) + h * sizeof(P)) | (bits(g) + h * sizeof(G)) |
                          (CODES ? 0 : (bits(m) + h * sizeof(float)) | (bits(v) + h * sizeof(float)));
    if (wide % 16 == 0 && (!CODES || (bits(m) | bits(v)) % 8 == 0)) return h;
  }
  return -1;
}

template <class P, class G, bool CODES, int N>
cudaError_t launch_table(const AdamwTensors& l, const AdamwStep& step, cudaStream_t stream) {
  Table<N> t;
  int64_t from = 0;
  while (from < l.count) {
    int k = 0;
    uint64_t chunks = 0;
    for (; from < l.count && k < N; ++from) {
      const int64_t n = l.n[from];
      if (n == 0) continue;
      const int head = head_of<P, G, CODES>(l.p[from], l.g[from], l.m[from], l.v[from]);
      const uint64_t rest = head > 0 && n > head ? n - head : n, mine = (rest + kChunk - 1) / kChunk;
      if (chunks + mine > INT32_MAX) break;  // checked: one tensor's fit
      t.g[k] = l.g[from], t.p[k] = l.p[from], t.m[k] = l.m[from], t.v[k] = l.v[from];
      t.ms[k] = CODES ? l.ms[from] : nullptr, t.vs[k] = CODES ? l.vs[from] : nullptr;
      t.n[k] = n;
      t.first[k] = (uint32_t)chunks;
      t.ordinal[k] = (uint32_t)from;
      t.head[k] = (int8_t)head;
      chunks += mine;
      ++k;
    }
    if (k == 0) continue;
    t.first[k] = (uint32_t)chunks;
    // CTAs in turn, not one round: chunks deal out evenly (20M fp32 in 200 tensors: 2
    // rounds 107 us, 16 98); with codes runs of some length
    const uint64_t most = (uint64_t)(CODES ? 5 * kCodesCtas : 16 * kCtas) * device_sm_count();
    const unsigned grid = (unsigned)(chunks < most ? chunks : most);
    auto kernel = CODES ? adamw_codes_kernel<P, G, N> : adamw_kernel<P, G, N>;
    const cudaError_t e = launch_pdl(kernel, grid, kThreads, 0, stream, t, k, step);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <class P, class G, bool CODES>
cudaError_t launch_list(const AdamwTensors& l, const AdamwStep& a, cudaStream_t stream) {
  return l.count <= kFewTensors ? launch_table<P, G, CODES, kFewTensors>(l, a, stream)
                                : launch_table<P, G, CODES, kManyTensors>(l, a, stream);
}

template <class P, class G>
cudaError_t launch_states(const AdamwTensors& l, const AdamwStep& a, cudaStream_t stream) {
  return l.ms != nullptr ? launch_list<P, G, true>(l, a, stream) : launch_list<P, G, false>(l, a, stream);
}

uint32_t mix_host(uint32_t x) {
  x ^= x >> 16;
  x *= 0x9E3779B9u;
  x ^= x >> 15;
  x *= 0x6A09E667u;
  return x ^ (x >> 16);
}

}  // namespace

uint32_t adamw_seed_key(uint64_t seed) { return mix_host((uint32_t)seed ^ mix_host((uint32_t)(seed >> 32))); }

// Parameters' and gradients' types: the same, fp32 gradients, or bf16 ones of fp32 parameters.
cudaError_t adamw(const AdamwTensors& l, const AdamwStep& a, cudaStream_t stream) {
  if (l.p_dtype == CUTIE_DTYPE_F32)
    return l.g_dtype == CUTIE_DTYPE_F32 ? launch_states<float, float>(l, a, stream)
                                        : launch_states<float, Bf16>(l, a, stream);
  if (l.p_dtype == CUTIE_DTYPE_BF16)
    return l.g_dtype == CUTIE_DTYPE_F32 ? launch_states<Bf16, float>(l, a, stream)
                                        : launch_states<Bf16, Bf16>(l, a, stream);
  return l.g_dtype == CUTIE_DTYPE_F32 ? launch_states<F16, float>(l, a, stream)
                                      : launch_states<F16, F16>(l, a, stream);
}

}  // namespace cutie
