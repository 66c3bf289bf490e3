// AdamW over many tensors in one launch (sm_100a). For each element, in fp32
// with every product and sum rounded by itself:
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
// Bound: memory, each value once. CTAs walk chunks of 4096 elements of one
// tensor, found by a search in the table that is the kernel's argument (no copy
// to the GPU, nothing to keep for a graph); a thread takes 8 neighbouring
// elements at a time, 16 lanes a group of 128.
#include <cuda_fp16.h>

#include "cutie.h"
#include "launch.cuh"

namespace cutie {
namespace {

constexpr int kThreads = 256, kEach = 8, kChunk = 4096, kGroup = 128;
constexpr int kCtas = 8;  // an SM, at most
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

// A magnitude at most 448 to one of its neighbours in e4m3 by 16 random bits: added
// below the three bits of mantissa that stay, the rest cut off. Subnormal codes
// have the spacing of the first binade, so they are rounded one binade up.
__device__ __forceinline__ float round8(float y, uint32_t bits) {
  const float up = y < 0x1p-6f ? 0x1p-6f : 0.f;
  const float z = __uint_as_float((__float_as_uint(__fadd_rn(y, up)) + (bits << 4)) & 0xfff00000u);
  return fminf(__fsub_rn(z, up), 448.f);
}

// Codes and scale of a group of 128 elements, 16 lanes with 8 each; bits: 16 random ones an element.
template <bool POSITIVE>
__device__ __forceinline__ void store_state(E4m3* p, float* scale, bool vec, int n, bool first,
                                            const float (&x)[kEach], const uint32_t (&bits)[kEach]) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) amax = fmaxf(amax, i < n ? fabsf(x[i]) : 0.f);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const float s = fmaxf(__fdiv_rn(amax, 448.f), kMinState), rs = __fdiv_rn(1.f, s);
  uint32_t w[2];
  float z[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const float y = __fmul_rn(fabsf(x[i]), rs);
    z[i] = round8(y, bits[i]);
    if (POSITIVE && x[i] > 0.f) z[i] = fmaxf(z[i], 0x1p-9f);
    if (!(y == y)) z[i] = y;  // NaN stays
    if (!POSITIVE) z[i] = copysignf(z[i], x[i]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = f4_to_e4m3x4(make_float2(z[4 * i], z[4 * i + 1]), make_float2(z[4 * i + 2], z[4 * i + 3]));
  if (first && n > 0) *scale = s;
  if (vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (i < n) p[i].bits = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ bool on16(const void* p) { return (reinterpret_cast<uint64_t>(p) & 15u) == 0; }

template <class P, class G, bool CODES, int N>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<N> t, int tensors,
                                                         const AdamwStep a) {
  __shared__ float factor[3];  // of the decay, of the root, of the update
  __shared__ uint32_t step_key;
  griddep_wait();
  griddep_launch_dependents();
  if (threadIdx.x == 0) {
    // 1 - b^t in 64 bits: in 32 its first digits are gone while b^t is near one
    const int64_t step = a.step_ptr != nullptr ? *a.step_ptr : a.step;
    const double lr = a.lr_ptr != nullptr ? (double)*a.lr_ptr : a.lr;
    factor[0] = (float)(1.0 - lr * a.decay);
    if (a.step_ptr != nullptr) {
      factor[1] = (float)rsqrt(1.0 - pow(a.beta2, (double)step));
      factor[2] = (float)(lr / (1.0 - pow(a.beta1, (double)step)));
    } else {
      factor[1] = a.root;
      factor[2] = (float)(lr / a.bias1);
    }
    step_key = mix(a.seed_key ^ (uint32_t)step);
  }
  __syncthreads();
  const float c = a.clip != nullptr ? *a.clip : 1.f;
  const float b1 = a.b1, b2 = a.b2, c1 = a.c1, c2 = a.c2;
  const float eps = a.eps, keep = factor[0], root = factor[1], rate = factor[2];
  using S = typename std::conditional<CODES, E4m3, float>::type;
  for (uint32_t chunk = blockIdx.x; chunk < t.first[tensors]; chunk += gridDim.x) {
  int lo = 0, hi = tensors;  // the last tensor whose chunks begin at this one or before
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  const int64_t begin = (int64_t)(chunk - t.first[lo]) * kChunk, size = t.n[lo];
  const G* g = static_cast<const G*>(t.g[lo]) + begin;
  P* p = static_cast<P*>(t.p[lo]) + begin;
  const int count = (int)min((int64_t)kChunk, size - begin);
  S *m = static_cast<S*>(t.m[lo]) + begin, *v = static_cast<S*>(t.v[lo]) + begin;
  const bool vec_all = on16(g) && on16(p) &&
                       (CODES ? ((reinterpret_cast<uint64_t>(m) | reinterpret_cast<uint64_t>(v)) & 7u) == 0
                              : on16(m) && on16(v));
  const uint32_t key = CODES ? mix(step_key ^ t.ordinal[lo]) : 0u;
  // whole warps go on: the lanes of a group exchange their maxima
  for (int at = (int)threadIdx.x * kEach; at - (int)(threadIdx.x & 31) * kEach < count; at += kThreads * kEach) {
    const int n = max(0, min(kEach, count - at));
    const bool vec = vec_all && n == kEach;
    float pf[kEach], gf[kEach], mf[kEach], vf[kEach];
    float ms = 0.f, vs = 0.f;
    const int64_t group = (begin + at) / kGroup;
    if (n > 0) {
      load8(g + at, vec, n, gf);
      load8(p + at, vec, n, pf);
      load8(m + at, vec, n, mf);
      load8(v + at, vec, n, vf);
      if (CODES) ms = t.ms[lo][group], vs = t.vs[lo][group];
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) pf[i] = gf[i] = mf[i] = vf[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (CODES) {
        mf[i] = __fmul_rn(mf[i], ms);
        const float r = __fmul_rn(vf[i], vs);
        vf[i] = __fmul_rn(r, r);
      }
      const float gc = __fmul_rn(gf[i], c);
      mf[i] = __fadd_rn(__fmul_rn(b1, mf[i]), __fmul_rn(c1, gc));
      vf[i] = __fadd_rn(__fmul_rn(b2, vf[i]), __fmul_rn(c2, __fmul_rn(gc, gc)));
      const float r = __fsqrt_rn(vf[i]);
      const float d = __fadd_rn(__fmul_rn(r, root), eps);
      pf[i] = __fsub_rn(__fmul_rn(pf[i], keep), __fmul_rn(rate, __fdiv_rn(mf[i], d)));
      if (CODES) vf[i] = r;
    }
    if (n > 0) store8(p + at, vec, n, pf);
    if constexpr (CODES) {
      uint32_t low[kEach], high[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const uint32_t h = mix((uint32_t)(begin + at + i) * 0x9E3779B9u + key);
        low[i] = h & 0xffffu, high[i] = h >> 16;
      }
      const bool first = (threadIdx.x & 15) == 0;
      store_state<false>(m + at, t.ms[lo] + group, vec, n, first, mf, low);
      store_state<true>(v + at, t.vs[lo] + group, vec, n, first, vf, high);
    } else if (n > 0) {
      store8(m + at, vec, n, mf);
      store8(v + at, vec, n, vf);
    }
  }
  }
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
      const uint64_t mine = ((uint64_t)n + kChunk - 1) / kChunk;
      if (chunks + mine > INT32_MAX) break;  // checked: one tensor's fit
      t.g[k] = l.g[from], t.p[k] = l.p[from], t.m[k] = l.m[from], t.v[k] = l.v[from];
      t.ms[k] = CODES ? l.ms[from] : nullptr, t.vs[k] = CODES ? l.vs[from] : nullptr;
      t.n[k] = n;
      t.first[k] = (uint32_t)chunks;
      t.ordinal[k] = (uint32_t)from;
      chunks += mine;
      ++k;
    }
    if (k == 0) continue;
    t.first[k] = (uint32_t)chunks;
    const uint64_t most = (uint64_t)kCtas * device_sm_count();
    const cudaError_t e = launch_pdl(adamw_kernel<P, G, CODES, N>, (unsigned)(chunks < most ? chunks : most), kThreads,
                                     0, stream, t, k, step);
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
