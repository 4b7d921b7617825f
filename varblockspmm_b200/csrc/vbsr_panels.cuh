// vbsr_panels.cuh — the pre-passes of the block-sparse layer operators: fp32 panels to operand
// pairs (layout and reasons in vbsr_pair.cuh).
#pragma once
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "vbsr_lm.cuh"
#include "vbsr_ptx.cuh"

namespace vbsr_b200 {

// Largest finite magnitudes are found by a grid of kAmaxCtas CTAs, one partial result each; every CTA
// of the following kernel takes the maximum of them. No atomics and nothing to clear.
constexpr int kAmaxCtas = 592;  // four per SM

// Exponent that brings a largest magnitude into [2^14, 2^15); between -113 and 126, so that 2^e is a
// normal number (numbers that are all subnormal keep fewer bits, as they have fewer).
__device__ __forceinline__ int pair_exponent(float amax) {
  if (!(amax > 0.0f)) return 0;
  const int e = 14 - ilogbf(amax);
  return e < 126 ? e : 126;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < __int_as_float(0x7f800000) ? a : 0.0f;  // false for NaN too
}

// x s as a pair. An infinity or NaN has no finite rest: both parts are then not finite.
__device__ __forceinline__ void to_pair(float x, float s, __half& hi, __half& lo) {
  const float v = x * s;
  hi = __float2half_rn(v);
  lo = __float2half_rn((v - __half2float(hi)) * 2048.0f);
}
__device__ __forceinline__ void to_pair8(const float (&x)[8], float s, uint4& hi, uint4& lo) {
  __half h[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) to_pair(x[i], s, h[i], l[i]);
  hi = *reinterpret_cast<uint4*>(h);
  lo = *reinterpret_cast<uint4*>(l);
}

// Maximum over the CTA; every thread gets it.
__device__ __forceinline__ float cta_max(float v) {
  __shared__ float red[32];
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < int(blockDim.x >> 5); ++i) v = fmaxf(v, red[i]);
  return v;
}
__device__ __forceinline__ int partial_exponent(const float* partial, int count) {
  float v = 0.0f;
  for (int i = threadIdx.x; i < count; i += blockDim.x) v = fmaxf(v, partial[i]);
  return pair_exponent(cta_max(v));
}

__device__ __forceinline__ void load8(const float* p, int vec, float (&v)[8]) {
  if (vec) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __ldg(p + i);
  }
}

// Sources of a panel's values: 8 features from 8 g of token t.
struct PlainSource {
  const float* x;
  long long features;  // multiple of 8
  int vec;             // x is 16-byte aligned
  static constexpr int parts = 1;
  __device__ __forceinline__ void load(long long t, long long g, float (&v)[1][8]) const {
    load8(x + t * features + 8 * g, vec, v[0]);
  }
};
// dG = dH U act'(G) and dU = dH act(G); two panels one behind the other.
struct GateSource {
  const float *G, *U, *dH;
  long long features;
  int vec, act;
  static constexpr int parts = 2;
  __device__ __forceinline__ void load(long long t, long long g, float (&v)[2][8]) const {
    const long long o = t * features + 8 * g;
    float a[8], u[8], d[8];
    load8(G + o, vec, a);
    load8(U + o, vec, u);
    load8(dH + o, vec, d);
    with_act(act, [&](auto kind) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float val, der;
        act_both<decltype(kind)::value>(a[i], val, der);
        v[0][i] = d[i] * u[i] * der;
        v[1][i] = d[i] * val;
      }
    });
  }
};

// The largest finite magnitude of a thread's groups.
template <class Source>
__device__ __forceinline__ float largest(const Source& src, long long tokens, long long first, long long step) {
  const long long groups = src.features >> 3, n = tokens * groups;
  float m = 0.0f;
  for (long long i = first; i < n; i += step) {
    float v[Source::parts][8];
    src.load(i / groups, i % groups, v);
#pragma unroll
    for (int q = 0; q < Source::parts; ++q)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[q][j]));
  }
  return m;
}

// A thread's share of the panel in pairs: per tile of R tokens, part and 8-feature group, [R of hi]
// [R of lo'] rows of 16 bytes. Neighbouring threads take neighbouring tokens (512 contiguous bytes written
// per warp; each reads one whole 32-byte sector).
template <class Source>
__device__ __forceinline__ void write_pairs(const Source& src, long long tokens, int R, int tiles, float s,
                                            uint4* out, long long first, long long step) {
  const long long groups = src.features >> 3, n = groups * tiles * R;
  for (long long i = first; i < n; i += step) {
    const int r = int(i % R);
    const long long g = (i / R) % groups, tile = i / R / groups, t = tile * R + r;
    float v[Source::parts][8] = {};
    if (t < tokens) src.load(t, g, v);
#pragma unroll
    for (int q = 0; q < Source::parts; ++q) {
      uint4 hi, lo;
      to_pair8(v[q], s, hi, lo);
      uint4* o = out + ((tile * Source::parts + q) * groups + g) * 2 * R + r;
      o[0] = hi;
      o[R] = lo;
    }
  }
}

template <class Source>
__global__ void __launch_bounds__(256) panel_amax_kernel(Source src, long long tokens, float* partial) {
  griddep_launch_dependents();
  const float m = cta_max(largest(src, tokens, blockIdx.x * 256ll + threadIdx.x, gridDim.x * 256ll));
  if (threadIdx.x == 0) partial[blockIdx.x] = m;
}

template <class Source>
__global__ void __launch_bounds__(256) panel_pair_kernel(Source src, long long tokens, int R, int tiles,
                                                         const float* partial, int count, uint4* out,
                                                         int* exponent) {
  griddep_launch_dependents();
  griddep_wait();
  const int e = partial_exponent(partial, count);
  if (blockIdx.x == 0 && threadIdx.x == 0) *exponent = e;
  write_pairs(src, tokens, R, tiles, pow2(e), out, blockIdx.x * 256ll + threadIdx.x, gridDim.x * 256ll);
}

// Both in one launch for a small panel: one cluster of kSmallCtas CTAs, which exchange their largest
// magnitudes through distributed shared memory and read their values a second time from the caches. Against
// the two kernels it saves a launch; above kSmallGroups 8-value groups its few SMs cost more than that.
constexpr int kSmallCtas = 8, kSmallThreads = 512;
constexpr int64_t kSmallGroups = 32768;
template <class Source>
__global__ void __cluster_dims__(kSmallCtas) __launch_bounds__(kSmallThreads)
    panel_small_kernel(Source src, long long tokens, int R, int tiles, uint4* out, int* exponent) {
  __shared__ float maxima[kSmallCtas];
  griddep_launch_dependents();
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const long long first = blockIdx.x * (long long)kSmallThreads + threadIdx.x;
  const long long step = (long long)kSmallCtas * kSmallThreads;
  float m = cta_max(largest(src, tokens, first, step));
  if (threadIdx.x < kSmallCtas) *cluster.map_shared_rank(&maxima[blockIdx.x], threadIdx.x) = m;
  cluster.sync();
#pragma unroll
  for (int i = 0; i < kSmallCtas; ++i) m = fmaxf(m, maxima[i]);
  const int e = pair_exponent(m);
  if (blockIdx.x == 0 && threadIdx.x == 0) *exponent = e;
  write_pairs(src, tokens, R, tiles, pow2(e), out, first, step);
}

}  // namespace vbsr_b200
