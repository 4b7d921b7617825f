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

// Sources of a panel's values, 8 at a time: the i-th 8 values of the [tokens, features] array (features is
// a multiple of 8).
struct PlainSource {
  const float* x;
  long long features;
  int vec;             // x is 16-byte aligned
  static constexpr int parts = 1;
  __device__ __forceinline__ void load(long long i, float (&v)[1][8]) const { load8(x + 8 * i, vec, v[0]); }
};
// dG = dH U act'(G) and dU = dH act(G); two panels one behind the other.
struct GateSource {
  const float *G, *U, *dH;
  long long features;
  int vec, act;
  static constexpr int parts = 2;
  __device__ __forceinline__ void load(long long i, float (&v)[2][8]) const {
    const long long o = 8 * i;
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

// Place i = (tile groups + g) R + r of a panel, i going up by `step`: divisions only at the start.
struct PanelWalk {
  long long g, tile, step_g, step_tile, groups;
  int r, step_r, R;
  __device__ __forceinline__ PanelWalk(long long first, long long step, int R_, long long groups_)
      : groups(groups_), R(R_) {
    const long long q = first / R, sq = step / R;
    r = int(first - q * R);
    step_r = int(step - sq * R);
    tile = q / groups;
    g = q - tile * groups;
    step_tile = sq / groups;
    step_g = sq - step_tile * groups;
  }
  __device__ __forceinline__ void next() {
    r += step_r;
    g += step_g;
    tile += step_tile;
    if (r >= R) {
      r -= R;
      ++g;
    }
    if (g >= groups) {
      g -= groups;
      ++tile;
    }
  }
};

// A panel cut into blocks of tt tokens (a power of two up to 32) x gg groups, tt gg = units.
struct PanelBlocks {
  int tt, tt_log, gg, gg_log, r_blocks, R;
  long long groups, g_blocks, items;
  struct Place {
    long long tile, g;
    int r;
  };
  __device__ __forceinline__ PanelBlocks(int R_, int tiles, long long groups_, int units) : R(R_), groups(groups_) {
    tt_log = R <= 1 ? 0 : min(5, 32 - __clz(R - 1));
    tt = 1 << tt_log;
    gg = units >> tt_log;
    gg_log = 31 - __clz(gg);
    r_blocks = (R + tt - 1) >> tt_log;
    g_blocks = (groups + gg - 1) >> gg_log;
    items = g_blocks * r_blocks * tiles;
  }
  __device__ __forceinline__ Place place(long long item) const {
    const long long q = item / g_blocks;
    return {q / r_blocks, (item - q * g_blocks) << gg_log, int(q % r_blocks) << tt_log};
  }
  // place of (token, group) in shared memory: tokens neighbouring, shifted by the group so that both the
  // writing along groups and the reading along tokens spread over the banks
  __device__ __forceinline__ int slot(int t, int g) const { return (g << tt_log) + ((t + g) & (tt - 1)); }
};

// The largest finite magnitude of a thread's groups.
template <class Source>
__device__ __forceinline__ float largest(const Source& src, long long tokens, long long first, long long step) {
  const long long n = tokens * (src.features >> 3);
  float m = 0.0f;
  for (long long i = first; i < n; i += step) {
    float v[Source::parts][8];
    src.load(i, v);
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
  const long long groups = src.features >> 3;
  for (PanelWalk w(first, step, R, groups); w.tile < tiles; w.next()) {
    const int r = w.r;
    const long long g = w.g, tile = w.tile, t = tile * R + r;
    float v[Source::parts][8] = {};
    if (t < tokens) src.load(t * groups + g, v);
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

// One panel to make: tiles of R tokens, largest magnitudes, pairs and exponent.
template <class Source>
struct PanelJob {
  Source src;
  int R, tiles;
  int amax_ctas, pair_ctas;
  float* partial;
  uint4* out;
  int* exponent;
};

template <class Source>
__device__ __forceinline__ void panel_amax(const PanelJob<Source>& j, long long tokens, int cta) {
  const float m = cta_max(largest(j.src, tokens, cta * 256ll + threadIdx.x, j.amax_ctas * 256ll));
  if (threadIdx.x == 0) j.partial[cta] = m;
}

// A block of TT tokens (a power of two) x GG groups at a time goes through shared memory: read along the
// features, written along the tokens, whole lines both ways.
constexpr int kPanelUnits = 1024;  // 8-value pieces of all parts
template <class Source>
__device__ __forceinline__ void panel_pairs(const PanelJob<Source>& j, long long tokens, int cta,
                                            uint4 (&buf)[2 * kPanelUnits]) {
  constexpr int P = Source::parts, UNITS = kPanelUnits / P;
  const int e = partial_exponent(j.partial, j.amax_ctas), R = j.R;
  if (cta == 0 && threadIdx.x == 0) *j.exponent = e;
  const float s = pow2(e);
  const PanelBlocks b(R, j.tiles, j.src.features >> 3, UNITS);
  for (long long item = cta; item < b.items; item += j.pair_ctas) {
    const PanelBlocks::Place at = b.place(item);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < UNITS / 256; ++k) {
      const int u = threadIdx.x + 256 * k, t = u >> b.gg_log, g = u & (b.gg - 1);
      const long long token = at.tile * R + at.r + t;
      float v[P][8] = {};
      if (at.r + t < R && token < tokens && at.g + g < b.groups) j.src.load(token * b.groups + at.g + g, v);
#pragma unroll
      for (int q = 0; q < P; ++q) {
        uint4* place = buf + 2 * q * UNITS + b.slot(t, g);
        to_pair8(v[q], s, place[0], place[UNITS]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < UNITS / 256; ++k) {
      const int u = threadIdx.x + 256 * k, t = u & (b.tt - 1), g = u >> b.tt_log;
      if (at.r + t >= R || at.g + g >= b.groups) continue;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        const uint4* place = buf + 2 * q * UNITS + b.slot(t, g);
        uint4* o = j.out + ((at.tile * P + q) * b.groups + at.g + g) * 2 * R + at.r + t;
        o[0] = place[0];
        o[R] = place[UNITS];
      }
    }
  }
}

// One panel, or two at once (the CTAs behind the first's), in two launches: largest magnitudes, then pairs.
template <class A, class C>
__global__ void __launch_bounds__(256) panel_amax_kernel(PanelJob<A> a, PanelJob<C> c, long long tokens) {
  griddep_launch_dependents();
  const int cta = blockIdx.x;
  if (cta < a.amax_ctas) panel_amax(a, tokens, cta);
  else panel_amax(c, tokens, cta - a.amax_ctas);
}
template <class A, class C>
__global__ void __launch_bounds__(256) panel_pair_kernel(PanelJob<A> a, PanelJob<C> c, long long tokens) {
  __shared__ uint4 buf[2 * kPanelUnits];
  griddep_launch_dependents();
  griddep_wait();
  const int cta = blockIdx.x;
  if (cta < a.pair_ctas) panel_pairs(a, tokens, cta, buf);
  else panel_pairs(c, tokens, cta - a.pair_ctas, buf);
}

// Small panels in one launch: a cluster of kSmallCtas CTAs for each, which exchange their largest magnitudes
// through distributed shared memory and read their values a second time from the caches. Against the two
// kernels it saves a launch; above kSmallGroups 8-value groups its few SMs cost more than that.
constexpr int kSmallCtas = 8, kSmallThreads = 512;
constexpr int64_t kSmallGroups = 32768;
template <class Source>
__device__ __forceinline__ void panel_small(const PanelJob<Source>& j, long long tokens, float* maxima) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = int(blockIdx.x % kSmallCtas);
  const long long first = cta * (long long)kSmallThreads + threadIdx.x;
  const long long step = (long long)kSmallCtas * kSmallThreads;
  float m = cta_max(largest(j.src, tokens, first, step));
  if (threadIdx.x < kSmallCtas) *cluster.map_shared_rank(&maxima[cta], threadIdx.x) = m;
  cluster.sync();
#pragma unroll
  for (int i = 0; i < kSmallCtas; ++i) m = fmaxf(m, maxima[i]);
  const int e = pair_exponent(m);
  if (cta == 0 && threadIdx.x == 0) *j.exponent = e;
  write_pairs(j.src, tokens, j.R, j.tiles, pow2(e), j.out, first, step);
}
template <class A, class C>
__global__ void __cluster_dims__(kSmallCtas) __launch_bounds__(kSmallThreads)
    panel_small_kernel(PanelJob<A> a, PanelJob<C> c, long long tokens) {
  __shared__ float maxima[kSmallCtas];
  griddep_launch_dependents();
  if (blockIdx.x < kSmallCtas) panel_small(a, tokens, maxima);
  else panel_small(c, tokens, maxima);
}

}  // namespace vbsr_b200
