// vbsr_panels.cuh — the pre-passes of the block-sparse layer operators: fp32 panels to operand
// pairs (layout and reasons in vbsr_pair.cuh).
#pragma once
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "vbsr_lm.cuh"
#include "vbsr_ptx.cuh"

namespace vbsr_b200 {

// Largest finite magnitudes are found by a grid of kAmaxCtas CTAs in partial results (of the weights one
// per CTA, of a token one per part), and the following kernel takes the maximum of them. No atomics and
// nothing to clear.
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

// The largest finite magnitude of groups first, first + step, ... of a token, over the lanes of a warp.
template <class Source>
__device__ __forceinline__ float largest(const Source& src, long long token, long long first, long long end,
                                         int step) {
  const long long row = token * (src.features >> 3);
  float m = 0.0f;
#pragma unroll 4
  for (long long g = first; g < end; g += step) {
    float v[Source::parts][8];
    src.load(row + g, v);
#pragma unroll
    for (int q = 0; q < Source::parts; ++q)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[q][j]));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// One panel to make. A token's exponent e brings its largest magnitude into [2^14, 2^15), so a token's
// accuracy does not depend on the others'; the output takes 2^e and the weights' power of two back with one
// factor, so that e is held where that is a normal number (products of largest magnitudes between 2^-98 and
// 2^154: smaller ones are held to 2^-147, larger ones overflow). Where tokens are summed over (the activations of the weight
// gradients, against gradients dY with exponents f) one exponent c has to serve all tokens of a stage: they
// are written with c - f, and c is the largest for which that is at most e for every token with a gradient.
// So a token with a small gradient takes no bits from the others, however large it is; without a gradient
// it has its own e.
template <class Source>
struct PanelJob {
  Source src;
  int R, tiles;  // tiles of R tokens
  int splits, amax_ctas, pair_ctas;
  float* partial;  // largest magnitudes of `splits` parts of every token
  uint4* out;
  const int* w_exp;  // the weights' exponent
  float* factor;   // for every token's output, or (summed) 2^-c of every tile
  const float* dy_partial;  // summed: the gradients' largest magnitudes, else null
  int dy_splits;
};

// 2^e down to the smallest subnormal number. A token of a stage's sums may have e below -126 where its x is near
// the largest fp32 number; below -149 its products are under 2^-35 of the stage's largest.
__device__ __forceinline__ float scale_for(int e) {
  return e >= -126 ? pow2(e) : (e >= -149 ? __int_as_float(1 << (e + 149)) : 0.0f);
}
// A token's exponent, with the weights' exponent w.
__device__ __forceinline__ int token_exponent(float amax, int w) {
  return min(126 - w, max(-126 - w, pair_exponent(amax)));
}
// Summed: the bound on c from a token with largest magnitudes x and dy, and the token's exponent.
__device__ __forceinline__ int sum_bound(float x, float dy, int w) {
  return x > 0.0f && dy > 0.0f ? min(126, max(-126, pair_exponent(x) + token_exponent(dy, w))) : 126;
}
__device__ __forceinline__ int sum_exponent(float x, float dy, int w, int c) {
  return min(c - token_exponent(dy, w), pair_exponent(x));
}

template <class Source>
__device__ __forceinline__ void panel_amax(const PanelJob<Source>& j, long long tokens, int cta) {
  const long long groups = j.src.features >> 3, parts = tokens * j.splits;
  const int lane = threadIdx.x & 31;
  for (long long i = cta * 8ll + (threadIdx.x >> 5); i < parts; i += j.amax_ctas * 8ll) {  // a warp each
    const long long t = i / j.splits, k = i - t * j.splits;
    const float m = largest(j.src, t, groups * k / j.splits + lane, groups * (k + 1) / j.splits, 32);
    if (lane == 0) j.partial[i] = m;
  }
}

// Exponents of a tile's tokens into e, several threads to a token; `write`: into the workspace too.
template <class Source>
__device__ __forceinline__ void tile_exponents(const PanelJob<Source>& j, long long tokens, long long tile, bool write,
                                               int (&e)[128]) {
  const int log = j.R <= 8 ? 5 : __clz(j.R - 1) - 24;  // 32 threads to a token, or 256 / (R rounded up)
  const int r = threadIdx.x >> log, first = threadIdx.x & ((1 << log) - 1);
  const long long t = tile * j.R + r;
  const bool live = r < j.R && t < tokens;
  const int w = *j.w_exp;
  float x = 0.0f, dy = 0.0f;
  if (live) {
    for (int i = first; i < j.splits; i += 1 << log) x = fmaxf(x, j.partial[t * j.splits + i]);
    if (j.dy_partial != nullptr)
      for (int i = first; i < j.dy_splits; i += 1 << log) dy = fmaxf(dy, j.dy_partial[t * j.dy_splits + i]);
  }
  for (int o = 1 << log >> 1; o; o >>= 1) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    dy = fmaxf(dy, __shfl_xor_sync(0xffffffffu, dy, o));
  }
  if (j.dy_partial != nullptr) {
    const int c = -int(cta_max(float(-sum_bound(x, dy, w))));
    if (first == 0 && r < j.R) e[r] = sum_exponent(x, dy, w, c);
    if (write && threadIdx.x == 0) j.factor[tile] = pow2(-c);
  } else if (first == 0 && r < j.R) {
    e[r] = token_exponent(x, w);
    if (write && live) j.factor[t] = pow2(-e[r] - w);
  }
}

// A block of TT tokens (a power of two) x GG groups at a time goes through shared memory: read along the
// features, written along the tokens, whole lines both ways. Per tile of R tokens, part and 8-feature group:
// [R of hi][R of lo'] rows of 16 bytes.
constexpr int kPanelUnits = 1024;  // 8-value pieces of all parts
template <class Source>
__device__ __forceinline__ void panel_pairs(const PanelJob<Source>& j, long long tokens, int cta,
                                            uint4 (&buf)[2 * kPanelUnits], int (&e)[128]) {
  constexpr int P = Source::parts, UNITS = kPanelUnits / P;
  const int R = j.R;
  const PanelBlocks b(R, j.tiles, j.src.features >> 3, UNITS);
  long long tile = -1;
  for (long long item = cta; item < b.items; item += j.pair_ctas) {
    const PanelBlocks::Place at = b.place(item);
    float v[UNITS / 256][P][8] = {};  // on their way while the exponents are found
#pragma unroll
    for (int k = 0; k < UNITS / 256; ++k) {
      const int u = threadIdx.x + 256 * k, t = u >> b.gg_log, g = u & (b.gg - 1);
      const long long token = at.tile * R + at.r + t;
      if (at.r + t < R && token < tokens && at.g + g < b.groups) j.src.load(token * b.groups + at.g + g, v[k]);
    }
    if (at.tile != tile || at.g == 0) tile_exponents(j, tokens, at.tile, at.g == 0, e);
    tile = at.tile;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < UNITS / 256; ++k) {
      const int u = threadIdx.x + 256 * k, t = u >> b.gg_log, g = u & (b.gg - 1);
      const float s = at.r + t < R ? scale_for(e[at.r + t]) : 0.0f;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        uint4* place = buf + 2 * q * UNITS + b.slot(t, g);
        to_pair8(v[k][q], s, place[0], place[UNITS]);
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
__global__ void __launch_bounds__(256, 4) panel_pair_kernel(PanelJob<A> a, PanelJob<C> c, long long tokens) {
  __shared__ uint4 buf[2 * kPanelUnits];
  __shared__ int e[128];
  griddep_launch_dependents();
  griddep_wait();
  const int cta = blockIdx.x;
  if (cta < a.pair_ctas) panel_pairs(a, tokens, cta, buf, e);
  else panel_pairs(c, tokens, cta - a.pair_ctas, buf, e);
}

// Small panels in one launch: a cluster of kSmallCtas CTAs for each, which exchange their tokens' largest
// magnitudes through distributed shared memory and read their values a second time from the caches. Against
// the two kernels it saves a launch; above kSmallGroups 8-value groups its few SMs cost more than that. The
// cluster of summed activations reads the gradients too, for their exponents.
constexpr int kSmallCtas = 8, kSmallThreads = 512;
constexpr int64_t kSmallGroups = 32768, kSmallTokens = 256;
struct SmallShared {
  float x[8 * kSmallTokens], dy[8 * kSmallTokens];  // per token, of the parts of the cluster's warps
  int e[kSmallTokens], bound[kSmallTokens], dy_e[kSmallTokens];
};

// Largest magnitudes of the tokens in every CTA's `table`: 8 << log parts a token, as many warps per token as
// there are for few tokens. `ready`: waits for the cluster's CTAs to have started (they have arrived) before
// it writes to them.
template <class Source>
__device__ __forceinline__ void small_amax(const Source& src, int tokens, int log, float* table, bool ready) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = int(blockIdx.x % kSmallCtas), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = cta << log | (warp & ((1 << log) - 1)), parts = kSmallCtas << log;
  auto of = [&](int t) {
    return t < tokens ? largest(src, t, 32 * part + lane, src.features >> 3, 32 * parts) : 0.0f;
  };
  int t = warp >> log;
  float m = of(t);
  if (ready) cluster.barrier_wait();
  for (; t < tokens; m = of(t)) {
    if (lane < kSmallCtas) *cluster.map_shared_rank(table + t * parts + part, lane) = m;
    t += kSmallThreads / 32 >> log;
  }
}

template <class A, class C>
__device__ __forceinline__ void panel_small(const PanelJob<A>& j, const PanelJob<C>& dy, int tokens, SmallShared& sh) {
  namespace cg = cooperative_groups;
  const int cta = int(blockIdx.x % kSmallCtas), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool summed = j.dy_partial != nullptr;
  const int w_exp = *j.w_exp;
  const int log = tokens > 8 ? 0 : 4 - (tokens > 1 ? 32 - __clz(tokens - 1) : 0), parts = kSmallCtas << log;
  small_amax(j.src, tokens, log, sh.x, true);
  if (summed) small_amax(dy.src, tokens, log, sh.dy, false);
  cg::this_cluster().sync();
  for (int t = warp; t < tokens; t += kSmallThreads / 32) {
    float x = 0.0f, d = 0.0f;
    for (int i = lane; i < parts; i += 32) {
      x = fmaxf(x, sh.x[t * parts + i]);
      if (summed) d = fmaxf(d, sh.dy[t * parts + i]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
      d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, o));
    }
    if (lane == 0) {
      if (summed) {
        sh.e[t] = pair_exponent(x);
        sh.bound[t] = sum_bound(x, d, w_exp);
        sh.dy_e[t] = token_exponent(d, w_exp);
      } else {
        const int e = token_exponent(x, w_exp);
        sh.e[t] = e;
        if (cta == 0) j.factor[t] = pow2(-e - w_exp);
      }
    }
  }
  __syncthreads();
  if (summed) {
    if (warp < j.tiles) {
      int c = 126;
      const int end = min(tokens, (warp + 1) * j.R);
      for (int t = warp * j.R + lane; t < end; t += 32) c = min(c, sh.bound[t]);
      c = __reduce_min_sync(0xffffffffu, c);
      for (int t = warp * j.R + lane; t < end; t += 32) sh.e[t] = min(c - sh.dy_e[t], sh.e[t]);
      if (cta == 0 && lane == 0) j.factor[warp] = pow2(-c);
    }
    __syncthreads();
  }
  // pairs: neighbouring threads take neighbouring tokens (512 contiguous bytes written per warp; each reads
  // one whole 32-byte sector)
  const long long groups = j.src.features >> 3;
  for (PanelWalk w(cta * (long long)kSmallThreads + threadIdx.x, kSmallCtas * (long long)kSmallThreads, j.R, groups);
       w.tile < j.tiles; w.next()) {
    const long long t = w.tile * j.R + w.r;
    float v[A::parts][8] = {}, s = 0.0f;
    if (t < tokens) {
      j.src.load(t * groups + w.g, v);
      s = scale_for(sh.e[t]);
    }
#pragma unroll
    for (int q = 0; q < A::parts; ++q) {
      uint4 hi, lo;
      to_pair8(v[q], s, hi, lo);
      uint4* o = j.out + ((w.tile * A::parts + q) * groups + w.g) * 2 * j.R + w.r;
      o[0] = hi;
      o[j.R] = lo;
    }
  }
}
// The first cluster makes a, a second one c, with a's largest magnitudes where c is summed over.
template <class A, class C>
__global__ void __cluster_dims__(kSmallCtas) __launch_bounds__(kSmallThreads)
    panel_small_kernel(PanelJob<A> a, PanelJob<C> c, int tokens) {
  __shared__ SmallShared sh;
  cooperative_groups::this_cluster().barrier_arrive();
  griddep_launch_dependents();
  if (blockIdx.x < kSmallCtas) panel_small(a, a, tokens, sh);
  else panel_small(c, a, tokens, sh);
}

}  // namespace vbsr_b200
