// vbsr_ortho.cu — orthogonalised block updates: Newton-Schulz steps on every block of a packed
// value array.
//
// Mathematics. With X the block (its shorter side as rows, m <= n <= 64; the formula commutes with
// transposition), a step is A = X X^T, P = b A + c A A, X <- a X + P X: three products. All of a block
// stays on chip from its one read to its one write, so global memory sees 8 bytes per value and the
// rest is tensor-core work, 4 m m n + 2 m^3 operations a step.
//
// Precision. Products are formed from fp16 pairs: X 2^5, A 2^10 and P 2^10 are hi + lo, both fp16, so an
// operand is held to 2^-23 of itself or 2^-30 (X) and 2^-35 (A, P) absolutely, and a product is
// hi lo + lo hi + hi hi in one fp32 accumulator (lo lo is below 2^-22 of it). With these powers of two a
// product comes out in the scale of the next operand: (2^5 X)(2^5 X)^T = 2^10 A. The iterates of a
// convergent iteration have entries of at most about one, and P of about 11; the scales leave room up to
// 2^11 in X and 64 in P. X itself is carried, as 2^5 X, in fp32 registers.
//
// Two forms, by the block's shorter side m.
//
// m <= 32, mma.sync: 16-row strips of X, one per warp, live in registers in the accumulator layout, which is
// also the A operand's layout, so a strip enters the next product without leaving the registers; the other
// operand (all of X, or all of A) is read from shared memory, rows padded by 16 bytes so that ldmatrix meets
// no bank conflict. A needs no transposed copy: it is symmetric. (M = 64 of a tcgen05 MMA would be mostly
// empty here.)
//
// m > 32, tcgen05: four warps own two blocks, one above the other, a thread one row of X. Operands are core
// matrices in shared memory, written once per product as pairs; X serves K-major as both operands of X X^T
// and MN-major as the second of P X. A product is read from TMEM, a row per thread. An MMA has
// M = 128, both blocks' rows, against the columns of both (X X^T, A A; the mixed quarters are not used) or
// one after the other (P X): with M = 64 the tensor core does the same work, but the accumulator fills
// 16 lanes of 32, and the conversions, which bound it, took twice the instructions (measured 1353 us for
// 32768 blocks of 8 to 64, 8192 of them above 48 x 48; mma.sync for all sizes: 701 us).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <new>
#include <vector>

#include "vbsr_internal.h"
#include "vbsr_lm.cuh"
#include "vbsr_pair_host.cuh"

using namespace vbsr_b200;

// The blocks of a CTA: two of more than 32 rows or of more than 16, or four (val = -1: none).
struct alignas(16) OrthoSlot {
  int64_t val;       // first value
  uint32_t shape;    // h | w << 8 | ceil(m / 16) << 16 | ceil(n / 16) << 24
  uint32_t pad;
};

struct vbsr_ortho {
  int device = 0, big_ctas = 0, small_ctas = 0;  // of blocks of more than 32 rows, which come first; others
  OrthoSlot* slots = nullptr;
  int* d_status = nullptr;
  char* memory = nullptr;  // of both
};

namespace {

constexpr float kScale = 32.0f;                // of X
constexpr float kSquare = 1.0f / 1024.0f;      // (2^10 A)(2^10 A) to 2^10 A A; (2^10 P)(2^5 X) to 2^5 P X

// Barrier of the MT warps of a block, the CTA's `group`-th.
template <int MT>
__device__ __forceinline__ void strip_sync(int group) {
  if (MT == 1)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(32 * MT) : "memory");
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  if (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// Two neighbouring values as packed fp16 hi and lo.
__device__ __forceinline__ void pair2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// |V| as 2^e |V / 2^e| with 2^e about the largest magnitude, so that the squares neither overflow nor vanish:
// the sum is 0 for a block of zeros alone, and not finite only where a value is not.
struct Norm {
  int e;
  float down;
  __device__ __forceinline__ explicit Norm(float amax) {
    const bool usable = amax > 0.0f && amax < __int_as_float(0x7f800000);
    e = usable ? max(-125, min(125, ilogbf(amax))) : 0;
    down = __int_as_float((127 - e) << 23);
  }
  __device__ __forceinline__ float add(float sum, float v) const {
    const float y = v * down;
    return fmaf(y, y, sum);
  }
  // kScale / (|V| + eps) times 2^e; 0 for a block of zeros (kScale / eps may overflow), NaN for one with a NaN or
  // an infinity
  __device__ __forceinline__ float inverse(float sum, float eps) const {
    if (sum == 0.0f) return 0.0f;
    return sum < __int_as_float(0x7f800000) ? kScale / (sqrtf(sum) + eps * down) : __int_as_float(0x7fc00000);
  }
  __device__ __forceinline__ float apply(float v, float inv) const { return v * down * inv; }
};

// A strip (T tiles of 8 columns) as pairs: the A operands of its T / 2 k-tiles.
template <int T>
struct StripPair {
  uint32_t hi[T / 2][4], lo[T / 2][4];
  __device__ __forceinline__ void set(const float (&x)[T][4]) {
#pragma unroll
    for (int j = 0; j < T; ++j) {
      pair2(x[j][0], x[j][1], hi[j / 2][(j & 1) * 2], lo[j / 2][(j & 1) * 2]);
      pair2(x[j][2], x[j][3], hi[j / 2][(j & 1) * 2 + 1], lo[j / 2][(j & 1) * 2 + 1]);
    }
  }
  // rows [16 strip, + 16) of a row-major matrix of row stride LD halves, lo behind hi at `lo_off` bytes
  template <int LD>
  __device__ __forceinline__ void store(char* base, int lo_off, int strip, int lane) const {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        char* p = base + ((16 * strip + g + 8 * half) * LD + 8 * j + 2 * t) * 2;
        *reinterpret_cast<uint32_t*>(p) = hi[j / 2][(j & 1) * 2 + half];
        *reinterpret_cast<uint32_t*>(p + lo_off) = lo[j / 2][(j & 1) * 2 + half];
      }
  }
};

// d (T tiles) = a (KT k-tiles) * B. TRANS: B[k][n] at row k of the matrix in shared memory; else at
// row n (its transpose).
template <int T, int KT, int LD, bool TRANS>
__device__ __forceinline__ void strip_product(float (&d)[T][4], const StripPair<2 * KT>& a, uint32_t base,
                                              int lo_off, int lane) {
#pragma unroll
  for (int j = 0; j < T; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) d[j][i] = 0.0f;
  const int r = lane & 7, q = lane >> 3;
  constexpr int J = T % 4 == 0 ? 4 : 2;  // tiles at a time: independent sums, an MMA waits for its sum's last one
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int j = 0; j < T; j += J) {
      uint32_t bh[J / 2][4], bl[J / 2][4];
#pragma unroll
      for (int i = 0; i < J / 2; ++i) {
        // the four 8 x 8 pieces: k halves of tile j + 2 i, then of the next
        const int n = 8 * (j + 2 * i + (q >> 1)), k = 16 * kt + 8 * (q & 1);
        const uint32_t addr = base + 2u * (TRANS ? (k + r) * LD + n : (n + r) * LD + k);
        ldsm4<TRANS>(addr, bh[i]);
        ldsm4<TRANS>(addr + lo_off, bl[i]);
      }
#pragma unroll
      for (int i = 0; i < J; ++i) mma16816(d[j + i], a.hi[kt], bl[i / 2][2 * (i & 1)], bl[i / 2][2 * (i & 1) + 1]);
#pragma unroll
      for (int i = 0; i < J; ++i) mma16816(d[j + i], a.lo[kt], bh[i / 2][2 * (i & 1)], bh[i / 2][2 * (i & 1) + 1]);
#pragma unroll
      for (int i = 0; i < J; ++i) mma16816(d[j + i], a.hi[kt], bh[i / 2][2 * (i & 1)], bh[i / 2][2 * (i & 1) + 1]);
    }
}

struct OrthoParams {
  const OrthoSlot* slots;
  const float* values;
  float* out;
  int steps;
  float eps, a, b, c;
  int* status;
};

// Shared memory of a block of MT x NT 16-tiles: X and A, each hi and lo.
template <int MT, int NT>
struct OrthoSmem {
  static constexpr int LDX = 16 * NT + 8, LDA = 16 * MT + 8;
  static constexpr int x_lo = 16 * MT * LDX * 2, x_bytes = 2 * x_lo;
  static constexpr int a_lo = 16 * MT * LDA * 2, a_at = x_bytes;
  static constexpr int red_at = a_at + 2 * a_lo;
  static constexpr int bytes = red_at + 2 * 16;
};
constexpr int kMax2(int a, int b) { return a > b ? a : b; }
constexpr int kSmallSmem = kMax2(2 * OrthoSmem<2, 4>::bytes, 4 * OrthoSmem<1, 4>::bytes);
// m > 32: X, and A or P, of two blocks as pairs, 128 x 64 each.
constexpr int kTileBytes = 128 * 64 * 2, kBigSmem = 4 * kTileBytes + 1024;

template <int MT, int NT>
__device__ __forceinline__ void orthogonalize(const OrthoParams& p, const OrthoSlot& s, char* sm, int group,
                                              int strip, int lane) {
  using S = OrthoSmem<MT, NT>;
  const int h = int(s.shape & 255u), w = int((s.shape >> 8) & 255u);
  const int m = min(h, w), n = max(h, w);
  const long long si = h <= w ? 1 : h, sj = h <= w ? h : 1;  // steps of X's row and column in the block
  const int g = lane >> 2, t = lane & 3;
  float* red = reinterpret_cast<float*>(sm + S::red_at);

  float x[2 * NT][4];
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < 2 * NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * strip + g + 8 * (i >> 1), col = 8 * j + 2 * t + (i & 1);
      x[j][i] = row < m && col < n ? p.values[s.val + row * si + col * sj] : 0.0f;
      amax = fmaxf(amax, fabsf(x[j][i]));
    }
  auto reduce = [&](float v, int slot, bool largest) {
    for (int d = 16; d; d >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, v, d);
      v = largest ? fmaxf(v, y) : v + y;
    }
    if (MT == 1) return v;
    if (lane == 0) red[4 * slot + strip] = v;
    strip_sync<MT>(group);
    v = red[4 * slot];
#pragma unroll
    for (int i = 1; i < MT; ++i) v = largest ? fmaxf(v, red[4 * slot + i]) : v + red[4 * slot + i];
    return v;
  };
  const Norm norm(reduce(amax, 0, true));
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < 2 * NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = norm.add(sum, x[j][i]);
  const float inv = norm.inverse(reduce(sum, 1, false), p.eps);
#pragma unroll
  for (int j = 0; j < 2 * NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[j][i] = norm.apply(x[j][i], inv);

  for (int step = 0; step < p.steps; ++step) {
    strip_sync<MT>(group);  // X may still be read by another warp
    char* xs = sm;
    float acc[2 * MT][4], sq[2 * MT][4];
    {
      StripPair<2 * NT> xp;
      xp.set(x);
      xp.template store<S::LDX>(xs, S::x_lo, strip, lane);
      strip_sync<MT>(group);
      strip_product<2 * MT, NT, S::LDX, false>(acc, xp, smem_addr(xs), S::x_lo, lane);
    }
    StripPair<2 * MT> ap;
    ap.set(acc);
    ap.template store<S::LDA>(sm + S::a_at, S::a_lo, strip, lane);
    strip_sync<MT>(group);
    strip_product<2 * MT, MT, S::LDA, false>(sq, ap, smem_addr(sm + S::a_at), S::a_lo, lane);
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sq[j][i] = fmaf(p.c * kSquare, sq[j][i], p.b * acc[j][i]);
    ap.set(sq);
    float px[2 * NT][4];
    strip_product<2 * NT, MT, S::LDX, true>(px, ap, smem_addr(xs), S::x_lo, lane);
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[j][i] = fmaf(px[j][i], kSquare, p.a * x[j][i]);
  }

#pragma unroll
  for (int j = 0; j < 2 * NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * strip + g + 8 * (i >> 1), col = 8 * j + 2 * t + (i & 1);
      if (row < m && col < n) p.out[s.val + row * si + col * sj] = x[j][i] * (1.0f / kScale);
    }
}

// Two warps a block of more than 16 rows, two of them in a CTA, or one warp a block, four in a CTA.
__global__ void __launch_bounds__(128, 4) ortho_small_kernel(OrthoParams p) {
  extern __shared__ __align__(16) char sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const OrthoSlot* slots = p.slots + 4ll * blockIdx.x;
  const int mt = int((slots[0].shape >> 16) & 255u);
  const int group = warp / mt, strip = warp % mt;
  const OrthoSlot s = slots[group];
  if (s.val >= 0) {
    const int nt = int(s.shape >> 24);
#define VBSR_ORTHO(M, N)                                                                     \
  case 8 * M + N:                                                                            \
    orthogonalize<M, N>(p, s, sm + group * OrthoSmem<M, N>::bytes, group, strip, lane);      \
    break;
    switch (8 * mt + nt) {
      VBSR_ORTHO(1, 1) VBSR_ORTHO(1, 2) VBSR_ORTHO(1, 3) VBSR_ORTHO(1, 4) VBSR_ORTHO(2, 2)
      VBSR_ORTHO(2, 3) VBSR_ORTHO(2, 4)
    }
#undef VBSR_ORTHO
  }
  griddep_wait();  // it may have started beside the large blocks' kernel: both are done when this one is
}

// ---- m > 32 --------------------------------------------------------------------------------------
//
// An operand: row r of the CTA's 128 (block r / 64), column group g (8 columns) at byte 2048 g + 16 r; hi, and
// lo kTileBytes behind.

struct OrthoTcShared {
  u64 done;
  uint32_t tmem;
  volatile int abort_flag;
  float red[2][4];
};

// A row's 64 values as pairs into an operand.
__device__ __forceinline__ void store_pairs(char* tile, int row, const float (&v)[64]) {
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    uint4 hi, lo;
    pair2(v[8 * g], v[8 * g + 1], hi.x, lo.x);
    pair2(v[8 * g + 2], v[8 * g + 3], hi.y, lo.y);
    pair2(v[8 * g + 4], v[8 * g + 5], hi.z, lo.z);
    pair2(v[8 * g + 6], v[8 * g + 7], hi.w, lo.w);
    char* o = tile + 2048 * g + 16 * row;
    *reinterpret_cast<uint4*>(o) = hi;
    *reinterpret_cast<uint4*>(o + kTileBytes) = lo;
  }
}

// 64 accumulator columns, loaded and waited for.
__device__ __forceinline__ void tc_ld64(uint32_t a, float (&v)[64]) {
#pragma unroll
  for (int i = 0; i < 64; i += 32) {
    float x[16], y[16];
    tc_ld16(a + i, a + i + 16, x, y);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      v[i + j] = x[j];
      v[i + 16 + j] = y[j];
    }
  }
}

__global__ void __launch_bounds__(128, 3) ortho_big_kernel(OrthoParams p) {
  extern __shared__ char sm[];
  __shared__ OrthoTcShared sh;
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, block = threadIdx.x >> 6, row = threadIdx.x & 63;
  const OrthoSlot* slots = p.slots + 4ll * blockIdx.x;
  const OrthoSlot s = slots[block];
  const int h = int(s.shape & 255u), w = int((s.shape >> 8) & 255u);
  const int m = min(h, w), n = max(h, w);
  // 16-column steps that cover both blocks
  const int mt = max(int((slots[0].shape >> 16) & 255u), int((slots[1].shape >> 16) & 255u));
  const int nt = max(int(slots[0].shape >> 24), int(slots[1].shape >> 24));
  const uint32_t base = (smem_addr(sm) + 1023u) & ~1023u;
  char* xt = sm + (base - smem_addr(sm));
  char* at = xt + 2 * kTileBytes;  // A, then P
  const uint32_t done = smem_addr(&sh.done);
  if (threadIdx.x == 0) {
    mbar_init(done, 1);
    sh.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    tc_alloc(smem_addr(&sh.tmem), 128);
    tc_relinquish();
  }
  tc_fence_before();
  const bool live = s.val >= 0 && row < m;
  const long long si = h <= w ? 1 : h, sj = h <= w ? h : 1;
  const float* v = p.values + s.val + row * si;
  float x[64];
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < 64; ++j) {
    x[j] = live && j < n ? v[j * sj] : 0.0f;
    amax = fmaxf(amax, fabsf(x[j]));
  }
  auto reduce = [&](float y, int slot, bool largest) {  // over the block's two warps
    for (int d = 16; d; d >>= 1) {
      const float z = __shfl_xor_sync(0xffffffffu, y, d);
      y = largest ? fmaxf(y, z) : y + z;
    }
    if (lane == 0) sh.red[slot][warp] = y;
    __syncthreads();
    const float a = sh.red[slot][2 * block], b = sh.red[slot][2 * block + 1];
    return largest ? fmaxf(a, b) : a + b;
  };
  const Norm norm(reduce(amax, 0, true));
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < 64; ++j) sum = norm.add(sum, x[j]);
  const float inv = norm.inverse(reduce(sum, 1, false), p.eps);
#pragma unroll
  for (int j = 0; j < 64; ++j) x[j] = norm.apply(x[j], inv);
  tc_fence_after();
  const uint32_t d = uniform(sh.tmem);  // A, then A A, then P X
  const uint32_t mine = (uint32_t(32 * warp) << 16) + 64u * block;  // this thread's lane and block's columns
  const uint32_t form = (1u << 4) | (8u << 24);  // D f32, A and B f16, M = 128
  const uint32_t leader = lane == 0;
  uint32_t parity = 0;
  bool ok = true;
  constexpr u64 LO = kTileBytes >> 4, STEP = 2 * 2048 >> 4;  // lo behind hi; two column groups
  auto run = [&](auto issue) {
    fence_proxy_async_smem();  // the operands were written by ordinary stores
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
      tc_fence_after();
      issue();
      tc_commit_by(done, leader);
    }
    // after an abort nothing is waited for, but the threads stay together (__syncthreads)
    if (ok) ok = wait_warp(done, parity, p.status, &sh.abort_flag);
    parity ^= 1u;
    tc_fence_after();
  };
  // D = T T^T for both blocks' rows at once, the small terms first
  auto gram = [&](uint32_t tile, int ksteps) {
    const u64 t = core_desc(tile, 2048, 128);
    const uint32_t id = form | (16u << 17);  // N = 128
    for (int k = 0; k < ksteps; ++k) {
      tc_mma_f16(d, t + STEP * k, t + STEP * k + LO, id, k > 0, leader);
      tc_mma_f16(d, t + STEP * k + LO, t + STEP * k, id, 1u, leader);
    }
    for (int k = 0; k < ksteps; ++k) tc_mma_f16(d, t + STEP * k, t + STEP * k, id, 1u, leader);
  };
  // columns 64 b .. of D = P X_b: X MN-major, 16 rows are two core matrices
  auto times_x = [&]() {
    const u64 a = core_desc(base + 2 * kTileBytes, 2048, 128);
    const uint32_t id = form | (1u << 16) | (8u << 17);  // N = 64
    const u64 b0 = core_desc(base, 128, 2048), b1 = core_desc(base + 1024, 128, 2048);
    for (int k = 0; k < mt; ++k) {  // the two blocks' sums are independent: one waits while the other runs
      tc_mma_f16(d, a + STEP * k, b0 + 16 * k + LO, id, k > 0, leader);
      tc_mma_f16(d + 64, a + STEP * k, b1 + 16 * k + LO, id, k > 0, leader);
      tc_mma_f16(d, a + STEP * k + LO, b0 + 16 * k, id, 1u, leader);
      tc_mma_f16(d + 64, a + STEP * k + LO, b1 + 16 * k, id, 1u, leader);
    }
    for (int k = 0; k < mt; ++k) {
      tc_mma_f16(d, a + STEP * k, b0 + 16 * k, id, 1u, leader);
      tc_mma_f16(d + 64, a + STEP * k, b1 + 16 * k, id, 1u, leader);
    }
  };
  const int r = threadIdx.x;
  for (int step = 0; step < p.steps; ++step) {
    store_pairs(xt, r, x);
    run([&] { gram(base, nt); });
    float a[64];
    tc_ld64(d + mine, a);
    store_pairs(at, r, a);
    run([&] { gram(base + 2 * kTileBytes, mt); });
#pragma unroll
    for (int i = 0; i < 64; i += 16) {
      float q[16];
      tc_ld16(d + mine + i, q);
#pragma unroll
      for (int j = 0; j < 16; ++j) a[i + j] = fmaf(p.c * kSquare, q[j], p.b * a[i + j]);
    }
    store_pairs(at, r, a);
    run([&] { times_x(); });
#pragma unroll
    for (int i = 0; i < 64; i += 16) {
      float q[16];
      tc_ld16(d + mine + i, q);
#pragma unroll
      for (int j = 0; j < 16; ++j) x[i + j] = fmaf(q[j], kSquare, p.a * x[i + j]);
    }
  }
  if (live) {
    float* o = p.out + s.val + row * si;
#pragma unroll
    for (int j = 0; j < 64; ++j)
      if (j < n) o[j * sj] = x[j] * (1.0f / kScale);
  }
  tc_fence_before();
  __syncthreads();
  if (sh.abort_flag) {  // a wait gave up: its MMAs may still run; give them time before the memory goes
    const long long t0 = clock64();
    while (clock64() - t0 < 20000000ll) __nanosleep(1000);
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 0) tc_dealloc(sh.tmem, 128);
}

void free_ortho(vbsr_ortho* p) {
  if (p == nullptr) return;
  DeviceGuard guard(p->device);
  cudaFree(p->memory);
  delete p;
}

vbsr_status build_ortho(vbsr_ortho* p, const MatrixData& d) {
  VBSR_CUDA(cudaFuncSetAttribute(ortho_small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmallSmem));
  VBSR_CUDA(cudaFuncSetAttribute(ortho_big_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBigSmem));
  std::vector<OrthoSlot> by_class[5][5];
  for (int i = 0; i < d.block_rows; ++i) {
    int64_t val = d.h_val_off_row[i];
    for (int b = d.h_row_ptr[i]; b < d.h_row_ptr[i + 1]; ++b) {
      const int h = d.h_row_size[i], w = d.h_col_size[d.h_block_col[b]];
      const int mt = (std::min(h, w) + 15) / 16, nt = (std::max(h, w) + 15) / 16;
      by_class[mt][nt].push_back({val, uint32_t(h) | uint32_t(w) << 8 | uint32_t(mt) << 16 |
                                           uint32_t(nt) << 24, 0});
      val += int64_t(h) * w;
    }
  }
  // the largest first
  std::vector<OrthoSlot> slots;
  auto pack = [&](const std::vector<OrthoSlot>& v, int per) {
    for (size_t i = 0; i < v.size(); i += per)
      for (int k = 0; k < 4; ++k) {
        const bool have = k < per && i + k < v.size();
        slots.push_back(have ? v[i + k] : OrthoSlot{-1, v[i].shape, 0});
      }
  };
  std::vector<OrthoSlot> big;
  for (int mt = 4; mt >= 3; --mt)
    for (int nt = 4; nt >= mt; --nt) big.insert(big.end(), by_class[mt][nt].begin(), by_class[mt][nt].end());
  pack(big, 2);
  p->big_ctas = int(slots.size() / 4);
  for (int mt = 2; mt >= 1; --mt)
    for (int nt = 4; nt >= mt; --nt) pack(by_class[mt][nt], mt == 2 ? 2 : 4);
  p->small_ctas = int(slots.size() / 4) - p->big_ctas;
  PlanMemory mem;
  mem.table(&p->slots, std::move(slots));
  mem.table(&p->d_status, std::vector<int>(kStatusWords));
  SetupStream s;  // after `mem`: it waits before that goes
  VBSR_CUDA(s.init());
  VBSR_CUDA(mem.make(&p->memory, s.s));
  VBSR_CUDA(s.finish());
  return VBSR_OK;
}

}  // namespace

extern "C" {

vbsr_status vbsr_ortho_create(const vbsr_matrix* m, vbsr_ortho** out) {
  clear_error();
  if (out == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null output");
  *out = nullptr;
  if (m == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null matrix");
  auto* p = new (std::nothrow) vbsr_ortho;
  if (p == nullptr) return set_error(VBSR_OUT_OF_MEMORY, "host allocation failed");
  p->device = m->d.device;
  DeviceGuard guard(p->device);
  vbsr_status st;
  try {
    st = build_ortho(p, m->d);
  } catch (const std::bad_alloc&) {
    st = set_error(VBSR_OUT_OF_MEMORY, "host allocation failed");
  }
  if (st != VBSR_OK) {
    free_ortho(p);
    return st;
  }
  *out = p;
  return VBSR_OK;
}

vbsr_status vbsr_ortho_destroy(vbsr_ortho* p) {
  clear_error();
  free_ortho(p);
  return VBSR_OK;
}

vbsr_status vbsr_ortho_execute(const vbsr_ortho* p, const float* values, float* out, int steps,
                               float eps, const float* coefficients, vbsr_stream_t stream) {
  clear_error();
  if (p == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null plan");
  if (steps < 0 || steps > 64)
    return set_error(VBSR_INVALID_ARGUMENT, "steps must be between 0 and 64");
  if (!(eps >= 0.0f) || std::isinf(eps))
    return set_error(VBSR_INVALID_ARGUMENT, "eps must be finite and not negative");
  if (coefficients == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null coefficients");
  if (p->big_ctas + p->small_ctas == 0) return VBSR_OK;
  if (values == nullptr || out == nullptr)
    return set_error(VBSR_INVALID_ARGUMENT, "null values or out");
  DeviceGuard guard(p->device);
  OrthoParams k{p->slots, values, out, steps, eps, coefficients[0], coefficients[1], coefficients[2], p->d_status};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p->big_ctas > 0) {
    ortho_big_kernel<<<unsigned(p->big_ctas), 128, kBigSmem, st>>>(k);
    VBSR_CUDA(cudaGetLastError());
  }
  if (p->small_ctas > 0) {
    k.slots += 4ll * p->big_ctas;
    if (p->big_ctas > 0) {
      VBSR_CUDA(launch_after(ortho_small_kernel, dim3(unsigned(p->small_ctas)), 128, kSmallSmem, st, k));
    } else {
      ortho_small_kernel<<<unsigned(p->small_ctas), 128, kSmallSmem, st>>>(k);
      VBSR_CUDA(cudaGetLastError());
    }
  }
  return VBSR_OK;
}

vbsr_status vbsr_ortho_check_status(const vbsr_ortho* p, vbsr_stream_t stream) {
  clear_error();
  if (p == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null plan");
  DeviceGuard guard(p->device);
  return read_status(p->d_status, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
