// vbsr_ortho.cu — orthogonalised block updates: Newton-Schulz steps on every block of a packed
// value array.
//
// Mathematics. With X the block (its shorter side as rows, m <= n <= 64; the formula commutes with
// transposition), a step is A = X X^T, P = b A + c A A, X <- a X + P X: three products. All of a block
// stays on chip from its one read to its one write, so global memory sees 8 bytes per value and the
// rest is tensor-core work, 4 m m n + 2 m^3 operations a step.
//
// Precision. Products are formed from fp16 pairs: x 2^10 = hi + lo, both fp16, so an operand is held
// to 2^-23 of itself or 2^-35 absolutely, and a product is hi lo + lo hi + hi hi in one fp32
// accumulator (lo lo is below 2^-22 of it). The iterates of a convergent iteration have entries of at
// most about one, and P of about 11; 2^10 leaves room up to 64. X itself is carried in fp32 registers.
//
// Layout. 16-row strips of X, one per warp, live in registers in the accumulator layout of mma.sync,
// which is also its A operand's layout, so a strip enters the next product without leaving the
// registers; the other operand (all of X, or all of A) is read from shared memory, rows padded by 16
// bytes so that ldmatrix meets no bank conflict. A needs no transposed copy: it is symmetric. mma.sync
// and not tcgen05, because the products are chained through elementwise steps and of any size from 8
// to 64: the result of each would go TMEM to registers to shared memory, and M = 64 is mostly
// empty for the small blocks.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <new>
#include <vector>

#include "vbsr_internal.h"
#include "vbsr_lm.cuh"
#include "vbsr_ptx.cuh"

using namespace vbsr_b200;

// The blocks of a CTA: one of more than 32 rows, two of more than 16, or four (val = -1: none).
struct alignas(16) OrthoSlot {
  int64_t val;       // first value
  uint32_t shape;    // h | w << 8 | ceil(m / 16) << 16 | ceil(n / 16) << 24
  uint32_t pad;
};

struct vbsr_ortho {
  const vbsr_matrix* m = nullptr;
  int device = 0, ctas = 0;
  OrthoSlot* slots = nullptr;
};

namespace {

constexpr float kScale = 1024.0f, kUnscale2 = 1.0f / (1024.0f * 1024.0f);

// Barrier of the MT warps of a block, the CTA's `group`-th.
template <int MT>
__device__ __forceinline__ void group_sync(int group) {
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

// Two neighbouring values times s as packed fp16 hi and lo.
__device__ __forceinline__ void pair2(float x, float y, float s, uint32_t& hi, uint32_t& lo) {
  x *= s;
  y *= s;
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// A strip (T tiles of 8 columns) as pairs: the A operands of its T / 2 k-tiles.
template <int T>
struct StripPair {
  uint32_t hi[T / 2][4], lo[T / 2][4];
  __device__ __forceinline__ void set(const float (&x)[T][4], float s) {
#pragma unroll
    for (int j = 0; j < T; ++j) {
      pair2(x[j][0], x[j][1], s, hi[j / 2][(j & 1) * 2], lo[j / 2][(j & 1) * 2]);
      pair2(x[j][2], x[j][3], s, hi[j / 2][(j & 1) * 2 + 1], lo[j / 2][(j & 1) * 2 + 1]);
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
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int j = 0; j < T; j += 2) {
      // the four 8 x 8 pieces: k halves of tile j, then of tile j + 1
      const int n = 8 * (j + (q >> 1)), k = 16 * kt + 8 * (q & 1);
      const uint32_t addr = base + 2u * (TRANS ? (k + r) * LD + n : (n + r) * LD + k);
      uint32_t bh[4], bl[4];
      ldsm4<TRANS>(addr, bh);
      ldsm4<TRANS>(addr + lo_off, bl);
      mma16816(d[j], a.hi[kt], bl[0], bl[1]);
      mma16816(d[j + 1], a.hi[kt], bl[2], bl[3]);
      mma16816(d[j], a.lo[kt], bh[0], bh[1]);
      mma16816(d[j + 1], a.lo[kt], bh[2], bh[3]);
      mma16816(d[j], a.hi[kt], bh[0], bh[1]);
      mma16816(d[j + 1], a.hi[kt], bh[2], bh[3]);
    }
}

struct OrthoParams {
  const OrthoSlot* slots;
  const float* values;
  float* out;
  int steps;
  float eps, a, b, c;
};

// Shared memory of a block of MT x NT 16-tiles: two buffers of X and one of A, each hi and lo.
template <int MT, int NT>
struct OrthoSmem {
  static constexpr int LDX = 16 * NT + 8, LDA = 16 * MT + 8;
  static constexpr int x_lo = 16 * MT * LDX * 2, x_bytes = 2 * x_lo;
  static constexpr int a_lo = 16 * MT * LDA * 2, a_at = 2 * x_bytes;
  static constexpr int red_at = a_at + 2 * a_lo;
  static constexpr int bytes = red_at + 2 * 16;
};
constexpr int kOrthoSmem = OrthoSmem<4, 4>::bytes;
static_assert(2 * OrthoSmem<2, 4>::bytes <= kOrthoSmem && 4 * OrthoSmem<1, 4>::bytes <= kOrthoSmem, "groups");

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
    group_sync<MT>(group);
    v = red[4 * slot];
#pragma unroll
    for (int i = 1; i < MT; ++i) v = largest ? fmaxf(v, red[4 * slot + i]) : v + red[4 * slot + i];
    return v;
  };
  // |V| as amax |V / amax|, so that the squares neither overflow nor vanish
  amax = reduce(amax, 0, true);
  const float scale = amax > 0.0f && amax < __int_as_float(0x7f800000) ? amax : 1.0f;
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < 2 * NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = x[j][i] / scale;
      sum = fmaf(y, y, sum);
    }
  sum = reduce(sum, 1, false);
  const float norm = scale * sqrtf(sum) + p.eps;
  if (norm != 0.0f) {
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[j][i] /= norm;
  }

  for (int step = 0; step < p.steps; ++step) {
    char* xs = sm + (step & 1) * S::x_bytes;  // the other buffer may still be read by another warp
    float acc[2 * MT][4], sq[2 * MT][4];
    {
      StripPair<2 * NT> xp;
      xp.set(x, kScale);
      xp.template store<S::LDX>(xs, S::x_lo, strip, lane);
      group_sync<MT>(group);
      strip_product<2 * MT, NT, S::LDX, false>(acc, xp, smem_addr(xs), S::x_lo, lane);
    }
    StripPair<2 * MT> ap;
    ap.set(acc, 1.0f / kScale);  // acc is 2^20 A
    ap.template store<S::LDA>(sm + S::a_at, S::a_lo, strip, lane);
    group_sync<MT>(group);
    strip_product<2 * MT, MT, S::LDA, false>(sq, ap, smem_addr(sm + S::a_at), S::a_lo, lane);
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sq[j][i] = fmaf(p.c, sq[j][i], p.b * acc[j][i]);  // 2^20 P
    ap.set(sq, 1.0f / kScale);
    float px[2 * NT][4];
    strip_product<2 * NT, MT, S::LDX, true>(px, ap, smem_addr(xs), S::x_lo, lane);
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[j][i] = fmaf(px[j][i], kUnscale2, p.a * x[j][i]);
  }

#pragma unroll
  for (int j = 0; j < 2 * NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * strip + g + 8 * (i >> 1), col = 8 * j + 2 * t + (i & 1);
      if (row < m && col < n) p.out[s.val + row * si + col * sj] = x[j][i];
    }
}

// Four warps: one block of more than 32 rows (three or four strips), two of more than 16 or four.
__global__ void __launch_bounds__(128, 3) ortho_kernel(OrthoParams p) {
  extern __shared__ __align__(16) char sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const OrthoSlot* slots = p.slots + 4ll * blockIdx.x;
  const int mt = int((slots[0].shape >> 16) & 255u);
  const int per = mt <= 1 ? 1 : (mt == 2 ? 2 : 4), group = warp / per, strip = warp % per;
  const OrthoSlot s = slots[group];
  if (s.val < 0 || strip >= mt) return;
  const int nt = int(s.shape >> 24);
#define VBSR_ORTHO(M, N)                                                                     \
  case 8 * M + N:                                                                            \
    orthogonalize<M, N>(p, s, sm + group * OrthoSmem<M, N>::bytes, group, strip, lane);      \
    break;
  switch (8 * mt + nt) {
    VBSR_ORTHO(1, 1) VBSR_ORTHO(1, 2) VBSR_ORTHO(1, 3) VBSR_ORTHO(1, 4) VBSR_ORTHO(2, 2)
    VBSR_ORTHO(2, 3) VBSR_ORTHO(2, 4) VBSR_ORTHO(3, 3) VBSR_ORTHO(3, 4) VBSR_ORTHO(4, 4)
  }
#undef VBSR_ORTHO
}

void free_ortho(vbsr_ortho* p) {
  if (p == nullptr) return;
  DeviceGuard guard(p->device);
  cudaFree(p->slots);
  delete p;
}

vbsr_status build_ortho(vbsr_ortho* p) {
  const MatrixData& d = p->m->d;
  VBSR_CUDA(cudaFuncSetAttribute(ortho_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kOrthoSmem));
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
  for (int mt = 4; mt >= 1; --mt)
    for (int nt = 4; nt >= mt; --nt) {
      const int per = mt >= 3 ? 1 : (mt == 2 ? 2 : 4);
      const std::vector<OrthoSlot>& v = by_class[mt][nt];
      for (size_t i = 0; i < v.size(); i += per)
        for (int k = 0; k < 4; ++k) {
          const bool have = k < per && i + k < v.size();
          slots.push_back(have ? v[i + k] : OrthoSlot{-1, v[i].shape, 0});
        }
    }
  p->ctas = int(slots.size() / 4);
  VBSR_CUDA(upload_array(&p->slots, slots));
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
  p->m = m;
  p->device = m->d.device;
  DeviceGuard guard(p->device);
  vbsr_status st;
  try {
    st = build_ortho(p);
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
  if (p->ctas == 0) return VBSR_OK;
  if (values == nullptr || out == nullptr)
    return set_error(VBSR_INVALID_ARGUMENT, "null values or out");
  DeviceGuard guard(p->device);
  const OrthoParams k{p->slots, values, out, steps, eps, coefficients[0], coefficients[1], coefficients[2]};
  ortho_kernel<<<unsigned(p->ctas), 128, kOrthoSmem, reinterpret_cast<cudaStream_t>(stream)>>>(k);
  VBSR_CUDA(cudaGetLastError());
  return VBSR_OK;
}

}  // extern "C"
