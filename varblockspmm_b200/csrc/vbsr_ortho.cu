// vbsr_ortho.cu — orthogonalised block updates: Newton-Schulz steps on every block of a packed
// value array.
#include <cuda_runtime.h>

#include <new>

#include "vbsr_internal.h"
#include "vbsr_lm.cuh"

using namespace vbsr_b200;

struct vbsr_ortho {
  const vbsr_matrix* m = nullptr;
  int device = 0;
};

namespace {

// One CTA per block. X is the block with its shorter side as rows (m <= n; the formula commutes with
// transposition), A = X X^T, P = b A + c A A.
__global__ void ortho_kernel(vbsr_device_matrix s, const float* values, float* out, int steps,
                             float eps, float ca, float cb, float cc) {
  extern __shared__ float sm[];
  float *X = sm, *A = sm + 4096, *P = sm + 8192, *Y = sm + 12288;
  __shared__ float red[8];
  const int b = blockIdx.x;
  const int h = s.row_size[row_of_block(s.row_ptr, s.block_rows, b)], w = s.col_size[s.block_col[b]];
  const int m = min(h, w), n = max(h, w), size = h * w;
  const float* v = values + s.value_off[b];
  float* o = out + s.value_off[b];
  auto at = [&](int i) {  // position in X (m x n, row-major) of packed element i
    const int r = i % h, c = i / h;
    return h <= w ? r * n + c : c * n + r;
  };
  // |V| as amax * |V / amax|, so that the squares neither overflow nor vanish
  auto reduce = [&](float x, bool largest) {
    for (int d = 16; d; d >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, x, d);
      x = largest ? fmaxf(x, y) : x + y;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
    __syncthreads();
    x = red[0];
    for (int i = 1; i < 8; ++i) x = largest ? fmaxf(x, red[i]) : x + red[i];
    return x;
  };
  float amax = 0.0f;
  for (int i = threadIdx.x; i < size; i += blockDim.x) amax = fmaxf(amax, fabsf(v[i]));
  amax = reduce(amax, true);
  const float scale = amax > 0.0f && amax < __int_as_float(0x7f800000) ? amax : 1.0f;
  float sum = 0.0f;
  for (int i = threadIdx.x; i < size; i += blockDim.x) {
    const float x = v[i] / scale;
    sum = fmaf(x, x, sum);
  }
  sum = reduce(sum, false);
  const float norm = scale * sqrtf(sum) + eps;
  for (int i = threadIdx.x; i < size; i += blockDim.x)
    X[at(i)] = norm > 0.0f || norm != norm ? v[i] / norm : 0.0f;
  __syncthreads();
  for (int step = 0; step < steps; ++step) {
    for (int i = threadIdx.x; i < m * m; i += blockDim.x) {
      const int r = i / m, c = i % m;
      float t = 0.0f;
      for (int k = 0; k < n; ++k) t = fmaf(X[r * n + k], X[c * n + k], t);
      A[i] = t;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < m * m; i += blockDim.x) {
      const int r = i / m, c = i % m;
      float t = 0.0f;
      for (int k = 0; k < m; ++k) t = fmaf(A[r * m + k], A[k * m + c], t);
      P[i] = cb * A[i] + cc * t;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < size; i += blockDim.x) {
      const int r = i / n, c = i % n;
      float t = 0.0f;
      for (int k = 0; k < m; ++k) t = fmaf(P[r * m + k], X[k * n + c], t);
      Y[i] = ca * X[i] + t;
    }
    __syncthreads();
    float* z = X;
    X = Y;
    Y = z;
  }
  for (int i = threadIdx.x; i < size; i += blockDim.x) o[i] = X[at(i)];
}
constexpr int kOrthoSmem = 4 * 4096 * 4;

}  // namespace

extern "C" {

vbsr_status vbsr_ortho_create(const vbsr_matrix* m, vbsr_ortho** out) {
  clear_error();
  if (out == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null output");
  *out = nullptr;
  if (m == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null matrix");
  DeviceGuard guard(m->d.device);
  VBSR_CUDA(cudaFuncSetAttribute(ortho_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kOrthoSmem));
  auto* p = new (std::nothrow) vbsr_ortho;
  if (p == nullptr) return set_error(VBSR_OUT_OF_MEMORY, "host allocation failed");
  p->m = m;
  p->device = m->d.device;
  *out = p;
  return VBSR_OK;
}

vbsr_status vbsr_ortho_destroy(vbsr_ortho* p) {
  clear_error();
  delete p;
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
  const MatrixData& d = p->m->d;
  if (d.nnzb == 0) return VBSR_OK;
  if (values == nullptr || out == nullptr)
    return set_error(VBSR_INVALID_ARGUMENT, "null values or out");
  DeviceGuard guard(p->device);
  ortho_kernel<<<unsigned(d.nnzb), 256, kOrthoSmem, reinterpret_cast<cudaStream_t>(stream)>>>(
      view_of(d), values, out, steps, eps, coefficients[0], coefficients[1], coefficients[2]);
  VBSR_CUDA(cudaGetLastError());
  return VBSR_OK;
}

}  // extern "C"
