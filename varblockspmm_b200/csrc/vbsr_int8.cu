// vbsr_int8.cu — products in 8-bit integers: C = diag(row_scale) (Aq Q) diag(token_scale).
#include <cuda_runtime.h>

#include <algorithm>
#include <new>

#include "vbsr_internal.h"
#include "vbsr_lm.cuh"
#include "vbsr_tiles.h"

using namespace vbsr_b200;

struct vbsr_int8 {
  const vbsr_matrix* m = nullptr;
  int device = 0;
  int64_t M = 0, K = 0;
  int8_t* values = nullptr;  // packed
  float* row_scale = nullptr;
  int* d_status = nullptr;
};

namespace {

constexpr int kTok = 8;                     // tokens per CTA
constexpr int64_t kMaxRowWidth = 131072;    // 127 * 127 * width stays below 2^31

// The integer nearest to x / s, ties to even, as of the exact quotient (s > 0, |x| <= 127.5 s up to
// rounding). The fp32 quotient can round onto or across a half; the residual x - q s is exact in
// fma (|q| <= 128 and the difference is at most about s), and its comparison with s / 2 decides.
__device__ __forceinline__ int quantize_exact(float x, float s) {
  float q = rintf(x / s);
  const float r = fmaf(-q, s, x), half = 0.5f * s;
  if (r > half || (r == half && (int(q) & 1))) q += 1.0f;
  if (r < -half || (r == -half && (int(q) & 1))) q -= 1.0f;
  return max(-127, min(127, int(q)));
}

// Largest magnitude of a CTA's values; NaN or infinity give NaN.
__device__ __forceinline__ float scale_of(float amax, bool finite) {
  return finite ? amax / 127.0f : __int_as_float(0x7fc00000);
}

__device__ float block_amax(float v, bool& finite) {
  __shared__ float red[32];
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  if (!finite) bad = 1;
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int i = 0; i < int(blockDim.x >> 5); ++i) v = fmaxf(v, red[i]);
  finite = bad == 0;
  __syncthreads();
  return v;
}

// One CTA per token.
__global__ void quantize_panel_kernel(const float* B, long long K, int8_t* Q, float* scale) {
  const float* x = B + (long long)blockIdx.x * K;
  int8_t* q = Q + (long long)blockIdx.x * K;
  float m = 0.0f;
  bool finite = true;
  for (long long i = threadIdx.x; i < K; i += blockDim.x) {
    m = fmaxf(m, fabsf(x[i]));
    finite = finite && isfinite(x[i]);
  }
  m = block_amax(m, finite);
  const float s = scale_of(m, finite);
  if (threadIdx.x == 0) scale[blockIdx.x] = s;
  for (long long i = threadIdx.x; i < K; i += blockDim.x)
    q[i] = int8_t(s > 0.0f ? quantize_exact(x[i], s) : 0);
}

// One warp per scalar row of a block row; one CTA per block row.
__global__ void quantize_rows_kernel(vbsr_device_matrix a, int8_t* values, float* row_scale) {
  const int row = blockIdx.x, h = a.row_size[row], lane = threadIdx.x & 31;
  for (int r = threadIdx.x >> 5; r < h; r += int(blockDim.x >> 5)) {
    float m = 0.0f, s = 0.0f;
    bool finite = true;
    for (int pass = 0; pass < 2; ++pass) {
      for (int b = a.row_ptr[row]; b < a.row_ptr[row + 1]; ++b) {
        const int w = a.col_size[a.block_col[b]];
        const long long vo = a.value_off[b];
        for (int k = lane; k < w; k += 32) {
          const float x = a.values[vo + blk_pos(h, w, r, k)];
          if (pass == 0) {
            m = fmaxf(m, fabsf(x));
            finite = finite && isfinite(x);
          } else {
            values[vo + r + (long long)k * h] = int8_t(s > 0.0f ? quantize_exact(x, s) : 0);
          }
        }
      }
      if (pass == 0) {
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        s = scale_of(m, __all_sync(0xffffffffu, finite));
        if (lane == 0) row_scale[a.row_scalar_off[row] + r] = s;
      }
    }
  }
}

// One CTA per block row and kTok tokens; a thread sums one (row, token).
__global__ void int8_kernel(vbsr_device_matrix a, const int8_t* v, const float* row_scale,
                            const int8_t* Q, const float* token_scale, long long tokens, float* C) {
  const int row = blockIdx.x, h = a.row_size[row];
  const long long t0 = (long long)blockIdx.y * kTok;
  for (int i = threadIdx.x; i < h * kTok; i += blockDim.x) {
    const int r = i % h;
    const long long t = t0 + i / h;
    if (t >= tokens) continue;
    int sum = 0;
    for (int b = a.row_ptr[row]; b < a.row_ptr[row + 1]; ++b) {
      const int c = a.block_col[b], w = a.col_size[c];
      const int8_t* x = Q + t * a.scalar_cols + a.col_scalar_off[c];
      const int8_t* av = v + a.value_off[b] + r;
      for (int k = 0; k < w; ++k) sum += int(av[(long long)k * h]) * int(x[k]);
    }
    const long long o = a.row_scalar_off[row] + r;
    C[t * a.scalar_rows + o] = float(sum) * (token_scale[t] * row_scale[o]);
  }
}

vbsr_status launch_quantize(const float* B, int64_t K, int64_t tokens, int8_t* Q, float* scale,
                            cudaStream_t s) {
  if (tokens > 0) quantize_panel_kernel<<<unsigned(tokens), 256, 0, s>>>(B, K, Q, scale);
  VBSR_CUDA(cudaGetLastError());
  return VBSR_OK;
}

vbsr_status launch_int8(const vbsr_int8* p, const int8_t* Q, const float* scale, int64_t tokens,
                        float* C, cudaStream_t s) {
  const MatrixData& d = p->m->d;
  const int64_t step = int64_t(kTok) * 65535;  // grid limit in y
  for (int64_t t0 = 0; t0 < tokens; t0 += step) {
    const int64_t n = std::min(step, tokens - t0);
    const dim3 grid(d.block_rows, unsigned((n + kTok - 1) / kTok));
    int8_kernel<<<grid, 256, 0, s>>>(view_of(d), p->values, p->row_scale, Q + t0 * p->K, scale + t0,
                                     n, C + t0 * p->M);
    VBSR_CUDA(cudaGetLastError());
  }
  return VBSR_OK;
}

int64_t q_bytes(const vbsr_int8* p, int64_t tokens) { return align256(p->K * tokens); }

void free_int8(vbsr_int8* p) {
  if (p == nullptr) return;
  DeviceGuard guard(p->device);
  cudaFree(p->values);
  cudaFree(p->row_scale);
  cudaFree(p->d_status);
  delete p;
}

vbsr_status build_int8(vbsr_int8* p, const int8_t* values, const float* row_scale) {
  const MatrixData& d = p->m->d;
  VBSR_CUDA(cudaMalloc(&p->values, std::max<int64_t>(1, d.nvalues)));
  VBSR_CUDA(cudaMalloc(&p->row_scale, 4 * d.M));
  VBSR_CUDA(cudaMalloc(&p->d_status, kStatusWords * sizeof(int)));
  VBSR_CUDA(cudaMemset(p->d_status, 0, kStatusWords * sizeof(int)));
  VBSR_CUDA(cudaMemcpy(p->values, values, d.nvalues, cudaMemcpyDeviceToDevice));
  VBSR_CUDA(cudaMemcpy(p->row_scale, row_scale, 4 * d.M, cudaMemcpyDeviceToDevice));
  VBSR_CUDA(cudaStreamSynchronize(nullptr));
  return VBSR_OK;
}

}  // namespace

extern "C" {

vbsr_status vbsr_int8_create(const vbsr_matrix* m, const int8_t* values, const float* row_scale,
                             vbsr_int8** out) {
  clear_error();
  if (out == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null output");
  *out = nullptr;
  if (m == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null matrix");
  if (row_scale == nullptr || (values == nullptr && m->d.nvalues > 0))
    return set_error(VBSR_INVALID_ARGUMENT, "null values or row_scale");
  for (int64_t w : m->d.h_sum_w)
    if (w > kMaxRowWidth)
      return set_error(VBSR_INVALID_ARGUMENT,
                       "a block row wider than 131072 columns could overflow the 32-bit sum");
  auto* p = new (std::nothrow) vbsr_int8;
  if (p == nullptr) return set_error(VBSR_OUT_OF_MEMORY, "host allocation failed");
  p->m = m;
  p->device = m->d.device;
  p->M = m->d.M;
  p->K = m->d.K;
  DeviceGuard guard(p->device);
  vbsr_status st;
  try {
    st = build_int8(p, values, row_scale);
  } catch (const std::bad_alloc&) {
    st = set_error(VBSR_OUT_OF_MEMORY, "host allocation failed");
  }
  if (st != VBSR_OK) {
    free_int8(p);
    return st;
  }
  *out = p;
  return VBSR_OK;
}

vbsr_status vbsr_int8_destroy(vbsr_int8* p) {
  clear_error();
  free_int8(p);
  return VBSR_OK;
}

vbsr_status vbsr_int8_workspace_bytes(const vbsr_int8* p, int64_t tokens, int64_t* bytes) {
  clear_error();
  if (p == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null plan");
  if (bytes == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null output");
  if (tokens < 0 || tokens > kMaxTokens)
    return set_error(VBSR_INVALID_ARGUMENT, "tokens must be between 0 and 2^22");
  *bytes = q_bytes(p, tokens) + align256(4 * tokens);
  return VBSR_OK;
}

vbsr_status vbsr_int8_execute(const vbsr_int8* p, const int8_t* Q, const float* token_scale,
                              int64_t tokens, float* C, void* workspace, int64_t workspace_bytes,
                              vbsr_stream_t stream) {
  clear_error();
  int64_t need = 0;
  vbsr_status st = vbsr_int8_workspace_bytes(p, tokens, &need);
  if (st == VBSR_OK) st = check_workspace(workspace, workspace_bytes, need);
  if (st != VBSR_OK || tokens == 0) return st;
  if (Q == nullptr || token_scale == nullptr || C == nullptr)
    return set_error(VBSR_INVALID_ARGUMENT, "null Q, token_scale or C");
  DeviceGuard guard(p->device);
  return launch_int8(p, Q, token_scale, tokens, C, reinterpret_cast<cudaStream_t>(stream));
}

vbsr_status vbsr_int8_execute_panel(const vbsr_int8* p, const float* B, int64_t tokens, float* C,
                                    void* workspace, int64_t workspace_bytes,
                                    vbsr_stream_t stream) {
  clear_error();
  int64_t need = 0;
  vbsr_status st = vbsr_int8_workspace_bytes(p, tokens, &need);
  if (st == VBSR_OK) st = check_workspace(workspace, workspace_bytes, need);
  if (st != VBSR_OK || tokens == 0) return st;
  if (B == nullptr || C == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null B or C");
  DeviceGuard guard(p->device);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int8_t* Q = static_cast<int8_t*>(workspace);
  float* scale = reinterpret_cast<float*>(Q + q_bytes(p, tokens));
  st = launch_quantize(B, p->K, tokens, Q, scale, s);
  if (st != VBSR_OK) return st;
  return launch_int8(p, Q, scale, tokens, C, s);
}

vbsr_status vbsr_int8_check_status(const vbsr_int8* p, vbsr_stream_t stream) {
  clear_error();
  if (p == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null plan");
  DeviceGuard guard(p->device);
  return read_status(p->d_status, reinterpret_cast<cudaStream_t>(stream));
}

vbsr_status vbsr_quantize_panel(const float* B, int64_t K, int64_t tokens, int8_t* Q,
                                float* token_scale, vbsr_stream_t stream) {
  clear_error();
  if (tokens < 0 || tokens > kMaxTokens)
    return set_error(VBSR_INVALID_ARGUMENT, "tokens must be between 0 and 2^22");
  if (K <= 0) return set_error(VBSR_INVALID_ARGUMENT, "K must be positive");
  if (tokens == 0) return VBSR_OK;
  if (B == nullptr || Q == nullptr || token_scale == nullptr)
    return set_error(VBSR_INVALID_ARGUMENT, "null B, Q or token_scale");
  return launch_quantize(B, K, tokens, Q, token_scale, reinterpret_cast<cudaStream_t>(stream));
}

vbsr_status vbsr_matrix_quantize(const vbsr_matrix* m, int8_t* values, float* row_scale,
                                 vbsr_stream_t stream) {
  clear_error();
  if (m == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null matrix");
  if (row_scale == nullptr || (values == nullptr && m->d.nvalues > 0))
    return set_error(VBSR_INVALID_ARGUMENT, "null values or row_scale");
  DeviceGuard guard(m->d.device);
  quantize_rows_kernel<<<m->d.block_rows, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      view_of(m->d), values, row_scale);
  VBSR_CUDA(cudaGetLastError());
  return VBSR_OK;
}

}  // extern "C"
