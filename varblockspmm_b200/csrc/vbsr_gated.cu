// vbsr_gated.cu — the gated feed-forward block: H = act(A_gate B) * (A_up B), and its backward pass.
#include <cuda_runtime.h>

#include <algorithm>
#include <new>
#include <vector>

#include "vbsr_internal.h"
#include "vbsr_lm.cuh"
#include "vbsr_tiles.h"

using namespace vbsr_b200;

struct vbsr_gated {
  const vbsr_matrix *gate = nullptr, *up = nullptr;
  int device = 0, act = 0;
  int32_t block_cols = 0;
  int64_t M = 0, K = 0;
  float* values[2] = {nullptr, nullptr};  // packed weights: gate, up
  // blocks by block column, gate then up: col_ptr[2 * j + which] .. col_ptr[2 * j + which + 1]
  int32_t* d_col_ptr = nullptr;
  int32_t* d_col_blk = nullptr;
  int32_t* d_col_row = nullptr;
  int* d_status = nullptr;
};

namespace {

constexpr int kTok = 8;  // tokens per CTA

// Packed values of a matrix from its device format.
__global__ void unpack_blocks(vbsr_device_matrix a, float* out) {
  const int b = blockIdx.x;
  const int h = a.row_size[row_of_block(a.row_ptr, a.block_rows, b)], w = a.col_size[a.block_col[b]];
  const long long vo = a.value_off[b];
  for (int i = threadIdx.x; i < h * w; i += blockDim.x)
    out[vo + i] = a.values[vo + blk_pos(h, w, i % h, i / h)];
}

// One CTA per block row and kTok tokens; a thread sums one (row, token) of G and U.
__global__ void gated_forward_kernel(vbsr_device_matrix ga, vbsr_device_matrix ua, const float* gv,
                                     const float* uv, const float* B, long long tokens, int act,
                                     float* H, float* G, float* U) {
  const int row = blockIdx.x, h = ga.row_size[row];
  const long long M = ga.scalar_rows, K = ga.scalar_cols, t0 = (long long)blockIdx.y * kTok;
  for (int i = threadIdx.x; i < h * kTok; i += blockDim.x) {
    const int r = i % h;
    const long long t = t0 + i / h;
    if (t >= tokens) continue;
    float s[2];
    for (int which = 0; which < 2; ++which) {
      const vbsr_device_matrix& a = which ? ua : ga;
      const float* v = which ? uv : gv;
      float sum = 0.0f;
      for (int b = a.row_ptr[row]; b < a.row_ptr[row + 1]; ++b) {
        const int c = a.block_col[b], w = a.col_size[c];
        const float* x = B + t * K + a.col_scalar_off[c];
        const float* av = v + a.value_off[b] + r;
        float part = 0.0f;
        for (int k = 0; k < w; ++k) part = fmaf(av[(long long)k * h], x[k], part);
        sum += part;
      }
      s[which] = sum;
    }
    const long long o = t * M + ga.row_scalar_off[row] + r;
    H[o] = act_value(act, s[0]) * s[1];
    if (G != nullptr) {
      G[o] = s[0];
      U[o] = s[1];
    }
  }
}

__global__ void gated_dact_kernel(const float* G, const float* U, const float* dH, long long n,
                                  int act, float* dG, float* dU) {
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n;
       i += (long long)gridDim.x * blockDim.x) {
    float a, da;
    act_both(act, G[i], a, da);
    dG[i] = dH[i] * U[i] * da;
    dU[i] = dH[i] * a;
  }
}

// One CTA per block column and kTok tokens: dB = A_gate^T dG + A_up^T dU.
__global__ void gated_dinput_kernel(vbsr_device_matrix ga, vbsr_device_matrix ua, const float* gv,
                                    const float* uv, const int32_t* col_ptr, const int32_t* col_blk,
                                    const int32_t* col_row, const float* dG, const float* dU,
                                    long long tokens, float* dB) {
  const int col = blockIdx.x, w = ga.col_size[col];
  const long long M = ga.scalar_rows, K = ga.scalar_cols, t0 = (long long)blockIdx.y * kTok;
  for (int i = threadIdx.x; i < w * kTok; i += blockDim.x) {
    const int c = i % w;
    const long long t = t0 + i / w;
    if (t >= tokens) continue;
    float sum = 0.0f;
    for (int which = 0; which < 2; ++which) {
      const vbsr_device_matrix& a = which ? ua : ga;
      const float* v = which ? uv : gv;
      const float* dy = (which ? dU : dG) + t * M;
      for (int e = col_ptr[2 * col + which]; e < col_ptr[2 * col + which + 1]; ++e) {
        const int row = col_row[e], h = a.row_size[row];
        const float* av = v + a.value_off[col_blk[e]] + (long long)c * h;
        const float* d = dy + a.row_scalar_off[row];
        float part = 0.0f;
        for (int r = 0; r < h; ++r) part = fmaf(av[r], d[r], part);
        sum += part;
      }
    }
    dB[t * K + ga.col_scalar_off[col] + c] = sum;
  }
}

// One CTA per block: dA = dY B^T at its h x w elements.
__global__ void gated_dweight_kernel(vbsr_device_matrix a, const float* B, const float* dY,
                                     long long tokens, float* out) {
  const int b = blockIdx.x, row = row_of_block(a.row_ptr, a.block_rows, b), c = a.block_col[b];
  const int h = a.row_size[row], w = a.col_size[c];
  for (int i = threadIdx.x; i < h * w; i += blockDim.x) {
    const float* d = dY + a.row_scalar_off[row] + i % h;
    const float* x = B + a.col_scalar_off[c] + i / h;
    float sum = 0.0f;
    for (long long t = 0; t < tokens; ++t) sum = fmaf(d[t * a.scalar_rows], x[t * a.scalar_cols], sum);
    out[a.value_off[b] + i] = sum;
  }
}

int64_t dact_bytes(const vbsr_gated* p, int64_t tokens) { return align256(4 * p->M * tokens); }

vbsr_status build_gated(vbsr_gated* p) {
  const MatrixData* m[2] = {&p->gate->d, &p->up->d};
  const int S = p->block_cols;
  std::vector<int32_t> ptr(size_t(2) * S + 1, 0);
  for (int which = 0; which < 2; ++which)
    for (int32_t c : m[which]->h_block_col) ++ptr[2 * size_t(c) + which + 1];
  for (size_t i = 1; i < ptr.size(); ++i) ptr[i] += ptr[i - 1];
  std::vector<int32_t> blk(std::max(1, ptr.back())), row(blk.size()), at(ptr.begin(), ptr.end() - 1);
  for (int which = 0; which < 2; ++which)
    for (int i = 0; i < m[which]->block_rows; ++i)
      for (int b = m[which]->h_row_ptr[i]; b < m[which]->h_row_ptr[i + 1]; ++b) {
        const int e = at[2 * size_t(m[which]->h_block_col[b]) + which]++;
        blk[e] = b;
        row[e] = i;
      }
  VBSR_CUDA(upload_array(&p->d_col_ptr, ptr));
  VBSR_CUDA(upload_array(&p->d_col_blk, blk));
  VBSR_CUDA(upload_array(&p->d_col_row, row));
  VBSR_CUDA(cudaMalloc(&p->d_status, kStatusWords * sizeof(int)));
  VBSR_CUDA(cudaMemset(p->d_status, 0, kStatusWords * sizeof(int)));
  for (int which = 0; which < 2; ++which) {
    VBSR_CUDA(cudaMalloc(&p->values[which], 4 * std::max<int64_t>(1, m[which]->nvalues)));
    if (m[which]->nnzb > 0)
      unpack_blocks<<<unsigned(m[which]->nnzb), 256>>>(view_of(*m[which]), p->values[which]);
  }
  VBSR_CUDA(cudaGetLastError());
  VBSR_CUDA(cudaStreamSynchronize(nullptr));
  return VBSR_OK;
}

void free_gated(vbsr_gated* p) {
  if (p == nullptr) return;
  DeviceGuard guard(p->device);
  cudaFree(p->values[0]);
  cudaFree(p->values[1]);
  cudaFree(p->d_col_ptr);
  cudaFree(p->d_col_blk);
  cudaFree(p->d_col_row);
  cudaFree(p->d_status);
  delete p;
}

vbsr_status check_panel(const vbsr_gated* p, int64_t tokens, const void* workspace,
                        int64_t workspace_bytes, int backward) {
  if (p == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null plan");
  int64_t need = 0;
  const vbsr_status st = vbsr_gated_workspace_bytes(p, tokens, backward, &need);
  if (st != VBSR_OK) return st;
  return check_workspace(workspace, workspace_bytes, need);
}

}  // namespace

extern "C" {

vbsr_status vbsr_gated_create(const vbsr_matrix* gate, const vbsr_matrix* up, int activation,
                              vbsr_gated** out) {
  clear_error();
  if (out == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null output");
  *out = nullptr;
  if (gate == nullptr || up == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null matrix");
  if (activation < VBSR_ACT_SILU || activation > VBSR_ACT_SIGMOID)
    return set_error(VBSR_INVALID_ARGUMENT, "unknown activation");
  const MatrixData &g = gate->d, &u = up->d;
  if (g.device != u.device)
    return set_error(VBSR_INVALID_ARGUMENT, "gate and up are on different devices");
  if (g.h_row_size != u.h_row_size || g.h_col_size != u.h_col_size)
    return set_error(VBSR_INVALID_ARGUMENT, "gate and up have different block partitions");
  auto* p = new (std::nothrow) vbsr_gated;
  if (p == nullptr) return set_error(VBSR_OUT_OF_MEMORY, "host allocation failed");
  p->gate = gate;
  p->up = up;
  p->device = g.device;
  p->act = activation;
  p->block_cols = g.block_cols;
  p->M = g.M;
  p->K = g.K;
  DeviceGuard guard(p->device);
  vbsr_status st;
  try {
    st = build_gated(p);
  } catch (const std::bad_alloc&) {
    st = set_error(VBSR_OUT_OF_MEMORY, "host allocation failed");
  }
  if (st != VBSR_OK) {
    free_gated(p);
    return st;
  }
  *out = p;
  return VBSR_OK;
}

vbsr_status vbsr_gated_destroy(vbsr_gated* p) {
  clear_error();
  free_gated(p);
  return VBSR_OK;
}

vbsr_status vbsr_gated_set_values(vbsr_gated* p, const float* gate_values, const float* up_values,
                                  vbsr_stream_t stream) {
  clear_error();
  if (p == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null plan");
  if ((gate_values == nullptr && p->gate->d.nvalues > 0) ||
      (up_values == nullptr && p->up->d.nvalues > 0))
    return set_error(VBSR_INVALID_ARGUMENT, "null values");
  DeviceGuard guard(p->device);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  VBSR_CUDA(cudaMemcpyAsync(p->values[0], gate_values, 4 * p->gate->d.nvalues,
                            cudaMemcpyDeviceToDevice, s));
  VBSR_CUDA(cudaMemcpyAsync(p->values[1], up_values, 4 * p->up->d.nvalues,
                            cudaMemcpyDeviceToDevice, s));
  return VBSR_OK;
}

vbsr_status vbsr_gated_workspace_bytes(const vbsr_gated* p, int64_t tokens, int backward,
                                       int64_t* bytes) {
  clear_error();
  if (p == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null plan");
  if (bytes == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null output");
  if (tokens < 0 || tokens > kMaxTokens)
    return set_error(VBSR_INVALID_ARGUMENT, "tokens must be between 0 and 2^22");
  *bytes = backward ? 2 * dact_bytes(p, tokens) : 0;
  return VBSR_OK;
}

vbsr_status vbsr_gated_forward(const vbsr_gated* p, const float* B, int64_t tokens, float* H,
                               float* G, float* U, void* workspace, int64_t workspace_bytes,
                               vbsr_stream_t stream) {
  clear_error();
  const vbsr_status st = check_panel(p, tokens, workspace, workspace_bytes, 0);
  if (st != VBSR_OK) return st;
  if ((G == nullptr) != (U == nullptr))
    return set_error(VBSR_INVALID_ARGUMENT, "G and U are given together or not at all");
  if (tokens == 0) return VBSR_OK;
  if (B == nullptr || H == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null B or H");
  DeviceGuard guard(p->device);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const MatrixData &g = p->gate->d, &u = p->up->d;
  const int64_t step = int64_t(kTok) * 65535;  // grid limit in y
  for (int64_t t0 = 0; t0 < tokens; t0 += step) {
    const int64_t n = std::min(step, tokens - t0);
    const dim3 grid(g.block_rows, unsigned((n + kTok - 1) / kTok));
    gated_forward_kernel<<<grid, 256, 0, s>>>(view_of(g), view_of(u), p->values[0], p->values[1],
                                              B + t0 * p->K, n, p->act, H + t0 * p->M,
                                              G ? G + t0 * p->M : nullptr,
                                              U ? U + t0 * p->M : nullptr);
    VBSR_CUDA(cudaGetLastError());
  }
  return VBSR_OK;
}

vbsr_status vbsr_gated_backward(const vbsr_gated* p, const float* B, const float* G,
                                const float* U, const float* dH, int64_t tokens, float* dB,
                                float* dgate, float* dup, void* workspace,
                                int64_t workspace_bytes, vbsr_stream_t stream) {
  clear_error();
  const vbsr_status st = check_panel(p, tokens, workspace, workspace_bytes, 1);
  if (st != VBSR_OK) return st;
  if ((dgate == nullptr) != (dup == nullptr))
    return set_error(VBSR_INVALID_ARGUMENT, "dgate and dup are given together or not at all");
  if (dgate == nullptr && dB == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "no output");
  if (tokens > 0 && (B == nullptr || G == nullptr || U == nullptr || dH == nullptr))
    return set_error(VBSR_INVALID_ARGUMENT, "null B, G, U or dH");
  DeviceGuard guard(p->device);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const MatrixData &g = p->gate->d, &u = p->up->d;
  if (tokens == 0) {
    if (dgate != nullptr) {
      VBSR_CUDA(cudaMemsetAsync(dgate, 0, 4 * g.nvalues, s));
      VBSR_CUDA(cudaMemsetAsync(dup, 0, 4 * u.nvalues, s));
    }
    return VBSR_OK;
  }
  float* dG = static_cast<float*>(workspace);
  float* dU = reinterpret_cast<float*>(static_cast<char*>(workspace) + dact_bytes(p, tokens));
  gated_dact_kernel<<<1184, 256, 0, s>>>(G, U, dH, p->M * tokens, p->act, dG, dU);
  VBSR_CUDA(cudaGetLastError());
  const int64_t step = int64_t(kTok) * 65535;
  for (int64_t t0 = 0; dB != nullptr && t0 < tokens; t0 += step) {
    const int64_t n = std::min(step, tokens - t0);
    const dim3 grid(p->block_cols, unsigned((n + kTok - 1) / kTok));
    gated_dinput_kernel<<<grid, 256, 0, s>>>(view_of(g), view_of(u), p->values[0], p->values[1],
                                             p->d_col_ptr, p->d_col_blk, p->d_col_row,
                                             dG + t0 * p->M, dU + t0 * p->M, n, dB + t0 * p->K);
    VBSR_CUDA(cudaGetLastError());
  }
  if (dgate != nullptr) {
    if (g.nnzb > 0)
      gated_dweight_kernel<<<unsigned(g.nnzb), 256, 0, s>>>(view_of(g), B, dG, tokens, dgate);
    if (u.nnzb > 0)
      gated_dweight_kernel<<<unsigned(u.nnzb), 256, 0, s>>>(view_of(u), B, dU, tokens, dup);
    VBSR_CUDA(cudaGetLastError());
  }
  return VBSR_OK;
}

vbsr_status vbsr_gated_check_status(const vbsr_gated* p, vbsr_stream_t stream) {
  clear_error();
  if (p == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null plan");
  DeviceGuard guard(p->device);
  return read_status(p->d_status, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
