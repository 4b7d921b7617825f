// vbsr_lm.cuh — pieces shared by the operators for block-sparse layers of language models
// (vbsr_gated.cu, vbsr_int8.cu, vbsr_ortho.cu).
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <memory>
#include <string>
#include <type_traits>
#include <utility>
#include <vector>

#include "vbsr_internal.h"

namespace vbsr_b200 {

constexpr int64_t kMaxTokens = int64_t(1) << 22;

inline int64_t align256(int64_t bytes) { return (bytes + 255) & ~int64_t(255); }

inline vbsr_status check_workspace(const void* ws, int64_t bytes, int64_t need) {
  if (need == 0) return VBSR_OK;
  if (ws == nullptr || bytes < need)
    return set_error(VBSR_INVALID_ARGUMENT, "workspace too small: " + std::to_string(need) +
                                                " bytes are needed");
  if (reinterpret_cast<uintptr_t>(ws) & 255u)
    return set_error(VBSR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
  return VBSR_OK;
}

// A plan's device memory: one allocation, with tables copied from the host and room for what kernels write, each
// 256-byte aligned.
class PlanMemory {
 public:
  template <class T>
  void table(T** dst, std::vector<T> src) {
    const auto kept = std::make_shared<std::vector<T>>(std::move(src));
    add(reinterpret_cast<void**>(dst), kept->size() * sizeof(T), kept->data(), kept);
  }
  template <class T>
  void room(T** dst, int64_t bytes) {
    add(reinterpret_cast<void**>(dst), size_t(bytes), nullptr, nullptr);
  }
  // Allocates *base, sets the pointers and enqueues the copies. This object must live until `s` has been waited for.
  cudaError_t make(char** base, cudaStream_t s) {
    cudaError_t e = cudaMalloc(reinterpret_cast<void**>(base), std::max<size_t>(bytes_, 1));
    for (size_t i = 0; i < parts_.size() && e == cudaSuccess; ++i) {
      const Part& p = parts_[i];
      *p.dst = *base + p.at;
      if (p.src != nullptr && p.bytes > 0) e = cudaMemcpyAsync(*p.dst, p.src, p.bytes, cudaMemcpyHostToDevice, s);
    }
    return e;
  }

 private:
  struct Part {
    void** dst;
    size_t at, bytes;
    const void* src;
    std::shared_ptr<void> kept;
  };
  void add(void** dst, size_t bytes, const void* src, std::shared_ptr<void> kept) {
    parts_.push_back({dst, bytes_, bytes, src, std::move(kept)});
    bytes_ += size_t(align256(int64_t(std::max<size_t>(bytes, 1))));
  }
  std::vector<Part> parts_;
  size_t bytes_ = 0;
};

// Reads and clears a plan's device status word after the work on `s`.
inline vbsr_status read_status(int* d_status, cudaStream_t s) {
  int st[kStatusWords] = {};
  VBSR_CUDA(cudaMemcpyAsync(st, d_status, sizeof(st), cudaMemcpyDeviceToHost, s));
  VBSR_CUDA(cudaMemsetAsync(d_status, 0, sizeof(st), s));
  VBSR_CUDA(cudaStreamSynchronize(s));
  if (st[kStatusCode] == VBSR_OK) return VBSR_OK;
  if (st[kStatusCode] == VBSR_TIMEOUT)
    return set_error(VBSR_TIMEOUT, "an in-kernel wait gave up (CTA " +
                                       std::to_string(st[kStatusInfo]) + ")");
  return set_error(VBSR_CUDA_ERROR, "kernel status " + std::to_string(st[kStatusCode]));
}

// Non-owning view of a matrix's device arrays (values in the device format).
inline vbsr_device_matrix view_of(const MatrixData& d) {
  return {d.block_rows, d.block_cols, int32_t(d.nnzb), d.M, d.K, d.d_row_ptr, d.d_block_col,
          d.d_row_size, d.d_col_size, d.d_row_off, d.d_col_off, d.d_value_off, d.d_values};
}

// An activation and its derivative. The exponential and the quotient are the fast ones, whose documented errors
// are (2 + 1.173 |x|) 2^-23 and 2^-22 of themselves. With t = exp(-|x|), the sigmoid of |x| is r = 1 / (1 + t) and
// that of -|x| is t r, so neither it nor its complement is a difference: both are off by at most
// (6 + 1.2 |x|) 2^-23 of themselves, and nothing overflows. GELU's (1 + erf) / 2 is off by about 2^-24 absolutely,
// which for x far below zero is not small against it.
template <int ACT>
__device__ __forceinline__ void act_both(float x, float& a, float& da) {
  if (ACT == VBSR_ACT_RELU) {
    a = x > 0.0f ? x : (x != x ? x : 0.0f);
    da = x > 0.0f ? 1.0f : 0.0f;
  } else if (ACT == VBSR_ACT_GELU) {
    const float cdf = 0.5f * (1.0f + erff(x * 0.70710678118654752f));
    a = x * cdf;
    da = cdf + x * __expf(-0.5f * x * x) * 0.39894228040143268f;
  } else {
    const float t = __expf(-fabsf(x)), r = __fdividef(1.0f, 1.0f + t), q = t * r;
    const float s = x >= 0.0f ? r : q, c = x >= 0.0f ? q : r;  // the sigmoids of x and of -x
    if (ACT == VBSR_ACT_SIGMOID) {
      a = s;
      da = s * c;
    } else {
      a = x * s;
      da = s * (1.0f + x * c);
    }
  }
}
// f(std::integral_constant<int, ACT>) for the activation at hand, chosen once.
template <class F>
__device__ __forceinline__ void with_act(int act, F f) {
  switch (act) {
    case VBSR_ACT_SILU: f(std::integral_constant<int, VBSR_ACT_SILU>()); break;
    case VBSR_ACT_GELU: f(std::integral_constant<int, VBSR_ACT_GELU>()); break;
    case VBSR_ACT_RELU: f(std::integral_constant<int, VBSR_ACT_RELU>()); break;
    default: f(std::integral_constant<int, VBSR_ACT_SIGMOID>()); break;
  }
}

}  // namespace vbsr_b200
