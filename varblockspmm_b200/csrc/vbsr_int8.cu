// vbsr_int8.cu — products in 8-bit integers: C = diag(row_scale) (Aq Q) diag(token_scale).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <new>
#include <vector>

#include "vbsr_internal.h"
#include "vbsr_lm.cuh"
#include "vbsr_pair_host.cuh"
#include "vbsr_panels.cuh"
#include "vbsr_tiles.h"

using namespace vbsr_b200;

// A block row in the packed layout and in ours (lay_weights_kernel).
struct LayRow {
  uint64_t val, out;   // first packed value, first byte
  uint32_t c0, chunks; // of chunk_src
  uint32_t row0, h;
};

struct vbsr_int8 {
  int device = 0, num_sm = 148, block_rows = 0;
  int64_t M = 0, K = 0, nvalues = 0;
  bool has_weights = false;
  char* w = nullptr;  // weights in 16-column chunks
  uint32_t* chunk_col = nullptr;
  // where the chunks' weights are in the packed layout
  LayRow* lay = nullptr;
  uint32_t* chunk_src = nullptr;
  RowUnit* rows[4] = {};
  int row_units[4] = {};
  int max_height = 64;
  float* row_scale = nullptr;
  int* d_status = nullptr;
  char* memory = nullptr;  // of all the above
};

namespace {

constexpr int64_t kMaxRowWidth = 131071;  // 128 * 128 * width stays below 2^31

// A scale ready for use: s is a normal number far from the smallest (tiny scales and the values that go
// with them are multiplied by 2^120, exactly); s = 0 stands for a scale that is 0 or NaN.
struct Quantizer {
  float s, inv, up;
  Quantizer() = default;
  __device__ __forceinline__ explicit Quantizer(float scale) {
    up = scale < 1e-30f ? __int_as_float((120 + 127) << 23) : 1.0f;
    s = scale > 0.0f ? scale * up : 0.0f;
    inv = s > 0.0f ? 1.0f / s : 0.0f;
  }
  // The integer nearest to x / s, ties to even, as of the exact quotient (|x| <= 127.5 s up to rounding).
  // x inv is off by less than 2^-15, which can take q across a half but not further; the residual x - q s
  // is exact in fma (|q| <= 128 and the difference is at most about s), and its comparison with s / 2
  // decides.
  __device__ __forceinline__ int operator()(float x) const {
    x *= up;
    int q = __float2int_rn(x * inv);
    const float r = fmaf(-float(q), s, x), half = 0.5f * s, a = fabsf(r);
    if (a > half || (a == half && (q & 1))) q += r > 0.0f ? 1 : -1;
    return s > 0.0f ? max(-127, min(127, q)) : 0;
  }
};

// The scale for a largest magnitude: times the fp32 number nearest to 1 / 127, one rounding; NaN where there
// is a NaN or an infinity.
__device__ __forceinline__ float scale_of(float amax, bool finite) {
  return finite ? amax * (1.0f / 127.0f) : __int_as_float(0x7fc00000);
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
  const Quantizer quant(s);
  if (threadIdx.x == 0) scale[blockIdx.x] = s;
  for (long long i = threadIdx.x; i < K; i += blockDim.x)
    q[i] = int8_t(quant(x[i]));
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
            values[vo + r + (long long)k * h] = int8_t(Quantizer(s)(x));
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

// ---- operands of the tensor-core product (pair_kernel<kInt8>, vbsr_pair.cuh) ----------------------
//
// An MMA step takes K = 32, two chunks of 16 columns. A block of width w is cut into chunks from its
// first column; the last chunk of a width that is 8 mod 16 is filled with zero weights (11% more bytes
// over the eight widths). Blocks start at multiples of 8, so the panel holds a 16-column chunk from
// every multiple of 8 on, each column twice: the even ones first, then the odd ones, so that the chunks
// of a block are neighbours and arrive with one copy. Per tile of R tokens, a chunk is R rows of 16
// bytes.
__host__ __device__ constexpr int64_t chunk_place(int64_t col8, int64_t K) {
  return (col8 & 1) * ((K / 8 + 1) / 2) + (col8 >> 1);
}

// A block row's weights from the packed layout, [chunk][h rows][16], and its scales. The columns of a chunk are
// neighbours in the packed layout; a thread takes 8 rows of a chunk, 8 bytes of every column, and turns them.
// chunk_src: first column of a chunk among the columns of its block row's blocks, in eights, times 2; + 1 where
// the chunk has 8 columns.
__global__ void __launch_bounds__(128) lay_weights_kernel(const LayRow* rows, const uint32_t* chunk_src,
                                                          const int8_t* values, int vec, const float* scale,
                                                          char* out, float* scale_out) {
  const LayRow r = rows[blockIdx.x];
  const uint32_t h8 = r.h / 8;
  if (threadIdx.x < r.h) scale_out[r.row0 + threadIdx.x] = scale[r.row0 + threadIdx.x];
  for (uint32_t i = threadIdx.x; i < r.chunks * h8; i += blockDim.x) {
    const uint32_t c = i / h8, g = i % h8, src = chunk_src[r.c0 + c];
    const int8_t* v = values + r.val + (unsigned long long)(src >> 1) * 8 * r.h + 8 * g;
    uint2 q[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      q[k] = make_uint2(0, 0);
      if (k >= 8 && (src & 1)) continue;
      if (vec) {
        q[k] = *reinterpret_cast<const uint2*>(v + k * r.h);
      } else {
        for (int b = 0; b < 4; ++b) {
          q[k].x |= uint32_t(uint8_t(v[k * r.h + b])) << 8 * b;
          q[k].y |= uint32_t(uint8_t(v[k * r.h + 4 + b])) << 8 * b;
        }
      }
    }
    uint4* o = reinterpret_cast<uint4*>(out + r.out + 16ull * (c * r.h + 8 * g));
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // row j: byte j of every column
      uint32_t w[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        auto half = [&](int k) { return j < 4 ? q[k].x : q[k].y; };
        const uint32_t pick = uint32_t(j & 3) | uint32_t(4 + (j & 3)) << 4;
        w[m] = __byte_perm(__byte_perm(half(4 * m), half(4 * m + 1), pick),
                           __byte_perm(half(4 * m + 2), half(4 * m + 3), pick), 0x5410);
      }
      o[j] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// Largest magnitude of each of `splits` equal parts of every token, or NaN: grid (splits, tokens).
__global__ void __launch_bounds__(256) token_amax_kernel(const float* B, long long K, int vec,
                                                         float* partial) {
  griddep_launch_dependents();
  const float* x = B + (long long)blockIdx.y * K;
  const long long g0 = (K / 8) * blockIdx.x / gridDim.x, g1 = (K / 8) * (blockIdx.x + 1) / gridDim.x;
  float m = 0.0f;
  bool finite = true;
  for (long long g = g0 + threadIdx.x; g < g1; g += blockDim.x) {
    float v[8];
    load8(x + 8 * g, vec, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m = fmaxf(m, fabsf(v[i]));
      finite = finite && isfinite(v[i]);
    }
  }
  m = block_amax(m, finite);
  if (threadIdx.x == 0)
    partial[(long long)blockIdx.y * gridDim.x + blockIdx.x] = finite ? m : __int_as_float(0x7fc00000);
}

// The panel's chunks of one tile per grid row. FLOAT: from fp32 values (partial maxima given, scales
// written), else from int8 ones. Blocks of tokens x groups (UNITS of 8 columns) go through shared memory, as
// panel_pair_kernel's; the group behind a block is read too, for the second half of its last chunk.
template <bool FLOAT, int UNITS>
__global__ void __launch_bounds__(256) chunk_panel_kernel(const void* src, long long tokens, long long K,
                                                          int R, int vec, const float* partial, int splits,
                                                          float* token_scale, char* out) {
  __shared__ Quantizer quant[128];
  __shared__ uint2 q8[UNITS + 32];
  griddep_launch_dependents();
  griddep_wait();
  const long long t0 = (long long)blockIdx.y * R, groups = K / 8;
  if (FLOAT) {
    for (int r = threadIdx.x; r < R && t0 + r < tokens; r += blockDim.x) {
      float m = 0.0f;
      bool finite = true;
      for (int i = 0; i < splits; ++i) {
        const float x = partial[(t0 + r) * splits + i];
        finite = finite && x == x;
        m = fmaxf(m, x);
      }
      const float s = scale_of(m, finite);
      quant[r] = Quantizer(s);
      if (blockIdx.x == 0) token_scale[t0 + r] = s;
    }
  }
  char* tile = out + t0 * groups * 16;
  const PanelBlocks b(R, 1, groups, UNITS);
  union Octet {
    int8_t q[8];
    uint2 u;
  };
  for (long long item = blockIdx.x; item < b.items; item += gridDim.x) {
    const PanelBlocks::Place at = b.place(item);
    auto live = [&](int r, int g) { return at.r + r < R && t0 + at.r + r < tokens && at.g + g < groups; };
    auto place = [&](int r, int g) { return (t0 + at.r + r) * K + 8 * (at.g + g); };
    auto octet = [&](int r, int g) {  // 8 columns as they are, or quantised
      Octet x;
      x.u = make_uint2(0, 0);
      if (!live(r, g)) return x.u;
      if (FLOAT) {
        float v[8];
        load8(static_cast<const float*>(src) + place(r, g), vec, v);
        const Quantizer q = quant[at.r + r];
#pragma unroll
        for (int k = 0; k < 8; ++k) x.q[k] = int8_t(q(v[k]));
      } else if (vec) {
        x.u = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(src) + place(r, g));
      } else {
        for (int k = 0; k < 8; ++k) x.q[k] = static_cast<const int8_t*>(src)[place(r, g) + k];
      }
      return x.u;
    };
    __syncthreads();
#pragma unroll
    for (int k = 0; k < UNITS / 256; ++k) {
      const int u = threadIdx.x + 256 * k, r = u >> b.gg_log, g = u & (b.gg - 1);
      q8[b.slot(r, g)] = octet(r, g);
    }
    if (int(threadIdx.x) < b.tt) q8[b.slot(threadIdx.x, b.gg)] = octet(threadIdx.x, b.gg);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < UNITS / 256; ++k) {
      const int u = threadIdx.x + 256 * k, r = u & (b.tt - 1), g = u >> b.tt_log;
      if (at.r + r >= R || at.g + g >= groups) continue;
      const uint2 first = q8[b.slot(r, g)], second = q8[b.slot(r, g + 1)];
      *reinterpret_cast<uint4*>(tile + (chunk_place(at.g + g, K) * R + at.r + r) * 16) =
          make_uint4(first.x, first.y, second.x, second.y);
    }
  }
}

// Few or long tokens, up to kHeldFeatures: scales and chunks in one launch, a cluster of kTokenCtas CTAs for two
// tokens. A lane takes 8 columns of one of them, kTokenHeld times, which stay in its registers from their one
// read until the CTAs have exchanged their largest magnitudes through distributed shared memory. A warp reads
// 16 neighbouring groups and writes the 15 chunks that begin in the first 15, the second half of a chunk coming
// from the lane of the next group: 16 bytes of both tokens side by side, a whole sector of 32. Against the two
// kernels above it saves a launch and a read, but every two tokens take a cluster, whose lanes short tokens leave
// idle. Whole calls, 64 block rows of 4 blocks, this and the two kernels, us:
//   tokens  K = 2048    4096        8192        16384       24576       38400
//   64      10.0  11.5  9.8   11.8  10.4  12.9  10.7  14.1  12.2  16.4  12.7  20.1
//   128     9.9   11.6  10.6  12.5  10.9  13.9  13.1  16.4  14.4  20.6  16.5  26.7
//   256     14.3  12.9  14.6  15.9  16.3  16.5  18.5  22.6  20.6  28.8  24.7  41.3
//   512     20.6  15.8  22.3  16.5  24.7  22.6  28.8  29.1  33.1  45.0  41.1  63.0
//   1024    34.5  18.5  37.0  22.6  41.1  30.7  51.3  51.3  59.2  69.4  71.8  102
//   4096    117   41    128   58    144   93    179   155   208   223   255   328
// So it takes up to 128 tokens, or one for every 24 features, and any number of tokens longer than 16384.
constexpr int kTokenCtas = 8, kTokenThreads = 256, kTokenWarps = kTokenThreads / 32, kTokenHeld = 5;
constexpr int64_t kHeldFeatures = 8ll * 15 * kTokenCtas * kTokenWarps * kTokenHeld;  // 38400
inline bool by_clusters(int64_t tokens, int64_t K) {
  return K <= kHeldFeatures && (tokens <= std::max<int64_t>(128, K / 24) || K > 16384);
}
__global__ void __cluster_dims__(kTokenCtas) __launch_bounds__(kTokenThreads, 4)
    token_chunks_kernel(const float* B, long long tokens, long long rows, long long K, int R, int vec,
                        float* token_scale, char* out) {
  __shared__ float red[kTokenWarps][2], maxima[kTokenCtas][2];
  griddep_launch_dependents();
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();  // its CTAs have started, before any writes to another
  const int cta = int(blockIdx.x % kTokenCtas), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, which = lane & 1;
  const long long t = blockIdx.x / kTokenCtas * 2 + which, groups = K / 8;
  const bool live = t < tokens;  // a tile's rows behind the last token are zeros
  const float* x = B + t * K;
  const long long warp_g = 15ll * (cta * kTokenWarps + warp), step = 15ll * kTokenCtas * kTokenWarps;
  auto load = [&](long long base, float (&v)[8]) {
    const long long g = base + (lane >> 1);
    if (live && g < groups) {
      load8(x + 8 * g, vec, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
  };
  constexpr float kInf = __builtin_huge_valf();  // marks a token that holds a NaN or an infinity
  float m = 0.0f;
  float v[kTokenHeld][8];
#pragma unroll
  for (int k = 0; k < kTokenHeld; ++k) load(warp_g + k * step, v[k]);
#pragma unroll
  for (int k = 0; k < kTokenHeld; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, isfinite(v[k][i]) ? fabsf(v[k][i]) : kInf);
#pragma unroll
  for (int o = 16; o > 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane < 2) red[warp][lane] = m;
  __syncthreads();
  cluster.barrier_wait();
  if (threadIdx.x < 2 * kTokenCtas) {
    m = 0.0f;
#pragma unroll
    for (int i = 0; i < kTokenWarps; ++i) m = fmaxf(m, red[i][which]);
    *cluster.map_shared_rank(&maxima[cta][which], threadIdx.x >> 1) = m;
  }
  cluster.sync();
  m = 0.0f;
#pragma unroll
  for (int i = 0; i < kTokenCtas; ++i) m = fmaxf(m, maxima[i][which]);
  const float s = scale_of(m, m < kInf);
  const Quantizer quant(s);
  if (cta == 0 && threadIdx.x < 2 && live) token_scale[t] = s;
  char* row = out + ((t / R) * R * groups + t % R) * 16;
  auto write = [&](long long base, const float (&w)[8]) {
    union {
      int8_t q[8];
      uint2 u;
    } y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y.q[i] = int8_t(quant(w[i]));
    const uint32_t next_x = __shfl_down_sync(0xffffffffu, y.u.x, 2), next_y = __shfl_down_sync(0xffffffffu, y.u.y, 2);
    const long long g = base + (lane >> 1);
    if (lane < 30 && t < rows && g < groups)
      *reinterpret_cast<uint4*>(row + chunk_place(g, K) * R * 16) = make_uint4(y.u.x, y.u.y, next_x, next_y);
  };
#pragma unroll
  for (int k = 0; k < kTokenHeld; ++k)
    if (warp_g + k * step < groups) write(warp_g + k * step, v[k]);
}

vbsr_status launch_quantize(const float* B, int64_t K, int64_t tokens, int8_t* Q, float* scale,
                            cudaStream_t s) {
  if (tokens > 0) quantize_panel_kernel<<<unsigned(tokens), 256, 0, s>>>(B, K, Q, scale);
  VBSR_CUDA(cudaGetLastError());
  return VBSR_OK;
}

// Geometry of a call: even tiles of at most 128 tokens; few tokens are searched for their largest
// magnitude by several CTAs each.
struct Geometry {
  int R = 0, splits = 1;
  int64_t tiles = 0, scale_at = 0, panel_at = 0, bytes = 0;
};
Geometry geometry_of(const vbsr_int8* p, int64_t tokens) {
  Geometry g;
  if (tokens == 0) return g;
  g.tiles = (tokens + 127) / 128;
  g.R = int((tokens + g.tiles - 1) / g.tiles);
  g.splits = int(std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(64, p->K / 1024), 296 / tokens)));
  g.scale_at = align256(4 * tokens * g.splits);
  g.panel_at = g.scale_at + align256(4 * tokens);
  g.bytes = g.panel_at + align256(g.tiles * g.R * (p->K / 8) * 16);
  return g;
}

vbsr_status launch_int8(const vbsr_int8* p, const Geometry& g, const float* scale, int64_t tokens,
                        const char* panel, float* C, cudaStream_t s) {
  PairParams k{};
  k.group_col = p->chunk_col;
  k.R = g.R;
  k.tokens = tokens;
  k.M = p->M;
  k.K = p->K;
  k.x = panel;
  k.w = p->w;
  k.row_scale = p->row_scale;
  k.token_scale = scale;
  k.out0 = C;
  k.vec = aligned16(C);
  k.status = p->d_status;
  choose_rows(k, p->rows, p->row_units, g.tiles, p->num_sm, p->max_height);
  return launch_pair<kInt8>(k, g.tiles, p->num_sm, s);
}

template <bool FLOAT>
vbsr_status launch_chunks(const vbsr_int8* p, const Geometry& g, const void* src, int vec, int64_t tokens,
                          char* ws, cudaStream_t s) {
  const float* partial = reinterpret_cast<const float*>(ws);
  float* scale = reinterpret_cast<float*>(ws + g.scale_at);
  // few values: small blocks, so that there are enough of them
  const bool small = p->K / 8 * g.R * g.tiles < 592 * 1024;
  const int64_t blocks = (p->K / 8 * g.R + (small ? 255 : 1023)) / (small ? 256 : 1024);
  // one grid row per tile (at most 32768, see kMaxTokens)
  const dim3 grid(unsigned(std::max<int64_t>(1, std::min(blocks, 1184 / g.tiles))), unsigned(g.tiles));
  const auto kernel = small ? chunk_panel_kernel<FLOAT, 256> : chunk_panel_kernel<FLOAT, 1024>;
  if (FLOAT) {
    VBSR_CUDA(launch_after(kernel, grid, 256, 0, s, src, tokens, p->K, g.R, vec, partial, g.splits, scale,
                           ws + g.panel_at));
  } else {  // the first kernel of its call: after everything before it
    kernel<<<grid, 256, 0, s>>>(src, tokens, p->K, g.R, vec, partial, g.splits, scale, ws + g.panel_at);
    VBSR_CUDA(cudaGetLastError());
  }
  return VBSR_OK;
}

void free_int8(vbsr_int8* p) {
  if (p == nullptr) return;
  DeviceGuard guard(p->device);
  cudaFree(p->memory);
  delete p;
}

vbsr_status lay_weights(vbsr_int8* p, const int8_t* values, const float* row_scale, cudaStream_t s) {
  lay_weights_kernel<<<unsigned(p->block_rows), 128, 0, s>>>(
      p->lay, p->chunk_src, values, (reinterpret_cast<uintptr_t>(values) & 7u) == 0, row_scale, p->w, p->row_scale);
  VBSR_CUDA(cudaGetLastError());
  p->has_weights = true;
  return VBSR_OK;
}

vbsr_status build_int8(vbsr_int8* p, const MatrixData& d, const int8_t* values, const float* row_scale) {
  p->max_height = *std::max_element(d.h_row_size.begin(), d.h_row_size.end());
  p->block_rows = d.block_rows;
  VBSR_CUDA(cudaDeviceGetAttribute(&p->num_sm, cudaDevAttrMultiProcessorCount, p->device));
  VBSR_CUDA(cudaFuncSetAttribute(pair_kernel<kInt8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kPairSmem));
  std::vector<uint32_t> cols, src;
  std::vector<LayRow> lay;
  std::vector<RowUnit> whole(d.block_rows);
  uint64_t at = 0;
  for (int i = 0; i < d.block_rows; ++i) {
    RowUnit& u = whole[i];
    u.row0 = uint32_t(d.h_row_off[i]);
    u.shape = uint32_t(d.h_row_size[i]);
    u.g0[0] = uint32_t(cols.size());
    u.w0[0] = at;
    uint32_t before = 0;  // columns of the row's blocks so far, in eights
    for (int b = d.h_row_ptr[i]; b < d.h_row_ptr[i + 1]; ++b) {
      const uint32_t col8 = d.h_blk_desc[b] >> 3, w8 = (d.h_blk_desc[b] & 7u) + 1u;
      for (uint32_t c = 0; c < w8; c += 2) {
        cols.push_back(uint32_t(chunk_place(col8 + c, p->K)));
        src.push_back((before + c) << 1 | (c + 1 == w8 ? 1u : 0u));
      }
      before += w8;
    }
    u.ng[0] = uint32_t(cols.size()) - u.g0[0];
    lay.push_back({uint64_t(d.h_val_off_row[i]), at, u.g0[0], u.ng[0], uint32_t(d.h_row_off[i]),
                   uint32_t(d.h_row_size[i])});
    at += uint64_t(16) * d.h_row_size[i] * u.ng[0];
  }
  PlanMemory mem;
  mem.table(&p->chunk_col, std::move(cols));
  mem.table(&p->chunk_src, std::move(src));
  mem.table(&p->lay, std::move(lay));
  add_row_units(mem, whole, p->num_sm, p->rows, p->row_units);
  mem.table(&p->d_status, std::vector<int>(kStatusWords));
  mem.room(&p->w, int64_t(at));
  mem.room(&p->row_scale, 4 * d.M);
  SetupStream s;  // after `mem`: it waits before that goes
  VBSR_CUDA(s.init());
  VBSR_CUDA(mem.make(&p->memory, s.s));
  if (row_scale != nullptr) {
    VBSR_CUDA(cudaDeviceSynchronize());  // the caller's arrays may come from any stream
    const vbsr_status laid = lay_weights(p, values, row_scale, s.s);
    if (laid != VBSR_OK) return laid;
  }
  VBSR_CUDA(s.finish());
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
  if ((row_scale == nullptr) != (values == nullptr) && (row_scale == nullptr || m->d.nvalues > 0))
    return set_error(VBSR_INVALID_ARGUMENT, "null values or row_scale");
  for (int64_t w : m->d.h_sum_w)
    if (w > kMaxRowWidth)
      return set_error(VBSR_INVALID_ARGUMENT,
                       "a block row of 131072 columns or more could overflow the 32-bit sum");
  auto* p = new (std::nothrow) vbsr_int8;
  if (p == nullptr) return set_error(VBSR_OUT_OF_MEMORY, "host allocation failed");
  p->device = m->d.device;
  p->M = m->d.M;
  p->K = m->d.K;
  p->nvalues = m->d.nvalues;
  DeviceGuard guard(p->device);
  vbsr_status st;
  try {
    st = build_int8(p, m->d, values, row_scale);
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

vbsr_status vbsr_int8_set_values(vbsr_int8* p, const int8_t* values, const float* row_scale,
                                 vbsr_stream_t stream) {
  clear_error();
  if (p == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null plan");
  if (row_scale == nullptr || (values == nullptr && p->nvalues > 0))
    return set_error(VBSR_INVALID_ARGUMENT, "null values or row_scale");
  DeviceGuard guard(p->device);
  return lay_weights(p, values, row_scale, reinterpret_cast<cudaStream_t>(stream));
}

vbsr_status vbsr_int8_workspace_bytes(const vbsr_int8* p, int64_t tokens, int64_t* bytes) {
  clear_error();
  if (p == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null plan");
  if (bytes == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null output");
  if (tokens < 0 || tokens > kMaxTokens)
    return set_error(VBSR_INVALID_ARGUMENT, "tokens must be between 0 and 2^22");
  *bytes = geometry_of(p, tokens).bytes;
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
  if (!p->has_weights) return set_error(VBSR_INVALID_ARGUMENT, "the plan has no weights yet");
  DeviceGuard guard(p->device);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const Geometry g = geometry_of(p, tokens);
  st = launch_chunks<false>(p, g, Q, (reinterpret_cast<uintptr_t>(Q) & 7u) == 0, tokens, ws, s);
  if (st != VBSR_OK) return st;
  return launch_int8(p, g, token_scale, tokens, ws + g.panel_at, C, s);
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
  if (!p->has_weights) return set_error(VBSR_INVALID_ARGUMENT, "the plan has no weights yet");
  DeviceGuard guard(p->device);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const Geometry g = geometry_of(p, tokens);
  const int vec = aligned16(B);
  if (by_clusters(tokens, p->K)) {
    const int64_t rows = g.tiles * g.R;
    token_chunks_kernel<<<unsigned((rows + 1) / 2 * kTokenCtas), kTokenThreads, 0, s>>>(
        B, tokens, rows, p->K, g.R, vec, reinterpret_cast<float*>(ws + g.scale_at), ws + g.panel_at);
    VBSR_CUDA(cudaGetLastError());
    return launch_int8(p, g, reinterpret_cast<const float*>(ws + g.scale_at), tokens, ws + g.panel_at, C, s);
  }
  for (int64_t t0 = 0; t0 < tokens; t0 += 65535) {  // grid limit in y
    const int64_t n = std::min<int64_t>(65535, tokens - t0);
    token_amax_kernel<<<dim3(unsigned(g.splits), unsigned(n)), 256, 0, s>>>(
        B + t0 * p->K, p->K, vec, reinterpret_cast<float*>(ws) + t0 * g.splits);
  }
  VBSR_CUDA(cudaGetLastError());
  st = launch_chunks<true>(p, g, B, vec, tokens, ws, s);
  if (st != VBSR_OK) return st;
  return launch_int8(p, g, reinterpret_cast<const float*>(ws + g.scale_at), tokens, ws + g.panel_at, C, s);
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
  if (m->d.structure_only) return set_error(VBSR_INVALID_ARGUMENT, "the matrix holds its structure only");
  if (row_scale == nullptr || (values == nullptr && m->d.nvalues > 0))
    return set_error(VBSR_INVALID_ARGUMENT, "null values or row_scale");
  DeviceGuard guard(m->d.device);
  quantize_rows_kernel<<<m->d.block_rows, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      view_of(m->d), values, row_scale);
  VBSR_CUDA(cudaGetLastError());
  return VBSR_OK;
}

}  // extern "C"
