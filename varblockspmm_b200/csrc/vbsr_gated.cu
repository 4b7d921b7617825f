// vbsr_gated.cu — the gated feed-forward block: H = act(A_gate B) * (A_up B), and its backward pass.
#include <cuda_runtime.h>

#include <algorithm>
#include <new>
#include <utility>
#include <vector>

#include "vbsr_internal.h"
#include "vbsr_lm.cuh"
#include "vbsr_pair_host.cuh"
#include "vbsr_panels.cuh"

using namespace vbsr_b200;

namespace vbsr_b200 {
// ---- weights -------------------------------------------------------------------------------------

static __global__ void __launch_bounds__(256) values_amax_kernel(const float* a, long long na, const float* b,
                                                          long long nb, float* partial) {
  griddep_launch_dependents();
  // both lengths are multiples of 64
  float m = 0.0f;
  auto scan = [&](const float* v, long long n) {
    const int vec = (reinterpret_cast<uintptr_t>(v) & 15u) == 0;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n / 8; i += gridDim.x * 256ll) {
      float x[8];
      load8(v + 8 * i, vec, x);
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_abs(x[k]));
    }
  };
  scan(a, na);
  scan(b, nb);
  m = cta_max(m);
  if (threadIdx.x == 0) partial[blockIdx.x] = m;
}

// A block row of a packed array in pairs; `row_val` is its first value, `groups` its 8-column groups.
// DEVICE: from the engine's device format (vbsr_tiles.h), else from the packed reference layout; a row
// is a sequence of groups of 8 h values in both.
template <bool DEVICE>
__device__ __forceinline__ void pack_row(const float* values, long long row_val, int h, long long groups,
                                         float s, char* out) {
  for (long long i = threadIdx.x; i < groups * h; i += blockDim.x) {
    const long long g = i / h;
    const int r = int(i % h);
    const float* src = values + row_val + g * 8 * h;
    float v[8];
#pragma unroll
    for (int c = 0; c < 8; ++c)
      v[c] = DEVICE ? src[r * 8 + (((c >> 2) ^ ((r >> 2) & 1)) * 4) + (c & 3)] : src[(long long)c * h + r];
    uint4 hi, lo;
    to_pair8(v, s, hi, lo);
    char* o = out + 4 * row_val + g * 32 * h + 16 * r;
    *reinterpret_cast<uint4*>(o) = hi;
    *reinterpret_cast<uint4*>(o + 16 * h) = lo;
  }
}
struct PackRow {
  uint64_t val;     // first value, in the array of its matrix
  uint32_t groups;  // 8-column groups
  uint32_t h_which; // h | which << 8
};
template <bool DEVICE>
__global__ void __launch_bounds__(256) pack_kernel(const PackRow* rows, const float* gate, const float* up,
                                                   long long up_byte, const float* partial, int count,
                                                   char* out, int* exponent) {
  griddep_launch_dependents();
  griddep_wait();
  const int e = partial_exponent(partial, count);
  if (blockIdx.x == 0 && threadIdx.x == 0) *exponent = e;
  const PackRow r = rows[blockIdx.x];
  const int which = int(r.h_which >> 8);
  pack_row<DEVICE>(which ? up : gate, (long long)r.val, int(r.h_which & 255u), r.groups, pow2(e),
                   out + (which ? up_byte : 0));
}
}  // namespace vbsr_b200

struct vbsr_gated {
  int device = 0, act = 0, num_sm = 148;
  int64_t M = 0, K = 0, gate_values = 0, up_values = 0;
  bool has_weights = false;
  char* w = nullptr;      // both weights in pairs
  int64_t up_byte = 0;    // where up's begin
  int* w_exp = nullptr;   // their exponent
  float* w_partial = nullptr;
  uint32_t* group_col = nullptr;
  PackRow* pack = nullptr;
  int pack_rows = 0;
  // work units with every block row (column) whole, and cut into 2, 4 and 8 parts, as far as calls choose them
  RowUnit* rows[4] = {};
  int row_units[4] = {};
  int max_height = 64;
  ColUnit* cols[4] = {};
  int col_units[4] = {};
  ColEntry* entries = nullptr;
  GradUnit* grads = nullptr;
  int grad_units = 0;
  int* d_status = nullptr;
  char* memory = nullptr;  // of all the above
};

namespace {

// Geometry of a call's panels.
struct Panels {
  int R = 0;        // tokens per tile
  int x_rows = 0;   // tokens per tile of the activations: R, or R / 2 (what a weight-gradient stage takes)
  int64_t tiles = 0;
  int x_splits = 0, dy_splits = 0;  // parts of a token for its largest magnitude
  int64_t dy_partial_at = 0, token_at = 0, stage_at = 0, x_at = 0, dy_at = 0, bytes = 0;
};

// Parts of at least 64 groups, and no more of all tokens than the warps of one grid.
int splits_of(int64_t features, int64_t tokens) {
  const int64_t most = std::min<int64_t>(64, features / 8 / 64);
  return int(std::max<int64_t>(1, std::min<int64_t>(most, 8 * kAmaxCtas / tokens)));
}

constexpr int64_t kPartialBytes = 4 * kAmaxCtas + (256 - 4 * kAmaxCtas % 256) % 256;

// Tiles of at most 128 tokens, evenly sized. In the forward direction any number goes: an MMA's rows behind
// the last token hold other bytes, and a row's result depends on that row alone. In the backward direction
// tokens are summed over, in stages of at most kGradTokens, a multiple of 16 (K = 16): a tile is one or two
// stages.
Panels panels_of(const vbsr_gated* p, int64_t tokens, bool backward) {
  Panels g;
  if (tokens == 0) return g;
  g.tiles = (tokens + 127) / 128;
  if (backward) {
    const int64_t stages = tokens <= kGradTokens ? 1 : 2 * g.tiles;
    g.x_rows = int(((tokens + stages - 1) / stages + 15) / 16 * 16);
    g.R = int(stages / g.tiles) * g.x_rows;
    g.tiles = (tokens + g.R - 1) / g.R;
  } else {
    g.R = g.x_rows = int((tokens + g.tiles - 1) / g.tiles);
  }
  g.x_splits = splits_of(p->K, tokens);
  g.dy_splits = splits_of(p->M, tokens);
  g.dy_partial_at = align256(4 * tokens * g.x_splits);
  g.token_at = g.dy_partial_at + (backward ? align256(4 * tokens * g.dy_splits) : 0);  // the tokens' factors
  g.stage_at = g.token_at + align256(4 * tokens);                                      // the stages'
  g.x_at = g.stage_at + (backward ? align256(4 * g.tiles * (g.R / g.x_rows)) : 0);
  g.dy_at = g.x_at + align256(g.tiles * g.R * (p->K / 8) * 32);
  g.bytes = backward ? g.dy_at + align256(g.tiles * g.R * (p->M / 4) * 32) : g.dy_at;
  return g;
}

PairParams params_of(const vbsr_gated* p, const Panels& g, int64_t tokens, char* ws) {
  PairParams k{};
  k.entries = p->entries;
  k.group_col = p->group_col;
  k.R = g.R;
  k.x_rows = g.x_rows;
  k.act = p->act;
  k.tokens = tokens;
  k.M = p->M;
  k.K = p->K;
  k.x = ws + g.x_at;
  k.dy = ws + g.dy_at;
  k.w = p->w;
  k.token_factor = reinterpret_cast<const float*>(ws + g.token_at);
  k.stage_factor = reinterpret_cast<const float*>(ws + g.stage_at);
  k.status = p->d_status;
  return k;
}

// The job of one panel. which: 0 the activations, 1 the gradients, 2 the activations of the backward pass.
template <class Source>
PanelJob<Source> job_of(const vbsr_gated* p, const Source& src, const Panels& g, int64_t tokens, char* ws,
                        int which) {
  const bool dy = which == 1;
  PanelJob<Source> j{src};
  j.R = dy ? g.R : g.x_rows;
  j.tiles = int(dy ? g.tiles : g.tiles * (g.R / g.x_rows));
  j.splits = dy ? g.dy_splits : g.x_splits;
  j.amax_ctas = ctas_for(32 * tokens * j.splits, kAmaxCtas);
  j.pair_ctas = ctas_for(src.features / 8 * g.tiles * g.R * Source::parts / 4, 148 * 7);
  j.partial = reinterpret_cast<float*>(ws + (dy ? g.dy_partial_at : 0));
  j.w_exp = p->w_exp;
  j.factor = reinterpret_cast<float*>(ws + (which == 2 ? g.stage_at : g.token_at));
  j.out = reinterpret_cast<uint4*>(ws + (dy ? g.dy_at : g.x_at));
  if (which == 2) {
    j.dy_partial = reinterpret_cast<const float*>(ws + g.dy_partial_at);
    j.dy_splits = g.dy_splits;
  }
  return j;
}

// Makes one panel, or two (`both`; the second may be summed over with the first).
template <class A, class C>
vbsr_status make_panels(const PanelJob<A>& a, const PanelJob<C>& c, bool both, int64_t tokens, cudaStream_t s) {
  auto small = [&](int64_t features, int parts) { return features / 8 * tokens * parts <= kSmallGroups; };
  if (tokens <= kSmallTokens && small(a.src.features, A::parts) && (!both || small(c.src.features, C::parts))) {
    panel_small_kernel<<<both ? 2 * kSmallCtas : kSmallCtas, kSmallThreads, 0, s>>>(a, c, int(tokens));
    VBSR_CUDA(cudaGetLastError());
    return VBSR_OK;
  }
  panel_amax_kernel<<<a.amax_ctas + (both ? c.amax_ctas : 0), 256, 0, s>>>(a, c, tokens);
  VBSR_CUDA(cudaGetLastError());
  VBSR_CUDA(launch_after(panel_pair_kernel<A, C>, dim3(unsigned(a.pair_ctas + (both ? c.pair_ctas : 0))), 256, 0, s,
                         a, c, tokens));
  return VBSR_OK;
}

template <bool DEVICE>
vbsr_status pack_weights(vbsr_gated* p, const float* gate, const float* up, cudaStream_t s) {
  const int64_t ng = p->gate_values, nu = p->up_values;
  const int n = ctas_for((ng + nu) / 8, kAmaxCtas);
  values_amax_kernel<<<n, 256, 0, s>>>(gate, ng, up, nu, p->w_partial);
  VBSR_CUDA(cudaGetLastError());
  VBSR_CUDA(launch_after(pack_kernel<DEVICE>, dim3(unsigned(p->pack_rows)), 256, 0, s, p->pack, gate, up,
                         p->up_byte, p->w_partial, n, p->w, p->w_exp));
  return VBSR_OK;
}

vbsr_status build_gated(vbsr_gated* p, const MatrixData& gate, const MatrixData& up) {
  const MatrixData* m[2] = {&gate, &up};
  const int R = m[0]->block_rows, S = m[0]->block_cols;
  p->max_height = *std::max_element(gate.h_row_size.begin(), gate.h_row_size.end());
  VBSR_CUDA(cudaDeviceGetAttribute(&p->num_sm, cudaDevAttrMultiProcessorCount, p->device));
  for (const void* k : {reinterpret_cast<const void*>(pair_kernel<kForward>),
                        reinterpret_cast<const void*>(pair_kernel<kInputGrad>),
                        reinterpret_cast<const void*>(pair_kernel<kWeightGrad>)})
    VBSR_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   kPairSmem));
  p->up_byte = align256(4 * m[0]->nvalues);

  // group lists, block rows of both matrices
  std::vector<uint32_t> group_col;
  std::vector<uint32_t> g0[2], ng[2];
  std::vector<PackRow> pack;
  int64_t columns = 0;
  for (const MatrixData* d : m)
    for (const int64_t w : d->h_sum_w) columns += w;
  group_col.reserve(size_t(columns / 8));
  pack.reserve(size_t(2 * R));
  for (int which = 0; which < 2; ++which) {
    const MatrixData& d = *m[which];
    for (int i = 0; i < R; ++i) {
      g0[which].push_back(uint32_t(group_col.size()));
      for (int b = d.h_row_ptr[i]; b < d.h_row_ptr[i + 1]; ++b) {
        const uint32_t col8 = d.h_blk_desc[b] >> 3, n = (d.h_blk_desc[b] & 7u) + 1u;
        for (uint32_t c = 0; c < n; ++c) group_col.push_back(col8 + c);
      }
      ng[which].push_back(uint32_t(group_col.size()) - g0[which].back());
      if (ng[which][i] >= (1u << 27))
        return set_error(VBSR_INVALID_ARGUMENT, "a block row is too long for the plan's index range");
      if (ng[which][i] > 0)
        pack.push_back({uint64_t(d.h_val_off_row[i]), ng[which][i],
                        uint32_t(d.h_row_size[i]) | uint32_t(which) << 8});
    }
  }
  if (group_col.size() >= (size_t(1) << 31))
    return set_error(VBSR_INVALID_ARGUMENT, "matrices exceed the plan's index range");
  PlanMemory mem;
  const size_t all_groups = group_col.size();
  mem.table(&p->group_col, std::move(group_col));
  p->pack_rows = int(std::max<size_t>(1, pack.size()));
  if (pack.empty()) pack.push_back({0, 0, 8});
  mem.table(&p->pack, std::move(pack));

  std::vector<RowUnit> whole_rows(R);
  for (int i = 0; i < R; ++i) {
    whole_rows[i].row0 = uint32_t(m[0]->h_row_off[i]);
    whole_rows[i].shape = uint32_t(m[0]->h_row_size[i]);
    for (int which = 0; which < 2; ++which) {
      whole_rows[i].g0[which] = g0[which][i];
      whole_rows[i].ng[which] = ng[which][i];
      whole_rows[i].w0[which] = uint64_t(4 * m[which]->h_val_off_row[i] + (which ? p->up_byte : 0));
    }
  }
  add_row_units(mem, whole_rows, p->num_sm, p->rows, p->row_units);

  // blocks by block column, gate then up, in stages of at most 64 rows: counted, then written
  std::vector<ColUnit> whole(S);
  std::vector<int64_t> col_rows(S, 0);
  std::vector<ColEntry> entries;
  struct Fill {
    uint32_t stages = 0, entries = 0, groups = 0;  // entries and groups of the last stage
  };
  for (const bool write : {false, true}) {
    std::vector<Fill> fill(S);
    for (int which = 0; which < 2; ++which) {
      const MatrixData& d = *m[which];
      for (int i = 0; i < R; ++i) {
        const uint32_t h = uint32_t(d.h_row_size[i]);
        int64_t val = d.h_val_off_row[i];
        for (int b = d.h_row_ptr[i]; b < d.h_row_ptr[i + 1]; ++b) {
          const int c = d.h_block_col[b];
          Fill& f = fill[c];
          if (f.stages == 0 || f.entries == kColEntries || f.groups + h / 8 > 8) f = {f.stages + 1, 0, 0};
          if (write)
            entries[size_t(whole[c].s0 + f.stages - 1) * kColEntries + f.entries] = {
                uint32_t((which ? p->M / 8 : 0) + d.h_row_off[i] / 8), h / 8,
                uint64_t(4 * val + (which ? p->up_byte : 0))};
          else
            col_rows[c] += h;
          ++f.entries;
          f.groups += h / 8;
          val += int64_t(h) * d.h_col_size[c];
        }
      }
    }
    if (write) break;
    uint32_t col0 = 0, stages = 0;
    for (int c = 0; c < S; ++c) {
      whole[c] = ColUnit{col0, uint32_t(m[0]->h_col_size[c]), stages, fill[c].stages, 0, {}};
      col0 += whole[c].w;
      stages += whole[c].ns;
    }
    entries.resize(size_t(stages) * kColEntries);
  }
  mem.table(&p->entries, std::move(entries));
  std::vector<std::pair<int64_t, ColUnit>> cols;  // with the rows that it sums over
  for (int f = 0; f < 4 && (f == 0 || finer_parts(p->col_units[f - 1], p->num_sm)); ++f) {
    cols.clear();
    for (int c = 0; c < S; ++c) {
      const int w = int(whole[c].w), wp = std::max(8, (w / 8 + (1 << f) - 1) / (1 << f) * 8);
      for (int c0 = 0; c0 < w; c0 += wp) {
        ColUnit u = whole[c];
        u.c0 = uint32_t(c0);
        u.col0 += u.c0;
        u.w = uint32_t(std::min(wp, w - c0));
        cols.push_back({col_rows[c], u});
      }
    }
    std::vector<ColUnit> sorted;
    sorted.reserve(cols.size());
    for (const auto& c : by_cost(cols, [](const auto& x) { return x.first * (32 + int64_t(x.second.w)); }))
      sorted.push_back(c.second);
    p->col_units[f] = int(sorted.size());
    mem.table(&p->cols[f], std::move(sorted));
  }

  // weight gradients: 16 groups (128 columns) of a block row at a time, the largest first
  std::vector<GradUnit> grads;
  grads.reserve(all_groups / 16 + 2 * size_t(R));
  for (int which = 0; which < 2; ++which)
    for (int i = 0; i < R; ++i)
      for (uint32_t g = 0; g < ng[which][i]; g += 16) {
        const int h = m[which]->h_row_size[i];
        grads.push_back({g0[which][i] + g, std::min(16u, ng[which][i] - g),
                         uint32_t((which ? p->M / 8 : 0) + m[which]->h_row_off[i] / 8), uint32_t(h),
                         uint64_t(m[which]->h_val_off_row[i] + int64_t(g) * 8 * h), uint32_t(which), 0});
      }
  mem.table(&p->grads, by_cost(grads, [](const GradUnit& u) { return (32 + u.h) * (8 + u.ng); }));
  p->grad_units = int(grads.size());

  mem.table(&p->d_status, std::vector<int>(kStatusWords));
  mem.room(&p->w, p->up_byte + 4 * up.nvalues);
  mem.room(&p->w_exp, sizeof(int));
  mem.room(&p->w_partial, kPartialBytes);
  SetupStream s;  // after `mem`: it waits before that goes
  VBSR_CUDA(s.init());
  VBSR_CUDA(mem.make(&p->memory, s.s));
  if ((!gate.structure_only && !up.structure_only) || gate.nvalues + up.nvalues == 0) {
    const vbsr_status st = pack_weights<true>(p, gate.d_values, up.d_values, s.s);
    if (st != VBSR_OK) return st;
    p->has_weights = true;
  }
  VBSR_CUDA(s.finish());
  return VBSR_OK;
}

void free_gated(vbsr_gated* p) {
  if (p == nullptr) return;
  DeviceGuard guard(p->device);
  cudaFree(p->memory);
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
  p->gate_values = g.nvalues;
  p->up_values = u.nvalues;
  p->device = g.device;
  p->act = activation;
  p->M = g.M;
  p->K = g.K;
  DeviceGuard guard(p->device);
  vbsr_status st;
  try {
    st = build_gated(p, g, u);
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
  if ((gate_values == nullptr && p->gate_values > 0) || (up_values == nullptr && p->up_values > 0))
    return set_error(VBSR_INVALID_ARGUMENT, "null values");
  DeviceGuard guard(p->device);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const vbsr_status st = pack_weights<false>(p, gate_values, up_values, s);
  p->has_weights |= st == VBSR_OK;
  return st;
}

vbsr_status vbsr_gated_workspace_bytes(const vbsr_gated* p, int64_t tokens, int backward,
                                       int64_t* bytes) {
  clear_error();
  if (p == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null plan");
  if (bytes == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "null output");
  if (tokens < 0 || tokens > kMaxTokens)
    return set_error(VBSR_INVALID_ARGUMENT, "tokens must be between 0 and 2^22");
  *bytes = std::max(panels_of(p, tokens, false).bytes, backward ? panels_of(p, tokens, true).bytes : 0);
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
  if (!p->has_weights) return set_error(VBSR_INVALID_ARGUMENT, "the plan has no weights yet");
  DeviceGuard guard(p->device);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const Panels g = panels_of(p, tokens, false);
  const auto x = job_of(p, PlainSource{B, p->K, aligned16(B)}, g, tokens, ws, 0);
  const vbsr_status st2 = make_panels(x, x, false, tokens, s);
  if (st2 != VBSR_OK) return st2;
  PairParams k = params_of(p, g, tokens, ws);
  k.out0 = H;
  k.out1 = G;
  k.out2 = U;
  k.vec = aligned16(H, G, U);
  choose_rows(k, p->rows, p->row_units, g.tiles, p->num_sm, p->max_height);
  return launch_pair<kForward>(k, g.tiles, p->num_sm, s);
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
  if (tokens > 0 && dgate == nullptr && dB == nullptr) return set_error(VBSR_INVALID_ARGUMENT, "no output");
  if (tokens > 0 && (B == nullptr || G == nullptr || U == nullptr || dH == nullptr))
    return set_error(VBSR_INVALID_ARGUMENT, "null B, G, U or dH");
  DeviceGuard guard(p->device);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (tokens == 0) {
    if (dgate != nullptr) {
      VBSR_CUDA(cudaMemsetAsync(dgate, 0, 4 * p->gate_values, s));
      VBSR_CUDA(cudaMemsetAsync(dup, 0, 4 * p->up_values, s));
    }
    return VBSR_OK;
  }
  if (!p->has_weights) return set_error(VBSR_INVALID_ARGUMENT, "the plan has no weights yet");
  char* ws = static_cast<char*>(workspace);
  const Panels n = panels_of(p, tokens, true);
  const auto dy = job_of(p, GateSource{G, U, dH, p->M, aligned16(G, U, dH), p->act}, n, tokens, ws, 1);
  const auto x = job_of(p, PlainSource{B, p->K, aligned16(B)}, n, tokens, ws, 2);
  vbsr_status st2 = make_panels(dy, x, dgate != nullptr, tokens, s);
  if (st2 != VBSR_OK) return st2;
  PairParams k = params_of(p, n, tokens, ws);
  if (dB != nullptr) {
    const int f = parts_for(p->col_units, n.tiles, p->num_sm);
    k.cols = p->cols[f];
    k.units = p->col_units[f];
    k.out0 = dB;
    k.vec = aligned16(dB);
    st2 = launch_pair<kInputGrad>(k, n.tiles, p->num_sm, s);
    if (st2 != VBSR_OK) return st2;
    k.beside = 1;  // the weight gradients need the panels only, which are complete
  }
  if (dgate != nullptr) {
    k.grads = p->grads;
    k.units = p->grad_units;
    k.out0 = dgate;
    k.out1 = dup;
    k.vec = aligned16(dgate, dup);
    return launch_pair<kWeightGrad>(k, n.tiles, p->num_sm, s);
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
