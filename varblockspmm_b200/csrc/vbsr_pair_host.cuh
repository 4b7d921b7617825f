// vbsr_pair_host.cuh — host side shared by the operators on pair_kernel: launches, work units.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "vbsr_lm.cuh"
#include "vbsr_pair.cuh"

namespace vbsr_b200 {

inline int ctas_for(int64_t threads, int most) {
  return int(std::max<int64_t>(1, std::min<int64_t>(most, (threads + 255) / 256)));
}

// Fewest parts per row (column) that give half of the SMs a work item. A part streams only its share of the
// weights but all the activations, and as many small copies instead of one per stage: parts for three items
// per SM took 16% longer over 14 drawn shapes (34.1 against 29.4 us, geometric mean), and 37 against 21 us at
// 177 block rows and one token.
inline int parts_for(const int (&units)[4], int64_t tiles, int num_sm) {
  int f = 0;
  while (f < 3 && 2 * units[f] * tiles < int64_t(num_sm)) ++f;
  return f;
}

// Row units for a call, and how a pipeline's memory is cut: two slots (four smaller ones were slower, 32
// tokens 158 against 144 us), and two accumulators where every part has at most 32 rows.
inline void choose_rows(PairParams& k, RowUnit* const (&rows)[4], const int (&units)[4], int64_t tiles,
                        int num_sm, int max_height) {
  const int f = parts_for(units, tiles, num_sm);
  k.rows = rows[f];
  k.units = units[f];
  k.ring_log = 1;
  k.acc_log = f >= 1 || max_height <= 32 ? 1 : 0;
}

// Launches a kernel that itself waits (griddep_wait) for the one before it on the stream: it may be set up
// while that one still runs.
template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

template <int MODE>
vbsr_status launch_pair(PairParams k, int64_t tiles, int num_sm, cudaStream_t s) {
  if (k.units == 0) return VBSR_OK;
  const int64_t most = MODE == kWeightGrad ? tiles : std::max<int64_t>(1, (int64_t(1) << 30) / k.units);
  for (int64_t t0 = 0; t0 < tiles; t0 += most) {
    k.tile0 = int(t0);
    k.tiles = int(std::min(most, tiles - t0));
    const int64_t items = MODE == kWeightGrad ? k.units : int64_t(k.units) * k.tiles;
    VBSR_CUDA(launch_after(pair_kernel<MODE>, dim3(unsigned(std::min<int64_t>(num_sm, items))), kPairThreads,
                           kPairSmem, s, k));
  }
  return VBSR_OK;
}

template <class... P>
int aligned16(const P*... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & 15u) == 0;
}

// Sorted by falling cost, equal ones in their order.
template <class T, class Cost>
std::vector<T> by_cost(const std::vector<T>& v, Cost cost) {
  std::vector<std::pair<uint64_t, uint32_t>> key(v.size());
  for (size_t i = 0; i < v.size(); ++i) key[i] = {~uint64_t(cost(v[i])), uint32_t(i)};
  std::sort(key.begin(), key.end());
  std::vector<T> out;
  out.reserve(v.size());
  for (const auto& k : key) out.push_back(v[k.second]);
  return out;
}

// Whether any call can choose parts finer than those that give `units` (parts_for, with one tile).
inline bool finer_parts(int units, int num_sm) { return 2 * int64_t(units) < num_sm; }

// Units of the block rows (given whole, shape = height), cut into 1, 2, 4 and 8 parts where their height
// allows and as far as calls can choose them, the largest first: the grid strides over them, which evens out
// the SMs' shares. A unit's cost is its weights' bytes and as much as 32 rows' for the activations.
inline void add_row_units(PlanMemory& mem, const std::vector<RowUnit>& whole, int num_sm, RowUnit* (&rows)[4],
                          int (&count)[4]) {
  std::vector<RowUnit> units;
  for (int f = 0; f < 4 && (f == 0 || finer_parts(count[f - 1], num_sm)); ++f) {
    units.clear();
    for (const RowUnit& w : whole) {
      const int h = int(w.shape), hp = std::max(8, (h / 8 + (1 << f) - 1) / (1 << f) * 8);
      for (int r0 = 0; r0 < h; r0 += hp) {
        RowUnit u = w;
        u.row0 += uint32_t(r0);
        u.shape = uint32_t(h) | uint32_t(std::min(hp, h - r0)) << 8 | uint32_t(r0) << 16;
        units.push_back(u);
      }
    }
    mem.table(&rows[f], by_cost(units, [](const RowUnit& u) {
                return uint64_t(u.ng[0] + u.ng[1]) * (32 + ((u.shape >> 8) & 255u));
              }));
    count[f] = int(units.size());
  }
}

}  // namespace vbsr_b200
