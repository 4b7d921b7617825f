// vbsr_pair.cuh — the tensor-core engine of the block-sparse layer operators (tcgen05, TMEM).
//
// FP32 accuracy from 16-bit tensor-core products. Every fp32 operand x is held as a pair of fp16
// numbers: with a power of two 2^e that brings the largest magnitude (of the weights, or of a token's
// activations or gradients) into [2^14, 2^15),
//   hi = fp16(x 2^e),  lo = fp16((x 2^e - hi) 2^11),   x 2^e = hi + lo 2^-11 (1 + d), |d| <= 2^-11,
// so the pair holds x to 2^-23 of itself (fp32 itself: 2^-24) for every |x| within 2^-27 of the
// largest, and to 2^-50 of the largest below that. The factor 2^11 keeps lo out of fp16's
// subnormals. A token has its own e because the tokens of a call may differ by any factor (padded places,
// outliers); where tokens are summed over, see PanelJob (vbsr_panels.cuh). A product of two operands is
// hi hi + 2^-11 (hi lo + lo hi); lo lo is below 2^-22 of it and left out. The two sums go to accumulators of their own (fp32, in TMEM) and are joined, and
// the powers of two taken back, in the epilogue. A pair is four bytes, as the fp32 number is: the
// weights are laid out as pairs once (4 bytes per value streamed, no conversion in the kernel), the
// activations by a pre-pass of each call. Against 3xTF32, which this replaces for these operators,
// the lo part needs no forming in shared memory and an MMA has K = 16 instead of 8.
//
// Layout. Everything is in 8 x 8 core matrices (8 rows of 16 bytes, 128 bytes contiguous), the
// unswizzled operand layout: an operand tile is any set of core matrices at one stride along each
// axis, and read "MN-major" the same bytes are the transposed operand. So one layout of the weights
// serves A x and A^T y, and one of the activations serves as K-major operand (products) and as
// MN-major operand (weight gradients, summed over tokens):
//   weights: block row by block row, 8-column group by group, [h rows of hi][h rows of lo'];
//            the group at packed value offset o starts at byte 4 o.
//   panels:  per tile of R tokens (at most 128; a multiple of 16 for the gradients) and 8-feature group,
//            [R tokens of hi][R tokens of lo'], zeros behind the last token.
// Block widths are multiples of 8, so any block is a whole number of groups; K = 16 steps take two
// groups, and an odd last one is paired with a tile of zeros (and, on the weights' side, with itself,
// so that no stale bytes are multiplied).
//
// Accumulation. The tensor core cuts off (does not round) each step's sum: 36 steps of 16 products
// into one accumulator were measured 1.1e-6 off (2-norm), against 2e-7 for fp32 arithmetic, and the
// error grows with the number of steps. So an accumulator takes at most kChunkSteps steps
// and is then added in fp32 registers by the epilogue warps, while the next steps go to another
// accumulator.
//
// The kernel: one persistent CTA per SM with four pipelines, each a producer warp, a ring of slots, an
// MMA warp and its accumulators; they take the accumulation chunks in turn. A producer issues a
// stage's bulk copies into a slot and writes down where its MMA steps begin; the MMA warp only works
// off that. Four, because both halves are latency: fetching a stage's list of places takes as
// long as several stages take to stream, and one warp that issued all MMAs was measured at 400 clocks
// a step where the operands need about 140 (517 tokens: 701 us with one pipeline, 384 us with four).
// Two epilogue groups of four warps, one warp per TMEM quadrant, take every second work item each. Tokens
// are on the M side (64 or 128 rows): with weights there, blocks of 8 to 56 rows would leave most of an
// MMA empty. What bounds it: the copies into shared memory. A weight group of 32 h bytes needs 32 R
// bytes of activations, from L2, so few tokens run at the weights' HBM rate and many at the
// L2-to-shared-memory rate, h / 2 operations per byte (517 tokens, 3.5 GB into shared memory: 12.5 TB/s).
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "vbsr_kernels_common.cuh"
#include "vbsr_lm.cuh"

namespace vbsr_b200 {

enum PairMode { kForward = 0, kInputGrad = 1, kWeightGrad = 2, kInt8 = 3 };

// A block row, or rows [r0, r0 + hp) of one (parts keep all SMs busy when there are few rows).
// which: 0 gate, 1 up (kInt8 uses 0 only).
struct alignas(16) RowUnit {
  uint32_t row0;   // first row of C
  uint32_t shape;  // h | hp << 8 | r0 << 16
  uint32_t ng[2];  // groups (kInt8: 16-column chunks)
  uint32_t g0[2];  // first entry of the group list
  uint64_t w0[2];  // byte of the first group's weights
  uint64_t pad;
};
static_assert(sizeof(RowUnit) == 48, "RowUnit layout");

// A block column, or columns [c0, c0 + w) of one, with its stages of at most kColEntries blocks.
struct alignas(16) ColUnit {
  uint32_t col0, w, s0, ns;  // first column of B, width, first stage, stages
  uint32_t c0, pad[3];
};
struct alignas(16) ColEntry {
  uint32_t dy_group;  // first 8-row group in the gradient panel (up: behind gate's M / 8 groups)
  uint32_t h8;        // h / 8; 0: no entry
  uint64_t w_byte;    // byte of the block's weights
};
constexpr int kColEntries = 8;  // entries of a stage, of 64 rows at most in total

// Up to 16 consecutive groups of a block row of one matrix: 128 columns of its gradient.
struct alignas(16) GradUnit {
  uint32_t g0, ng;       // group list
  uint32_t dy_group, h;  // gradient panel groups, height
  uint64_t out;          // element of the packed output
  uint32_t which, pad;
};

struct PairParams {
  const RowUnit* rows;
  const ColUnit* cols;
  const ColEntry* entries;
  const GradUnit* grads;
  const uint32_t* group_col;  // per group: scalar column / 8
  int units, tiles, tile0;    // work items are units x tiles from tile0 on (kWeightGrad: units)
  int R, act;
  int x_rows;                 // kWeightGrad: tokens per tile of x, R or R / 2, and per stage
  int beside;                 // kWeightGrad: may run beside the launch before it (kInputGrad)
  int ring_log, acc_log;      // slots and accumulators per pipeline
  long long tokens, M, K;
  const char* x;              // activation panel in pairs (kInt8: in 16-column chunks), K / 8 a tile
  const char* dy;             // gradient panel in pairs
  const char* w;              // weights in pairs (kInt8: int8 chunks)
  // take back the powers of two of x or dy and the weights, per token; kWeightGrad: of x and dy, per stage
  const float *token_factor, *stage_factor;
  const float* row_scale;     // kInt8
  const float* token_scale;
  float *out0, *out1, *out2;  // kForward: H, G, U; kInputGrad: dB; kWeightGrad: dgate, dup; kInt8: C
  int vec;                    // outputs are 16-byte aligned
  int* status;
};

// One K step: two MMAs (kInt8: one; gradients: three). a and b are shared-memory descriptors; a flag is in
// the unused top bits of a.
struct PairStep {
  u64 a, b;
};
constexpr u64 kStepOdd = 1ull << 58;    // the second K half of A is the tile of zeros
constexpr u64 kStepMask = (1ull << 56) - 1;
constexpr int kMaxSteps = 16;

// Slot header: steps | N/8 << 8 | flags. No steps: end of the work. First, last stage of an accumulation
// chunk; odd: the last step has one group (kForward, kInt8).
constexpr uint32_t kHdrFirst = 1u << 16, kHdrLast = 1u << 17, kHdrOdd = 1u << 18;
constexpr uint32_t kHdrGroup = 1u << 19;  // the item's epilogue group

__host__ __device__ constexpr bool by_rows(int mode) { return mode == kForward || mode == kInt8; }
constexpr int kPipes = 4;  // producer warps 0 .. 3, MMA warps 4 .. 7
// A pipeline's share of shared memory, cut into 2^ring_log slots, and of the 512 TMEM columns, cut into
// 2^acc_log accumulators of 128 or 64 columns (hi sums, then lo sums).
constexpr uint32_t kPipeBytes = 48 * 1024;
constexpr int kMaxSlots = 8, kMaxAccs = 8;
constexpr int kEpilogueWarp = 8, kEpilogueGroups = 2;
constexpr int kPairThreads = 32 * (kEpilogueWarp + 4 * kEpilogueGroups);
// The 128 registers per thread that the kernel is launched with, shared out again over its four
// warpgroups: producers, MMA warps, and two of the epilogue.
constexpr int kProducerRegs = 88, kMmaRegs = 40, kEpilogueRegs = 192;
static_assert(kPairThreads == 512 && kProducerRegs + kMmaRegs + 2 * kEpilogueRegs <= 4 * 128, "registers");
// Against 64 bits (2-norm) and fp32 arithmetic's 1.5e-7 to 3.3e-7, six shapes forward: 8 steps 2.9e-7 to 3.8e-7, 12
// steps 4.3e-7 to 5.1e-7. 12 steps are faster for few tokens: 1 token 142 and 150 us with its weights laid out, 8
// tokens of 256 rows 26.6 and 27.7, 32 tokens 290 and 293; 517 tokens and the training steps are the same within 1%.
constexpr int kChunkSteps = 8;
constexpr int kZeroBytes = 2048;   // 128 rows of 16 bytes
constexpr int kTailBytes = 4096;   // MMAs read up to this far behind a tile's own rows
constexpr int kGradTokens = 64;    // kWeightGrad: tokens per stage, at most
// kForward, kInt8: results pass through shared memory (but see the epilogue), R rows and 2^stage_log columns
// (rows padded by 16 bytes, except rows of 32) of two matrices or one; a buffer for each of the two epilogue
// groups.
constexpr int kScaleAhead = 3, kScaleBytes = 4 * 256;  // kInt8: ring of row scales, behind the rows
constexpr int kStageBytes = 10 * 1024 + 256 + kScaleBytes;
__host__ __device__ constexpr int stage_log(int mode, int R) {
  return (R <= 16 ? 6 : (R <= 32 ? 5 : (R <= 64 ? 4 : 3))) + (mode == kInt8 && R > 16 ? 1 : 0);
}
__host__ __device__ constexpr int stage_ld(int log) { return log == 3 ? 8 : (1 << log) + 4; }
constexpr int kPairSmem = kPipes * kPipeBytes + kZeroBytes + kTailBytes + 2 * kStageBytes + 1024;

__device__ __forceinline__ u64 core_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return u64((addr >> 4) & 0x3FFFu) | (u64((lbo >> 4) & 0x3FFFu) << 16) |
         (u64((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}

// MMAs and commits are issued by the lane with leader != 0; the whole warp runs the code around them, so that
// descriptors stay in uniform registers (issued from a branch of one lane, each operand is first moved there).
__device__ __forceinline__ void tc_mma_f16(uint32_t d, u64 a, u64 b, uint32_t idesc, uint32_t acc,
                                           uint32_t leader) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tc_mma_i8(uint32_t d, u64 a, u64 b, uint32_t idesc, uint32_t acc,
                                          uint32_t leader) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tc_commit_by(uint32_t bar, uint32_t leader) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar),
      "r"(leader)
      : "memory");
}
// A value that is the same in all lanes, as a uniform one.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ u64 uniform(u64 x) {
  return u64(uniform(uint32_t(x))) | u64(uniform(uint32_t(x >> 32))) << 32;
}

// Bulk copy without an L2 hint (bulk_g2s has one).
__device__ __forceinline__ void bulk_g2s_plain(uint32_t dst, const void* src, uint32_t bytes,
                                               uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

// 16 accumulator columns from one or two places, loaded and waited for in one statement (the registers are
// not valid before the wait).
__device__ __forceinline__ void tc_ld16(uint32_t a, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, "
      "%8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]),
        "=f"(v[15])
      : "r"(a)
      : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t a, uint32_t b, float (&v)[16], float (&w)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, "
      "%8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16, %17, %18, %19, %20, %21, %22, %23, "
      "%24, %25, %26, %27, %28, %29, %30, %31}, [%33];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]),
        "=f"(v[15]), "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3]), "=f"(w[4]), "=f"(w[5]), "=f"(w[6]),
        "=f"(w[7]), "=f"(w[8]), "=f"(w[9]), "=f"(w[10]), "=f"(w[11]), "=f"(w[12]), "=f"(w[13]),
        "=f"(w[14]), "=f"(w[15])
      : "r"(a), "r"(b)
      : "memory");
}

// Bounded wait of one thread; false after a timeout (recorded) or another role's abort.
constexpr long long kPairWaitLimit = 4000000000ll;  // SM clocks, about 2 s
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, int* status,
                                         volatile int* abort_flag) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_hint(bar, parity, kWaitHintNs)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kPairWaitLimit) {
      record_status(status, VBSR_TIMEOUT, int(blockIdx.x));
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int* status,
                                          volatile int* abort_flag) {
  return __all_sync(0xffffffffu, wait_one(bar, parity, status, abort_flag)) != 0;
}

// n / d for 0 <= n < 2^27 and 1 <= d <= 32, with m = ceil(2^32 / d) (d = 1: m = 0): n m / 2^32 is off
// by n (m d - 2^32) / 2^32 < 1 / d.
__device__ __forceinline__ uint32_t div_magic(uint32_t d) {
  return d == 1 ? 0u : uint32_t((0x100000000ull + d - 1) / d);
}
__device__ __forceinline__ int div_by(int n, uint32_t magic) {
  return magic ? int(__umulhi(uint32_t(n), magic)) : n;
}

// Stages and accumulation chunks of the row units of one height: groups per stage, stages per chunk. An
// integer division takes tens of clocks and every role would do several per work item, so they are
// worked out once per height.
struct RowStages {
  int cap, per_chunk;  // kInt8: one chunk, per_chunk = 0
  uint32_t cap_magic, chunk_magic;
  template <int MODE>
  __device__ __forceinline__ void init(const PairParams& p, int hp) {
    cap = int(kPipeBytes >> p.ring_log) / ((MODE == kInt8 ? 16 : 32) * (p.R + hp));
    const int most = MODE == kInt8 ? 32 : 2 * kChunkSteps;
    cap = (cap < most ? cap : most) & ~1;
    per_chunk = MODE == kInt8 ? 0 : (2 * kChunkSteps) / cap;
    cap_magic = div_magic(cap);
    chunk_magic = MODE == kInt8 ? 0u : div_magic(per_chunk);
  }
  __device__ __forceinline__ int stages(int groups) const { return div_by(groups + cap - 1, cap_magic); }
  __device__ __forceinline__ int chunks(int groups) const {
    if (per_chunk == 0) return groups > 0;
    return div_by(stages(groups) + per_chunk - 1, chunk_magic);
  }
};
// kInputGrad, kWeightGrad: a stage (of at most 8 and 4 steps) is a chunk.

// The units of this CTA's work items, 32 at a time in the lanes' registers and the next 32 on their
// way; get() broadcasts one.
template <class Unit>
struct UnitWin {
  static constexpr int W = sizeof(Unit) / 16;
  uint4 cur[W], next[W];
  const Unit* units;
  int items, tiles, first;
  __device__ __forceinline__ void load(int k, uint4 (&v)[W]) const {
    const long long item = blockIdx.x + (long long)k * gridDim.x;
    if (item < items) {
      const uint4* q = reinterpret_cast<const uint4*>(units + int(item) / tiles);
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = __ldg(q + i);
    }
  }
  __device__ __forceinline__ void init(const Unit* u, int items_, int tiles_, int lane) {
    units = u;
    items = items_;
    tiles = tiles_;
    first = 0;
    load(lane, cur);
    load(32 + lane, next);
  }
  // the CTA's k-th item; k never decreases and grows by at most one
  __device__ __forceinline__ Unit get(int k, int lane) {
    if (k - first == 32) {
      first += 32;
#pragma unroll
      for (int i = 0; i < W; ++i) cur[i] = next[i];
      load(first + 32 + lane, next);
    }
    Unit u;
    uint4* o = reinterpret_cast<uint4*>(&u);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      o[i].x = __shfl_sync(0xffffffffu, cur[i].x, k - first);
      o[i].y = __shfl_sync(0xffffffffu, cur[i].y, k - first);
      o[i].z = __shfl_sync(0xffffffffu, cur[i].z, k - first);
      o[i].w = __shfl_sync(0xffffffffu, cur[i].w, k - first);
    }
    return u;
  }
};

// Token tile of the CTA's items, item = unit x tiles + tile, kept without divisions.
struct TileWalk {
  int tile, step, tiles;
  __device__ __forceinline__ TileWalk(int tiles_)
      : tile(int(blockIdx.x) % tiles_), step(int(gridDim.x) % tiles_), tiles(tiles_) {}
  __device__ __forceinline__ void next() {
    tile += step;
    if (tile >= tiles) tile -= tiles;
  }
};

struct PairBars {
  uint32_t full, empty, acc_full, acc_empty, drain;  // first barrier of each array
};

struct PairShared {
  RowStages stages[8];  // by height / 8 - 1
  u64 full[kMaxSlots], empty[kMaxSlots], acc_full[2 * kMaxAccs], acc_empty[kMaxAccs], drain[kPipes];
  PairStep steps[kMaxSlots][kMaxSteps];
  uint32_t header[kMaxSlots];
  uint32_t tmem;
  volatile int abort_flag;
};

// ---- producers -----------------------------------------------------------------------------------
//
// Pipeline q takes the CTA's accumulation chunks c with c % kPipes == q. A producer fetches its next
// stage's list before it issues the one in hand.

// A pipeline's slots: its stage i is in slot i % ring.
struct Pipe {
  int q, log;
  uint32_t i = 0;
  __device__ __forceinline__ Pipe(const PairParams& p, int q_) : q(q_), log(p.ring_log) {}
  __device__ __forceinline__ uint32_t slot() const {
    return (uint32_t(q) << log) + (i & ((1u << log) - 1u));
  }
  __device__ __forceinline__ uint32_t parity() const { return (i >> log) & 1u; }
  __device__ __forceinline__ uint32_t base(uint32_t slots) const {
    return slots + slot() * (kPipeBytes >> log);
  }
};
__device__ __forceinline__ bool wait_slot(const PairParams& p, PairShared& sh, const PairBars& bars,
                                          const Pipe& pipe) {
  return wait_warp(bars.empty + 8 * pipe.slot(), pipe.parity() ^ 1u, p.status, &sh.abort_flag);
}
// Announces the slot's list and bytes; the lanes' list entries are written before.
__device__ __forceinline__ void announce(PairShared& sh, uint32_t slot, uint32_t full, uint32_t header,
                                         uint32_t bytes, int lane) {
  if (lane == 0) sh.header[slot] = header;
  __syncwarp();
  if (lane == 0) mbar_arrive_expect_tx(full, bytes);
  __syncwarp();
}
// The end marker, a stage without steps.
__device__ __forceinline__ void produce_end(const PairParams& p, PairShared& sh, const PairBars& bars,
                                            const Pipe& pipe, int lane) {
  if (!wait_slot(p, sh, bars, pipe)) return;
  if (lane == 0) {
    sh.header[pipe.slot()] = 0u;
    mbar_arrive(bars.full + 8 * pipe.slot());
  }
}

template <int MODE>
__device__ void produce_rows(const PairParams& p, PairShared& sh, uint32_t slots, uint32_t zero,
                             const PairBars& bars, int warp, int lane) {
  constexpr bool I8 = MODE == kInt8;
  const uint32_t xb = (I8 ? 16u : 32u) * uint32_t(p.R);  // panel bytes of a group
  const uint64_t pol_x = policy_evict_last(), pol_w = policy_evict_first();
  const long long per_tile = p.K >> 3;
  const int items = p.units * p.tiles;
  struct Stage {
    uint32_t shape, flags, col;  // flags: of the header
    int n, tile;
    const char* w;
  };
  Pipe pipe(p, warp);
  auto issue = [&](const Stage& st) {
    if (!wait_slot(p, sh, bars, pipe)) return false;
    const int h = int(st.shape & 255u), hp = int((st.shape >> 8) & 255u), r0 = int(st.shape >> 16);
    const uint32_t wb = (I8 ? 16u : 32u) * uint32_t(hp), n = uint32_t(st.n);
    const uint32_t slot = pipe.slot(), base = pipe.base(slots), full = bars.full + 8 * slot;
    const uint32_t xbase = base + n * wb, steps = (n + 1) / 2;  // weights first: 128-byte aligned
    // the steps are evenly spaced: the list holds the first and, if the number of groups is odd, the last
    if (lane == 0) {
      sh.steps[slot][0] = {core_desc(xbase, xb, 128), core_desc(base, wb, 128)};
      const uint32_t a = xbase + (n - 1) * xb;
      if (n & 1u) sh.steps[slot][1] = {core_desc(a, zero - a, 128), core_desc(base + (n - 1) * wb, 0u, 128)};
    }
    announce(sh, slot, full, steps | uint32_t(hp) << 5 | st.flags | (n & 1u ? kHdrOdd : 0u), n * (xb + wb),
             lane);
    // weights: one run, or per group the part's rows of hi and of lo'
    if (hp == h) {
      if (lane == 0) {
        if (p.tiles == 1)
          bulk_g2s(base, st.w, n * wb, full, pol_w);
        else
          bulk_g2s_plain(base, st.w, n * wb, full);
      }
    } else if (lane < st.n) {
      const char* g = st.w + (long long)lane * (I8 ? 16 : 32) * h + 16 * r0;
      bulk_g2s_plain(base + lane * wb, g, 16u * hp, full);
      if (!I8) bulk_g2s_plain(base + lane * wb + 16u * hp, g + 16 * h, 16u * hp, full);
    }
    if (pipe.i == 0) griddep_wait();
    // activations: one copy per run of neighbouring groups
    const uint32_t before = __shfl_up_sync(0xffffffffu, st.col, 1);
    const bool head = lane < st.n && (lane == 0 || st.col != before + 1);
    const uint32_t heads = __ballot_sync(0xffffffffu, head) | (n < 32 ? 1u << n : 0u);
    if (head) {
      const uint32_t rest = lane < 31 ? heads >> (lane + 1) : 0u;
      const uint32_t run = rest ? uint32_t(__ffs(rest)) : uint32_t(32 - lane);
      bulk_g2s(xbase + lane * xb, p.x + (st.tile * per_tile + st.col) * xb, run * xb, full, pol_x);
    }
    ++pipe.i;
    return true;
  };
  UnitWin<RowUnit> win;
  win.init(p.rows, items, p.tiles, lane);
  Stage held{};
  bool have = false;
  uint32_t c0 = 0;  // chunks before this item
  int k = 0;
  TileWalk walk(p.tiles);
  for (int item = blockIdx.x; item < items; item += gridDim.x, ++k, walk.next()) {
    const RowUnit u = win.get(k, lane);
    const RowStages rs = sh.stages[((u.shape >> 11) & 31u) - 1u];
    const int n0 = rs.chunks(int(u.ng[0])), total = n0 + rs.chunks(int(u.ng[1]));
    for (int ch = int((uint32_t(warp) - c0) % kPipes); ch < total; ch += kPipes) {
      const bool up = ch >= n0;
      const int groups = int(up ? u.ng[1] : u.ng[0]), ns = rs.stages(groups);
      const int j0 = (up ? ch - n0 : ch) * rs.per_chunk, j1 = I8 ? ns : min(ns, j0 + rs.per_chunk);
      for (int j = j0; j < j1; ++j) {
        const int off = j * rs.cap;
        Stage st;
        st.shape = u.shape;
        st.n = min(rs.cap, groups - off);
        st.tile = p.tile0 + walk.tile;
        st.flags = (j == j0 ? kHdrFirst : 0u) | (j + 1 == j1 ? kHdrLast : 0u) | (k & 1 ? kHdrGroup : 0u);
        st.col = lane < st.n ? __ldg(p.group_col + (up ? u.g0[1] : u.g0[0]) + off + lane) : 0u;
        st.w = p.w + (up ? u.w0[1] : u.w0[0]) + (long long)off * (I8 ? 16 : 32) * int(u.shape & 255u);
        if (have && !issue(held)) return;
        held = st;
        have = true;
      }
    }
    c0 += uint32_t(total);
  }
  if (have && !issue(held)) return;
  produce_end(p, sh, bars, pipe, lane);
}

__device__ __forceinline__ void produce_cols(const PairParams& p, PairShared& sh, uint32_t slots,
                                             uint32_t zero, const PairBars& bars, int warp, int lane) {
  const uint32_t xb = 32u * uint32_t(p.R);
  const uint64_t pol_x = policy_evict_last();
  const int items = p.units * p.tiles;
  const long long per_tile = 2 * (p.M >> 3);
  struct Stage {
    uint32_t w, c0, flags;
    int tile;
    ColEntry e;
  };
  Pipe pipe(p, warp);
  auto issue = [&](const Stage& st) {
    const ColEntry& e = st.e;
    // places of the entries: groups before this one, and its steps
    uint32_t g = e.h8, steps = (e.h8 + 1) / 2;
#pragma unroll
    for (int d = 1; d < kColEntries; d *= 2) {
      const uint32_t g2 = __shfl_up_sync(0xffffffffu, g, d), s2 = __shfl_up_sync(0xffffffffu, steps, d);
      if (lane >= d) {
        g += g2;
        steps += s2;
      }
    }
    const uint32_t groups = __shfl_sync(0xffffffffu, g, kColEntries - 1);
    const uint32_t all_steps = __shfl_sync(0xffffffffu, steps, kColEntries - 1);
    const uint32_t g_before = g - e.h8, s_before = steps - (e.h8 + 1) / 2;
    if (!wait_slot(p, sh, bars, pipe)) return false;
    const uint32_t slot = pipe.slot(), base = pipe.base(slots), full = bars.full + 8 * slot;
    const uint32_t a0 = base + g_before * xb, b0 = base + groups * xb + g_before * 32u * st.w;
    const uint32_t h = 8u * e.h8;
    if (lane < kColEntries)
      for (uint32_t j = 0; 2 * j < e.h8; ++j) {
        const bool pair = 2 * j + 1 < e.h8;
        const uint32_t a = a0 + 2 * j * xb;
        PairStep& out = sh.steps[slot][s_before + j];
        out.a = core_desc(a, pair ? xb : zero - a, 128) | (pair ? 0 : kStepOdd);
        // columns 8 apart are 16 h apart (hi and lo' tiles alternate), rows 8 apart 128 bytes
        out.b = core_desc(b0 + 256u * j, pair ? 128u : 0u, 16u * h);
      }
    announce(sh, slot, full, all_steps | st.w << 5 | st.flags, groups * (xb + 32u * st.w), lane);
    if (e.h8) bulk_g2s_plain(b0, p.w + e.w_byte + (long long)(st.c0 >> 3) * 32 * h, 4u * h * st.w, full);
    if (pipe.i == 0) griddep_wait();
    if (e.h8) bulk_g2s(a0, p.dy + (st.tile * per_tile + e.dy_group) * xb, e.h8 * xb, full, pol_x);
    ++pipe.i;
    return true;
  };
  UnitWin<ColUnit> win;
  win.init(p.cols, items, p.tiles, lane);
  Stage held{};
  bool have = false;
  uint32_t c0 = 0;
  int k = 0;
  TileWalk walk(p.tiles);
  for (int item = blockIdx.x; item < items; item += gridDim.x, ++k, walk.next()) {
    const ColUnit u = win.get(k, lane);
    for (uint32_t j = (uint32_t(warp) - c0) % kPipes; j < u.ns; j += kPipes) {
      Stage st;
      st.w = u.w;
      st.c0 = u.c0;
      st.flags = kHdrFirst | kHdrLast | (k & 1 ? kHdrGroup : 0u);
      st.tile = p.tile0 + walk.tile;
      st.e = ColEntry{};
      if (lane < kColEntries) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.entries) +
                              (long long)(u.s0 + j) * kColEntries + lane);
        st.e.dy_group = v.x;
        st.e.h8 = v.y;
        st.e.w_byte = u64(v.z) | u64(v.w) << 32;
      }
      if (have && !issue(held)) return;
      held = st;
      have = true;
    }
    c0 += u.ns;
  }
  if (have && !issue(held)) return;
  produce_end(p, sh, bars, pipe, lane);
}

// Token stages of a weight-gradient unit: x_rows tokens of the unit's 16 activation groups, a copy each, and
// of its h / 8 gradient groups, which are R tokens long, a copy for hi and one for lo'.
__device__ __forceinline__ void produce_grads(const PairParams& p, PairShared& sh, uint32_t slots,
                                              const PairBars& bars, int warp, int lane) {
  const uint32_t nt = uint32_t(p.x_rows), GB = 32u * nt, dyb = 32u * uint32_t(p.R);
  const uint64_t pol_x = policy_evict_last();
  const int per_tile = p.R / p.x_rows, total = p.tiles * per_tile;
  UnitWin<GradUnit> win;
  win.init(p.grads, p.units, 1, lane);
  Pipe pipe(p, warp);
  uint32_t c0 = 0, next_col = 0;
  int k = 0;
  auto load_col = [&](const GradUnit& u) {
    return lane < int(u.ng) ? __ldg(p.group_col + u.g0 + lane) : 0u;
  };
  GradUnit nu{};
  if (int(blockIdx.x) < p.units) {
    nu = win.get(0, lane);
    next_col = load_col(nu);
  }
  uint32_t group = 0;
  for (int item = blockIdx.x; item < p.units; item += gridDim.x, group ^= kHdrGroup) {
    const GradUnit u = nu;
    const uint32_t col = next_col;
    if (item + int(gridDim.x) < p.units) {
      nu = win.get(++k, lane);
      next_col = load_col(nu);
    }
    const uint32_t h8 = u.h / 8;
    const bool is_x = lane < int(u.ng), is_dy = lane >= 16 && lane < 16 + int(h8);
    const char* src0 = is_x ? p.x + (long long)col * GB : p.dy + ((long long)u.dy_group + lane - 16) * dyb;
    for (int j = int((uint32_t(warp) - c0) % kPipes); j < total; j += kPipes, ++pipe.i) {
      if (!wait_slot(p, sh, bars, pipe)) return;
      const uint32_t slot = pipe.slot(), base = pipe.base(slots), full = bars.full + 8 * slot;
      const uint32_t steps = nt / 16;
      if (lane < int(steps)) {
        PairStep& out = sh.steps[slot][lane];
        out.a = core_desc(base + 256u * lane, 128u, GB);
        out.b = core_desc(base + 16u * GB + 256u * lane, 128u, GB / 2);
      }
      announce(sh, slot, full, steps | u.h << 5 | kHdrFirst | kHdrLast | group, (u.ng + h8) * GB, lane);
      const uint32_t dst = base + lane * GB;
      if (is_x) {
        bulk_g2s(dst, src0 + (long long)j * (p.K >> 3) * GB, GB, full, pol_x);
      } else if (is_dy) {
        const char* src = src0 + (long long)(j / per_tile) * 2 * (p.M >> 3) * dyb + 16 * nt * (j % per_tile);
        bulk_g2s(dst, src, GB / 2, full, pol_x);
        bulk_g2s(dst + GB / 2, src + 16 * p.R, GB / 2, full, pol_x);
      }
    }
    c0 += uint32_t(total);
  }
  produce_end(p, sh, bars, pipe, lane);
}

// Accumulator of a pipeline's chunk, and the TMEM columns of one.
__device__ __forceinline__ uint32_t acc_of(const PairParams& p, uint32_t q, uint32_t chunk) {
  return q + kPipes * (chunk & ((1u << p.acc_log) - 1u));
}
__device__ __forceinline__ uint32_t acc_cols(const PairParams& p) { return 128u >> p.acc_log; }

// ---- MMA warps -----------------------------------------------------------------------------------

template <int MODE>
__device__ void issue_mmas(const PairParams& p, PairShared& sh, const PairBars& bars, int q_, int lane) {
  const uint32_t q = uniform(uint32_t(q_)), leader = lane == 0;
  const int m = MODE == kWeightGrad ? 128 : (p.R > 64 ? 128 : 64);
  // D f32, A and B f16 (kInt8: D s32, A and B s8); transposed (MN-major) operands in bits 15 and 16
  const uint32_t form = (MODE == kInt8 ? (2u << 4) | (1u << 7) | (1u << 10) : (1u << 4)) |
                        (MODE == kWeightGrad ? 1u << 15 : 0u) |
                        (MODE == kWeightGrad || MODE == kInputGrad ? 1u << 16 : 0u) |
                        (uint32_t(m >> 4) << 24);
  const uint32_t xb16 = (MODE == kInt8 ? 1u : 2u) * uint32_t(p.R);  // panel group, in 16 bytes
  const u64 lo = MODE == kWeightGrad ? u64(p.x_rows) : u64(p.R);  // hi to lo' tile of A, in 16 bytes
  const uint32_t tmem = uniform(sh.tmem);
  Pipe pipe(p, int(q));
  uint32_t chunk = 0;  // of this pipeline: accumulator q + kPipes (chunk % accumulators)
  for (;; ++pipe.i) {
    const uint32_t slot = pipe.slot();
    if (!wait_warp(bars.full + 8 * slot, pipe.parity(), p.status, &sh.abort_flag)) return;
    const uint32_t hdr = uniform(*reinterpret_cast<volatile uint32_t*>(&sh.header[slot]));
    const int steps = int(hdr & 63u), n = int((hdr >> 8) & 15u) * 8;
    if (steps == 0) break;
    // the list, one step to a lane
    const PairStep list = sh.steps[slot][lane & (kMaxSteps - 1)];
    const u64 a0 = uniform(list.a), b0 = uniform(list.b);
    const uint32_t acc_no = acc_of(p, q, chunk), d = tmem + acc_no * acc_cols(p);
    if (hdr & kHdrFirst)
      if (!wait_warp(bars.acc_empty + 8 * acc_no, ((chunk >> p.acc_log) & 1u) ^ 1u, p.status, &sh.abort_flag))
        return;
    tc_fence_after();
    // N of one tile of n columns: a multiple of 16 for M = 128 (one tile more is read, and its
    // columns are not used)
    const int n1 = m == 128 || MODE == kInt8 ? (n + 15) & ~15 : n;
    const uint32_t i1 = form | (uint32_t(n1 >> 3) << 17);
    [[maybe_unused]] const uint32_t i2 = form | (uint32_t(2 * n >> 3) << 17);
    uint32_t acc = (hdr & kHdrFirst) ? 0u : 1u;
    if constexpr (MODE == kForward || MODE == kInt8) {
      const u64 da = 2u * xb16, db = (MODE == kInt8 ? 2u : 4u) * uint32_t(n);  // two groups, in 16 bytes
      const int even = steps - ((hdr & kHdrOdd) ? 1 : 0);
      u64 a = a0, b = b0;
      auto step = [&](u64 a1, u64 a2, u64 b1) {
        if (MODE == kInt8) {
          tc_mma_i8(d, a1, b1, i1, acc, leader);
        } else {  // hi x [hi; lo'], then lo' x hi into the columns of hi lo'
          tc_mma_f16(d, a1, b1, i2, acc, leader);
          tc_mma_f16(d + n, a2, b1, i1, 1u, leader);
        }
        acc = 1u;
      };
      for (int s = 0; s < even; ++s, a += da, b += db) step(a, a + lo, b);
      if (hdr & kHdrOdd) {  // the second K half of A is the tile of zeros, which has no lo' tile behind it
        const PairStep last = sh.steps[slot][1];
        const u64 a1 = uniform(last.a);
        step(a1, a1 + lo - (lo << 16), uniform(last.b));
      }
    } else {
      auto step = [&](u64 a, u64 a2, u64 b) {  // B's hi and lo' tiles alternate: every second one
        const u64 sbo = (b >> 32) & 0x3FFFull, bh = b + (sbo << 32);
        tc_mma_f16(d, a, bh, i1, acc, leader);
        tc_mma_f16(d + 64u, a, bh + sbo, i1, acc, leader);
        tc_mma_f16(d + 64u, a2, bh, i1, 1u, leader);
        acc = 1u;
      };
      if constexpr (MODE == kWeightGrad) {  // 16 tokens are two core matrices, 256 bytes, further in both
        u64 a = a0, b = b0;
        for (int s = 0; s < steps; ++s, a += 16, b += 16) step(a, a + lo, b);
      } else {
        for (int s = 0; s < steps; ++s) {
          const uint32_t a_lo = __shfl_sync(0xffffffffu, uint32_t(list.a), s);
          const uint32_t a_hi = __shfl_sync(0xffffffffu, uint32_t(list.a >> 32), s);
          const uint32_t b_lo = __shfl_sync(0xffffffffu, uint32_t(list.b), s);
          const uint32_t b_hi = __shfl_sync(0xffffffffu, uint32_t(list.b >> 32), s);
          const u64 a = (u64(a_hi) << 32 | a_lo) & kStepMask, b = u64(b_hi) << 32 | b_lo;
          step(a, a + lo - ((a_hi & uint32_t(kStepOdd >> 32)) ? lo << 16 : 0ull), b);
        }
      }
    }
    tc_commit_by(bars.empty + 8 * slot, leader);
    if (hdr & kHdrLast) {
      tc_commit_by(bars.acc_full + 8 * (acc_no + ((hdr & kHdrGroup) ? kMaxAccs : 0)), leader);
      ++chunk;
    }
  }
  tc_commit_by(bars.drain + 8 * q, leader);  // nothing may arrive on a barrier of a CTA that has gone
  wait_warp(bars.drain + 8 * q, 0, p.status, &sh.abort_flag);
}

// ---- epilogue ------------------------------------------------------------------------------------

__device__ __forceinline__ void store8(float* dst, const float* v) {
  reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void put8(float* dst, const float* v, int vec) {
  if (vec) {
    store8(dst, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = v[i];
  }
}
__device__ __forceinline__ void store4(float* dst, const float (&v)[4], int vec) {
  if (vec) {
    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = v[i];
  }
}
__device__ __forceinline__ void group_sync(int e) {
  asm volatile("bar.sync %0, 128;" ::"r"(e + 1) : "memory");
}
constexpr float kLoUnit = 1.0f / 2048.0f;  // 2^-11

// Adds a 16-column tile of an accumulation chunk: hi sums at column `hi`, lo sums at `lo` (kInt8: the
// integers at `hi`, carried as they are; kWeightGrad: times the stage's power of two f).
template <int MODE>
__device__ __forceinline__ void add_tile(float (&acc)[16], uint32_t hi, uint32_t lo, float f) {
  if constexpr (MODE == kInt8) {
    tc_ld16(hi, acc);
  } else {
    float v[16], w[16];
    tc_ld16(hi, lo, v, w);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float sum = fmaf(w[i], kLoUnit, v[i]);
      acc[i] = MODE == kWeightGrad ? fmaf(sum, f, acc[i]) : acc[i] + sum;
    }
  }
}

// Output of a row unit's tile from the staged sums: a thread takes four neighbouring elements of a row, so
// that few tokens' activations are shared out too and whole lines are stored. Two rows at a time, because
// an element is a chain of latencies (shared memory, exponential, quotient).
template <int MODE>
__device__ __forceinline__ void write_staged(const PairParams& p, const float* st, const float* st_up, int ld,
                                             int step, int sc, int sr, int rows, long long o, const float* rs,
                                             const float* tokens, const float* factors) {
  // o: place of (row 0, column sc) in the output
  // tokens: the tile's token scales (few, and read again by every unit: they stay in L1)
  auto finish = [&](long long at, float (&v)[4], float (&w)[4], float ts) {
    float hv[4];
    if constexpr (MODE == kForward) {
      with_act(p.act, [&](auto kind) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float a, da;
          act_both<decltype(kind)::value>(v[i], a, da);
          hv[i] = a * w[i];
        }
      });
      if (p.out1 != nullptr) {
        store4(p.out1 + at, v, p.vec);
        store4(p.out2 + at, w, p.vec);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) hv[i] = float(__float_as_int(v[i])) * (ts * rs[i]);
    }
    store4(p.out0 + at, hv, p.vec);
  };
  auto load = [&](int r, float (&v)[4], float (&w)[4]) {
    *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(st + r * ld + sc);
    if constexpr (MODE == kForward) {
      *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(st_up + r * ld + sc);
      const float f = factors[r];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] *= f;
        w[i] *= f;
      }
    }
  };
  const long long hop = step * p.M;
  o += sr * p.M;
  for (int r = sr; r < rows; r += 2 * step, o += 2 * hop) {
    float v[2][4], w[2][4], ts[2] = {};
    const bool two = r + step < rows;
    if constexpr (MODE == kInt8) {
      ts[0] = tokens[r];
      ts[1] = tokens[two ? r + step : r];
    }
    load(r, v[0], w[0]);
    load(two ? r + step : r, v[1], w[1]);
    finish(o, v[0], w[0], ts[0]);
    if (two) finish(o + hop, v[1], w[1], ts[1]);
  }
}

// TMEM quadrants that hold tokens: M = 64 puts 16 rows in a quadrant, M = 128 32.
template <int MODE>
__device__ __forceinline__ int live_quads(const PairParams& p) {
  if (MODE == kWeightGrad) return 4;
  return p.R > 64 ? (p.R + 31) / 32 : (p.R + 15) / 16;
}

// The part of a unit that the epilogue reads, 16 bytes.
template <int MODE>
__device__ __forceinline__ uint4 unit_head(const PairParams& p, int unit) {
  if constexpr (by_rows(MODE)) return __ldg(reinterpret_cast<const uint4*>(p.rows + unit));
  else if constexpr (MODE == kInputGrad) return __ldg(reinterpret_cast<const uint4*>(p.cols + unit));
  else return __ldg(reinterpret_cast<const uint4*>(p.grads + unit));
}

// Epilogue group e (four warps, one per TMEM quadrant) takes every second of the CTA's work items, so that
// one item's sums are added while the other's output is worked out.
template <int MODE>
__device__ void epilogue(const PairParams& p, PairShared& sh, const PairBars& bars, float* stage, int quad,
                         int e, int lane) {
  const bool wide = MODE == kWeightGrad || p.R > 64;  // M = 128; M = 64 fills lanes 0..15
  const int row = wide ? 32 * quad + lane : 16 * quad + lane;
  const bool in_tile = (wide || lane < 16) && (MODE == kWeightGrad || row < p.R);
  const int tiles = MODE == kWeightGrad ? 1 : p.tiles, items = p.units * tiles, grid = int(gridDim.x);
  if (MODE != kWeightGrad || !p.beside) griddep_wait();
  if (MODE == kInputGrad) griddep_launch_dependents();
  constexpr bool per_token = MODE == kForward || MODE == kInputGrad;
  float stage_factor = 0.0f;  // kWeightGrad: of 32 stages, one to a lane
  const int quads = live_quads<MODE>(p);
  const int thread = 32 * quad + lane, slog = stage_log(MODE, p.R), ld = stage_ld(slog), log4 = slog - 2;
  const int sc = 4 * (thread & ((1 << log4) - 1)), sr = thread >> log4;  // staged output: column, first row
  uint32_t use = 0, phases = 0;  // chunks of the CTA so far; parity of this group's phase per accumulator
  bool ok = true;
  // the units of the next 32 items in the lanes' registers, and the 32 after them on their way
  TileWalk walk(tiles);
  uint4 heads, heads2;
  int head0 = 0;
  auto fetch = [&](int k) {
    const long long item = blockIdx.x + (long long)(k + lane) * grid;
    return item < items ? unit_head<MODE>(p, int(item) / tiles) : make_uint4(0, 0, 0, 0);
  };
  heads = fetch(0);
  heads2 = fetch(32);
  // kInt8: row scales come through a ring in shared memory, kScaleAhead of the group's items ahead: a load of
  // the epilogue waits behind the bulk copies in flight, longer than a small item takes
  float* row_scales = stage + (kStageBytes - kScaleBytes) / 4;
  // kForward, kInputGrad: the same place holds the factors of the tile's tokens, two tiles in turn
  float* token_factors = row_scales;
  auto fetch_scales = [&](int k) {  // of the CTA's item k
    if constexpr (MODE == kInt8) {
      const uint32_t x1 = __shfl_sync(0xffffffffu, heads.x, k & 31), x2 = __shfl_sync(0xffffffffu, heads2.x, k & 31);
      const uint32_t y1 = __shfl_sync(0xffffffffu, heads.y, k & 31), y2 = __shfl_sync(0xffffffffu, heads2.y, k & 31);
      const bool near = k < head0 + 32;
      const int n = int(((near ? y1 : y2) >> 8) & 255u);
      if (quad == 0) {
        if (blockIdx.x + (long long)k * grid < items && 4 * lane < n)
          cp_async16(smem_addr(row_scales + 64 * ((k >> 1) & 3) + 4 * lane), p.row_scale + (near ? x1 : x2) + 4 * lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
    }
  };
  for (int i = 0; i < kScaleAhead; ++i) fetch_scales(e + 2 * i);
  for (int item = blockIdx.x, k = 0; item < items; item += grid, ++k, walk.next()) {
    if (k > 0 && (k & 31) == 0) {
      heads = heads2;
      heads2 = fetch(k + 32);
      head0 = k;
    }
    uint4 u;
    u.x = __shfl_sync(0xffffffffu, heads.x, k & 31);
    u.y = __shfl_sync(0xffffffffu, heads.y, k & 31);
    u.z = __shfl_sync(0xffffffffu, heads.z, k & 31);
    u.w = __shfl_sync(0xffffffffu, heads.w, k & 31);
    int n, chunks[2] = {0, 0};
    if constexpr (by_rows(MODE)) {
      n = int((u.y >> 8) & 255u);
      const RowStages rs = sh.stages[n / 8 - 1];
      chunks[0] = rs.chunks(int(u.z));
      chunks[1] = rs.chunks(int(u.w));
    } else if constexpr (MODE == kInputGrad) {
      n = int(u.y);
      chunks[0] = int(u.w);
    } else {
      n = int(u.w);
      chunks[0] = p.tiles * (p.R / p.x_rows);
    }
    if ((k & 1) != e) {
      use += uint32_t(chunks[0] + chunks[1]);
      continue;
    }
    const long long t0 = (long long)(p.tile0 + walk.tile) * p.R;
    float* factors = token_factors + (tiles > 1 ? 128 * ((k >> 1) & 1) : 0);
    if (per_token && (tiles > 1 || k == e) && in_tile && t0 + row < p.tokens)
      cp_async4(smem_addr(factors + row), p.token_factor + t0 + row);
    uint4 g2 = make_uint4(0, 0, 0, 0);
    if constexpr (MODE == kWeightGrad) g2 = __ldg(reinterpret_cast<const uint4*>(p.grads + item) + 1);
    float acc[MODE == kForward ? 2 : 1][4][16] = {};
    if (quad < quads) {
#pragma unroll
      for (int which = 0; which < (MODE == kForward ? 2 : 1); ++which) {
        for (int ch = 0; ch < chunks[which]; ++ch, ++use) {
          [[maybe_unused]] float f = 1.0f;
          if constexpr (MODE == kWeightGrad) {
            if ((ch & 31) == 0 && (ch > 0 || k == e || chunks[0] > 32))
              stage_factor = ch + lane < chunks[0] ? p.stage_factor[ch + lane] : 0.0f;
            f = __shfl_sync(0xffffffffu, stage_factor, ch & 31);
          }
          const uint32_t buf = acc_of(p, use % kPipes, use / kPipes);
          // after an abort nothing is waited for, but the warps stay together (group_sync)
          if (ok)
            ok = wait_warp(bars.acc_full + 8 * (buf + kMaxAccs * e), (phases >> buf) & 1u, p.status, &sh.abort_flag);
          phases ^= 1u << buf;
          tc_fence_after();
          const uint32_t d = sh.tmem + acc_cols(p) * buf + (uint32_t(32 * quad) << 16);
          const uint32_t lo = d + (MODE == kForward ? n : 64);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (16 * j >= n) break;  // an odd last tile of 8 reads 8 columns more of its accumulator
            add_tile<MODE>(acc[which][j], d + 16 * j, lo + 16 * j, f);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars.acc_empty + 8 * buf);
        }
      }
    } else {
      use += uint32_t(chunks[0] + chunks[1]);
    }
    [[maybe_unused]] const float* row_scale = row_scales + 64 * ((k >> 1) & 3);
    if constexpr (MODE == kInt8) {
      group_sync(e);  // the group's last item, whose place in the ring is filled again, has been written
      fetch_scales(k + 2 * kScaleAhead);
      if (quad == 0) asm volatile("cp.async.wait_group %0;" ::"n"(kScaleAhead) : "memory");
      group_sync(e);
    }
    if (per_token) cp_async_wait_all();
    if (by_rows(MODE) && p.R > 64 && p.out1 == nullptr) {
      // Every lane has a token, one output: straight from the registers, a 32-byte sector of a row at a time.
      // (1436 block rows, 765 tokens: 172 us, and 237 us through shared memory as below, whose barriers and
      // copies, 8 columns at a time for lack of room, cost more than whole lines save. With three outputs the
      // scattered stores cost more: a training step of 1000 tokens 1195 us, and 1168 us as below.)
      if (in_tile && t0 + row < p.tokens) {
        float* o = p.out0 + (t0 + row) * p.M + u.x;
        [[maybe_unused]] float ts = 0.0f;
        [[maybe_unused]] const float f = factors[row];
        if constexpr (MODE == kInt8) ts = p.token_scale[t0 + row];
#pragma unroll 1
        for (int j = 0; 8 * j < n; ++j, o += 8) {
          float v[8], w[8], hv[8];
          auto pick = [&](auto c) {  // registers cannot be indexed by j
            constexpr int J = decltype(c)::value;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              v[i] = acc[0][J / 2][8 * (J & 1) + i];
              if constexpr (MODE == kForward) {
                v[i] = v[i] * f;
                w[i] = acc[1][J / 2][8 * (J & 1) + i] * f;
              }
            }
          };
          switch (j) {
            case 0: pick(std::integral_constant<int, 0>()); break;
            case 1: pick(std::integral_constant<int, 1>()); break;
            case 2: pick(std::integral_constant<int, 2>()); break;
            case 3: pick(std::integral_constant<int, 3>()); break;
            case 4: pick(std::integral_constant<int, 4>()); break;
            case 5: pick(std::integral_constant<int, 5>()); break;
            case 6: pick(std::integral_constant<int, 6>()); break;
            default: pick(std::integral_constant<int, 7>()); break;
          }
          if constexpr (MODE == kForward) {
            with_act(p.act, [&](auto kind) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float a, da;
                act_both<decltype(kind)::value>(v[i], a, da);
                hv[i] = a * w[i];
              }
            });
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) hv[i] = float(__float_as_int(v[i])) * (ts * row_scale[8 * j + i]);
          }
          put8(o, hv, p.vec);
        }
      }
    } else if constexpr (by_rows(MODE)) {
      float* st_up = stage + p.R * ld;
      const int rows = int(min((long long)p.R, p.tokens - t0));
      for (int c0 = 0; c0 < n; c0 += 1 << slog) {
        group_sync(e);  // the buffer has been read
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = 8 * j - c0;
          if (!in_tile || c < 0 || c >= (1 << slog) || 8 * j >= n) continue;
          float* v = acc[0][j / 2] + 8 * (j & 1);
          store8(stage + row * ld + c, v);
          if constexpr (MODE == kForward) store8(st_up + row * ld + c, acc[1][j / 2] + 8 * (j & 1));
        }
        group_sync(e);
        if (c0 + sc < n)
          write_staged<MODE>(p, stage, st_up, ld, 128 >> log4, sc, sr, rows, t0 * p.M + u.x + c0 + sc,
                             row_scale + c0 + sc, p.token_scale + t0, factors);
      }
    } else {
      const bool live = MODE == kWeightGrad ? row < int(u.y) * 8 : in_tile && t0 + row < p.tokens;
      if (!live) continue;
      [[maybe_unused]] const float f = factors[row];
      float* dst = MODE == kInputGrad
                       ? p.out0 + (t0 + row) * p.K + u.x
                       : ((g2.z & 1u) ? p.out1 : p.out0) + (u64(g2.x) | u64(g2.y) << 32) + (long long)row * n;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (8 * j >= n) break;
        float* a = acc[0][j / 2] + 8 * (j & 1);
        if constexpr (MODE == kInputGrad) {
#pragma unroll
          for (int i = 0; i < 8; ++i) a[i] *= f;
        }
        put8(dst + 8 * j, a, p.vec);
      }
    }
  }
}

// ---- the kernel ----------------------------------------------------------------------------------

template <int MODE>
__global__ void __launch_bounds__(kPairThreads, 1) pair_kernel(PairParams p) {
  extern __shared__ char dyn[];
  __shared__ PairShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t slots = (smem_addr(dyn) + 1023u) & ~1023u, zero = slots + kPipes * kPipeBytes;
  char* zero_ptr = dyn + (zero - smem_addr(dyn));
  const PairBars bars{smem_addr(sh.full), smem_addr(sh.empty), smem_addr(sh.acc_full),
                      smem_addr(sh.acc_empty), smem_addr(sh.drain)};
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxSlots; ++s) {
      mbar_init(bars.full + 8 * s, 1);
      mbar_init(bars.empty + 8 * s, 1);
    }
    for (int b = 0; b < kMaxAccs; ++b) {
      mbar_init(bars.acc_full + 8 * b, 1);  // one for each epilogue group, which see only their own phases
      mbar_init(bars.acc_full + 8 * (kMaxAccs + b), 1);
      mbar_init(bars.acc_empty + 8 * b, live_quads<MODE>(p));
    }
    for (int b = 0; b < kPipes; ++b) mbar_init(bars.drain + 8 * b, 1);
    sh.abort_flag = 0;
    mbar_fence_init();
  }
  for (int i = threadIdx.x; i < kZeroBytes / 16; i += kPairThreads)
    reinterpret_cast<uint4*>(zero_ptr)[i] = make_uint4(0, 0, 0, 0);
  if (by_rows(MODE) && warp == 1 && lane < 8) sh.stages[lane].template init<MODE>(p, 8 * (lane + 1));
  fence_proxy_async_smem();
  if (warp == kPipes) {
    tc_alloc(smem_addr(&sh.tmem), 512);
    tc_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  if (warp < kPipes) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
    // the launch before makes the panel; by rows and columns the first weights are fetched meanwhile
    if (MODE == kWeightGrad && !p.beside) griddep_wait();
    if constexpr (by_rows(MODE))
      produce_rows<MODE>(p, sh, slots, zero, bars, warp, lane);
    else if constexpr (MODE == kInputGrad)
      produce_cols(p, sh, slots, zero, bars, warp, lane);
    else
      produce_grads(p, sh, slots, bars, warp, lane);
  } else if (warp < 2 * kPipes) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs));
    issue_mmas<MODE>(p, sh, bars, warp - kPipes, lane);
  } else if (warp >= kEpilogueWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpilogueRegs));
    const int group = (warp - kEpilogueWarp) >> 2;
    float* stage = reinterpret_cast<float*>(zero_ptr + kZeroBytes + kTailBytes + group * kStageBytes);
    epilogue<MODE>(p, sh, bars, stage, (warp - kEpilogueWarp) & 3, group, lane);
  }
  tc_fence_before();
  __syncthreads();
  if (sh.abort_flag) {
    // a wait gave up: copies and MMAs may still be in flight; give them time before the memory goes
    const long long t0 = clock64();
    while (clock64() - t0 < 20000000ll) __nanosleep(1000);
    __syncthreads();
  }
  tc_fence_after();
  if (warp == kPipes) tc_dealloc(sh.tmem, 512);
  if (MODE == kWeightGrad && p.beside) griddep_wait();  // the launch beside it is done when this one is
}

}  // namespace vbsr_b200
