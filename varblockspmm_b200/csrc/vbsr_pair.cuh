// vbsr_pair.cuh — the tensor-core engine of the block-sparse layer operators (tcgen05, TMEM).
//
// FP32 accuracy from 16-bit tensor-core products. Every fp32 operand x is held as a pair of fp16
// numbers: with a power of two 2^e that brings the operand's largest magnitude into [2^14, 2^15),
//   hi = fp16(x 2^e),  lo = fp16((x 2^e - hi) 2^11),   x 2^e = hi + lo 2^-11 (1 + d), |d| <= 2^-12,
// so the pair holds x to 2^-23 of itself (fp32 itself: 2^-24) for every |x| within 2^-28 of the
// largest, and to 2^-51 of the largest below that. The factor 2^11 keeps lo out of fp16's
// subnormals. A product of two operands is hi hi + 2^-11 (hi lo + lo hi); lo lo is below 2^-22 of it
// and left out. The two sums go to accumulators of their own (fp32, in TMEM) and are joined, and
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
//   panels:  per tile of R tokens (a multiple of 8, at most 128) and 8-feature group,
//            [R tokens of hi][R tokens of lo'], zeros behind the last token.
// Block widths are multiples of 8, so any block is a whole number of groups; K = 16 steps take two
// groups, and an odd last one is paired with a tile of zeros (and, on the weights' side, with itself,
// so that no stale bytes are multiplied).
//
// The kernel: one persistent CTA per SM; a producer warp (bulk copies into a ring of slots, and each
// slot's list of MMA steps), one MMA thread that only works off those lists, four epilogue warps on
// two accumulator buffers. Tokens are on the M side (64 or 128 rows): with weights there, blocks of
// 8 to 56 rows would leave most of an MMA empty. What bounds it: the copies into shared memory.
// A weight group of 32 h bytes needs 32 R bytes of activations, from L2, so few tokens run at the
// weights' HBM rate and many at the L2-to-shared-memory rate, h / 2 operations per byte.
#pragma once
#include <cuda_fp16.h>

#include "vbsr_kernels_common.cuh"

namespace vbsr_b200 {

enum PairMode { kForward = 0, kInputGrad = 1, kWeightGrad = 2, kInt8 = 3 };

// A block row, or rows [r0, r0 + hp) of one (parts keep all SMs busy when there are few rows).
// which: 0 gate, 1 up (kInt8 uses 0 only).
struct alignas(16) RowUnit {
  uint32_t row0;   // first row of C
  uint32_t shape;  // h | hp << 8 | r0 << 16
  uint32_t g0[2];  // first entry of the group list
  uint32_t ng[2];  // groups (kInt8: 16-column chunks)
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
  long long tokens, M, K;
  const char* x;              // activation panel in pairs (kInt8: in 16-column chunks)
  const char* dy;             // gradient panel in pairs
  const char* w;              // weights in pairs (kInt8: int8 chunks)
  const int* exps;            // exponents of x and dy: the call's
  const int* w_exp;           // exponent of the weights: the plan's
  const float* row_scale;     // kInt8
  const float* token_scale;
  float *out0, *out1, *out2;  // kForward: H, G, U; kInputGrad: dB; kWeightGrad: dgate, dup; kInt8: C
  int vec;                    // outputs are 16-byte aligned
  int* status;
};

// One K step: two MMAs (kInt8: one). a and b are shared-memory descriptors; their unused top bits
// carry flags.
struct PairStep {
  u64 a, b;
};
constexpr u64 kStepFresh = 1ull << 60;  // first step into its accumulator: overwrite
constexpr u64 kStepUp = 1ull << 59;     // second accumulator (up)
constexpr u64 kStepOdd = 1ull << 58;    // the second K half of A is the tile of zeros
constexpr u64 kStepMask = (1ull << 56) - 1;
constexpr int kMaxSteps = 32;

// Slot header: steps | N/8 << 8 | flags. No steps: end of the work.
constexpr uint32_t kHdrFirst = 1u << 16, kHdrLast = 1u << 17;

template <int MODE>
struct PairShape {
  static constexpr int slots = MODE == kForward || MODE == kInt8 ? 8 : 4;
  static constexpr int slot_bytes = MODE == kForward || MODE == kInt8 ? 24 * 1024 : 48 * 1024;
};
constexpr int kPairThreads = 256;
constexpr int kZeroBytes = 2048;   // 128 rows of 16 bytes
constexpr int kTailBytes = 4096;   // MMAs read up to this far behind a tile's own rows
constexpr int kGradTokens = 64;    // kWeightGrad: tokens per stage
template <int MODE>
constexpr int pair_smem() {
  return PairShape<MODE>::slots * PairShape<MODE>::slot_bytes + kZeroBytes + kTailBytes + 1024;
}

__device__ __forceinline__ u64 core_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return u64((addr >> 4) & 0x3FFFu) | (u64((lbo >> 4) & 0x3FFFu) << 16) |
         (u64((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}

__device__ __forceinline__ void tc_mma_f16(uint32_t d, u64 a, u64 b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tc_mma_i8(uint32_t d, u64 a, u64 b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
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

// 8 accumulator columns each from one, three or four places, loaded and waited for in one statement
// (the registers are not valid before the wait).
__device__ __forceinline__ void tc_ld8_1(uint32_t a, float (&v)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
      : "r"(a)
      : "memory");
}
__device__ __forceinline__ void tc_ld8_3(uint32_t a, uint32_t b, uint32_t c, float (&v)[8],
                                         float (&w)[8], float (&x)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%24];\n"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8, %9, %10, %11, %12, %13, %14, %15}, [%25];\n"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%16, %17, %18, %19, %20, %21, %22, %23}, [%26];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3]), "=f"(w[4]), "=f"(w[5]),
        "=f"(w[6]), "=f"(w[7]), "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]),
        "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
      : "r"(a), "r"(b), "r"(c)
      : "memory");
}
__device__ __forceinline__ void tc_ld8_4(uint32_t a, uint32_t b, uint32_t c, uint32_t d,
                                         float (&v)[8], float (&w)[8], float (&x)[8], float (&y)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%32];\n"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8, %9, %10, %11, %12, %13, %14, %15}, [%33];\n"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%16, %17, %18, %19, %20, %21, %22, %23}, [%34];\n"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%24, %25, %26, %27, %28, %29, %30, %31}, [%35];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3]), "=f"(w[4]), "=f"(w[5]),
        "=f"(w[6]), "=f"(w[7]), "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]),
        "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(y[0]), "=f"(y[1]), "=f"(y[2]), "=f"(y[3]),
        "=f"(y[4]), "=f"(y[5]), "=f"(y[6]), "=f"(y[7])
      : "r"(a), "r"(b), "r"(c), "r"(d)
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

// 2^-e in two factors that neither overflow nor vanish, for |e| <= 252.
__device__ __forceinline__ void unscale(int e, float& f1, float& f2) {
  const int a = -e / 2, b = -e - a;
  f1 = __int_as_float((a + 127) << 23);
  f2 = __int_as_float((b + 127) << 23);
}

struct PairBars {
  uint32_t full, empty, acc_full, acc_empty, drain;  // first barrier of each array
};

// The producer's ring position.
struct Ring {
  uint32_t slot = 0, parity = 1;  // parity of the empty barrier to wait for
  uint32_t filled = 0;            // stages issued
  template <int SLOTS>
  __device__ __forceinline__ void next() {
    ++filled;
    if (++slot == SLOTS) {
      slot = 0;
      parity ^= 1u;
    }
  }
};

struct PairShared {
  u64 full[8], empty[8], acc_full[2], acc_empty[2], drain;
  PairStep steps[8][kMaxSteps];
  uint32_t header[8];
  uint32_t tmem;
  volatile int abort_flag;
};

// ---- producer: kForward and kInt8 ----------------------------------------------------------------

template <int MODE>
__device__ void produce_rows(const PairParams& p, PairShared& sh, uint32_t slots, uint32_t zero,
                             const PairBars& bars, int lane) {
  constexpr bool I8 = MODE == kInt8;
  constexpr int SLOTS = PairShape<MODE>::slots, BYTES = PairShape<MODE>::slot_bytes;
  const uint32_t xb = (I8 ? 16u : 32u) * uint32_t(p.R);  // panel bytes of a group
  const uint64_t pol_x = policy_evict_last(), pol_w = policy_evict_first();
  const int items = p.units * p.tiles;
  Ring ring;
  int item = blockIdx.x;
  // work ahead: the unit of the next item, the group columns of the next stage
  RowUnit u{};
  if (item < items) u = p.rows[item / p.tiles];
  auto seek = [&](int& it, RowUnit& un, int& which) {  // next item with groups
    while (it < items && un.ng[0] + un.ng[1] == 0) {
      it += gridDim.x;
      if (it < items) un = p.rows[it / p.tiles];
    }
    which = it < items && un.ng[0] == 0 ? 1 : 0;
  };
  int which = 0, off = 0;
  seek(item, u, which);
  int nitem = item + int(gridDim.x);
  RowUnit nu{};
  if (nitem < items) nu = p.rows[nitem / p.tiles];
  auto load_cols = [&](const RowUnit& un, int wh, int of) {
    return of + lane < int(un.ng[wh]) ? p.group_col[un.g0[wh] + of + lane] : 0u;
  };
  uint32_t col = item < items ? load_cols(u, which, 0) : 0u;
  bool ok = true;
  while (item < items) {
    const int h = int(u.shape & 255u), hp = int((u.shape >> 8) & 255u), r0 = int(u.shape >> 16);
    const uint32_t wb = (I8 ? 16u : 32u) * uint32_t(hp);
    int cap = BYTES / int(xb + wb);
    cap = (cap < 32 ? cap : 32) & ~1;
    const int n = min(cap, int(u.ng[which]) - off);
    // the next stage
    int w2 = which, o2 = off + n, it2 = item;
    RowUnit u2 = u;
    if (o2 >= int(u.ng[w2])) {
      o2 = 0;
      if (w2 == 0 && u.ng[1] > 0) {
        w2 = 1;
      } else {
        it2 = nitem;
        u2 = nu;
        seek(it2, u2, w2);
        nitem = it2 + int(gridDim.x);
        if (nitem < items) nu = p.rows[nitem / p.tiles];
      }
    }
    const bool last = it2 != item;
    const uint32_t col2 = it2 < items ? load_cols(u2, w2, o2) : 0u;

    if (!(ok = wait_warp(bars.empty + 8 * ring.slot, ring.parity, p.status, &sh.abort_flag))) break;
    const uint32_t base = slots + ring.slot * BYTES, full = bars.full + 8 * ring.slot;
    const uint32_t wbase = base + uint32_t(n) * xb;
    const int steps = (n + 1) / 2;
    if (lane < steps) {
      const bool pair = 2 * lane + 1 < n;
      const uint32_t a = base + 2u * lane * xb, b = wbase + 2u * lane * wb;
      sh.steps[ring.slot][lane].a = core_desc(a, pair ? xb : zero - a, 128) |
                                    (lane == 0 && off == 0 ? kStepFresh : 0) |
                                    (which ? kStepUp : 0) | (pair ? 0 : kStepOdd);
      sh.steps[ring.slot][lane].b = core_desc(b, pair ? wb : 0u, 128);
    }
    if (lane == 0)
      sh.header[ring.slot] = uint32_t(steps) | uint32_t(hp) << 5 |
                             (off == 0 && (which == 0 || u.ng[0] == 0) ? kHdrFirst : 0u) |
                             (last ? kHdrLast : 0u);
    __syncwarp();
    if (lane == 0) mbar_arrive_expect_tx(full, uint32_t(n) * (xb + wb));
    __syncwarp();
    // weights: one run, or per group the part's rows of hi and of lo'
    const char* wsrc = p.w + u.w0[which] + (long long)off * (I8 ? 16 : 32) * h;
    if (hp == h) {
      if (lane == 0) {
        if (p.tiles == 1)
          bulk_g2s(wbase, wsrc, uint32_t(n) * wb, full, pol_w);
        else
          bulk_g2s_plain(wbase, wsrc, uint32_t(n) * wb, full);
      }
    } else if (lane < n) {
      const char* g = wsrc + (long long)lane * (I8 ? 16 : 32) * h + 16 * r0;
      bulk_g2s_plain(wbase + lane * wb, g, 16u * hp, full);
      if (!I8) bulk_g2s_plain(wbase + lane * wb + 16u * hp, g + 16 * h, 16u * hp, full);
    }
    // activations: one copy per run of neighbouring groups
    const uint32_t before = __shfl_up_sync(0xffffffffu, col, 1);
    const bool head = lane < n && (lane == 0 || col != before + 1);
    const uint32_t heads = __ballot_sync(0xffffffffu, head) | (n < 32 ? 1u << n : 0u);
    if (head) {
      const uint32_t rest = lane < 31 ? heads >> (lane + 1) : 0u;
      const uint32_t run = rest ? uint32_t(__ffs(rest)) : uint32_t(32 - lane);
      const long long tile = p.tile0 + item % p.tiles;
      const long long per_tile = I8 ? (p.K >> 3) + 1 : p.K >> 3;  // see panel8_chunks
      bulk_g2s(base + lane * xb, p.x + (tile * per_tile + col) * xb, run * xb, full, pol_x);
    }
    ring.next<SLOTS>();
    item = it2;
    which = w2;
    off = o2;
    u = u2;
    col = col2;
  }
  if (ok) {  // end marker
    ok = wait_warp(bars.empty + 8 * ring.slot, ring.parity, p.status, &sh.abort_flag);
    if (ok && lane == 0) {
      sh.header[ring.slot] = 0u;
      mbar_arrive(bars.full + 8 * ring.slot);
    }
    if (ok) ring.next<SLOTS>();
  }
}

// ---- producer: kInputGrad ------------------------------------------------------------------------

__device__ __forceinline__ void produce_cols(const PairParams& p, PairShared& sh, uint32_t slots,
                                             uint32_t zero, const PairBars& bars, int lane) {
  constexpr int SLOTS = PairShape<kInputGrad>::slots, BYTES = PairShape<kInputGrad>::slot_bytes;
  const uint32_t xb = 32u * uint32_t(p.R);
  const uint64_t pol_x = policy_evict_last();
  const int items = p.units * p.tiles;
  const long long per_tile = 2 * (p.M >> 3);
  Ring ring;
  bool ok = true;
  int item = blockIdx.x;
  ColUnit nu{};
  if (item < items) nu = p.cols[item / p.tiles];
  for (; ok && item < items; item += gridDim.x) {
    const ColUnit u = nu;
    if (item + int(gridDim.x) < items) nu = p.cols[(item + gridDim.x) / p.tiles];
    const char* dy = p.dy + (p.tile0 + item % p.tiles) * per_tile * xb;
    auto load = [&](uint32_t s) {
      ColEntry e{};
      if (lane < kColEntries && s < u.ns) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.entries) +
                              (long long)(u.s0 + s) * kColEntries + lane);
        e.dy_group = v.x;
        e.h8 = v.y;
        e.w_byte = u64(v.z) | u64(v.w) << 32;
      }
      return e;
    };
    ColEntry next = load(0);
    for (uint32_t s = 0; s < u.ns; ++s) {
      const ColEntry e = next;
      next = load(s + 1);
      // places of the entries: groups before this one, and its steps
      uint32_t g = e.h8, st = (e.h8 + 1) / 2;
#pragma unroll
      for (int d = 1; d < kColEntries; d *= 2) {
        const uint32_t g2 = __shfl_up_sync(0xffffffffu, g, d), s2 = __shfl_up_sync(0xffffffffu, st, d);
        if (lane >= d) {
          g += g2;
          st += s2;
        }
      }
      const uint32_t groups = __shfl_sync(0xffffffffu, g, kColEntries - 1);
      const uint32_t steps = __shfl_sync(0xffffffffu, st, kColEntries - 1);
      const uint32_t g_before = g - e.h8, s_before = st - (e.h8 + 1) / 2;
      if (!(ok = wait_warp(bars.empty + 8 * ring.slot, ring.parity, p.status, &sh.abort_flag))) break;
      const uint32_t base = slots + ring.slot * BYTES, full = bars.full + 8 * ring.slot;
      const uint32_t a0 = base + g_before * xb, b0 = base + groups * xb + g_before * 32u * u.w;
      const uint32_t h = 8u * e.h8;
      if (lane < kColEntries)
        for (uint32_t j = 0; 2 * j < e.h8; ++j) {
          const bool pair = 2 * j + 1 < e.h8;
          const uint32_t a = a0 + 2 * j * xb;
          PairStep& out = sh.steps[ring.slot][s_before + j];
          out.a = core_desc(a, pair ? xb : zero - a, 128) |
                  (s == 0 && s_before + j == 0 ? kStepFresh : 0) | (pair ? 0 : kStepOdd);
          // columns 8 apart are 16 h apart (hi and lo' tiles alternate), rows 8 apart 128 bytes
          out.b = core_desc(b0 + 256u * j, pair ? 128u : 0u, 16u * h);
        }
      if (lane == 0)
        sh.header[ring.slot] = steps | u.w << 5 | (s == 0 ? kHdrFirst : 0u) |
                               (s + 1 == u.ns ? kHdrLast : 0u);
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(full, groups * (xb + 32u * u.w));
      __syncwarp();
      if (e.h8) {
        bulk_g2s(a0, dy + (long long)e.dy_group * xb, e.h8 * xb, full, pol_x);
        bulk_g2s_plain(b0, p.w + e.w_byte + (long long)(u.c0 >> 3) * 32 * h, 4u * h * u.w, full);
      }
      ring.next<SLOTS>();
    }
  }
  if (ok) {
    ok = wait_warp(bars.empty + 8 * ring.slot, ring.parity, p.status, &sh.abort_flag);
    if (ok && lane == 0) {
      sh.header[ring.slot] = 0u;
      mbar_arrive(bars.full + 8 * ring.slot);
    }
  }
}

// ---- producer: kWeightGrad -----------------------------------------------------------------------

// A stage is kGradTokens tokens (the last of a tile fewer) of the unit's 16 activation groups and of
// its h / 8 gradient groups, each group [kGradTokens of hi][kGradTokens of lo'].
__device__ __forceinline__ void produce_grads(const PairParams& p, PairShared& sh, uint32_t slots,
                                              const PairBars& bars, int lane) {
  constexpr int SLOTS = PairShape<kWeightGrad>::slots, BYTES = PairShape<kWeightGrad>::slot_bytes;
  constexpr uint32_t GB = 32u * kGradTokens;
  const uint32_t xb = 32u * uint32_t(p.R);
  const uint64_t pol_x = policy_evict_last();
  Ring ring;
  bool ok = true;
  int item = blockIdx.x;
  GradUnit nu{};
  uint32_t ncol = 0;
  if (item < p.units) {
    nu = p.grads[item];
    ncol = lane < int(nu.ng) ? p.group_col[nu.g0 + lane] : 0u;
  }
  for (; ok && item < p.units; item += gridDim.x) {
    const GradUnit u = nu;
    const uint32_t col = ncol;
    if (item + int(gridDim.x) < p.units) {
      nu = p.grads[item + gridDim.x];
      ncol = lane < int(nu.ng) ? p.group_col[nu.g0 + lane] : 0u;
    }
    const uint32_t h8 = u.h / 8;
    for (int tile = 0; ok && tile < p.tiles; ++tile) {
      const char* x = p.x + ((long long)tile * (p.K >> 3) + col) * xb;
      const char* dy = p.dy + ((long long)tile * 2 * (p.M >> 3) + u.dy_group + lane - 16) * xb;
      for (int t0 = 0; t0 < p.R; t0 += kGradTokens) {
        const int nt = min(kGradTokens, p.R - t0);
        if (!(ok = wait_warp(bars.empty + 8 * ring.slot, ring.parity, p.status, &sh.abort_flag)))
          break;
        const uint32_t base = slots + ring.slot * BYTES, full = bars.full + 8 * ring.slot;
        const int steps = nt / 16;
        if (lane < steps) {
          PairStep& out = sh.steps[ring.slot][lane];
          out.a = core_desc(base + 256u * lane, 128u, GB) |
                  (tile == 0 && t0 == 0 && lane == 0 ? kStepFresh : 0);
          out.b = core_desc(base + 16u * GB + 256u * lane, 128u, GB / 2);
        }
        if (lane == 0)
          sh.header[ring.slot] = uint32_t(steps) | u.h << 5 |
                                 (tile == 0 && t0 == 0 ? kHdrFirst : 0u) |
                                 (tile + 1 == p.tiles && t0 + kGradTokens >= p.R ? kHdrLast : 0u);
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(full, (u.ng + h8) * 32u * uint32_t(nt));
        __syncwarp();
        const bool is_x = lane < int(u.ng), is_dy = lane >= 16 && lane < 16 + int(h8);
        if (is_x || is_dy) {
          const char* src = (is_x ? x : dy) + 16 * t0;
          const uint32_t dst = base + lane * GB;
          bulk_g2s(dst, src, 16u * nt, full, pol_x);
          bulk_g2s(dst + GB / 2, src + 16 * p.R, 16u * nt, full, pol_x);
        }
        ring.next<SLOTS>();
      }
    }
  }
  if (ok) {
    ok = wait_warp(bars.empty + 8 * ring.slot, ring.parity, p.status, &sh.abort_flag);
    if (ok && lane == 0) {
      sh.header[ring.slot] = 0u;
      mbar_arrive(bars.full + 8 * ring.slot);
    }
  }
}

// ---- MMA thread ----------------------------------------------------------------------------------

template <int MODE>
__device__ void issue_mmas(const PairParams& p, PairShared& sh, const PairBars& bars) {
  constexpr int SLOTS = PairShape<MODE>::slots;
  const int m = MODE == kWeightGrad ? 128 : (p.R > 64 ? 128 : 64);
  // D f32, A and B f16 (kInt8: D s32, A and B s8); transposed (MN-major) operands in bits 15 and 16
  const uint32_t form = (MODE == kInt8 ? (2u << 4) | (1u << 7) | (1u << 10) : (1u << 4)) |
                        (MODE == kWeightGrad ? 1u << 15 : 0u) |
                        (MODE == kWeightGrad || MODE == kInputGrad ? 1u << 16 : 0u) |
                        (uint32_t(m >> 4) << 24);
  const u64 lo = MODE == kWeightGrad ? kGradTokens : u64(p.R);  // hi to lo' tile of A, in 16 bytes
  uint32_t slot = 0, parity = 0, use = 0;
  while (true) {
    if (!wait_one(bars.full + 8 * slot, parity, p.status, &sh.abort_flag)) return;
    const uint32_t hdr = *reinterpret_cast<volatile uint32_t*>(&sh.header[slot]);
    const int steps = int(hdr & 63u), n = int((hdr >> 8) & 15u) * 8;
    if (steps == 0) break;
    const uint32_t buf = use & 1u;
    if (hdr & kHdrFirst)
      if (!wait_one(bars.acc_empty + 8 * buf, ((use >> 1) & 1u) ^ 1u, p.status, &sh.abort_flag)) return;
    tc_fence_after();
    const uint32_t d0 = sh.tmem + 256u * buf;
    // N of one tile of n columns: a multiple of 16 for M = 128 (one tile more is read, and its
    // columns are not used)
    const int n1 = m == 128 || MODE == kInt8 ? (n + 15) & ~15 : n;
    const uint32_t i1 = form | (uint32_t(n1 >> 3) << 17), i2 = form | (uint32_t(2 * n >> 3) << 17);
    for (int s = 0; s < steps; ++s) {
      const PairStep st = sh.steps[slot][s];
      const u64 a = st.a & kStepMask, b = st.b;
      const uint32_t acc = (st.a & kStepFresh) ? 0u : 1u;
      const uint32_t d = d0 + ((st.a & kStepUp) ? 128u : 0u);
      if (MODE == kInt8) {
        tc_mma_i8(d, a, b, i1, acc);
        continue;
      }
      // hi x [hi; lo'] and lo' x hi
      const u64 a2 = a + lo - ((st.a & kStepOdd) ? lo << 16 : 0ull);
      tc_mma_f16(d, a, b, i2, acc);
      if (MODE == kForward)  // columns [n, 2n) hold hi lo'; lo' hi joins them
        tc_mma_f16(d + n, a2, b, i1, 1u);
      else  // hi and lo' columns alternate by 8: every second tile, into columns of its own
        tc_mma_f16(d + 128u, a2, b + (b & (0x3FFFull << 32)), i1, acc);
    }
    tc_commit(bars.empty + 8 * slot);
    if (hdr & kHdrLast) {
      tc_commit(bars.acc_full + 8 * buf);
      ++use;
    }
    if (++slot == SLOTS) {
      slot = 0;
      parity ^= 1u;
    }
  }
  tc_commit(bars.drain);  // nothing may arrive on a barrier of a CTA that has gone
  wait_one(bars.drain, 0, p.status, &sh.abort_flag);
}

// ---- epilogue ------------------------------------------------------------------------------------

__device__ __forceinline__ void store8(float* dst, const float (&v)[8], int vec) {
  if (vec) {
    reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = v[i];
  }
}
constexpr float kLoUnit = 1.0f / 2048.0f;  // 2^-11

template <int MODE>
__device__ void epilogue(const PairParams& p, PairShared& sh, const PairBars& bars, int quad, int lane) {
  const bool wide = MODE == kWeightGrad || p.R > 64;  // M = 128; M = 64 fills lanes 0..15
  const int row = wide ? 32 * quad + lane : 16 * quad + lane;
  const bool in_tile = wide || lane < 16;
  const int items = MODE == kWeightGrad ? p.units : p.units * p.tiles;
  float f1 = 1.0f, f2 = 1.0f;
  if (MODE == kForward) unscale(p.exps[0] + *p.w_exp, f1, f2);
  if (MODE == kInputGrad) unscale(p.exps[1] + *p.w_exp, f1, f2);
  if (MODE == kWeightGrad) unscale(p.exps[0] + p.exps[1], f1, f2);
  uint32_t use = 0;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const uint32_t buf = use & 1u;
    const uint32_t d0 = sh.tmem + 256u * buf + (uint32_t(32 * quad) << 16);
    const long long t = MODE == kWeightGrad ? 0 : (long long)(p.tile0 + item % p.tiles) * p.R + row;
    bool work = true;
    int n = 0;
    bool live = false;
    RowUnit ru{};
    ColUnit cu{};
    GradUnit gu{};
    if (MODE == kForward || MODE == kInt8) {
      ru = p.rows[item / p.tiles];
      n = int((ru.shape >> 8) & 255u);
      work = ru.ng[0] + ru.ng[1] > 0;
      live = in_tile && row < p.R && t < p.tokens;
    } else if (MODE == kInputGrad) {
      cu = p.cols[item / p.tiles];
      n = int(cu.w);
      work = cu.ns > 0;
      live = in_tile && row < p.R && t < p.tokens;
    } else {
      gu = p.grads[item];
      n = int(gu.h);
      live = row < int(gu.ng) * 8;
    }
    if (work) {
      if (!wait_warp(bars.acc_full + 8 * buf, (use >> 1) & 1u, p.status, &sh.abort_flag)) return;
      tc_fence_after();
    }
    float rs = 0.0f;
    if (MODE == kInt8 && live) rs = p.token_scale[t];
    for (int c = 0; c < n; c += 8) {
      if (MODE == kForward) {
        float g[8] = {}, u[8] = {}, gl[8] = {}, ul[8] = {};
        if (work) tc_ld8_4(d0 + c, d0 + n + c, d0 + 128 + c, d0 + 128 + n + c, g, gl, u, ul);
        if (live) {
          float hv[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // a matrix without blocks here left its columns unwritten
            g[i] = ru.ng[0] ? fmaf(gl[i], kLoUnit, g[i]) * f1 * f2 : 0.0f;
            u[i] = ru.ng[1] ? fmaf(ul[i], kLoUnit, u[i]) * f1 * f2 : 0.0f;
            hv[i] = act_value(p.act, g[i]) * u[i];
          }
          const long long o = t * p.M + ru.row0 + c;
          store8(p.out0 + o, hv, p.vec);
          if (p.out1 != nullptr) {
            store8(p.out1 + o, g, p.vec);
            store8(p.out2 + o, u, p.vec);
          }
        }
      } else if (MODE == kInt8) {
        float v[8] = {};
        if (work) tc_ld8_1(d0 + c, v);
        if (live) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[i] = float(__float_as_int(v[i])) * (rs * p.row_scale[ru.row0 + c + i]);
          store8(p.out0 + t * p.M + ru.row0 + c, v, p.vec);
        }
      } else {
        float v[8] = {}, l1[8] = {}, l2[8] = {};
        if (work) tc_ld8_3(d0 + 2 * c, d0 + 2 * c + 8, d0 + 128 + c, v, l1, l2);
        if (live) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = fmaf(l1[i] + l2[i], kLoUnit, v[i]) * f1 * f2;
          float* dst = MODE == kInputGrad
                           ? p.out0 + t * p.K + cu.col0 + c
                           : (gu.which ? p.out1 : p.out0) + gu.out + (long long)row * n + c;
          store8(dst, v, p.vec);
        }
      }
    }
    if (work) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars.acc_empty + 8 * buf);
      ++use;
    }
  }
}

// ---- the kernel ----------------------------------------------------------------------------------

template <int MODE>
__global__ void __launch_bounds__(kPairThreads, 1) pair_kernel(PairParams p) {
  constexpr int SLOTS = PairShape<MODE>::slots, BYTES = PairShape<MODE>::slot_bytes;
  extern __shared__ char dyn[];
  __shared__ PairShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t slots = (smem_addr(dyn) + 1023u) & ~1023u, zero = slots + SLOTS * BYTES;
  char* zero_ptr = dyn + (zero - smem_addr(dyn));
  const PairBars bars{smem_addr(sh.full), smem_addr(sh.empty), smem_addr(sh.acc_full),
                      smem_addr(sh.acc_empty), smem_addr(&sh.drain)};
  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(bars.full + 8 * s, 1);
      mbar_init(bars.empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bars.acc_full + 8 * b, 1);
      mbar_init(bars.acc_empty + 8 * b, 4);
    }
    mbar_init(bars.drain, 1);
    sh.abort_flag = 0;
    mbar_fence_init();
  }
  for (int i = threadIdx.x; i < kZeroBytes / 16; i += kPairThreads)
    reinterpret_cast<uint4*>(zero_ptr)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  if (warp == 1) {
    tc_alloc(smem_addr(&sh.tmem), 512);
    tc_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  if (warp == 0) {
    if (MODE == kForward || MODE == kInt8)
      produce_rows<MODE>(p, sh, slots, zero, bars, lane);
    else if (MODE == kInputGrad)
      produce_cols(p, sh, slots, zero, bars, lane);
    else
      produce_grads(p, sh, slots, bars, lane);
  } else if (warp == 1) {
    if (lane == 0) issue_mmas<MODE>(p, sh, bars);
    __syncwarp();
  } else if (warp >= 4) {
    epilogue<MODE>(p, sh, bars, warp - 4, lane);
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
  if (warp == 1) tc_dealloc(sh.tmem, 512);
}

}  // namespace vbsr_b200
