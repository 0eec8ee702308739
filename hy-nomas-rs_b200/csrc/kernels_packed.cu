// kernels_packed.cu — softmax attention of packed sequences with grouped
// heads: the masked current-segment part that joins the history part of
// nkv_bank_attend_history, whole prompts, and chunks of new tokens (down to
// one) over a longer cache.
//
// For token i of a sequence of q_len new tokens over k_len keys, key j is
// visible iff j < lim(i); lim(i) = k_len, or, causal, the end of the block of
// `block` tokens that holds key position i + k_len - q_len (block 1: the
// token itself is the last; block = tokens per frame: a frame sees itself and
// the frames before it).  Per head
//   S = scale * q k^T, o = softmax(S over visible keys) v, lse = log sum e^S,
// and with a history part (o_h, lse_h) the two-part merge
//   o = (e^lse_h o_h + e^lse o) / (e^lse_h + e^lse).
// A row that sees nothing gives o = 0, lse = -inf.
//
// Rows of one key/value head are packed: row r of a sequence is token r / G,
// query head kvh * G + r % G (G = heads / kv_heads), so a group's heads share
// every K / V tile and a single new token of a grouped model fills G rows.  A
// work item is two halves of up to 128 rows (whole tokens) of one sequence and
// key/value head over a range of 128-key tiles.  A plan made once per set of
// lengths deals the items to persistent CTAs, one per SM, and splits the key
// range of long rows when there are too few items to fill the GPU (their
// partial rows are merged by k_packed_combine).
//
// Per step of 64 keys: S_h = Q_h K^T and O_h += P_h V as tcgen05.mma (kind::f16,
// f32 in TMEM), P written over S_h in TMEM as the A operand, the running
// maximum moved only when a step exceeds it by more than 8 (base 2).  Scores,
// maxima, sums and O stay in f32; P is rounded to the type of V because the
// tensor core takes both operands in one type: an error of half a step of that
// type per probability, the size of the output's own rounding, or, where that is
// more in f16, of 2^-32 of the row's largest one (2^-32 n max|v| for n keys;
// kRaise).  The sum uses the unrounded values.
//
// A key past a row's limit has P = 0, but 0 times an infinity or a NaN in its
// V row is a NaN: the V rows that some but not all rows of an item see are
// checked in shared memory first (non-finite values zeroed and remembered; V
// rows that none sees zeroed), and rows that do see such a value get it added
// to their output at the end.
//
// Every wait on an mbarrier gives up after 1 s; the CTA then sets bit 0 of the
// plan's status word, frees the TMEM, fills its rows with NaN and returns.  A
// plan whose status word is set gives NaN until it is cleared: what such a call
// left in its outputs and workspace must not pass for a result.
//
// Measured, and what bounds it (copy 6.5 TB/s, matrix product 1,679 TFLOP/s):
// - 6,496 frame-causal queries, 24 heads of 128, history merged (319 GFLOP):
//   295 to 355 us by the GPU's power limit (clock down to 1,650 MHz), 0.9 to
//   1.08 PFLOP/s; tensor pipe 59 %, issue 52 %: the softmax warps' chain of
//   latencies per step (about 1,450 cycles for both halves, 1,280 of them tensor
//   time at head_dim 128: S at N = 64 takes 48 cycles per MMA, bound by shared
//   memory, where N = 128 would need 512 more TMEM columns).
// - 16,383 causal queries, 16 heads of 64 (550 GFLOP): 800 us, 0.69 PFLOP/s, the
//   exponentials and that chain.
// - one token over 29,056 keys, 24 heads of 128 (357 MB): 65 us, 5.5 TB/s.
// - chunks of 1 to 64 tokens over caches of up to 9,001 (59 MB): 26 us, of which
//   13 the loop at memory speed, the rest start, output and merge.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "nkv_device.cuh"
#include "nkv_kernels.h"
#include "nkv_tcgen05.cuh"

namespace nkv {
using namespace tc;
namespace {

constexpr int PQ = kPackedHalfRows;  // rows per half (TMEM lanes)
constexpr int PK = kPackedTileKeys;  // keys per K / V tile
constexpr int SK = kPackedStepKeys;  // keys per softmax step
static_assert(PQ == 128 && PK == 128 && SK == 64, "");
// warps 0-7 softmax (half = warp / 4), 8-9 MMA issue (one per half), 10 TMA, 11 V scrub
constexpr int kSoftmaxWarps = 8, kMmaWarp = 8, kTmaWarp = 10, kScrubWarp = 11;
constexpr int kThreads = 384;

// Shared memory for head_dim <= DP: the two Q halves, a ring of K tiles, a
// ring of V tiles, 4 KB per softmax warp to turn rows into lines.
template <int DP>
struct Shape {
  static constexpr int kTile = (DP / 64) * HALF_BYTES;  // 128 rows x DP 16-bit values
  static constexpr int kStages = DP == 128 ? 2 : 4;     // of each ring
  static constexpr int kK = 2 * kTile, kV = kK + kStages * kTile, kStage = kV + kStages * kTile,
                       kBars = kStage + kSoftmaxWarps * 4096;
  static constexpr int kSmem = kBars + 512 + 1024;
  static_assert(kSmem <= 232448, "shared memory");
};

// f32 accumulate, A and B both bf16 (1) or f16 (0); S: both K-major, N = 64
// keys.  O: B (V) MN-major, N = DP.
template <int DT>
constexpr uint32_t kIdescIn = (1u << 4) | (uint32_t(DT == BF16) << 7) | (uint32_t(DT == BF16) << 10) |
                              (uint32_t(PQ >> 4) << 24);
template <int DT>
constexpr uint32_t kIdescS = kIdescIn<DT> | (uint32_t(SK >> 3) << 17);
template <int DT, int DP>
constexpr uint32_t kIdescO = kIdescIn<DT> | (1u << 16) | (uint32_t(DP >> 3) << 17);

// 64 columns x 128 consecutive tokens of one head (a 3-D map: values, head,
// token), 128-byte swizzled, completing on `bar`; x is 0 or 64 values
// (16-byte aligned).  Columns past head_dim and tokens past the end read 0.
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* map, int x, int h, int tok, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(h), "r"(tok), "r"(bar)
      : "memory");
}

// Bounded wait as tc::bar_wait, but small: the roles' code runs from the
// instruction cache at once, and two dozen waits with their retries unrolled
// made it 120 KB.  (A suspend-time hint on the wait: the one-token case 76 us
// instead of 65.)
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
  if (bar_try(bar, parity)) return true;
  const uint64_t t0 = gtimer();
  uint32_t tries = 0;
#pragma unroll 1
  do {
    if (bar_try(bar, parity)) return true;
  } while ((++tries & 31u) || gtimer() - t0 <= kWaitNs);
  return false;
}

// Lane 0's arrival, predicated rather than branched around.
__device__ __forceinline__ void arrive_lane0(uint32_t bar, int lane) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.eq.s32 p, %1, 0;\n\t"
      "@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar),
      "r"(lane)
      : "memory");
}

// Keys visible to token i (causal or not), as documented above.
__device__ __forceinline__ int key_limit(const PackedArgs& a, const PackedItem& it, int i) {
  if (!a.causal) return it.k_len;
  const int64_t p = int64_t(i) + it.k_len - it.q_len;
  if (p < 0) return 0;
  const int64_t lim = a.block == 1 ? p + 1 : (int64_t(uint32_t(p) / uint32_t(a.block)) + 1) * a.block;
  return lim < it.k_len ? int(lim) : it.k_len;
}

// An item read anew: its fields need no registers while the steps run.
__device__ __forceinline__ PackedItem read_item(const PackedItem* p) {
  PackedItem it;
  static_assert(sizeof(PackedItem) == 64, "");
  int32_t* w = reinterpret_cast<int32_t*>(&it);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    asm volatile("ld.global.nc.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[4 * k]), "=r"(w[4 * k + 1]), "=r"(w[4 * k + 2]), "=r"(w[4 * k + 3])
                 : "l"(reinterpret_cast<const int4*>(p) + k));
  return it;
}

// NaN for all rows of the items first .. last - 1 (a part's maximum and sum
// carry it through the merge).  Not inlined: the steps' registers would be dealt
// out anew (six prompts of f16 217 us instead of 214, 8 bytes of spills at
// head_dim 64).
__device__ __noinline__ void fill_nan(const PackedArgs* a, int first, int last) {
  const int warp = int(threadIdx.x) >> 5, lane = int(threadIdx.x) & 31, G = a->G;
  const float nan = __int_as_float(0x7FFFFFFF);
#pragma unroll 1
  for (int i = first; i < last; ++i) {
    const PackedItem it = read_item(a->items + i);
#pragma unroll 1
    for (int r = warp; r < it.rows; r += kThreads / 32) {
      const int tok = (it.row0 + r) / G, h = it.kvh * G + (it.row0 + r) - tok * G;
      const int64_t q = int64_t(it.q_start) + tok;
      if (it.part_row >= 0) {
        if (lane == 0) reinterpret_cast<float2*>(a->part_ml)[int64_t(it.part_row) + r] = make_float2(nan, nan);
        continue;
      }
      if (lane == 0) a->lse[int64_t(h) * a->lse_head + q] = nan;
#pragma unroll 1
      for (int c = lane; c < a->D; c += 32) {
        const int64_t at = (q * a->H + h) * a->D + c;
        if (a->out_f32) static_cast<float*>(a->out)[at] = nan;
        else static_cast<uint16_t*>(a->out)[at] = uint16_t(0x7FFFu);
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return DT == BF16 ? dev::bf16x2_bits_nonnan(a, b) : dev::f16x2_bits_nonnan(a, b);
}

// 2^x on the FMA pipes: x = n + f with n the nearest integer (the low bits of x
// + 1.5 2^23), a degree-4 polynomial of 2^f on [-1/2, 1/2] (a fit of the least
// maximal relative error with the constant held at 1: 2.9e-6, a hundredth of
// P's rounding), n added to the exponent.  x is held at -127 from below, where
// f = 0, the polynomial is exactly 1 and the sum of the exponents leaves the
// bits of +0: a masked score (-inf) has P = 0.  (Held at -125 a masked key would
// weigh 2^-125, a normal bf16 number: 8 next to a value of 3.4e38.)  Between -127
// and -126 the result falls from 2^-126 to 0, 0 next to any row's sum.  x at most
// 2^7; a NaN is lost here and caught by the row maximum.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  x = make_float2(fmaxf(x.x, -127.0f), fmaxf(x.y, -127.0f));
  auto both = [](float v) { return make_float2(v, v); };
  const float2 t = __fadd2_rn(x, both(12582912.0f));
  const float2 f = __ffma2_rn(__fadd2_rn(t, both(-12582912.0f)), both(-1.0f), x);
  float2 p = __ffma2_rn(both(0.009582817554473877f), f, both(0.05590637028217316f));
  p = __ffma2_rn(p, f, both(0.24024099111557007f));
  p = __ffma2_rn(p, f, both(0.6931241750717163f));
  p = __ffma2_rn(p, f, both(1.0f));
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}

// Three-input maximum that keeps a NaN.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max2_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// What the running maximum m lies below a row's scores' (base 2), so that the
// largest probabilities are 2^kRaise to 2^(kRaise + 8).  f16 has no exponents to
// spare below: held near 1, every probability under 2^-25 of the largest became
// 0 in P but not in the sum (131,072 keys 17.4 nats below one: 0.36 % of the
// row's mass lost).  Raised by 2^7 (32,768 at most, of 65,504) that border is at
// 2^-32.  l and O carry the factor as well, and m accounts for it in lse and in
// the merge of parts.
template <int DT>
constexpr float kRaise = DT == F16 ? 7.0f : 0.0f;

// Exponent all ones: the smallest pattern of a non-finite value without sign.
template <int DT>
constexpr uint32_t kNonFinite = DT == BF16 ? 0x7F80u : 0x7C00u;
// The non-finite 16-bit halves of w.
template <int DT>
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t w) {
  constexpr uint32_t e = kNonFinite<DT>;
  return ((w & e) == e ? 0xFFFFu : 0u) | ((w & (e << 16)) == (e << 16) ? 0xFFFF0000u : 0u);
}

// Steps of 64 keys, two score buffers per half: TMEM columns
//   S_h: buffers at 128 h + 64 (u & 1) for step u; P_h(u) over its first 32
//   O_h: 256 + 128 h.
// A half's MMA warp keeps both of its buffers filled,
//   S(0) S(1) | PV(0) S(2) | PV(1) S(3) | ...
// so its softmax warps find the next step's scores ready when they hand over P
// and do not wait for the tensor core's latency.  A warp's MMAs complete in
// issue order: S(u + 2) overwrites P(u) only after PV(u) read it.  The core's
// queue is short and an issuing warp stalls on it, so with one warp for both
// halves the core stood still during that warp's waits (3,900 cycles per 128
// keys at head_dim 128); two warps cover each other's.
//
// Between items nothing drains: the TMA warp brings the next item's first K
// tile and, once the last scores are out, its Q; its first scores are computed
// while the softmax warps still write the last output (its first PV waits for
// that).  Counters run on across items, so every barrier's phases are seen in
// turn by whoever waits on it.
template <int DT, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    k_attend_packed(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap hmap,
                    const __grid_constant__ PackedArgs a) {
  using Sh = Shape<DP>;
  constexpr int NST = Sh::kStages;
  extern __shared__ unsigned char packed_raw[];
  unsigned char* base =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(packed_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + Sh::kBars);
  // barriers: scores full and P full (half, buffer); a half's last two PV of
  // an item done; Q full, Q free, O free (half); history full and read (half,
  // columns); per K stage full and empty, per V stage full, scrubbed and empty
  constexpr int kS = 0, kP = 4, kPv = 8, kQf = 12, kQe = 14, kOf = 16, kH = 18, kHr = 22, kKf = 26, kKe = kKf + NST,
                kVf = kKe + NST, kVc = kVf + NST, kVe = kVc + NST, kBarCount = kVe + NST;
  static_assert(kBarCount * 8 + 16 <= 512, "barriers");
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + kBarCount);
  volatile uint32_t* abort_flag = tslot + 1;
  volatile uint32_t* dirty_flag = tslot + 2;  // some V value was zeroed in this CTA
  volatile uint32_t* failed_flag = tslot + 3;  // the plan's status word at the start
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  asm volatile("griddepcontrol.launch_dependents;");  // the merge may take SMs that have nothing left to do
  const int G = a.G;
  const int first = a.cta_begin[blockIdx.x], last = a.cta_begin[blockIdx.x + 1];  // this CTA's items
  auto B = [&](int i) { return smem_addr(&bars[i]); };

  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tslot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  PackedItem head{};  // the TMA warp's: the first loads wait for one read of the list, not for two in turn
  if (warp == kTmaWarp) {
    head = read_item(a.first + blockIdx.x);
    for (const CUtensorMap* m : {&kmap, &qmap, &vmap})
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
    // arrivals per phase: P, O free and history read by the half's 4 warps, K / V empty by both MMA warps, else 1
#pragma unroll 1
    for (int i = lane; i < kBarCount; i += 32) {
      const bool by_half = (i >= kP && i < kP + 4) || (i >= kOf && i < kOf + 2) || (i >= kHr && i < kHr + 4);
      const int count = by_half ? 4 : (i >= kKe && i < kKe + NST) || i >= kVe ? 2 : 1;
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(B(i)), "r"(count) : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
    if (lane == 0) *abort_flag = *dirty_flag = 0u;
  }
  // The barriers and flags are the TMA warp's, which needs nothing of the
  // others': it only announces them and goes on to its loads.
  uint32_t tmem = 0u;
  if (warp == kTmaWarp) {
    __syncwarp();
    asm volatile("bar.arrive 1, %0;" ::"n"(kThreads) : "memory");
  } else {
    tc_before();
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
    tc_after();
    tmem = *tslot;
  }
  bool ok = true;
  auto fail = [&]() {
    *abort_flag = 1u;
    ok = false;
  };

  if (warp == kMmaWarp || warp == kMmaWarp + 1) {
    // --------------------------------------------------------- MMA issue
    // The whole warp runs its half's schedule, so addresses stay warp-uniform;
    // one elected lane issues.
    const int hf = warp - kMmaWarp;
    const uint32_t dq = desc_k_lo(smem_addr(base + hf * Sh::kTile)), dk = desc_k_lo(smem_addr(base + Sh::kK)),
                   dv = desc_mn_lo(smem_addr(base + Sh::kV));
    constexpr uint32_t kTileLo = Sh::kTile >> 4;
    const uint32_t s_tmem = tmem + uint32_t(hf * 128), o_tmem = tmem + uint32_t(256 + hf * 128);
    auto wait = [&](int i, uint32_t parity) {
      bool r = __all_sync(0xFFFFFFFFu, bar_try(B(i), parity));
      if (!r) {
        r = __all_sync(0xFFFFFFFFu, wait_for(B(i), parity));
        if (!r) fail();
      }
      tc_after();
      return r;
    };
    uint32_t tiles = 0, use0 = 0, use1 = 0;  // K / V tiles and uses of the score buffers so far
#pragma unroll 1
    for (int i = first; i < last && ok; ++i) {
      const PackedItem& it = a.items[i];
      const int n0 = it.steps0, n1 = it.steps1, nh = hf ? n1 : n0, n = (max(n0, n1) + 1) / 2;
      const uint32_t item_ph = uint32_t(i - first) & 1u;
      // scores of step u: keys 64 (u & 1).. (8 groups of 8 rows) of the K tile in stage st
      auto s_mmas = [&](int u, uint32_t st) {
        const uint32_t odd = uint32_t(u) & 1u;
        const uint32_t b = dk + st * kTileLo + odd * uint32_t(8 * 1024 >> 4);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
          mma_ss_lo(s_tmem + odd * SK, dq, b, uint32_t(((kk >> 2) * HALF_BYTES + (kk & 3) * 32) >> 4), kIdescS<DT>,
                    kk > 0 ? 1u : 0u);
        mma_commit(B(kS + 2 * hf + odd));
        if (u == nh - 1) mma_commit(B(kQe + hf));  // Q has been read
      };
      auto pv_mmas = [&](int u, uint32_t st) {
        const uint32_t odd = uint32_t(u) & 1u;
        const uint32_t b = dv + st * kTileLo + odd * uint32_t(8 * 1024 >> 4);
#pragma unroll
        for (int kk = 0; kk < SK / 16; ++kk)
          mma_ts_lo(o_tmem, s_tmem + odd * SK + uint32_t(kk * 8), b, uint32_t(kk * 2 * 1024 >> 4), kIdescO<DT, DP>,
                    (u > 0 || kk > 0) ? 1u : 0u);
        if (u >= nh - 2) mma_commit(B(kPv + 2 * hf + (u == nh - 1)));
      };
      if (!wait(kQf + hf, item_ph)) break;
      if (n > 0 && !wait(kKf + tiles % NST, (tiles / NST) & 1u)) break;
      if (elect_one()) {
        if (nh > 0) s_mmas(0, tiles % NST);
        if (nh > 1) s_mmas(1, tiles % NST);
        if (nh == 0) mma_commit(B(kQe + hf));
        if (n > 0) mma_commit(B(kKe + tiles % NST));
      }
      __syncwarp();
      // the first PV overwrites O, which the last item's output is read from
      if (i > first && !wait(kOf + hf, item_ph ^ 1u)) break;
      // a half without steps has its "last PV" here: its softmax warps, which
      // wait for nothing else, must not free O twice before the wait above
      if (nh == 0 && elect_one()) mma_commit(B(kPv + 2 * hf + 1));
      __syncwarp();
      // One round per tile; this half may need fewer steps than the other, but
      // returns every stage to the rings.
#pragma unroll 1
      for (int t = 0; t < n && ok; ++t) {
        const int u = 2 * t;
        const uint32_t x = tiles + uint32_t(t), st = x % NST, next = (x + 1) % NST;
        const bool more = t + 1 < n;
        if (!wait(kVc + st, (x / NST) & 1u)) break;
        if (more && !wait(kKf + next, ((x + 1) / NST) & 1u)) break;
        if (u < nh && !wait(kP + 2 * hf, (use0 + uint32_t(t)) & 1u)) break;
        if (elect_one()) {
          if (u < nh) pv_mmas(u, st);
          if (u + 2 < nh) s_mmas(u + 2, next);
        }
        __syncwarp();
        if (u + 1 < nh && !wait(kP + 2 * hf + 1, (use1 + uint32_t(t)) & 1u)) break;
        if (elect_one()) {
          if (u + 1 < nh) pv_mmas(u + 1, st);
          mma_commit(B(kVe + st));
          if (u + 3 < nh) s_mmas(u + 3, next);
          if (more) mma_commit(B(kKe + next));
        }
        __syncwarp();
      }
      tiles += uint32_t(n);
      use0 += uint32_t(nh + 1) / 2;
      use1 += uint32_t(nh) / 2;
    }
  } else if (warp == kTmaWarp) {
    // --------------------------------------------------------------- TMA
    if (lane == 0) {
      uint32_t kt = 0, vt = 0, slots = 0, hists = 0;  // K tiles, V tiles, V-ring slots, histories so far
      uint32_t held = 0, parity = 0;  // per V stage (4 bits): free 0, a tile 1, history columns 2 + e; loads of e modulo 2
      const uint32_t q_bytes = uint32_t(DP / 64) * uint32_t(a.half_rows) * 128u;
      auto wait = [&](int i, uint32_t parity) {
        if (ok && !wait_for(B(i), parity)) fail();
        return ok && *abort_flag == 0u;
      };
      auto load_k = [&](const PackedItem& it, int t) {
        const uint32_t st = kt % NST;
        if (kt >= NST && !wait(kKe + st, (kt / NST - 1) & 1u)) return false;
        bar_expect_tx(B(kKf + st), uint32_t(Sh::kTile));
#pragma unroll
        for (int x = 0; x < DP / 64; ++x)
          tma_tile(smem_addr(base + Sh::kK + st * Sh::kTile) + uint32_t(x * HALF_BYTES), &kmap, 64 * x, it.kvh,
                   it.k_start + (it.t_lo + t) * PK, B(kKf + st));
        ++kt;
        return true;
      };
      // V tiles and history columns share the V ring (an item takes four
      // history slots, a multiple of both ring lengths, so a V tile's stage
      // stays its count modulo the length); a slot is free once what it held
      // has been read: a tile by the MMA warps, history by the softmax warps
      auto slot_free = [&](uint32_t st, uint32_t next) {
        const uint32_t what = (held >> (4 * st)) & 15u;
        held = (held & ~(15u << (4 * st))) | (next << (4 * st));
        if (what == 0) return true;
        if (what == 1) return wait(kVe + st, ((vt + NST - 1 - st) / NST - 1) & 1u);
        return wait(kHr + what - 2, ((parity >> (what - 2)) & 1u) ^ 1u);
      };
      auto load_v = [&](const PackedItem& it, int t) {
        const uint32_t st = slots % NST;
        if (!slot_free(st, 1u)) return false;
        bar_expect_tx(B(kVf + st), uint32_t(Sh::kTile));
#pragma unroll
        for (int x = 0; x < DP / 64; ++x)
          tma_tile(smem_addr(base + Sh::kV + st * Sh::kTile) + uint32_t(x * HALF_BYTES), &vmap, 64 * x, it.kvh,
                   it.k_start + (it.t_lo + t) * PK, B(kVf + st));
        ++slots, ++vt;
        return true;
      };
      // Q of item i: the box is the group's heads by half_rows / G tokens; rows
      // behind the sequence belong to rows that are not kept
      auto load_q = [&](int i, const PackedItem& it) {
#pragma unroll 1
        for (int hf = 0; hf < 2; ++hf) {
          if (i > first && !wait(kQe + hf, uint32_t(i - first - 1) & 1u)) return false;
          bar_expect_tx(B(kQf + hf), q_bytes);
#pragma unroll
          for (int x = 0; x < DP / 64; ++x)
            tma_tile(smem_addr(base + hf * Sh::kTile) + uint32_t(x * HALF_BYTES), &qmap, 64 * x, it.kvh * G,
                     it.q_start + (it.row0 + hf * a.half_rows) / G, B(kQf + hf));
        }
        return true;
      };
      auto load_history = [&](const PackedItem& it) {
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {  // half e / 2, columns (e & 1) * DP / 2
          const uint32_t st = slots % NST;
          if (!slot_free(st, 2u + uint32_t(e))) return false;
          parity ^= 1u << e;
          bar_expect_tx(B(kH + e), uint32_t(DP / 64) * uint32_t(a.half_rows) * 128u);
#pragma unroll
          for (int x = 0; x < DP / 64; ++x)
            tma_tile(smem_addr(base + Sh::kV + st * Sh::kTile) + uint32_t(x * HALF_BYTES), &hmap,
                     (e & 1) * (DP / 2) + 32 * x, it.kvh * G, it.q_start + (it.row0 + (e >> 1) * a.half_rows) / G,
                     B(kH + e));
          ++slots;
        }
        ++hists;
        return true;
      };
      auto tiles_of = [&](const PackedItem& it) { return (max(it.steps0, it.steps1) + 1) / 2; };
      if (first < last) {
        if (tiles_of(head) > 0) load_k(head, 0);
        load_q(first, head);
      }
      int qs = first < last ? 1 : 0;
#pragma unroll 1
    for (int i = first; i < last && ok; ++i) {
        const PackedItem it = i == first ? head : read_item(a.items + i);
        const int n = tiles_of(it);
        bool run = true;
#pragma unroll 1
        for (int t = 0; t < n && run; ++t) run = load_v(it, t) && (t + 1 == n || load_k(it, t + 1));
        if (run && i + 1 < last) {
          const PackedItem up = read_item(a.items + i + 1);
          run = (tiles_of(up) == 0 || load_k(up, 0)) && load_q(i + 1, up);
          qs += run;
        }
        if (run && a.hist_o && it.part_row < 0) run = load_history(it);
        if (!run) break;
      }
      // no copy in flight when the CTA ends: wait (bounded) for the last load
      // on every barrier; on the normal path they have all been consumed
#pragma unroll 1
      for (uint32_t x = kt > NST ? kt - NST : 0; x < kt; ++x) wait_for(B(kKf + x % NST), (x / NST) & 1u);
#pragma unroll 1
      for (uint32_t x = vt > NST ? vt - NST : 0; x < vt; ++x) wait_for(B(kVf + x % NST), (x / NST) & 1u);
      if (qs)
#pragma unroll 1
        for (int hf = 0; hf < 2; ++hf) wait_for(B(kQf + hf), uint32_t(qs - 1) & 1u);
      if (hists)
#pragma unroll 1
        for (int e = 0; e < 4; ++e) wait_for(B(kH + e), (hists - 1) & 1u);
    }
    __syncwarp();
  } else if (warp == kScrubWarp) {
    // ----------------------------------------------------------- V scrub
    if (lane == 0) *failed_flag = *static_cast<const volatile uint32_t*>(a.status);
    uint32_t vt = 0;
#pragma unroll 1
    for (int i = first; i < last && ok; ++i) {
      const PackedItem& it = a.items[i];
      const int n = (max(it.steps0, it.steps1) + 1) / 2, lo_vis = it.lo_vis, hi_vis = it.hi_vis;
#pragma unroll 1
      for (int t = 0; t < n; ++t, ++vt) {
        const uint32_t st = vt % NST;
        if (!__all_sync(0xFFFFFFFFu, wait_for(B(kVf + st), (vt / NST) & 1u))) {
          fail();
          break;
        }
        // rows [lo, hi) of the tile: seen by some rows of the item only; rows from hi on: by none
        const int lo = max(0, min(PK, lo_vis - t * PK)), hi = max(0, min(PK, hi_vis - t * PK));
        if (lo < PK) {
          unsigned char* tile = base + Sh::kV + st * Sh::kTile;
#pragma unroll 1
          for (int x = 0; x < DP / 64; ++x, tile += HALF_BYTES) {
            uint4* p = reinterpret_cast<uint4*>(tile);  // 8 chunks of 16 bytes per row, swizzled within the row
            uint32_t top = 0u;
#pragma unroll 4
            for (int c = 8 * lo + lane; c < 8 * hi; c += 32) {
              const uint4 v = p[c];
              top = __vmaxu2(__vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu),
                                      __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu)), top);
            }
            const bool bad = max(top & 0xFFFFu, top >> 16) >= kNonFinite<DT>;
            if (__any_sync(0xFFFFFFFFu, bad)) {
              *dirty_flag = 1u;
#pragma unroll 1
              for (int c = 8 * lo + lane; c < 8 * hi; c += 32) {
                const uint4 v = p[c];
                p[c] = make_uint4(v.x & ~nonfinite_mask<DT>(v.x), v.y & ~nonfinite_mask<DT>(v.y),
                                  v.z & ~nonfinite_mask<DT>(v.z), v.w & ~nonfinite_mask<DT>(v.w));
              }
            }
#pragma unroll 1
            for (int c = 8 * hi + lane; c < 8 * PK; c += 32) p[c] = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_async_smem();
        }
        __syncwarp();
        arrive_lane0(B(kVc + st), lane);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int hf = warp >> 2;
    const int row = (warp & 3) * 32 + lane;  // packed row of the half
    const uint32_t lane_q = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_cols = tmem + lane_q + uint32_t(hf * 128);
    const uint32_t o_cols = tmem + lane_q + uint32_t(256 + hf * 128);
    // phases so far, one bit each: the score buffers (0, 1), the last PV and
    // the one before (2, 3), the history (4); V tiles modulo the ring (5, 6)
    uint32_t bits = 0;
#pragma unroll 1
    for (int i = first; i < last && ok; ++i) {
      int nh, lim;  // the half's steps; the row's visible keys, from the item's first tile
      bool idle;    // no row of the warp's: it only hands its part of P over
      {
        const PackedItem it = read_item(a.items + i);
        nh = hf ? it.steps1 : it.steps0;
        const int jt = int((uint32_t(row) * a.g_magic) >> 16);  // row / G
        const int n_rows = min(a.half_rows, it.rows - hf * a.half_rows);
        // lanes without a row mask nothing: their scores and output are never
        // kept, and a few of them must not send the warp through the masks
        lim = row < n_rows ? key_limit(a, it, (it.row0 + hf * a.half_rows) / G + jt) - it.t_lo * PK : 1 << 30;
        idle = (warp & 3) * 32 >= n_rows;
        const uint32_t tiles = uint32_t((max(it.steps0, it.steps1) + 1) / 2);
        bits = (bits & 31u) | ((((bits >> 5) + tiles) & 3u) << 5);
      }
      float m = -INFINITY, l = 0.0f;
      // Each phase of a step is a chain of latencies (TMEM, barriers), so the
      // next step's barrier is tried before the second half of the exponentials
      // and its scores are requested right after them, to arrive behind the end
      // of this step.
      float sv[SK];
      auto request = [&](int u) {
        tc_after();
        tmem_load32_async(s_cols + (u & 1) * SK, sv);
        tmem_load32_async(s_cols + (u & 1) * SK + 32, sv + 32);
      };
      auto s_phase = [&](int u) { return ((bits >> (u & 1)) ^ uint32_t(u >> 1)) & 1u; };
      // votes keep the warp together for the TMEM accesses
      auto scores_full = [&](int u, bool tried) {
        if (__all_sync(0xFFFFFFFFu, tried)) return true;
        const bool r = __all_sync(0xFFFFFFFFu, wait_for(B(kS + 2 * hf + (u & 1)), s_phase(u)));
        if (!r) fail();
        return r;
      };
      bool before_seen = false;  // the last PV but one of this item
#pragma unroll 1
      for (int u = 0; idle && u < nh && scores_full(u, false); ++u) arrive_lane0(B(kP + 2 * hf + (u & 1)), lane);
      if (!idle && nh > 0 && scores_full(0, false)) request(0);
#pragma unroll 1
      for (int u = 0; !idle && u < nh && ok; ++u) {
        const int buf = u & 1;
        tmem_load_wait();
        tmem_regs_after_wait(sv);
        tmem_regs_after_wait(sv + 32);
        const int vis = lim - u * SK;
        if (__any_sync(0xFFFFFFFFu, vis < SK)) {
#pragma unroll
          for (int j = 0; j < SK; ++j)
            if (j >= vis) sv[j] = -INFINITY;
        }
        float mx[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) mx[c] = max2_nan(sv[c], sv[8 + c]);
#pragma unroll
        for (int j = 16; j < SK; j += 16)
#pragma unroll
          for (int c = 0; c < 8; ++c) mx[c] = max3_nan(mx[c], sv[j + c], sv[j + 8 + c]);
        const float top = max3_nan(max3_nan(mx[0], mx[1], mx[2]), max3_nan(mx[3], mx[4], mx[5]),
                                   max2_nan(mx[6], mx[7]));
        const float mt = fmaf(top, a.scale_log2, -kRaise<DT>);
        const bool move = mt > m + 8.0f;
        const float mn = move ? mt : m;
        const float alpha = move ? exp2f(m - mn) : 1.0f;  // 0 on a row's first visible step
        // a row that has seen no key yet keeps m = -inf: its scores are all -inf
        // and must not give inf - inf
        const float nm = mn == -INFINITY ? 0.0f : -mn;
        const float2 sc2 = make_float2(a.scale_log2, a.scale_log2), nm2 = make_float2(nm, nm);
        float2 ls[4] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f),
                        make_float2(0.0f, 0.0f)};
        auto exponentiate = [&](int ch) {
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int k0 = ch * 32 + 2 * j;
            const float2 x = __ffma2_rn(make_float2(sv[k0], sv[k0 + 1]), sc2, nm2);
            // a quarter of the exponentials on the FMA pipes, the others on the
            // special-function unit, which alone would take 8 cycles each (16,383
            // queries of 64: 800 us; an eighth 814, three eighths 845)
            const float2 p = j % 4 == 3 ? exp2_fma(x) : make_float2(fast_exp2(x.x), fast_exp2(x.y));
            ls[j & 3] = __fadd2_rn(ls[j & 3], p);
            w[j] = pack2<DT>(p.x, p.y);
          }
          tmem_store16(s_cols + buf * SK + ch * 16, w);
        };
        exponentiate(0);
        const bool next = u + 1 < nh;
        const bool tried = next && bar_try(B(kS + 2 * hf + (buf ^ 1)), s_phase(u + 1));
        exponentiate(1);
        if (next) {
          if (!scores_full(u + 1, tried)) break;
          request(u + 1);
        }
        const float2 l01 = __fadd2_rn(ls[0], ls[1]), l23 = __fadd2_rn(ls[2], ls[3]);
        float lsum = (l01.x + l01.y) + (l23.x + l23.y);
        if (!(mt < INFINITY)) lsum = __int_as_float(0x7FFFFFFF);  // a NaN or infinite score: the row is NaN
        if (u > 0 && __any_sync(0xFFFFFFFFu, move)) {
          // O_h's rows rescaled between PV_h(u - 1), which was issued before
          // S_h(u + 1) and so is over, and PV_h(u), which waits for P_h(u)
          if (!next) {
            if (!__all_sync(0xFFFFFFFFu, wait_for(B(kPv + 2 * hf), (bits >> 3) & 1u))) {
              fail();
              break;
            }
            before_seen = true;
          }
          tc_after();
#pragma unroll 1
          for (int ch = 0; ch < DP / 32; ++ch) {
            float ov[32];
            tmem_load32(o_cols + ch * 32, ov);
#pragma unroll
            for (int j = 0; j < 32; ++j) ov[j] *= alpha;
            tmem_store32(o_cols + ch * 32, ov);
          }
        }
        tmem_store_wait();
        l = l * alpha + lsum;
        m = mn;
        tc_before();
        __syncwarp();
        arrive_lane0(B(kP + 2 * hf + buf), lane);
      }
      const PackedItem it = read_item(a.items + i);
      bits ^= uint32_t((nh + 1) / 2) & 1u;
      bits ^= (uint32_t(nh / 2) & 1u) << 1;
      if (ok) {
        bool r = nh < 2 || before_seen || wait_for(B(kPv + 2 * hf), (bits >> 3) & 1u);
        r = wait_for(B(kPv + 2 * hf + 1), (bits >> 2) & 1u) && r;
        if (!__all_sync(0xFFFFFFFFu, r)) fail();
        bits ^= nh > 1 ? 12u : 4u;
        tc_after();
      }
      if (!__all_sync(0xFFFFFFFFu, ok)) {
        ok = false;
        break;
      }
      // ---- the item's output
      const int row_tok = int((uint32_t(row) * a.g_magic) >> 16), row_head = row - row_tok * G;
      const int n_rows = min(a.half_rows, it.rows - hf * a.half_rows);  // the half's rows
      const bool have = row < n_rows;
      const int64_t q = int64_t(it.q_start) + (it.row0 + hf * a.half_rows) / G + row_tok;
      const int h = it.kvh * G + row_head;
      const bool whole = it.part_row < 0, hist = a.hist_o && whole;
      // the line (row of the output or of the partial buffers) of the half's
      // first row; row j is j / G lines of H and j % G lines further
      const int64_t line0 = whole ? q * a.H + h - (int64_t(row_tok) * a.H + row_head)
                                  : int64_t(it.part_row) + hf * a.half_rows;
      const int64_t line_tok = whole ? a.H : G;
      // normalisation and the history part's weights (base 2)
      float wo = 1.0f, wh = 0.0f;
      if (whole) {
        const float z = l > 0.0f || l != l ? m + log2f(l) : -INFINITY;  // NaN stays NaN
        wo = z == -INFINITY ? 0.0f : 1.0f / l;
        float lse2 = z;
        if (hist && have) {
          const float zh = __ldg(a.hist_lse + int64_t(h) * a.hist_lse_head + q) * 1.4426950408889634f;
          const float M = fmaxf(z, zh);
          if (z == -INFINITY && zh == -INFINITY) {  // (not M, which forgets a NaN)
            wo = 0.0f;
          } else {
            const float e0 = exp2f(z - M), e1 = exp2f(zh - M), inv = 1.0f / (e0 + e1);
            wo *= e0 * inv;
            wh = e1 * inv;
            lse2 = M + log2f(e0 + e1);
          }
        }
        if (have) a.lse[int64_t(h) * a.lse_head + q] = lse2 * 0.69314718055994531f;
      } else if (have) {
        reinterpret_cast<float2*>(a.part_ml)[int64_t(it.part_row) + hf * a.half_rows + row] = make_float2(m, l);
      }
      // The weighted rows leave through the warp's 4 KB, 128 bytes of each of
      // its 32 rows at a time (64 16-bit values or 32 f32), 16-byte chunks XORed
      // with the row, so that eight lanes write 128 consecutive bytes.
      const bool slow = *dirty_flag != 0u;
      const bool wide = !whole || a.out_f32;  // f32 rows
      unsigned char* dst = whole ? static_cast<unsigned char*>(a.out) : reinterpret_cast<unsigned char*>(a.part_o);
      const int esize = wide ? 4 : 2;
      unsigned char* stage = base + Sh::kStage + warp * 4096;
#pragma unroll 1
      for (int c0 = 0; c0 < DP; c0 += 32) {
        float ov[32];
        __syncwarp();
        if (nh > 0) tmem_load32(o_cols + c0, ov);
        if (c0 + 32 == DP) {  // O may be overwritten
          tc_before();
          __syncwarp();
          arrive_lane0(B(kOf + hf), lane);
        }
        if (nh == 0 || l == 0.0f) {  // nothing visible here (the MMA, if any, ran on P = 0)
#pragma unroll
          for (int j = 0; j < 32; ++j) ov[j] = 0.0f;
        }
        if (slow && have) {
          // the zeroed values of keys that this row does see
          const int hi = min(lim, nh * SK);
#pragma unroll 1
          for (int k = it.lo_vis; k < hi; ++k) {
            const uint16_t* vr = a.v + (int64_t(it.k_start) + it.t_lo * PK + k) * a.v_token +
                                 int64_t(it.kvh) * a.v_head + c0;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c0 + j < a.D) {
                const float x = dev::load_elem<DT>(vr, uint64_t(j));
                if (!(fabsf(x) <= 3.4e38f)) ov[j] += x;
              }
          }
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) ov[j] *= wo;
        if (hist) {
          constexpr int kCols = DP / 2;  // columns per history slot
          const int e = c0 / kCols;
          if (c0 % kCols == 0 && !__all_sync(0xFFFFFFFFu, wait_for(B(kH + 2 * hf + e), (bits >> 4) & 1u))) {
            fail();
            break;
          }
          // its slots are behind the V tiles so far (and earlier histories,
          // four slots each, a multiple of the ring's length)
          const uint32_t st = ((bits >> 5) + uint32_t(2 * hf + e)) % NST;
          if (wh != 0.0f) {
            const unsigned char* src = base + Sh::kV + st * Sh::kTile + ((c0 % kCols) / 32) * HALF_BYTES + row * 128;
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              const float4 x = *reinterpret_cast<const float4*>(src + ((d ^ (row & 7)) << 4));
              ov[4 * d] = fmaf(x.x, wh, ov[4 * d]);
              ov[4 * d + 1] = fmaf(x.y, wh, ov[4 * d + 1]);
              ov[4 * d + 2] = fmaf(x.z, wh, ov[4 * d + 2]);
              ov[4 * d + 3] = fmaf(x.w, wh, ov[4 * d + 3]);
            }
          }
          if ((c0 + 32) % kCols == 0) {  // read: back to the ring
            __syncwarp();
            arrive_lane0(B(kHr + 2 * hf + e), lane);
          }
        }
        // into the staging rows
        if (wide) {
#pragma unroll
          for (int d = 0; d < 8; ++d)
            *reinterpret_cast<float4*>(stage + lane * 128 + ((d ^ (lane & 7)) << 4)) =
                make_float4(ov[4 * d], ov[4 * d + 1], ov[4 * d + 2], ov[4 * d + 3]);
        } else {
#pragma unroll
          for (int d = 0; d < 4; ++d)
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((((c0 & 32) / 8 + d) ^ (lane & 7)) << 4)) =
                make_uint4(pack2<DT>(ov[8 * d], ov[8 * d + 1]), pack2<DT>(ov[8 * d + 2], ov[8 * d + 3]),
                           pack2<DT>(ov[8 * d + 4], ov[8 * d + 5]), pack2<DT>(ov[8 * d + 6], ov[8 * d + 7]));
          if (!(c0 & 32)) continue;
        }
        // and out: lane / 8 the row within four, lane % 8 the 16 bytes
        __syncwarp();
        const int c = (wide ? c0 : c0 - 32) + (lane & 7) * (16 / esize);  // first column of the 16 bytes
        const bool col_ok = c < a.D;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int rr = 4 * k + (lane >> 3), j = (warp & 3) * 32 + rr;  // row of the warp, of the half
          const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
          const int jt = int((uint32_t(j) * a.g_magic) >> 16);  // j / G
          const int64_t line = line0 + jt * line_tok + (j - jt * G);
          if (j < n_rows && col_ok) *reinterpret_cast<uint4*>(dst + (line * a.D + c) * esize) = v;
        }
      }
      bits ^= hist ? 16u : 0u;
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (*abort_flag && tid == 0) atomicOr(a.status, 1u);
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  if (*abort_flag | *failed_flag) fill_nan(&a, first, last);
}

// The merge of a split unit's partial rows (and the history part), one warp
// per row: with M the largest maximum, o = sum_p 2^(m_p - M) O_p / L,
// L = sum_p 2^(m_p - M) l_p, lse = (M + log2 L) ln 2.  It moves a few hundred
// kilobytes, so what counts is how many times it waits for memory: lane p takes
// part p's (m, l), and the first parts' rows are asked for at the same time.
// It is launched while k_attend_packed's last CTAs run and waits for them here.
// One part after the other and launched behind: the one-token case above 69 us
// instead of 66, the chunks 31 instead of 27.
template <int DT>
__global__ void __launch_bounds__(256) k_packed_combine(const PackedArgs a) {
  const PackedUnit u = a.units[blockIdx.x];
  const int lane = int(threadIdx.x) & 31;
  const int row = int(blockIdx.y) * 8 + (int(threadIdx.x) >> 5);
  const int G = a.G, r = u.row0 + row, tok = r / G, h = u.kvh * G + r - tok * G;
  const int64_t q = int64_t(u.q_start) + tok;
  const bool live = 4 * lane < a.D;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (row >= u.rows) return;
  float M = -INFINITY, L = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (a.hist_o) {  // a first part of sum 1
    const float4 x = live ? __ldg(reinterpret_cast<const float4*>(a.hist_o + (q * a.H + h) * a.D) + lane) : acc;
    M = __ldg(a.hist_lse + int64_t(h) * a.hist_lse_head + q) * 1.4426950408889634f;
    if (M != -INFINITY) {  // (a NaN stays in the sum)
      L = M == M ? 1.0f : M;
      acc = x;
    }
  }
  constexpr int kBatch = 8;
  for (int p0 = 0; p0 < u.parts; p0 += 32) {
    const int cnt = min(32, u.parts - p0);
    const int64_t first = int64_t(u.part_row) + int64_t(p0) * u.rows + row;
    float2 v = make_float2(-INFINITY, 0.0f);
    if (lane < cnt) v = reinterpret_cast<const float2*>(a.part_ml)[first + int64_t(lane) * u.rows];
    float w = 0.0f;  // this lane's part's weight
    for (int b = 0; b < cnt; b += kBatch) {
      float4 o[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (live && b + k < cnt)
          o[k] = reinterpret_cast<const float4*>(a.part_o + (first + int64_t(b + k) * u.rows) * a.D)[lane];
      if (b == 0) {
        float top = v.x;
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        const float to = fmaxf(M, top), nm = to == -INFINITY ? 0.0f : to;
        const float keep = M == -INFINITY ? 1.0f : exp2f(M - nm);  // (nothing yet: L and acc are 0)
        w = exp2f(v.x - nm);
        float l = w * v.y;
#pragma unroll
        for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, d);
        L = fmaf(L, keep, l);
        acc.x *= keep, acc.y *= keep, acc.z *= keep, acc.w *= keep;
        M = to;
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const float wk = __shfl_sync(0xFFFFFFFFu, w, b + k);
        if (live && b + k < cnt && (wk != 0.0f || wk != wk)) {
          acc.x = fmaf(wk, o[k].x, acc.x);
          acc.y = fmaf(wk, o[k].y, acc.y);
          acc.z = fmaf(wk, o[k].z, acc.z);
          acc.w = fmaf(wk, o[k].w, acc.w);
        }
      }
    }
  }
  const bool empty = L == 0.0f;
  const float inv = empty ? 0.0f : 1.0f / L;
  if (live) {
    const int64_t o_off = (q * a.H + h) * a.D + 4 * lane;
    acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
    if (a.out_f32)
      *reinterpret_cast<float4*>(static_cast<float*>(a.out) + o_off) = acc;
    else
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + o_off) =
          make_uint2(pack2<DT>(acc.x, acc.y), pack2<DT>(acc.z, acc.w));
  }
  if (lane == 0)
    a.lse[int64_t(h) * a.lse_head + q] = empty ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
}

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 enc = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  return enc;
}

// (tokens, heads, D) with strides in elements as (values, head, token); boxes
// of 128 bytes of values x `box_heads` heads x `box_tokens` tokens, 128-byte
// swizzled.  A key / value tile is one head by 128 tokens, half the rows of an
// item are G heads by 128 / G tokens.
bool make_map(CUtensorMap* m, const void* base, int dt, int64_t tokens, int heads, int D, int64_t token_stride,
              int64_t head_stride, int box_heads, int box_tokens) {
  const PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return false;
  const size_t es = dtype_size(dt);
  const cuuint64_t dims[3] = {cuuint64_t(D), cuuint64_t(heads), cuuint64_t(tokens)};
  // a dimension of one element has no stride: give it a valid one
  const cuuint64_t strides[2] = {cuuint64_t(heads > 1 ? head_stride : D) * es,
                                 cuuint64_t(tokens > 1 ? token_stride : int64_t(D) * heads) * es};
  const cuuint32_t box[3] = {uint32_t(128 / es), uint32_t(box_heads), uint32_t(box_tokens)};
  const cuuint32_t estr[3] = {1u, 1u, 1u};
  const CUtensorMapDataType type = dt == F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dt == BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(m, type, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Maps {
  CUtensorMap q, k, v, h;
};

template <int DT, int DP>
cudaError_t launch_shape(const Maps& m, const PackedArgs& a, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(k_attend_packed<DT, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Shape<DP>::kSmem);
  if (e != cudaSuccess) return e;
  k_attend_packed<DT, DP><<<unsigned(a.n_ctas), kThreads, Shape<DP>::kSmem, s>>>(m.q, m.k, m.v, m.h, a);
  e = cudaGetLastError();
  if (e != cudaSuccess || a.n_units == 0) return e;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.n_units), unsigned((a.max_unit_rows + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cfg.attrs = &early, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_packed_combine<DT>, a);
}

}  // namespace

bool launch_attend_packed(PackedArgs a, int dtype, const void* k, int64_t q_tokens, int64_t k_tokens, int64_t k_token,
                          int64_t k_head, cudaStream_t s, cudaError_t* err) {
  *err = cudaSuccess;
  if (a.n_ctas == 0) return true;
  const int box_tokens = kPackedHalfRows / a.G;
  a.half_rows = a.G * box_tokens;
  a.g_magic = 65536u / uint32_t(a.G) + 1u;  // (j * g_magic) >> 16 = j / G for j < 128, G <= 128
  Maps m{};
  if (!make_map(&m.q, a.q, dtype, q_tokens, a.H, a.D, a.q_token, a.q_head, a.G, box_tokens)) return false;
  // no key at all: no item has a tile and the maps are never read
  if (k_tokens > 0 &&
      (!make_map(&m.k, k, dtype, k_tokens, a.H / a.G, a.D, k_token, k_head, 1, kPackedTileKeys) ||
       !make_map(&m.v, a.v, dtype, k_tokens, a.H / a.G, a.D, a.v_token, a.v_head, 1, kPackedTileKeys)))
    return false;
  if (a.hist_o && !make_map(&m.h, a.hist_o, F32, q_tokens, a.H, a.D, int64_t(a.H) * a.D, a.D, a.G, box_tokens))
    return false;
  // head_dim up to 64 in tiles of its own width: 4,096 queries, 24 heads of 64
  // take 94 us, padded to 128 114; four tokens over 20,000 keys 101 and 119
  if (dtype == BF16)
    *err = a.D <= 64 ? launch_shape<BF16, 64>(m, a, s) : launch_shape<BF16, 128>(m, a, s);
  else
    *err = a.D <= 64 ? launch_shape<F16, 64>(m, a, s) : launch_shape<F16, 128>(m, a, s);
  return true;
}

}  // namespace nkv
