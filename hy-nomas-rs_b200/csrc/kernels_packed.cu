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
// work item is up to 256 rows (two halves of 128) of one sequence and
// key/value head over a range of 128-key tiles; a plan made once per set of
// lengths lists the items, longest first, and splits the key range of long
// rows when there are too few items to fill the GPU (their partial rows are
// merged by k_packed_combine).
//
// Per tile: S_h = Q_h K^T and O_h += P_h V as tcgen05.mma (kind::f16, f32 in
// TMEM), P written over S_h in TMEM as the A operand, the running maximum
// moved only when a tile exceeds it by more than 8 (base 2).  Scores, maxima,
// sums and O stay in f32; P is rounded to the type of V because the tensor
// core takes both operands in one type (an error of half a step of that type
// per probability, the size of the output's own rounding); the sum uses the
// unrounded values.
//
// A key past a row's limit has P = 0, but 0 times an infinity or a NaN in its
// V row is a NaN: V tiles that some row of the item does not wholly see are
// scrubbed in shared memory first (rows past the sequence zeroed, non-finite
// values zeroed and remembered), and rows that do see such a value get it
// added to their output at the end.
//
// Every wait on an mbarrier gives up after 1 s, sets bit 0 of the plan's
// status word, frees the TMEM and returns.
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

constexpr int PQ = 128;             // rows per half (TMEM lanes)
constexpr int PK = kPackedTileKeys;  // keys per K / V tile
constexpr int SK = kPackedStepKeys;  // keys per softmax step
static_assert(PK == 128 && SK == 64, "");
// warps 0-7 softmax (half = warp / 4), 8-9 MMA issue (one per half), 10 TMA, 11 V scrub
constexpr int kSoftmaxWarps = 8, kMmaWarp = 8, kTmaWarp = 10, kScrubWarp = 11;
constexpr int kThreads = 384;

// Shared memory for head_dim <= DP: the two Q halves, then a ring of K / V
// tiles (K_0 V_0 K_1 V_1 ...).
template <int DP>
struct Shape {
  static constexpr int kTile = (DP / 64) * HALF_BYTES;  // 128 rows x DP 16-bit values
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr int kSmem = (2 + kStages) * kTile + 512 + 1024;
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
  const int64_t lim = a.block == 1 ? p + 1 : (p / a.block + 1) * a.block;
  return lim < it.k_len ? int(lim) : it.k_len;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return DT == BF16 ? dev::bf16x2_bits_nonnan(a, b) : dev::f16x2_bits_nonnan(a, b);
}

// 2^x on the FMA pipes: x = n + f with n the nearest integer (the low bits of x
// + 1.5 2^23), a degree-4 polynomial of 2^f on [-1/2, 1/2] (a fit of the least
// maximal relative error with the constant held at 1: 2.9e-6, a hundredth of
// P's rounding), n added to the exponent.  Below 2^-125 it stays at 2^-125: 0
// next to any row's sum.  x at most 2^7; a NaN is lost here and caught by the
// row maximum.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  x = make_float2(fmaxf(x.x, -125.0f), fmaxf(x.y, -125.0f));
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

// Non-finite 16-bit halves of w (exponent all ones).
template <int DT>
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t w) {
  constexpr uint32_t e = DT == BF16 ? 0x7F80u : 0x7C00u;
  uint32_t m = 0u;
  if ((w & e) == e) m |= 0xFFFFu;
  if ((w & (e << 16)) == (e << 16)) m |= 0xFFFF0000u;
  return m;
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
template <int DT, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    k_attend_packed(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const PackedArgs a) {
  using Sh = Shape<DP>;
  constexpr int NST = Sh::kStages;
  extern __shared__ unsigned char packed_raw[];
  unsigned char* base =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(packed_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* Qs = base;
  unsigned char* Rs = base + 2 * Sh::kTile;  // the ring
  // barriers: S full and P full (half, buffer); a half's last two PV done
  // (once each); then per ring stage: full, empty, scrubbed, scrub wanted.
  // A waiter sees every phase of a barrier in turn, never one early or late.
  uint64_t* bars = reinterpret_cast<uint64_t*>(Rs + NST * Sh::kTile);
  constexpr int kS = 0, kP = 4, kPv = 8, kFull = 12, kEmpty = kFull + NST, kClean = kFull + 2 * NST,
                kGo = kFull + 3 * NST;
  // tiles between two V tiles in the same stage, for the phases of the two
  // scrub barriers (a stage is scrubbed again only after its last use was
  // released, so neither side falls a phase behind)
  constexpr int kVPeriod = NST % 2 ? NST : NST / 2;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + kFull + 4 * NST);
  volatile uint32_t* abort_flag = tslot + 1;
  volatile uint32_t* dirty_flag = tslot + 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PackedItem it = a.items[blockIdx.x];
  const int G = a.G;
  auto B = [&](int i) { return smem_addr(&bars[i]); };

  const int n0 = it.steps0, n1 = it.steps1, nu = max(n0, n1);  // steps of the halves
  const int n = (nu + 1) / 2;                                  // K / V tiles
  const int first_partial = it.first_partial;  // tiles from this one on are not wholly visible to every row

  // the TMA thread's load of ring entry idx (K_t, then V_t)
  auto load_tile = [&](int idx) {
    const int st = idx % NST;
    bar_expect_tx(B(kFull + st), uint32_t(Sh::kTile));
    const int tok = it.k_start + (it.t_lo + (idx >> 1)) * PK;
#pragma unroll
    for (int x = 0; x < DP / 64; ++x)
      tma_tile(smem_addr(Rs + st * Sh::kTile) + uint32_t(x * HALF_BYTES), (idx & 1) ? &vmap : &kmap, 64 * x, it.kvh,
               tok, B(kFull + st));
    if ((idx & 1) && (idx >> 1) >= first_partial) bar_arrive(B(kGo + st));
  };

  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tslot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 32 * kTmaWarp) {
    for (int i = 0; i < 4; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(B(kS + i)) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(B(kP + i)), "r"(PQ / 32) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(B(kPv + i)) : "memory");
    }
    for (int i = 0; i < NST; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 32;" ::"r"(B(kClean + i)) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(B(kGo + i)) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(B(kFull + i)) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 2;" ::"r"(B(kEmpty + i)) : "memory");  // both MMA warps
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *abort_flag = 0u;
    *dirty_flag = 0u;
    // the first K tile sets out beside Q; the others follow once Q has landed
    if (n > 0) load_tile(0);
  }
  // Q: each softmax warp loads its 32 packed rows, consecutive lanes along a
  // row (a row per thread would touch 32 lines with every load), zeros past the
  // item's rows and past head_dim
  if (warp < kSoftmaxWarps) {
    unsigned char* Qh = Qs + (warp >> 2) * Sh::kTile;
    constexpr int kLanes = DP / 8, kRows = 32 / kLanes;  // lanes per row, rows per round
    const int c = lane % kLanes;
    constexpr int kBatch = 8;  // loads in flight per lane
#pragma unroll
    for (int i0 = 0; i0 < 32; i0 += kRows * kBatch) {
      uint4 v[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int j = warp * 32 + i0 + b * kRows + lane / kLanes;
        v[b] = make_uint4(0u, 0u, 0u, 0u);
        if (j < it.rows && 8 * c < a.D) {
          const int r = it.row0 + j, tok = G == 1 ? r : r / G;
          v[b] = __ldg(reinterpret_cast<const uint4*>(a.q + (int64_t(it.q_start) + tok) * a.q_token +
                                                      int64_t(it.kvh * G + r - tok * G) * a.q_head) + c);
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int j = warp * 32 + i0 + b * kRows + lane / kLanes;
        *reinterpret_cast<uint4*>(Qh + swz(j & 127, c)) = v[b];
      }
    }
    fence_async_smem();
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tslot;
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
    const int nh = hf ? n1 : n0;
    const uint32_t dq = desc_k_lo(smem_addr(Qs + hf * Sh::kTile)), dr_k = desc_k_lo(smem_addr(Rs)),
                   dr_v = desc_mn_lo(smem_addr(Rs));
    constexpr uint32_t kTileLo = Sh::kTile >> 4;
    const uint32_t s_tmem = tmem + uint32_t(hf * 128), o_tmem = tmem + uint32_t(256 + hf * 128);
    auto wait = [&](int i, uint32_t parity) {
      bool r = __all_sync(0xFFFFFFFFu, bar_try(B(i), parity));
      if (!r) {
        r = __all_sync(0xFFFFFFFFu, bar_wait(B(i), parity));
        if (!r) fail();
      }
      tc_after();
      return r;
    };
    // scores of step parity `odd` from ring stage st: keys 64 odd.. (8 groups of 8 rows)
    auto s_mmas = [&](uint32_t odd, uint32_t st) {
      const uint32_t b = dr_k + st * kTileLo + odd * uint32_t(8 * 1024 >> 4);
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
        mma_ss_lo(s_tmem + odd * SK, dq, b, uint32_t(((kk >> 2) * HALF_BYTES + (kk & 3) * 32) >> 4), kIdescS<DT>,
                  kk > 0 ? 1u : 0u);
      mma_commit(B(kS + 2 * hf + odd));
    };
    auto pv_mmas = [&](uint32_t odd, uint32_t st, uint32_t acc, int u) {
      const uint32_t b = dr_v + st * kTileLo + odd * uint32_t(8 * 1024 >> 4);
#pragma unroll
      for (int kk = 0; kk < SK / 16; ++kk)
        mma_ts_lo(o_tmem, s_tmem + odd * SK + uint32_t(kk * 8), b, uint32_t(kk * 2 * 1024 >> 4), kIdescO<DT, DP>,
                  kk > 0 ? 1u : acc);
      if (u >= nh - 2) mma_commit(B(kPv + 2 * hf + (u == nh - 1)));
    };
    // ring stage and phase of V_t; K_(t + 1) is the next
    uint32_t v_st = 1, v_ph = 0;
    if (nu > 0 && wait(kFull, 0)) {
      if (elect_one()) {
        if (nh > 0) s_mmas(0, 0);
        if (nh > 1) s_mmas(1, 0);
        mma_commit(B(kEmpty));
      }
      __syncwarp();
    }
    // One round per tile; this half may need fewer steps than the other, but
    // returns every stage to the ring.
    for (int t = 0; t < n && ok; ++t) {
      const int u = 2 * t;
      const uint32_t ph = uint32_t(t) & 1u;
      uint32_t kn_st = v_st + 1, kn_ph = v_ph;
      if (kn_st == NST) kn_st = 0, kn_ph ^= 1u;
      if (t >= first_partial) {
        if (!wait(kClean + v_st, uint32_t((t - first_partial) / kVPeriod) & 1u)) break;
      } else if (!wait(kFull + v_st, v_ph)) {
        break;
      }
      const bool more = t + 1 < n;
      if (more && !wait(kFull + kn_st, kn_ph)) break;
      if (u < nh && !wait(kP + 2 * hf, ph)) break;
      if (elect_one()) {
        if (u < nh) pv_mmas(0, v_st, t > 0 ? 1u : 0u, u);
        if (u + 2 < nh) s_mmas(0, kn_st);
      }
      __syncwarp();
      if (u + 1 < nh && !wait(kP + 2 * hf + 1, ph)) break;
      if (elect_one()) {
        if (u + 1 < nh) pv_mmas(1, v_st, 1u, u + 1);
        mma_commit(B(kEmpty + v_st));
        if (u + 3 < nh) s_mmas(1, kn_st);
        if (more) mma_commit(B(kEmpty + kn_st));
      }
      __syncwarp();
      v_st = kn_st + 1, v_ph = kn_ph;
      if (v_st == NST) v_st = 0, v_ph ^= 1u;
    }
  } else if (warp == kTmaWarp) {
    // --------------------------------------------------------------- TMA
    if (lane == 0 && n > 0) {
      int idx = 1;
      for (; idx < 2 * n; ++idx) {
        if (idx >= NST && !bar_wait(B(kEmpty + idx % NST), uint32_t(idx / NST - 1) & 1u)) {
          fail();
          break;
        }
        if (*abort_flag) break;
        load_tile(idx);
      }
      // no copy in flight when the CTA ends: wait (bounded) for the last
      // load of every stage; on the normal path they have all been consumed
      for (int u = max(0, idx - NST); u < idx; ++u) bar_wait(B(kFull + u % NST), uint32_t(u / NST) & 1u);
    }
    __syncwarp();
  } else if (warp >= kScrubWarp) {
    // ----------------------------------------------------------- V scrub
    if (a.hist_o && it.part_row < 0) {
      // the history rows that the end of the item reads, brought to L2
      for (int i = lane; i < it.rows; i += 32) {
        const int r = it.row0 + i, tok = r / G;
        const float* src = a.hist_o + ((int64_t(it.q_start) + tok) * a.H + it.kvh * G + r - tok * G) * a.D;
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(a.D * 4) : "memory");
      }
    }
    for (int t = first_partial; t < n; ++t) {
      const int idx = 2 * t + 1, st = idx % NST;
      // the load was issued, so the stage's earlier phases are over: without
      // that its full barrier could still answer for the phase before them
      if (!bar_wait(B(kGo + st), uint32_t((t - first_partial) / kVPeriod) & 1u) ||
          !bar_wait(B(kFull + st), uint32_t(idx / NST) & 1u)) {
        fail();
        break;
      }
      const int left = it.k_len - (it.t_lo + t) * PK;  // rows of the tile that are keys
      bool bad = false;
      // whole 16-byte chunks, consecutive lanes on consecutive chunks, eight in flight
      uint4* tile = reinterpret_cast<uint4*>(Rs + st * Sh::kTile);
      for (int c0 = lane; c0 < Sh::kTile / 16; c0 += 32 * 8) {
        uint4 v[8];
#pragma unroll
        for (int b = 0; b < 8; ++b) v[b] = tile[c0 + 32 * b];
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          const int c = c0 + 32 * b, row = (c >> 3) & 127;  // 8 chunks per row of a 64-column half
          const uint32_t m0 = nonfinite_mask<DT>(v[b].x), m1 = nonfinite_mask<DT>(v[b].y),
                         m2 = nonfinite_mask<DT>(v[b].z), m3 = nonfinite_mask<DT>(v[b].w);
          if (row >= left) {
            tile[c] = make_uint4(0u, 0u, 0u, 0u);
          } else if (m0 | m1 | m2 | m3) {
            bad = true;
            tile[c] = make_uint4(v[b].x & ~m0, v[b].y & ~m1, v[b].z & ~m2, v[b].w & ~m3);
          }
        }
      }
      if (bad) *dirty_flag = 1u;
      fence_async_smem();
      bar_arrive(B(kClean + st));
      if (*abort_flag) break;
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int hf = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const int nh = hf ? n1 : n0;
    const uint32_t lane_q = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_cols = tmem + lane_q + uint32_t(hf * 128);
    const uint32_t o_cols = tmem + lane_q + uint32_t(256 + hf * 128);
    const bool have = hf * PQ + row < it.rows;
    const int r = it.row0 + hf * PQ + row, tok = have ? r / G : 0;
    // visible keys, counted from the item's first tile
    const int lim = have ? key_limit(a, it, tok) - it.t_lo * PK : 0;
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
    // votes keep the warp together for the TMEM accesses
    auto scores_full = [&](int u, bool tried) {
      if (__all_sync(0xFFFFFFFFu, tried)) return true;
      const bool r = __all_sync(0xFFFFFFFFu, bar_wait(B(kS + 2 * hf + (u & 1)), uint32_t(u >> 1) & 1u));
      if (!r) fail();
      return r;
    };
    if (nh > 0 && scores_full(0, false)) request(0);
    for (int u = 0; u < nh && ok; ++u) {
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
      const float mt = max3_nan(max3_nan(mx[0], mx[1], mx[2]), max3_nan(mx[3], mx[4], mx[5]),
                                max2_nan(mx[6], mx[7])) * a.scale_log2;
      const bool move = mt > m + 8.0f;
      const float mn = move ? mt : m;
      const float alpha = move ? exp2f(m - mn) : 1.0f;  // 0 on a row's first visible step
      // a row that has seen no key yet keeps m = -inf: its scores are all -inf
      // and must give 0, not inf - inf
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
          // special-function unit, which alone would take 8 cycles each
          const float2 p = j % 4 == 3 ? exp2_fma(x) : make_float2(fast_exp2(x.x), fast_exp2(x.y));
          ls[j & 3] = __fadd2_rn(ls[j & 3], p);
          w[j] = pack2<DT>(p.x, p.y);
        }
        tmem_store16(s_cols + buf * SK + ch * 16, w);
      };
      exponentiate(0);
      const bool next = u + 1 < nh;
      const bool tried = next && bar_try(B(kS + 2 * hf + (buf ^ 1)), uint32_t((u + 1) >> 1) & 1u);
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
        if (!next && !__all_sync(0xFFFFFFFFu, bar_wait(B(kPv + 2 * hf), 0))) {
          fail();
          break;
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
    if (ok && nh > 0) {
      // the half's last PV is done, and with it everything that read its Q
      if (!__all_sync(0xFFFFFFFFu, bar_wait(B(kPv + 2 * hf + 1), 0))) fail();
      tc_after();
    }
    if (__all_sync(0xFFFFFFFFu, ok && *abort_flag == 0u)) {
      const int64_t q = int64_t(it.q_start) + tok;
      const int h = it.kvh * G + (r - tok * G);
      const bool whole = it.part_row < 0;
      // normalisation and the history part's weights (base 2)
      float wo = 1.0f, wh = 0.0f;
      if (whole) {
        const float z = l > 0.0f || l != l ? m + log2f(l) : -INFINITY;  // NaN stays NaN
        wo = z == -INFINITY ? 0.0f : 1.0f / l;
        float lse2 = z;
        if (a.hist_o && have) {
          const float zh = __ldg(a.hist_lse + int64_t(h) * a.hist_lse_head + q) * 1.4426950408889634f;
          const float M = fmaxf(z, zh);
          if (M == -INFINITY) {
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
        reinterpret_cast<float2*>(a.part_ml)[int64_t(it.part_row) + hf * PQ + row] = make_float2(m, l);
      }
      // The weighted rows leave through shared memory, DP / 2 columns at a
      // time, so that consecutive lanes write consecutive bytes of a row: the
      // warp's 32 rows in its quarter of the half's Q tile, 16-byte chunks
      // XORed with the row.
      constexpr int kCols = DP / 2, kLanes = kCols / 4, kRows = 32 / kLanes, kBatch = 8;
      unsigned char* stage = Qs + hf * Sh::kTile + (warp & 3) * (32 * kCols * 4);
      const bool slow = *dirty_flag != 0u;
      const int n_rows = min(32, it.rows - hf * PQ - (warp & 3) * 32);  // the warp's rows
      const int64_t my_off = whole ? (q * a.H + h) * a.D : (int64_t(it.part_row) + hf * PQ + row) * a.D;
      const int c = lane % kLanes;
#pragma unroll 1
      for (int c0 = 0; c0 < DP; c0 += kCols) {
#pragma unroll 1
        for (int ch = 0; ch < kCols; ch += 32) {
          float ov[32];
          __syncwarp();
          if (nh > 0) tmem_load32(o_cols + c0 + ch, ov);
          if (nh == 0 || l == 0.0f) {  // nothing visible here (the MMA, if any, ran on P = 0)
#pragma unroll
            for (int j = 0; j < 32; ++j) ov[j] = 0.0f;
          }
          if (slow && have) {
            // the scrubbed values of keys that this row does see
            const int hi = min(lim, nh * SK);
            for (int k = first_partial * PK; k < hi; ++k) {
              const uint16_t* vr = a.v + (int64_t(it.k_start) + it.t_lo * PK + k) * a.v_token +
                                   int64_t(it.kvh) * a.v_head + c0 + ch;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (c0 + ch + j < a.D) {
                  const float x = dev::load_elem<DT>(vr, uint64_t(j));
                  if (!(fabsf(x) <= 3.4e38f)) ov[j] += x;
                }
            }
          }
#pragma unroll
          for (int d = 0; d < 8; ++d)
            *reinterpret_cast<float4*>(stage + lane * (kCols * 4) + (((ch / 4 + d) ^ (lane & 7)) << 4)) =
                make_float4(ov[4 * d] * wo, ov[4 * d + 1] * wo, ov[4 * d + 2] * wo, ov[4 * d + 3] * wo);
        }
        __syncwarp();
        for (int i0 = 0; i0 < n_rows; i0 += kRows * kBatch) {
          float4 o[kBatch], x[kBatch];
          float w[kBatch];
          int64_t off[kBatch];
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            const int j = i0 + b * kRows + lane / kLanes;
            off[b] = __shfl_sync(0xFFFFFFFFu, my_off, j) + c0 + 4 * c;
            w[b] = __shfl_sync(0xFFFFFFFFu, wh, j);
            if (j >= n_rows || c0 + 4 * c >= a.D) off[b] = -1;
            x[b] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (off[b] >= 0 && w[b] != 0.0f) x[b] = __ldg(reinterpret_cast<const float4*>(a.hist_o + off[b]));
            o[b] = *reinterpret_cast<const float4*>(stage + j * (kCols * 4) + ((c ^ (j & 7)) << 4));
          }
          if (a.hist_o) {
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
              if (w[b] != 0.0f) {
                o[b].x = fmaf(x[b].x, w[b], o[b].x);
                o[b].y = fmaf(x[b].y, w[b], o[b].y);
                o[b].z = fmaf(x[b].z, w[b], o[b].z);
                o[b].w = fmaf(x[b].w, w[b], o[b].w);
              }
          }
          if (!whole || a.out_f32) {
            float* dst = whole ? static_cast<float*>(a.out) : a.part_o;
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
              if (off[b] >= 0) *reinterpret_cast<float4*>(dst + off[b]) = o[b];
          } else {
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
              if (off[b] >= 0)
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + off[b]) =
                    make_uint2(pack2<DT>(o[b].x, o[b].y), pack2<DT>(o[b].z, o[b].w));
          }
        }
        __syncwarp();
      }
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (*abort_flag && tid == 0) atomicOr(a.status, 1u);
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// The merge of a split unit's partial rows (and the history part), one warp
// per row: with M the largest maximum, o = sum_p 2^(m_p - M) O_p / L,
// L = sum_p 2^(m_p - M) l_p, lse = (M + log2 L) ln 2.
template <int DT>
__global__ void __launch_bounds__(256) k_packed_combine(const PackedArgs a) {
  const PackedUnit u = a.units[blockIdx.x];
  const int lane = int(threadIdx.x) & 31;
  const int row = int(blockIdx.y) * 8 + (int(threadIdx.x) >> 5);
  if (row >= u.rows) return;
  const int G = a.G, r = u.row0 + row, tok = r / G, h = u.kvh * G + r - tok * G;
  const int64_t q = int64_t(u.q_start) + tok;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
  float M = -INFINITY;
  for (int p = 0; p < u.parts; ++p) M = fmaxf(M, ml[int64_t(u.part_row) + int64_t(p) * u.rows + row].x);
  float zh = -INFINITY;
  if (a.hist_o) zh = __ldg(a.hist_lse + int64_t(h) * a.hist_lse_head + q) * 1.4426950408889634f;
  M = fmaxf(M, zh);
  const float nm = M == -INFINITY ? 0.0f : M;
  const bool live = 4 * lane < a.D;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float L = 0.0f;
  if (a.hist_o) {
    const float w = exp2f(zh - nm);
    L = w;
    if (live && w != 0.0f) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(a.hist_o + (q * a.H + h) * a.D) + lane);
      acc = make_float4(w * x.x, w * x.y, w * x.z, w * x.w);
    }
  }
  for (int p = 0; p < u.parts; ++p) {
    const int64_t pr = int64_t(u.part_row) + int64_t(p) * u.rows + row;
    const float2 v = ml[pr];
    const float w = exp2f(v.x - nm);
    L = fmaf(w, v.y, L);
    if (live && (w != 0.0f || w != w)) {
      const float4 o = reinterpret_cast<const float4*>(a.part_o + pr * a.D)[lane];
      acc.x = fmaf(w, o.x, acc.x);
      acc.y = fmaf(w, o.y, acc.y);
      acc.z = fmaf(w, o.z, acc.z);
      acc.w = fmaf(w, o.w, acc.w);
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

// (tokens, heads, D) with strides in elements as (values, head, token), boxes
// of 64 values x 1 head x 128 tokens.
bool make_kv_map(CUtensorMap* m, const void* base, int dt, int64_t tokens, int heads, int D, int64_t token_stride,
                 int64_t head_stride) {
  const PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return false;
  const cuuint64_t dims[3] = {cuuint64_t(D), cuuint64_t(heads), cuuint64_t(tokens)};
  // a dimension of one element has no stride: give it a valid one
  const cuuint64_t strides[2] = {cuuint64_t(heads > 1 ? head_stride : D) * 2,
                                 cuuint64_t(tokens > 1 ? token_stride : int64_t(D) * heads) * 2};
  const cuuint32_t box[3] = {64u, 1u, uint32_t(PK)};
  const cuuint32_t estr[3] = {1u, 1u, 1u};
  return enc(m, dt == BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
             const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DT, int DP>
cudaError_t launch_shape(const CUtensorMap& km, const CUtensorMap& vm, const PackedArgs& a, cudaStream_t s) {
  cudaError_t e = cudaFuncSetAttribute(k_attend_packed<DT, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::kSmem);
  if (e != cudaSuccess) return e;
  k_attend_packed<DT, DP><<<unsigned(a.n_items), kThreads, Shape<DP>::kSmem, s>>>(km, vm, a);
  e = cudaGetLastError();
  if (e != cudaSuccess || a.n_units == 0) return e;
  k_packed_combine<DT><<<dim3(unsigned(a.n_units), unsigned((a.max_unit_rows + 7) / 8)), 256, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

bool launch_attend_packed(const PackedArgs& a, int dtype, const void* k, int64_t k_tokens, int64_t k_token,
                          int64_t k_head, int kv_heads, cudaStream_t s, cudaError_t* err) {
  *err = cudaSuccess;
  if (a.n_items == 0) return true;
  CUtensorMap km{}, vm{};
  if (k_tokens > 0) {  // no key at all: no item has a tile and the maps are never read
    if (!make_kv_map(&km, k, dtype, k_tokens, kv_heads, a.D, k_token, k_head) ||
        !make_kv_map(&vm, a.v, dtype, k_tokens, kv_heads, a.D, a.v_token, a.v_head))
      return false;
  }
  if (dtype == BF16)
    *err = a.D <= 64 ? launch_shape<BF16, 64>(km, vm, a, s) : launch_shape<BF16, 128>(km, vm, a, s);
  else
    *err = a.D <= 64 ? launch_shape<F16, 64>(km, vm, a, s) : launch_shape<F16, 128>(km, vm, a, s);
  return true;
}

}  // namespace nkv
