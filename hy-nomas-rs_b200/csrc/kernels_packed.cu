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

constexpr int PQ = 128;  // rows per half (TMEM lanes)
constexpr int PK = kPackedTileKeys;
static_assert(PK == 128, "");
// warps 0-7 softmax (half = warp / 4), 8 MMA issue, 9 TMA, 10-11 V scrub
constexpr int kSoftmaxWarps = 8, kMmaWarp = 8, kTmaWarp = 9, kScrubWarp = 10, kScrubWarps = 2;
constexpr int kThreads = 384;
// Registers after the split: 256 x 208 + 128 x 88 = 64,512 = 384 x 168.
constexpr int kRegsLaunch = 168, kRegsSoftmax = 208, kRegsOther = 88;
static_assert(kRegsSoftmax * 32 * kSoftmaxWarps + kRegsOther * 128 <= kRegsLaunch * kThreads,
              "register split exceeds the launch's registers");

// Shared memory for head_dim <= DP: the two Q halves, then a ring of K / V
// tiles (K_0 V_0 K_1 V_1 ...).
template <int DP>
struct Shape {
  static constexpr int kTile = (DP / 64) * HALF_BYTES;  // 128 rows x DP 16-bit values
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr int kSmem = (2 + kStages) * kTile + 512 + 1024;
  static_assert(kSmem <= 232448, "shared memory");
};

// f32 accumulate, A and B both bf16 (1) or f16 (0); S: both K-major, N = 128
// keys.  O: B (V) MN-major, N = DP.
template <int DT>
constexpr uint32_t kIdescIn = (1u << 4) | (uint32_t(DT == BF16) << 7) | (uint32_t(DT == BF16) << 10) |
                              (uint32_t(PQ >> 4) << 24);
template <int DT>
constexpr uint32_t kIdescS = kIdescIn<DT> | (uint32_t(PK >> 3) << 17);
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

// Keys visible to token i (causal or not), as documented above.
__device__ __forceinline__ int key_limit(const PackedArgs& a, const PackedItem& it, int i) {
  if (!a.causal) return it.k_len;
  const int64_t p = int64_t(i) + it.k_len - it.q_len;
  if (p < 0) return 0;
  const int64_t lim = (p / a.block + 1) * a.block;
  return lim < it.k_len ? int(lim) : it.k_len;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return DT == BF16 ? dev::bf16x2_bits_nonnan(a, b) : dev::f16x2_bits_nonnan(a, b);
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
  // barriers: 0-1 S full (half), 2-3 P full (half), 4 O done, then per ring
  // stage: full, empty, scrubbed, scrub wanted
  uint64_t* bars = reinterpret_cast<uint64_t*>(Rs + NST * Sh::kTile);
  constexpr int kFull = 5, kEmpty = 5 + NST, kClean = 5 + 2 * NST, kGo = 5 + 3 * NST;
  // tiles between two V tiles in the same stage, for the phases of the two
  // scrub barriers (a stage is scrubbed again only after its last use was
  // released, so neither side falls a phase behind)
  constexpr int kVPeriod = NST % 2 ? NST : NST / 2;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + 5 + 4 * NST);
  volatile uint32_t* abort_flag = tslot + 1;
  volatile uint32_t* dirty_flag = tslot + 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PackedItem it = a.items[blockIdx.x];
  const int G = a.G;
  auto B = [&](int i) { return smem_addr(&bars[i]); };

  // tiles of this item that each half needs (limits grow with the row)
  auto half_tiles = [&](int hf) {
    const int rows = min(PQ, it.rows - hf * PQ);
    if (rows <= 0) return 0;
    const int lim = key_limit(a, it, (it.row0 + hf * PQ + rows - 1) / G);
    const int hi = min(it.t_hi, (lim + PK - 1) / PK);
    return max(0, hi - it.t_lo);
  };
  const int n0 = half_tiles(0), n1 = half_tiles(1), n = max(n0, n1);
  // tiles from this one on are not wholly visible to every row
  const int first_partial = max(0, key_limit(a, it, it.row0 / G) / PK - it.t_lo);

  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tslot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 32 * kTmaWarp) {
    for (int i = 0; i < 2; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(B(i)) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(B(2 + i)), "r"(PQ) : "memory");
    }
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(B(4)) : "memory");
    for (int i = 0; i < NST; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(B(kClean + i)), "r"(32 * kScrubWarps) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(B(kGo + i)) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(B(kFull + i)) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(B(kEmpty + i)) : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *abort_flag = 0u;
    *dirty_flag = 0u;
  }
  // Q: softmax thread j loads packed row j (zeros past the item's rows and
  // past head_dim)
  if (warp < kSoftmaxWarps) {
    unsigned char* Qh = Qs + (tid >> 7) * Sh::kTile;
    const bool have = tid < it.rows;
    const int r = it.row0 + tid, tok = r / G;
    const uint16_t* src = a.q + (int64_t(it.q_start) + tok) * a.q_token + int64_t(it.kvh * G + r - tok * G) * a.q_head;
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (have && 8 * c < a.D) v = __ldg(reinterpret_cast<const uint4*>(src) + c);
      *reinterpret_cast<uint4*>(Qh + swz(tid & 127, c)) = v;
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

  if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == kMmaWarp && n > 0) {
      // ------------------------------------------------------- MMA issue
      // The whole warp runs the schedule; one elected lane issues.
      const uint32_t dq = desc_k_lo(smem_addr(Qs)), dr_k = desc_k_lo(smem_addr(Rs)),
                     dr_v = desc_mn_lo(smem_addr(Rs));
      constexpr uint32_t kTileLo = Sh::kTile >> 4;
      auto wait = [&](int i, uint32_t parity) {
        int r = 1;
        if (lane == 0) r = bar_wait(B(i), parity) ? 1 : 0;
        r = __shfl_sync(0xFFFFFFFFu, r, 0);
        if (!r) fail();
        tc_after();
        return r != 0;
      };
      auto wait_full = [&](int idx) { return wait(kFull + idx % NST, uint32_t(idx / NST) & 1u); };
      auto issue_s = [&](int t, int hf) {
        if (elect_one()) {
          const uint32_t b = dr_k + uint32_t((2 * t) % NST) * kTileLo;
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            mma_ss_lo(tmem + uint32_t(hf * 128), dq + uint32_t(hf) * kTileLo, b,
                      uint32_t(((kk >> 2) * HALF_BYTES + (kk & 3) * 32) >> 4), kIdescS<DT>, kk > 0 ? 1u : 0u);
          mma_commit(B(hf));
        }
        __syncwarp();
      };
      auto issue_pv = [&](int t, int hf) {
        if (elect_one()) {
          const uint32_t b = dr_v + uint32_t((2 * t + 1) % NST) * kTileLo;
#pragma unroll
          for (int kk = 0; kk < PK / 16; ++kk)
            mma_ts_lo(tmem + uint32_t(256 + hf * 128), tmem + uint32_t(hf * 128 + kk * 8), b,
                      uint32_t(kk * 2 * 1024 >> 4), kIdescO<DT, DP>, (t > 0 || kk > 0) ? 1u : 0u);
        }
        __syncwarp();
      };
      auto release = [&](int idx) {
        if (elect_one()) mma_commit(B(kEmpty + idx % NST));
        __syncwarp();
      };
      if (wait_full(0)) {
        if (n0 > 0) issue_s(0, 0);
        if (n1 > 0) issue_s(0, 1);
        release(0);
      }
      for (int t = 0; t < n && ok; ++t) {
        if (__shfl_sync(0xFFFFFFFFu, int(*abort_flag), 0)) break;
        if (t >= first_partial) {
          if (!wait(kClean + (2 * t + 1) % NST, uint32_t((t - first_partial) / kVPeriod) & 1u)) break;
        } else if (!wait_full(2 * t + 1)) {
          break;
        }
        const bool more = t + 1 < n;
        if (t < n0) {
          if (!wait(2, uint32_t(t) & 1u)) break;
          issue_pv(t, 0);
        }
        if (more) {
          if (!wait_full(2 * t + 2)) break;
          if (t + 1 < n0) issue_s(t + 1, 0);
        }
        if (t < n1) {
          if (!wait(3, uint32_t(t) & 1u)) break;
          issue_pv(t, 1);
        }
        release(2 * t + 1);
        if (more) {
          if (t + 1 < n1) issue_s(t + 1, 1);
          release(2 * t + 2);
        }
      }
      if (elect_one()) mma_commit(B(4));
      __syncwarp();
    } else if (warp == kTmaWarp && n > 0) {
      // ------------------------------------------------------------- TMA
      if (lane == 0) {
        int idx = 0;
        for (; idx < 2 * n; ++idx) {
          const int st = idx % NST;
          if (idx >= NST && !bar_wait(B(kEmpty + st), uint32_t(idx / NST - 1) & 1u)) {
            fail();
            break;
          }
          if (*abort_flag) break;
          bar_expect_tx(B(kFull + st), uint32_t(Sh::kTile));
          const int tok = it.k_start + (it.t_lo + (idx >> 1)) * PK;
#pragma unroll
          for (int x = 0; x < DP / 64; ++x)
            tma_tile(smem_addr(Rs + st * Sh::kTile) + uint32_t(x * HALF_BYTES), (idx & 1) ? &vmap : &kmap, 64 * x,
                     it.kvh, tok, B(kFull + st));
          if ((idx & 1) && (idx >> 1) >= first_partial) bar_arrive(B(kGo + st));
        }
        // no copy in flight when the CTA ends: wait (bounded) for the last
        // load of every stage; on the normal path they have all been consumed
        for (int u = max(0, idx - NST); u < idx; ++u) bar_wait(B(kFull + u % NST), uint32_t(u / NST) & 1u);
      }
      __syncwarp();
    } else if (warp >= kScrubWarp && first_partial < n) {
      // --------------------------------------------------------- V scrub
      const int j = tid - 32 * kScrubWarp;
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
        // whole 16-byte chunks, consecutive threads on consecutive chunks
        for (int c = j; c < Sh::kTile / 16; c += 32 * kScrubWarps) {
          const int row = (c >> 3) & 127;  // 8 chunks per row of a 64-column half
          uint4* p = reinterpret_cast<uint4*>(Rs + st * Sh::kTile) + c;
          if (row >= left) {
            *p = make_uint4(0u, 0u, 0u, 0u);
          } else {
            uint4 v = *p;
            const uint32_t m0 = nonfinite_mask<DT>(v.x), m1 = nonfinite_mask<DT>(v.y), m2 = nonfinite_mask<DT>(v.z),
                           m3 = nonfinite_mask<DT>(v.w);
            if (m0 | m1 | m2 | m3) {
              bad = true;
              *p = make_uint4(v.x & ~m0, v.y & ~m1, v.z & ~m2, v.w & ~m3);
            }
          }
        }
        if (bad) *dirty_flag = 1u;
        fence_async_smem();
        bar_arrive(B(kClean + st));
        if (*abort_flag) break;
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
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
    for (int t = 0; t < nh; ++t) {
      // votes keep the warp together for the TMEM accesses
      if (!__all_sync(0xFFFFFFFFu, bar_wait(B(hf), uint32_t(t) & 1u))) {
        fail();
        break;
      }
      tc_after();
      float sv[PK];
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) tmem_load32_async(s_cols + ch * 32, sv + ch * 32);
      tmem_load_wait();
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) tmem_regs_after_wait(sv + ch * 32);
      const int vis = lim - t * PK;
      if (__any_sync(0xFFFFFFFFu, vis < PK)) {
#pragma unroll
        for (int j = 0; j < PK; ++j)
          if (j >= vis) sv[j] = -INFINITY;
      }
      float mx[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) mx[c] = fmaxf(sv[c], sv[8 + c]);
#pragma unroll
      for (int j = 16; j < PK; j += 16)
#pragma unroll
        for (int c = 0; c < 8; ++c) mx[c] = max3(mx[c], sv[j + c], sv[j + 8 + c]);
      const float mt =
          max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) * a.scale_log2;
      const bool move = mt > m + 8.0f;
      const float mn = move ? mt : m;
      const float alpha = move ? exp2f(m - mn) : 1.0f;  // 0 on a row's first visible tile
      // a row that has seen no key yet keeps m = -inf: its scores are all -inf
      // and must give 0, not inf - inf
      const float nm = mn == -INFINITY ? 0.0f : -mn;
      const float2 sc2 = make_float2(a.scale_log2, a.scale_log2), nm2 = make_float2(nm, nm);
      float2 ls[4] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f),
                      make_float2(0.0f, 0.0f)};
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int k0 = ch * 32 + 2 * j;
          const float2 x = __ffma2_rn(make_float2(sv[k0], sv[k0 + 1]), sc2, nm2);
          const float2 p = make_float2(fast_exp2(x.x), fast_exp2(x.y));
          ls[j & 3] = __fadd2_rn(ls[j & 3], p);
          w[j] = pack2<DT>(p.x, p.y);
        }
        tmem_store16(s_cols + ch * 16, w);
      }
      const float2 l01 = __fadd2_rn(ls[0], ls[1]), l23 = __fadd2_rn(ls[2], ls[3]);
      const float lsum = (l01.x + l01.y) + (l23.x + l23.y);
      if (t > 0 && __any_sync(0xFFFFFFFFu, move)) {
        // O_h's row rescaled; PV_h(t - 1) completed before S_h(t) did
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
      bar_arrive(B(2 + hf));
      if (__any_sync(0xFFFFFFFFu, *abort_flag != 0u)) {
        ok = false;
        break;
      }
    }
    if (ok && nh > 0) {
      if (!__all_sync(0xFFFFFFFFu, bar_wait(B(4), 0))) fail();
      tc_after();
    }
    if (__all_sync(0xFFFFFFFFu, ok && *abort_flag == 0u)) {
      const int64_t q = int64_t(it.q_start) + tok;
      const int h = it.kvh * G + (r - tok * G);
      const bool whole = it.part_row < 0;
      // normalisation and the history part's weights (base 2)
      float wo = 1.0f, wh = 0.0f, lse2 = -INFINITY;
      if (whole) {
        const float z = l > 0.0f || l != l ? m + log2f(l) : -INFINITY;  // NaN stays NaN
        wo = z == -INFINITY ? 0.0f : 1.0f / l;
        lse2 = z;
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
      }
      const bool slow = *dirty_flag != 0u;
#pragma unroll 1
      for (int ch = 0; ch < DP / 32; ++ch) {
        float ov[32];
        __syncwarp();
        if (nh > 0) {
          tmem_load32(o_cols + ch * 32, ov);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) ov[j] = 0.0f;
        }
        if (!have || ch * 32 >= a.D) continue;
        if (l == 0.0f) {  // nothing visible here (the MMA ran on P = 0)
#pragma unroll
          for (int j = 0; j < 32; ++j) ov[j] = 0.0f;
        }
        if (slow) {
          // the scrubbed values of keys that this row does see
          const int hi = min(lim, nh * PK);
          for (int k = first_partial * PK; k < hi; ++k) {
            const uint16_t* vr = a.v + (int64_t(it.k_start) + it.t_lo * PK + k) * a.v_token +
                                 int64_t(it.kvh) * a.v_head + ch * 32;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (ch * 32 + j < a.D) {
                const float x = dev::load_elem<DT>(vr, uint64_t(j));
                if (!(fabsf(x) <= 3.4e38f)) ov[j] += x;
              }
          }
        }
        if (!whole) {
          float4* dst = reinterpret_cast<float4*>(a.part_o + (int64_t(it.part_row) + hf * PQ + row) * a.D + ch * 32);
#pragma unroll
          for (int d = 0; d < 8; ++d)
            if (ch * 32 + 4 * d < a.D) dst[d] = make_float4(ov[4 * d], ov[4 * d + 1], ov[4 * d + 2], ov[4 * d + 3]);
          continue;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) ov[j] *= wo;
        const int64_t o_off = (q * a.H + h) * a.D + ch * 32;
        if (wh != 0.0f) {
          const float4* hp = reinterpret_cast<const float4*>(a.hist_o + o_off);
#pragma unroll
          for (int d = 0; d < 8; ++d)
            if (ch * 32 + 4 * d < a.D) {
              const float4 x = __ldg(hp + d);
              ov[4 * d] = fmaf(x.x, wh, ov[4 * d]);
              ov[4 * d + 1] = fmaf(x.y, wh, ov[4 * d + 1]);
              ov[4 * d + 2] = fmaf(x.z, wh, ov[4 * d + 2]);
              ov[4 * d + 3] = fmaf(x.w, wh, ov[4 * d + 3]);
            }
        }
        if (a.out_f32) {
          float4* dst = reinterpret_cast<float4*>(static_cast<float*>(a.out) + o_off);
#pragma unroll
          for (int d = 0; d < 8; ++d)
            if (ch * 32 + 4 * d < a.D) dst[d] = make_float4(ov[4 * d], ov[4 * d + 1], ov[4 * d + 2], ov[4 * d + 3]);
        } else {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + o_off);
#pragma unroll
          for (int d = 0; d < 4; ++d)
            if (ch * 32 + 8 * d < a.D)
              dst[d] = make_uint4(pack2<DT>(ov[8 * d], ov[8 * d + 1]), pack2<DT>(ov[8 * d + 2], ov[8 * d + 3]),
                                  pack2<DT>(ov[8 * d + 4], ov[8 * d + 5]), pack2<DT>(ov[8 * d + 6], ov[8 * d + 7]));
        }
      }
      if (have) {
        if (whole)
          a.lse[int64_t(h) * a.lse_head + q] = lse2 * 0.69314718055994531f;
        else
          reinterpret_cast<float2*>(a.part_ml)[int64_t(it.part_row) + hf * PQ + row] = make_float2(m, l);
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
  // the register split's increase waits for registers the launch must hold:
  // refuse a build whose launch count differs from the split's
  cudaFuncAttributes fa{};
  cudaError_t e = cudaFuncGetAttributes(&fa, k_attend_packed<DT, DP>);
  if (e != cudaSuccess) return e;
  if (fa.numRegs != kRegsLaunch) return cudaErrorInvalidConfiguration;
  e = cudaFuncSetAttribute(k_attend_packed<DT, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::kSmem);
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
