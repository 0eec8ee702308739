// kernels_rotary.cu — rotary positions with several axes: the cos / sin
// tables that nkv_kv_project takes, and the per-head RMS norm and rotation
// applied to q (and k) directly.
//
// Pair p of a head belongs to one axis a with dims[a] of the rotated R =
// sum(dims) values, index i inside it; its angle at token t is
//   pos[t][a] * theta^(-2 i / dims[a]).
// The rotation takes (x, y) to (x c - y s, y c + x s) on the values (2p, 2p+1)
// (interleaved, the layout of rope.rs:257-306) or (p, p + R/2); values at and
// past R pass through.  With norm the head is first divided by its RMS
// (norm.rs:55-65) and multiplied by the gain.
//
// Numerics: the angle and its reduction to [-pi/4, pi/4] are taken in f64 (a
// position of 10^6 would lose every digit of its fastest angles in f32), the
// sine and cosine of the remainder in f32; norm and rotation run in f32 from
// the input and round once, at the store (nkv_kv_project rounds after the norm
// as well, as the reference does between its two modules).
//
// The rotation moves bytes: each value is read and written once.  A token's
// D / 2 angles serve all its heads: a CTA computes those of its tokens, each
// lane takes the ones of its own columns into registers, and a group of lanes
// streams a token's heads, several rows ahead.  Measured: q and k of 6,496
// tokens, 2 x 24 heads of 128, bf16, norm and three axes (160 MB): 30 us,
// 5.3 TB/s, where a plain copy of as many bytes takes 29; 4,099 tokens, 40
// heads of 128, f16, 80 values rotated in half-split pairs (84 MB): 21 us,
// 4.0 TB/s (a copy: 17).  One token: 4 us, a launch.
#include <type_traits>

#include "nkv_device.cuh"
#include "nkv_kernels.h"

namespace nkv {
namespace {

constexpr int kRotThreads = 256, kVecThreads = 128;
constexpr int kRotMaxPairs = kRotaryMaxDim / 2;

// cos and sin of an f64 angle in f32.  The quadrant reduction in f64 (two parts
// of pi / 2; the product with the first is exact inside the fma) leaves |r| <=
// pi / 4, where the Taylor sums sin r = r - r^3/3! + ... + r^9/9! and cos r = 1
// - r^2/2! + ... + r^10/10! stop below 2^-29 of 1 and each last rounding is one
// of f32.  Their few multiply-adds replace library calls whose argument
// reduction this kernel has no use for.
__device__ __forceinline__ float2 cos_sin(double a) {
  const double n = rint(a * 0.63661977236758134308);  // 2 / pi
  double r = fma(-n, 1.5707963267948965580, a);       // pi / 2 rounded to 53 bits
  r = fma(-n, 6.1232339957367660359e-17, r);          // the next 53 bits
  const int q = int(__double2ll_rn(n)) & 3;
  const float x = float(r), y = x * x;
  float s = fmaf(2.7557319e-6f, y, -1.9841270e-4f);  // 1/9!, -1/7!
  s = fmaf(s, y, 8.3333333e-3f);                      // 1/5!
  s = fmaf(s, y, -1.6666667e-1f);                     // -1/3!
  s = fmaf(s * y, x, x);
  float c = fmaf(-2.7557319e-7f, y, 2.4801587e-5f);  // -1/10!, 1/8!
  c = fmaf(c, y, -1.3888889e-3f);                     // -1/6!
  c = fmaf(c, y, 4.1666667e-2f);                      // 1/4!
  c = fmaf(c, y, -0.5f);
  c = fmaf(c, y, 1.0f);
  if (q & 1) {
    const float t = s;
    s = c;
    c = -t;
  }
  if (q & 2) {
    s = -s;
    c = -c;
  }
  return make_float2(c, s);
}

__device__ __forceinline__ double position(const RopePositions& P, uint64_t t, int axis) {
  const uint64_t i = t * uint64_t(P.n_axes) + uint64_t(axis);
  if (P.dtype == POS_I32) return double(__ldg(static_cast<const int32_t*>(P.data) + i));
  if (P.dtype == POS_I64) return double(__ldg(static_cast<const long long*>(P.data) + i));
  return double(__ldg(static_cast<const float*>(P.data) + i));
}

// Calls f(token, pair, cos, sin) for the CTA's tokens t0 .. t0 + nt.  A thread
// keeps its pairs p, p + blockDim.x, ... over all its tokens: the frequencies
// lie in the kernel's parameters, where lanes that index differently are
// served one at a time, so each is read once per thread.
template <typename F>
__device__ __forceinline__ void for_angles(const RopePositions& P, uint64_t t0, int nt, F&& f) {
  const int lanes = min(P.pairs, int(blockDim.x));      // threads along the pairs
  const int rows = int(blockDim.x) / lanes;             // tokens at a time
  const int row = int(threadIdx.x) / lanes;
  if (row >= rows) return;
  for (int p = int(threadIdx.x) - row * lanes; p < P.pairs; p += lanes) {
    const double freq = P.freq[p];
    const int axis = P.axis[p];
    for (int t = row; t < nt; t += rows) {
      const float2 cs = cos_sin(position(P, t0 + uint64_t(t), axis) * freq);
      f(t, p, cs);
    }
  }
}

__global__ void __launch_bounds__(kRotThreads) k_rope_tables(const RopePositions P, uint64_t tokens, int per_cta,
                                                             float* cos_out, float* sin_out) {
  const uint64_t t0 = uint64_t(blockIdx.x) * uint64_t(per_cta);
  const int nt = int(min(uint64_t(per_cta), tokens - t0));
  for_angles(P, t0, nt, [&](int t, int p, float2 cs) {
    const uint64_t i = (t0 + uint64_t(t)) * uint64_t(P.pairs) + uint64_t(p);
    cos_out[i] = cs.x;
    sin_out[i] = cs.y;
  });
}

template <int DT>
struct Chunk;  // 8 values as loaded
template <>
struct Chunk<F32> {
  float4 a, b;
};
template <>
struct Chunk<BF16> {
  uint4 a;
};
template <>
struct Chunk<F16> {
  uint4 a;
};

template <int DT>
__device__ __forceinline__ Chunk<DT> load_chunk(const void* base, int64_t elem) {
  Chunk<DT> c;
  if constexpr (DT == F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + elem);
    c.a = p[0];
    c.b = p[1];
  } else {
    c.a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + elem);
  }
  return c;
}

template <int DT>
__device__ __forceinline__ void unpack(const Chunk<DT>& c, float* x) {
  if constexpr (DT == F32) {
    x[0] = c.a.x, x[1] = c.a.y, x[2] = c.a.z, x[3] = c.a.w, x[4] = c.b.x, x[5] = c.b.y, x[6] = c.b.z, x[7] = c.b.w;
  } else {
    const uint32_t w[4] = {c.a.x, c.a.y, c.a.z, c.a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == BF16) {
        x[2 * j] = __uint_as_float(w[j] << 16);
        x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        x[2 * j] = f.x;
        x[2 * j + 1] = f.y;
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ void store_chunk(void* base, int64_t elem, const float* x) {
  if constexpr (DT == F32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + elem);
    p[0] = make_float4(x[0], x[1], x[2], x[3]);
    p[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = DT == BF16 ? dev::bf16x2_bits_nonnan(x[2 * j], x[2 * j + 1])
                        : dev::f16x2_bits_nonnan(x[2 * j], x[2 * j + 1]);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + elem) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// head_dim 16 * LPR, 16-byte aligned rows: LPR lanes per (token, head), each
// two chunks of 8 values; consecutive lanes take consecutive chunks, so an
// access covers whole lines.  Interleaved pairs: chunks l and l + LPR.
// Half-split pairs: chunk l of the first and of the second half of the rotated
// values, so both members of a pair meet in one thread; lanes past R / 16 take
// two chunks of the values that pass through (R is a multiple of 16).
// 2^log_hp such groups share a token's heads, where one group per token would
// leave the GPU empty.
//
// What bounded it was the count of instructions, 65 % of the issue slots at 260
// per row and warp: row addresses by 64-bit products, an angle per lane and
// group, masks on every row.  Pointers that advance, angles shared by the CTA
// and a path of its own for warps whose pairs all rotate took the 160 MB above
// from 35 to 30 us, the 84 MB from 27.5 to 21 (5 CTAs of 128 threads an SM at
// 96 registers; 6 at 80 spill: 31 and 23; 4: 29 and 22).  Rows ahead: 2 take
// 32.7 us, 4 take 30.4, 8 take 31.0.
template <int DT, int LPR>
__global__ void __launch_bounds__(kVecThreads, 5) k_rotary_vec(const RotaryParams a) {
  constexpr int D = 16 * LPR;
  constexpr int kSize = DT == F32 ? 4 : 2;
  // rows a thread has in flight, by cp.async into its own bytes of shared memory
  constexpr int kAhead = DT == F32 ? 2 : 4, kPieces = DT == F32 ? 2 : 1;  // 16-byte pieces per chunk
  __shared__ uint4 ring[kAhead][2][kPieces][kVecThreads];
  constexpr int kGroups = kVecThreads / LPR;
  __shared__ float2 angles[kGroups * (D / 2)];  // of the CTA's tokens
  const RopePositions& P = a.pos;
  __shared__ double freq[D / 2];
  __shared__ uint8_t axis[D / 2];
  const int l = int(threadIdx.x) % LPR;
  const uint64_t group = (uint64_t(blockIdx.x) * kVecThreads + threadIdx.x) / LPR;
  const int hp = 1 << a.log_hp, h0 = int(group) & (hp - 1);
  const uint64_t t = group >> a.log_hp;
  const bool live = t < a.tokens;
  const int R = 2 * P.pairs;
  int c0 = l, c1 = l + LPR;
  int n_rot0 = 0, n_rot1 = 0;  // rotated pairs of the chunks (half-split: of both together, in n_rot0)
  if (a.interleaved) {
    n_rot0 = max(0, min(4, P.pairs - 4 * c0));
    n_rot1 = max(0, min(4, P.pairs - 4 * c1));
  } else if (l < R / 16) {
    c1 = l + R / 16;
    n_rot0 = 8;
  } else {
    c0 = R / 8 + (l - R / 16);
    c1 = c0 + (D - R) / 16;
  }
  // The rows are q's heads h0, h0 + hp, ... and then k's.  Every group goes
  // through the same number of each (the shuffles want whole warps); the last
  // may not exist.
  struct Side {
    int steps, rows;  // of every group, of this one
  };
  auto side_of = [&](int sd) {
    const int heads = a.side[sd].heads;
    return Side{(heads + hp - 1) >> a.log_hp, live ? max(0, (heads - h0 + hp - 1) >> a.log_hp) : 0};
  };
  const Side sides[2] = {side_of(0), side_of(1)};
  auto first_row = [&](const void* base, int64_t token, int64_t head) {
    return reinterpret_cast<uintptr_t>(base) + uintptr_t((int64_t(t) * token + h0 * head + 8 * c0) * kSize);
  };
  const int gap = 8 * (c1 - c0) * kSize;  // bytes from the first chunk to the second
  int asked = 0, ask_left = sides[0].rows;
  uintptr_t src = first_row(a.side[0].in, a.side[0].in_token, a.side[0].in_head);
  int64_t src_step = a.side[0].in_head * kSize << a.log_hp;
  const uint32_t ring0 = static_cast<uint32_t>(__cvta_generic_to_shared(&ring[0][0][0][threadIdx.x]));
  constexpr uint32_t kPiece = kVecThreads * 16, kRow = 2 * kPieces * kPiece;
  auto request = [&](uint32_t slot) {
    if (asked == sides[0].steps) {
      ask_left = sides[1].rows;
      src = first_row(a.side[1].in, a.side[1].in_token, a.side[1].in_head);
      src_step = a.side[1].in_head * kSize << a.log_hp;
    }
    ++asked;
    if (--ask_left >= 0) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int p = 0; p < kPieces; ++p)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring0 + slot * kRow +
                                                                        uint32_t(k * kPieces + p) * kPiece),
                       "l"(src + (k ? gap : 0) + 16 * p)
                       : "memory");
    }
    src += uintptr_t(src_step);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto arrived = [&](uint32_t slot, int k, float* x) {
    Chunk<DT> c;
    c.a = *reinterpret_cast<const decltype(c.a)*>(&ring[slot][k][0][threadIdx.x]);
    if constexpr (DT == F32) c.b = *reinterpret_cast<const float4*>(&ring[slot][k][kPieces - 1][threadIdx.x]);
    unpack<DT>(c, x);
  };
  // the first rows are on their way while the angles are computed
#pragma unroll
  for (uint32_t b = 0; b < kAhead; ++b) request(b);
  // (the parameters serve lanes that index differently one at a time)
  if (threadIdx.x < P.pairs) {
    freq[threadIdx.x] = P.freq[threadIdx.x];
    axis[threadIdx.x] = P.axis[threadIdx.x];
  }
  __syncthreads();
  // one angle per thread at a time; the groups of a token share them
  const uint64_t t0 = (uint64_t(blockIdx.x) * kGroups) >> a.log_hp;
  const int nt = int(min(uint64_t(max(1, kGroups >> a.log_hp)), a.tokens - t0));
  for (int i = int(threadIdx.x); i < nt * P.pairs; i += kVecThreads) {
    const int row = i / P.pairs, p = i - row * P.pairs;
    angles[i] = cos_sin(position(P, t0 + uint64_t(row), axis[p]) * freq[p]);
  }
  __syncthreads();
  // Pair j of this thread is (x[ia(j)], x[ib(j)]) of its 16 values: with the
  // gains w folded in,
  //   a' = a (w_a c) - b (w_b s),  b' = b (w_b c) + a (w_a s),
  // on two pairs at a time.  A pair that passes through is only multiplied by
  // its gains: its partner is masked to 0 (a sine of 0 alone would turn an
  // infinite partner into a NaN) and its sine to -0 (0 * -0 + x is x, for x = -0
  // too).
  float2 cs[8];
  uint32_t mask[8];
  bool all = true;
  {
    const int pa = a.interleaved ? 4 * c0 : 8 * c0, pb = a.interleaved ? 4 * c1 : 8 * c0 + 4;
    const int na = a.interleaved ? n_rot0 : n_rot0 / 2, nb = a.interleaved ? n_rot1 : n_rot0 / 2;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool rotates = j < 4 ? j < na : j - 4 < nb;
      cs[j] = rotates && live ? angles[int(t - t0) * P.pairs + (j < 4 ? pa + j : pb + j - 4)] : make_float2(1.0f, 0.0f);
      mask[j] = rotates ? 0xFFFFFFFFu : 0u;
      all &= rotates;
    }
  }
  uint32_t slot = 0;
  auto stream = [&](auto inter_, auto all_) {
    constexpr bool kInter = decltype(inter_)::value, kAll = decltype(all_)::value;
    auto ia = [](int j) { return kInter ? 2 * j : j; };
    auto ib = [](int j) { return kInter ? 2 * j + 1 : 8 + j; };
    auto masked = [&](float2 v, int j) {
      if (kAll) return v;
      return make_float2(__uint_as_float(__float_as_uint(v.x) & mask[2 * j]),
                         __uint_as_float(__float_as_uint(v.y) & mask[2 * j + 1]));
    };
#pragma unroll 1
    for (int sd = 0; sd < 2; ++sd) {
      const int steps = sd ? sides[1].steps : sides[0].steps, rows = sd ? sides[1].rows : sides[0].rows;
      if (steps == 0) continue;
      const RotarySide& S = a.side[sd];
      float w[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) w[j] = 1.0f;
      if (a.norm && S.weight) {
        unpack<DT>(load_chunk<DT>(S.weight, 8 * c0), w);
        unpack<DT>(load_chunk<DT>(S.weight, 8 * c1), w + 8);
      }
      float2 ca[4], sb[4], cb[4], sa[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 u = cs[2 * j], v = cs[2 * j + 1];
        const float a0 = w[ia(2 * j)], a1 = w[ia(2 * j + 1)], b0 = w[ib(2 * j)], b1 = w[ib(2 * j + 1)];
        ca[j] = make_float2(a0 * u.x, a1 * v.x);
        cb[j] = make_float2(b0 * u.x, b1 * v.x);
        const bool r0 = kAll || mask[2 * j], r1 = kAll || mask[2 * j + 1];
        sb[j] = make_float2(r0 ? -b0 * u.y : -0.0f, r1 ? -b1 * v.y : -0.0f);
        sa[j] = make_float2(r0 ? a0 * u.y : -0.0f, r1 ? a1 * v.y : -0.0f);
      }
      uintptr_t dst = first_row(S.out, S.out_token, S.out_head);
      const int64_t dst_step = S.out_head * kSize << a.log_hp;
#pragma unroll 1
      for (int n = 0; n < steps; ++n) {
        float x[16];
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        arrived(slot, 0, x);
        arrived(slot, 1, x + 8);
        request(slot);
        slot = (slot + 1) & (kAhead - 1);
        float2 A[4], Bv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          A[j] = make_float2(x[ia(2 * j)], x[ia(2 * j + 1)]);
          Bv[j] = make_float2(x[ib(2 * j)], x[ib(2 * j + 1)]);
        }
        float2 inv2 = make_float2(1.0f, 1.0f);
        if (a.norm) {
          float2 s0 = __fmul2_rn(A[0], A[0]), s1 = __fmul2_rn(Bv[0], Bv[0]);
#pragma unroll
          for (int j = 1; j < 4; ++j) {
            s0 = __ffma2_rn(A[j], A[j], s0);
            s1 = __ffma2_rn(Bv[j], Bv[j], s1);
          }
          const float2 s = __fadd2_rn(s0, s1);
          float ss = s.x + s.y;
#pragma unroll
          for (int d = 1; d < LPR; d <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
          const float inv = rsqrtf(fmaf(ss, 1.0f / D, a.eps));
          inv2 = make_float2(inv, inv);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 ra = __ffma2_rn(masked(Bv[j], j), sb[j], __fmul2_rn(A[j], ca[j]));
          const float2 rb = __ffma2_rn(masked(A[j], j), sa[j], __fmul2_rn(Bv[j], cb[j]));
          const float2 na = __fmul2_rn(ra, inv2), nb = __fmul2_rn(rb, inv2);
          x[ia(2 * j)] = na.x, x[ia(2 * j + 1)] = na.y;
          x[ib(2 * j)] = nb.x, x[ib(2 * j + 1)] = nb.y;
        }
        if (n < rows) {
          store_chunk<DT>(reinterpret_cast<void*>(dst), 0, x);
          store_chunk<DT>(reinterpret_cast<void*>(dst + gap), 0, x + 8);
        }
        dst += uintptr_t(dst_step);
      }
    }
  };
  all = __all_sync(0xFFFFFFFFu, all);
  if (a.interleaved) {
    if (all) stream(std::true_type(), std::true_type());
    else stream(std::true_type(), std::false_type());
  } else {
    if (all) stream(std::false_type(), std::true_type());
    else stream(std::false_type(), std::false_type());
  }
}

// Any even head_dim up to kRotaryMaxDim, any strides and alignment (what
// k_rotary_vec cannot take: where both can, the 160 MB above take 129 us here,
// 29 there): one warp per (token,
// head), each lane owning whole pair slots (slot p < pairs: the rotated pair
// p; the slots after them: two consecutive values that pass through), so a
// row may be rotated in place.
template <int DT>
__global__ void __launch_bounds__(kRotThreads) k_rotary_any(const RotaryParams a) {
  extern __shared__ float2 table[];
  const RopePositions& P = a.pos;
  const uint64_t t0 = uint64_t(blockIdx.x) * uint64_t(a.tokens_per_cta);
  const int nt = int(min(uint64_t(a.tokens_per_cta), a.tokens - t0));
  for_angles(P, t0, nt, [&](int t, int p, float2 cs) { table[t * P.pairs + p] = cs; });
  __syncthreads();
  const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
  const int heads = a.side[0].heads + a.side[1].heads, slots = a.D / 2;
  constexpr int kMaxSlots = kRotMaxPairs / 32;
  for (int row = warp; row < nt * heads; row += kRotThreads / 32) {
    const int t = row / heads;
    int h = row - t * heads;
    const int sd = h >= a.side[0].heads ? 1 : 0;
    const RotarySide& S = a.side[sd];
    if (sd) h -= a.side[0].heads;
    const int64_t ib = int64_t(t0 + uint64_t(t)) * S.in_token + int64_t(h) * S.in_head;
    const int64_t ob = int64_t(t0 + uint64_t(t)) * S.out_token + int64_t(h) * S.out_head;
    float x[kMaxSlots], y[kMaxSlots], ss = 0.0f;
    auto first = [&](int p) { return a.interleaved || p >= P.pairs ? 2 * p : p; };
    auto second = [&](int p) { return a.interleaved || p >= P.pairs ? 2 * p + 1 : p + P.pairs; };
#pragma unroll
    for (int k = 0; k < kMaxSlots; ++k) {
      const int p = lane + 32 * k;
      x[k] = y[k] = 0.0f;
      if (p < slots) {
        x[k] = dev::load_elem<DT>(S.in, uint64_t(ib + first(p)));
        y[k] = dev::load_elem<DT>(S.in, uint64_t(ib + second(p)));
      }
      ss = fmaf(x[k], x[k], fmaf(y[k], y[k], ss));
    }
    float inv = 1.0f;
    if (a.norm) {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
      inv = 1.0f / sqrtf(ss / float(a.D) + a.eps);
    }
#pragma unroll
    for (int k = 0; k < kMaxSlots; ++k) {
      const int p = lane + 32 * k;
      if (p >= slots) continue;
      float u = x[k], v = y[k];
      if (a.norm) {
        u *= S.weight ? inv * dev::load_elem<DT>(S.weight, uint64_t(first(p))) : inv;
        v *= S.weight ? inv * dev::load_elem<DT>(S.weight, uint64_t(second(p))) : inv;
      }
      if (p < P.pairs) {
        const float2 r = table[t * P.pairs + p];
        const float w = fmaf(u, r.x, -v * r.y);
        v = fmaf(v, r.x, u * r.y);
        u = w;
      }
      dev::store_elem<DT>(S.out, uint64_t(ob + first(p)), u);
      dev::store_elem<DT>(S.out, uint64_t(ob + second(p)), v);
    }
  }
}

template <int DT>
cudaError_t launch_dt(const RotaryParams& a, bool vec, unsigned grid, size_t smem, cudaStream_t s) {
  if (vec) {
    switch (a.D) {
      case 16: k_rotary_vec<DT, 1><<<grid, kVecThreads, smem, s>>>(a); break;
      case 32: k_rotary_vec<DT, 2><<<grid, kVecThreads, smem, s>>>(a); break;
      case 64: k_rotary_vec<DT, 4><<<grid, kVecThreads, smem, s>>>(a); break;
      case 128: k_rotary_vec<DT, 8><<<grid, kVecThreads, smem, s>>>(a); break;
      default: k_rotary_vec<DT, 16><<<grid, kVecThreads, smem, s>>>(a); break;
    }
  } else {
    k_rotary_any<DT><<<grid, kRotThreads, smem, s>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rope_tables(const RopePositions& p, uint64_t tokens, float* cos_out, float* sin_out,
                               cudaStream_t s) {
  const uint64_t total = tokens * uint64_t(p.pairs);
  if (total == 0) return cudaSuccess;
  // a few angles per thread, and CTAs for every SM
  const uint64_t rows = uint64_t(kRotThreads / (p.pairs < kRotThreads ? p.pairs : kRotThreads));
  uint64_t per = (tokens + 148 * 8 - 1) / (148 * 8);
  per = (per + rows - 1) / rows * rows;
  k_rope_tables<<<unsigned((tokens + per - 1) / per), kRotThreads, 0, s>>>(p, tokens, int(per), cos_out, sin_out);
  return cudaGetLastError();
}

cudaError_t launch_rotary(RotaryParams a, int dtype, cudaStream_t s) {
  const int heads = a.side[0].heads + a.side[1].heads;
  if (a.tokens == 0 || heads == 0) return cudaSuccess;
  const size_t es = dtype_size(dtype);
  bool vec = a.D == 16 || a.D == 32 || a.D == 64 || a.D == 128 || a.D == 256;
  if (!a.interleaved && (2 * a.pos.pairs) % 16) vec = false;
  for (const RotarySide& sd : a.side) {
    if (!sd.heads) continue;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(sd.in) | reinterpret_cast<uintptr_t>(sd.out) |
                           reinterpret_cast<uintptr_t>(sd.weight) |
                           uintptr_t((sd.in_token | sd.in_head | sd.out_token | sd.out_head) * int64_t(es));
    if (bits & 15u) vec = false;
  }
  uint64_t grid;
  size_t smem = 0;
  if (vec) {
    // groups per token: enough for some 768 threads an SM (6,496 tokens of 48
    // heads: 4 groups, 30 us; 2 groups: 37), at least three rows each
    const int lanes = a.D / 16;
    a.log_hp = 0;
    while ((a.tokens << a.log_hp) * uint64_t(lanes) < 148 * 768 && (heads >> a.log_hp) > 3) ++a.log_hp;
    grid = ((a.tokens << a.log_hp) * uint64_t(lanes) + kVecThreads - 1) / kVecThreads;
  } else {
    // a row per warp: enough rows that a CTA's angles serve several
    int nt = (4 * kRotThreads + heads * 32 - 1) / (heads * 32);
    nt = nt < 1 ? 1 : nt > 32 ? 32 : nt;
    a.tokens_per_cta = nt;
    grid = (a.tokens + uint64_t(nt) - 1) / uint64_t(nt);
    smem = size_t(nt) * a.pos.pairs * sizeof(float2);  // <= 32 * 128 * 8 = 32 KB
  }
  switch (dtype) {
    case F32: return launch_dt<F32>(a, vec, unsigned(grid), smem, s);
    case BF16: return launch_dt<BF16>(a, vec, unsigned(grid), smem, s);
    default: return launch_dt<F16>(a, vec, unsigned(grid), smem, s);
  }
}

}  // namespace nkv
