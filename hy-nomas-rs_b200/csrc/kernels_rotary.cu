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
// Both kernels move bytes: each value is read and written once.  A token's
// D/2 angles serve all its heads, so a CTA computes them once into shared
// memory for a few tokens and then streams those tokens' rows.
#include "nkv_device.cuh"
#include "nkv_kernels.h"

namespace nkv {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotMaxPairs = kRotaryMaxDim / 2;

// cos and sin of an f64 angle, rounded to f32.  The quadrant reduction (three
// parts of pi/2: the product n * P1 is exact inside the fma, what P1 lacks is
// added by P2 and P3) leaves |r| <= pi/4, where the f32 functions are within
// 2 ulp.
__device__ __forceinline__ float2 cos_sin(double a) {
  const double n = rint(a * 0.63661977236758134308);  // 2 / pi
  double r = fma(-n, 1.5707963267948965580, a);       // pi / 2 rounded to 53 bits
  r = fma(-n, 6.1232339957367660359e-17, r);          // the next 53 bits
  const int q = int(__double2ll_rn(n)) & 3;
  float s, c;
  sincosf(float(r), &s, &c);
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

__global__ void __launch_bounds__(kRotThreads) k_rope_tables(const RopePositions P, uint64_t tokens, float* cos_out,
                                                             float* sin_out) {
  const uint64_t total = tokens * uint64_t(P.pairs);
  for (uint64_t i = blockIdx.x * uint64_t(kRotThreads) + threadIdx.x; i < total;
       i += uint64_t(gridDim.x) * kRotThreads) {
    const uint64_t t = i / uint64_t(P.pairs);
    const int p = int(i - t * uint64_t(P.pairs));
    const float2 cs = cos_sin(position(P, t, P.axis[p]) * P.freq[p]);
    cos_out[i] = cs.x;
    sin_out[i] = cs.y;
  }
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

// The angles of this CTA's tokens as (cos, sin) pairs [token][pair].
__device__ __forceinline__ void fill_angles(const RopePositions& P, float2* table, uint64_t t0, int nt) {
  for (int i = threadIdx.x; i < nt * P.pairs; i += blockDim.x) {
    const int t = i / P.pairs, p = i - t * P.pairs;
    table[i] = cos_sin(position(P, t0 + uint64_t(t), P.axis[p]) * P.freq[p]);
  }
}

// head_dim 16 * LPR, 16-byte aligned rows: LPR lanes per (token, head), each
// two 16-byte (f32: 32-byte) chunks.  Interleaved pairs: chunks 2l, 2l + 1.
// Half-split pairs: chunk l of the first and of the second half of the rotated
// values, so both members of a pair meet in one thread; lanes past R / 16 take
// two chunks of the values that pass through (R is a multiple of 16).
template <int DT, int LPR>
__global__ void __launch_bounds__(kRotThreads) k_rotary_vec(const RotaryParams a) {
  extern __shared__ float2 table[];
  constexpr int D = 16 * LPR;
  const RopePositions& P = a.pos;
  const uint64_t t0 = uint64_t(blockIdx.x) * uint64_t(a.tokens_per_cta);
  const int nt = int(min(uint64_t(a.tokens_per_cta), a.tokens - t0));
  fill_angles(P, table, t0, nt);
  __syncthreads();
  const int l = int(threadIdx.x) % LPR, slot = int(threadIdx.x) / LPR;
  constexpr int kSlots = kRotThreads / LPR;
  const int R = 2 * P.pairs, heads = a.side[0].heads + a.side[1].heads;
  int c0 = 2 * l, c1 = 2 * l + 1;
  int n_rot;  // pairs this thread rotates
  int p0;     // its first pair
  if (a.interleaved) {
    p0 = 8 * l;
    n_rot = max(0, min(8, P.pairs - p0));
  } else if (l < R / 16) {
    c0 = l;
    c1 = l + R / 16;
    p0 = 8 * l;
    n_rot = 8;
  } else {
    c0 = R / 8 + 2 * (l - R / 16);
    c1 = c0 + 1;
    p0 = 0;
    n_rot = 0;
  }
  const int rows = nt * heads, rounds = (rows + kSlots - 1) / kSlots;
  for (int it = 0; it < rounds; ++it) {
    const int row = it * kSlots + slot;
    const bool have = row < rows;  // every lane stays for the shuffles
    const int t = have ? row / heads : 0;
    int h = have ? row - t * heads : 0;
    const int sd = h >= a.side[0].heads ? 1 : 0;
    const RotarySide& S = a.side[sd];
    if (sd) h -= a.side[0].heads;
    float x[16];
    if (have) {
      const int64_t base = int64_t(t0 + uint64_t(t)) * S.in_token + int64_t(h) * S.in_head;
      const Chunk<DT> u = load_chunk<DT>(S.in, base + 8 * c0), v = load_chunk<DT>(S.in, base + 8 * c1);
      unpack<DT>(u, x);
      unpack<DT>(v, x + 8);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = 0.0f;
    }
    if (a.norm) {
      float s[2] = {0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j & 1] = fmaf(x[j], x[j], s[j & 1]);
      float ss = s[0] + s[1];
#pragma unroll
      for (int d = 1; d < LPR; d <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
      const float inv = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
      if (S.weight) {
        float w[16];
        unpack<DT>(load_chunk<DT>(S.weight, 8 * c0), w);
        unpack<DT>(load_chunk<DT>(S.weight, 8 * c1), w + 8);
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] *= inv * w[j];
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] *= inv;
      }
    }
    if (!have) continue;
    const float2* cs = table + t * P.pairs + p0;
    if (a.interleaved) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n_rot) {
          const float2 r = cs[j];
          const float xr = x[2 * j], xi = x[2 * j + 1];
          x[2 * j] = fmaf(xr, r.x, -xi * r.y);
          x[2 * j + 1] = fmaf(xi, r.x, xr * r.y);
        }
    } else if (n_rot) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 r = cs[j];
        const float xr = x[j], xi = x[8 + j];
        x[j] = fmaf(xr, r.x, -xi * r.y);
        x[8 + j] = fmaf(xi, r.x, xr * r.y);
      }
    }
    const int64_t base = int64_t(t0 + uint64_t(t)) * S.out_token + int64_t(h) * S.out_head;
    store_chunk<DT>(S.out, base + 8 * c0, x);
    store_chunk<DT>(S.out, base + 8 * c1, x + 8);
  }
}

// Any even head_dim up to kRotaryMaxDim, any strides: one warp per (token,
// head), each lane owning whole pair slots (slot p < pairs: the rotated pair
// p; the slots after them: two consecutive values that pass through), so a
// row may be rotated in place.
template <int DT>
__global__ void __launch_bounds__(kRotThreads) k_rotary_any(const RotaryParams a) {
  extern __shared__ float2 table[];
  const RopePositions& P = a.pos;
  const uint64_t t0 = uint64_t(blockIdx.x) * uint64_t(a.tokens_per_cta);
  const int nt = int(min(uint64_t(a.tokens_per_cta), a.tokens - t0));
  fill_angles(P, table, t0, nt);
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
      case 16: k_rotary_vec<DT, 1><<<grid, kRotThreads, smem, s>>>(a); break;
      case 32: k_rotary_vec<DT, 2><<<grid, kRotThreads, smem, s>>>(a); break;
      case 64: k_rotary_vec<DT, 4><<<grid, kRotThreads, smem, s>>>(a); break;
      case 128: k_rotary_vec<DT, 8><<<grid, kRotThreads, smem, s>>>(a); break;
      default: k_rotary_vec<DT, 16><<<grid, kRotThreads, smem, s>>>(a); break;
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
  const uint64_t ctas = (total + kRotThreads - 1) / kRotThreads;
  k_rope_tables<<<unsigned(ctas < 148 * 32 ? ctas : 148 * 32), kRotThreads, 0, s>>>(p, tokens, cos_out, sin_out);
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
  // Tokens per CTA: enough rows that a CTA's angles (about one per thread)
  // serve several rows per thread, and at most 32.
  const int lanes = vec ? a.D / 16 : 32;
  int nt = (4 * kRotThreads + heads * lanes - 1) / (heads * lanes);
  nt = nt < 1 ? 1 : nt > 32 ? 32 : nt;
  a.tokens_per_cta = nt;
  const uint64_t grid = (a.tokens + uint64_t(nt) - 1) / uint64_t(nt);
  const size_t smem = size_t(nt) * a.pos.pairs * sizeof(float2);  // <= 32 * 128 * 8 = 32 KB
  switch (dtype) {
    case F32: return launch_dt<F32>(a, vec, unsigned(grid), smem, s);
    case BF16: return launch_dt<BF16>(a, vec, unsigned(grid), smem, s);
    default: return launch_dt<F16>(a, vec, unsigned(grid), smem, s);
  }
}

}  // namespace nkv
