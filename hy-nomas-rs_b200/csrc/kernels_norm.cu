// kernels_norm.cu — the residual stream between two blocks in one pass:
//   h = x + gate * post(branch)                      (the block's end)
//   y = norm(h) * weight * (1 + scale) + shift       (the next block's start)
// post and norm are RMS (v / sqrt(mean v^2 + eps), norm.rs:55-65) or layer
// norms ((v - mean) / sqrt(var + eps)); gate, scale and shift are rows of
// per-group modulation vectors picked by mod_index (one row per frame of a
// segment, say).  y is what nkv_kv_project takes as x.
//
// Numerics: f32 throughout, the variance from the centred values (two passes
// over registers, no cancellation); y comes from the unrounded h, and h and y
// round once, at their stores.
//
// The pass is bound by its bytes: x and branch read once, h and y written
// once.  A row lives in the registers of one CTA, 16 columns a thread.  A CTA
// takes a run of consecutive rows and keeps the products gate * post_weight
// and weight * (1 + scale) and the shift of the current group in registers:
// reading their five vectors anew for every row (20 bytes a column from L2)
// would cost more than the row itself.  That leaves room for two CTAs an SM at
// 5,120 columns, too few loads in flight for HBM if they went to registers as
// well: rows arrive by cp.async, several ahead, each thread waiting for its own
// bytes only.  Measured: 6,496 rows of 5,120 bf16 columns with norms on both
// sides and five modulation groups (266 MB): 53 us, 5.1 TB/s, where a plain
// copy of as many bytes takes 47.  One row: 5 us, a launch.
#include <algorithm>

#include "nkv_device.cuh"
#include "nkv_kernels.h"

namespace nkv {
namespace {

// One element by the hardware conversions (a NaN stays one, its payload does
// not matter here).
template <int DT>
__device__ __forceinline__ float get(const void* p, int64_t i) {
  if constexpr (DT == F32) return __ldg(static_cast<const float*>(p) + i);
  const uint16_t v = __ldg(static_cast<const uint16_t*>(p) + i);
  return DT == BF16 ? __uint_as_float(uint32_t(v) << 16) : __half2float(__ushort_as_half(v));
}
template <int DT>
__device__ __forceinline__ void put(void* p, int64_t i, float v) {
  if constexpr (DT == F32) static_cast<float*>(p)[i] = v;
  else if constexpr (DT == BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Sum over the CTA's `threads` (blockDim.x, at most 1024); `slot` alternates
// between consecutive calls, so one barrier per call keeps a call's partials
// apart from the next one's.  Every thread adds the warps' partials itself:
// their few broadcast reads are shorter than a second round of shuffles.
__device__ __forceinline__ float cta_sum(float v, float4* part, int& slot) {
  const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5, warps = int(blockDim.x) >> 5;
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  if (warps == 1) return v;
  float4* p = part + 8 * slot;
  slot ^= 1;
  if (lane == 0) reinterpret_cast<float*>(p)[warp] = v;
  // the last warp clears what the last float4 has behind the partials
  if (warp == warps - 1 && lane > 0 && warp + lane < ((warps + 3) & ~3)) reinterpret_cast<float*>(p)[warp + lane] = 0.0f;
  __syncthreads();
  float4 s = p[0];
  for (int k = 1; 4 * k < warps; ++k) {
    const float4 u = p[k];
    s.x += u.x, s.y += u.y, s.z += u.z, s.w += u.w;
  }
  return (s.x + s.y) + (s.z + s.w);
}

// 1 / sqrt of the mean square of v over `dim` values (layer: after taking the
// mean off v).  N values per thread, absent ones 0 and not counted.
template <int N>
__device__ __forceinline__ float normalise(float (&v)[N], int n, float inv_dim, float eps, int kind, float4* part,
                                           int& slot) {
  if (kind == NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) s += v[j];
    const float mean = cta_sum(s, part, slot) * inv_dim;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < n ? v[j] - mean : 0.0f;
  }
  // two running sums in one packed register pair
  static_assert(N % 2 == 0, "");
  float2 q2 = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const float2 p = make_float2(v[j], v[j + 1]);
    q2 = __ffma2_rn(p, p, q2);
  }
  const float q = q2.x + q2.y;
  return rsqrtf(fmaf(cta_sum(q, part, slot), inv_dim, eps));
}

template <int DT>
struct Raw8 {  // 8 values as loaded
  uint4 w[DT == F32 ? 2 : 1];
};

template <int DT>
__device__ __forceinline__ Raw8<DT> load_row8(const void* base, int64_t elem) {
  Raw8<DT> r;
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(base) + elem * (DT == F32 ? 4 : 2));
#pragma unroll
  for (int k = 0; k < (DT == F32 ? 2 : 1); ++k) r.w[k] = p[k];
  return r;
}

template <int DT>
__device__ __forceinline__ void unpack_row8(const Raw8<DT>& r, float* x) {
#pragma unroll
  for (int k = 0; k < (DT == F32 ? 2 : 1); ++k) {
    const uint32_t w[4] = {r.w[k].x, r.w[k].y, r.w[k].z, r.w[k].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == F32) {
        x[4 * k + j] = __uint_as_float(w[j]);
      } else if constexpr (DT == BF16) {
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
__device__ __forceinline__ void store_row8(void* base, int64_t elem, const float* x) {
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

// 8 consecutive elements of such a vector, 16-byte aligned.
template <int DT>
__device__ __forceinline__ void vec8(const void* p, int dt, int64_t i, float* x) {
  if (dt == F32) unpack_row8<F32>(load_row8<F32>(p, i), x);
  else unpack_row8<DT>(load_row8<DT>(p, i), x);
}

// The modulation group of row t: -1 when its index is outside the rows there
// are (such a row is filled with NaN: an index is device data, which the host
// cannot check, and a row computed with another group's vectors would pass
// unnoticed).
__device__ __forceinline__ int group_of(const ResidualNormParams& a, uint64_t t) {
  if (!a.mod_index) return 0;
  const int g = __ldg(a.mod_index + t);
  return g >= 0 && g < a.mod_rows ? g : -1;
}

// The products of group g (-1: NaN) for the 8 columns from i on.
template <int DT>
__device__ __forceinline__ void products8(const ResidualNormParams& a, int g, int64_t i, float* G, float* W, float* S) {
  const int64_t m = int64_t(max(g, 0)) * a.dim + i;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) G[j] = W[j] = 1.0f, S[j] = 0.0f;
  if (a.gate) vec8<DT>(a.gate, a.mod_dtype, m, G);
  if (a.shift) vec8<DT>(a.shift, a.mod_dtype, m, S);
  if (a.weight) vec8<DT>(a.weight, a.weight_dtype, i, W);
  if (a.post_weight) {
    vec8<DT>(a.post_weight, a.weight_dtype, i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) G[j] *= v[j];
  }
  if (a.scale) {
    vec8<DT>(a.scale, a.mod_dtype, m, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) W[j] *= 1.0f + v[j];
  }
  if (g < 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) G[j] = W[j] = S[j] = __int_as_float(0x7FFFFFFF);
  }
}

// dim a multiple of 8 up to 8192, everything 16-byte aligned: thread j of the
// CTA owns the 8-column chunks j and j + threads, and in shared memory the
// bytes of its chunks of the kAhead rows on their way.
//
// 96 registers a thread, so that two CTAs of 320 threads share an SM (at 100
// only one does).  The instructions
// count next: addresses that advance row by row, and x unpacked only when the
// branch's norm is known, took 583 instructions per row and warp to 427 and
// 61 us to 54 (8,192 columns: 94 to 75).  Two rows on their way are enough (53
// us; without modulation groups 49, with three or four rows 52).
constexpr int kAhead = 2;
template <int DT>
__global__ void __maxnreg__(96) k_residual_norm_vec(const ResidualNormParams a) {
  extern __shared__ uint4 ring[];
  __shared__ float4 part[16];
  int slot = 0;
  constexpr int kSize = DT == F32 ? 4 : 2, kPieces = DT == F32 ? 2 : 1;  // 16-byte pieces per chunk
  const int threads = int(blockDim.x), chunks = int(a.dim / 8);
  const int c0 = int(threadIdx.x);
  const bool have[2] = {c0 < chunks, c0 + threads < chunks};
  const int n = 8 * (int(have[0]) + int(have[1]));  // values this thread holds
  const float inv_dim = 1.0f / float(a.dim);
  const uint64_t r0 = uint64_t(blockIdx.x) * a.rows_per_cta;
  const int rows = int(min(a.tokens - r0, a.rows_per_cta));
  // Every address advances by a row at a time; in a row of the ring x comes
  // before the branch, a chunk's pieces `chunks` apart.
  auto first = [&](const void* base, int64_t stride) {
    return reinterpret_cast<uintptr_t>(base) + uintptr_t((int64_t(r0) * stride + 8 * c0) * kSize);
  };
  uintptr_t x_src = first(a.x, a.x_stride), b_src = first(a.branch, a.branch_stride);
  uintptr_t h_dst = first(a.h_out, a.h_stride), y_dst = first(a.y_out, a.y_stride);
  const int gap = 8 * threads * kSize;  // bytes to the second chunk in a row of a tensor; in the ring:
  const uint32_t ring_gap = uint32_t(threads) * 16u, ring_piece = uint32_t(chunks) * 16u,
                 ring_row = 2u * kPieces * ring_piece;
  const uint32_t ring0 = static_cast<uint32_t>(__cvta_generic_to_shared(ring + c0));
  const uint32_t ring_end = ring0 + kAhead * ring_row;
  auto copy = [&](uint32_t dst, uintptr_t src) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int p = 0; p < kPieces; ++p)
        if (have[k])
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + uint32_t(k) * ring_gap +
                                                                        uint32_t(p) * ring_piece),
                       "l"(src + (k ? gap : 0) + 16 * p)
                       : "memory");
  };
  int left = rows;  // rows not asked for yet
  auto request = [&](uint32_t at) {
    if (left-- > 0) {
      copy(at, x_src);
      x_src += uintptr_t(a.x_stride * kSize);
      if (a.branch) {
        copy(at + kPieces * ring_piece, b_src);
        b_src += uintptr_t(a.branch_stride * kSize);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto arrived = [&](uint32_t at, int k, float* x) {  // chunk k; absent: zeros
    Raw8<DT> raw;
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      raw.w[p] = make_uint4(0u, 0u, 0u, 0u);
      if (have[k])
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(raw.w[p].x), "=r"(raw.w[p].y), "=r"(raw.w[p].z), "=r"(raw.w[p].w)
                     : "r"(at + uint32_t(k) * ring_gap + uint32_t(p) * ring_piece)
                     : "memory");
    }
    unpack_row8<DT>(raw, x);
  };
  // v * inv * P + Q of 8 values, on packed pairs
  auto scaled = [](const float* v, float inv, const float* P, const float* Q, float* out) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2 u = __ffma2_rn(__fmul2_rn(make_float2(v[j], v[j + 1]), make_float2(inv, inv)),
                                  make_float2(P[j], P[j + 1]), make_float2(Q[j], Q[j + 1]));
      out[j] = u.x, out[j + 1] = u.y;
    }
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d) request(ring0 + uint32_t(d) * ring_row);
  uint32_t at = ring0;
  const int32_t* index = a.mod_index ? a.mod_index + r0 : nullptr;
  int next_group = group_of(a, r0), group = -2;
  float G[16], W[16], S[16];
#pragma unroll 1
  for (int r = rows; r > 0; --r) {
    if (next_group != group) {
      group = next_group;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (have[k]) products8<DT>(a, group, 8 * int64_t(c0 + k * threads), G + 8 * k, W + 8 * k, S + 8 * k);
    }
    if (index && r > 1) {
      next_group = __ldg(++index);
      if (uint32_t(next_group) >= uint32_t(a.mod_rows)) next_group = -1;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    float h[16];  // the branch, then the stream
    if (a.branch) {
#pragma unroll
      for (int k = 0; k < 2; ++k) arrived(at + kPieces * ring_piece, k, h + 8 * k);
      const float inv = a.post ? normalise(h, n, inv_dim, a.eps, a.post, part, slot) : 1.0f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float x[8];
        arrived(at, k, x);
        scaled(h + 8 * k, inv, G + 8 * k, x, h + 8 * k);
        if (have[k]) store_row8<DT>(reinterpret_cast<void*>(h_dst + (k ? gap : 0)), 0, h + 8 * k);
        else
#pragma unroll
          for (int j = 0; j < 8; ++j) h[8 * k + j] = 0.0f;
      }
      h_dst += uintptr_t(a.h_stride * kSize);
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) arrived(at, k, h + 8 * k);
    }
    request(at);
    at += ring_row;
    if (at == ring_end) at = ring0;
    if (a.norm) {
      const float inv = normalise(h, n, inv_dim, a.eps, a.norm, part, slot);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float y[8];
        scaled(h + 8 * k, inv, W + 8 * k, S + 8 * k, y);
        if (have[k]) store_row8<DT>(reinterpret_cast<void*>(y_dst + (k ? gap : 0)), 0, y);
      }
      y_dst += uintptr_t(a.y_stride * kSize);
    }
  }
}

// The n values tid, tid + threads, ... of a row from element `base` on, others 0.
template <int DT, int E>
__device__ __forceinline__ void get_row(const void* p, int64_t base, int n, int threads, float (&v)[E]) {
  const int64_t at = base + int64_t(threadIdx.x);
#pragma unroll
  for (int k = 0; k < E; ++k) v[k] = k < n ? get<DT>(p, at + k * threads) : 0.0f;
}
// The same of a vector that is f32 or the stream's type.
template <int DT, int E>
__device__ __forceinline__ void get_vec(const void* p, int dt, int64_t base, int n, int threads, float (&v)[E]) {
  if (dt == F32) get_row<F32>(p, base, n, threads, v);
  else get_row<DT>(p, base, n, threads, v);
}
template <int DT, int E>
__device__ __forceinline__ void put_row(void* p, int64_t base, int n, int threads, const float (&v)[E]) {
  const int64_t at = base + int64_t(threadIdx.x);
#pragma unroll
  for (int k = 0; k < E; ++k)
    if (k < n) put<DT>(p, at + k * threads, v[k]);
}

// Any dim and any alignment (what k_residual_norm_vec cannot take, rows above
// 8,192 columns among it: where both can, 6,496 rows of 5,120 columns take 152
// us here, 52 there; of 128 columns 9 and 8).  One value per load and up to five
// waits for memory or a barrier in turn bound it: blockDim.x threads per row, each holding the E
// values tid, tid + blockDim.x, ...; one row per CTA, or one per warp when 32
// threads suffice.  Up to 2,048 columns at 40 registers, for more rows at once
// (6,000 rows of 2,047: 53 us; at 48 58, at 32 54).
template <int DT, int E, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads, kMaxThreads == 256 ? 6 : 1) k_residual_norm_any(const ResidualNormParams a) {
  __shared__ float4 part[16];
  int slot = 0;
  const int tid = int(threadIdx.x), threads = int(blockDim.x), dim = int(a.dim);
  const uint64_t t = uint64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  if (t >= a.tokens) return;  // only where a row is a warp: no barrier is skipped
  const float inv_dim = 1.0f / float(dim), nan = __int_as_float(0x7FFFFFFF);
  const int n = tid < dim ? (dim - tid + threads - 1) / threads : 0;
  float h[E], v[E];
  get_row<DT>(a.x, int64_t(t) * a.x_stride, n, threads, h);
  const int g = group_of(a, t);
  const int64_t mrow = int64_t(max(g, 0)) * a.dim;
  if (a.branch) {
    get_row<DT>(a.branch, int64_t(t) * a.branch_stride, n, threads, v);
    const float inv = a.post ? normalise(v, n, inv_dim, a.eps, a.post, part, slot) : 1.0f;
    const float one = g < 0 ? nan : inv;
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] *= one;
    float w[E];
    if (a.post_weight) {
      get_vec<DT>(a.post_weight, a.weight_dtype, 0, n, threads, w);
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] *= w[k];
    }
    if (a.gate) {
      get_vec<DT>(a.gate, a.mod_dtype, mrow, n, threads, w);
#pragma unroll
      for (int k = 0; k < E; ++k) v[k] *= w[k];
    }
#pragma unroll
    for (int k = 0; k < E; ++k) h[k] += v[k];
    put_row<DT>(a.h_out, int64_t(t) * a.h_stride, n, threads, h);
  }
  if (!a.norm) return;
  const float inv = normalise(h, n, inv_dim, a.eps, a.norm, part, slot);
  const float one = g < 0 ? nan : inv;
#pragma unroll
  for (int k = 0; k < E; ++k) h[k] *= one;
  if (a.weight) {
    get_vec<DT>(a.weight, a.weight_dtype, 0, n, threads, v);
#pragma unroll
    for (int k = 0; k < E; ++k) h[k] *= v[k];
  }
  if (a.scale) {
    get_vec<DT>(a.scale, a.mod_dtype, mrow, n, threads, v);
#pragma unroll
    for (int k = 0; k < E; ++k) h[k] = fmaf(h[k], v[k], h[k]);
  }
  if (a.shift) {
    get_vec<DT>(a.shift, a.mod_dtype, mrow, n, threads, v);
#pragma unroll
    for (int k = 0; k < E; ++k) h[k] += v[k];
  }
  put_row<DT>(a.y_out, int64_t(t) * a.y_stride, n, threads, h);
}

template <int DT>
cudaError_t launch_vec(ResidualNormParams a, cudaStream_t s) {
  const int64_t chunks = a.dim / 8;
  const int threads = int(((chunks + 1) / 2 + 31) / 32 * 32);
  // as many CTAs as 96 registers a thread and the rings (x and branch of each
  // row; at most 128 KB) let an SM hold
  const size_t smem = size_t(a.dim) * 2 * dtype_size(DT) * kAhead;
  const uint64_t per_sm = std::max<uint64_t>(1, std::min<uint64_t>({640u / uint64_t(threads), 220 * 1024 / (smem + 1280), 12}));
  a.rows_per_cta = (a.tokens + per_sm * 148 - 1) / (per_sm * 148);
  const unsigned grid = unsigned((a.tokens + a.rows_per_cta - 1) / a.rows_per_cta);
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(k_residual_norm_vec<DT>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
    if (e != cudaSuccess) return e;
  }
  k_residual_norm_vec<DT><<<grid, threads, smem, s>>>(a);
  return cudaGetLastError();
}

template <int DT>
cudaError_t launch_any(const ResidualNormParams& a, cudaStream_t s) {
  // values per thread: 8 up to 2,048 columns (20,000 rows of 130: 21 us, with 16
  // 33; of 1,155 the same); four rows of one warp each in a CTA (of 255: 23 us
  // against 25 alone)
  const int per = a.dim <= 2048 ? 8 : 16;
  const int threads = a.dim <= 16384 ? int((a.dim + 32 * per - 1) / (32 * per) * 32) : 1024;
  const dim3 block(threads, threads == 32 ? 4 : 1);
  const unsigned grid = unsigned((a.tokens + block.y - 1) / block.y);
  if (per == 8) k_residual_norm_any<DT, 8, 256><<<grid, block, 0, s>>>(a);
  else if (a.dim <= 16384) k_residual_norm_any<DT, 16, 1024><<<grid, block, 0, s>>>(a);
  else k_residual_norm_any<DT, 32, 1024><<<grid, block, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_residual_norm(const ResidualNormParams& a, int dtype, cudaStream_t s) {
  if (a.tokens == 0) return cudaSuccess;
  const size_t es = dtype_size(dtype);
  uintptr_t bits = uintptr_t((a.x_stride | a.branch_stride | a.h_stride | a.y_stride) * int64_t(es));
  for (const void* p : {a.x, a.branch, static_cast<const void*>(a.h_out), static_cast<const void*>(a.y_out),
                        a.post_weight, a.weight, a.gate, a.scale, a.shift})
    bits |= reinterpret_cast<uintptr_t>(p);
  const bool vec = a.dim % 8 == 0 && a.dim <= 8192 && (bits & 15u) == 0;
  switch (dtype) {
    case F32: return vec ? launch_vec<F32>(a, s) : launch_any<F32>(a, s);
    case BF16: return vec ? launch_vec<BF16>(a, s) : launch_any<BF16>(a, s);
    default: return vec ? launch_vec<F16>(a, s) : launch_any<F16>(a, s);
  }
}

}  // namespace nkv
