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
// once.  A row lives in the registers of one CTA; a CTA keeps the products
// gate * post_weight and weight * (1 + scale) and the shift of the current
// group in registers over a run of consecutive rows, because reading them
// again per row (20 bytes a column from L2) would cost more than the row
// itself.
#include "nkv_device.cuh"
#include "nkv_kernels.h"

namespace nkv {
namespace {

// Element i of a vector that is f32 or the stream's 16-bit type.
template <int DT>
__device__ __forceinline__ float vec_elem(const void* p, int dt, int64_t i) {
  return dt == F32 ? __ldg(static_cast<const float*>(p) + i) : dev::load_elem<DT>(p, uint64_t(i));
}

// Sum over the CTA; `slot` alternates between consecutive calls, so one
// barrier per call keeps a call's partials apart from the next one's.
__device__ __forceinline__ float cta_sum(float v, float* part, int& slot) {
  const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5, warps = int(blockDim.x) >> 5;
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  if (warps == 1) return v;
  float* p = part + 32 * slot;
  slot ^= 1;
  if (lane == 0) p[warp] = v;
  __syncthreads();
  v = lane < warps ? p[lane] : 0.0f;
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  return v;
}

// 1 / sqrt of the mean square of v over `dim` values (layer: after taking the
// mean off v).  N values per thread, absent ones 0 and not counted.
template <int N>
__device__ __forceinline__ float normalise(float (&v)[N], int n, float inv_dim, float eps, int kind, float* part,
                                           int& slot) {
  if (kind == NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) s += v[j];
    const float mean = cta_sum(s, part, slot) * inv_dim;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < n ? v[j] - mean : 0.0f;
  }
  float q = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) q = fmaf(v[j], v[j], q);
  return 1.0f / sqrtf(cta_sum(q, part, slot) * inv_dim + eps);
}

template <int DT>
__device__ __forceinline__ void load_row8(const void* base, int64_t elem, float* x) {
  if constexpr (DT == F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + elem);
    const float4 a = p[0], b = p[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 r = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + elem);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
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

// The modulation group of row t: -1 when its index is outside the rows there
// are (such a row is filled with NaN: an index is device data, which the host
// cannot check, and a row computed with another group's vectors would pass
// unnoticed).
__device__ __forceinline__ int group_of(const ResidualNormParams& a, uint64_t t) {
  if (!a.mod_index) return 0;
  const int g = __ldg(a.mod_index + t);
  return g >= 0 && g < a.mod_rows ? g : -1;
}

// dim a multiple of 8 with 16-byte aligned rows: thread j of the CTA owns the
// 8-value chunks j, j + threads, ... (V of them).
template <int DT, int V>
__global__ void __launch_bounds__(1024) k_residual_norm_vec(const ResidualNormParams a) {
  __shared__ float part[64];
  int slot = 0;
  const int tid = int(threadIdx.x), threads = int(blockDim.x);
  const int chunks = int(a.dim / 8);
  const float inv_dim = 1.0f / float(a.dim);
  const uint64_t r0 = uint64_t(blockIdx.x) * a.rows_per_cta;
  const uint64_t r1 = min(a.tokens, r0 + a.rows_per_cta);
  // the group's vectors
  float G[8 * V], W[8 * V], S[8 * V];
  int group = -2;
  int n = 0;  // values this thread holds
#pragma unroll
  for (int k = 0; k < V; ++k) n += tid + k * threads < chunks ? 8 : 0;
  for (uint64_t t = r0; t < r1; ++t) {
    const int g = group_of(a, t);
    float h[8 * V], b[8 * V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = tid + k * threads;
      if (c < chunks) {
        load_row8<DT>(a.x, int64_t(t) * a.x_stride + 8 * c, h + 8 * k);
        if (a.branch) load_row8<DT>(a.branch, int64_t(t) * a.branch_stride + 8 * c, b + 8 * k);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[8 * k + j] = b[8 * k + j] = 0.0f;
      }
    }
    if (g != group) {
      group = g;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = tid + k * threads;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float gg = 1.0f, ww = 1.0f, ss = 0.0f;
          if (c < chunks) {
            const int64_t i = 8 * int64_t(c) + j, m = int64_t(max(g, 0)) * a.dim + i;
            if (a.gate) gg = vec_elem<DT>(a.gate, a.mod_dtype, m);
            if (a.post_weight) gg *= vec_elem<DT>(a.post_weight, a.weight_dtype, i);
            if (a.weight) ww = vec_elem<DT>(a.weight, a.weight_dtype, i);
            if (a.scale) ww *= 1.0f + vec_elem<DT>(a.scale, a.mod_dtype, m);
            if (a.shift) ss = vec_elem<DT>(a.shift, a.mod_dtype, m);
          }
          if (g < 0) gg = ww = ss = __int_as_float(0x7FFFFFFF);
          G[8 * k + j] = gg;
          W[8 * k + j] = ww;
          S[8 * k + j] = ss;
        }
      }
    }
    if (a.branch) {
      float inv = 1.0f;
      if (a.post) inv = normalise(b, n, inv_dim, a.eps, a.post, part, slot);
#pragma unroll
      for (int j = 0; j < 8 * V; ++j) h[j] = fmaf(b[j] * inv, G[j], h[j]);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = tid + k * threads;
        if (c < chunks && a.h_out) store_row8<DT>(a.h_out, int64_t(t) * a.h_stride + 8 * c, h + 8 * k);
      }
    }
    if (a.norm) {
      const float inv = normalise(h, n, inv_dim, a.eps, a.norm, part, slot);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = tid + k * threads;
        if (c < chunks) {
          float y[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = fmaf(h[8 * k + j] * inv, W[8 * k + j], S[8 * k + j]);
          store_row8<DT>(a.y_out, int64_t(t) * a.y_stride + 8 * c, y);
        }
      }
    }
  }
}

// Any dim up to kResidualNormMaxDim and any alignment: one CTA per row, the
// row's f32 values in shared memory (each thread touches only its own).
template <int DT>
__global__ void __launch_bounds__(512) k_residual_norm_any(const ResidualNormParams a) {
  extern __shared__ float row[];
  __shared__ float part[64];
  int slot = 0;
  const int tid = int(threadIdx.x), threads = int(blockDim.x), dim = int(a.dim);
  const float inv_dim = 1.0f / float(dim), nan = __int_as_float(0x7FFFFFFF);
  const uint64_t t = blockIdx.x;
  const int g = group_of(a, t);
  const int64_t mrow = int64_t(max(g, 0)) * a.dim;
  auto norm_of = [&](int kind, float& mean) {
    mean = 0.0f;
    if (kind == NORM_LAYER) {
      float s = 0.0f;
      for (int i = tid; i < dim; i += threads) s += row[i];
      mean = cta_sum(s, part, slot) * inv_dim;
    }
    float q = 0.0f;
    for (int i = tid; i < dim; i += threads) q = fmaf(row[i] - mean, row[i] - mean, q);
    return 1.0f / sqrtf(cta_sum(q, part, slot) * inv_dim + a.eps);
  };
  float mean = 0.0f, inv = 1.0f;
  if (a.branch) {
    if (a.post) {
      for (int i = tid; i < dim; i += threads)
        row[i] = dev::load_elem<DT>(a.branch, uint64_t(int64_t(t) * a.branch_stride + i));
      inv = norm_of(a.post, mean);
    }
    for (int i = tid; i < dim; i += threads) {
      const float b = a.post ? row[i] : dev::load_elem<DT>(a.branch, uint64_t(int64_t(t) * a.branch_stride + i));
      float gg = a.gate ? vec_elem<DT>(a.gate, a.mod_dtype, mrow + i) : 1.0f;
      if (a.post_weight) gg *= vec_elem<DT>(a.post_weight, a.weight_dtype, i);
      if (g < 0) gg = nan;
      const float h =
          fmaf((b - mean) * inv, gg, dev::load_elem<DT>(a.x, uint64_t(int64_t(t) * a.x_stride + i)));
      row[i] = h;
      if (a.h_out) dev::store_elem<DT>(a.h_out, uint64_t(int64_t(t) * a.h_stride + i), h);
    }
  } else {
    for (int i = tid; i < dim; i += threads)
      row[i] = dev::load_elem<DT>(a.x, uint64_t(int64_t(t) * a.x_stride + i));
  }
  if (!a.norm) return;
  inv = norm_of(a.norm, mean);
  for (int i = tid; i < dim; i += threads) {
    float ww = a.weight ? vec_elem<DT>(a.weight, a.weight_dtype, i) : 1.0f;
    if (a.scale) ww *= 1.0f + vec_elem<DT>(a.scale, a.mod_dtype, mrow + i);
    float ss = a.shift ? vec_elem<DT>(a.shift, a.mod_dtype, mrow + i) : 0.0f;
    if (g < 0) ww = ss = nan;
    dev::store_elem<DT>(a.y_out, uint64_t(int64_t(t) * a.y_stride + i), fmaf((row[i] - mean) * inv, ww, ss));
  }
}

template <int DT>
cudaError_t launch_dt(ResidualNormParams a, bool vec, cudaStream_t s) {
  if (vec) {
    const int chunks = int(a.dim / 8);
    const int v = chunks <= 1024 ? 1 : 2;
    const int threads = ((chunks + v - 1) / v + 31) / 32 * 32;
    // runs of consecutive rows, about four CTAs of 256 threads' worth per SM
    const uint64_t want = uint64_t(148) * uint64_t(threads >= 1024 ? 1 : 1024 / threads);
    a.rows_per_cta = (a.tokens + want - 1) / want;
    const unsigned grid = unsigned((a.tokens + a.rows_per_cta - 1) / a.rows_per_cta);
    if (v == 1) k_residual_norm_vec<DT, 1><<<grid, threads, 0, s>>>(a);
    else k_residual_norm_vec<DT, 2><<<grid, threads, 0, s>>>(a);
  } else {
    const int threads = a.dim <= 1024 ? 128 : a.dim <= 4096 ? 256 : 512;
    const size_t smem = size_t(a.dim) * sizeof(float);
    if (smem > 40 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(k_residual_norm_any<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 int(kResidualNormMaxDim * sizeof(float)));
      if (e != cudaSuccess) return e;
    }
    k_residual_norm_any<DT><<<unsigned(a.tokens), threads, smem, s>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_residual_norm(const ResidualNormParams& a, int dtype, cudaStream_t s) {
  if (a.tokens == 0) return cudaSuccess;
  const size_t es = dtype_size(dtype);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.branch) |
                         reinterpret_cast<uintptr_t>(a.h_out) | reinterpret_cast<uintptr_t>(a.y_out) |
                         uintptr_t((a.x_stride | a.branch_stride | a.h_stride | a.y_stride) * int64_t(es));
  const bool vec = a.dim % 8 == 0 && a.dim <= 16384 && (bits & 15u) == 0;
  switch (dtype) {
    case F32: return launch_dt<F32>(a, vec, s);
    case BF16: return launch_dt<BF16>(a, vec, s);
    default: return launch_dt<F16>(a, vec, s);
  }
}

}  // namespace nkv
