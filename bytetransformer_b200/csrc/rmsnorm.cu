// Root-mean-square norm with the residual's addition, the result in fp16 or in 8 bits (e4m3) with scales:
//
//   s = x + residual
//   y = s / sqrt(mean(s^2) + eps) * gamma
//   fp16:  out = y
//   e4m3:  scale = max(max |y| over the group, 2^-100) / 448,  out = y * (1 / scale);  a group is a row or 128 columns of it
//
// The reciprocal is rounded, so before its rounding to 8 bits a value is off by up to 2^-23 of y / scale: about one in 4 million, next
// to a tie, takes the neighbouring number.  A division for each value costs 2 to 19 % of the kernel's time (75,776 x 768 by row
// 61.7 -> 63.2 us, 4000 x 16384 fp32 by 128 columns 100.7 -> 119.8).
// s also leaves as fp16 where the caller wants it (the next residual); the statistics are those of the fp32 sum, not of
// its rounded copy.  HBM bound: every byte is read and written once, a row lives in registers between the two.
// Measured on B200 (of the copy's 6.45 TB/s): 75776 x 768 fp16 69.9 us (1.03), 18645 x 1024 fp32 -> e4m3 with a scale per 128
// columns 29.1 us (0.92), per row 28.0 (0.95), 4000 x 16384 fp32 -> fp16 98.3 us (1.03); 48 x 768 2.15 us, a launch.
#include <cuda_fp8.h>

#include "common.cuh"
#include "kernels.h"
#include "../../include/bt_b200.h"

namespace bt {

namespace {

struct RmsArgs {
  const void* x;
  const __half* residual;
  const void* gamma;
  __half* sum_out;
  void* out;
  float* scales;
  const int* m_dev;
  int rows, hidden;
  float eps;
};

enum RmsOut { kRmsHalf = 0, kRmsRowScale = 1, kRmsGroupScale = 2 };

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_half2(f[0], f[1]), pack_half2(f[2], f[3]), pack_half2(f[4], f[5]), pack_half2(f[6], f[7]));
}
__device__ __forceinline__ uint2 pack8_e4m3(const float (&f)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i], f[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2], f[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// The larger of two, NaN if either is: a group with NaN gets a scale that says so.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum or maximum over the WARPS warps of a row (one warp: lanes only).  No barrier stands behind the last reads of `scratch`: each
// call in a kernel has a row of it to itself.
template <int WARPS, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? max_or_nan(v, u) : v + u;
  }
  if (WARPS == 1) return v;
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) v = MAX ? max_or_nan(v, scratch[w]) : v + scratch[w];
  return v;
}

constexpr int kRmsWarpRows = 4;  // rows (warps) of a CTA where a warp takes a row

// WARPS warps to a row, NVEC vectors of 8 columns to a lane: hidden <= WARPS * 32 * 8 * NVEC.
template <bool X_FP32, bool G_FP32, int OUT, int WARPS, int NVEC>
__global__ void __launch_bounds__(WARPS == 1 ? kRmsWarpRows * 32 : WARPS * 32, WARPS >= 12 ? 2 : 1) add_residual_rmsnorm_kernel(const RmsArgs a) {
  __shared__ float scratch[2][WARPS];
  pdl_launch_dependents();
  constexpr int kLanes = WARPS * 32;
  constexpr int kRows = WARPS == 1 ? kRmsWarpRows : 1;
  const int t = threadIdx.x % kLanes;
  const int nvec = a.hidden >> 3;
  pdl_wait();
  int rows = a.rows;
  if (a.m_dev != nullptr) rows = min(rows, *a.m_dev);
  const unsigned row = blockIdx.x * kRows + threadIdx.x / kLanes;  // (the last block's rows may pass 2^31)
  if (rows <= 0 || row >= static_cast<unsigned>(rows)) return;       // (of a row's warps all or none)
  const size_t at = static_cast<size_t>(row) * nvec;
  uint4 xv[NVEC][X_FP32 ? 2 : 1], rv[NVEC];
#pragma unroll
  for (int i = 0; i < NVEC; ++i) {
    const int v = i * kLanes + t;
    if (v >= nvec) continue;
    if (X_FP32) {
      xv[i][0] = reinterpret_cast<const uint4*>(a.x)[(at + v) * 2];
      xv[i][X_FP32 ? 1 : 0] = reinterpret_cast<const uint4*>(a.x)[(at + v) * 2 + 1];
    } else {
      xv[i][0] = reinterpret_cast<const uint4*>(a.x)[at + v];
    }
    rv[i] = a.residual != nullptr ? reinterpret_cast<const uint4*>(a.residual)[at + v] : make_uint4(0u, 0u, 0u, 0u);
  }
  float s[NVEC][8];
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NVEC; ++i) {
    const int v = i * kLanes + t;
    if (v < nvec) {
      float r[8];
      unpack8(rv[i], r);
      if (X_FP32) {
        const uint32_t w[8] = {xv[i][0].x, xv[i][0].y, xv[i][0].z, xv[i][0].w, xv[i][X_FP32 ? 1 : 0].x, xv[i][X_FP32 ? 1 : 0].y,
                               xv[i][X_FP32 ? 1 : 0].z, xv[i][X_FP32 ? 1 : 0].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] = __uint_as_float(w[j]);
      } else {
        unpack8(xv[i][0], s[i]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[i][j] += r[j];
        sq = fmaf(s[i][j], s[i][j], sq);
      }
      if (a.sum_out != nullptr) reinterpret_cast<uint4*>(a.sum_out)[at + v] = pack8(s[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[i][j] = 0.f;
    }
  }
  sq = row_reduce<WARPS, false>(sq, scratch[0]);
  const float rstd = 1.0f / sqrtf(sq / static_cast<float>(a.hidden) + a.eps);
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < NVEC; ++i) {
    const int v = i * kLanes + t;
    if (v < nvec) {
      float g[8];
      if (G_FP32) {
        const float4 g0 = __ldg(reinterpret_cast<const float4*>(a.gamma) + 2 * v);
        const float4 g1 = __ldg(reinterpret_cast<const float4*>(a.gamma) + 2 * v + 1);
        g[0] = g0.x; g[1] = g0.y; g[2] = g0.z; g[3] = g0.w; g[4] = g1.x; g[5] = g1.y; g[6] = g1.z; g[7] = g1.w;
      } else {
        unpack8(__ldg(reinterpret_cast<const uint4*>(a.gamma) + v), g);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[i][j] = s[i][j] * rstd * g[j];
        if (OUT == kRmsRowScale) top = max_or_nan(top, fabsf(s[i][j]));
      }
      if (OUT == kRmsHalf) reinterpret_cast<uint4*>(a.out)[at + v] = pack8(s[i]);
    }
  }
  if (OUT == kRmsRowScale) {
    top = row_reduce<WARPS, true>(top, scratch[1]);
    const float scale = max_or_nan(top, 0x1p-100f) / 448.0f;
    const float inv = 1.0f / scale;
    if (t == 0) a.scales[row] = scale;
#pragma unroll
    for (int i = 0; i < NVEC; ++i) {
      const int v = i * kLanes + t;
      if (v < nvec) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] *= inv;
        reinterpret_cast<uint2*>(a.out)[at + v] = pack8_e4m3(s[i]);
      }
    }
  }
  if (OUT == kRmsGroupScale) {
    const int groups = (a.hidden + 127) / 128;
#pragma unroll
    for (int i = 0; i < NVEC; ++i) {  // sixteen neighbouring lanes hold a group (those without columns hold zeros)
      const int v = i * kLanes + t;
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max_or_nan(m, fabsf(s[i][j]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = max_or_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float scale = max_or_nan(m, 0x1p-100f) / 448.0f;
      const float inv = 1.0f / scale;
      if (v < nvec) {
        if ((t & 15) == 0) a.scales[static_cast<size_t>(row) * groups + (v >> 4)] = scale;
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] *= inv;
        reinterpret_cast<uint2*>(a.out)[at + v] = pack8_e4m3(s[i]);
      }
    }
  }
}

template <bool X_FP32, bool G_FP32, int OUT, int WARPS, int NVEC>
cudaError_t launch_one(const RmsArgs& a, cudaStream_t stream) {
  constexpr int kRows = WARPS == 1 ? kRmsWarpRows : 1;
  return launch_pdl(add_residual_rmsnorm_kernel<X_FP32, G_FP32, OUT, WARPS, NVEC>, dim3((static_cast<unsigned>(a.rows) + kRows - 1) / kRows),
                    dim3(WARPS == 1 ? kRmsWarpRows * 32 : WARPS * 32), 0, stream, a);
}

template <bool X_FP32, bool G_FP32, int OUT>
cudaError_t launch_by_width(const RmsArgs& a, cudaStream_t stream) {
  // A warp to a row as far as four vectors to a lane go; beyond, as many warps as leave two to four.  Rows of more than 8192 keep two
  // CTAs to an SM by registers (one: 4000 x 16384 fp32 107.9 us instead of 98.3).
  const int nvec = a.hidden / 8;
  if (nvec <= 32) return launch_one<X_FP32, G_FP32, OUT, 1, 1>(a, stream);
  if (nvec <= 64) return launch_one<X_FP32, G_FP32, OUT, 1, 2>(a, stream);
  if (nvec <= 96) return launch_one<X_FP32, G_FP32, OUT, 1, 3>(a, stream);
  if (nvec <= 128) return launch_one<X_FP32, G_FP32, OUT, 1, 4>(a, stream);
  if (nvec <= 256) return launch_one<X_FP32, G_FP32, OUT, 4, 2>(a, stream);
  if (nvec <= 512) return launch_one<X_FP32, G_FP32, OUT, 8, 2>(a, stream);
  if (nvec <= 1024) return launch_one<X_FP32, G_FP32, OUT, 8, 4>(a, stream);
  if (nvec <= 1536) return launch_one<X_FP32, G_FP32, OUT, 12, 4>(a, stream);
  return launch_one<X_FP32, G_FP32, OUT, 16, 4>(a, stream);
}

template <int OUT>
cudaError_t launch_rms(const RmsArgs& a, bool x_fp32, bool g_fp32, cudaStream_t stream) {
  if (x_fp32) return g_fp32 ? launch_by_width<true, true, OUT>(a, stream) : launch_by_width<true, false, OUT>(a, stream);
  return g_fp32 ? launch_by_width<false, true, OUT>(a, stream) : launch_by_width<false, false, OUT>(a, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int rms(const void* x, int x_fp32, const void* residual, const void* gamma, int gamma_fp32, void* sum_out, void* out,
        float* scales, int kind, const int* m_dev, int m_rows, int hidden, float eps, void* stream) {
  if (!x || !gamma || !out || m_rows <= 0 || hidden <= 0 || hidden % 8 != 0 || hidden > 16384 || !(eps >= 0.f)) return BT_ERR_INVALID_ARG;
  if (!aligned16(x) || !aligned16(residual) || !aligned16(gamma) || !aligned16(sum_out) || !aligned16(out)) return BT_ERR_INVALID_ARG;
  // In place only element for element: rows go on at once, and where elements differ in size one row's results lie on another's
  // input.
  if (out == sum_out || (out == x && (x_fp32 || kind != kRmsHalf)) || (out == residual && kind != kRmsHalf) || (sum_out == x && x_fp32))
    return BT_ERR_INVALID_ARG;
  RmsArgs a{x, static_cast<const __half*>(residual), gamma, static_cast<__half*>(sum_out), out, scales, m_dev, m_rows, hidden, eps};
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (kind == kRmsHalf)
    e = launch_rms<kRmsHalf>(a, x_fp32 != 0, gamma_fp32 != 0, s);
  else if (kind == kRmsRowScale)
    e = launch_rms<kRmsRowScale>(a, x_fp32 != 0, gamma_fp32 != 0, s);
  else
    e = launch_rms<kRmsGroupScale>(a, x_fp32 != 0, gamma_fp32 != 0, s);
  return e == cudaSuccess ? BT_OK : BT_ERR_CUDA;
}

}  // namespace

}  // namespace bt

using namespace bt;

extern "C" {

int bt_add_residual_rmsnorm(const void* x, int x_fp32, const void* residual, const void* gamma, int gamma_fp32, void* sum_out,
                            void* out, const int* m_dev, int m_rows, int hidden, float eps, void* stream) {
  return rms(x, x_fp32, residual, gamma, gamma_fp32, sum_out, out, nullptr, kRmsHalf, m_dev, m_rows, hidden, eps, stream);
}

int bt_add_residual_rmsnorm_e4m3(const void* x, int x_fp32, const void* residual, const void* gamma, int gamma_fp32,
                                 void* sum_out, void* out, float* scales, int group, const int* m_dev, int m_rows, int hidden,
                                 float eps, void* stream) {
  if (!scales || (reinterpret_cast<uintptr_t>(scales) & 3u) != 0 || (group != 0 && group != 128)) return BT_ERR_INVALID_ARG;
  return rms(x, x_fp32, residual, gamma, gamma_fp32, sum_out, out, scales, group == 0 ? kRmsRowScale : kRmsGroupScale, m_dev,
             m_rows, hidden, eps, stream);
}

}  // extern "C"
