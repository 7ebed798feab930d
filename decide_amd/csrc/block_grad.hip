// Backward kernels of the training-block operators.
#include <algorithm>

#include "block_ops.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kRowParts = 256;  // partial sums of the weight gradients

__device__ __forceinline__ float block_sum(float v, float *lds) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; i++) s += lds[i];
  return s;
}

int row_parts(int64_t rows) { return (int)std::min<int64_t>(kRowParts, (rows + 7) / 8); }

// The input gradients, one workgroup per row: with xh = (h - mean) rstd and
// g = dy w, dres = dh + rstd (g - mean(g) - xh mean(g xh)) and dx = dropout's
// gradient of it (the forward's mask and scale), from the unrounded sum.
template <class D, class S, class X, bool BOUNDARY>
__global__ __launch_bounds__(kThreads) void norm_grad_kernel(NormGradArgs a) {
  __shared__ float lds[kThreads / 64];
  const int blocks = (a.cols + 7) / 8;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    auto terms = [&](int k, int n, float(&g)[8], float(&xh)[8]) {
      float w[8];
      load8((const D *)a.dy + row * a.lddy + 8 * k, n, g);
      load8((const S *)a.h + row * a.ldh + 8 * k, n, xh);
      if (a.w) load8(a.w + 8 * k, n, w);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        xh[j] = j < n ? (xh[j] - mean) * rstd : 0.0f;
        g[j] *= a.w ? w[j] : 1.0f;
      }
    };
    float s1 = 0, s2 = 0;
    for (int k = threadIdx.x; k < blocks; k += kThreads) {
      float g[8], xh[8];
      terms(k, a.cols - 8 * k, g, xh);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        s1 += g[j];
        s2 += g[j] * xh[j];
      }
    }
    const float c1 = block_sum(s1, lds) / (float)a.cols, c2 = block_sum(s2, lds) / (float)a.cols;
    for (int k = threadIdx.x; k < blocks; k += kThreads) {
      const int n = a.cols - 8 * k;
      float g[8], xh[8];
      terms(k, n, g, xh);
#pragma unroll
      for (int j = 0; j < 8; j++) g[j] = rstd * (g[j] - c1 - xh[j] * c2);
      if constexpr (BOUNDARY) {
        if (a.dh) {
          float r[8];
          load8((const S *)a.dh + row * a.lddh + 8 * k, n, r);
#pragma unroll
          for (int j = 0; j < 8; j++) g[j] = r[j] + g[j];
        }
      }
      store8((S *)a.dres + row * a.lddres + 8 * k, n, g);
      if constexpr (BOUNDARY) {
        drop8(a.mask, (uint32_t)row, k, g);
        store8((X *)a.dx + row * a.lddx + 8 * k, n, g);
      }
    }
  }
}

// Partial sums over every gridDim.y-th row: work[part][0][c] = sum dy xh,
// work[part][1][c] = sum dy.
template <class D, class S>
__global__ __launch_bounds__(kThreads) void norm_sums_kernel(NormGradArgs a) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.cols) return;
  float sw = 0, sb = 0;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float dy = (float)((const D *)a.dy)[row * a.lddy + c];
    const float h = (float)((const S *)a.h)[row * a.ldh + c];
    sw += dy * ((h - a.mean[row]) * a.rstd[row]);
    sb += dy;
  }
  float *out = a.work + (int64_t)blockIdx.y * 2 * a.cols;
  out[c] = sw;
  out[a.cols + c] = sb;
}

__global__ __launch_bounds__(kThreads) void norm_sums_join_kernel(NormGradArgs a, int parts) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.cols) return;
  float sw = 0, sb = 0;
  for (int p = 0; p < parts; p++) {
    sw += a.work[(int64_t)p * 2 * a.cols + c];
    sb += a.work[((int64_t)p * 2 + 1) * a.cols + c];
  }
  if (a.dw) a.dw[c] = a.accumulate ? a.dw[c] + sw : sw;
  if (a.db) a.db[c] = a.accumulate ? a.db[c] + sb : sb;
}

template <class D, class S, class X, bool BOUNDARY>
hipError_t grad_launch(const NormGradArgs &a, hipStream_t s) {
  const int parts = row_parts(a.rows);
  const unsigned cb = (unsigned)((a.cols + kThreads - 1) / kThreads);
  if (a.dw || a.db) {
    // The sums first: dres may be written over dy or h.
    if (parts > 0) {
      hipLaunchKernelGGL((norm_sums_kernel<D, S>), dim3(cb, parts), dim3(kThreads), 0, s, a);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(norm_sums_join_kernel, dim3(cb), dim3(kThreads), 0, s, a, parts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (a.rows == 0) return hipSuccess;
  hipLaunchKernelGGL((norm_grad_kernel<D, S, X, BOUNDARY>), dim3((unsigned)std::min<int64_t>(a.rows, 1 << 20)),
                     dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

template <class T>
hipError_t norm_grad_pick(int dy_type, int x_type, const NormGradArgs &a, hipStream_t s) {
  if (x_type == PREC_F32)
    return dy_type == PREC_F32 ? grad_launch<float, float, float, false>(a, s)
                               : grad_launch<T, float, float, false>(a, s);
  return grad_launch<T, T, T, false>(a, s);
}

template <class T>
hipError_t boundary_grad_pick(int dy_type, int stream_type, int dx_type, const NormGradArgs &a, hipStream_t s) {
  if (stream_type != PREC_F32) return grad_launch<T, T, T, true>(a, s);
  if (dx_type == PREC_F32) return grad_launch<float, float, float, true>(a, s);
  return dy_type == PREC_F32 ? grad_launch<float, float, T, true>(a, s) : grad_launch<T, float, T, true>(a, s);
}

}  // namespace

int64_t norm_grad_work(int64_t rows, int cols) { return (int64_t)row_parts(rows) * 2 * cols; }

hipError_t launch_norm_grad(int dy_type, int x_type, const NormGradArgs &a, hipStream_t s) {
  return dy_type == PREC_F16 ? norm_grad_pick<f16>(dy_type, x_type, a, s) : norm_grad_pick<bf16>(dy_type, x_type, a, s);
}

hipError_t launch_boundary_grad(int dy_type, int stream_type, int dx_type, const NormGradArgs &a, hipStream_t s) {
  return dx_type == PREC_F16 ? boundary_grad_pick<f16>(dy_type, stream_type, dx_type, a, s)
                             : boundary_grad_pick<bf16>(dy_type, stream_type, dx_type, a, s);
}
