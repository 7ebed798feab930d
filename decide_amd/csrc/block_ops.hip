// Forward kernels of the training-block operators: LayerNorm, dropout, and the
// residual boundary made of both.
#include <algorithm>

#include "block_ops.hpp"

namespace {

constexpr int kThreads = 256;

// The sum of v over the workgroup, in every thread.
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

// One workgroup per row.
template <class X, class S, class Y, bool BOUNDARY>
__global__ __launch_bounds__(kThreads) void norm_kernel(NormArgs a) {
  __shared__ float lds[kThreads / 64];
  const int blocks = (a.cols + 7) / 8;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const X *x = (const X *)a.x + row * a.ldx;
    const S *in = BOUNDARY ? (const S *)a.h + row * a.ldh : (const S *)a.x + row * a.ldx;
    float sum = 0;
    for (int k = threadIdx.x; k < blocks; k += kThreads) {
      const int n = a.cols - 8 * k;
      float v[8];
      load8(x + 8 * k, n, v);
      if constexpr (BOUNDARY) {
        drop8(a.mask, (uint32_t)row, k, v);
        float r[8];
        load8((const S *)a.res + row * a.ldres + 8 * k, n, r);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = (float)to_elem<S>(r[j] + v[j]);
        store8((S *)a.h + row * a.ldh + 8 * k, n, v);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) sum += v[j];
    }
    const float mean = block_sum(sum, lds) / (float)a.cols;
    float sq = 0;
    for (int k = threadIdx.x; k < blocks; k += kThreads) {
      const int n = a.cols - 8 * k;
      float v[8];
      load8(in + 8 * k, n, v);
#pragma unroll
      for (int j = 0; j < 8; j++) sq += j < n ? (v[j] - mean) * (v[j] - mean) : 0.0f;
    }
    const float rstd = 1.0f / sqrtf(block_sum(sq, lds) / (float)a.cols + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    for (int k = threadIdx.x; k < blocks; k += kThreads) {
      const int n = a.cols - 8 * k;
      float v[8], w[8], b[8];
      load8(in + 8 * k, n, v);
      if (a.w) load8(a.w + 8 * k, n, w);
      if (a.b) load8(a.b + 8 * k, n, b);
#pragma unroll
      for (int j = 0; j < 8; j++)
        v[j] = (v[j] - mean) * rstd * (a.w ? w[j] : 1.0f) + (a.b ? b[j] : 0.0f);
      store8((Y *)a.y + row * a.ldy + 8 * k, n, v);
    }
  }
}

template <class X, class Y>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropArgs a) {
  const int64_t per_row = (a.cols + 7) / 8, total = per_row * a.rows;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / per_row, k = i % per_row;
    const int n = (int)(a.cols - 8 * k < 8 ? a.cols - 8 * k : 8);
    float v[8];
    load8((const X *)a.x + row * a.ldx + 8 * k, n, v);
    drop8(a.mask, (uint32_t)row, (uint32_t)k, v);
    if (a.res) {
      float r[8];
      load8((const Y *)a.res + row * a.ldres + 8 * k, n, r);
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = r[j] + v[j];
    }
    store8((Y *)a.y + row * a.ldy + 8 * k, n, v);
  }
}

template <class X, class S, class Y, bool BOUNDARY>
hipError_t norm_launch(const NormArgs &a, hipStream_t s) {
  if (a.rows == 0) return hipSuccess;
  hipLaunchKernelGGL((norm_kernel<X, S, Y, BOUNDARY>), dim3((unsigned)std::min<int64_t>(a.rows, 1 << 20)),
                     dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

template <class T>
hipError_t norm_pick(int x_type, int y_type, const NormArgs &a, hipStream_t s) {
  if (x_type == PREC_F32)
    return y_type == PREC_F32 ? norm_launch<float, float, float, false>(a, s)
                              : norm_launch<float, float, T, false>(a, s);
  return norm_launch<T, T, T, false>(a, s);
}

template <class T>
hipError_t boundary_pick(int x_type, int stream_type, int y_type, const NormArgs &a, hipStream_t s) {
  if (stream_type != PREC_F32) return norm_launch<T, T, T, true>(a, s);
  if (y_type == PREC_F32) return norm_launch<float, float, float, true>(a, s);
  return x_type == PREC_F32 ? norm_launch<float, float, T, true>(a, s) : norm_launch<T, float, T, true>(a, s);
}

template <class X, class Y>
hipError_t dropout_launch(const DropArgs &a, hipStream_t s) {
  const int64_t total = (a.cols + 7) / 8 * a.rows;
  if (total == 0) return hipSuccess;
  hipLaunchKernelGGL((dropout_kernel<X, Y>), dim3((unsigned)std::min<int64_t>((total + kThreads - 1) / kThreads, 2048)),
                     dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

template <class T>
hipError_t dropout_pick(int x_type, int y_type, const DropArgs &a, hipStream_t s) {
  if (x_type == PREC_F32) return y_type == PREC_F32 ? dropout_launch<float, float>(a, s) : dropout_launch<float, T>(a, s);
  return y_type == PREC_F32 ? dropout_launch<T, float>(a, s) : dropout_launch<T, T>(a, s);
}

}  // namespace

hipError_t launch_norm(int x_type, int y_type, const NormArgs &a, hipStream_t s) {
  return y_type == PREC_F16 ? norm_pick<f16>(x_type, y_type, a, s) : norm_pick<bf16>(x_type, y_type, a, s);
}

hipError_t launch_boundary(int x_type, int stream_type, int y_type, const NormArgs &a, hipStream_t s) {
  return y_type == PREC_F16 ? boundary_pick<f16>(x_type, stream_type, y_type, a, s)
                            : boundary_pick<bf16>(x_type, stream_type, y_type, a, s);
}

hipError_t launch_dropout(int x_type, int y_type, const DropArgs &a, hipStream_t s) {
  return x_type == PREC_F16 || y_type == PREC_F16 ? dropout_pick<f16>(x_type, y_type, a, s)
                                                  : dropout_pick<bf16>(x_type, y_type, a, s);
}
