// Backward kernels of the training-block operators.
#include <algorithm>

#include "block_ops.hpp"

namespace {

// Workgroups of the gradient, each with partial sums of its own that cost a
// slice of the workspace to write and to read again: up to three per CU while
// they make 16 waves together, one for wide rows.
int row_parts(int64_t rows, int cols, int rows_per_group, int threads) {
  const int most = 256 * (cols > 4096 ? 1 : std::clamp(1024 / threads, 1, 3));
  return (int)std::min<int64_t>(most, (rows + rows_per_group - 1) / rows_per_group);
}

// All gradients in one pass over rows held in registers: with xh = (h - mean) rstd and g = dy w,
// dres = dh + rstd (g - mean(g) - xh mean(g xh)) and dx = dropout's gradient of
// it (the forward's mask and scale), from the unrounded sum. Each thread adds
// dy xh and dy of its columns over its rows; a workgroup's sums go to its
// slice of the workspace, [2][cols].
template <class D, class S, class X, bool BOUNDARY, class Shape>
__global__ __launch_bounds__(Shape::MAXT) void norm_grad_kernel(NormGradArgs a) {
  constexpr int VEC = Shape::VEC, LPR = Shape::LPR, VPT = Shape::VPT;
  constexpr bool WAVES = LPR == 0;
  // The widest rows' threads have 128 registers: dh is read after the row's sums there.
  constexpr bool LATE = BOUNDARY && Shape::MAXT == 1024 && VEC * VPT == 16;
  __shared__ float slots[2][WAVES ? 32 : 1];
  const int lpr = WAVES ? blockDim.x : LPR, lane = WAVES ? threadIdx.x : threadIdx.x % lpr, cols = a.cols;
  const float inv = 1.0f / (float)cols;
  float sw[VPT][VEC], sb[VPT][VEC];
#pragma unroll
  for (int j = 0; j < VPT; j++)
#pragma unroll
    for (int i = 0; i < VEC; i++) sw[j][i] = 0.0f, sb[j][i] = 0.0f;
  int turn = 0;
  for (int64_t row = row_of<LPR>((int64_t)blockIdx.x * Shape::ROWS); row < a.rows;
       row += (int64_t)gridDim.x * Shape::ROWS, turn ^= 1) {
    // The weights are read again for every row (from the caches): held, they
    // would cost the registers of a wave per SIMD.
    const float *weight = a.w;
    asm volatile("" : "+s"(weight));
    Raw<S, VEC> h[VPT], dh[BOUNDARY ? VPT : 1];
    Raw<D, VEC> dy[VPT];
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const int c = VEC * (lane + j * lpr);
      h[j] = fetch<S, VEC>((const S *)a.h + row * a.ldh, c, cols);
      dy[j] = fetch<D, VEC>((const D *)a.dy + row * a.lddy, c, cols);
    }
    auto fetch_dh = [&] {
      if (a.dh)
#pragma unroll
        for (int j = 0; j < (BOUNDARY ? VPT : 0); j++)
          dh[j] = fetch<S, VEC>((const S *)a.dh + row * a.lddh, VEC * (lane + j * lpr), cols);
    };
    if constexpr (BOUNDARY && !LATE) fetch_dh();
    const float mean = a.mean[row], rstd = a.rstd[row];
    float g[VPT][VEC], xh[VPT][VEC];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const int c = VEC * (lane + j * lpr);
      float w[VEC];
#pragma unroll
      for (int i = 0; i < VEC; i++) w[i] = 1.0f;
      if (weight) load<float, VEC>(weight, c, cols, w);
      unpack<S, VEC>(h[j], cols - c, xh[j]);
      unpack<D, VEC>(dy[j], cols - c, g[j]);
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        // Columns past the row hold dy = 0.
        xh[j][i] = (xh[j][i] - mean) * rstd;
        sw[j][i] += g[j][i] * xh[j][i];
        sb[j][i] += g[j][i];
        g[j][i] *= w[i];
        s[0] += g[j][i];
        s[1] += g[j][i] * xh[j][i];
      }
    }
    row_sum<LPR>(s, slots[turn]);
    if constexpr (LATE) fetch_dh();
    const float c1 = mul_rounded(s[0], inv), c2 = mul_rounded(s[1], inv);
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const int c = VEC * (lane + j * lpr);
#pragma unroll
      for (int i = 0; i < VEC; i++) g[j][i] = rstd * (g[j][i] - c1 - xh[j][i] * c2);
      if constexpr (BOUNDARY)
        if (a.dh) {
          float r[VEC];
          unpack<S, VEC>(dh[j], cols - c, r);
#pragma unroll
          for (int i = 0; i < VEC; i++) g[j][i] += r[i];
        }
      store<S, VEC>((S *)a.dres + row * a.lddres, c, cols, g[j]);
    }
    if constexpr (BOUNDARY) {
      Columns<WAVES, VPT, VEC>::drop(a.mask, (uint32_t)row, lane, lpr, cols, g);
#pragma unroll
      for (int j = 0; j < VPT; j++) {
#pragma unroll
        for (int i = 0; i < VEC; i++) g[j][i] *= a.mask.scale;
        store<X, VEC>((X *)a.dx + row * a.lddx, VEC * (lane + j * lpr), cols, g[j]);
      }
    }
  }
  if (!a.work) return;
  float *out = a.work + (int64_t)blockIdx.x * 2 * cols;
  if constexpr (WAVES) {
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const int c = VEC * (lane + j * lpr);
      store<float, VEC>(out, c, cols, sw[j]);
      store<float, VEC>(out + cols, c, cols, sb[j]);
    }
  } else {
    // Rows of one wave in registers, then the four waves through LDS in order.
    constexpr int N = kRowThreads / 64, COLS = LPR * VPT * VEC;
    __shared__ float part[N][COLS];
    auto join = [&](float(&v)[VPT][VEC], float *to) {
#pragma unroll
      for (int j = 0; j < VPT; j++)
#pragma unroll
        for (int i = 0; i < VEC; i++) {
#pragma unroll
          for (int m = LPR; m < 64; m <<= 1) v[j][i] += __shfl_xor(v[j][i], m);
        }
      if ((threadIdx.x & 63) < LPR)
#pragma unroll
        for (int j = 0; j < VPT; j++)
#pragma unroll
          for (int i = 0; i < VEC; i++) part[threadIdx.x >> 6][VEC * (lane + j * lpr) + i] = v[j][i];
      __syncthreads();
      for (int c = threadIdx.x; c < cols; c += kRowThreads) {
        float t = 0;
#pragma unroll
        for (int k = 0; k < N; k++) t += part[k][c];
        to[c] = t;
      }
      __syncthreads();
    };
    join(sw, out);
    join(sb, out + cols);
  }
}

// The workgroups' sums in order: blockIdx.y 0 dw, 1 db; 16 columns of a
// workgroup, 64 threads each, whose loads are made eight at a time.
__global__ __launch_bounds__(1024) void norm_join_kernel(NormGradArgs a, int parts) {
  constexpr int COLS = 16, SPLIT = 1024 / COLS, BATCH = 8;
  __shared__ float lds[SPLIT][COLS + 1];
  float *to = blockIdx.y ? a.db : a.dw;
  if (!to) return;
  const int i = threadIdx.x % COLS, c = blockIdx.x * COLS + i, k = threadIdx.x / COLS;
  const float *from = a.work + (int64_t)blockIdx.y * a.cols + min(c, a.cols - 1);
  float s = 0;
  for (int p = k; p < parts; p += SPLIT * BATCH) {
    float v[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; j++) v[j] = from[(int64_t)min(p + j * SPLIT, parts - 1) * 2 * a.cols];
#pragma unroll
    for (int j = 0; j < BATCH; j++) s += p + j * SPLIT < parts ? v[j] : 0.0f;
  }
  lds[k][i] = s;
  __syncthreads();
  if (k < 8) {
    s = 0;
#pragma unroll
    for (int j = 0; j < SPLIT / 8; j++) s += lds[k * (SPLIT / 8) + j][i];
    lds[k * (SPLIT / 8)][i] = s;
  }
  __syncthreads();
  if (k == 0 && c < a.cols) {
    s = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) s += lds[j * (SPLIT / 8)][i];
    to[c] = a.accumulate ? to[c] + s : s;
  }
}

// The gradient's threads also hold two sums per column, so its shapes have
// fewer columns a thread than the forward's.
template <int WIDE, class F>
hipError_t with_grad_shape(int cols, F f) {
  if (cols < WIDE) return f(RowShape<1, 8, 1>{});
  if constexpr (WIDE == 8)
    return pick_shape<RowShape<8, 8, 1>, RowShape<8, 16, 1>, RowShape<8, 32, 1>, RowShape<8, 64, 1>, RowShape<8, 64, 2>,
                      RowShape<8, 0, 1, 512>, RowShape<8, 0, 2, 512>, RowShape<8, 0, 2, 1024>>(cols, f);
  else
    return pick_shape<RowShape<4, 8, 1>, RowShape<4, 16, 1>, RowShape<4, 32, 1>, RowShape<4, 64, 1>, RowShape<4, 64, 2>,
                      RowShape<4, 64, 3>, RowShape<4, 64, 4>, RowShape<4, 0, 1, 512>, RowShape<4, 0, 2, 1024>,
                      RowShape<4, 0, 4, 1024>>(cols, f);
}

template <class D, class S, class X, bool BOUNDARY>
hipError_t grad_launch(const NormGradArgs &args, hipStream_t s) {
  return with_grad_shape<vec_of<D, S, X>>(args.cols, [&](auto shape) {
    using Shape = decltype(shape);
    NormGradArgs a = args;
    const int threads = Shape::threads(a.cols), parts = row_parts(a.rows, a.cols, Shape::ROWS, threads);
    if (!a.dw && !a.db) a.work = nullptr;
    if (parts > 0)
      hipLaunchKernelGGL((norm_grad_kernel<D, S, X, BOUNDARY, Shape>), dim3(parts), dim3(threads), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && (a.dw || a.db)) {
      hipLaunchKernelGGL(norm_join_kernel, dim3((a.cols + 15) / 16, a.db ? 2 : 1), dim3(1024), 0, s, a, parts);
      e = hipGetLastError();
    }
    return e;
  });
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

// The larger of what calls with and without an fp32 array use.
int64_t norm_grad_work(int64_t rows, int cols) {
  int parts = 0;
  auto most = [&](auto shape) {
    using Shape = decltype(shape);
    parts = std::max(parts, row_parts(rows, cols, Shape::ROWS, Shape::threads(cols)));
    return hipSuccess;
  };
  (void)with_grad_shape<4>(cols, most);
  (void)with_grad_shape<8>(cols, most);
  return (int64_t)parts * 2 * cols;
}

hipError_t launch_norm_grad(int dy_type, int x_type, const NormGradArgs &a, hipStream_t s) {
  return dy_type == PREC_F16 ? norm_grad_pick<f16>(dy_type, x_type, a, s) : norm_grad_pick<bf16>(dy_type, x_type, a, s);
}

hipError_t launch_boundary_grad(int dy_type, int stream_type, int dx_type, const NormGradArgs &a, hipStream_t s) {
  return dx_type == PREC_F16 ? boundary_grad_pick<f16>(dy_type, stream_type, dx_type, a, s)
                             : boundary_grad_pick<bf16>(dy_type, stream_type, dx_type, a, s);
}
