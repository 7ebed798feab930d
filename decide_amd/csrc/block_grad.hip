// Backward kernels of the training-block operators.
#include <algorithm>

#include "block_ops.hpp"

namespace {

// Calls of at most this many rows sum each column over all of them in
// workgroups beside those of the rows: one launch (of ~3.5 us on the host)
// instead of two, for a second read of dy and h from the caches. Norm gradient,
// bf16 dy and fp32 stream, one launch and two, us (arrays in the cache):
//   columns        768          2,304          4,096          8,192
//   256 rows    5.2   7.8     5.2   8.9      7.1  11.2      7.5  16.0
//   512         5.2   8.0     9.1  11.5     15.1  15.8     14.3  16.3
//   640         5.9   7.8    10.6  12.8     19.6  15.5     18.3  17.8
//   1,024      11.4   8.3    17.1  14.6     29.0  15.7     27.6  21.9
// One number for all widths: up to 2,304 columns one launch still wins at 768
// rows; the boundary's gradient at 4,096 columns wants two from about 450 on
// (512 rows of fp32: 19.9 and 15.7).
constexpr int64_t kSmallRows = 512;
// Columns of such a workgroup: few, so that many threads share the rows, or 32
// where the columns alone make enough workgroups and narrow reads cost more
// (the same gradient at 512 rows, 8 and 32: 768 columns 5.2 and 11.6 us, 2,304
// 9.2 and 12.5, 4,000 13.6 and 14.1, 4,096 14.8 and 13.9, 6,144 22.3 and 13.5,
// 8,192 30.4 and 14.3; all in bf16 4,000 12.4 and 13.3, 4,104 12.8 and 18.8,
// 6,144 19.3 and 17.9).
__host__ __device__ constexpr int slab_cols(int cols) { return cols <= 4096 ? 8 : 32; }

// Workgroups of the gradient of many rows, each with partial sums of its own
// that cost a slice of the workspace to write and to read again: up to three
// per CU while they make 16 waves together (12,288 x 768: 768 workgroups 37.4
// us, 512 39.0, 1,024 38.2), one past 4,096 columns (4,096 x 8,192: 256
// workgroups 75 us, 512 82).
int row_parts(int64_t rows, int cols, int rows_per_group, int threads) {
  const int most = 256 * (cols > 4096 ? 1 : std::clamp(1024 / threads, 1, 3));
  return (int)std::min<int64_t>(most, (rows + rows_per_group - 1) / rows_per_group);
}

// Floats between the sums of a workgroup's dw and db, and of one workgroup and
// the next: whole float4s, the last one's rest unused.
__host__ __device__ constexpr int sum_stride(int cols) { return (cols + 3) / 4 * 4; }

// dw and db of COLS columns over all rows (of few), by one workgroup: its
// threads share the rows, eight loaded at a time, and their sums are added in
// order.
template <class D, class S, int COLS>
__device__ __forceinline__ void column_sums(const NormGradArgs &a, int slab) {
  constexpr int BATCH = 8;
  __shared__ float lds[2][1024 / COLS][COLS + 1];
  const int i = threadIdx.x % COLS, k = threadIdx.x / COLS, step = blockDim.x / COLS, rows = (int)a.rows;
  const int c = slab * COLS + i, at = min(c, a.cols - 1);
  float sw = 0.0f, sb = 0.0f;
  for (int r = k; r < rows; r += step * BATCH) {
    float dy[BATCH], h[BATCH], mean[BATCH], rstd[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; j++) {
      const int64_t row = min(r + j * step, rows - 1);
      dy[j] = (float)((const D *)a.dy)[row * a.lddy + at];
      h[j] = (float)((const S *)a.h)[row * a.ldh + at];
      mean[j] = a.mean[row];
      rstd[j] = a.rstd[row];
    }
#pragma unroll
    for (int j = 0; j < BATCH; j++) {
      if (r + j * step >= rows) break;
      sw += dy[j] * ((h[j] - mean[j]) * rstd[j]);
      sb += dy[j];
    }
  }
  lds[0][k][i] = sw;
  lds[1][k][i] = sb;
  __syncthreads();
  if (k >= 2 || c >= a.cols) return;
  float *to = k ? a.db : a.dw;
  if (!to) return;
  float s = 0.0f;
#pragma unroll 8
  for (int j = 0; j < step; j++) s += lds[k][j][i];
  to[c] = a.accumulate ? to[c] + s : s;
}

// All gradients in one pass over rows held in registers: with xh = (h - mean)
// rstd and g = dy w, dres = dh + rstd (g - mean(g) - xh mean(g xh)) and dx =
// dropout's gradient of it (the forward's mask and scale), from the unrounded
// sum. Each thread adds dy xh and dy of its columns over its rows; a
// workgroup's sums go to its slice of the workspace. SMALL: the
// workgroups past `groups` sum the columns instead.
//
// HBM-bound: 12,288 x 768 (dy bf16, stream fp32) 20 us, with dropout's gradient
// 31, both 4.7 to 4.9 TB/s; the sums that follow (norm_join_kernel) 4 to 5 us more. The
// rows of a workgroup come from a loop, since its sums live in registers; three
// to four waves per SIMD cover the loop's wait for its stores.
template <class D, class S, class X, bool BOUNDARY, bool SMALL, class Shape>
__global__ __launch_bounds__(Shape::MAXT) void norm_grad_kernel(NormGradArgs a, int groups) {
  if constexpr (SMALL)
    if ((int)blockIdx.x >= groups) {
      const int slab = blockIdx.x - groups;
      return slab_cols(a.cols) == 8 ? column_sums<D, S, 8>(a, slab) : column_sums<D, S, 32>(a, slab);
    }
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
       row += (int64_t)groups * Shape::ROWS, turn ^= 1) {
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
      // Columns past the row hold dy = 0 and xh = 0 (of h = mean: mean * rstd may be infinite where no column's xh is).
      unpack<S, VEC>(h[j], cols - c, xh[j], mean);
      unpack<D, VEC>(dy[j], cols - c, g[j]);
#pragma unroll
      for (int i = 0; i < VEC; i++) {
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
  if (SMALL || !a.work) return;
  const int stride = sum_stride(cols);
  float *out = a.work + (int64_t)blockIdx.x * 2 * stride;
  if constexpr (WAVES) {
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const int c = VEC * (lane + j * lpr);
      if (a.dw) store<float, VEC>(out, c, cols, sw[j]);
      if (a.db) store<float, VEC>(out + stride, c, cols, sb[j]);
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
    if (a.dw) join(sw, out);
    if (a.db) join(sb, out + stride);
  }
}

// The workgroups' sums in order: blockIdx.y 0 dw, 1 db; 32 columns of a
// workgroup, four per thread, the parts shared by 128 threads that load eight
// at a time; a wave's sums in registers, then the waves' through LDS.
__global__ __launch_bounds__(1024) void norm_join_kernel(NormGradArgs a, int parts) {
  constexpr int COLS = 32, SPLIT = 128, BATCH = 8;
  __shared__ float lds[16][COLS];
  float *to = blockIdx.y ? a.db : a.dw;
  if (!to) return;
  const int i = threadIdx.x % 8, k = threadIdx.x / 8, c = blockIdx.x * COLS + 4 * i;
  const int stride = sum_stride(a.cols);
  const float *from = a.work + (int64_t)blockIdx.y * stride;
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < a.cols)
    for (int p = k; p < parts; p += SPLIT * BATCH) {
      float v[BATCH][4];
#pragma unroll
      for (int j = 0; j < BATCH; j++)
        __builtin_memcpy(v[j], from + (int64_t)min(p + j * SPLIT, parts - 1) * 2 * stride + c, sizeof(v[j]));
#pragma unroll
      for (int j = 0; j < BATCH; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[e] += p + j * SPLIT < parts ? v[j][e] : 0.0f;
    }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    s[e] += __uint_as_float(dpp_u32<0x128>(__float_as_uint(s[e])));  // the other half of 16 lanes: row_ror 8
    const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(s[e]), __float_as_uint(s[e]), false, false);
    s[e] = __uint_as_float(q[0]) + __uint_as_float(q[1]);
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(s[e]), __float_as_uint(s[e]), false, false);
    s[e] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if ((threadIdx.x & 63) < 8)
#pragma unroll
    for (int e = 0; e < 4; e++) lds[threadIdx.x >> 6][4 * i + e] = s[e];
  __syncthreads();
  const int out = blockIdx.x * COLS + threadIdx.x;
  if (threadIdx.x < COLS && out < a.cols) {
    float t = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; j++) t += lds[j][threadIdx.x];
    to[out] = a.accumulate ? to[out] + t : t;
  }
}

// The gradient's threads also hold two sums per column, so its shapes have
// fewer columns a thread than the forward's. Past 4,096 columns two vectors of
// eight in 512 threads (4,096 x 8,192: 69 us) before one in 1,024 (76).
// With an fp32 array three vectors of four reach 12,288 columns without a
// spilled register, where four spill up to 39 (boundary, bf16 with an fp32
// stream, 8,200 columns: 52 and 88 us); four are what 16,384 columns need.
template <int WIDE, class F>
hipError_t with_grad_shape(int cols, F f) {
  if (cols < WIDE) return f(RowShape<1, 8, 1>{});
  if constexpr (WIDE == 8)
    return pick_shape<RowShape<8, 8, 1>, RowShape<8, 16, 1>, RowShape<8, 32, 1>, RowShape<8, 64, 1>, RowShape<8, 64, 2>,
                      RowShape<8, 0, 1, 512>, RowShape<8, 0, 2, 512>, RowShape<8, 0, 2, 1024>>(cols, f);
  else
    return pick_shape<RowShape<4, 8, 1>, RowShape<4, 16, 1>, RowShape<4, 32, 1>, RowShape<4, 64, 1>, RowShape<4, 64, 2>,
                      RowShape<4, 64, 3>, RowShape<4, 64, 4>, RowShape<4, 0, 1, 512>, RowShape<4, 0, 2, 1024>,
                      RowShape<4, 0, 3, 1024>, RowShape<4, 0, 4, 1024>>(cols, f);
}

template <class D, class S, class X, bool BOUNDARY>
hipError_t grad_launch(const NormGradArgs &args, hipStream_t s) {
  return with_grad_shape<vec_of<D, S, X>>(args.cols, [&](auto shape) {
    using Shape = decltype(shape);
    NormGradArgs a = args;
    const int threads = Shape::threads(a.cols);
    const bool sums = a.dw || a.db;
    if (a.rows <= kSmallRows) {
      const int groups = ((int)a.rows + Shape::ROWS - 1) / Shape::ROWS, slab = slab_cols(a.cols);
      const int slabs = sums ? (a.cols + slab - 1) / slab : 0;
      auto run = [&](int grid, int row_groups) {
        if (grid > 0)
          hipLaunchKernelGGL((norm_grad_kernel<D, S, X, BOUNDARY, true, Shape>), dim3(grid), dim3(threads), 0, s, a,
                             row_groups);
        return hipGetLastError();
      };
      // Where an output takes the place of what the sums read, the sums go first.
      const bool over = a.dres == a.dy || a.dres == a.h || (BOUNDARY && (a.dx == a.dy || a.dx == a.h));
      if (!over) return run(groups + slabs, groups);
      const hipError_t e = run(slabs, 0);
      return e == hipSuccess ? run(groups, groups) : e;
    }
    const int parts = row_parts(a.rows, a.cols, Shape::ROWS, threads);
    if (!sums) a.work = nullptr;
    hipLaunchKernelGGL((norm_grad_kernel<D, S, X, BOUNDARY, false, Shape>), dim3(parts), dim3(threads), 0, s, a, parts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !sums) return e;
    hipLaunchKernelGGL(norm_join_kernel, dim3((a.cols + 31) / 32, a.db ? 2 : 1), dim3(1024), 0, s, a, parts);
    return hipGetLastError();
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
  if (rows <= kSmallRows) return 0;
  int parts = 0;
  auto most = [&](auto shape) {
    using Shape = decltype(shape);
    parts = std::max(parts, row_parts(rows, cols, Shape::ROWS, Shape::threads(cols)));
    return hipSuccess;
  };
  (void)with_grad_shape<4>(cols, most);
  (void)with_grad_shape<8>(cols, most);
  return (int64_t)parts * 2 * sum_stride(cols);
}

hipError_t launch_norm_grad(int dy_type, int x_type, const NormGradArgs &a, hipStream_t s) {
  return dy_type == PREC_F16 ? norm_grad_pick<f16>(dy_type, x_type, a, s) : norm_grad_pick<bf16>(dy_type, x_type, a, s);
}

hipError_t launch_boundary_grad(int dy_type, int stream_type, int dx_type, const NormGradArgs &a, hipStream_t s) {
  return dx_type == PREC_F16 ? boundary_grad_pick<f16>(dy_type, stream_type, dx_type, a, s)
                             : boundary_grad_pick<bf16>(dy_type, stream_type, dx_type, a, s);
}
