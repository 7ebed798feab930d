// Forward kernels of the training-block operators: LayerNorm, dropout, and the
// residual boundary made of both.
#include <algorithm>

#include "block_ops.hpp"

namespace {

#ifndef DROP_GRID
#define DROP_GRID 2048
#endif
constexpr int kThreads = 256;
// Most workgroups of a launch (fewer than 2^32 threads); more rows take several.
constexpr int kGrid = 1 << 20;

// LayerNorm of rows held in registers: LPR threads per row, VPT vectors of VEC
// columns each. BOUNDARY: the row is res + dropout(x), stored to h.
template <class X, class S, class Y, bool BOUNDARY, int VEC, int LPR, int VPT>
__global__ __launch_bounds__(row_threads(LPR)) void norm_kernel(NormArgs a, int64_t first) {
  constexpr int GROUPS = row_threads(LPR) / LPR, W = LPR > 64 ? LPR / 64 : 1;
  __shared__ float slots[3 * W];
  const int lane = threadIdx.x % LPR, cols = a.cols;
  const float inv = 1.0f / (float)cols;
  const int64_t row = row_of<LPR>(first + (int64_t)blockIdx.x * GROUPS);
  if (row >= a.rows) return;  // whole groups; a row of several waves has its workgroup to itself
  Raw<X, VEC> x[VPT];
  Raw<S, VEC> res[BOUNDARY ? VPT : 1];
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    const int c = VEC * (lane + j * LPR);
    x[j] = fetch<X, VEC>((const X *)a.x + row * a.ldx, c, cols);
    if constexpr (BOUNDARY) res[j] = fetch<S, VEC>((const S *)a.res + row * a.ldres, c, cols);
  }
  float v[VPT][VEC];
#pragma unroll
  for (int j = 0; j < VPT; j++) unpack<X, VEC>(x[j], cols - VEC * (lane + j * LPR), v[j]);
  if constexpr (BOUNDARY) {
    Columns<LPR, VPT, VEC>::drop(a.mask, (uint32_t)row, lane, cols, v);
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const int c = VEC * (lane + j * LPR);
      float r[VEC];
      unpack<S, VEC>(res[j], cols - c, r);
#pragma unroll
      for (int i = 0; i < VEC; i++) v[j][i] = (float)to_elem<S>(r[i] + v[j][i]);
      store<S, VEC>((S *)a.h + row * a.ldh, c, cols, v[j]);
    }
  }
  float s[1] = {0.0f};
#pragma unroll
  for (int j = 0; j < VPT; j++)
#pragma unroll
    for (int i = 0; i < VEC; i++) s[0] += v[j][i];
  row_sum<LPR>(s, slots);
  const float mean = mul_rounded(s[0], inv);
  // The squares of the differences, and the differences' own sum: what the
  // mean's rounding leaves is taken out of both.
  float q[2] = {0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    const int n = cols - VEC * (lane + j * LPR);
#pragma unroll
    for (int i = 0; i < VEC; i++) v[j][i] -= mean;
    if (n < VEC)
#pragma unroll
      for (int i = 0; i < VEC; i++) v[j][i] = i < n ? v[j][i] : 0.0f;
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      q[0] += v[j][i];
      q[1] += v[j][i] * v[j][i];
    }
  }
  row_sum<LPR>(q, slots + W);
  const float rest = mul_rounded(q[0], inv);
  const float var = q[1] * inv - rest * rest;  // a NaN stays one
  const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + a.eps);
  if (lane == 0) {
    if (a.mean) a.mean[row] = mean + rest;
    if (a.rstd) a.rstd[row] = rstd;
  }
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    const int c = VEC * (lane + j * LPR);
    float w[VEC], b[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) w[i] = 1.0f, b[i] = 0.0f;
    if (a.w) load<float, VEC>(a.w, c, cols, w);
    if (a.b) load<float, VEC>(a.b, c, cols, b);
#pragma unroll
    for (int i = 0; i < VEC; i++) v[j][i] = (v[j][i] - rest) * rstd * w[i] + b[i];
    store<Y, VEC>((Y *)a.y + row * a.ldy, c, cols, v[j]);
  }
}

// How the threads of the elementwise kernel walk over the blocks of eight
// columns: `per_row` blocks a row, the last of `tail` columns; from one of its
// blocks to its next a thread goes `rows` rows and `blocks` blocks on, and one
// row more where that passes the row's end.
struct Walk {
  uint32_t per_row, tail, rows, blocks;
};

// Elementwise: thread i takes blocks i, i + threads, ..., DEPTH of them loaded
// before the first is computed; rows, blocks and offsets are carried along
// (no product or division in the loop). NARROW: rows of less than eight
// columns, element by element.
template <class X, class Y, bool RES, bool NARROW>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropArgs a, Walk w) {
  constexpr int DEPTH = 2;
  const uint32_t first = blockIdx.x * kThreads + threadIdx.x, rows = (uint32_t)a.rows;
  uint32_t row = first / w.per_row, k = first - row * w.per_row;
  struct At {
    int64_t x, res, y;
  };
  auto along = [&](int64_t r, int64_t b) { return At{r * a.ldx + 8 * b, r * a.ldres + 8 * b, r * a.ldy + 8 * b}; };
  auto plus = [](At p, At q) { return At{p.x + q.x, RES ? p.res + q.res : 0, p.y + q.y}; };
  const At step = along(w.rows, w.blocks), wrap = along(1, -(int64_t)w.per_row);
  At at = along(row, k);
  auto read = [&](auto base, int64_t off, int n) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(base)>>;
    Raw<T, 8> q;
    if constexpr (NARROW) {
      T t[8];
#pragma unroll
      for (int j = 0; j < 8; j++) t[j] = base[off + min(j, n - 1)];
      __builtin_memcpy(&q, t, sizeof(q));
    } else {  // a partial last block as the eight elements that end with the row
      __builtin_memcpy(&q, base + off - (8 - n), sizeof(q));
    }
    return q;
  };
  while (row < rows) {
    Raw<X, 8> x[DEPTH];
    Raw<Y, 8> res[RES ? DEPTH : 1];
    uint32_t r[DEPTH], block[DEPTH];
    At to[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
      r[d] = row;
      block[d] = k;
      to[d] = at;
      // Past the last row the first block is read again: no branch stands between the loads.
      const int e = d > 0 && row >= rows ? 0 : d, n = block[e] == w.per_row - 1 ? w.tail : 8;
      x[d] = read((const X *)a.x, to[e].x, n);
      if constexpr (RES) res[d] = read((const Y *)a.res, to[e].res, n);
      row += w.rows;
      k += w.blocks;
      at = plus(at, step);
      if (k >= w.per_row) {
        k -= w.per_row;
        row++;
        at = plus(at, wrap);
      }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
      if (d > 0 && r[d] >= rows) break;
      const int n = block[d] == w.per_row - 1 ? w.tail : 8, moved = NARROW ? 8 : n;
      float v[1][8];
      unpack<X, 8>(x[d], moved, v[0]);
      Columns<1, 1, 8>::drop(a.mask, r[d], (int)block[d], 0, v);
      if constexpr (RES) {
        float z[8];
        unpack<Y, 8>(res[d], moved, z);
#pragma unroll
        for (int j = 0; j < 8; j++) v[0][j] = z[j] + v[0][j];
      }
      store<Y, 8>((Y *)a.y + to[d].y, 0, n, v[0]);
    }
  }
}

template <class X, class S, class Y, bool BOUNDARY>
hipError_t norm_launch(const NormArgs &a, hipStream_t s) {
  if (a.rows == 0) return hipSuccess;
  return with_row_shape<vec_of<X, S, Y>>(a.cols, [&](auto vec, auto lpr, auto vpt) -> hipError_t {
    constexpr int VEC = vec, LPR = lpr, VPT = vpt, THREADS = row_threads(LPR), GROUPS = THREADS / LPR;
    for (int64_t first = 0; first < a.rows; first += (int64_t)kGrid * GROUPS) {
      const int64_t groups = (std::min<int64_t>(a.rows - first, (int64_t)kGrid * GROUPS) + GROUPS - 1) / GROUPS;
      hipLaunchKernelGGL((norm_kernel<X, S, Y, BOUNDARY, VEC, LPR, VPT>), dim3((unsigned)groups), dim3(THREADS), 0, s, a,
                         first);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  });
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
  const int64_t per_row = (a.cols + 7) / 8, total = per_row * a.rows;
  if (total == 0) return hipSuccess;
  // Enough threads to fill the CUs; more blocks are more rounds of the loop.
  const int64_t grid = std::min<int64_t>((total + kThreads - 1) / kThreads, DROP_GRID), threads = grid * kThreads;
  const Walk w{(uint32_t)per_row, (uint32_t)(a.cols - 8 * (per_row - 1)), (uint32_t)(threads / per_row),
               (uint32_t)(threads % per_row)};
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kThreads), 0, s, a, w);
    return hipGetLastError();
  };
  if (a.cols < 8) return a.res ? run(dropout_kernel<X, Y, true, true>) : run(dropout_kernel<X, Y, false, true>);
  return a.res ? run(dropout_kernel<X, Y, true, false>) : run(dropout_kernel<X, Y, false, false>);
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
