// Forward kernels of the training-block operators: LayerNorm, dropout, and the
// residual boundary made of both.
#include <algorithm>

#include "block_ops.hpp"

namespace {

constexpr int kThreads = 256;
// Most workgroups of a launch (fewer than 2^32 threads); more rows take several.
constexpr int kGrid = 1 << 20;

// LayerNorm of rows held in registers: one read of each input, one write of
// each output. BOUNDARY: the row is res + dropout(x), stored to h.
//
// HBM-bound from a few thousand rows on; a launch's latency below. A row per
// wave (or part of one) up to 1,024 columns, a row per workgroup above, one row
// per thread group and no loop over rows: loads and stores share one counter
// (vmcnt), so that a loop's next row waits for this row's stores (32,768 x 768
// with a row prefetched in a loop 58 us, without a loop 29.5, 5.1 TB/s, the
// rate of a large copy; 12,288 rows with dropout 45 and 23.9, 4.7 TB/s). The
// weights are read after the sums, not held: at most 64 registers, eight waves
// per SIMD. 768 x 64 rows: 3.1 us on the GPU, 4.6 a call.
template <class X, class S, class Y, bool BOUNDARY, class Shape>
__global__ __launch_bounds__(Shape::MAXT) void norm_kernel(NormArgs a, int64_t first) {
  constexpr int VEC = Shape::VEC, LPR = Shape::LPR, VPT = Shape::VPT;
  constexpr bool WAVES = LPR == 0;
  __shared__ float slots[WAVES ? 48 : 1];
  const int lpr = WAVES ? blockDim.x : LPR, lane = WAVES ? threadIdx.x : threadIdx.x % lpr, cols = a.cols;
  const float inv = 1.0f / (float)cols;
  const int64_t row = row_of<LPR>(first + (int64_t)blockIdx.x * Shape::ROWS);
  if (row >= a.rows) return;  // all threads of the row
  Raw<X, VEC> x[VPT];
  Raw<S, VEC> res[BOUNDARY ? VPT : 1];
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    const int c = VEC * (lane + j * lpr);
    x[j] = fetch<X, VEC>((const X *)a.x + row * a.ldx, c, cols);
    if constexpr (BOUNDARY) res[j] = fetch<S, VEC>((const S *)a.res + row * a.ldres, c, cols);
  }
  float v[VPT][VEC];
#pragma unroll
  for (int j = 0; j < VPT; j++) unpack<X, VEC>(x[j], cols - VEC * (lane + j * lpr), v[j]);
  if constexpr (BOUNDARY) {
    Columns<WAVES, VPT, VEC>::drop(a.mask, (uint32_t)row, lane, lpr, cols, v);
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const int c = VEC * (lane + j * lpr);
      if (WAVES && j > 0 && c >= cols) break;  // waves past the row; within a wave the branch costs more
      float r[VEC];
      unpack<S, VEC>(res[j], cols - c, r);
#pragma unroll
      for (int i = 0; i < VEC; i++) v[j][i] = (float)to_elem<S>(fmaf(v[j][i], a.mask.scale, r[i]));
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
    const int n = cols - VEC * (lane + j * lpr);
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
  row_sum<LPR>(q, slots + (WAVES ? 16 : 0));
  const float rest = mul_rounded(q[0], inv);
  const float var = q[1] * inv - rest * rest;  // a NaN stays one
  const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + a.eps);
  if (lane == 0) {
    if (a.mean) a.mean[row] = mean + rest;
    if (a.rstd) a.rstd[row] = rstd;
  }
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    const int c = VEC * (lane + j * lpr);
    if (WAVES && j > 0 && c >= cols) break;
    float w[VEC], b[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) w[i] = 1.0f, b[i] = 0.0f;
    if (a.w) load<float, VEC>(a.w, c, cols, w);
    if (a.b) load<float, VEC>(a.b, c, cols, b);
    // rest is within the mean's rounding, so that its product may be rounded.
#pragma unroll
    for (int i = 0; i < VEC; i++) v[j][i] = fmaf(fmaf(v[j][i], rstd, -rest * rstd), w[i], b[i]);
    store<Y, VEC>((Y *)a.y + row * a.ldy, c, cols, v[j]);
  }
}

// Elementwise dropout. HBM-bound (32,768 x 1,152 bf16 29.4 us, 5.1 TB/s) with the
// VALU 75% busy, most of it the generator's twenty 32 x 32 -> 64-bit products
// per eight columns. No loop, for norm_kernel's reason (2,048 workgroups in a loop
// 37.8 us); rows and blocks from one 32-bit division per vector.
//
// A thread takes a vector of eight columns, or (VEC 4, with an fp32 array) two of
// four: the launch's vectors i and i + 64 of the 128 of a wave, so that a wave's
// 16-byte accesses lie side by side (fp32 12 M elements 22.0 -> 20.2 us). The two
// lanes of a generator block then share its work (drop_pair). A row has `per_row`
// blocks of eight columns, the last of `tail`; the launch starts at block k0 of
// row r0. NARROW: rows of less than eight columns, element by element.
template <class X, class Y, bool RES, bool NARROW>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropArgs a, uint32_t r0, uint32_t k0, uint32_t per_row,
                                                           uint32_t tail) {
  constexpr int VEC = NARROW ? 8 : vec_of<X, Y>, VPT = VEC == 4 ? 2 : 1;
  uint32_t row[VPT], k[VPT];
  int n[VPT], half[VPT];
  int64_t col[VPT];
  Raw<X, VEC> x[VPT];
  Raw<Y, VEC> res[VPT];
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    const uint32_t wave = (blockIdx.x * kThreads + threadIdx.x) & ~63u, lane = threadIdx.x & 63;
    const uint32_t vector = wave * VPT + lane + 64 * j;       // fewer than 2^30
    const uint32_t i = k0 + (VEC == 4 ? vector / 2 : vector);  // k0 < per_row < 2^31
    const uint32_t down = i / per_row;
    row[j] = r0 + down;
    k[j] = i - down * per_row;
    half[j] = VEC == 4 ? vector & 1 : 0;
    const int left = k[j] == per_row - 1 ? (int)tail - 4 * half[j] : VEC;
    n[j] = row[j] < (uint32_t)a.rows ? min(left, VEC) : 0;
    col[j] = 8 * (int64_t)k[j] + 4 * half[j];
  }
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    auto read = [&](auto base, int64_t ld) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(base)>>;
      Raw<T, VEC> q;
      if constexpr (NARROW) {
        T t[8];
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = n[j] > 0 ? base[row[j] * ld + min(i, n[j] - 1)] : T(0.0f);
        __builtin_memcpy(&q, t, sizeof(q));
      } else {
        // A partial vector as the VEC elements that end with the row; where there is none, the first row's first.
        const T *p = n[j] > 0 ? base + row[j] * ld + col[j] - (VEC - n[j]) : base;
        __builtin_memcpy(&q, p, sizeof(q));
      }
      return q;
    };
    x[j] = read((const X *)a.x, a.ldx);
    if constexpr (RES) res[j] = read((const Y *)a.res, a.ldres);
  }
  float v[VPT][VEC];
#pragma unroll
  for (int j = 0; j < VPT; j++) unpack<X, VEC>(x[j], NARROW ? VEC : n[j], v[j]);
  if (a.mask.threshold) {
    if constexpr (VEC == 8) {
      const uint4 r = philox(k[0], row[0], a.mask.o0, a.mask.o1, a.mask.k0, a.mask.k1);
      const uint32_t word[4] = {r.x, r.y, r.z, r.w};
      drop_by<8>(a.mask, word, v[0]);
    } else {
      const bool odd = threadIdx.x & 1;
      drop_pair(a.mask, odd, philox(odd ? k[VPT - 1] : k[0], odd ? row[VPT - 1] : row[0], a.mask.o0, a.mask.o1,
                                    a.mask.k0, a.mask.k1),
                v[0], v[VPT - 1]);
    }
  }
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    if constexpr (RES) {
      float z[VEC];
      unpack<Y, VEC>(res[j], NARROW ? VEC : n[j], z);
#pragma unroll
      for (int i = 0; i < VEC; i++) v[j][i] = fmaf(v[j][i], a.mask.scale, z[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i++) v[j][i] *= a.mask.scale;
    }
    store<Y, VEC>((Y *)a.y + row[j] * a.ldy + col[j], 0, n[j], v[j]);
  }
}

template <class X, class S, class Y, bool BOUNDARY>
hipError_t norm_launch(const NormArgs &a, hipStream_t s) {
  auto run = [&](auto shape) -> hipError_t {
    using Shape = decltype(shape);
    for (int64_t first = 0; first < a.rows; first += (int64_t)kGrid * Shape::ROWS) {
      const int64_t rows = std::min<int64_t>(a.rows - first, (int64_t)kGrid * Shape::ROWS);
      hipLaunchKernelGGL((norm_kernel<X, S, Y, BOUNDARY, Shape>), dim3((unsigned)((rows + Shape::ROWS - 1) / Shape::ROWS)),
                         dim3(Shape::threads(a.cols)), 0, s, a, first);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  };
  // Vectors per thread past 1,024 columns: 1, 2 and 3 of eight, 2, 3 and 4 of
  // four measured within 5% of each other; the most is what 16,384 columns need.
  if constexpr (vec_of<X, S, Y> == 8) {
    if (a.cols < 8) return run(RowShape<1, 8, 1>{});
    return pick_shape<RowShape<8, 8, 1>, RowShape<8, 16, 1>, RowShape<8, 32, 1>, RowShape<8, 32, 2>, RowShape<8, 32, 3>,
                      RowShape<8, 64, 2>, RowShape<8, 0, 2, 1024>>(a.cols, run);
  } else {
    if (a.cols < 4) return run(RowShape<1, 8, 1>{});
    return pick_shape<RowShape<4, 8, 1>, RowShape<4, 16, 1>, RowShape<4, 32, 1>, RowShape<4, 64, 1>, RowShape<4, 64, 2>,
                      RowShape<4, 64, 3>, RowShape<4, 64, 4>, RowShape<4, 0, 4, 1024>>(a.cols, run);
  }
}

template <class X, class Y>
hipError_t dropout_launch(const DropArgs &a, hipStream_t s) {
  const int64_t per_row = (a.cols + 7) / 8, total = per_row * a.rows, most = (int64_t)kGrid * kThreads;
  for (int64_t first = 0; first < total; first += most) {
    // A thread per block of eight columns, whether as one vector or as halves of two.
    const int64_t blocks = std::min<int64_t>(total - first, most), groups = (blocks + kThreads - 1) / kThreads;
    auto run = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(kThreads), 0, s, a, (uint32_t)(first / per_row),
                         (uint32_t)(first % per_row), (uint32_t)per_row, (uint32_t)(a.cols - 8 * (per_row - 1)));
      return hipGetLastError();
    };
    const hipError_t e = a.cols < 8
                             ? (a.res ? run(dropout_kernel<X, Y, true, true>) : run(dropout_kernel<X, Y, false, true>))
                             : (a.res ? run(dropout_kernel<X, Y, true, false>) : run(dropout_kernel<X, Y, false, false>));
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
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
