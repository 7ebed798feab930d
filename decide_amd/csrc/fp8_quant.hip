// RMS norm with an 8-bit output, and the block quantiser.
//
// A block's scale is its largest magnitude over the type's largest value
// (v / scale reaches the whole range; its rounding costs a relative 2^-24, the
// element's 2^-4 or 2^-3), its elements are v * (largest value / largest
// magnitude) rounded to nearest, ties to even, by the conversion instructions.
#include <algorithm>

#include "block_ops.hpp"
#include "fp8_ops.hpp"

namespace {

constexpr int kThreads = 256;
// Most workgroups of a launch (fewer than 2^32 threads); more work takes several.
constexpr int kGrid = 1 << 20;

// Magnitudes below this count as this: a block of zeros has a scale that can be
// inverted.
constexpr float kLeast = 0x1p-100f;

__device__ __forceinline__ float largest(int e5m2) { return e5m2 ? 57344.0f : 448.0f; }

// The largest v over LANES consecutive lanes, in all of them. A NaN among
// numbers is passed over: it reaches its own element alone.
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
  auto with = [&](unsigned x) { v = fmaxf(v, __uint_as_float(x)); };
  with(dpp_u32<0xB1>(__float_as_uint(v)));   // quad_perm 1,0,3,2
  with(dpp_u32<0x4E>(__float_as_uint(v)));   // quad_perm 2,3,0,1
  with(dpp_u32<0x141>(__float_as_uint(v)));  // row_half_mirror
  if constexpr (LANES >= 16) with(dpp_u32<0x140>(__float_as_uint(v)));  // row_mirror
  if constexpr (LANES >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

// N elements times `by`, rounded to 8 bits and packed (N a multiple of 4).
template <int N>
__device__ __forceinline__ void pack8(const float (&v)[N], float by, int e5m2, uint32_t (&q)[N / 4]) {
#pragma unroll
  for (int j = 0; j < N / 4; j++) {
    const float *p = v + 4 * j;
    if (e5m2) {
      const int lo = __builtin_amdgcn_cvt_pk_bf8_f32(p[0] * by, p[1] * by, 0, false);
      q[j] = (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(p[2] * by, p[3] * by, lo, true);
    } else {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(p[0] * by, p[1] * by, 0, false);
      q[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(p[2] * by, p[3] * by, lo, true);
    }
  }
}

// VEC elements at column c of a row of cols 8-bit ones; those past it are not written.
template <int VEC>
__device__ __forceinline__ void store8(uint8_t *row, int c, int cols, const float (&v)[VEC], float by, int e5m2) {
  float t[VEC < 4 ? 4 : VEC];
  uint32_t q[(VEC < 4 ? 4 : VEC) / 4];
#pragma unroll
  for (int i = 0; i < (VEC < 4 ? 4 : VEC); i++) t[i] = v[i < VEC ? i : 0];
  pack8(t, by, e5m2, q);
  if (cols - c >= VEC) {
    __builtin_memcpy(row + (unsigned)c, q, VEC);
  } else {
#pragma unroll
    for (int i = 0; i < VEC - 1; i++)
      if (c + i < cols) row[(unsigned)(c + i)] = (uint8_t)(q[i / 4] >> (8 * (i % 4)));
  }
}

// h = res + x, y = h rstd w with rstd = 1 / sqrt(mean(h^2) + eps), and y in 8
// bits: rows in registers, one read of each input and one write of each output,
// one row per thread group without a loop, as norm_kernel. Bound by HBM: 32,768 x
// 768, bf16 x and fp32 stream, 51.4 us, 5.4 TB/s (a 1 GiB copy 5.1); rows of 4,099
// columns by their ramp and drain and unaligned stores (4,001 rows 33.5 us, 4.4).
template <class X, class S, class Y, class Shape>
__global__ __launch_bounds__(Shape::MAXT) void rms_kernel(RmsArgs a, int64_t first) {
  constexpr int VEC = Shape::VEC, LPR = Shape::LPR, VPT = Shape::VPT;
  constexpr bool WAVES = LPR == 0;
  // Lanes that share a block of 128 columns (a row of fewer lanes is one block).
  constexpr int LANES = LPR && LPR < kFp8Block / VEC ? LPR : kFp8Block / VEC < 64 ? kFp8Block / VEC : 8;
  static_assert(VEC > 1 || LPR == 8, "one lane per column: rows narrower than a vector");
  __shared__ float slots[WAVES ? 16 : 1];
  const int lpr = WAVES ? blockDim.x : LPR, lane = WAVES ? threadIdx.x : threadIdx.x % lpr, cols = a.cols;
  const int64_t row = row_of<LPR>(first + (int64_t)blockIdx.x * Shape::ROWS);
  if (row >= a.rows) return;  // all threads of the row
  Raw<X, VEC> x[VPT];
  Raw<S, VEC> res[VPT];
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    const int c = VEC * (lane + j * lpr);
    x[j] = fetch<X, VEC>((const X *)a.x + row * a.ldx, c, cols);
    if (a.res) res[j] = fetch<S, VEC>((const S *)a.res + row * a.ldres, c, cols);
  }
  float v[VPT][VEC];
#pragma unroll
  for (int j = 0; j < VPT; j++) unpack<X, VEC>(x[j], cols - VEC * (lane + j * lpr), v[j]);
  if (a.res)
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const int c = VEC * (lane + j * lpr);
      if (WAVES && j > 0 && c >= cols) break;
      float r[VEC];
      unpack<S, VEC>(res[j], cols - c, r);
#pragma unroll
      for (int i = 0; i < VEC; i++) v[j][i] = (float)to_elem<S>(v[j][i] + r[i]);
      store<S, VEC>((S *)a.h + row * a.ldh, c, cols, v[j]);
    }
  float s[1] = {0.0f};
#pragma unroll
  for (int j = 0; j < VPT; j++)
#pragma unroll
    for (int i = 0; i < VEC; i++) s[0] += v[j][i] * v[j][i];
  row_sum<LPR>(s, slots);
  const float rstd = 1.0f / sqrtf(s[0] / (float)cols + a.eps);
  if (lane == 0 && a.rstd) a.rstd[row] = rstd;
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    const int c = VEC * (lane + j * lpr);
    if (WAVES && j > 0 && VEC * ((lane & ~63) + j * lpr) >= cols) break;  // a block's lanes stay together
    float w[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) w[i] = 1.0f;
    if (a.w) load<float, VEC>(a.w, c, cols, w);
    if (a.q) {
      // y / scale without y's own rounding: rstd, which all of a block shares,
      // cancels. Not so in a block whose y or h w is zeros, tiny or not finite,
      // where rstd times either side's inverse would leave fp32's range: y itself.
      float p[VEC], most = 0.0f;
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        p[i] = v[j][i] * w[i];
        most = fmaxf(most, fabsf(p[i]));
      }
      most = lanes_max<LANES>(most);
      float of_y = most * rstd;
      if (!(most >= kLeast && of_y >= kLeast && of_y < INFINITY)) {
        most = kLeast;
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          p[i] = v[j][i] * rstd * w[i];
          most = fmaxf(most, fabsf(p[i]));
        }
        of_y = most = lanes_max<LANES>(most);
      }
      const float top = largest(a.e5m2);
      store8<VEC>((uint8_t *)a.q + row * a.ldq, c, cols, p, top / most, a.e5m2);
      if (lane % LANES == 0 && c < cols) a.scale[c / kFp8Block * a.ldscale + row] = of_y / top;
    }
    if (a.y) {
#pragma unroll
      for (int i = 0; i < VEC; i++) v[j][i] = v[j][i] * rstd * w[i];
      store<Y, VEC>((Y *)a.y + row * a.ldy, c, cols, v[j]);
    }
  }
}

template <class X, class S, class Y>
hipError_t rms_launch(const RmsArgs &a, hipStream_t s) {
  auto run = [&](auto shape) -> hipError_t {
    using Shape = decltype(shape);
    for (int64_t first = 0; first < a.rows; first += (int64_t)kGrid * Shape::ROWS) {
      const int64_t rows = std::min<int64_t>(a.rows - first, (int64_t)kGrid * Shape::ROWS);
      hipLaunchKernelGGL((rms_kernel<X, S, Y, Shape>), dim3((unsigned)((rows + Shape::ROWS - 1) / Shape::ROWS)),
                         dim3(Shape::threads(a.cols)), 0, s, a, first);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  };
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

template <class T>
hipError_t rms_pick(int x_type, int stream_type, int y_type, const RmsArgs &a, hipStream_t s) {
  if (stream_type != PREC_F32) return rms_launch<T, T, T>(a, s);
  if (y_type == PREC_F32) return rms_launch<float, float, float>(a, s);
  return x_type == PREC_F32 ? rms_launch<float, float, T>(a, s) : rms_launch<T, float, T>(a, s);
}

// Blocks of 1 x 128 of rows: 128 / VEC lanes a block, consecutive blocks of a
// row side by side. Blocks are numbered from `first` on in row order. Bound by the
// launch at 112 x 1,152 (5.8 us a call), by HBM where bytes count: bf16 12,288 x
// 2,304 16.5 us, 5.2 TB/s, x 4,099 31.5 us, 4.9; fp32 12,288 x 768 10.1 us, 4.7.
template <class X, int VEC, int LANES>
__global__ __launch_bounds__(kThreads) void quantise_rows_kernel(QuantArgs a, int64_t first, uint32_t per_row) {
  const int lane = threadIdx.x % LANES, cols = (int)a.cols;
  const int64_t block = first + (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  // first < rows * per_row, which passes 32 bits in arrays of over 2^39 elements alone.
  const int64_t row = block >> 32 ? block / per_row : (uint32_t)block / per_row;
  if (row >= a.rows) return;  // all lanes of the block
  const int b = (int)(block - row * per_row), c = b * kFp8Block + VEC * lane;
  float v[VEC];
  load<X, VEC>((const X *)a.x + row * a.ldx, c, cols, v);
  float most = kLeast;
#pragma unroll
  for (int i = 0; i < VEC; i++) most = fmaxf(most, fabsf(v[i]));
  most = lanes_max<LANES>(most);
  const float top = largest(a.e5m2);
  store8<VEC>((uint8_t *)a.q + row * a.ldq, c, cols, v, top / most, a.e5m2);
  if (lane == 0) a.scale[b * a.ldscale + row] = most / top;
}

// 128 x 128 elements of x as values and as their transpose, one read. Thread
// (rg, cg) holds rows 8 rg .. + 7 of columns 8 cg .. + 7; a row's block is 16
// lanes, a column's 16 rows of threads (four of a wave, then the waves through
// LDS). The transpose goes through LDS in runs of eight rows, swizzled by the
// column group so that neither side's accesses share a bank. 12,288 x 2,304 bf16
// into both: 29.2 us, 3.9 TB/s (a 1 GiB copy 5.1); blocks of 128 x 128 into both:
// 8,192 x 4,096 fp32 41 us, 4.9 TB/s, 8,192 x 8,192 bf16 60 us, 4.5.
template <class X>
__global__ __launch_bounds__(kThreads) void quantise_tile_kernel(QuantArgs a, int64_t first, uint32_t per_row) {
  constexpr int T = kFp8Block;
  __shared__ float most_of[4][T];
  __shared__ __attribute__((aligned(16))) uint8_t turned[T * T];
  const int64_t tile = first + blockIdx.x;
  const int64_t rb = tile / per_row, cb = tile - rb * per_row;
  const int64_t r0 = rb * T, c0 = cb * T;
  const int rows = (int)min((int64_t)T, a.rows - r0), cols = (int)min((int64_t)T, a.cols - c0);
  const int cg = threadIdx.x % 16, rg = threadIdx.x / 16, wave = threadIdx.x / 64;
  const float top = largest(a.e5m2);
  float v[8][8];
  Raw<X, 8> raw[8];
  if (a.cols >= 8) {
#pragma unroll
    for (int p = 0; p < 8; p++)
      raw[p] = fetch<X, 8>((const X *)a.x + (r0 + min(8 * rg + p, rows - 1)) * a.ldx, (int)(c0 + 8 * cg), (int)a.cols);
#pragma unroll
    for (int p = 0; p < 8; p++) unpack<X, 8>(raw[p], 8 * rg + p < rows ? cols - 8 * cg : 0, v[p]);
  } else {
#pragma unroll
    for (int p = 0; p < 8; p++)
#pragma unroll
      for (int i = 0; i < 8; i++)
        v[p][i] = 8 * rg + p < rows && 8 * cg + i < cols
                      ? (float)((const X *)a.x)[(r0 + 8 * rg + p) * a.ldx + 8 * cg + i]
                      : 0.0f;
  }
  float row_most[8], col_most[8];
#pragma unroll
  for (int i = 0; i < 8; i++) row_most[i] = col_most[i] = kLeast;
#pragma unroll
  for (int p = 0; p < 8; p++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      row_most[p] = fmaxf(row_most[p], fabsf(v[p][i]));
      col_most[i] = fmaxf(col_most[i], fabsf(v[p][i]));
    }
  if (a.qt || a.square) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(col_most[i]), __float_as_uint(col_most[i]), false, false);
      col_most[i] = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
      r = __builtin_amdgcn_permlane32_swap(__float_as_uint(col_most[i]), __float_as_uint(col_most[i]), false, false);
      col_most[i] = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
      if (threadIdx.x % 64 < 16) most_of[wave][8 * cg + i] = col_most[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++)
      col_most[i] = fmaxf(fmaxf(most_of[0][8 * cg + i], most_of[1][8 * cg + i]),
                          fmaxf(most_of[2][8 * cg + i], most_of[3][8 * cg + i]));
  }
  if (a.square) {
    float most = kLeast;
#pragma unroll
    for (int i = 0; i < 8; i++) most = fmaxf(most, col_most[i]);
    most = lanes_max<16>(most);
#pragma unroll
    for (int i = 0; i < 8; i++) row_most[i] = col_most[i] = most;
    if (threadIdx.x == 0) {
      if (a.q) a.scale[cb * a.ldscale + rb] = most / top;
      if (a.qt) a.scalet[rb * a.ldscalet + cb] = most / top;
    }
  }
  if (a.q) {
#pragma unroll
    for (int p = 0; p < 8; p++) {
      if (!a.square) row_most[p] = lanes_max<16>(row_most[p]);
      if (8 * rg + p < rows) {
        const int64_t row = r0 + 8 * rg + p;
        store8<8>((uint8_t *)a.q + row * a.ldq + c0, 8 * cg, cols, v[p], top / row_most[p], a.e5m2);
        if (!a.square && cg == 0) a.scale[cb * a.ldscale + row] = row_most[p] / top;
      }
    }
  }
  if (!a.qt) return;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    float t[8];
    uint32_t q[2];
#pragma unroll
    for (int p = 0; p < 8; p++) t[p] = v[p][i];
    pack8(t, top / col_most[i], a.e5m2, q);
    *(uint2 *)(turned + (8 * cg + i) * T + 8 * (rg ^ cg)) = make_uint2(q[0], q[1]);
    if (!a.square && rg == 0 && 8 * cg + i < cols) a.scalet[rb * a.ldscalet + c0 + 8 * cg + i] = col_most[i] / top;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const int c = 32 * k + threadIdx.x / 8, r = threadIdx.x % 8 * 16, g = c / 8;
    if (c >= cols || r >= rows) continue;
    const uint4 u = *(const uint4 *)(turned + c * T + 16 * (r / 16 ^ g / 2));
    const uint4 w = g & 1 ? make_uint4(u.z, u.w, u.x, u.y) : u;
    uint8_t *to = (uint8_t *)a.qt + (c0 + c) * a.ldqt + r0 + r;
    if (rows - r >= 16) {
      __builtin_memcpy(to, &w, 16);
    } else {
      const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 15; i++)
        if (r + i < rows) to[i] = (uint8_t)(q[i / 4] >> (8 * (i % 4)));
    }
  }
}

template <class X>
hipError_t quantise_launch(const QuantArgs &a, hipStream_t s) {
  const int64_t per_row = fp8_blocks(a.cols);
  const bool tiles = a.qt || a.square;
  auto run = [&](auto kernel, int64_t total, int each) {
    for (int64_t first = 0; first < total; first += (int64_t)kGrid * each) {
      const int64_t some = std::min<int64_t>(total - first, (int64_t)kGrid * each);
      hipLaunchKernelGGL(kernel, dim3((unsigned)((some + each - 1) / each)), dim3(kThreads), 0, s, a, first,
                         (uint32_t)per_row);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  };
  if (tiles) return run(quantise_tile_kernel<X>, per_row * fp8_blocks(a.rows), 1);
  constexpr int VEC = vec_of<X>, LANES = kFp8Block / VEC;
  if (a.cols < VEC) return run(quantise_rows_kernel<X, 1, 8>, per_row * a.rows, kThreads / 8);
  return run(quantise_rows_kernel<X, VEC, LANES>, per_row * a.rows, kThreads / LANES);
}

}  // namespace

hipError_t launch_rms(int x_type, int stream_type, int y_type, const RmsArgs &a, hipStream_t s) {
  return y_type == PREC_F16 ? rms_pick<f16>(x_type, stream_type, y_type, a, s)
                            : rms_pick<bf16>(x_type, stream_type, y_type, a, s);
}

hipError_t launch_quantise(int x_type, const QuantArgs &a, hipStream_t s) {
  if (x_type == PREC_F32) return quantise_launch<float>(a, s);
  return x_type == PREC_F16 ? quantise_launch<f16>(a, s) : quantise_launch<bf16>(a, s);
}
