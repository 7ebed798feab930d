// Argument checks of the 8-bit operators (fp8_ops.cpp), host code without HIP.
// Each returns {0, ""} or the status and message of a refusal.
#pragma once

#include "block_check.hpp"
#include "fp8_args.hpp"

namespace blockchk {

inline bool known8(int t) { return t == DN_FP8_E4M3 || t == DN_FP8_E5M2; }

// Rows, columns and depth of an 8-bit array: a tile's number and a place
// inside a row fit 32 bits.
constexpr int64_t kMaxFp8 = 0x7fffffff;
// Columns of a product: a row of tiles is one launch.
constexpr int64_t kMaxFp8Out = 1 << 26;

inline Refusal rms(int x_type, int stream_type, int y_type, int q_type, const RmsArgs &a) {
  const char *op = "dn_add_rms_norm_device";
  if (!a.y) y_type = x_type;
  BLOCKCHK(types(op, known(x_type) && known(stream_type) && known(y_type) && known8(q_type),
                 boundary_types_ok(x_type, stream_type, y_type) && (a.res || x_type == stream_type)));
  BLOCKCHK(sizes(op, a.rows, a.cols, 1, kNormMaxCols));
  BLOCKCHK(epsilon(op, a.eps));
  if (!a.y && !a.q && a.rows > 0) return {DN_INVALID_ARG, said(op) + "y and q are both NULL"};
  const int64_t R = a.rows, C = a.cols;
  const Array v[] = {{"x", a.x, R, C, a.ldx, width(x_type), false, true, true},
                     {"res", a.res, R, C, a.ldres, width(stream_type), false, false, true},
                     {"h", a.res ? a.h : nullptr, R, C, a.ldh, width(stream_type), true, a.res != nullptr, true},
                     {"y", a.y, R, C, a.ldy, width(y_type), true, false, true},
                     {"q", a.q, R, C, a.ldq, 1, true, false, true},
                     {"scale", a.q ? a.scale : nullptr, fp8_blocks(C), R, a.ldscale, 4, true, a.q != nullptr, false},
                     {"w", a.w, 1, C, C, 4, false, false, false},
                     {"rstd", a.rstd, 1, R, R, 4, true, false, false}};
  return arrays(op, v, 8);
}

inline Refusal rms_grad(int dy_type, int stream_type, int dx_type, const NormGradArgs &a, int64_t work_floats,
                        int64_t work_bytes) {
  const char *op = "dn_add_rms_norm_backward_device";
  if (!a.dx) dx_type = dy_type;
  BLOCKCHK(types(op, known(dy_type) && known(stream_type) && known(dx_type),
                 boundary_types_ok(dy_type, stream_type, dx_type)));
  BLOCKCHK(sizes(op, a.rows, a.cols, 1, kNormMaxCols));
  const int64_t R = a.rows, C = a.cols, W = a.dw ? work_floats : 0;
  if (work_bytes < 4 * W) return {DN_INVALID_ARG, said(op) + "the workspace is too small"};
  const Array v[] = {{"dy", a.dy, R, C, a.lddy, width(dy_type), false, true, true},
                     {"dh", a.dh, R, C, a.lddh, width(stream_type), false, false, true},
                     {"h", a.h, R, C, a.ldh, width(stream_type), false, true, true},
                     {"w", a.w, 1, C, C, 4, false, false, false},
                     {"rstd", a.rstd, 1, R, R, 4, false, true, false},
                     {"dres", a.dres, R, C, a.lddres, width(stream_type), true, true, true},
                     {"dx", a.dx, R, C, a.lddx, width(dx_type), true, false, true},
                     {"dw", a.dw, 1, C, C, 4, true, false, false},
                     {"work", a.work, 1, W, W, 4, true, true, false}};
  return arrays(op, v, 9);
}

inline Refusal quantise(int x_type, int q_type, int block_rows, const QuantArgs &a) {
  const char *op = "dn_quantize_blocks_device";
  BLOCKCHK(types(op, known(x_type) && known8(q_type), true));
  if (block_rows != 1 && block_rows != kFp8Block)
    return {DN_INVALID_ARG, said(op) + "a block has 1 or 128 rows"};
  BLOCKCHK(sizes(op, a.rows, a.cols, 0, kMaxFp8));
  if (!a.q && !a.qt && a.rows > 0 && a.cols > 0) return {DN_INVALID_ARG, said(op) + "q and qt are both NULL"};
  const int64_t R = a.rows, C = a.cols;
  const int64_t SR = block_rows == 1 ? R : fp8_blocks(R), SC = block_rows == 1 ? C : fp8_blocks(C);
  const Array v[] = {{"x", a.x, R, C, a.ldx, width(x_type), false, true, false},
                     {"q", a.q, R, C, a.ldq, 1, true, false, false},
                     {"scale", a.q ? a.scale : nullptr, fp8_blocks(C), SR, a.ldscale, 4, true, a.q != nullptr, false},
                     {"qt", a.qt, C, R, a.ldqt, 1, true, false, false},
                     {"scalet", a.qt ? a.scalet : nullptr, fp8_blocks(R), SC, a.ldscalet, 4, true, a.qt != nullptr,
                      false}};
  return arrays(op, v, 5);
}

inline Refusal gemm_sizes(const char *op, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0) return {DN_INVALID_ARG, said(op) + "a size is negative"};
  if (M > kMaxFp8 || N > kMaxFp8Out || K > kMaxFp8)
    return {DN_UNSUPPORTED, said(op) + "M and K of at most 2147483647, N of at most 67108864"};
  return {};
}

inline Refusal gemm(int a_type, int b_type, int c_type, int b_rows, const Fp8GemmArgs &a, int64_t need,
                    int64_t work_bytes) {
  const char *op = "dn_gemm_fp8_device";
  BLOCKCHK(types(op, known8(a_type) && known8(b_type) && known(c_type), !a.accumulate || c_type == DN_PRECISION_FP32));
  if (b_rows != 1 && b_rows != kFp8Block) return {DN_INVALID_ARG, said(op) + "a block of B has 1 or 128 rows"};
  BLOCKCHK(gemm_sizes(op, a.M, a.N, a.K));
  if (work_bytes < need) return {DN_INVALID_ARG, said(op) + "the workspace is too small"};
  const int64_t M = a.M, N = a.N, K = a.K, W = need / 4;
  const int64_t m = N ? M : 0, n = M ? N : 0;  // an empty product reads nothing
  const Array v[] = {{"A", a.A, m, K, a.lda, 1, false, true, false},
                     {"the scale of A", a.sa, fp8_blocks(K), m, a.ldsa, 4, false, true, false},
                     {"B", a.B, n, K, a.ldb, 1, false, true, false},
                     {"the scale of B", a.sb, fp8_blocks(K), b_rows == 1 ? n : fp8_blocks(n), a.ldsb, 4, false, true,
                      false},
                     {"C", a.C, m, n, a.ldc, width(c_type), true, true, false},
                     {"work", a.work, 1, W, W, 4, true, true, false}};
  return arrays(op, v, 6);
}

}  // namespace blockchk
