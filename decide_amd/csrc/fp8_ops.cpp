// C ABI of the 8-bit operators: RMS norm with an 8-bit output and its gradient,
// block quantiser, block-scaled product. As block_ops.cpp's, each call checks
// its arguments on the host and enqueues its kernels on the context's stream,
// without allocating, copying or waiting.
#include <hip/hip_runtime.h>

#include "block_ops.hpp"
#include "device_call.hpp"
#include "fp8_check.hpp"
#include "fp8_ops.hpp"

extern "C" {

int dn_add_rms_norm_device(dn_ctx *c, int x_type, int stream_type, int y_type, int q_type, int64_t rows, int cols,
                           const void *d_x, int64_t ldx, const void *d_res, int64_t ldres, const float *d_w, float eps,
                           void *d_h, int64_t ldh, void *d_y, int64_t ldy, void *d_q, int64_t ldq, float *d_scale,
                           int64_t ldscale, float *d_rstd) {
  RmsArgs a{};
  a.rows = rows;
  a.cols = cols;
  a.x = d_x;
  a.ldx = ldx;
  a.res = d_res;
  a.ldres = ldres;
  a.w = d_w;
  a.eps = eps;
  a.h = d_h;
  a.ldh = ldh;
  a.y = d_y;
  a.ldy = ldy;
  a.q = d_q;
  a.ldq = ldq;
  a.scale = d_scale;
  a.ldscale = ldscale;
  a.rstd = d_rstd;
  a.e5m2 = q_type == DN_FP8_E5M2;
  return device_call(c, "add_rms_norm", [&] { return blockchk::rms(x_type, stream_type, y_type, q_type, a); },
                     [&] { return launch_rms(x_type, stream_type, d_y ? y_type : x_type, a, c->stream); });
}

int dn_add_rms_norm_backward_device(dn_ctx *c, int dy_type, int stream_type, int dx_type, int64_t rows, int cols,
                                    const void *d_dy, int64_t lddy, const void *d_dh, int64_t lddh, const void *d_h,
                                    int64_t ldh, const float *d_w, const float *d_rstd, void *d_dres, int64_t lddres,
                                    void *d_dx, int64_t lddx, float *d_dw, int accumulate, void *d_work,
                                    int64_t work_bytes) {
  NormGradArgs a{};
  a.rows = rows;
  a.cols = cols;
  a.dy = d_dy;
  a.lddy = lddy;
  a.dh = d_dh;
  a.lddh = lddh;
  a.h = d_h;
  a.ldh = ldh;
  a.w = d_w;
  a.rstd = d_rstd;
  a.dres = d_dres;
  a.lddres = lddres;
  a.dx = d_dx;
  a.lddx = lddx;
  a.dw = d_dw;
  a.accumulate = accumulate ? 1 : 0;
  a.work = (float *)d_work;
  const int64_t bytes = dn_norm_backward_workspace(rows, cols);  // -1: sizes that the checks refuse
  return device_call(c, "add_rms_norm_backward",
                     [&] {
                       return blockchk::rms_grad(dy_type, stream_type, dx_type, a, bytes > 0 ? bytes / 4 : 0,
                                                 work_bytes);
                     },
                     [&] { return launch_rms_grad(dy_type, stream_type, d_dx ? dx_type : dy_type, a, c->stream); });
}

int dn_quantize_blocks_device(dn_ctx *c, int x_type, int q_type, int64_t rows, int64_t cols, int block_rows,
                              const void *d_x, int64_t ldx, void *d_q, int64_t ldq, float *d_scale, int64_t ldscale,
                              void *d_qt, int64_t ldqt, float *d_scalet, int64_t ldscalet) {
  QuantArgs a{};
  a.rows = rows;
  a.cols = cols;
  a.x = d_x;
  a.ldx = ldx;
  a.q = d_q;
  a.ldq = ldq;
  a.scale = d_scale;
  a.ldscale = ldscale;
  a.qt = d_qt;
  a.ldqt = ldqt;
  a.scalet = d_scalet;
  a.ldscalet = ldscalet;
  a.square = block_rows == kFp8Block;
  a.e5m2 = q_type == DN_FP8_E5M2;
  return device_call(c, "quantize_blocks", [&] { return blockchk::quantise(x_type, q_type, block_rows, a); },
                     [&] { return rows && cols ? launch_quantise(x_type, a, c->stream) : hipSuccess; });
}

int64_t dn_gemm_fp8_workspace(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || M > blockchk::kMaxFp8 || N < 0 || N > blockchk::kMaxFp8Out || K < 0 || K > blockchk::kMaxFp8) return -1;
  return gemm_fp8_work(M, N, K) * (int64_t)sizeof(float);
}

int dn_gemm_fp8_device(dn_ctx *c, int a_type, int b_type, int c_type, int64_t M, int64_t N, int64_t K,
                       const void *d_A, int64_t lda, const float *d_sa, int64_t ldsa, const void *d_B, int64_t ldb,
                       int b_rows, const float *d_sb, int64_t ldsb, void *d_C, int64_t ldc, int accumulate,
                       void *d_work, int64_t work_bytes) {
  Fp8GemmArgs a{};
  a.M = M;
  a.N = N;
  a.K = K;
  a.A = d_A;
  a.lda = lda;
  a.sa = d_sa;
  a.ldsa = ldsa;
  a.B = d_B;
  a.ldb = ldb;
  a.sb = d_sb;
  a.ldsb = ldsb;
  a.C = d_C;
  a.ldc = ldc;
  a.b_square = b_rows == kFp8Block;
  a.accumulate = accumulate ? 1 : 0;
  a.work = (float *)d_work;
  return device_call(c, "gemm_fp8",
                     [&] {
                       const int64_t need = dn_gemm_fp8_workspace(M, N, K);  // -1: sizes that the checks refuse
                       return blockchk::gemm(a_type, b_type, c_type, b_rows, a, need > 0 ? need : 0, work_bytes);
                     },
                     [&] {
                       if (M == 0 || N == 0) return hipSuccess;
                       return launch_gemm_fp8(a_type == DN_FP8_E5M2, b_type == DN_FP8_E5M2, c_type, a, c->stream);
                     });
}

}  // extern "C"
