// C ABI of the training-block operators: LayerNorm, dropout and the residual
// boundary on device arrays. Each call checks its arguments on the host
// (block_check.hpp) and enqueues its kernels on the context's stream; nothing
// is allocated, copied or waited for, so the calls can be captured into a graph.
#include <hip/hip_runtime.h>

#include "block_check.hpp"
#include "block_ops.hpp"
#include "device_call.hpp"

namespace {

// Floats of workspace for sizes that the checks pass; 0 for others, which they refuse.
int64_t work_floats(int64_t rows, int cols) {
  const bool taken = rows >= 0 && rows <= blockchk::kMaxRows && cols >= 1 && cols <= kNormMaxCols;
  return taken ? norm_grad_work(rows, cols) : 0;
}

}  // namespace

extern "C" {

int dn_layer_norm_device(dn_ctx *c, int x_type, int y_type, int64_t rows, int cols, const void *d_x, int64_t ldx,
                         const float *d_w, const float *d_b, float eps, void *d_y, int64_t ldy, float *d_mean,
                         float *d_rstd) {
  NormArgs a{};
  a.rows = rows;
  a.cols = cols;
  a.x = d_x;
  a.ldx = ldx;
  a.w = d_w;
  a.b = d_b;
  a.eps = eps;
  a.y = d_y;
  a.ldy = ldy;
  a.mean = d_mean;
  a.rstd = d_rstd;
  return device_call(c, "layer_norm", [&] { return blockchk::norm(x_type, y_type, a); },
                     [&] { return launch_norm(x_type, y_type, a, c->stream); });
}

int64_t dn_norm_backward_workspace(int64_t rows, int cols) {
  if (rows < 0 || rows > blockchk::kMaxRows || cols < 1 || cols > kNormMaxCols) return -1;
  return norm_grad_work(rows, cols) * (int64_t)sizeof(float);
}

int dn_layer_norm_backward_device(dn_ctx *c, int dy_type, int x_type, int64_t rows, int cols, const void *d_dy,
                                  int64_t lddy, const void *d_x, int64_t ldx, const float *d_w, const float *d_mean,
                                  const float *d_rstd, void *d_dx, int64_t lddx, float *d_dw, float *d_db,
                                  int accumulate, void *d_work, int64_t work_bytes) {
  NormGradArgs a{};
  a.rows = rows;
  a.cols = cols;
  a.dy = d_dy;
  a.lddy = lddy;
  a.h = d_x;
  a.ldh = ldx;
  a.w = d_w;
  a.mean = d_mean;
  a.rstd = d_rstd;
  a.dres = d_dx;
  a.lddres = lddx;
  a.dw = d_dw;
  a.db = d_db;
  a.accumulate = accumulate ? 1 : 0;
  a.work = (float *)d_work;
  return device_call(c, "layer_norm_backward",
                     [&] { return blockchk::norm_grad(dy_type, x_type, a, work_floats(rows, cols), work_bytes); },
                     [&] { return launch_norm_grad(dy_type, x_type, a, c->stream); });
}

int dn_dropout_device(dn_ctx *c, int x_type, int y_type, int64_t rows, int64_t cols, const void *d_x, int64_t ldx,
                      const void *d_res, int64_t ldres, float p, uint64_t seed, uint64_t offset, void *d_y,
                      int64_t ldy) {
  DropArgs a{};
  a.rows = rows;
  a.cols = cols;
  a.x = d_x;
  a.ldx = ldx;
  a.res = d_res;
  a.ldres = ldres;
  a.y = d_y;
  a.ldy = ldy;
  return device_call(c, "dropout", [&] { return blockchk::dropout(x_type, y_type, p, seed, offset, &a); },
                     [&] { return launch_dropout(x_type, y_type, a, c->stream); });
}

int dn_dropout_add_norm_device(dn_ctx *c, int x_type, int stream_type, int y_type, int64_t rows, int cols,
                               const void *d_x, int64_t ldx, const void *d_res, int64_t ldres, float p,
                               uint64_t seed, uint64_t offset, const float *d_w, const float *d_b, float eps,
                               void *d_h, int64_t ldh, void *d_y, int64_t ldy, float *d_mean, float *d_rstd) {
  NormArgs a{};
  a.rows = rows;
  a.cols = cols;
  a.x = d_x;
  a.ldx = ldx;
  a.res = d_res;
  a.ldres = ldres;
  a.w = d_w;
  a.b = d_b;
  a.eps = eps;
  a.h = d_h;
  a.ldh = ldh;
  a.y = d_y;
  a.ldy = ldy;
  a.mean = d_mean;
  a.rstd = d_rstd;
  return device_call(c, "dropout_add_norm",
                     [&] { return blockchk::boundary(x_type, stream_type, y_type, p, seed, offset, &a); },
                     [&] { return launch_boundary(x_type, stream_type, y_type, a, c->stream); });
}

int dn_dropout_add_norm_backward_device(dn_ctx *c, int dy_type, int stream_type, int dx_type, int64_t rows, int cols,
                                        const void *d_dy, int64_t lddy, const void *d_dh, int64_t lddh,
                                        const void *d_h, int64_t ldh, float p, uint64_t seed, uint64_t offset,
                                        const float *d_w, const float *d_mean, const float *d_rstd, void *d_dres,
                                        int64_t lddres, void *d_dx, int64_t lddx, float *d_dw, float *d_db,
                                        int accumulate, void *d_work, int64_t work_bytes) {
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
  a.mean = d_mean;
  a.rstd = d_rstd;
  a.dres = d_dres;
  a.lddres = lddres;
  a.dx = d_dx;
  a.lddx = lddx;
  a.dw = d_dw;
  a.db = d_db;
  a.accumulate = accumulate ? 1 : 0;
  a.work = (float *)d_work;
  return device_call(c, "dropout_add_norm_backward",
                     [&] {
                       return blockchk::boundary_grad(dy_type, stream_type, dx_type, p, seed, offset, &a,
                                                      work_floats(rows, cols), work_bytes);
                     },
                     [&] { return launch_boundary_grad(dy_type, stream_type, dx_type, a, c->stream); });
}

}  // extern "C"
