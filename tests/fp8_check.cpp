// The argument checks of the 8-bit operators as functions that ctypes can call
// without a GPU: each returns the refusal's status and copies its message out.
#include <cstring>

#include "../decide_amd/csrc/fp8_check.hpp"

namespace {
int give(const blockchk::Refusal &r, char *msg, int cap) {
  std::strncpy(msg, r.msg.c_str(), cap - 1);
  msg[cap - 1] = 0;
  return r.code;
}
}  // namespace

extern "C" {

struct Fp8Call {
  int x_type, stream_type, y_type, q_type, b_type, block_rows, accumulate;
  float eps;
  int64_t rows, cols, depth;
  uintptr_t x, res, h, y, q, qt, scale, scalet, w, rstd, dy, dh, dres, dx, dw, work, A, B, sa, sb, C;
  int64_t ldx, ldres, ldh, ldy, ldq, ldqt, ldscale, ldscalet, lddy, lddh, lddres, lddx, ldA, ldB, ldsa, ldsb, ldC;
  int64_t work_floats, work_bytes;
};

int check_rms(const Fp8Call *c, char *msg, int cap) {
  RmsArgs a{};
  a.rows = c->rows, a.cols = (int)c->cols, a.eps = c->eps;
  a.x = (const void *)c->x, a.ldx = c->ldx, a.res = (const void *)c->res, a.ldres = c->ldres;
  a.w = (const float *)c->w, a.h = (void *)c->h, a.ldh = c->ldh, a.y = (void *)c->y, a.ldy = c->ldy;
  a.q = (void *)c->q, a.ldq = c->ldq, a.scale = (float *)c->scale, a.ldscale = c->ldscale, a.rstd = (float *)c->rstd;
  return give(blockchk::rms(c->x_type, c->stream_type, c->y_type, c->q_type, a), msg, cap);
}

int check_rms_grad(const Fp8Call *c, char *msg, int cap) {
  NormGradArgs a{};
  a.rows = c->rows, a.cols = (int)c->cols;
  a.dy = (const void *)c->dy, a.lddy = c->lddy, a.dh = (const void *)c->dh, a.lddh = c->lddh;
  a.h = (const void *)c->h, a.ldh = c->ldh, a.dres = (void *)c->dres, a.lddres = c->lddres;
  a.dx = (void *)c->dx, a.lddx = c->lddx, a.w = (const float *)c->w, a.rstd = (const float *)c->rstd;
  a.dw = (float *)c->dw, a.work = (float *)c->work;
  return give(blockchk::rms_grad(c->x_type, c->stream_type, c->y_type, a, c->work_floats, c->work_bytes), msg, cap);
}

int check_quantise(const Fp8Call *c, char *msg, int cap) {
  QuantArgs a{};
  a.rows = c->rows, a.cols = c->cols;
  a.x = (const void *)c->x, a.ldx = c->ldx, a.q = (void *)c->q, a.ldq = c->ldq;
  a.scale = (float *)c->scale, a.ldscale = c->ldscale;
  a.qt = (void *)c->qt, a.ldqt = c->ldqt, a.scalet = (float *)c->scalet, a.ldscalet = c->ldscalet;
  return give(blockchk::quantise(c->x_type, c->q_type, c->block_rows, a), msg, cap);
}

int check_gemm(const Fp8Call *c, char *msg, int cap) {
  Fp8GemmArgs a{};
  a.M = c->rows, a.N = c->cols, a.K = c->depth;
  a.A = (const void *)c->A, a.lda = c->ldA, a.sa = (const float *)c->sa, a.ldsa = c->ldsa;
  a.B = (const void *)c->B, a.ldb = c->ldB, a.sb = (const float *)c->sb, a.ldsb = c->ldsb;
  a.C = (void *)c->C, a.ldc = c->ldC, a.accumulate = c->accumulate, a.work = (float *)c->work;
  return give(blockchk::gemm(c->q_type, c->b_type, c->y_type, c->block_rows, a, 4 * c->work_floats, c->work_bytes),
              msg, cap);
}

}  // extern "C"
