// The argument checks of the training-block operators as functions that ctypes
// can call without a GPU: each returns the refusal's status and copies its
// message out.
#include <cstring>

#include "../decide_amd/csrc/block_check.hpp"

namespace {
int give(const blockchk::Refusal &r, char *msg, int cap) {
  std::strncpy(msg, r.msg.c_str(), cap - 1);
  msg[cap - 1] = 0;
  return r.code;
}
}  // namespace

extern "C" {

struct NormCall {
  int a_type, stream_type, b_type, cols;
  int64_t rows;
  float p, eps;
  // norm: x, y; dropout and boundary: x, res, h, y; gradients: dy, dh, h, dres, dx
  uintptr_t x, res, h, y, dy, dh, dres, dx, w, b, mean, rstd, dw, db, work;
  int64_t ldx, ldres, ldh, ldy, lddy, lddh, lddres, lddx, drop_cols, work_floats, work_bytes;
};

static NormArgs forward(const NormCall &c) {
  NormArgs a{};
  a.rows = c.rows, a.cols = c.cols, a.eps = c.eps;
  a.x = (const void *)c.x, a.ldx = c.ldx, a.res = (const void *)c.res, a.ldres = c.ldres;
  a.w = (const float *)c.w, a.b = (const float *)c.b;
  a.h = (void *)c.h, a.ldh = c.ldh, a.y = (void *)c.y, a.ldy = c.ldy;
  a.mean = (float *)c.mean, a.rstd = (float *)c.rstd;
  return a;
}

static NormGradArgs gradient(const NormCall &c) {
  NormGradArgs a{};
  a.rows = c.rows, a.cols = c.cols;
  a.dy = (const void *)c.dy, a.lddy = c.lddy, a.dh = (const void *)c.dh, a.lddh = c.lddh;
  a.h = (const void *)c.h, a.ldh = c.ldh, a.dres = (void *)c.dres, a.lddres = c.lddres;
  a.dx = (void *)c.dx, a.lddx = c.lddx;
  a.w = (const float *)c.w, a.mean = (const float *)c.mean, a.rstd = (const float *)c.rstd;
  a.dw = (float *)c.dw, a.db = (float *)c.db, a.work = (float *)c.work;
  return a;
}

int check_norm(const NormCall *c, char *msg, int cap) {
  return give(blockchk::norm(c->stream_type, c->b_type, forward(*c)), msg, cap);
}

int check_boundary(const NormCall *c, char *msg, int cap) {
  NormArgs a = forward(*c);
  return give(blockchk::boundary(c->a_type, c->stream_type, c->b_type, c->p, 1, 2, &a), msg, cap);
}

int check_norm_grad(const NormCall *c, char *msg, int cap) {
  return give(blockchk::norm_grad(c->a_type, c->stream_type, gradient(*c), c->work_floats, c->work_bytes), msg, cap);
}

int check_boundary_grad(const NormCall *c, char *msg, int cap) {
  NormGradArgs a = gradient(*c);
  return give(blockchk::boundary_grad(c->a_type, c->stream_type, c->b_type, c->p, 1, 2, &a, c->work_floats,
                                      c->work_bytes),
              msg, cap);
}

int check_dropout(const NormCall *c, char *msg, int cap) {
  DropArgs a{};
  a.rows = c->rows, a.cols = c->drop_cols;
  a.x = (const void *)c->x, a.ldx = c->ldx, a.res = (const void *)c->res, a.ldres = c->ldres;
  a.y = (void *)c->y, a.ldy = c->ldy;
  return give(blockchk::dropout(c->a_type, c->b_type, c->p, 1, 2, &a), msg, cap);
}

int mask_of(float p, uint64_t seed, uint64_t offset, uint32_t *out5, float *scale) {
  DropMask m{};
  const blockchk::Refusal r = blockchk::mask("mask", p, seed, offset, &m);
  out5[0] = m.threshold, out5[1] = m.k0, out5[2] = m.k1, out5[3] = m.o0, out5[4] = m.o1;
  *scale = m.scale;
  return r.code;
}

}  // extern "C"
