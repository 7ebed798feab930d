// Argument checks of the training-block operators (block_ops.cpp), host code
// without HIP. Each returns {0, ""} or the status and message of a refusal.
#pragma once

#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/decide_hip.h"
#include "block_args.hpp"

namespace blockchk {

struct Refusal {
  int code = DN_OK;
  std::string msg;
};

// Rows an operator takes: the mask's counter holds a row in 32 bits, and a
// launch's loops count rows in 64.
constexpr int64_t kMaxRows = 0x7fffffff;
// Columns of the elementwise dropout: the mask's counter holds a block of
// eight columns in 32 bits.
constexpr int64_t kMaxDropCols = ((int64_t)1 << 34) - 8;

inline bool known(int t) { return t == DN_PRECISION_FP32 || t == DN_PRECISION_BF16 || t == DN_PRECISION_FP16; }
inline int width(int t) { return t == DN_PRECISION_FP32 ? 4 : 2; }

// The type combinations that are built. 16-bit arrays of a call are all of one
// type. A norm: its input fp32 or the type of the other side (y, or dy).
inline bool norm_types_ok(int x, int y) { return x == DN_PRECISION_FP32 || x == y; }
// A boundary (a = x or dy, b = y or dx): a 16-bit stream has 16-bit neighbours
// on both sides; an fp32 stream fp32 or 16-bit ones, also a = fp32 beside a
// 16-bit b.
inline bool boundary_types_ok(int a, int stream, int b) {
  if (stream != DN_PRECISION_FP32) return a == stream && b == stream;
  return a == b || (a == DN_PRECISION_FP32 && b != DN_PRECISION_FP32);
}
inline bool dropout_types_ok(int x, int y) { return x == y || x == DN_PRECISION_FP32 || y == DN_PRECISION_FP32; }

// One array of a call. Vectors over the columns or rows are arrays of one row.
struct Array {
  const char *name;
  const void *p;
  int64_t rows, cols, ld;
  int es;         // element size
  bool out;       // written
  bool required;  // may not be NULL
  bool matrix;    // rows x cols of the call (an output may be an input's very array)
};

// Whether two arrays share no element. Their byte ranges are apart, or they
// are columns of one buffer (equal row strides, the columns side by side).
inline bool apart(const Array &a, const Array &b) {
  auto lo = [](const Array &x) { return (uintptr_t)x.p; };
  auto span = [](const Array &x) { return (uint64_t)(((x.rows - 1) * x.ld + x.cols) * x.es); };
  if (lo(a) + span(a) <= lo(b) || lo(b) + span(b) <= lo(a)) return true;
  if (a.rows < 2 || b.rows < 2) return false;  // a single row's stride is any number
  const int64_t sa = a.ld * a.es, sb = b.ld * b.es;
  if (sa != sb) return false;
  // b's first byte within a's row, modulo the stride.
  const int64_t d = lo(b) >= lo(a) ? (int64_t)((lo(b) - lo(a)) % (uint64_t)sa)
                                   : (sa - (int64_t)((lo(a) - lo(b)) % (uint64_t)sa)) % sa;
  return d >= a.cols * a.es && d + b.cols * b.es <= sa;
}

inline std::string said(const char *op) { return std::string("decide_hip: ") + op + ": "; }

inline Refusal arrays(const char *op, const Array *v, int n) {
  for (int i = 0; i < n; i++) {
    const Array &a = v[i];
    if (a.rows == 0 || a.cols == 0) continue;
    if (!a.p) {
      if (a.required) return {DN_INVALID_ARG, said(op) + a.name + " is NULL"};
      continue;
    }
    if ((uintptr_t)a.p % a.es) return {DN_INVALID_ARG, said(op) + a.name + " is not aligned to its elements"};
    if (a.rows > 1 && a.ld < a.cols)
      return {DN_INVALID_ARG, said(op) + "the row stride of " + a.name + " is less than its columns"};
    if (a.rows > 1 && a.ld > ((int64_t)1 << 56) / a.rows)
      return {DN_INVALID_ARG, said(op) + "the row stride of " + a.name + " passes the address range"};
  }
  for (int i = 0; i < n; i++)
    for (int j = i + 1; j < n; j++) {
      const Array &a = v[i], &b = v[j];
      if (!a.p || !b.p || !(a.out || b.out) || a.rows == 0 || a.cols == 0 || b.rows == 0 || b.cols == 0) continue;
      const bool same = a.p == b.p && a.es == b.es && (a.ld == b.ld || a.rows == 1) && a.matrix && b.matrix;
      if (same && a.out != b.out) continue;  // in place
      if (!apart(a, b)) return {DN_INVALID_ARG, said(op) + a.name + " overlaps " + b.name};
    }
  return {};
}

inline Refusal sizes(const char *op, int64_t rows, int64_t cols, int64_t min_cols, int64_t max_cols) {
  if (rows < 0 || cols < min_cols) return {DN_INVALID_ARG, said(op) + "bad number of rows or columns"};
  if (rows > kMaxRows || cols > max_cols)
    return {DN_UNSUPPORTED, said(op) + "at most 2147483647 rows and " + std::to_string(max_cols) + " columns"};
  return {};
}

inline Refusal types(const char *op, bool all_known, bool built) {
  if (!all_known) return {DN_INVALID_ARG, said(op) + "unknown precision"};
  if (!built) return {DN_UNSUPPORTED, said(op) + "this combination of types is not built"};
  return {};
}

// The mask of a dropout probability: threshold = p in units of 2^-16, to nearest.
inline Refusal mask(const char *op, float p, uint64_t seed, uint64_t offset, DropMask *m) {
  if (!(p >= 0.0f && p <= 1.0f))
    return {DN_INVALID_ARG, said(op) + "the dropout probability is not in [0, 1]"};
  m->threshold = (uint32_t)std::nearbyint((double)p * 65536.0);
  m->scale = m->threshold < 65536 ? (float)(65536.0 / (65536 - m->threshold)) : 0.0f;
  m->k0 = (uint32_t)seed;
  m->k1 = (uint32_t)(seed >> 32);
  m->o0 = (uint32_t)offset;
  m->o1 = (uint32_t)(offset >> 32);
  return {};
}

inline Refusal epsilon(const char *op, float eps) {
  if (!(eps > 0.0f) || !std::isfinite(eps))
    return {DN_INVALID_ARG, said(op) + "eps is not a positive number"};
  return {};
}

#define BLOCKCHK(expr)                      \
  do {                                      \
    const blockchk::Refusal r_ = (expr);    \
    if (r_.code) return r_;                 \
  } while (0)

inline Refusal norm(int x_type, int y_type, const NormArgs &a) {
  const char *op = "dn_layer_norm_device";
  BLOCKCHK(types(op, known(x_type) && known(y_type), norm_types_ok(x_type, y_type)));
  BLOCKCHK(sizes(op, a.rows, a.cols, 1, kNormMaxCols));
  BLOCKCHK(epsilon(op, a.eps));
  const int64_t R = a.rows, C = a.cols;
  const Array v[] = {{"x", a.x, R, C, a.ldx, width(x_type), false, true, true},
                     {"y", a.y, R, C, a.ldy, width(y_type), true, true, true},
                     {"w", a.w, 1, C, C, 4, false, false, false},
                     {"b", a.b, 1, C, C, 4, false, false, false},
                     {"mean", a.mean, 1, R, R, 4, true, false, false},
                     {"rstd", a.rstd, 1, R, R, 4, true, false, false}};
  return arrays(op, v, 6);
}

inline Refusal norm_grad(int dy_type, int x_type, const NormGradArgs &a, int64_t work_floats, int64_t work_bytes) {
  const char *op = "dn_layer_norm_backward_device";
  BLOCKCHK(types(op, known(dy_type) && known(x_type), norm_types_ok(x_type, dy_type)));
  BLOCKCHK(sizes(op, a.rows, a.cols, 1, kNormMaxCols));
  const int64_t R = a.rows, C = a.cols, W = a.dw || a.db ? work_floats : 0;
  if (work_bytes < 4 * W) return {DN_INVALID_ARG, said(op) + "the workspace is too small"};
  const Array v[] = {{"dy", a.dy, R, C, a.lddy, width(dy_type), false, true, true},
                     {"x", a.h, R, C, a.ldh, width(x_type), false, true, true},
                     {"w", a.w, 1, C, C, 4, false, false, false},
                     {"mean", a.mean, 1, R, R, 4, false, true, false},
                     {"rstd", a.rstd, 1, R, R, 4, false, true, false},
                     {"dx", a.dres, R, C, a.lddres, width(x_type), true, true, true},
                     {"dw", a.dw, 1, C, C, 4, true, false, false},
                     {"db", a.db, 1, C, C, 4, true, false, false},
                     {"work", a.work, 1, W, W, 4, true, true, false}};
  return arrays(op, v, 9);
}

inline Refusal dropout(int x_type, int y_type, float p, uint64_t seed, uint64_t offset, DropArgs *a) {
  const char *op = "dn_dropout_device";
  BLOCKCHK(types(op, known(x_type) && known(y_type), dropout_types_ok(x_type, y_type)));
  BLOCKCHK(sizes(op, a->rows, a->cols, 0, kMaxDropCols));
  BLOCKCHK(mask(op, p, seed, offset, &a->mask));
  const int64_t R = a->rows, C = a->cols;
  const Array v[] = {{"x", a->x, R, C, a->ldx, width(x_type), false, true, true},
                     {"res", a->res, R, C, a->ldres, width(y_type), false, false, true},
                     {"y", a->y, R, C, a->ldy, width(y_type), true, true, true}};
  return arrays(op, v, 3);
}

inline Refusal boundary(int x_type, int stream_type, int y_type, float p, uint64_t seed, uint64_t offset,
                        NormArgs *a) {
  const char *op = "dn_dropout_add_norm_device";
  BLOCKCHK(types(op, known(x_type) && known(stream_type) && known(y_type),
                 boundary_types_ok(x_type, stream_type, y_type)));
  BLOCKCHK(sizes(op, a->rows, a->cols, 1, kNormMaxCols));
  BLOCKCHK(mask(op, p, seed, offset, &a->mask));
  BLOCKCHK(epsilon(op, a->eps));
  const int64_t R = a->rows, C = a->cols;
  const Array v[] = {{"x", a->x, R, C, a->ldx, width(x_type), false, true, true},
                     {"res", a->res, R, C, a->ldres, width(stream_type), false, true, true},
                     {"h", a->h, R, C, a->ldh, width(stream_type), true, true, true},
                     {"y", a->y, R, C, a->ldy, width(y_type), true, true, true},
                     {"w", a->w, 1, C, C, 4, false, false, false},
                     {"b", a->b, 1, C, C, 4, false, false, false},
                     {"mean", a->mean, 1, R, R, 4, true, false, false},
                     {"rstd", a->rstd, 1, R, R, 4, true, false, false}};
  return arrays(op, v, 8);
}

inline Refusal boundary_grad(int dy_type, int stream_type, int dx_type, float p, uint64_t seed, uint64_t offset,
                             NormGradArgs *a, int64_t work_floats, int64_t work_bytes) {
  const char *op = "dn_dropout_add_norm_backward_device";
  BLOCKCHK(types(op, known(dy_type) && known(stream_type) && known(dx_type),
                 boundary_types_ok(dy_type, stream_type, dx_type)));
  BLOCKCHK(sizes(op, a->rows, a->cols, 1, kNormMaxCols));
  BLOCKCHK(mask(op, p, seed, offset, &a->mask));
  const int64_t R = a->rows, C = a->cols, W = a->dw || a->db ? work_floats : 0;
  if (work_bytes < 4 * W) return {DN_INVALID_ARG, said(op) + "the workspace is too small"};
  const Array v[] = {{"dy", a->dy, R, C, a->lddy, width(dy_type), false, true, true},
                     {"dh", a->dh, R, C, a->lddh, width(stream_type), false, false, true},
                     {"h", a->h, R, C, a->ldh, width(stream_type), false, true, true},
                     {"w", a->w, 1, C, C, 4, false, false, false},
                     {"mean", a->mean, 1, R, R, 4, false, true, false},
                     {"rstd", a->rstd, 1, R, R, 4, false, true, false},
                     {"dres", a->dres, R, C, a->lddres, width(stream_type), true, true, true},
                     {"dx", a->dx, R, C, a->lddx, width(dx_type), true, true, true},
                     {"dw", a->dw, 1, C, C, 4, true, false, false},
                     {"db", a->db, 1, C, C, 4, true, false, false},
                     {"work", a->work, 1, W, W, 4, true, true, false}};
  return arrays(op, v, 11);
}

}  // namespace blockchk
