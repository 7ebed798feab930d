// Arguments of the training-block operators, without the HIP headers: the
// argument checks (block_check.hpp) are host code of their own.
#pragma once

#include <stdint.h>

// Widest row of the norms: 1,024 threads hold it in registers, 16 elements each.
constexpr int kNormMaxCols = 16384;

// A dropout mask: the element in column c of row r is kept where its 16
// random bits are at least `threshold`, and scaled by `scale` = 65536 / (65536
// - threshold). threshold 0 keeps every element unscaled, 65536 none.
struct DropMask {
  uint32_t threshold;
  float scale;
  uint32_t k0, k1;  // the seed: the generator's key
  uint32_t o0, o1;  // the offset: the upper half of its counter
};

// Row r of an array starts at base + r * ld elements.
struct NormArgs {
  int64_t rows;
  int cols;
  const void *x;  // the norm's input, or the sub-layer's output that is dropped and added to res
  int64_t ldx;
  const void *res;  // null: the plain norm of x
  int64_t ldres;
  DropMask mask;
  const float *w, *b;  // [cols]; null: 1 and 0
  float eps;
  void *h;  // res + dropout(x) (with res)
  int64_t ldh;
  void *y;
  int64_t ldy;
  float *mean, *rstd;  // [rows]; either may be null
};

struct NormGradArgs {
  int64_t rows;
  int cols;
  const void *dy;
  int64_t lddy;
  const void *dh;  // the gradient that reaches h beside the norm; null: 0
  int64_t lddh;
  const void *h;  // the norm's input
  int64_t ldh;
  const float *w, *mean, *rstd;
  void *dres;  // the gradient of the norm's input, dh included
  int64_t lddres;
  DropMask mask;
  void *dx;  // dropout's gradient of dres; null: the plain norm
  int64_t lddx;
  float *dw, *db;  // [cols]; either may be null
  int accumulate;  // dw, db += instead of =
  float *work;     // norm_grad_work(rows, cols) floats
};

struct DropArgs {
  int64_t rows, cols;
  const void *x;
  int64_t ldx;
  const void *res;  // null: 0
  int64_t ldres;
  DropMask mask;
  void *y;
  int64_t ldy;
};
