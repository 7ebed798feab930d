// Arguments of the 8-bit operators, without the HIP headers: the argument
// checks (fp8_check.hpp) are host code of their own.
#pragma once

#include <stdint.h>

// Columns (and rows, of a square block) that share a scale.
constexpr int kFp8Block = 128;
inline int64_t fp8_blocks(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }

// Row r of an array starts at base + r * ld elements. Scales are held block by
// block: row (or block of rows) r, block of columns b at scale[b * ldscale + r].
struct RmsArgs {
  int64_t rows;
  int cols;
  const void *x;
  int64_t ldx;
  const void *res;  // null: the norm of x
  int64_t ldres;
  const float *w;  // [cols]; null: 1
  float eps;
  void *h;  // res + x (with res)
  int64_t ldh;
  void *y;  // null: q only
  int64_t ldy;
  void *q;  // null: y only
  int64_t ldq;
  float *scale;
  int64_t ldscale;
  float *rstd;  // [rows]; may be null
  int e5m2;     // q's type
};

struct QuantArgs {
  int64_t rows, cols;
  const void *x;
  int64_t ldx;
  void *q;  // null: the transpose only
  int64_t ldq;
  float *scale;
  int64_t ldscale;
  void *qt;  // [cols x rows]; null: x itself only
  int64_t ldqt;
  float *scalet;
  int64_t ldscalet;
  int square;  // blocks of 128 x 128 instead of 1 x 128
  int e5m2;
};

struct Fp8GemmArgs {
  int64_t M, N, K;
  const void *A;  // M x K
  int64_t lda;
  const float *sa;  // of 1 x 128 blocks
  int64_t ldsa;
  const void *B;  // N x K
  int64_t ldb;
  const float *sb;  // of 1 x 128 blocks or (b_square) 128 x 128 ones
  int64_t ldsb;
  void *C;  // M x N
  int64_t ldc;
  int b_square;
  int accumulate;  // C += instead of =
  float *work;
};
