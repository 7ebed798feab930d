// The training-block operators (block_ops.hip, block_grad.hip; C entry points
// in block_ops.cpp): LayerNorm, dropout by a counter-based generator, and the
// residual boundary h = res + dropout(x), y = LayerNorm(h), with their
// gradients.
#pragma once

#include "block_args.hpp"
#include "common.hpp"

// Launchers. Types are PREC_* codes that block_check.hpp's rules allow; the
// arguments have passed its checks.
hipError_t launch_norm(int x_type, int y_type, const NormArgs &a, hipStream_t s);
hipError_t launch_boundary(int x_type, int stream_type, int y_type, const NormArgs &a, hipStream_t s);
hipError_t launch_norm_grad(int dy_type, int x_type, const NormGradArgs &a, hipStream_t s);
hipError_t launch_boundary_grad(int dy_type, int stream_type, int dx_type, const NormGradArgs &a, hipStream_t s);
int64_t norm_grad_work(int64_t rows, int cols);
hipError_t launch_dropout(int x_type, int y_type, const DropArgs &a, hipStream_t s);

#ifdef __HIPCC__

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC'11): ten rounds of two 32 x 32 -> 64-bit products, the
// published multipliers and key increments.
__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 10; i++) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Drops the elements of columns 8 * block .. 8 * block + 7 of a row in place:
// one generator block gives their eight 16-bit draws. A dropped element is 0
// whatever it was (also an infinity or a NaN), so it is selected, not multiplied.
__device__ __forceinline__ void drop8(const DropMask &m, uint32_t row, uint32_t block, float (&v)[8]) {
  if (m.threshold == 0) return;
  const uint4 r = philox(block, row, m.o0, m.o1, m.k0, m.k1);
  const uint32_t word[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int j = 0; j < 4; j++) {
    v[2 * j] = (word[j] & 0xffffu) >= m.threshold ? v[2 * j] * m.scale : 0.0f;
    v[2 * j + 1] = (word[j] >> 16) >= m.threshold ? v[2 * j + 1] * m.scale : 0.0f;
  }
}

// Eight consecutive elements from an address aligned to the element only: the
// hardware takes 16-byte accesses at any element's alignment, so odd row
// strides need no variant of their own. n < 8 (a row's last, partial block):
// element by element, zeros past n.
template <class T>
__device__ __forceinline__ void load8(const T *p, int n, float (&v)[8]) {
  if (n >= 8) {
    T t[8];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = (float)t[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = j < n ? (float)p[j] : 0.0f;
  }
}
template <class T>
__device__ __forceinline__ void store8(T *p, int n, const float (&v)[8]) {
  if (n >= 8) {
    T t[8];
#pragma unroll
    for (int j = 0; j < 8; j++) t[j] = to_elem<T>(v[j]);
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (j < n) p[j] = to_elem<T>(v[j]);
  }
}

#endif
