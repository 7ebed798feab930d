// The training-block operators (block_ops.hip, block_grad.hip; C entry points
// in block_ops.cpp): LayerNorm, dropout by a counter-based generator, and the
// residual boundary h = res + dropout(x), y = LayerNorm(h), with their
// gradients.
#pragma once

#include <type_traits>

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
  auto xor3 = [](uint32_t x, uint32_t y, uint32_t z) { return __builtin_amdgcn_bitop3_b32(x, y, z, 0x96); };
#pragma unroll
  for (int i = 0; i < 10; i++) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = xor3((uint32_t)(b >> 32), c1, k0);
    c1 = (uint32_t)b;
    c2 = xor3((uint32_t)(a >> 32), c3, k1);
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Drops elements in place (the scale of the others is the caller's, one
// multiply-add with what they are added to), from the generator's words that
// hold their 16-bit draws: element j takes half j % 2 (0 low) of word j / 2. A
// dropped element is 0 whatever it was (also an infinity or a NaN), so it is
// selected, not multiplied. A half is at least the threshold t > 0 where its
// word, with that half in the upper bits, is above 65536 t - 1: the lower bits
// only add, and at t = 65536 nothing is above 2^32 - 1.
__device__ __forceinline__ float keep(const DropMask &m, uint32_t upper, float v) {
  return upper > (m.threshold << 16) - 1u ? v : 0.0f;
}
template <int N>
__device__ __forceinline__ void drop_by(const DropMask &m, const uint32_t (&word)[N / 2], float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N / 2; j++) {
    v[2 * j] = keep(m, word[j] << 16, v[2 * j]);
    v[2 * j + 1] = keep(m, word[j], v[2 * j + 1]);
  }
}

// Two vectors of four columns, halves of two generator blocks that the lane and
// its neighbour share: of the first vectors' block r is in the even lane, of
// the second ones' in the odd lane, and each hands the other its half (the even
// lane holds the lower four columns of both). Both lanes take part.
__device__ __forceinline__ void drop_pair(const DropMask &m, bool odd, const uint4 &r, float (&first)[4],
                                          float (&second)[4]) {
  const uint32_t low[2] = {r.x, r.y}, high[2] = {r.z, r.w};
  uint32_t a[2], b[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const uint32_t mine = odd ? high[i] : low[i];
    const uint32_t other = dpp_u32<0xB1>(odd ? low[i] : high[i]);  // the neighbour's: quad_perm 1,0,3,2
    a[i] = odd ? other : mine;
    b[i] = odd ? mine : other;
  }
  drop_by<4>(m, a, first);
  drop_by<4>(m, b, second);
}

// The columns of a row that one of its `lpr` threads holds: VPT vectors of VEC,
// vector j at column VEC * (lane + j * lpr). WAVES: the row has several waves.
template <bool WAVES, int VPT, int VEC>
struct Columns {
  // The elements of a row of `cols` dropped in place. One generator block covers
  // eight columns: a vector of eight, or the vectors of four of two neighbouring
  // lanes (drop_pair), or a row of less than eight columns with one lane each.
  // Waves that lie past the row skip a vector, both lanes of a pair or neither.
  static __device__ __forceinline__ void drop(const DropMask &m, uint32_t row, int lane, int lpr, int cols,
                                              float (&v)[VPT][VEC]) {
    if (m.threshold == 0) return;
    if constexpr (VEC == 8) {
#pragma unroll
      for (int j = 0; j < VPT; j++) {
        const int block = lane + j * lpr;
        if (WAVES && j > 0 && 8 * block >= cols) break;
        const uint4 r = philox((uint32_t)block, row, m.o0, m.o1, m.k0, m.k1);
        const uint32_t word[4] = {r.x, r.y, r.z, r.w};
        drop_by<8>(m, word, v[j]);
      }
    } else if constexpr (VEC == 1) {
      const uint4 r = philox(0, row, m.o0, m.o1, m.k0, m.k1);
      const uint32_t word = lane < 4 ? (lane < 2 ? r.x : r.y) : (lane < 6 ? r.z : r.w);
      v[0][0] = keep(m, lane & 1 ? word : word << 16, v[0][0]);
    } else {
      const bool odd = lane & 1;
#pragma unroll
      for (int j = 0; j < VPT; j += 2) {
        const bool pair = j + 1 < VPT;
        if (WAVES && j > 0 && 4 * ((lane & ~1) + j * lpr) >= cols) break;
        const uint4 r = philox((uint32_t)(lane + (j + (pair && odd ? 1 : 0)) * lpr) >> 1, row, m.o0, m.o1, m.k0, m.k1);
        if (pair) {
          drop_pair(m, odd, r, v[j], v[j + 1 < VPT ? j + 1 : j]);
        } else {
          const uint32_t word[2] = {odd ? r.z : r.x, odd ? r.w : r.y};
          drop_by<4>(m, word, v[j]);
        }
      }
    }
  }
};

// VEC consecutive elements of a row as they lie in memory. The address needs
// the elements' alignment only: the hardware takes accesses of up to 16 bytes
// at any address, so odd strides and offsets need no variant of their own.
template <class T, int VEC>
struct Raw {
  uint32_t q[VEC * sizeof(T) / 4];
  __device__ __forceinline__ float at(int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(q[j]);
    else return j & 1 ? hi16<T>(q[j / 2]) : lo16<T>(q[j / 2]);
  }
};
template <class T>
struct Raw<T, 1> {
  T q;
  __device__ __forceinline__ float at(int) const { return (float)q; }
};

// Columns c .. c + VEC - 1 of a row of cols >= VEC. Where those pass the row's
// end (its last, partial vector, and threads past it) the VEC elements that end
// with the row are read instead, so that every lane makes the same loads and no
// branch stands between them; unpack moves them into place.
template <class T, int VEC>
__device__ __forceinline__ Raw<T, VEC> fetch(const T *row, int c, int cols) {
  Raw<T, VEC> r;
  __builtin_memcpy(&r, row + (unsigned)min(c, cols - VEC), sizeof(r));
  return r;
}

// The vector's elements as floats, `past` past the row. n: columns from c on.
template <class T, int VEC>
__device__ __forceinline__ void unpack(const Raw<T, VEC> &r, int n, float (&v)[VEC], float past = 0.0f) {
#pragma unroll
  for (int j = 0; j < VEC; j++) v[j] = r.at(j);
  if (n < VEC) {
    const int by = VEC - max(n, 0);  // elements down, 1 .. VEC
#pragma unroll
    for (int step = VEC; step > 0; step >>= 1)
#pragma unroll
      for (int j = 0; j < VEC; j++) v[j] = by & step ? (j + step < VEC ? v[j + step] : past) : v[j];
  }
}

template <class T, int VEC>
__device__ __forceinline__ void load(const T *row, int c, int cols, float (&v)[VEC]) {
  unpack<T, VEC>(fetch<T, VEC>(row, c, cols), cols - c, v);
}

template <class T, int VEC>
__device__ __forceinline__ void store(T *row, int c, int cols, const float (&v)[VEC]) {
  if (cols - c >= VEC) {
    T t[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) t[j] = to_elem<T>(v[j]);
    __builtin_memcpy(row + (unsigned)c, t, sizeof(t));
  } else if (c < cols) {
    asm volatile("");  // keeps the compiler from splitting the store above to share its parts with these
#pragma unroll
    for (int j = 0; j < VEC - 1; j++)
      if (c + j < cols) row[(unsigned)(c + j)] = to_elem<T>(v[j]);
  }
}

// The sum of each v[i] over the threads that share a row, in all of them: LPR
// consecutive threads, or (0) the workgroup. DPP moves within 16 lanes and row
// swaps across them (no LDS round trips: steps of ~8 cycles where a shuffle
// takes ~60), and for a workgroup one exchange of its waves' sums (at most 16)
// through LDS. The order of the sum depends on the number of threads alone.
// `slot`: N * 16 floats of LDS that no other reduction of the same row uses, so
// that one barrier per reduction is enough.
template <int LPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float *slot) {
  auto add = [&](auto move) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] += __uint_as_float(move(__float_as_uint(v[i])));
  };
  auto add16 = [&] {
    add([](unsigned x) { return dpp_u32<0xB1>(x); });   // quad_perm 1,0,3,2
    add([](unsigned x) { return dpp_u32<0x4E>(x); });   // quad_perm 2,3,0,1
    add([](unsigned x) { return dpp_u32<0x141>(x); });  // row_half_mirror
    if constexpr (LPR != 8) add([](unsigned x) { return dpp_u32<0x140>(x); });  // row_mirror
  };
  add16();
  if constexpr (LPR == 0 || LPR >= 32)
#pragma unroll
    for (int i = 0; i < N; i++) {
      const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
  if constexpr (LPR == 0 || LPR >= 64)
#pragma unroll
    for (int i = 0; i < N; i++) {
      const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
  if constexpr (LPR == 0) {
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; i++) slot[16 * i + (threadIdx.x >> 6)] = v[i];
    __syncthreads();
    const int k = threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = k < (int)(blockDim.x >> 6) ? slot[16 * i + k] : 0.0f;
    add16();
  }
}

// a * b, rounded: never fused into an addition that uses it. A row's mean has
// to be one number for all of its columns.
__device__ __forceinline__ float mul_rounded(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// Threads of a workgroup whose rows have LPR threads each.
constexpr int kRowThreads = 256;

// The row a thread works on, of those that start at `first`: LPR threads per
// row, or (0) the workgroup. One register for the wave where all of its lanes
// share the row, so that the row's addresses are scalar.
template <int LPR>
__device__ __forceinline__ int64_t row_of(int64_t first) {
  if constexpr (LPR == 0) return first;
  const int group = threadIdx.x / (LPR ? LPR : 1);
  if constexpr (LPR == 64) return first + __builtin_amdgcn_readfirstlane(group);
  return first + group;
}

// How the threads share rows of a width: LPR threads of a workgroup of
// kRowThreads per row, or (LPR 0) a workgroup per row of as many waves as VPT
// vectors of VEC columns per thread need, MAXT threads at most.
template <int VEC_, int LPR_, int VPT_, int MAXT_ = kRowThreads>
struct RowShape {
  static constexpr int VEC = VEC_, LPR = LPR_, VPT = VPT_, MAXT = MAXT_;
  static constexpr int ROWS = LPR ? kRowThreads / (LPR ? LPR : 1) : 1;  // of a workgroup
  static int threads(int cols) {
    return LPR ? kRowThreads : ((cols + VEC * VPT - 1) / (VEC * VPT) + 63) / 64 * 64;
  }
  static bool takes(int cols) { return cols <= VEC * VPT * (LPR ? LPR : MAXT); }
};

// Calls f with the first shape of the list that takes the width.
template <class First, class... Rest, class F>
hipError_t pick_shape(int cols, F f) {
  if (First::takes(cols)) return f(First{});
  if constexpr (sizeof...(Rest) > 0) return pick_shape<Rest...>(cols, f);
  return hipErrorInvalidValue;
}

// Columns of a vector for a call with arrays of these types: 4 with an fp32
// array (16 bytes of it per lane, consecutive lanes side by side), else 8. Rows
// narrower than that take a lane per column.
template <class... T>
constexpr int vec_of = (... || (sizeof(T) == 4)) ? 4 : 8;

#endif
