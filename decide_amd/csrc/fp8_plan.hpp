// Which kernels a block-scaled 8-bit product runs, in which launches, by its
// sizes, types and alignment: host code without HIP (fp8_gemm.hip launches it).
#pragma once

#include <algorithm>

#include "fp8_args.hpp"

namespace fp8plan {

// Most tiles of a launch (fewer than 2^32 threads).
constexpr int64_t kGrid = 1 << 22;

inline int64_t tiles_of(int64_t n, int each) { return (n + each - 1) / each; }

// Small: 16 x 16, 32 x 32 and 64 x 32 outputs by eight waves that share K.
// Tile: 128 x 128 outputs; Wide: 128 x 256.
enum class Kind { Small11, Small22, Small42, Tile, Wide };
inline int rows_of(Kind k) { return k == Kind::Small11 ? 16 : k == Kind::Small22 ? 32 : k == Kind::Small42 ? 64 : 128; }
inline int cols_of(Kind k) { return k == Kind::Small11 ? 16 : k == Kind::Tile ? 128 : k == Kind::Wide ? 256 : 32; }

// The kernel of a product of these sizes. Median times in us of the kernel alone,
// bf16 C with 128 x 128 scales unless said:
//                          16 x 16  32 x 32  64 x 32  128 x 128  128 x 256
//   1 x 8,192 x 8,192        13.4     13.9     16.4      38.6
//   16 x 8,192 x 4,096       10.6      9.6     11.1      21.1
//   64 x 8,192 x 4,096       31.8     19.7     15.2      21.8
//   100 x 768 x 768           4.2      4.6      5.6       7.3
//   200 x 768 x 2,304         9.6      7.8      9.8      13.8
//   512 x 768 x 768           9.1      7.0      6.0       7.8
//   512 x 2,304 x 768        21.8     14.4     14.2       8.4
//   4,096 x 2,304 x 768                                  18.6       20.0
//   12,288 x 768 x 2,304                                 34.6       37.2
//   4,096 x 4,096 x 4,096                                74.0       72.4
//   32,768 x 2,304 x 768                                 96.3       90.0
// The small kernel as long as one round of the CUs holds its tiles (its waves
// share K, so that past 64 rows a long K goes to tiles whose parts workgroups
// share: 384 x 384 x 12,288 into fp32 39.4 and 17.6 a call).
inline Kind kind_of(int64_t M, int64_t N, int64_t K) {
  if (M > 64 && K > 64 * 128) return Kind::Tile;
  if (tiles_of(M, 16) * tiles_of(N, 16) <= 384) return Kind::Small11;
  if (tiles_of(M, 32) * tiles_of(N, 32) <= 256) return Kind::Small22;
  if (M <= 64 || tiles_of(M, 64) * tiles_of(N, 32) <= 256) return Kind::Small42;
  return Kind::Tile;
}

// Workgroups that share a 128 x 128 tile's blocks along K, by what they cost: a
// block 0.65 us (EXACT 1.2), half as much again for two workgroups on a CU, and
// the join 7 us (a launch) and the partial sums' bytes (2,304 x 768 x 12,288
// into fp32: one 125 us, two 74, three 78, four 67; 512 x 4,096 x 4,096 into bf16:
// one 22, two 23, four 25).
inline int split_of(int64_t M, int64_t N, int64_t K, bool exact) {
  if (kind_of(M, N, K) != Kind::Tile) return 1;
  const int64_t tiles = tiles_of(M, 128) * tiles_of(N, 128), blocks = tiles_of(K, 128);
  int best = 1;
  double least = 0.0;
  for (int split = 1; split <= 16 && split * tiles <= 512 && (split == 1 || split * 4 <= blocks); split++) {
    const double each = (exact ? 1.2 : 0.65) * (split * tiles > 256 ? 1.5 : 1.0);
    const double cost = tiles_of(blocks, split) * each + (split > 1 ? 7.0 + split * (double)M * N * 8 / 4.5e6 : 0.0);
    if (split == 1 || cost < least) best = split, least = cost;
  }
  return best;
}

// Floats of workspace of a product of these sizes.
inline int64_t work_of(int64_t M, int64_t N, int64_t K) {
  const int split = M && N ? std::max(split_of(M, N, K, false), split_of(M, N, K, true)) : 1;
  return split > 1 ? split * M * N : 0;
}

// Whether the tile kernels' direct loads take an operand: rows of whole 16-byte
// chunks, and offsets that fit a buffer load's 31 bits.
inline bool direct(uintptr_t p, int64_t ld, int64_t ld_scale, int64_t K) {
  const int64_t blocks = tiles_of(K, 128);
  return K <= 1 << 23 && p % 16 == 0 && ld % 16 == 0 && ld >= 0 && ld <= 1 << 23 &&
         (blocks <= 1 || (ld_scale <= 1 << 28 && ld_scale * blocks < 1 << 29));
}

// One launch: rows m .. m + M - 1 and columns n .. n + N - 1 of C by tiles_m x
// tiles_n workgroups, times `parts` that share K by `each` blocks (the tile kernels).
struct Launch {
  Kind kind;
  int64_t m, M, n, N;
  uint32_t tiles_m, tiles_n, each;
  int parts;
};

// Calls launch(Launch) for every launch of a product, M, N > 0, until one does
// not give `ok`. exact: an fp32 C. direct: both operands are direct(). Parts > 1
// leave partial sums in the workspace, to be joined.
template <class E, class F>
E for_launches(int64_t M, int64_t N, int64_t K, bool exact, bool square, bool direct, E ok, F launch) {
  const int64_t blocks = tiles_of(K, 128);
  // Rows of tiles in launches of at most kGrid tiles.
  auto rows = [&](Kind kind, int64_t n, int64_t cols, uint32_t each, int parts) -> E {
    const int bm = rows_of(kind), bn = cols_of(kind);
    const int64_t tn = tiles_of(cols, bn), most = std::max<int64_t>(1, kGrid / tn) * bm;
    for (int64_t m = 0; m < M; m += most) {
      const int64_t some = std::min(M - m, most);
      const E e = launch(Launch{kind, m, some, n, cols, (uint32_t)tiles_of(some, bm), (uint32_t)tn, each, parts});
      if (e != ok) return e;
    }
    return ok;
  };
  const Kind kind = kind_of(M, N, K);
  if (kind != Kind::Tile) return rows(kind, 0, N, (uint32_t)blocks, 1);
  if (!exact && square && direct && tiles_of(M, 128) * tiles_of(N, 256) >= 512) {
    // A last column of tiles that is nearly empty and costs a round of the
    // CUs goes to the small kernel: in one launch and in two, us a call,
    //   4,001 x 4,099 x 8,200    204  169     8,065 x 2,051 x 2,064     62   51
    //   4,001 x 4,128 x 8,192    165  144     8,065 x 2,080 x 2,064     62   52
    //   4,001 x 4,128 x 2,048     49   43    16,257 x 1,056 x 4,096     94   87
    // Below 16 blocks of K and past 32 columns it would gain at some sizes too
    // (4,001 x 4,112 x 768 27 and 23, 4,001 x 4,160 x 2,048 50 and 43) and at some
    // not (16,257 x 1,056 x 768 26 and 26, 32,641 x 273 x 1,536 27 and 27). Where
    // it is the only column, one launch stays (in the small kernel and in this
    // one: 65,536 x 32 x 2,048 47 and 38, 70,000 x 1 x 2,048 37 and 51).
    auto rounds = [&](int64_t cols) { return tiles_of(tiles_of(M, 128) * tiles_of(cols, 256), 512); };
    int64_t cols = N;
    const int64_t over = N % 256;
    if (over > 0 && over <= 32 && over < N && blocks >= 16 && rounds(N - over) < rounds(N)) {
      cols -= over;
      const E e = rows(over <= 16 ? Kind::Small11 : Kind::Small22, cols, over, (uint32_t)blocks, 1);
      if (e != ok) return e;
    }
    return rows(Kind::Wide, 0, cols, (uint32_t)blocks, 1);
  }
  const int split = split_of(M, N, K, exact);
  const uint32_t each = (uint32_t)tiles_of(blocks, split);
  return rows(Kind::Tile, 0, N, each, each ? (int)tiles_of(blocks, each) : 1);
}

}  // namespace fp8plan
