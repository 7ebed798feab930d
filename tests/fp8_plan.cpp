// The launches of a block-scaled product as a function that ctypes can call
// without a GPU.
#include "../decide_amd/csrc/fp8_plan.hpp"

extern "C" {

struct Fp8Launch {
  int64_t kind, m, M, n, N, tiles_m, tiles_n, each, parts;
};

int tile_rows(int kind) { return fp8plan::rows_of((fp8plan::Kind)kind); }
int tile_cols(int kind) { return fp8plan::cols_of((fp8plan::Kind)kind); }
int64_t work_floats(int64_t M, int64_t N, int64_t K) { return fp8plan::work_of(M, N, K); }
int takes_direct(uint64_t p, int64_t ld, int64_t ld_scale, int64_t K) {
  return fp8plan::direct((uintptr_t)p, ld, ld_scale, K);
}

// The number of launches, or -1 past `cap`.
int launches(int64_t M, int64_t N, int64_t K, int exact, int square, int direct, Fp8Launch *out, int cap) {
  int n = 0;
  const int bad = fp8plan::for_launches(M, N, K, exact, square, direct, 0, [&](const fp8plan::Launch &l) {
    if (n == cap) return 1;
    out[n++] = {(int64_t)l.kind, l.m, l.M, l.n, l.N, l.tiles_m, l.tiles_n, l.each, l.parts};
    return 0;
  });
  return bad ? -1 : n;
}

}  // extern "C"
