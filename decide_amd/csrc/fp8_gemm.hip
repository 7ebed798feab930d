// C = A . B^T of 8-bit arrays with a scale for each block of 128 along K:
//   C[m][n] = sum over blocks b of sa[b][m] sb[b][n] sum over k in b of A[m][k] B[n][k]
// One MFMA (16 x 16 x 128) is one block's inner sum of 16 x 16 outputs; its
// result is scaled and added to the fp32 sums in registers.
#include "fp8_ops.hpp"
#include "fp8_plan.hpp"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// One 16 x 16 x 128 product. Lane l feeds row l % 16 of each operand with 32 of
// the block's elements, the same ones for both (which ones is free: the sum over
// the block does not tell), and owns rows 4 (l / 16) .. + 3 of the first operand
// in column l % 16 of the second. E5A, E5B: the operands are e5m2.
//
// EXACT: on the 16-bit matrix instructions, of operands widened to fp16 (which
// holds every e4m3 and e5m2 value): products are exact and sums keep fp32's 24
// bits. The 8-bit instruction has twice the rate, but it adds eight products at
// a time, cut towards zero at 13 bits below two to the largest sum of two
// exponents: sums off by 1.2e-5 to 1.5e-5 of their norm for normal operands (the
// 16-bit one: 1e-8). That is far below the rounding of a 16-bit C and far above
// that of an fp32 one. At most seven products lose 2^-13 of the largest, 2^-10 of
// the terms' magnitudes; a subnormal counts with the least normal exponent, up to
// three bits above its own (e5m2 two), so that 2^-7 (2^-8) is the most where such a
// product is the largest. Zeros do not count.
template <bool EXACT, bool E5>
struct Operand {
  i32x8 v;
  __device__ __forceinline__ explicit Operand(const uint4 &lo, const uint4 &hi)
      : v{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w} {}
};
template <bool E5>
struct Operand<true, E5> {
  f16x8 v[4];
  __device__ __forceinline__ explicit Operand(const uint4 &lo, const uint4 &hi) {
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    auto widen = [](uint32_t q, auto upper) {
      constexpr bool U = decltype(upper)::value;
      if constexpr (E5) return __builtin_amdgcn_cvt_scalef32_pk_f16_bf8((int)q, 1.0f, U);
      else return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)q, 1.0f, U);
    };
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const auto l = widen(w[i], std::false_type{}), h = widen(w[i], std::true_type{});
      const int at = 4 * (i & 1);
      v[i / 2][at] = l[0], v[i / 2][at + 1] = l[1], v[i / 2][at + 2] = h[0], v[i / 2][at + 3] = h[1];
    }
  }
};
template <bool E5A, bool E5B>
__device__ __forceinline__ f32x4 mma_block(const Operand<false, E5A> &a, const Operand<false, E5B> &b) {
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, zero, E5A, E5B, 0, 0, 0, 0);
}
template <bool E5A, bool E5B>
__device__ __forceinline__ f32x4 mma_block(const Operand<true, E5A> &a, const Operand<true, E5B> &b) {
  f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 4; i++) c = mma16x16<f16>(a.v[i], b.v[i], c);
  return c;
}

// 16 bytes at column k of a row of K; zeros past its end.
__device__ __forceinline__ uint4 chunk_of(const uint8_t *row, int64_t k, int64_t K) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (k + 16 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (k < K) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 15; i++)
      if (k + i < K) w[i / 4] |= (uint32_t)row[k + i] << (8 * (i % 4));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}

// Eight consecutive outputs of a row from column n on.
template <class T>
__device__ __forceinline__ void put8(T *row, int64_t n, int64_t N, float (&v)[8], bool accumulate) {
  if (n + 8 <= N) {
    T t[8];
    if constexpr (sizeof(T) == 4)
      if (accumulate) {
        __builtin_memcpy(t, row + n, sizeof(t));
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] += t[i];
      }
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = to_elem<T>(v[i]);
    __builtin_memcpy(row + n, t, sizeof(t));
  } else {
#pragma unroll
    for (int i = 0; i < 7; i++)
      if (n + i < N) row[n + i] = to_elem<T>(sizeof(T) == 4 && accumulate ? (float)row[n + i] + v[i] : v[i]);
  }
}

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A buffer of `bytes` from `base` on, for loads that read nothing past its end (a
// load whose 4 bytes are not all inside gives 0). At most 2^31: what lies there or
// behind is past the end.
__device__ __forceinline__ i32x4 buffer(const void *base, int64_t bytes) {
  const uint64_t at = (uint64_t)base;
  const int64_t n = max((int64_t)0, min(bytes, (int64_t)1 << 31));
  return {__builtin_amdgcn_readfirstlane((int)at), __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff),
          __builtin_amdgcn_readfirstlane((int)(uint32_t)n), 0x00027000};
}
// An 8-bit operand's buffer: its bytes are rounded up to the 16 of the aligned
// chunk that the last one lies in, on the same page.
__device__ __forceinline__ i32x4 operand_buffer(const void *base, int64_t bytes) {
  return buffer(base, (bytes + 15) & -16);
}
__device__ __forceinline__ uint32_t lds_at(const char *p) {
  return (uint32_t)(size_t)(const __attribute__((address_space(3))) char *)p;
}
// Loads BYTES a lane from `off` in a buffer to LDS, the lanes' side by side from
// `dst` on. In assembly (no register is written) because the compiler would wait
// for the builtin's loads before the next read of LDS, which here is of the other
// slot; the caller waits (vmcnt) before it reads this one. s_nop: for m0.
template <int BYTES>
__device__ __forceinline__ void to_lds(uint32_t dst, uint32_t off, i32x4 from) {
  static_assert(BYTES == 16 || BYTES == 4, "a load's width");
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(off), "s"(from)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(dst), "v"(off), "s"(from)
                 : "memory", "m0");
}

// A workgroup's tile of the product, and the blocks along K that it sums.
// Consecutive workgroups go round-robin over the 8 XCDs: each XCD takes a
// contiguous range of the tiles, in patches of kPatch rows of tiles so that the
// tiles that run there together share panels of both operands in its L2.
constexpr int kPatch = 8;
struct TileAt {
  int64_t m, n;
  __device__ __forceinline__ TileAt(uint32_t tiles_m, uint32_t tiles_n) {
    const uint32_t bid = blockIdx.x, nt = gridDim.x, q = nt >> 3, r = nt & 7, xcd = bid & 7;
    const uint32_t t = xcd * q + min(xcd, r) + (bid >> 3);
    const uint32_t patch = t / (kPatch * tiles_n), in = t - patch * kPatch * tiles_n;
    const uint32_t tall = min((uint32_t)kPatch, tiles_m - patch * kPatch);
    m = patch * kPatch + in % tall;
    n = in / tall;
  }
};

// A tile of BM x BN outputs by WGM x WGN waves, its operands through LDS by
// direct loads (buffer_load ... lds), two blocks of K in turn: one lands while
// the other is multiplied. LDS rows of 128 bytes, their 16-byte chunks swizzled
// on the global side of the load so that 16 lanes read distinct banks. The
// operands' rows start at multiples of 16 bytes; what a load reads past a row's
// end is its padding or the next row (nothing past the array's last chunk), and
// the last block's is cleared in LDS before it is multiplied. RAGGED: rows of any
// alignment, through registers, whose unaligned loads bound it (4,001 x 4,099 x
// 8,200 406 us, aligned 161; 4,096 x 768 x 768 16 and 8).
//
// B is the instruction's first operand, its rows dealt to the tiles of a wave so
// that a lane holds runs of eight consecutive columns of C: 16 bytes of a 16-bit
// C straight from registers, four lanes side by side.
//
// ONE_B: B has one slot, since a wave holds a block's B in registers before the
// next one's is needed: two workgroups of 128 x 256 tiles fit a CU's LDS, each of
// which computes while the other waits (32,768 x 2,304 x 768: 90 us, 128 x 128 96;
// 8,192 cubed 499 and 559).
//
// At 8,192 cubed (495 us, 2.2 PFLOP/s; a library product without block scales 2.7)
// bound by power: the matrix cores are 63% busy, LDS 28%, no bank conflicts, and
// launches of equal cycles take 482 us at 1.8 GHz and 575 at 1.5. At K = 768
// (32,768 x 2,304, 1.3 PFLOP/s) the matrix cores are 38% busy: the tiles without
// their stores take 58 us and the stores alone 31, which overlap only between a
// CU's two workgroups, and the last of 4.5 rounds leaves half of the places empty.
// EXACT (928 us at 8,192 cubed, 1.2 PFLOP/s): the vector unit, which widens the
// operands, and the matrix cores share a wave's issue: 50% and 60% busy.
template <bool EXACT, bool E5A, bool E5B, bool SQUARE, int BM, int BN, int WGM, int WGN, bool ONE_B, bool RAGGED>
__global__ __launch_bounds__(64 * WGM * WGN, 2) void gemm_fp8_tile_kernel(Fp8GemmArgs g, int c_type, uint32_t tiles_m,
                                                                         uint32_t tiles_n, uint32_t each) {
  constexpr int NW = WGM * WGN, WM = BM / WGM, WN = BN / WGN, TM = WM / 16, TN = WN / 16;
  constexpr int LOADS_A = BM / (8 * NW), LOADS_B = BN / (8 * NW), LOADS_S = (BM + BN + 64 * NW - 1) / (64 * NW);
  static_assert(NW % 4 == 0 && LOADS_A * 8 * NW == BM && LOADS_B * 8 * NW == BN && WN == 64, "a wave's share of a stage");
  static_assert(!ONE_B || !EXACT, "the loop that keeps B in registers across blocks");
  static_assert(!RAGGED || (!ONE_B && BM + BN == 64 * NW), "a thread brings one scale");
  constexpr int AT_B = 2 * BM * 128, AT_S = AT_B + (ONE_B ? 1 : 2) * BN * 128, SCALES = LOADS_S * 256 * NW;
  __shared__ __attribute__((aligned(1024))) char smem[AT_S + 2 * SCALES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WGN, wn = wave % WGN, r16 = lane & 15, g4 = lane >> 4;
  const TileAt at(tiles_m, tiles_n);
  const int64_t m0 = at.m * BM, n0 = at.n * BN;
  // This workgroup's blocks: `count` from kb0 on, `whole` of them 128 wide.
  const int blocks = (int)((g.K + 127) / 128), kb0 = blockIdx.y * each, count = min(blocks - kb0, (int)each);
  const int whole = min(count, (int)(g.K / 128) - kb0);
  auto slot_a = [&](int slot) { return smem + slot * BM * 128; };
  auto slot_b = [&](int slot) { return smem + AT_B + (ONE_B ? 0 : slot) * BN * 128; };
  auto slot_s = [&](int slot) { return smem + AT_S + slot * SCALES; };

  // Loads: instruction i of a wave fills rows 8 (wave + NW i) .. + 7; lane l row l / 8, place l % 8 of its chunks.
  const int lrow = 8 * wave + (lane >> 3);
  auto swz_a = [](int r) { return (r >> 1) & 7; };
  auto swz_b = [](int r) { return (r >> 1 & 1) | (r >> 2 & 6); };
  const uint32_t off_a = (uint32_t)lrow * (uint32_t)g.lda + ((lane & 7) ^ swz_a(lrow)) * 16;
  const uint32_t off_b = (uint32_t)lrow * (uint32_t)g.ldb + ((lane & 7) ^ swz_b(lrow)) * 16;
  // The operands' buffers begin at the tile's first row and block, so that only
  // the lanes' offsets move on. Past the last block these lie past the end (no
  // branch stands between the loads).
  i32x4 from_a = operand_buffer((const char *)g.A + m0 * g.lda + kb0 * 128, (g.M - m0 - 1) * g.lda + g.K - kb0 * 128);
  i32x4 from_b = operand_buffer((const char *)g.B + n0 * g.ldb + kb0 * 128, (g.N - n0 - 1) * g.ldb + g.K - kb0 * 128);
  i32x4 from_s[LOADS_S];
  uint32_t off_s[LOADS_S], step_s[LOADS_S];
#pragma unroll
  for (int i = 0; i < LOADS_S; i++) {
    // Scales of 64 rows: those of A's, then of B's.
    const int row = 64 * (wave + i * NW);
    const bool b = row >= BM;
    const int64_t s0 = b ? (SQUARE ? n0 / 128 : n0 + row - BM) : m0 + row, ld = b ? g.ldsb : g.ldsa;
    const int64_t rows = b ? (SQUARE ? (g.N + 127) / 128 : g.N) : g.M;
    from_s[i] = buffer((b ? g.sb : g.sa) + s0 + kb0 * ld, row < BM + BN ? ((blocks - kb0 - 1) * ld + rows - s0) * 4 : 0);
    off_s[i] = 4 * (SQUARE && b ? (row - BM + lane) / 128 : lane);
    step_s[i] = 4 * (uint32_t)ld;
    asm volatile("s_nop 4" : "+s"(from_a), "+s"(from_b), "+s"(from_s[i]));  // written by vector instructions, read by to_lds
  }
  // RAGGED: through registers instead, a block ahead of their way into LDS.
  uint4 held_a[RAGGED ? LOADS_A : 1], held_b[RAGGED ? LOADS_B : 1];
  float held_s = 0.0f;
  auto hold = [&](int n) __attribute__((always_inline)) {
    if (n >= count) return;
    const int64_t k = (int64_t)(kb0 + n) * 128;
    auto each = [&](auto read) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < (RAGGED ? LOADS_A : 0); i++)
        held_a[i] = read((const uint8_t *)g.A + min(m0 + lrow + i * 8 * NW, g.M - 1) * g.lda,
                         k + ((lane & 7) ^ swz_a(lrow)) * 16);
#pragma unroll
      for (int i = 0; i < (RAGGED ? LOADS_B : 0); i++)
        held_b[i] = read((const uint8_t *)g.B + min(n0 + lrow + i * 8 * NW, g.N - 1) * g.ldb,
                         k + ((lane & 7) ^ swz_b(lrow)) * 16);
    };
    if (k + 128 <= g.K)
      each([](const uint8_t *row, int64_t at) {
        uint4 v;
        __builtin_memcpy(&v, row + at, 16);
        return v;
      });
    else
      each([&](const uint8_t *row, int64_t at) { return chunk_of(row, at, g.K); });
    const int64_t row = tid < BM ? min(m0 + tid, g.M - 1) : min(n0 + tid - BM, g.N - 1) / (SQUARE ? 128 : 1);
    held_s = tid < BM ? g.sa[(kb0 + n) * g.ldsa + row] : g.sb[(kb0 + n) * g.ldsb + row];
  };
  auto let_go = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < (RAGGED ? LOADS_A : 0); i++)
      *(uint4 *)(slot_a(slot) + (wave + i * NW) * 1024 + lane * 16) = held_a[i];
#pragma unroll
    for (int i = 0; i < (RAGGED ? LOADS_B : 0); i++)
      *(uint4 *)(slot_b(slot) + (wave + i * NW) * 1024 + lane * 16) = held_b[i];
    ((float *)slot_s(slot))[tid] = held_s;
  };
  auto at_block = [&](int n, uint32_t step) { return n < count ? n * step : 1u << 31; };  // n: from kb0 on
  auto issue_a = [&](int slot, int n) {
    const uint32_t k = at_block(n, 128);
#pragma unroll
    for (int i = 0; i < LOADS_A; i++)
      to_lds<16>(lds_at(slot_a(slot)) + (wave + i * NW) * 1024, off_a + i * 8 * NW * (uint32_t)g.lda + k, from_a);
#pragma unroll
    for (int i = 0; i < LOADS_S; i++)
      to_lds<4>(lds_at(slot_s(slot)) + 256 * (wave + i * NW), off_s[i] + at_block(n, step_s[i]), from_s[i]);
  };
  auto issue_b = [&](int slot, int n) {
    const uint32_t k = at_block(n, 128);
#pragma unroll
    for (int i = 0; i < LOADS_B; i++)
      to_lds<16>(lds_at(slot_b(slot)) + (wave + i * NW) * 1024, off_b + i * 8 * NW * (uint32_t)g.ldb + k, from_b);
  };

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = {0.0f, 0.0f, 0.0f, 0.0f};

  // A wave's operands in a block's slots: row i of A's 16 x 128 pieces, piece j of B's, and their scales.
  typedef Operand<EXACT, E5A> OpA;
  typedef Operand<EXACT, E5B> OpB;
  const int ar = wm * WM + r16, br = wn * WN + 8 * (r16 >> 2) + (r16 & 3);
  int at_a[2], at_b[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    at_a[h] = ar * 128 + ((g4 ^ swz_a(ar) ^ 4 * h) << 4);
    at_b[h] = br * 128 + ((g4 ^ swz_b(br) ^ 4 * h) << 4);
  }
  auto get_a = [&](int slot, int i) {
    const char *const s = slot_a(slot) + i * 2048;
    return OpA(*(const uint4 *)(s + at_a[0]), *(const uint4 *)(s + at_a[1]));
  };
  auto get_b = [&](int slot, int j) {
    const char *const s = slot_b(slot) + (32 * (j >> 1) + 4 * (j & 1)) * 128;
    return OpB(*(const uint4 *)(s + at_b[0]), *(const uint4 *)(s + at_b[1]));
  };
  auto scale_a = [&](int slot, int i) { return ((const float *)slot_s(slot))[ar + 16 * i]; };
  auto scale_b = [&](int slot) { return SQUARE ? ((const float *)slot_s(slot))[BM + wn * WN] : 1.0f; };
  auto scale_row = [&](int slot, int j) {
    return *(const f32x4 *)(slot_s(slot) + 4 * (BM + wn * WN + 32 * (j >> 1) + 4 * (j & 1) + 8 * g4));
  };
  // acc += p * s (* t, the columns' own scales).
  auto add = [&](f32x4 &sum, const f32x4 &p, float s, const f32x4 &t) {
#pragma unroll
    for (int e = 0; e < 4; e++) sum[e] = fmaf(p[e], SQUARE ? s : s * t[e], sum[e]);
  };
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  // One block of K. One row of 16 x 16 tiles after the other: the next one's
  // operand is read and the last one's products are scaled and added while this
  // one multiplies.
  auto multiply = [&](int slot) {
    const OpB b[4] = {get_b(slot, 0), get_b(slot, 1), get_b(slot, 2), get_b(slot, 3)};
    const float sb = scale_b(slot);
    float sa = scale_a(slot, 0), before = 0.0f;
    OpA a[2] = {get_a(slot, 0), get_a(slot, 0)};
    f32x4 p[2][TN];
#pragma unroll
    for (int i = 0; i <= TM; i++) {
      const float s = sa * sb;
      if (i + 1 < TM) {
        a[(i + 1) & 1] = get_a(slot, i + 1);
        sa = scale_a(slot, i + 1);
      }
      if (i < TM)
#pragma unroll
        for (int j = 0; j < TN; j++) p[i & 1][j] = mma_block(b[j], a[i & 1]);
      if (i > 0)
#pragma unroll
        for (int j = 0; j < TN; j++) add(acc[i - 1][j], p[(i - 1) & 1][j], before, SQUARE ? zero : scale_row(slot, j));
      before = s;
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // A block's slots are read once it has landed for every wave, and written once
  // every wave is done with them: from here on block n + 1 is read, n + 2 sent for.
  auto change_over = [&](int slot, int n) __attribute__((always_inline)) {
    if constexpr (RAGGED) {
      let_go(slot ^ 1);
      __syncthreads();
      hold(n + 2);
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      issue_a(slot, n + 2);
      if constexpr (!ONE_B) issue_b(slot, n + 2);
    }
  };
  auto done = [] {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
  };
  int slot = 0;
  if constexpr (RAGGED) {
    hold(0);
  } else {
    issue_a(0, 0);
    issue_b(0, 0);
  }
  change_over(1, -1);
  if constexpr (EXACT) {
    for (int n = 0; n < whole; n++, slot ^= 1) {
      multiply(slot);
      change_over(slot, n);
    }
  } else if (whole > 0) {
    // As multiply(), across the blocks: the slots change over at row TM - 2,
    // with this block's reads of A all done, and each of the last row's products
    // makes room for a piece of the next block's B.
    OpB b[4] = {get_b(0, 0), get_b(0, 1), get_b(0, 2), get_b(0, 3)};
    OpA a[2] = {get_a(0, 0), get_a(0, 0)};
    float sa = scale_a(0, 0), sb = scale_b(0), before = 0.0f;
    f32x4 p[TN], t[SQUARE ? 1 : TN];
#pragma unroll
    for (int j = 0; j < TN; j++) p[j] = t[SQUARE ? 0 : j] = zero;
    for (int n = 0; n < whole; n++, slot ^= 1) {
      const int next = slot ^ 1;
      if constexpr (ONE_B) {
        done();  // every wave has B in registers
        issue_b(0, n + 1);
      }
#pragma unroll
      for (int i = 0; i < TM; i++) {
        const float s = sa * sb;
        if (i + 1 < TM) {
          a[(i + 1) & 1] = get_a(slot, i + 1);
          sa = scale_a(slot, i + 1);
        } else {
          a[0] = get_a(next, 0);
          sa = scale_a(next, 0);
          sb = scale_b(next);
        }
        if (i == TM - 2) {
          change_over(slot, n);
        }
#pragma unroll
        for (int j = 0; j < TN; j++) {
          // The row before, of the block before in the first.
          add(acc[(i + TM - 1) % TM][j], p[j], before, t[SQUARE ? 0 : j]);
          if constexpr (!SQUARE)
            if (i == 0) t[j] = scale_row(slot, j);
          p[j] = mma_block(b[j], a[i & 1]);
          if (i == TM - 1) b[j] = get_b(next, j);
          __builtin_amdgcn_sched_barrier(0);
        }
        before = s;
      }
    }
#pragma unroll
    for (int j = 0; j < TN; j++) add(acc[TM - 1][j], p[j], before, t[SQUARE ? 0 : j]);
  }
  if (whole < count) {
    // The last block ends inside: what lies past the end of K is cleared.
    const int rem = (int)(g.K % 128);
    if constexpr (ONE_B) done();
    for (int c = tid; c < (BM + BN) * 8; c += 64 * NW) {
      const int r = c >> 3, n = rem - 16 * ((c & 7) ^ (r < BM ? swz_a(r) : swz_b(r - BM)));
      if (n >= 16) continue;
      uint32_t *const w = (uint32_t *)(r < BM ? slot_a(slot) + 16 * c : slot_b(slot) + 16 * (c - 8 * BM));
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = n >= 4 * i + 4 ? w[i] : n <= 4 * i ? 0u : w[i] & ((1u << 8 * (n - 4 * i)) - 1u);
    }
    __syncthreads();
    multiply(slot);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load to LDS outlives the workgroup

  auto put = [&](auto *C, int64_t ldc, bool accumulate) {
#pragma unroll
    for (int i = 0; i < TM; i++) {
      const int64_t m = m0 + wm * WM + 16 * i + r16;
      if (m >= g.M) continue;
#pragma unroll
      for (int j = 0; j < TN / 2; j++) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = acc[i][2 * j + (e >> 2)][e & 3];
        put8(C + m * ldc, n0 + wn * WN + 32 * j + 8 * g4, g.N, v, accumulate);
      }
    }
  };
  if (gridDim.y > 1) put(g.work + blockIdx.y * g.M * g.N, g.N, false);
  else if (c_type == PREC_F32) put((float *)g.C, g.ldc, g.accumulate);
  else if (c_type == PREC_BF16) put((bf16 *)g.C, g.ldc, false);
  else put((f16 *)g.C, g.ldc, false);
}

// Few rows (or few outputs): a tile of 16 TM x 16 TN outputs by eight waves that
// share the blocks along K, each with its operands straight from memory to
// registers one block ahead; their sums are joined through LDS in order. Rows of
// any alignment.
constexpr int kSmallWaves = 8;
template <bool EXACT, bool E5A, bool E5B, bool SQUARE, int TM, int TN, int DEPTH>
__global__ __launch_bounds__(64 * kSmallWaves, 2) void gemm_fp8_small_kernel(Fp8GemmArgs g, int c_type, uint32_t tiles_m,
                                                                            uint32_t tiles_n) {
  constexpr int BM = 16 * TM, BN = 16 * TN, NT = 64 * kSmallWaves;
  __shared__ __attribute__((aligned(16))) float part[kSmallWaves][BM][BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;
  const TileAt at(tiles_m, tiles_n);
  const int64_t m0 = at.m * BM, n0 = at.n * BN;
  const int blocks = (int)((g.K + 127) / 128);
  const uint8_t *pa[TM], *pb[TN];
  uint32_t row_a[TM], row_b[SQUARE ? 1 : 4 * TN];  // places of the scales in a block of columns
#pragma unroll
  for (int i = 0; i < TM; i++) {
    const int64_t m = min(m0 + 16 * i + r16, g.M - 1);
    pa[i] = (const uint8_t *)g.A + m * g.lda;
    row_a[i] = (uint32_t)m;
  }
#pragma unroll
  for (int j = 0; j < TN; j++) {
    pb[j] = (const uint8_t *)g.B + min(n0 + 16 * j + r16, g.N - 1) * g.ldb;
    if constexpr (!SQUARE)
#pragma unroll
      for (int e = 0; e < 4; e++) row_b[4 * j + e] = (uint32_t)min(n0 + 16 * j + 4 * g4 + e, g.N - 1);
  }
  if constexpr (SQUARE) row_b[0] = (uint32_t)(n0 / 128);
  struct Stage {
    uint4 a[TM][2], b[TN][2];
    float sa[TM], sb[SQUARE ? 1 : 4 * TN];
  };
  auto fetch = [&](Stage &s, int kb) {
    const int64_t k = (int64_t)kb * 128 + 16 * g4;
    if ((int64_t)(kb + 1) * 128 <= g.K) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int j = 0; j < TN; j++) __builtin_memcpy(&s.b[j][h], pb[j] + k + 64 * h, 16);
#pragma unroll
        for (int i = 0; i < TM; i++) __builtin_memcpy(&s.a[i][h], pa[i] + k + 64 * h, 16);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int j = 0; j < TN; j++) s.b[j][h] = chunk_of(pb[j], k + 64 * h, g.K);
#pragma unroll
        for (int i = 0; i < TM; i++) s.a[i][h] = chunk_of(pa[i], k + 64 * h, g.K);
      }
    }
#pragma unroll
    for (int i = 0; i < TM; i++) s.sa[i] = (g.sa + kb * g.ldsa)[row_a[i]];
#pragma unroll
    for (int j = 0; j < (SQUARE ? 1 : 4 * TN); j++) s.sb[j] = (g.sb + kb * g.ldsb)[row_b[j]];
  };
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) acc[i][j] = {0.0f, 0.0f, 0.0f, 0.0f};
  Stage st[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; d++)
    if (wave + d * kSmallWaves < blocks) fetch(st[d], wave + d * kSmallWaves);
  for (int kb = wave; kb < blocks; kb += DEPTH * kSmallWaves)
#pragma unroll
    for (int d = 0; d < DEPTH; d++) {
      const int now = kb + d * kSmallWaves;
      if (now >= blocks) break;
      Stage &s = st[d];
#pragma unroll
      for (int j = 0; j < TN; j++) {
        const Operand<EXACT, E5B> ob(s.b[j][0], s.b[j][1]);
#pragma unroll
        for (int i = 0; i < TM; i++) {
          const f32x4 p = mma_block(ob, Operand<EXACT, E5A>(s.a[i][0], s.a[i][1]));
#pragma unroll
          for (int e = 0; e < 4; e++) acc[i][j][e] = fmaf(p[e], s.sa[i] * s.sb[SQUARE ? 0 : 4 * j + e], acc[i][j][e]);
        }
      }
      if (now + DEPTH * kSmallWaves < blocks) fetch(s, now + DEPTH * kSmallWaves);
    }
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++) *(f32x4 *)&part[wave][16 * i + r16][16 * j + 4 * g4] = acc[i][j];
  __syncthreads();
  const int waves = max(1, min(blocks, kSmallWaves));  // the others' sums are 0
  auto put = [&](auto *C, bool accumulate) {
    using T = std::remove_pointer_t<decltype(C)>;
    for (int c = tid; c < BM * BN / 4; c += NT) {
      const int r = c / (BN / 4), col = 4 * (c % (BN / 4));
      const int64_t m = m0 + r, n = n0 + col;
      if (m >= g.M || n >= g.N) continue;
      f32x4 v = *(const f32x4 *)&part[0][r][col];
      for (int w = 1; w < waves; w++) {
        const f32x4 t = *(const f32x4 *)&part[w][r][col];
        v += t;
      }
      T *const to = C + m * g.ldc + n;
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (sizeof(T) == 4 && accumulate && n + e < g.N) v[e] += (float)to[e];
      T t[4] = {to_elem<T>(v[0]), to_elem<T>(v[1]), to_elem<T>(v[2]), to_elem<T>(v[3])};
      if (n + 4 <= g.N) {
        __builtin_memcpy(to, t, sizeof(t));
      } else {
#pragma unroll
        for (int e = 0; e < 3; e++)
          if (n + e < g.N) to[e] = t[e];
      }
    }
  };
  if (c_type == PREC_F32) put((float *)g.C, g.accumulate);
  else if (c_type == PREC_BF16) put((bf16 *)g.C, false);
  else put((f16 *)g.C, false);
}

// The partial sums of a product whose blocks along K several workgroups share,
// added in order: four outputs a thread.
template <class T>
__global__ __launch_bounds__(256) void gemm_fp8_join_kernel(Fp8GemmArgs g, int parts, int64_t per_row) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / per_row, n = 4 * (i - m * per_row);
  if (m >= g.M) return;
  const float *from = g.work + m * g.N + n;
  T *const to = (T *)g.C + m * g.ldc + n;
  const int have = (int)min((int64_t)4, g.N - n);
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (have == 4) {
#pragma unroll 4
    for (int p = 0; p < parts; p++, from += g.M * g.N) {
      float t[4];
      __builtin_memcpy(t, from, 16);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] += t[e];
    }
  } else {
    for (int p = 0; p < parts; p++, from += g.M * g.N)
#pragma unroll
      for (int e = 0; e < 3; e++)
        if (e < have) v[e] += from[e];
  }
  T t[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (sizeof(T) == 4 && g.accumulate && e < have) v[e] += (float)to[e];
    t[e] = to_elem<T>(v[e]);
  }
  if (have == 4) {
    __builtin_memcpy(to, t, sizeof(t));
  } else {
#pragma unroll
    for (int e = 0; e < 3; e++)
      if (e < have) to[e] = t[e];
  }
}

}  // namespace

int64_t gemm_fp8_work(int64_t M, int64_t N, int64_t K) { return fp8plan::work_of(M, N, K); }

hipError_t launch_gemm_fp8(int a_e5m2, int b_e5m2, int c_type, const Fp8GemmArgs &args, hipStream_t s) {
  using fp8plan::Kind;
  using fp8plan::Launch;
  const bool direct = fp8plan::direct((uintptr_t)args.A, args.lda, args.ldsa, args.K) &&
                      fp8plan::direct((uintptr_t)args.B, args.ldb, args.ldsb, args.K);
  auto with = [&](auto ex, auto ea, auto eb, auto sq) -> hipError_t {
    constexpr bool X = decltype(ex)::value, A = decltype(ea)::value, B = decltype(eb)::value, S = decltype(sq)::value;
    int parts = 1;
    auto launch = [&](const Launch &l) -> hipError_t {
      Fp8GemmArgs a = args;
      a.M = l.M;
      a.N = l.N;
      a.A = (const char *)args.A + l.m * args.lda;
      a.sa = args.sa + l.m;
      a.B = (const char *)args.B + l.n * args.ldb;
      a.sb = args.sb + (S ? l.n / kFp8Block : l.n);
      a.C = (char *)args.C + (l.m * args.ldc + l.n) * (c_type == PREC_F32 ? 4 : 2);
      parts = l.parts;
      const uint32_t tm = l.tiles_m, tn = l.tiles_n;
      auto small = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(tm * tn), dim3(64 * kSmallWaves), 0, s, a, c_type, tm, tn);
        return hipGetLastError();
      };
      auto tile = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(tm * tn, parts), dim3(256), 0, s, a, c_type, tm, tn, l.each);
        return hipGetLastError();
      };
      if (l.kind == Kind::Small11) return small(gemm_fp8_small_kernel<X, A, B, S, 1, 1, 3>);
      if (l.kind == Kind::Small22) return small(gemm_fp8_small_kernel<X, A, B, S, 2, 2, 2>);
      if (l.kind == Kind::Small42) return small(gemm_fp8_small_kernel<X, A, B, S, 4, 2, 2>);
      if constexpr (!X && S)
        if (l.kind == Kind::Wide) return tile(gemm_fp8_tile_kernel<X, A, B, S, 128, 256, 1, 4, true, false>);
      return direct ? tile(gemm_fp8_tile_kernel<X, A, B, S, 128, 128, 2, 2, false, false>)
                    : tile(gemm_fp8_tile_kernel<X, A, B, S, 128, 128, 2, 2, false, true>);
    };
    const hipError_t e = fp8plan::for_launches(args.M, args.N, args.K, X, S, direct, hipSuccess, launch);
    if (e != hipSuccess || parts == 1) return e;
    const int64_t per_row = fp8plan::tiles_of(args.N, 4);  // at most 512 tiles are split: one launch
    const dim3 grid((unsigned)fp8plan::tiles_of(args.M * per_row, 256));
    if (X) hipLaunchKernelGGL(gemm_fp8_join_kernel<float>, grid, dim3(256), 0, s, args, parts, per_row);
    else if (c_type == PREC_BF16) hipLaunchKernelGGL(gemm_fp8_join_kernel<bf16>, grid, dim3(256), 0, s, args, parts, per_row);
    else hipLaunchKernelGGL(gemm_fp8_join_kernel<f16>, grid, dim3(256), 0, s, args, parts, per_row);
    return hipGetLastError();
  };
  const std::true_type yes;
  const std::false_type no;
  auto square = [&](auto ex, auto ea, auto eb) { return args.b_square ? with(ex, ea, eb, yes) : with(ex, ea, eb, no); };
  auto type_b = [&](auto ex, auto ea) { return b_e5m2 ? square(ex, ea, yes) : square(ex, ea, no); };
  auto type_a = [&](auto ex) { return a_e5m2 ? type_b(ex, yes) : type_b(ex, no); };
  return c_type == PREC_F32 ? type_a(yes) : type_a(no);
}
