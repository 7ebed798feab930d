// The 8-bit operators (fp8_quant.hip, fp8_gemm.hip; C entry points in
// fp8_ops.cpp): the RMS norm that writes a product's 8-bit operand, the block
// quantiser, and the product of block-scaled 8-bit arrays.
#pragma once

#include "common.hpp"
#include "fp8_args.hpp"

// Launchers. Types are PREC_* codes that fp8_check.hpp's rules allow; the
// arguments have passed its checks.
hipError_t launch_rms(int x_type, int stream_type, int y_type, const RmsArgs &a, hipStream_t s);
hipError_t launch_quantise(int x_type, const QuantArgs &a, hipStream_t s);
// a_e5m2, b_e5m2: the operands' types (0 e4m3). M, N > 0.
hipError_t launch_gemm_fp8(int a_e5m2, int b_e5m2, int c_type, const Fp8GemmArgs &a, hipStream_t s);
// Floats of workspace of a product of these sizes.
int64_t gemm_fp8_work(int64_t M, int64_t N, int64_t K);
