// Launchers of linear.hip (internal; the public surface is include/dion_hip.h).
#pragma once
#include "common.h"

namespace dion {

enum LinAct { kActNone, kActRelu, kActReluSquared, kActGelu, kActGeluTanh, kActSilu, kActCount };

// C[M][N] = sum over K of P[m][k] Q[n][k], operands bf16, sums fp32, then (has_epilogue) act(. + bias) + residual.
// An operand lies with the reduction along its rows ([M][K], [N][K]) or, *_kmajor, along its columns ([K][M], [K][N]).
// Rows of an operand are whole 16-byte chunks: they start on 16-byte boundaries, and where their extent is not a multiple of 8
// elements, what lies behind it up to one belongs to the row too: zeros where the reduction runs along the rows.
struct LinProduct {
  const bf16_t *P, *Q;
  int64_t ldp, ldq;  // elements between rows, at most kLinMaxLd
  int p_kmajor, q_kmajor;
  int M, N, K;
  bf16_t* C;  // [M][N], dense
  // epilogue
  int act;
  const void* bias;  // [N] or null
  int bias_dtype;    // 0 bf16, 1 fp32
  const bf16_t* R;   // [M][N] addend or null, ldr elements between rows
  int64_t ldr;
  uint16_t* slope;  // [M][N rounded up to 8] act'(z), 16-byte aligned, or null: see linear.hip
  // partial sums of a split reduction: lin_product_scratch(...) bytes
  float* scratch;
};
constexpr int64_t kLinMaxLd = int64_t(1) << 21;

size_t lin_product_scratch(int M, int N, int K, int p_kmajor, int q_kmajor);
hipError_t launch_lin_product(const LinProduct& p, hipStream_t st);

// dst[rows][cols rounded up to 8] = src (times slope, laid out like dst), bf16, zero behind column cols;
// partial[lin_sum_parts(rows)][cols]: sums over runs of rows, in fp32, before rounding.  dst or partial may be null.
int lin_sum_parts(int rows);
hipError_t launch_lin_prepare(const bf16_t* src, int64_t ld, const uint16_t* slope, int act, int rows, int cols, bf16_t* dst,
                              float* partial, hipStream_t st);
hipError_t launch_lin_sum(const float* partial, int parts, int cols, void* out, int out_dtype, hipStream_t st);

}  // namespace dion
