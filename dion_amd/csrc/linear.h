// Launchers of linear.hip and gated.hip (internal; the public surface is include/dion_hip.h).
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

// How a product runs: on which tiles, and in how many parts of the reduction, of so many slabs of 64.
enum LinTile { kLinFew, kLin128, kLinWide, kLin256 };
struct LinPlan {
  LinTile tile;
  int splits, slabs;
};
LinPlan lin_plan(int M, int N, int K, int p_kmajor, int q_kmajor, bool may_be_few = true);

size_t lin_product_scratch(int M, int N, int K, int p_kmajor, int q_kmajor);
hipError_t launch_lin_product(const LinProduct& p, hipStream_t st);

// dst[rows][cols rounded up to 8] = src (times slope, laid out like dst), bf16, zero behind column cols;
// partial[lin_sum_parts(rows)][cols]: sums over runs of rows, in fp32, before rounding.  dst or partial may be null.
int lin_sum_parts(int rows);
hipError_t launch_lin_prepare(const bf16_t* src, int64_t ld, const uint16_t* slope, int act, int rows, int cols, bf16_t* dst,
                              float* partial, hipStream_t st);
hipError_t launch_lin_sum(const float* partial, int parts, int cols, void* out, int out_dtype, hipStream_t st);
// ... of partial[parts][2][cols]: out from the first, out2 from the second; either may be null.
hipError_t launch_lin_sum(const float* partial, int parts, int cols, void* out, int out_dtype, hipStream_t st, void* out2, int out2_dtype);
// C[M][N] = the sum of part[0 .. splits)[M][N], in that order, rounded once.
hipError_t launch_lin_join(const float* part, int splits, int M, int N, bf16_t* C, hipStream_t st);

// ---- gated.hip: h = act(x Wg^T + bg) * (x Wu^T + bu).  Operands as above; the rows of both weights are as long and as many.
struct GatedProduct {
  const bf16_t *X, *Wg, *Wu;
  int64_t ldx, ldg, ldu;
  int M, N, K;  // tokens, columns of h, columns of x
  bf16_t* H;    // [M][N], dense
  int act;
  const void *bg, *bu;  // [N] or null
  int bg_dtype, bu_dtype;
  void* kept;  // gated_kept_bytes(M, N, wide), 16-byte aligned, or null: what launch_gated_dz reads
  int wide;    // of 32 bits a value instead of 24
  float* scratch;  // gated_product_scratch(M, N, K) bytes
};
size_t gated_kept_bytes(int M, int N, bool wide);
size_t gated_product_scratch(int M, int N, int K);
hipError_t launch_gated_product(const GatedProduct& p, hipStream_t st);

// dz[rows][2 * (cols rounded up to 8)]: the gradients at x Wg^T + bg and, behind them in a row, at x Wu^T + bu, zeros behind column
// cols; sums[lin_sum_parts(rows)][2][cols]: their sums over runs of rows, in fp32, before rounding.  dz or sums may be null.
hipError_t launch_gated_dz(const bf16_t* dh, int64_t ld, const void* kept, bool wide, int rows, int cols, bf16_t* dz, float* sums,
                           hipStream_t st);

// C[M][N] = P Q + P2 Q2, sums over K each: P, P2 [M][K], ldp elements between rows, Q, Q2 [K][N].
struct PairProduct {
  const bf16_t *P, *P2, *Q, *Q2;
  int64_t ldp, ldq, ldq2;
  int M, N, K;
  bf16_t* C;
  float* scratch;  // pair_product_scratch(M, N, K) bytes
};
size_t pair_product_scratch(int M, int N, int K);
hipError_t launch_pair_product(const PairProduct& p, hipStream_t st);

}  // namespace dion
