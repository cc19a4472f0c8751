// The product a weight matrix stands for, y = act(x W^T + b) + residual, and its gradients:
//   z = x W^T + b        x [T][K], W [N][K]: both with the reduction along rows
//   dz = dy act'(z)      (elementwise, bf16: an operand of two products; db = column sums of it before rounding)
//   dx = dz W            W [N][K] read as it lies, reduction along its columns
//   dW = dz^T x          both operands read as they lie, reduction (the tokens) along their columns
// Operands bf16, sums fp32 in the accumulators of v_mfma_f32_16x16x32_bf16, one rounding where a result is stored.
//
// For the backward pass the forward one keeps act'(z), not z, in 16 bits: slopes of relu, gelu and silu are bounded and are
// kept in fp16 (eleven bits); those of the squared relu, 2 max(z, 0), have no sign and no bound, and are kept as seven bits of
// exponent and nine of mantissa, from 2^-63 to where z^2 leaves fp32.  bf16's eight bits would add an error of the size of
// the rounding of dz itself; so it stays an eighth (a quarter) of that, for the same bytes.
//
// Large products are bound by the matrix units at the clock the power limit leaves (a 256-wide slab takes 1.37 us of ordinary
// values, 1.06 of zeros) and by the output, which all CUs write at once when a round of tiles ends (134 MB of 8192 x 8192 with
// a reduction of 64, where little else is left: 39 us, with an activation's slopes 63). us, y with nothing in the epilogue / dx
// / dW: 8192 x 2048 x 8192 (tokens, fan-in, fan-out) 205 / 193 / 195, 16384 x 4096 x 14336 1349 / 1334 / 1715, 4096 x 2048 x
// 2048 31.7 / 30.8 / 33.1; 8192 x 8192 x 8192 757 / 755 / 776, 1.45 PFLOP/s.
#include "lin_tile.h"

namespace dion {

// Finishes and stores elements (row, col .. col + 3), where the activation is not worth a kernel of its own.
static __device__ __forceinline__ void finish4_any(const LinEpilogue& p, int row, int col, f32x4 z) {
  if (row >= p.M || col >= p.N) return;
  const f32x4 b = bias4(p, col);
  const uint2 r = residual4(p, row, col);
  uint2 y, s;
  switch (p.act) {
    case kActRelu: finish4<kActRelu, true>(p, z, b, r, y, s); break;
    case kActReluSquared: finish4<kActReluSquared, true>(p, z, b, r, y, s); break;
    case kActGelu: finish4<kActGelu, true>(p, z, b, r, y, s); break;
    case kActGeluTanh: finish4<kActGeluTanh, true>(p, z, b, r, y, s); break;
    case kActSilu: finish4<kActSilu, true>(p, z, b, r, y, s); break;
    default: finish4<kActNone, true>(p, z, b, r, y, s); break;
  }
  if (p.slope) *(uint2*)(p.slope + (int64_t)row * slope_pitch(p.N) + col) = s;
  store4(p, p.C + (int64_t)row * p.N + col, col, y);
}

// Adds the parts of a split reduction, in their order, and finishes: four elements per thread.  Ten parts of 32 x 2048 4.4 us,
// of which 2 are the launch; the parts come from L2 and the memory-side cache.
__global__ __launch_bounds__(256) void lin_join_kernel(const LinEpilogue p, const float* __restrict__ part, int splits) {
  const int per_row = (p.N + 3) / 4;
  const int64_t all = (int64_t)p.M * per_row, one = (int64_t)p.M * p.N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int row = (int)(i / per_row), col = (int)(i - (int64_t)row * per_row) * 4;
    const float* q = part + (int64_t)row * p.N + col;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (p.N % 4 == 0) {
#pragma unroll 4
      for (int k = 0; k < splits; ++k) s += *(const f32x4*)(q + k * one);
    } else {
      for (int k = 0; k < splits; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < p.N) s[e] += q[k * one + e];
    }
    finish4_any(p, row, col, s);
  }
}

// ---------------------------------------------------------------------------------------------- few tokens
// Up to 32 rows of x and a weight of a few megabytes: latency is what counts.  A workgroup takes 16 rows of W, its wavefronts an
// equal run of the reduction each; fragments go from memory to registers with no LDS between (a lane's chunk is its MFMA operand
// as it lies), the next U steps' while the MFMAs of these run.  MFMA row: a row of W; column: a token (past the last one, the
// last one again).  The wavefronts' sums meet in LDS and are added in their order.  Bound by the weight's bytes: one token of 4096 to 14336
// 24.4 us (4.8 TB/s, the weight from HBM), of 768 to 768 4.7 us (launch, one way to memory, LDS).
template <int TB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void lin_few_kernel(const LinEpilogue p, const bf16_t* __restrict__ x, int64_t ldx,
                                                             const bf16_t* __restrict__ w, int64_t ldw, int K) {
  constexpr int U = 4;
  __shared__ f32x4 sums[WAVES][TB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l16 = lane & 15, quad = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int wrow = n0 + l16 < p.N ? n0 + l16 : p.N - 1;
  const bf16_t* wp = w + (int64_t)wrow * ldw + quad * 8;
  const bf16_t* xp[TB];
#pragma unroll
  for (int b = 0; b < TB; ++b) xp[b] = x + (int64_t)(b * 16 + l16 < p.M ? b * 16 + l16 : p.M - 1) * ldx + quad * 8;
  f32x4 acc[TB];
#pragma unroll
  for (int b = 0; b < TB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = (K + 31) / 32;
  const int s0 = (int)((int64_t)steps * wave / WAVES), s1 = (int)((int64_t)steps * (wave + 1) / WAVES);
  struct Set {
    bf16x8 w[U], x[TB][U];
  };
  auto fetch = [&](Set& f, int s) {  // steps s .. s + U - 1, zeros behind the run's end and the reduction's
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = s + u < s1 && (s + u) * 32 + quad * 8 < K;
      const bf16x8 zero = {};
      f.w[u] = in ? *(const bf16x8*)(wp + (s + u) * 32) : zero;
#pragma unroll
      for (int b = 0; b < TB; ++b) f.x[b][u] = in ? *(const bf16x8*)(xp[b] + (s + u) * 32) : zero;
    }
  };
  auto multiply = [&](const Set& f) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int b = 0; b < TB; ++b) acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.w[u], f.x[b][u], acc[b], 0, 0, 0);
  };
  Set even, odd;
  fetch(even, s0);
  for (int s = s0; s < s1; s += 2 * U) {
    fetch(odd, s + U);
    multiply(even);
    fetch(even, s + 2 * U);
    multiply(odd);
  }
#pragma unroll
  for (int b = 0; b < TB; ++b) sums[wave][b][lane] = acc[b];
  __syncthreads();
  for (int i = threadIdx.x; i < TB * 64; i += WAVES * 64) {
    const int b = i >> 6, l = i & 63;
    f32x4 t = sums[0][b][l];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) t += sums[k][b][l];
    const int row = b * 16 + (l & 15), col = n0 + 4 * (l >> 4);
    finish4_any(p, row, col, t);
  }
}

// ---------------------------------------------------------------------------------------------- operands and column sums
constexpr int kPrepCols = 256;  // columns of a workgroup: 32 threads of eight, by eight rows

// Rows of a part, a multiple of eight: about 128 parts, which fill the chip where there are few columns.
static int sum_rows(int rows) { return (rows + 1023) / 1024 * 8; }
int lin_sum_parts(int rows) { return (rows + sum_rows(rows) - 1) / sum_rows(rows); }

// One pass for what the products cannot read as it lies: dz, its column sums, and rows that are not whole chunks.  HBM: 6 bytes an
// element with slopes, 8192 x 8192 72 us (5.6 TB/s); 4 bytes for a copy, 2 for sums alone (4096 x 2048 4.7 us).
// SLOPE: src is dy, and dz = dy * act'(z) goes on.  W: elements of src that are read at once; 8: every row is whole chunks.
// NT: non-temporal loads of dy and the slopes, which nothing reads again.
template <bool SLOPE, bool DST, bool SUM, int W, bool NT>
__global__ __launch_bounds__(256) void lin_prepare_kernel(const bf16_t* __restrict__ src, int64_t ld,
                                                          const uint16_t* __restrict__ slope, int act, int rows, int cols,
                                                          bf16_t* __restrict__ dst, float* __restrict__ partial, int per) {
  __shared__ float sums[8][kPrepCols];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c0 = blockIdx.x * kPrepCols + tx * 8, padded = slope_pitch(cols);
  const int r_first = blockIdx.y * per, r_end = r_first + per < rows ? r_first + per : rows;
  float acc[8] = {};
  if (c0 < cols) {
#pragma unroll 2
    for (int r = r_first + ty; r < r_end; r += 8) {
      const bf16_t* q = src + (int64_t)r * ld + c0;
      float v[8];
      if constexpr (W == 8) {
        const u32x4_t w = NT ? __builtin_nontemporal_load((const u32x4_t*)q) : *(const u32x4_t*)q;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float((e & 1) ? (w[e >> 1] & 0xffff0000u) : (w[e >> 1] << 16));
      } else if constexpr (W == 2) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {  // (an even number of columns)
          const uint32_t w = c0 + e < cols ? *(const uint32_t*)(q + e) : 0;
          v[e] = __uint_as_float(w << 16);
          v[e + 1] = __uint_as_float(w & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c0 + e < cols ? bf16_to_f32(q[e]) : 0.f;
      }
      if constexpr (SLOPE) {
        const u32x4_t* sp = (const u32x4_t*)(slope + (int64_t)r * padded + c0);
        const u32x4_t s = NT ? __builtin_nontemporal_load(sp) : *sp;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = slope_unpack(act, (uint16_t)(s[e >> 1] >> (16 * (e & 1))));
          v[e] = c0 + e < cols ? v[e] * f : 0.f;
        }
      }
      if constexpr (DST) st_store8<bf16_t>(dst + (int64_t)r * padded + c0, 0, v);
      if constexpr (SUM)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += v[e];
    }
  }
  if constexpr (SUM) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[ty][tx * 8 + e] = acc[e];
    __syncthreads();
    const int c = blockIdx.x * kPrepCols + threadIdx.x;
    if (c < cols) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += sums[k][threadIdx.x];
      partial[(int64_t)blockIdx.y * cols + c] = s;
    }
  }
}

// out[c] = sum of partial[0 .. parts)[c]: 16 columns of a workgroup, sixteen threads a column.  3 us: a launch and eight loads in a row.
// (out2: of partial[parts][2][cols] the first and the second; `cols` is then that of both.)
__global__ __launch_bounds__(256) void lin_sum_kernel(const float* __restrict__ partial, int parts, int cols, void* out,
                                                      int out_dtype, int split, void* out2, int out2_dtype) {
  __shared__ float sums[16][17];
  const int tx = threadIdx.x & 15, g = threadIdx.x >> 4, c = blockIdx.x * 16 + tx;
  float s = 0.f;
  if (c < cols)
#pragma unroll 4
    for (int k = g; k < parts; k += 16) s += partial[(int64_t)k * cols + c];
  sums[g][tx] = s;
  __syncthreads();
  if (g == 0 && c < cols) {
    s = sums[0][tx];
#pragma unroll
    for (int k = 1; k < 16; ++k) s += sums[k][tx];
    void* const to = c < split ? out : out2;
    const int at = c < split ? c : c - split;
    if (!to) return;
    if (c < split ? out_dtype : out2_dtype) ((float*)to)[at] = s;
    else ((bf16_t*)to)[at] = f32_to_bf16(s);
  }
}

// ---------------------------------------------------------------------------------------------- host
// How a product runs: on which tiles, and in how many parts of the reduction: what is estimated to take least.  us:
//   a round of the 256 CUs: so much a slab and so much for itself (first loads, epilogue).  Measured over reductions of 1024 / 8192,
//     128-wide tiles 12.9 / 63, 256 x 128 21 / 122, 256-wide 34 / 224; from HBM full 128-wide tiles, which read the most, take 0.62 a
//     slab (512 tokens of 4096 x 14336, weights not cached: two parts of them 78, four of 256 x 128 63), from caches 0.45;
//   never less than the bytes at what so many CUs draw from HBM: 4096 x 14336 and one to sixteen tokens in 160 / 256 parts of
//     tiles 28.8 / 25.6, 14336 x 4096 and 128 tokens in 112 / 224 45 / 37;
//   the kernel that joins the parts: 3 and the sums both ways (32 tokens of 2048 x 8192, 16 tiles, in 1 / 4 / 16 parts 46 / 16.8 /
//     13.4).
// lin_few_kernel takes so long per 512 of the reduction, its tokens and a workgroup per CU.  Few / tiles at 1, 8, 16, 32 tokens of
// a weight from HBM: 768 x 768 3.8, 4.1, 4.2, 5.2 / 7.1 to 7.7; 4096 x 4096 8.6, 10.0, 11.9, 16.4 / 11.8 to 12.7; 4096 x 14336
// 23.5, 28.5, 34.8, 50.3 / 25.2 to 25.9; 50304 x 768 15.5, 20.0, 24.5, 57 / 20.4 to 21.7.
LinPlan lin_plan(int M, int N, int K, int p_kmajor, int q_kmajor, bool may_be_few) {
  const int KT = (K + 63) / 64;
  LinPlan best{kLin128, 1, KT};
  double least = 1e30;
  const double bytes = 2.0 * ((double)M * K + (double)N * K + (double)M * N);
  for (int t = kLin128; t <= kLin256; ++t) {
    const int bm = t == kLin128 ? 128 : 256, bn = t == kLin256 ? 256 : 128;
    const double slab = t == kLin256 ? 1.65 : t == kLinWide ? 0.9 : M > 64 && bytes > 64e6 ? 0.55 : 0.45;
    const double fixed = t == kLin256 ? 8.0 : t == kLinWide ? 5.0 : 4.5;
    const int64_t tiles = (int64_t)((M + bm - 1) / bm) * ((N + bn - 1) / bn);
    for (int s = 1; s <= 16 && s <= KT; ++s) {
      const int slabs = (KT + s - 1) / s;
      const int parts = (KT + slabs - 1) / slabs;
      if (parts != s) continue;
      double us = (double)((tiles * parts + 255) / 256) * (slabs * slab + fixed);
      const double streaming = 3.0 + bytes / (tiles * parts >= 256 ? 6.1e6 : tiles * parts > 128 ? 5.1e6 : 3.0e6);
      if (us < streaming) us = streaming;
      if (parts > 1) us += 3.0 + (double)M * N * parts * 8.0 / 6e6;
      if (us < least) {
        least = us;
        best = {(LinTile)t, parts, slabs};
      }
    }
  }
  if (M <= 32 && !p_kmajor && !q_kmajor && may_be_few) {
    const double wgs = (N + 15) / 16, each = M <= 16 ? 0.77 + 0.033 * (M - 1) : 1.5;
    if (2.5 + each * (K / 512.0) * (wgs > 256 ? wgs / 256 : 1) < least) return {kLinFew, 1, 0};
  }
  return best;
}

size_t lin_product_scratch(int M, int N, int K, int p_kmajor, int q_kmajor) {
  const LinPlan plan = lin_plan(M, N, K, p_kmajor, q_kmajor);
  return plan.splits > 1 ? (size_t)plan.splits * M * N * sizeof(float) : 0;
}

template <class Cfg, int ACT>
static hipError_t launch_act(const LinTileParams& tp, hipStream_t st) {
  return tp.e.slope ? launch_tile<Cfg, false, false, ACT, true, false>(tp, st)
                    : launch_tile<Cfg, false, false, ACT, false, false>(tp, st);
}

template <class Cfg>
static hipError_t launch_tiles(const LinProduct& p, LinTileParams tp, hipStream_t st) {
  if (!lin_tile_list<Cfg>(p.M, p.N, tp)) return hipErrorInvalidValue;
  // P past the 256 MB memory-side cache, Q well within it: the XCDs then work on the same rows of P at the same time.  us, a run
  // for each XCD / interleaved: 16384 x 4096 x 14336 1531 / 1434, with W K-major 1501 / 1436, 14336 x 4096 x 16384 both K-major
  // 1729 / 1615, 32768 x 4096 x 8192 1740 / 1615; with Q as large 16384 x 8192 x 16384 3369 / 3534, with P the smaller one
  // 4096 x 14336 x 16384 1571 / 1629.
  tp.interleave = Cfg::BM == 256 && Cfg::BN == 256 && (int64_t)p.M * p.K >= (int64_t(128) << 20) && (int64_t)p.N * p.K <= (int64_t(96) << 20);
  const bool split = tp.splits > 1;
  if (p.p_kmajor)
    return split ? launch_tile<Cfg, true, true, kActNone, false, true>(tp, st) : launch_tile<Cfg, true, true, kActNone, false, false>(tp, st);
  if (p.q_kmajor)
    return split ? launch_tile<Cfg, false, true, kActNone, false, true>(tp, st) : launch_tile<Cfg, false, true, kActNone, false, false>(tp, st);
  if (split) return launch_tile<Cfg, false, false, kActNone, false, true>(tp, st);
  switch (tp.e.act) {
    case kActNone: return launch_tile<Cfg, false, false, kActNone, false, false>(tp, st);
    case kActRelu: return launch_act<Cfg, kActRelu>(tp, st);
    case kActReluSquared: return launch_act<Cfg, kActReluSquared>(tp, st);
    case kActGelu: return launch_act<Cfg, kActGelu>(tp, st);
    case kActGeluTanh: return launch_act<Cfg, kActGeluTanh>(tp, st);
    case kActSilu: return launch_act<Cfg, kActSilu>(tp, st);
    default: return hipErrorInvalidValue;
  }
}

static hipError_t launch_join(const LinEpilogue& e, const float* part, int splits, hipStream_t st) {
  const int64_t wg = ((int64_t)e.M * ((e.N + 3) / 4) + 255) / 256;
  const dim3 grid((unsigned)(wg < 65536 ? wg : 65536));
  hipLaunchKernelGGL(lin_join_kernel, grid, dim3(256), 0, st, e, part, splits);
  return hipGetLastError();
}

hipError_t launch_lin_join(const float* part, int splits, int M, int N, bf16_t* C, hipStream_t st) {
  LinEpilogue e = {};
  e.C = C;
  e.M = M;
  e.N = N;
  e.vec = lin_vec(C, nullptr, N, 0);
  return launch_join(e, part, splits, st);
}

hipError_t launch_lin_product(const LinProduct& p, hipStream_t st) {
  if (p.M <= 0 || p.N <= 0 || p.K <= 0) return hipErrorInvalidValue;
  if (!lin_chunks(p.P, p.ldp, p.p_kmajor ? p.M : p.K) || !lin_chunks(p.Q, p.ldq, p.q_kmajor ? p.N : p.K)) return hipErrorInvalidValue;
  if ((p.p_kmajor && !p.q_kmajor) || (p.q_kmajor && (p.act != kActNone || p.bias || p.R || p.slope))) return hipErrorInvalidValue;
  LinEpilogue e;
  e.C = p.C;
  e.bias = p.bias;
  e.R = p.R;
  e.slope = p.slope;
  e.ldr = p.ldr;
  e.M = p.M;
  e.N = p.N;
  e.act = p.act;
  e.bias_dtype = p.bias_dtype;
  e.vec = lin_vec(p.C, p.R, p.N, p.ldr);
  const LinPlan plan = lin_plan(p.M, p.N, p.K, p.p_kmajor, p.q_kmajor);
  if (plan.tile == kLinFew) {
    const dim3 grid((unsigned)((p.N + 15) / 16));
    auto go = [&](auto tbc, auto wavesc) {
      constexpr int TB = decltype(tbc)::value, WAVES = decltype(wavesc)::value;
      hipLaunchKernelGGL((lin_few_kernel<TB, WAVES>), grid, dim3(WAVES * 64), 0, st, e, p.P, p.ldp, p.Q, p.ldq, p.K);
    };
    // Sixteen wavefronts share a reduction, or four where the rows of W make two workgroups of those per CU: one token of
    // 14336 x 4096 26.0 / 24.0 us, of 50304 x 768 33.5 / 15.8, of 4096 x 14336 24.0 / 26.5, of 2048 x 8192 11.4 / 13.6.
    typedef std::integral_constant<int, 16> many;
    if (p.M > 16) go(std::integral_constant<int, 2>(), many());
    else if (p.N >= 8192) go(std::integral_constant<int, 1>(), std::integral_constant<int, 4>());
    else go(std::integral_constant<int, 1>(), many());
    return hipGetLastError();
  }
  LinTileParams tp;
  tp.e = e;
  tp.P = p.P;
  tp.Q = p.Q;
  tp.ldp = (int)p.ldp;
  tp.ldq = (int)p.ldq;
  tp.K = p.K;
  tp.part = p.scratch;
  tp.splits = plan.splits;
  tp.slabs = plan.slabs;
  if (plan.splits > 1 && !p.scratch) return hipErrorInvalidValue;
  if (hipError_t err = plan.tile == kLin256 ? launch_tiles<Lin256>(p, tp, st)
                       : plan.tile == kLinWide ? launch_tiles<LinWide>(p, tp, st) : launch_tiles<Lin128>(p, tp, st))
    return err;
  if (plan.splits > 1) return launch_join(e, p.scratch, plan.splits, st);
  return hipGetLastError();
}

template <bool SLOPE, bool DST, bool SUM>
static hipError_t launch_prepare(const bf16_t* src, int64_t ld, const uint16_t* slope, int act, int rows, int cols, bf16_t* dst,
                                 float* partial, hipStream_t st) {
  const dim3 grid((cols + kPrepCols - 1) / kPrepCols, lin_sum_parts(rows));
  const uint64_t bytes = (uint64_t)src | (uint64_t)cols * 2 | (uint64_t)ld * 2;
  auto go = [&](auto wc, auto ntc) {
    hipLaunchKernelGGL((lin_prepare_kernel<SLOPE, DST, SUM, decltype(wc)::value, decltype(ntc)::value>), grid, dim3(256), 0, st, src, ld,
                       slope, act, rows, cols, dst, partial, sum_rows(rows));
  };
  if constexpr (SLOPE) {
    // From 30 MB of dy, slopes and dz on.  us without / with, dz alone and with its sums: 777 x 2736 5.0 / 5.2 and 4.5 / 4.8,
    // 4096 x 2048 12.3 / 11.9 and 12.0 / 10.2, 4096 x 14336 69 / 67 and 70 / 66, 8192 x 8192 84 / 69 and 83 / 67.
    if (bytes % 16 == 0 && (int64_t)rows * cols >= (5 << 20)) {
      go(std::integral_constant<int, 8>(), std::true_type());
      return hipGetLastError();
    }
  }
  if (bytes % 16 == 0) go(std::integral_constant<int, 8>(), std::false_type());
  else if (bytes % 4 == 0) go(std::integral_constant<int, 2>(), std::false_type());
  else go(std::integral_constant<int, 1>(), std::false_type());
  return hipGetLastError();
}

hipError_t launch_lin_prepare(const bf16_t* src, int64_t ld, const uint16_t* slope, int act, int rows, int cols, bf16_t* dst,
                              float* partial, hipStream_t st) {
  if (rows <= 0 || cols <= 0 || (!dst && !partial) || ((uint64_t)dst & 15) || ((uint64_t)slope & 15)) return hipErrorInvalidValue;
  if (slope) {
    if (dst && partial) return launch_prepare<true, true, true>(src, ld, slope, act, rows, cols, dst, partial, st);
    if (dst) return launch_prepare<true, true, false>(src, ld, slope, act, rows, cols, dst, partial, st);
    return launch_prepare<true, false, true>(src, ld, slope, act, rows, cols, dst, partial, st);
  }
  if (dst && partial) return launch_prepare<false, true, true>(src, ld, slope, act, rows, cols, dst, partial, st);
  if (dst) return launch_prepare<false, true, false>(src, ld, slope, act, rows, cols, dst, partial, st);
  return launch_prepare<false, false, true>(src, ld, slope, act, rows, cols, dst, partial, st);
}

hipError_t launch_lin_sum(const float* partial, int parts, int cols, void* out, int out_dtype, hipStream_t st) {
  hipLaunchKernelGGL(lin_sum_kernel, dim3((cols + 15) / 16), dim3(256), 0, st, partial, parts, cols, out, out_dtype, cols, nullptr, 0);
  return hipGetLastError();
}
hipError_t launch_lin_sum(const float* partial, int parts, int cols, void* out, int out_dtype, hipStream_t st, void* out2, int out2_dtype) {
  hipLaunchKernelGGL(lin_sum_kernel, dim3((2 * cols + 15) / 16), dim3(256), 0, st, partial, parts, 2 * cols, out, out_dtype, cols, out2,
                     out2_dtype);
  return hipGetLastError();
}

}  // namespace dion
