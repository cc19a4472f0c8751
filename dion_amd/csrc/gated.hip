// Both projections of a gated feed-forward block, h = act(g) u with g = x Wg^T + bg, u = x Wu^T + bu, and their gradients:
//   forward    one product whose tiles hold the same columns of g and of u, so that h leaves the registers of the sums
//   dg = dh u act'(g),  du = dh act(g)   elementwise, from two values of 24 (32) bits an element that the forward pass keeps
//   dx = dg Wg + du Wu                   one reduction over both (pair form): dx is rounded once and no sum goes through memory
//   dWg = dg^T x,  dWu = du^T x          one product of linear.hip where the results lie behind one another
// Operands bf16, sums fp32.  Tiles, ring and epilogue are lin_tile.h's; like linear.hip's products, large ones are bound by the matrix
// units at the clock the power limit leaves, and by what all CUs store when a round of tiles ends.
// us, medians of kernel traces (from card to card 4 % apart): 8192 x 4096 x 14336 (tokens, fan-in, fan-out) forward 1371 to 1435, 1.34 to 1.40
// PFLOP/s; 8192 x 2048 x 5632 forward with what is kept 369 to 380 (277 MB of it; 1408 tiles of 256 x 256, 5.5 rounds of the CUs), dz
// 110, dx 289 to 295, dW 334 to 345 (704 tiles of 256 x 128, 2.75 rounds); 8192 x 2048 x 8192 507, 175, 437, 441, forward without keeping 431
// (1.28 PFLOP/s).  Two workgroups a CU of 128 x 128 tiles in a ring of two slots, so that one stores while the other multiplies, took 452
// where these took 351, and 571 where 424: their operands come twice as often.
#include "lin_tile.h"

namespace dion {

// What every kernel that finishes elements needs.
struct GatedEpilogue : LinEpilogue {  // (C: h, slope: kept)
  const void* bias2;
  int bias2_dtype, wide;
};

// Finishes and stores elements (row, col .. col + 3) from their two sums, where the activation is not worth a kernel of its own.
static __device__ __forceinline__ void gated4_any(const GatedEpilogue& p, int row, int col, f32x4 g, f32x4 u) {
  if (row >= p.M || col >= p.N) return;
  g += bias4(p, col);
  u += bias4(p.bias2, p.bias2_dtype, p.N, col);
  f32x4 h, s;  // h, act'(g) u; g becomes act(g)
  switch (p.act) {
    case kActRelu: gate4<kActRelu>(g, u, h, s); break;
    case kActReluSquared: gate4<kActReluSquared>(g, u, h, s); break;
    case kActGelu: gate4<kActGelu>(g, u, h, s); break;
    case kActGeluTanh: gate4<kActGeluTanh>(g, u, h, s); break;
    case kActSilu: gate4<kActSilu>(g, u, h, s); break;
    default: gate4<kActNone>(g, u, h, s); break;
  }
  if (p.slope) {
    char* k = (char*)p.slope + (int64_t)row * kept_pitch(p.N, p.wide) + (col >> 5) * kept_block(p.wide);
    const int c = col & 31;
    const Kept4 to_gate = p.wide ? kept4<true>(s) : kept4<false>(s), to_up = p.wide ? kept4<true>(g) : kept4<false>(g);
    *(uint2*)(k + 2 * c) = to_gate.high;
    *(uint2*)(k + 64 + 2 * c) = to_up.high;
    if (p.wide) {
      *(uint2*)(k + 128 + 2 * c) = to_gate.low;
      *(uint2*)(k + 192 + 2 * c) = to_up.low;
    } else {
      *(uint32_t*)(k + 128 + c) = to_gate.low.x;
      *(uint32_t*)(k + 160 + c) = to_up.low.x;
    }
  }
  store4(p, p.C + (int64_t)row * p.N + col, col, make_uint2(pack_bf16x2(h[0], h[1]), pack_bf16x2(h[2], h[3])));
}

// Adds the parts of a split reduction, in their order, and finishes: four elements per thread.  24 x 8192 in eight parts 4 us.
__global__ __launch_bounds__(256) void gated_join_kernel(const GatedEpilogue p, const float* __restrict__ part, int splits) {
  const int per_row = (p.N + 3) / 4;
  const int64_t all = (int64_t)p.M * per_row, one = (int64_t)p.M * p.N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int row = (int)(i / per_row), col = (int)(i - (int64_t)row * per_row) * 4;
    const float* q = part + (int64_t)row * p.N + col;
    f32x4 g = {0.f, 0.f, 0.f, 0.f}, u = g;
    if (p.N % 4 == 0) {
#pragma unroll 4
      for (int k = 0; k < splits; ++k) {
        g += *(const f32x4*)(q + 2 * k * one);
        u += *(const f32x4*)(q + (2 * k + 1) * one);
      }
    } else {
      for (int k = 0; k < splits; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < p.N) {
            g[e] += q[2 * k * one + e];
            u[e] += q[(2 * k + 1) * one + e];
          }
    }
    gated4_any(p, row, col, g, u);
  }
}

// ---------------------------------------------------------------------------------------------- few tokens
// Up to 32 rows of x: a workgroup takes eight rows of each weight, which are the sixteen rows of an MFMA operand, and its wavefronts
// an equal run of the reduction each; fragments go from memory to registers, the next U steps' while the MFMAs of these run.
// The wavefronts' sums meet in LDS and are added in their order; rows 0-7 of a product are g's, 8-15 u's.  Bound by the weights'
// bytes: one token of 4096 x 14336 41.5 us (5.7 TB/s, the weights from HBM); of 768 x 2048 4.9 (launch, one way to memory, LDS).
template <int TB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void gated_few_kernel(const GatedEpilogue p, const bf16_t* __restrict__ x, int64_t ldx,
                                                               const bf16_t* __restrict__ wg, int64_t ldg,
                                                               const bf16_t* __restrict__ wu, int64_t ldu, int K) {
  constexpr int U = 4;
  __shared__ f32x4 sums[WAVES][TB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l16 = lane & 15, quad = lane >> 4;
  const int n0 = blockIdx.x * 8;
  const int wrow = n0 + (l16 & 7) < p.N ? n0 + (l16 & 7) : p.N - 1;
  const bf16_t* wp = (l16 < 8 ? wg + (int64_t)wrow * ldg : wu + (int64_t)wrow * ldu) + quad * 8;
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
  for (int i = threadIdx.x; i < TB * 32; i += WAVES * 64) {
    const int b = i >> 5, l = i & 31;
    f32x4 g = sums[0][b][l], u = sums[0][b][l + 32];
#pragma unroll 5  // (all fifteen at once would not fit the registers)
    for (int k = 1; k < WAVES; ++k) {
      g += sums[k][b][l];
      u += sums[k][b][l + 32];
    }
    gated4_any(p, b * 16 + (l & 15), n0 + 4 * (l >> 4), g, u);
  }
}

// ---------------------------------------------------------------------------------------------- gradients at g and u
constexpr int kDzCols = 256;  // columns of a workgroup: 32 threads of eight, by eight rows

// One pass for both: 12 bytes an element (14 with 32 bits kept), 8192 x 5632 108 us (5.1 TB/s).  Four rows at a time instead of two
// take 17 us more; results stored around the caches, where the products then do not find them, 19 with these.
// W: elements of dh that are read at once; 8: every row is whole chunks.
template <bool WIDE, bool DST, bool SUM, int W>
__global__ __launch_bounds__(256) void gated_dz_kernel(const bf16_t* __restrict__ dh, int64_t ld, const char* __restrict__ kept,
                                                       int rows, int cols, bf16_t* __restrict__ dz, float* __restrict__ partial,
                                                       int per) {
  __shared__ float sums[2][8][kDzCols];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c0 = blockIdx.x * kDzCols + tx * 8, padded = slope_pitch(cols);
  const int64_t pitch = kept_pitch(cols, WIDE);
  const int r_first = blockIdx.y * per, r_end = r_first + per < rows ? r_first + per : rows;
  float acc_g[8] = {}, acc_u[8] = {};
  if (c0 < cols) {
#pragma unroll 2
    for (int r = r_first + ty; r < r_end; r += 8) {
      const bf16_t* q = dh + (int64_t)r * ld + c0;
      float v[8], g[8], u[8];
      if constexpr (W == 8) {
        const u32x4_t w = __builtin_nontemporal_load((const u32x4_t*)q);
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
      const char* k = kept + (int64_t)r * pitch + (c0 >> 5) * kept_block(WIDE);
      auto read = [&](int which, float* to) __attribute__((always_inline)) {
        const u32x4_t high = __builtin_nontemporal_load((const u32x4_t*)(k + which * 64 + (c0 & 31) * 2));
        if constexpr (WIDE) {
          const u32x4_t low = __builtin_nontemporal_load((const u32x4_t*)(k + 128 + which * 64 + (c0 & 31) * 2));
#pragma unroll
          for (int e = 0; e < 8; ++e)
            to[e] = __uint_as_float(__builtin_amdgcn_perm(high[e >> 1], low[e >> 1], e & 1 ? 0x07060302u : 0x05040100u));
        } else {
          const u32x2_t low = __builtin_nontemporal_load((const u32x2_t*)(k + 128 + which * 32 + (c0 & 31)));
#pragma unroll
          for (int e = 0; e < 8; ++e)  // bytes: zero, the low one, the two high ones
            to[e] = __uint_as_float(__builtin_amdgcn_perm(high[e >> 1], low[e >> 2], (e & 1 ? 0x0706000cu : 0x0504000cu) | (e & 3) << 8));
        }
      };
      read(0, g);
      read(1, u);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = W == 8 || c0 + e < cols;
        g[e] = in ? v[e] * g[e] : 0.f;
        u[e] = in ? v[e] * u[e] : 0.f;
      }
      if constexpr (DST) {
        bf16_t* o = dz + (int64_t)r * 2 * padded + c0;
        st_store8<bf16_t>(o, 0, g);
        st_store8<bf16_t>(o + padded, 0, u);
      }
      if constexpr (SUM)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          acc_g[e] += g[e];
          acc_u[e] += u[e];
        }
    }
  }
  if constexpr (SUM) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sums[0][ty][tx * 8 + e] = acc_g[e];
      sums[1][ty][tx * 8 + e] = acc_u[e];
    }
    __syncthreads();
    const int c = blockIdx.x * kDzCols + threadIdx.x;
    if (c < cols) {
      float g = 0.f, u = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        g += sums[0][k][threadIdx.x];
        u += sums[1][k][threadIdx.x];
      }
      partial[(int64_t)blockIdx.y * 2 * cols + c] = g;
      partial[((int64_t)blockIdx.y * 2 + 1) * cols + c] = u;
    }
  }
}

// ---------------------------------------------------------------------------------------------- host
size_t gated_kept_bytes(int M, int N, bool wide) { return (size_t)M * kept_pitch(N, wide); }

// Up to 32 tokens: gated_few_kernel where it is estimated to take less than tiles, which pass the weights at 5.4 TB/s and then join the
// parts of their reductions (8 us).  us, few / tiles, weights from HBM: 4096 x 14336, 1 token 44 / 52, 4 tokens 47 / 52, 16 tokens
// 68 / 53; 2048 x 8192, 8 tokens 15.6 / 18.1, 24 tokens 39.6 / 19.4.
static LinPlan gated_plan(int M, int N, int K) {
  if (M <= 32) {
    const double wgs = (N + 7) / 8, each = M <= 16 ? 0.74 + 0.03 * (M - 1) : 2.3;
    const double few = 2.5 + each * (K / 512.0) * (wgs > 256 ? wgs / 256 : 1), tiles = 8.0 + 4.0 * N * K / 5.4e6;
    if (few < tiles) return {kLinFew, 1, 0};
  }
  return lin_plan(M, 2 * N, K, 0, 0, false);
}

size_t gated_product_scratch(int M, int N, int K) {
  const LinPlan plan = gated_plan(M, N, K);
  return plan.splits > 1 ? (size_t)plan.splits * M * N * 2 * sizeof(float) : 0;
}

template <class Cfg, int ACT>
static hipError_t launch_act(const LinTwoParams& tp, bool wide, hipStream_t st) {
  if (tp.e.slope && wide) return launch_tile<Cfg, false, false, ACT, true, false, kLinGatedWide>(tp, st);
  return tp.e.slope ? launch_tile<Cfg, false, false, ACT, true, false, kLinGated>(tp, st)
                    : launch_tile<Cfg, false, false, ACT, false, false, kLinGated>(tp, st);
}

template <class Cfg>
static hipError_t launch_tiles(const GatedProduct& p, LinTwoParams tp, hipStream_t st) {
  if (!lin_tile_list<Cfg>(p.M, ((int64_t)p.N * 2 + Cfg::BN - 1) / Cfg::BN * Cfg::BN, tp)) return hipErrorInvalidValue;
  // As in linear.hip, with half its bound on a weight: there are two.  us, a run for each XCD / interleaved, with 24 bits kept: 16384 x 8192 x
  // 4096 1699 / 1579, 65536 x 2048 x 8192 3871 / 3708, but 32768 x 4096 x 8192 3420 / 3469; larger weights 16384 x 4096 x 14336 2951 / 3054
  // (16384 x 8192 x 8192 3399 / 3251 the other way), a smaller x 32768 x 2048 x 16384 3773 / 3983, 16384 x 4096 x 4096 837 / 834.
  tp.interleave = Cfg::BM == 256 && Cfg::BN == 256 && (int64_t)p.M * p.K >= (int64_t(128) << 20) &&
                  (int64_t)p.N * p.K <= (int64_t(48) << 20);
  if (tp.splits > 1) return launch_tile<Cfg, false, false, kActNone, false, true, kLinGated>(tp, st);
  switch (tp.e.act) {
    case kActNone: return launch_act<Cfg, kActNone>(tp, p.wide, st);
    case kActRelu: return launch_act<Cfg, kActRelu>(tp, p.wide, st);
    case kActReluSquared: return launch_act<Cfg, kActReluSquared>(tp, p.wide, st);
    case kActGelu: return launch_act<Cfg, kActGelu>(tp, p.wide, st);
    case kActGeluTanh: return launch_act<Cfg, kActGeluTanh>(tp, p.wide, st);
    case kActSilu: return launch_act<Cfg, kActSilu>(tp, p.wide, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_gated_product(const GatedProduct& p, hipStream_t st) {
  if (p.M <= 0 || p.N <= 0 || p.K <= 0) return hipErrorInvalidValue;
  if (!lin_chunks(p.X, p.ldx, p.K) || !lin_chunks(p.Wg, p.ldg, p.K) || !lin_chunks(p.Wu, p.ldu, p.K)) return hipErrorInvalidValue;
  GatedEpilogue e = {};
  e.C = p.H;
  e.bias = p.bg;
  e.slope = (uint16_t*)p.kept;
  e.M = p.M;
  e.N = p.N;
  e.act = p.act;
  e.bias_dtype = p.bg_dtype;
  e.vec = lin_vec(p.H, nullptr, p.N, 0);
  e.bias2 = p.bu;
  e.bias2_dtype = p.bu_dtype;
  e.wide = p.wide;
  const LinPlan plan = gated_plan(p.M, p.N, p.K);
  if (plan.tile == kLinFew) {
    const dim3 grid((unsigned)((p.N + 7) / 8));
    auto go = [&](auto tbc, auto wavesc) {
      constexpr int TB = decltype(tbc)::value, WAVES = decltype(wavesc)::value;
      hipLaunchKernelGGL((gated_few_kernel<TB, WAVES>), grid, dim3(WAVES * 64), 0, st, e, p.X, p.ldx, p.Wg, p.ldg, p.Wu, p.ldu, p.K);
    };
    typedef std::integral_constant<int, 16> many;
    if (p.M > 16) go(std::integral_constant<int, 2>(), many());
    else if (p.N >= 4096) go(std::integral_constant<int, 1>(), std::integral_constant<int, 4>());
    else go(std::integral_constant<int, 1>(), many());
    return hipGetLastError();
  }
  LinTwoParams tp = {};
  tp.e = e;
  tp.P = p.X;
  tp.Q = p.Wg;
  tp.Q2 = p.Wu;
  tp.ldp = (int)p.ldx;
  tp.ldq = (int)p.ldg;
  tp.ldq2 = (int)p.ldu;
  tp.K = p.K;
  tp.part = p.scratch;
  tp.splits = plan.splits;
  tp.slabs = plan.slabs;
  tp.bias2 = p.bu;
  tp.bias2_dtype = p.bu_dtype;
  if (plan.splits > 1 && !p.scratch) return hipErrorInvalidValue;
  if (hipError_t err = plan.tile == kLin256 ? launch_tiles<Lin256>(p, tp, st)
                       : plan.tile == kLinWide ? launch_tiles<LinWide>(p, tp, st) : launch_tiles<Lin128>(p, tp, st))
    return err;
  if (plan.splits > 1) {
    const int64_t wg = ((int64_t)p.M * ((p.N + 3) / 4) + 255) / 256;
    const dim3 grid((unsigned)(wg < 65536 ? wg : 65536));
    hipLaunchKernelGGL(gated_join_kernel, grid, dim3(256), 0, st, e, p.scratch, plan.splits);
  }
  return hipGetLastError();
}

hipError_t launch_gated_dz(const bf16_t* dh, int64_t ld, const void* kept, bool wide, int rows, int cols, bf16_t* dz, float* sums,
                           hipStream_t st) {
  if (rows <= 0 || cols <= 0 || !kept || (!dz && !sums) || ((uint64_t)dz & 15) || ((uint64_t)kept & 15))
    return hipErrorInvalidValue;
  const int parts = lin_sum_parts(rows), per = (rows + 1023) / 1024 * 8;
  const dim3 grid((cols + kDzCols - 1) / kDzCols, parts);
  const uint64_t bytes = (uint64_t)dh | (uint64_t)cols * 2 | (uint64_t)ld * 2;
  auto go = [&](auto widec, auto dstc, auto sumc, auto wc) {
    hipLaunchKernelGGL((gated_dz_kernel<decltype(widec)::value, decltype(dstc)::value, decltype(sumc)::value, decltype(wc)::value>), grid, dim3(256), 0, st, dh,
                       ld, (const char*)kept, rows, cols, dz, sums, per);
  };
  auto sized = [&](auto widec, auto dstc, auto sumc) {
    if (bytes % 16 == 0) go(widec, dstc, sumc, std::integral_constant<int, 8>());
    else if (bytes % 4 == 0) go(widec, dstc, sumc, std::integral_constant<int, 2>());
    else go(widec, dstc, sumc, std::integral_constant<int, 1>());
  };
  auto with = [&](auto dstc, auto sumc) {
    if (wide) sized(std::true_type(), dstc, sumc);
    else sized(std::false_type(), dstc, sumc);
  };
  if (dz && sums) with(std::true_type(), std::true_type());
  else if (dz) with(std::true_type(), std::false_type());
  else with(std::false_type(), std::true_type());
  return hipGetLastError();
}

// ---- dg Wg + du Wu
static LinPlan pair_plan(int M, int N, int K) { return lin_plan(M, N, (K + 63) / 64 * 128, 0, 1); }

size_t pair_product_scratch(int M, int N, int K) {
  const LinPlan plan = pair_plan(M, N, K);
  return plan.splits > 1 ? (size_t)plan.splits * M * N * sizeof(float) : 0;
}

template <class Cfg>
static hipError_t launch_pair_tiles(const PairProduct& p, LinTwoParams tp, hipStream_t st) {
  if (!lin_tile_list<Cfg>(p.M, p.N, tp)) return hipErrorInvalidValue;
  // Two of each operand: half of linear.hip's bounds.  us with dz, a run for each XCD / interleaved: 16384 x 4096 x 4096 (tokens, fan-in,
  // fan-out) 956 / 929, 32768 x 4096 x 8192 3946 / 3833, 65536 x 4096 x 8192 7993 / 7751, but 65536 x 1024 x 8192 3068 / 3140; smaller dg
  // and du 8192 x 2048 x 5632 370 / 367, larger weights 8192 x 4096 x 14336 1643 / 1644 (16384 x 4096 x 14336 3397 / 3304).
  tp.interleave = Cfg::BM == 256 && Cfg::BN == 256 && (int64_t)p.M * p.K >= (int64_t(64) << 20) &&
                  (int64_t)p.N * p.K <= (int64_t(48) << 20);
  return tp.splits > 1 ? launch_tile<Cfg, false, true, kActNone, false, true, kLinPair>(tp, st)
                       : launch_tile<Cfg, false, true, kActNone, false, false, kLinPair>(tp, st);
}

hipError_t launch_pair_product(const PairProduct& p, hipStream_t st) {
  if (p.M <= 0 || p.N <= 0 || p.K <= 0) return hipErrorInvalidValue;
  if (!lin_chunks(p.P, p.ldp, p.K) || !lin_chunks(p.P2, p.ldp, p.K) || !lin_chunks(p.Q, p.ldq, p.N) || !lin_chunks(p.Q2, p.ldq2, p.N))
    return hipErrorInvalidValue;
  const LinPlan plan = pair_plan(p.M, p.N, p.K);
  LinTwoParams tp = {};
  tp.e.C = p.C;
  tp.e.M = p.M;
  tp.e.N = p.N;
  tp.e.vec = lin_vec(p.C, nullptr, p.N, 0);
  tp.P = p.P;
  tp.P2 = p.P2;
  tp.Q = p.Q;
  tp.Q2 = p.Q2;
  tp.ldp = (int)p.ldp;
  tp.ldq = (int)p.ldq;
  tp.ldq2 = (int)p.ldq2;
  tp.K = p.K;
  tp.part = p.scratch;
  tp.splits = plan.splits;
  tp.slabs = plan.slabs;
  if (plan.splits > 1 && !p.scratch) return hipErrorInvalidValue;
  if (hipError_t err = plan.tile == kLin256 ? launch_pair_tiles<Lin256>(p, tp, st)
                       : plan.tile == kLinWide ? launch_pair_tiles<LinWide>(p, tp, st) : launch_pair_tiles<Lin128>(p, tp, st))
    return err;
  return plan.splits > 1 ? launch_lin_join(p.scratch, plan.splits, p.M, p.N, p.C, st) : hipGetLastError();
}

}  // namespace dion
