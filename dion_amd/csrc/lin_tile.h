// What the products of weights share: activations, the tile kernel in its forms, and its launch (linear.hip: y = act(x W^T + b) +
// residual and its gradients; gated.hip: act(x Wg^T + bg) * (x Wu^T + bu) and its own).
#pragma once
#include <atomic>

#include "gemm_tile.h"
#include "linear.h"

namespace dion {

// ---------------------------------------------------------------------------------------------- activations
static __device__ __forceinline__ float rcp_fast(float v) { return __builtin_amdgcn_rcpf(v); }

// act(z), and act'(z) in `slope`, for slope_pack2.  Exponentials and quotients by the hardware's approximations (1 ulp): the
// result is rounded to bf16, the slope to eleven bits.
template <int ACT>
static __device__ __forceinline__ float activate(float z, float& slope) {
  if constexpr (ACT == kActRelu) {
    slope = z <= 0.f ? 0.f : 1.f;  // (where z is NaN the gradient goes on, and the value stays NaN)
    return z < 0.f ? 0.f : z;
  } else if constexpr (ACT == kActReluSquared) {
    const float r = z <= 0.f ? 0.f : z;  // (never -0, which has no code; NaN stays)
    slope = r;  // (half of it: slope_pack2 doubles)
    return r * r;
  } else if constexpr (ACT == kActSilu) {
    const float s = rcp_fast(1.f + __expf(-z));
    slope = s * (1.f + z * (1.f - s));
    return z * s;
  } else if constexpr (ACT == kActGelu) {
    // The normal distribution's upper tail at a = |z| is exp(-a^2 / 2) t P(t), t = 1 / (1 + 0.3 a), P fitted to it with a
    // relative error of 1.7e-7 up to a = 14, where fp32 ends: one exponential for the tail and the density.  In fp32 the rounding of
    // a^2 / 2 adds to that: 7e-7 up to a = 4, 2.4e-6 up to 10, 4.3e-6 up to 13; behind it the tail is below fp32's normal numbers.
    const float a = fabsf(z), t = rcp_fast(1.f + 0.3f * a), e = __expf(-0.5f * z * z);
    float q = 0.03567495f;
    q = fmaf(q, t, -0.15720376f);
    q = fmaf(q, t, 0.20635456f);
    q = fmaf(q, t, -0.053684533f);
    q = fmaf(q, t, 0.12856206f);
    q = fmaf(q, t, 0.09991337f);
    q = fmaf(q, t, 0.12075397f);
    q = fmaf(q, t, 0.1196293f);
    const float tail = q * t * e;
    const float cdf = z > 0.f ? 1.f - tail : tail;
    slope = cdf + z * 0.39894228f * e;
    return z * cdf;
  } else if constexpr (ACT == kActGeluTanh) {
    // (past |z| = 100, where s is 0 or 1, the square stands still: none that leaves fp32 meets 1 - s = 0)
    const float zz = fminf(z * z, 1e4f);
    const float u = 0.79788456f * z * (1.f + 0.044715f * zz);
    const float s = rcp_fast(1.f + __expf(-2.f * u));  // (1 + tanh u) / 2
    slope = s + z * s * (1.f - s) * 1.5957691f * (1.f + 0.134145f * zz);
    return z * s;
  } else {
    slope = 1.f;
    return z;
  }
}

// Two slopes as the forward pass keeps them.
template <int ACT>
static __device__ __forceinline__ uint32_t slope_pack2(float a, float b) {
  if constexpr (ACT != kActReluSquared) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
  } else {
    // Doubled and rounded to nine bits of mantissa; code 0 is zero (and 2^-63 and below), 0xffff NaN and everything past 2^65.
    auto code = [](float half) {  // in the upper bits
      const uint32_t twice = __builtin_elementwise_add_sat(__float_as_uint(half), 0x802000u);  // (a NaN may have a sign)
      return min(__builtin_elementwise_sub_sat(twice, 64u << 23), 0x3fffffffu);
    };
    return code(a) >> 14 | (code(b) << 2 & 0xffff0000u);
  }
}
static __device__ __forceinline__ float slope_unpack(int act, uint16_t c) {
  if (act != kActReluSquared) return (float)__builtin_bit_cast(_Float16, c);
  if (c == 0) return 0.f;
  return c == 0xffffu ? __uint_as_float(0x7fc00000u) : __uint_as_float(((uint32_t)c << 14) + (64u << 23));
}

// What every kernel that finishes elements needs.
struct LinEpilogue {
  bf16_t* C;
  const void* bias;
  const bf16_t* R;
  uint16_t* slope;
  int64_t ldr;
  int M, N, act, bias_dtype;
  int vec;  // 8, 4, 2, 1: neighbours of a row that N, ldr and the addresses allow to be moved at once
};

// Bias of columns col .. col + 3.
static __device__ __forceinline__ f32x4 bias4(const void* bias, int dtype, int N, int col) {
  f32x4 b = {0.f, 0.f, 0.f, 0.f};
  if (bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < N) b[e] = dtype ? ((const float*)bias)[col + e] : bf16_to_f32(((const bf16_t*)bias)[col + e]);
  }
  return b;
}
static __device__ __forceinline__ f32x4 bias4(const LinEpilogue& p, int col) { return bias4(p.bias, p.bias_dtype, p.N, col); }
// The addend of elements (row, col .. col + 3), as four bf16.
static __device__ __forceinline__ uint2 residual4(const LinEpilogue& p, int row, int col) {
  uint2 w = make_uint2(0, 0);
  if (!p.R || row >= p.M || col >= p.N) return w;
  const bf16_t* r = p.R + (int64_t)row * p.ldr + col;
  if (p.vec >= 4) return *(const uint2*)r;
  if (p.vec == 2) {
    w.x = *(const uint32_t*)r;
    if (col + 2 < p.N) w.y = *(const uint32_t*)(r + 2);
    return w;
  }
  w.x = r[0];
  if (col + 1 < p.N) w.x |= (uint32_t)r[1] << 16;
  if (col + 2 < p.N) w.y = r[2];
  if (col + 3 < p.N) w.y |= (uint32_t)r[3] << 16;
  return w;
}
// Stores four 16-bit elements of a row, as far as it goes.
static __device__ __forceinline__ void store4(const LinEpilogue& p, uint16_t* o, int col, uint2 w) {
  if (p.vec >= 4) {
    *(uint2*)o = w;
  } else if (p.vec == 2) {
    *(uint32_t*)o = w.x;
    if (col + 2 < p.N) *(uint32_t*)(o + 2) = w.y;
  } else {
    o[0] = (uint16_t)w.x;
    if (col + 1 < p.N) o[1] = (uint16_t)(w.x >> 16);
    if (col + 2 < p.N) o[2] = (uint16_t)w.y;
    if (col + 3 < p.N) o[3] = (uint16_t)(w.y >> 16);
  }
}
// Slopes lie in whole 16-byte chunks, whatever N is.
static __host__ __device__ __forceinline__ int slope_pitch(int n) { return (n + 7) & ~7; }

// Four sums of a row as they are stored, y and the slopes.
template <int ACT, bool SLOPE>
static __device__ __forceinline__ void finish4(const LinEpilogue& p, f32x4 z, f32x4 b, uint2 r, uint2& y, uint2& slopes) {
  float v[4], s[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = activate<ACT>(z[e] + b[e], s[e]);
  if constexpr (SLOPE) slopes = make_uint2(slope_pack2<ACT>(s[0], s[1]), slope_pack2<ACT>(s[2], s[3]));
  if (p.R) {
    v[0] += __uint_as_float(r.x << 16);
    v[1] += __uint_as_float(r.x & 0xffff0000u);
    v[2] += __uint_as_float(r.y << 16);
    v[3] += __uint_as_float(r.y & 0xffff0000u);
  }
  y = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// ---------------------------------------------------------------------------------------------- gated products
// What the backward pass of h = act(g) u needs of an element: act'(g) u and act(g), rounded to the upper 24 bits of fp32.  In bf16
// their rounding would be as large as that of the gradients at g and u themselves (dx and dW off by 0.0029 of their norm instead of
// 0.0024), and fp16 ends at 65504.  `wide`: all 32 bits, for sums that are stored as fp32 (24 bits: off by 4e-6, 32: 3e-7).  Of 32
// columns of a row lie in 192 (256) bytes: the upper 16 bits of the one, of the other, then the lower 8 (16) of the one, of the other.
static __host__ __device__ __forceinline__ constexpr int kept_block(bool wide) { return wide ? 256 : 192; }
static __host__ __device__ __forceinline__ int64_t kept_pitch(int n, bool wide) { return (int64_t)((n + 31) / 32) * kept_block(wide); }

struct Kept4 {  // of four neighbours
  uint2 high, low;  // (low.x alone: eight bits each)
};
template <bool WIDE>
static __device__ __forceinline__ Kept4 kept4(f32x4 v) {
  uint32_t b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    b[e] = __float_as_uint(v[e]);
    if constexpr (!WIDE)  // (a NaN stays one: saturated apart from its sign)
      b[e] = (uint32_t)__builtin_elementwise_add_sat((int)(b[e] & 0x7fffffffu), 0x80) | (b[e] & 0x80000000u);
  }
  const uint2 high = make_uint2(__builtin_amdgcn_perm(b[1], b[0], 0x07060302), __builtin_amdgcn_perm(b[3], b[2], 0x07060302));
  if constexpr (WIDE)
    return {high, make_uint2(__builtin_amdgcn_perm(b[1], b[0], 0x05040100), __builtin_amdgcn_perm(b[3], b[2], 0x05040100))};
  else
    return {high, make_uint2(__builtin_amdgcn_perm(b[1], b[0], 0x0c0c0501) | __builtin_amdgcn_perm(b[3], b[2], 0x05010c0c), 0)};
}

// Four elements of a row from their sums: h = act(g) u, s = act'(g) u, and act(g) in g.
template <int ACT>
static __device__ __forceinline__ void gate4(f32x4& g, f32x4 u, f32x4& h, f32x4& s) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float slope;
    const float a = activate<ACT>(g[e], slope);
    h[e] = a * u[e];
    s[e] = (ACT == kActReluSquared ? 2.f * slope : slope) * u[e];
    g[e] = a;
  }
}
// ... as they are stored: h, and (KEEP) what is kept for the backward pass (not from h: act(g) may be zero).
template <int ACT, bool KEEP, bool WIDE>
static __device__ __forceinline__ void gated4(f32x4 g, f32x4 u, uint2& h, Kept4& to_gate, Kept4& to_up) {
  f32x4 v, s;
  gate4<ACT>(g, u, v, s);
  h = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  if constexpr (KEEP) {
    to_gate = kept4<WIDE>(s);
    to_up = kept4<WIDE>(g);
  }
}

// ---------------------------------------------------------------------------------------------- tiles
template <int BM_, int BN_, int WM_, int WN_, int NS_>
struct LinCfg {
  static constexpr int BM = BM_, BN = BN_, BK = 64, WM = WM_, WN = WN_, NS = NS_;
  static constexpr int NT = WM * WN * 64;
  static constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
  static constexpr int HALVES = TM / 4, ST = BK / 32;
  static constexpr int PB = BM * BK * 2, QB = BN * BK * 2;  // bytes of an operand's slab
  static constexpr int RING_BYTES = NS * (PB + QB);
  static constexpr int STG_BYTES = 16 * 128;  // a wavefront's staging: 16 rows of 64 16-bit elements
  static constexpr int LDS_BYTES = RING_BYTES + WM * WN * STG_BYTES;
  static constexpr int PL = PB / (NT * 16), QL = QB / (NT * 16), LPS = PL + QL;  // loads of a thread per slab
  static_assert(TN == 4 && (TM == 4 || TM == 8) && LPS <= 8 && LDS_BYTES <= 160 * 1024, "wavefronts of 64 or 128 rows by 64 columns");
};
typedef LinCfg<256, 256, 2, 4, 2> Lin256;   // 8 wavefronts of 128 x 64
typedef LinCfg<256, 128, 4, 2, 3> LinWide;  // 8 wavefronts of 64 x 64
typedef LinCfg<128, 128, 2, 2, 4> Lin128;   // 4 wavefronts of 64 x 64

// Issue order of the fragment reads behind the MFMAs, and how many LDS instructions may be outstanding when an MFMA issues (the
// LDS returns in order).  A 32-deep step is HALVES halves of sixteen MFMAs (A fragment q / 4 against B fragment q % 4); while a half
// runs, the next one's fragments are requested: A0 B0..B3 A1..A3 behind MFMAs 0..7 where it starts a step, A4..A7 behind every
// fourth where it does not.  A fragment that lies along the reduction is one read, one across it two transposing ones (AI, BI).
template <int HALVES, int ST, int AI, int BI>
struct LinSched {
  static constexpr bool full(int hp) { return (hp + 1) % HALVES == 0; }
  static constexpr int read_behind(int hp, int q) { return full(hp) ? (q < 8 ? q : -1) : (q % 4 == 1 ? q / 4 : -1); }
  static constexpr int behind(int hp, int q) {
    const int r = read_behind(hp, q);
    return r < 0 ? 0 : full(hp) ? (r >= 1 && r <= 4 ? BI : AI) : AI;
  }
  static constexpr int allowed(int hp, int q) {
    const int i = q / 4, j = q % 4, prev = (hp + HALVES * ST - 1) % (HALVES * ST);
    int need = 4 * i + 1;
    if (hp % HALVES == 0) {
      const int ra = i == 0 ? 0 : 4 + i, rb = 1 + j;
      need = ra > rb ? ra : rb;
    }
    int n = 0;
    for (int k = need + 1; k < 16; ++k) n += behind(prev, k);
    for (int k = 0; k < q; ++k) n += behind(hp, k);
    return n < 15 ? n : 15;  // (the counter has four bits)
  }
};

struct LinTileParams {
  LinEpilogue e;
  const bf16_t *P, *Q;
  int ldp, ldq, K;
  float* part;  // [splits][M][N] sums, where the reduction is split
  int tilesM, tilesN, splits, slabs;  // slabs: of 64, per split
  int total, grid;                    // tiles of the list, workgroups
  int interleave;
  uint32_t inv_tiles, inv_group, inv_tail;
};

// Forms of the tile kernel.
//   plain  C = P Q^T.
//   gated  e.C = act(P Q^T + e.bias) * (P Q2^T + bias2), both [M][e.N], in one tile: sixteen rows of Q, sixteen of Q2 and so on take
//          turns along the tile's columns, so that a lane holds both sums of an element.  Every wavefront loads rows of one of
//          the two.  e.slope: what gated4 keeps, of 24 bits or (gated_wide) 32.  Split: parts [splits][2][M][e.N].
//   pair   C = P Q + P2 Q2 (K-major Q, Q2; rows of P and P2 equally far apart), one reduction of twice the slabs of K: the ring
//          runs on from the first pair's last slab, whose chunks behind K arrive as zeros, into the second pair's.
enum LinForm { kLinPlain, kLinGated, kLinGatedWide, kLinPair };
struct LinTwoParams : LinTileParams {
  const bf16_t *P2, *Q2;
  int ldq2;
  const void* bias2;  // gated
  int bias2_dtype;
};

// One workgroup per CU walks a list of output tiles (of parts of the reduction).  Operand slabs reach a ring of NS slots in LDS
// by direct-to-LDS buffer loads, whose descriptors end where the matrix does: rows past an edge arrive as zeros, and need no
// padded copy.  Chunks behind the reduction's end in the last slab of an operand with the reduction along rows get an offset past
// the end.  The ring runs on across tiles: the last slabs of one are computed while the first ones of the next arrive.
// XOR swizzles keep the LDS writes and the fragment reads free of bank conflicts.  The MFMA operands are swapped (B
// fragment first), so that a lane's four sums are neighbours of one row of C: 8-byte accesses to C, the addend and the slopes.
// SPLIT: the sums of a part go to p.part as fp32, and lin_join_kernel finishes them.
// What the steps to this form measured, us, 8192 x 2048 x 8192 with the squared relu and its slopes: a workgroup per tile, sums
// through LDS to the activation 329; activation in the registers of the sums 293; one workgroup per CU that walks its tiles,
// results through LDS in lines 255. Tiles of 256 x 128 whose fragments are a slab ahead: 4096 x 2048 x 2048 37 to 32, dW of it
// 48 to 34. Four wavefronts of 128 x 128 instead of eight gain nothing in the loop (1.34 to 1.41 us a slab against 1.37) and
// lose in the epilogue; neither staggered starts of the workgroups nor non-temporal stores make the rounds' ends cheaper.
template <class Cfg, bool PK, bool QK, int ACT, bool SLOPE, bool SPLIT, int FORM = kLinPlain>
__global__ __launch_bounds__(Cfg::NT, 2) void lin_tile_kernel(const std::conditional_t<FORM == kLinPlain, LinTileParams, LinTwoParams> p) {
  constexpr bool WIDE = FORM == kLinGatedWide, GATED = FORM == kLinGated || WIDE, PAIR = FORM == kLinPair;
  static_assert(!GATED || (!PK && !QK), "gated: the reduction along the rows of all operands");
  static_assert(!PAIR || (!PK && QK), "pair: the reduction along the rows of P, across those of Q");
  constexpr int BM = Cfg::BM, BN = Cfg::BN, BK = Cfg::BK, TM = Cfg::TM, TN = Cfg::TN, ST = Cfg::ST, HALVES = Cfg::HALVES;
  constexpr int HP = HALVES * ST, PB = Cfg::PB, QB = Cfg::QB, NT = Cfg::NT, NS = Cfg::NS, PL = Cfg::PL, QL = Cfg::QL, LPS = Cfg::LPS;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;

  // ---- tile `pid` of the list, eight rows of tiles at a time, columns first within them.  Every XCD has one contiguous run of it,
  // or (p.interleave) 32 consecutive tiles of every 256, those behind the last whole 256 in runs again.
  struct Tile {
    int part, ti, tj, KT;  // KT: slabs of its reduction
  };
  auto tile = [&](int pid) __attribute__((always_inline)) {
    Tile t;
    const int base = p.interleave ? p.total & ~255 : 0, xcd = pid & 7, q = (p.total - base) >> 3, r = p.total & 7;
    const int lt = pid < base ? (pid & ~255) + xcd * 32 + ((pid & 255) >> 3) : base + xcd * q + (xcd < r ? xcd : r) + ((pid - base) >> 3);
    int in_part, tg;
    t.part = div_known(lt, p.tilesM * p.tilesN, p.inv_tiles, in_part);
    const int first = div_known(in_part, 8 * p.tilesN, p.inv_group, tg) * 8;
    if (p.tilesM - first >= 8) {
      t.ti = first + (tg & 7);
      t.tj = tg >> 3;
    } else {
      int row;
      t.tj = div_known(tg, p.tilesM - first, p.inv_tail, row);
      t.ti = first + row;
    }
    t.part = __builtin_amdgcn_readfirstlane(t.part);
    t.ti = __builtin_amdgcn_readfirstlane(t.ti);
    t.tj = __builtin_amdgcn_readfirstlane(t.tj);
    t.KT = min((PAIR ? 2 : 1) * ((p.K + BK - 1) / BK) - t.part * p.slabs, p.slabs);
    return t;
  };

  // ---- global -> LDS: an operand's slab is a tile of BM (BN) rows of 64, or (K-major) of 64 rows of BM (BN); 16-byte chunk
  // j * NT + tid of it, in LDS order, is load j's.  Rows along the reduction are 128 bytes: chunk c of row r lies at
  // c ^ (r / 2) % 8.  K-major rows: 64-byte group g of row r at g ^ r % 4, its 32-byte halves swapped where r / 8 is odd.
  // A descriptor ends where the operand's rows do: past the last row of the tile with the reduction along the rows (wherever along
  // it the slab is: that is the scalar offset), past the last index of the reduction K-major.  Chunks that start behind the end of a
  // row -- the reduction's or, K-major, the matrix's -- get an offset past every descriptor's end.
  constexpr int P_ROWS = PK ? NT / (BM / 8) : NT / 8, Q_ROWS = QK ? NT / (BN / 8) : NT / 8;  // between two loads of a slab
  static_assert(P_ROWS % 16 == 0 && Q_ROWS % 16 == 0, "the swizzles repeat every 16 rows");
  constexpr uint32_t kEnd = 0xb0000000u;  // past every descriptor's end, with room for the rows between the loads
  static_assert(kEnd + 256ull * kLinMaxLd * 2 < (1ull << 32) && 256ull * kLinMaxLd * 2 < kEnd, "offsets within a tile");
  // The thread's number where what follows from it is not to be kept in registers over the loops.
  auto again = [&]() __attribute__((always_inline)) {
    int v = tid;
    asm volatile("" : "+v"(v));
    return v;
  };
  auto offset = [&](int tid, bool kmajor, int width, int ld, int in, bool turns = false) __attribute__((always_inline)) {  // in: elements of a row from the tile's start
    const int cpr = kmajor ? width / 8 : 8, row = tid / cpr, c = tid % cpr;
    const int chunk = kmajor ? (((c >> 2) ^ (row & 3)) << 2) | ((c & 3) ^ (((row >> 3) & 1) << 1)) : c ^ ((row >> 1) & 7);
    const int from = turns ? ((row >> 5) << 4) | (row & 15) : row;  // (turns: of the operand whose sixteen rows these are)
    return chunk * 8 < in ? (uint32_t)(from * ld + chunk * 8) * 2u : kEnd;
  };
  // gated: rows 8 w .. 8 w + 7 of every load are wavefront w's, of Q2 where w / 2 is odd
  const bool second = GATED && ((wave >> 1) & 1);
  int ldq = p.ldq;
  if constexpr (GATED) ldq = second ? p.ldq2 : p.ldq;
  constexpr int Q_FROM = GATED ? Q_ROWS / 2 : Q_ROWS;  // rows of Q between two loads
  // 64-row wavefront tiles have a register for every load's offset; 128-row ones one per operand, the rest is added.
  constexpr int VP = TM == 4 ? PL : 1, VQ = TM == 4 ? QL : 1;
  uint32_t voffP[VP], voffQ[VQ];
  auto set_offsets = [&](int inP, int inQ) __attribute__((always_inline)) {
    const int t = again();
    const uint32_t vp = offset(t, PK, BM, p.ldp, inP), vq = offset(t, QK, BN, ldq, inQ, GATED);
#pragma unroll
    for (int j = 0; j < VP; ++j) voffP[j] = vp + (uint32_t)j * (uint32_t)(P_ROWS * p.ldp * 2);
#pragma unroll
    for (int j = 0; j < VQ; ++j) voffQ[j] = vq + (uint32_t)j * (uint32_t)(Q_FROM * ldq * 2);
  };
  // what is loaded next: slab nxt of a tile of KT_in, into slot slot_in
  const char *baseP = (const char*)p.P, *baseQ = (const char*)p.Q;
  const int64_t stepP = PK ? (int64_t)BK * p.ldp * 2 : 0;
  int64_t stepQ = QK ? (int64_t)BK * p.ldq * 2 : 0;
  int pid_in = blockIdx.x, k_in = 0, nxt = 0, KT_in = 0, slot_in = 0, soff = 0, endP = 0, endQ = 0, inP = 0, inQ = 0;
  int recsP = 0, recsQ = 0;
  int at_P = 0, at_Q = 0, behind_in = 0, odd_in = 0;  // pair: the tile, its slabs of the second pair, whether it has an odd number
  // What changes with the last slab of a tile and behind it.  (Slabs behind an odd number of them, and behind the last tile, are
  // loaded as zeros: the loop is two slabs long, and its waits count on every load.)
  auto turn = [&]() __attribute__((always_inline)) {
    auto starts = [&]() __attribute__((always_inline)) {
      if constexpr (PAIR) return behind_in > 0 ? nxt >= KT_in : nxt >= KT_in + odd_in && pid_in < p.total;
      else return nxt >= ((KT_in + 1) & ~1) && pid_in < p.total;
    };
    if (starts()) {
      const bf16_t *fromP = p.P, *fromQ = p.Q;
      if constexpr (PAIR) {
        // a tile's slabs of the first pair, then those of the second: a run each
        const int KS = (p.K + BK - 1) / BK;
        ldq = p.ldq;
        if (behind_in > 0) {
          KT_in = behind_in;
          behind_in = 0;
          k_in = 0;
          fromP = p.P2, fromQ = p.Q2, ldq = p.ldq2;
        } else {
          const Tile t = tile(pid_in);
          pid_in += p.grid;
          at_P = t.ti * BM;
          at_Q = t.tj * BN;
          odd_in = t.KT & 1;
          const int first = t.part * p.slabs;
          KT_in = t.KT;
          k_in = first * BK;
          if (first >= KS) {
            k_in -= KS * BK;
            fromP = p.P2, fromQ = p.Q2, ldq = p.ldq2;
          } else if (first + t.KT > KS) {
            KT_in = KS - first;
            behind_in = t.KT - KT_in;
          }
        }
        stepQ = (int64_t)BK * ldq * 2;
      } else {
        const Tile t = tile(pid_in);
        pid_in += p.grid;
        KT_in = t.KT;
        k_in = t.part * p.slabs * BK;
        at_P = t.ti * BM;
        at_Q = t.tj * (GATED ? BN / 2 : BN);
      }
      if constexpr (GATED) fromQ = second ? p.Q2 : p.Q;
      nxt = 0;
      soff = 0;
      auto begin = [&](const bf16_t* base, bool kmajor, int extent, int at, int ld, const char*& from, int& end, int& recs,
                       int& in) __attribute__((always_inline)) {
        from = (const char*)(base + (kmajor ? (int64_t)k_in * ld + at : (int64_t)at * ld + k_in));
        // (K-major: rows from the tile's last slab on; all of a slab's rows are there before it)
        const int64_t n = (int64_t)(kmajor ? p.K - k_in - (KT_in - 1) * BK : extent - at) * ld * 2;
        end = (int)(uint32_t)(n < (int64_t)kEnd ? n : (int64_t)kEnd);
        recs = kmajor ? (int)kEnd : end;
        in = kmajor ? ((extent + 7) & ~7) - at : BK;
      };
      begin(fromP, PK, p.e.M, at_P, p.ldp, baseP, endP, recsP, inP);
      begin(fromQ, QK, p.e.N, at_Q, ldq, baseQ, endQ, recsQ, inQ);
      set_offsets(inP, inQ);
    }
    const bool last = nxt == KT_in - 1, behind = nxt >= KT_in;
    recsP = behind ? 0 : PK && last ? endP : recsP;
    recsQ = behind ? 0 : QK && last ? endQ : recsQ;
    soff = behind ? 0 : soff;  // (a scalar offset past a descriptor's end may turn its check around)
    if ((!PK || !QK) && last && (p.K & (BK - 1))) {  // the reduction may end inside this slab
      const int in = p.K - k_in - nxt * BK;
      set_offsets(PK ? inP : in, QK ? inQ : in);
    }
  };
  // LDS: the slots of P, then those of Q
  auto load = [&](int slot, auto jc) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value, jo = j < PL ? j : j - PL;
    constexpr bool isP = j < PL, kmajor = isP ? PK : QK;
    uint32_t v;
    if constexpr (TM == 4) {
      v = isP ? voffP[isP ? jo : 0] : voffQ[isP ? 0 : jo];
    } else {
      // (the sums stay here instead of in registers of the whole loop)
      if constexpr (isP) asm volatile("" : "+v"(voffP[0]));
      else asm volatile("" : "+v"(voffQ[0]));
      v = isP ? voffP[0] : voffQ[0];
      if constexpr (jo != 0) v += (uint32_t)jo * (uint32_t)((isP ? P_ROWS * p.ldp : Q_FROM * ldq) * 2);
    }
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)(isP ? baseP : baseQ), 0, isP ? recsP : recsQ, 0x00020000);
    char* l = lds + (isP ? slot * PB : NS * PB + slot * QB) + jo * (NT * 16) + wave * (64 * 16);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LDS_PTR(l), 16, (int)v, kmajor ? 0 : soff, 0, 0);
  };
  auto loaded = [&]() __attribute__((always_inline)) {
    slot_in = slot_in == NS - 1 ? 0 : slot_in + 1;
    if constexpr (!PK || !QK) soff += BK * 2;
    if constexpr (PK) baseP += stepP;
    if constexpr (QK) baseQ += stepQ;
    if (++nxt >= KT_in - 1) turn();
  };

  // ---- LDS -> fragments: lane l holds row (column) l % 16 and reduction indices 8 (l / 16) .. + 7 of a 32-deep step
  const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)lds;
  const int l16 = lane & 15, quad = lane >> 4;
  // (fragments f and f + 1 of a K-major operand differ in bit 5 of the address: where registers are short, one serves both)
  constexpr int AF = PK ? (TM == 8 ? 2 : 1) : 1, NA = PK ? TM / AF : ST, NB = QK ? TN : ST;
  uint32_t aoff[NA], boff[NB];
  auto kmajor_off = [&](int base, int width, int at, int f) {
    return lds_base + (uint32_t)(base + (8 * quad + (l16 >> 2)) * (width * 2) + ((((at + f * 16) >> 5) ^ (l16 >> 2)) << 6) +
                                 ((f ^ quad) & 1) * 32 + (l16 & 3) * 8);
  };
  auto row_off = [&](int base, int at, int st) {
    return lds_base + (uint32_t)(base + (at + l16) * (BK * 2) + ((st * 4 + quad) ^ (l16 >> 1)) * 16);
  };
#pragma unroll
  for (int f = 0; f < NA; ++f) aoff[f] = PK ? kmajor_off(0, BM, wm * Cfg::WTM, f * AF) : row_off(0, wm * Cfg::WTM, f);
#pragma unroll
  for (int f = 0; f < NB; ++f)
    boff[f] = QK ? kmajor_off(NS * PB, BN, wn * Cfg::WTN, f) : row_off(NS * PB, wn * Cfg::WTN, f);

  f32x4 acc[TM][TN];
  auto clear_acc = [&]() {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  clear_acc();

  typedef std::integral_constant<int, 0> ic0;
  typedef std::integral_constant<int, 1> ic1;
  // AHEAD (64 x 64 wavefront tiles): the fragments of a whole slab are requested one slab ahead, by parity of the slab, with
  // one wait for them and one barrier per slab.  128-row wavefront tiles have registers for half a step ahead: A by parity
  // of the half (four fragments), B by parity of the step.
  constexpr bool AHEAD = TM == 4;
  bf16x8 fa[2][AHEAD ? ST * 4 : 4], fb[2][AHEAD ? ST * TN : TN];
  auto read_a = [&](auto slotc, auto stc, auto ic, bf16x8& dst) {
    constexpr int slot = decltype(slotc)::value, st = decltype(stc)::value, i = decltype(ic)::value;
    if constexpr (PK && AF == 2) {
      asm volatile("" : "+v"(aoff[i / 2]));  // (the other address is not kept)
      lds_read_tr<slot * PB + st * (32 * BM * 2), 4 * BM * 2>(dst, aoff[i / 2] ^ (i & 1 ? 32u : 0u));
    } else if constexpr (PK) lds_read_tr<slot * PB + st * (32 * BM * 2), 4 * BM * 2>(dst, aoff[i]);
    else lds_read16<slot * PB + i * (16 * BK * 2)>(dst, aoff[st]);
  };
  auto read_b = [&](auto slotc, auto stc, auto jc, bf16x8& dst) {
    constexpr int slot = decltype(slotc)::value, st = decltype(stc)::value, j = decltype(jc)::value;
    if constexpr (QK) lds_read_tr<slot * QB + st * (32 * BN * 2), 4 * BN * 2>(dst, boff[j]);
    else lds_read16<slot * QB + j * (16 * BK * 2)>(dst, boff[st]);
  };
  // To the next slot, where slots are in the offsets (more than two: P's would pass the reads' 16-bit offset).
  int slot_out = 0;
  auto next_slot = [&]() {
    if constexpr (NS > 2) {
      const bool wrap = slot_out == NS - 1;
      const uint32_t dp = wrap ? (uint32_t)(-(NS - 1) * PB) : (uint32_t)PB, dq = wrap ? (uint32_t)(-(NS - 1) * QB) : (uint32_t)QB;
      slot_out = wrap ? 0 : slot_out + 1;
#pragma unroll
      for (int f = 0; f < NA; ++f) aoff[f] += dp;
#pragma unroll
      for (int f = 0; f < NB; ++f) boff[f] += dq;
    }
  };

  typedef LinSched<HALVES, ST, PK ? 2 : 1, QK ? 2 : 1> FS;
  auto read_frag = [&](auto slotc, auto hnc, auto rc) {  // read r of those half hn of a slab needs (not AHEAD)
    constexpr int hn = decltype(hnc)::value, r = decltype(rc)::value, st = hn / HALVES, half = hn % HALVES;
    typedef std::integral_constant<int, st> stc;
    if constexpr (half != 0) read_a(slotc, stc(), std::integral_constant<int, 4 + r>(), fa[hn & 1][r]);
    else if constexpr (r == 0 || r > 4) read_a(slotc, stc(), std::integral_constant<int, (r == 0 ? 0 : r - 4)>(), fa[hn & 1][r == 0 ? 0 : r - 4]);
    else read_b(slotc, stc(), std::integral_constant<int, r - 1>(), fb[st & 1][r - 1]);
  };
  auto read_ahead = [&](auto parc, auto rc) {  // read r of a slab's sixteen, from where the offsets point
    constexpr int par = decltype(parc)::value, r = decltype(rc)::value, st = r / 8, f = r % 8;
    typedef std::integral_constant<int, st> stc;
    if constexpr (f < 4) read_a(ic0(), stc(), std::integral_constant<int, f>(), fa[par][st * 4 + f]);
    else read_b(ic0(), stc(), std::integral_constant<int, f - 4>(), fb[par][st * TN + f - 4]);
  };
  // every fragment of that parity that may be in flight has arrived
  auto landed = [&](auto parc) {
    auto& a = fa[decltype(parc)::value];
    auto& b = fb[decltype(parc)::value];
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(b[0]), "+v"(b[1]), "+v"(b[2]), "+v"(b[3]));
    if constexpr (AHEAD)
      asm volatile("" : "+v"(a[4]), "+v"(a[5]), "+v"(a[6]), "+v"(a[7]), "+v"(b[4]), "+v"(b[5]), "+v"(b[6]), "+v"(b[7]));
  };

  // One slab, whose first fragments (AHEAD: all of them) are on their way, in slot `slotc` (0, 1) where there are two.
  auto slab = [&](auto slotc) __attribute__((always_inline)) {
    constexpr int here = NS == 2 ? decltype(slotc)::value : 0, next = NS == 2 ? here ^ 1 : 0, par = decltype(slotc)::value;
    if constexpr (AHEAD) {
      pipeline_barrier<(NS - 2) * LPS>();  // the next slab has landed, this one is read: its slot is refilled
      landed(slotc);
      next_slot();
      __builtin_amdgcn_sched_barrier(0);
      static_for<0, 32>([&](auto qc) {
        constexpr int q = decltype(qc)::value, st = q / 16, i = (q % 16) / 4, j = q % 4;
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[par][st * TN + j], fa[par][st * 4 + i], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        // a refill behind every fourth MFMA, a read behind each of the others
        constexpr bool refill = q % 4 == 3 && q / 4 < LPS;
        constexpr int r = q - (q / 4 < LPS ? q / 4 : LPS);
        if constexpr (refill) load(slot_in, std::integral_constant<int, q / 4>());
        else if constexpr (r < 16) read_ahead(std::integral_constant<int, par ^ 1>(), std::integral_constant<int, r>());
        __builtin_amdgcn_sched_barrier(0);
      });
      loaded();
    } else {
      static_for<0, HP>([&](auto hpc) {
        constexpr int hp = decltype(hpc)::value, st = hp / HALVES, half = hp % HALVES;
        constexpr bool last = hp == HP - 1;
        if constexpr (last) pipeline_barrier<(NS - 2) * LPS>();
        static_for<0, 16>([&](auto qc) {
          constexpr int q = decltype(qc)::value, i = q / 4, j = q % 4;
          frag_wait<FS::allowed(hp, q)>(fa[hp & 1][i], fb[st & 1][j]);
          acc[half * 4 + i][j] =
              __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[st & 1][j], fa[hp & 1][i], acc[half * 4 + i][j], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (FS::read_behind(hp, q) >= 0) {
            typedef std::integral_constant<int, FS::read_behind(hp, q)> rc;
            if constexpr (last) read_frag(std::integral_constant<int, next>(), ic0(), rc());
            else read_frag(std::integral_constant<int, here>(), std::integral_constant<int, hp + 1>(), rc());
          }
          if constexpr (last && (q & 1) && q / 2 < LPS) load(here, std::integral_constant<int, q / 2>());
          __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (last) loaded();
      });
    }
  };

  // ---- the ring is filled; slab 0's fragments
  turn();
  static_for<0, NS>([&](auto sc) {
    static_for<0, LPS>([&](auto jc) { load(decltype(sc)::value, jc); });
    loaded();
  });
  pipeline_barrier<(NS - 1) * LPS>();
  if constexpr (AHEAD) static_for<0, 16>([&](auto rc) { read_ahead(ic0(), rc); });
  else static_for<0, 8>([&](auto rc) { read_frag(ic0(), ic0(), rc); });
  __builtin_amdgcn_sched_barrier(0);

  for (int pid = blockIdx.x;;) {
    const Tile t = tile(pid);
    for (int kt = 0; kt < t.KT; kt += 2) {  // (a slab of zeros behind an odd number)
      slab(ic0());
      slab(ic1());
    }
    // The first fragments of the next tile are on their way: they land before the epilogue, whose register traffic must not
    // meet a read in flight.
    landed(ic0());

    // ---- element e of a lane: row l16, column 4 * quad + e of its 16 x 16 tile
    const int lane = again() & 63, l16 = lane & 15, quad = lane >> 4;
    constexpr int STEP = GATED ? 2 : 1;  // 16-column groups of a tile per group of C
    const int row0 = t.ti * BM + wm * Cfg::WTM + l16, col0 = (t.tj * BN + wn * Cfg::WTN) / STEP + 4 * quad;
    if constexpr (SPLIT) {
      float* out = p.part + (int64_t)t.part * STEP * p.e.M * p.e.N;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int row = row0 + i * 16, col = col0 + j / STEP * 16;
          if (row >= p.e.M || col >= p.e.N) continue;
          float* o = out + ((int64_t)(j % STEP) * p.e.M + row) * p.e.N + col;
          if (p.e.N % 4 == 0) {
            *(f32x4*)o = acc[i][j];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < p.e.N) o[e] = acc[i][j][e];
          }
        }
    } else {
      f32x4 b[TN];
      if constexpr (GATED) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
          b[j] = j % 2 ? bias4(p.bias2, p.bias2_dtype, p.e.N, col0 + j / 2 * 16) : bias4(p.e, col0 + j / 2 * 16);
      } else if constexpr (!PK && !QK) {
#pragma unroll
        for (int j = 0; j < TN; ++j) b[j] = bias4(p.e, col0 + j * 16);
      }
      // Sixteen rows at a time through the wavefront's staging, so that C and the slopes leave in whole 128-byte lines, as
      // wide as rows of C allow: an 8-byte piece q of row r lies at q ^ 2 ((r / 2) % 8), which spreads writes and reads over
      // all banks.
      constexpr int RB = TM == 8 ? 2 : 4;
      char* const stg = lds + Cfg::RING_BYTES + wave * Cfg::STG_BYTES;
      const int wrow = t.ti * BM + wm * Cfg::WTM, wcol = t.tj * BN + wn * Cfg::WTN;  // (gated: half of it in C, all in e.slope)
      auto put = [&](int j, uint2 w) { *(uint2*)(stg + l16 * 128 + (((4 * j + quad) ^ (((l16 >> 1) & 7) << 1)) << 3)) = w; };
      auto send = [&](auto widthc, uint16_t* o, int pitch, int row) __attribute__((always_inline)) {
        constexpr int W = decltype(widthc)::value, LANES = 64 / W;  // elements of a lane, lanes of a row
        typedef std::conditional_t<W == 8, uint4, std::conditional_t<W == 4, uint2, std::conditional_t<W == 2, uint32_t, uint16_t>>> piece_t;
        const int sr = lane / LANES, sc = lane % LANES * W;
        asm volatile("" ::: "memory");
#pragma unroll
        for (int h = 0; h < 16; h += W) {
          const int r = sr + h;
          const piece_t w = *(const piece_t*)(stg + r * 128 + (((sc >> 2) ^ (((r >> 1) & 7) << 1)) << 3) + (sc & 3) * 2);
          if (row + r < p.e.M && wcol + sc < pitch) *(piece_t*)(o + (int64_t)(row + r) * pitch + wcol + sc) = w;
        }
        asm volatile("" ::: "memory");
      };
      // Rows of 64 bytes: their 16-byte piece s at s ^ (r / 4) % 4, behind `at` bytes of the staging.
      auto half_at = [&](int at, int r, int s) { return stg + at + r * 64 + ((s ^ (r >> 2)) << 4); };
      auto send_half = [&](auto widthc, uint16_t* o, int pitch, int row) __attribute__((always_inline)) {
        constexpr int W = decltype(widthc)::value, LANES = 32 / W;
        typedef std::conditional_t<W == 8, uint4, std::conditional_t<W == 4, uint2, std::conditional_t<W == 2, uint32_t, uint16_t>>> piece_t;
        const int sr = lane / LANES, sc = lane % LANES * W, at = wcol / 2 + sc;
#pragma unroll
        for (int h = 0; h < 16; h += 2 * W) {
          const int r = sr + h;
          const piece_t w = *(const piece_t*)(half_at(0, r, sc >> 3) + (sc & 7) * 2);
          if (row + r < p.e.M && at < pitch) *(piece_t*)(o + (int64_t)(row + r) * pitch + at) = w;
        }
      };
      if constexpr (GATED) {
        char* const kept = (char*)p.e.slope;
        const int64_t pitch = kept_pitch(p.e.N, WIDE);
        const int kept_at = wcol / 64 * kept_block(WIDE);
        // sixteen rows of 128 bytes (put) to byte `at` of their blocks
        auto send_kept = [&](int at, int row) __attribute__((always_inline)) {
          asm volatile("" ::: "memory");
#pragma unroll
          for (int k = 0; k < 16; k += 8) {
            const int r = lane / 8 + k, s = lane % 8;
            const uint4 w = *(const uint4*)(stg + r * 128 + ((2 * s ^ (((r >> 1) & 7) << 1)) << 3));
            if (row + r < p.e.M && kept_at < pitch) *(uint4*)(kept + (int64_t)(row + r) * pitch + kept_at + at + s * 16) = w;
          }
          asm volatile("" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          uint2 h[TN / 2];
          uint2 low[TN];
#pragma unroll
          for (int j = 0; j < TN / 2; ++j) {
            Kept4 to_gate, to_up;
            gated4<ACT, SLOPE, WIDE>(acc[i][2 * j] + b[2 * j], acc[i][2 * j + 1] + b[2 * j + 1], h[j], to_gate, to_up);
            if constexpr (SLOPE) {
              put(j, to_gate.high);
              put(TN / 2 + j, to_up.high);
              low[j] = to_gate.low;
              low[TN / 2 + j] = to_up.low;
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          const int row = wrow + i * 16;
          if constexpr (SLOPE) {
            send_kept(0, row);
#pragma unroll
            for (int j = 0; j < TN; ++j) {
              if constexpr (WIDE) put(j, low[j]);
              else *(uint32_t*)(half_at(1024, l16, j) + quad * 4) = low[j].x;
            }
            if constexpr (WIDE) send_kept(128, row);
          }
#pragma unroll
          for (int j = 0; j < TN / 2; ++j) *(uint2*)(half_at(0, l16, 2 * j + (quad >> 1)) + (quad & 1) * 8) = h[j];
          asm volatile("" ::: "memory");
          if constexpr (SLOPE && !WIDE) {
            const int r = lane / 4, s = lane % 4;
            const uint4 w = *(const uint4*)half_at(1024, r, s);
            if (row + r < p.e.M && kept_at < pitch) *(uint4*)(kept + (int64_t)(row + r) * pitch + kept_at + 128 + s * 16) = w;
          }
          if (p.e.vec == 8) send_half(std::integral_constant<int, 8>(), p.e.C, p.e.N, row);
          else if (p.e.vec == 4) send_half(std::integral_constant<int, 4>(), p.e.C, p.e.N, row);
          else if (p.e.vec == 2) send_half(std::integral_constant<int, 2>(), p.e.C, p.e.N, row);
          else send_half(std::integral_constant<int, 1>(), p.e.C, p.e.N, row);
          asm volatile("" ::: "memory");
          __builtin_amdgcn_sched_barrier(0);
        }
      } else
#pragma unroll
      for (int i0 = 0; i0 < TM; i0 += RB) {
        uint2 r[RB][TN];  // (the addend of RB * 16 rows in one go: one way to memory)
        if constexpr (!PK && !QK)
#pragma unroll
          for (int i = 0; i < RB; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) r[i][j] = residual4(p.e, row0 + (i0 + i) * 16, col0 + j * 16);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          uint2 y[TN];
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const f32x4 z = acc[i0 + i][j];
            uint2 sl;
            if constexpr (PK || QK) y[j] = make_uint2(pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3]));  // a gradient: nothing to add
            else finish4<ACT, SLOPE>(p.e, z, b[j], r[i][j], y[j], sl);
            if constexpr (SLOPE) {
              put(j, sl);
              __builtin_amdgcn_sched_barrier(0);  // (four elements' intermediate values at a time: more would not fit)
            }
          }
          const int row = wrow + (i0 + i) * 16;
          if constexpr (SLOPE) send(std::integral_constant<int, 8>(), p.e.slope, slope_pitch(p.e.N), row);
#pragma unroll
          for (int j = 0; j < TN; ++j) put(j, y[j]);
          if (p.e.vec == 8) send(std::integral_constant<int, 8>(), p.e.C, p.e.N, row);
          else if (p.e.vec == 4) send(std::integral_constant<int, 4>(), p.e.C, p.e.N, row);
          else if (p.e.vec == 2) send(std::integral_constant<int, 2>(), p.e.C, p.e.N, row);
          else send(std::integral_constant<int, 1>(), p.e.C, p.e.N, row);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    pid += p.grid;
    if (pid >= p.total) break;
    clear_acc();
    __builtin_amdgcn_sched_barrier(0);
  }
  wait_vmcnt<0>();  // loads of zeros behind the last tile land before the LDS is given back
#pragma unroll
  for (int i = 0; i < (int)(sizeof(fa[0]) / sizeof(fa[0][0])); ++i) {
    asm volatile("" ::"v"(fa[0][i]));
    asm volatile("" ::"v"(fb[0][i]));
  }
}

// ---- host
// Whether rows of an operand are whole 16-byte chunks, as far apart as the kernels can address.
static inline bool lin_chunks(const void* ptr, int64_t ld, int extent) {
  return ((uint64_t)ptr & 15) == 0 && ld % 8 == 0 && ld >= ((extent + 7) & ~7) && ld <= kLinMaxLd;
}
// LinEpilogue::vec
static inline int lin_vec(const void* C, const void* R, int N, int64_t ldr) {
  const uint64_t bytes = ((uint64_t)C | (uint64_t)R) | (uint64_t)N * 2 | (R ? (uint64_t)ldr * 2 : 0);
  return bytes % 16 == 0 ? 8 : bytes % 8 == 0 ? 4 : bytes % 4 == 0 ? 2 : 1;
}
// The tiles of M x N results and what the kernel divides by; false where there are too many.
template <class Cfg>
static bool lin_tile_list(int M, int64_t N, LinTileParams& tp) {
  tp.tilesM = (M + Cfg::BM - 1) / Cfg::BM;
  tp.tilesN = (int)((N + Cfg::BN - 1) / Cfg::BN);
  if ((int64_t)tp.tilesM * tp.tilesN > 0x7fffffff || (int64_t)tp.tilesN * 8 > 0x7fffffff) return false;
  tp.inv_tiles = (uint32_t)(0xffffffffu / ((int64_t)tp.tilesM * tp.tilesN));
  tp.inv_group = (uint32_t)(0xffffffffu / (8 * (int64_t)tp.tilesN));
  tp.inv_tail = tp.tilesM % 8 ? 0xffffffffu / (tp.tilesM % 8) : 0;
  return true;
}

template <class Cfg, bool PK, bool QK, int ACT, bool SLOPE, bool SPLIT, int FORM = kLinPlain>
static hipError_t launch_tile(std::conditional_t<FORM == kLinPlain, LinTileParams, LinTwoParams> tp, hipStream_t st) {
  static std::atomic<uint64_t> attr_done{0};
  auto kern = lin_tile_kernel<Cfg, PK, QK, ACT, SLOPE, SPLIT, FORM>;
  if (hipError_t e = set_max_dynamic_lds_once((const void*)kern, Cfg::LDS_BYTES, attr_done)) return e;
  const int64_t total = (int64_t)tp.tilesM * tp.tilesN * tp.splits;
  if (total > 0x7fffffff) return hipErrorInvalidValue;
  static std::atomic<int> cu_count[64];
  int dev = 0;
  if (hipError_t e = hipGetDevice(&dev)) return e;
  int cus = cu_count[dev & 63].load(std::memory_order_relaxed);
  if (cus == 0) {
    if (hipError_t e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev)) return e;
    if (cus <= 0) return hipErrorInvalidValue;
    cu_count[dev & 63].store(cus, std::memory_order_relaxed);
  }
  tp.total = (int)total;
  tp.grid = total < cus ? (int)total : cus;
  hipLaunchKernelGGL(kern, dim3((unsigned)tp.grid), dim3(Cfg::NT), Cfg::LDS_BYTES, st, tp);
  return hipGetLastError();
}

}  // namespace dion
