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
static __device__ __forceinline__ f32x4 bias4(const LinEpilogue& p, int col) {
  f32x4 b = {0.f, 0.f, 0.f, 0.f};
  if (p.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < p.N) b[e] = p.bias_dtype ? ((const float*)p.bias)[col + e] : bf16_to_f32(((const bf16_t*)p.bias)[col + e]);
  }
  return b;
}
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
template <class Cfg, bool PK, bool QK, int ACT, bool SLOPE, bool SPLIT>
__global__ __launch_bounds__(Cfg::NT, 2) void lin_tile_kernel(const LinTileParams p) {
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
    t.KT = min((p.K + BK - 1) / BK - t.part * p.slabs, p.slabs);
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
  auto offset = [&](int tid, bool kmajor, int width, int ld, int in) __attribute__((always_inline)) {  // in: elements of a row from the tile's start
    const int cpr = kmajor ? width / 8 : 8, row = tid / cpr, c = tid % cpr;
    const int chunk = kmajor ? (((c >> 2) ^ (row & 3)) << 2) | ((c & 3) ^ (((row >> 3) & 1) << 1)) : c ^ ((row >> 1) & 7);
    return chunk * 8 < in ? (uint32_t)(row * ld + chunk * 8) * 2u : kEnd;
  };
  // 64-row wavefront tiles have a register for every load's offset; 128-row ones one per operand, the rest is added.
  constexpr int VP = TM == 4 ? PL : 1, VQ = TM == 4 ? QL : 1;
  uint32_t voffP[VP], voffQ[VQ];
  auto set_offsets = [&](int inP, int inQ) __attribute__((always_inline)) {
    const int t = again();
    const uint32_t vp = offset(t, PK, BM, p.ldp, inP), vq = offset(t, QK, BN, p.ldq, inQ);
#pragma unroll
    for (int j = 0; j < VP; ++j) voffP[j] = vp + (uint32_t)j * (uint32_t)(P_ROWS * p.ldp * 2);
#pragma unroll
    for (int j = 0; j < VQ; ++j) voffQ[j] = vq + (uint32_t)j * (uint32_t)(Q_ROWS * p.ldq * 2);
  };
  // what is loaded next: slab nxt of a tile of KT_in, into slot slot_in
  const char *baseP = (const char*)p.P, *baseQ = (const char*)p.Q;
  const int64_t stepP = PK ? (int64_t)BK * p.ldp * 2 : 0, stepQ = QK ? (int64_t)BK * p.ldq * 2 : 0;
  int pid_in = blockIdx.x, k_in = 0, nxt = 0, KT_in = 0, slot_in = 0, soff = 0, endP = 0, endQ = 0, inP = 0, inQ = 0;
  int recsP = 0, recsQ = 0;
  // What changes with the last slab of a tile and behind it.  (Slabs behind an odd number of them, and behind the last tile, are
  // loaded as zeros: the loop is two slabs long, and its waits count on every load.)
  auto turn = [&]() __attribute__((always_inline)) {
    if (nxt >= ((KT_in + 1) & ~1) && pid_in < p.total) {
      const Tile t = tile(pid_in);
      pid_in += p.grid;
      nxt = 0;
      soff = 0;
      KT_in = t.KT;
      k_in = t.part * p.slabs * BK;
      auto begin = [&](const bf16_t* base, bool kmajor, int extent, int at, int ld, const char*& from, int& end, int& recs,
                       int& in) __attribute__((always_inline)) {
        from = (const char*)(base + (kmajor ? (int64_t)k_in * ld + at : (int64_t)at * ld + k_in));
        // (K-major: rows from the tile's last slab on; all of a slab's rows are there before it)
        const int64_t n = (int64_t)(kmajor ? p.K - k_in - (t.KT - 1) * BK : extent - at) * ld * 2;
        end = (int)(uint32_t)(n < (int64_t)kEnd ? n : (int64_t)kEnd);
        recs = kmajor ? (int)kEnd : end;
        in = kmajor ? ((extent + 7) & ~7) - at : BK;
      };
      begin(p.P, PK, p.e.M, t.ti * BM, p.ldp, baseP, endP, recsP, inP);
      begin(p.Q, QK, p.e.N, t.tj * BN, p.ldq, baseQ, endQ, recsQ, inQ);
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
      if constexpr (jo != 0) v += (uint32_t)jo * (uint32_t)((isP ? P_ROWS * p.ldp : Q_ROWS * p.ldq) * 2);
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
    const int row0 = t.ti * BM + wm * Cfg::WTM + l16, col0 = t.tj * BN + wn * Cfg::WTN + 4 * quad;
    if constexpr (SPLIT) {
      float* out = p.part + (int64_t)t.part * p.e.M * p.e.N;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int row = row0 + i * 16, col = col0 + j * 16;
          if (row >= p.e.M || col >= p.e.N) continue;
          float* o = out + (int64_t)row * p.e.N + col;
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
      if constexpr (!PK && !QK)
#pragma unroll
        for (int j = 0; j < TN; ++j) b[j] = bias4(p.e, col0 + j * 16);
      // Sixteen rows at a time through the wavefront's staging, so that C and the slopes leave in whole 128-byte lines, as
      // wide as rows of C allow: an 8-byte piece q of row r lies at q ^ 2 ((r / 2) % 8), which spreads writes and reads over
      // all banks.
      constexpr int RB = TM == 8 ? 2 : 4;
      char* const stg = lds + Cfg::RING_BYTES + wave * Cfg::STG_BYTES;
      const int wrow = t.ti * BM + wm * Cfg::WTM, wcol = t.tj * BN + wn * Cfg::WTN;
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
__global__ __launch_bounds__(256) void lin_sum_kernel(const float* __restrict__ partial, int parts, int cols, void* out,
                                                      int out_dtype) {
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
    if (out_dtype) ((float*)out)[c] = s;
    else ((bf16_t*)out)[c] = f32_to_bf16(s);
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
enum LinTile { kLinFew, kLin128, kLinWide, kLin256 };
struct LinPlan {
  LinTile tile;
  int splits, slabs;
};
static LinPlan lin_plan(int M, int N, int K, int p_kmajor, int q_kmajor) {
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
  if (M <= 32 && !p_kmajor && !q_kmajor) {
    const double wgs = (N + 15) / 16, each = M <= 16 ? 0.77 + 0.033 * (M - 1) : 1.5;
    if (2.5 + each * (K / 512.0) * (wgs > 256 ? wgs / 256 : 1) < least) return {kLinFew, 1, 0};
  }
  return best;
}

size_t lin_product_scratch(int M, int N, int K, int p_kmajor, int q_kmajor) {
  const LinPlan plan = lin_plan(M, N, K, p_kmajor, q_kmajor);
  return plan.splits > 1 ? (size_t)plan.splits * M * N * sizeof(float) : 0;
}

template <class Cfg, bool PK, bool QK, int ACT, bool SLOPE, bool SPLIT>
static hipError_t launch_tile(LinTileParams tp, hipStream_t st) {
  static std::atomic<uint64_t> attr_done{0};
  auto kern = lin_tile_kernel<Cfg, PK, QK, ACT, SLOPE, SPLIT>;
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

template <class Cfg, int ACT>
static hipError_t launch_act(const LinTileParams& tp, hipStream_t st) {
  return tp.e.slope ? launch_tile<Cfg, false, false, ACT, true, false>(tp, st)
                    : launch_tile<Cfg, false, false, ACT, false, false>(tp, st);
}

template <class Cfg>
static hipError_t launch_tiles(const LinProduct& p, LinTileParams tp, hipStream_t st) {
  tp.tilesM = (p.M + Cfg::BM - 1) / Cfg::BM;
  tp.tilesN = (p.N + Cfg::BN - 1) / Cfg::BN;
  if ((int64_t)tp.tilesM * tp.tilesN > 0x7fffffff || (int64_t)tp.tilesN * 8 > 0x7fffffff) return hipErrorInvalidValue;
  tp.inv_tiles = (uint32_t)(0xffffffffu / ((int64_t)tp.tilesM * tp.tilesN));
  tp.inv_group = (uint32_t)(0xffffffffu / (8 * (int64_t)tp.tilesN));
  tp.inv_tail = tp.tilesM % 8 ? 0xffffffffu / (tp.tilesM % 8) : 0;
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

hipError_t launch_lin_product(const LinProduct& p, hipStream_t st) {
  if (p.M <= 0 || p.N <= 0 || p.K <= 0) return hipErrorInvalidValue;
  auto whole = [](const void* ptr, int64_t ld, int extent) {
    return ((uint64_t)ptr & 15) == 0 && ld % 8 == 0 && ld >= ((extent + 7) & ~7) && ld <= kLinMaxLd;
  };
  if (!whole(p.P, p.ldp, p.p_kmajor ? p.M : p.K) || !whole(p.Q, p.ldq, p.q_kmajor ? p.N : p.K)) return hipErrorInvalidValue;
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
  const uint64_t bytes = ((uint64_t)p.C | (uint64_t)p.R) | (uint64_t)p.N * 2 | (p.R ? (uint64_t)p.ldr * 2 : 0);
  e.vec = bytes % 16 == 0 ? 8 : bytes % 8 == 0 ? 4 : bytes % 4 == 0 ? 2 : 1;
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
  if (plan.splits > 1) {
    const int64_t wg = ((int64_t)p.M * ((p.N + 3) / 4) + 255) / 256;
    const dim3 grid((unsigned)(wg < 65536 ? wg : 65536));
    hipLaunchKernelGGL(lin_join_kernel, grid, dim3(256), 0, st, e, p.scratch, plan.splits);
  }
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
  hipLaunchKernelGGL(lin_sum_kernel, dim3((cols + 15) / 16), dim3(256), 0, st, partial, parts, cols, out, out_dtype);
  return hipGetLastError();
}

}  // namespace dion
