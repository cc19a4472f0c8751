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
#include <hip/hip_fp16.h>

#include <atomic>

#include "gemm_tile.h"
#include "linear.h"

namespace dion {

// ---------------------------------------------------------------------------------------------- activations
static __device__ __forceinline__ float rcp_fast(float v) { return __builtin_amdgcn_rcpf(v); }

// act(z), and act'(z) in `slope`.  Exponentials and quotients by the hardware's approximations (1 ulp): the result is rounded
// to bf16, the slope to eleven bits.
static __device__ __forceinline__ float activate(int act, float z, float& slope) {
  switch (act) {
    case kActRelu:
      slope = z > 0.f ? 1.f : 0.f;
      return z < 0.f ? 0.f : z;  // (NaN stays)
    case kActReluSquared: {
      const float r = z < 0.f ? 0.f : z;
      slope = 2.f * r;
      return r * r;
    }
    case kActSilu: {
      const float s = rcp_fast(1.f + __expf(-z));
      slope = s * (1.f + z * (1.f - s));
      return z * s;
    }
    case kActGelu: {
      const float cdf = 0.5f * (1.f + erff(z * 0.70710678f));
      slope = cdf + z * 0.39894228f * __expf(-0.5f * z * z);
      return z * cdf;
    }
    case kActGeluTanh: {
      const float u = 0.79788456f * z * (1.f + 0.044715f * z * z);
      const float t = 1.f - 2.f * rcp_fast(1.f + __expf(2.f * u));
      slope = 0.5f * (1.f + t) + 0.5f * z * (1.f - t * t) * 0.79788456f * (1.f + 0.134145f * z * z);
      return 0.5f * z * (1.f + t);
    }
    default:
      slope = 1.f;
      return z;
  }
}

static __device__ __forceinline__ uint16_t slope_pack(int act, float s) {
  if (act != kActReluSquared) return __builtin_bit_cast(uint16_t, (_Float16)s);
  // Round to nine bits of mantissa; code 0 is zero, 0xffff NaN and everything past 2^65.
  const uint32_t b = __float_as_uint(s) + 0x2000u;
  if (b < (64u << 23) + (1u << 14)) return 0;
  const uint32_t c = (b >> 14) - (64u << 9);
  return c > 0xffffu ? 0xffffu : (uint16_t)c;
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
  int vec;  // N, ldr and the addresses allow 8-byte accesses to four neighbours
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
  if (p.vec) return *(const uint2*)r;
  w.x = r[0];
  if (col + 1 < p.N) w.x |= (uint32_t)r[1] << 16;
  if (col + 2 < p.N) w.y = r[2];
  if (col + 3 < p.N) w.y |= (uint32_t)r[3] << 16;
  return w;
}
// Finishes and stores elements (row, col .. col + 3).  ACT: an activation may be there.
template <bool ACT>
static __device__ __forceinline__ void finish4(const LinEpilogue& p, int row, int col, f32x4 z, f32x4 b, uint2 r) {
  if (row >= p.M || col >= p.N) return;
  float v[4], s[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = z[e] + b[e];
    if constexpr (ACT) v[e] = activate(p.act, v[e], s[e]);
  }
  const int64_t at = (int64_t)row * p.N + col;
  if constexpr (ACT) {
    if (p.slope) {
      uint16_t c[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] = slope_pack(p.act, s[e]);
      if (p.vec) {
        *(uint2*)(p.slope + at) = make_uint2(c[0] | (uint32_t)c[1] << 16, c[2] | (uint32_t)c[3] << 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < p.N) p.slope[at + e] = c[e];
      }
    }
  }
  if (p.R) {
    v[0] += __uint_as_float(r.x << 16);
    v[1] += __uint_as_float(r.x & 0xffff0000u);
    v[2] += __uint_as_float(r.y << 16);
    v[3] += __uint_as_float(r.y & 0xffff0000u);
  }
  if (p.vec) {
    *(uint2*)(p.C + at) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < p.N) p.C[at + e] = f32_to_bf16(v[e]);
  }
}

// ---------------------------------------------------------------------------------------------- tiles
template <int BM_, int BN_, int WM_, int WN_>
struct LinCfg {
  static constexpr int BM = BM_, BN = BN_, BK = 64, WM = WM_, WN = WN_;
  static constexpr int NT = WM * WN * 64;
  static constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
  static constexpr int HALVES = TM / 4, ST = BK / 32;
  static constexpr int OP_BYTES = BM * BK * 2;  // one operand of one slab
  static constexpr int LDS_BYTES = 4 * OP_BYTES;
  static constexpr int OP_LOADS = OP_BYTES / (NT * 16);
  static_assert(BM == BN && TN == 4 && (TM == 4 || TM == 8) && OP_LOADS == 4, "square tiles, wavefronts of 64 or 128 rows by 64 columns");
};
typedef LinCfg<256, 256, 2, 4> Lin256;  // 8 wavefronts: one workgroup per CU
typedef LinCfg<128, 128, 2, 2> Lin128;  // 4 wavefronts: two workgroups per CU

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
  uint32_t inv_tiles, inv_group, inv_tail;
};

// One output tile (of one part of the reduction) per workgroup.  Operand slabs reach a two-slot LDS ring by direct-to-LDS
// buffer loads, whose descriptors end where the matrix does: rows past an edge arrive as zeros, and need no padded copy.  Chunks
// behind the reduction's end in the last slab of an operand with the reduction along rows get an offset past the end.  XOR
// swizzles keep the LDS writes and the fragment reads free of bank conflicts.  The MFMA operands are swapped (B fragment
// first), so that a lane's four sums are neighbours of one row of C: 8-byte accesses to C, the addend and the slopes.
// SPLIT: the sums of a part go to p.part as fp32, and lin_join_kernel finishes them.
template <class Cfg, bool PK, bool QK, bool ACT, bool SPLIT>
__global__ __launch_bounds__(Cfg::NT, 2) void lin_tile_kernel(const LinTileParams p) {
  constexpr int BM = Cfg::BM, BN = Cfg::BN, BK = Cfg::BK, TM = Cfg::TM, TN = Cfg::TN, ST = Cfg::ST, HALVES = Cfg::HALVES;
  constexpr int HP = HALVES * ST, OPB = Cfg::OP_BYTES, NT = Cfg::NT;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;

  // ---- which tile: every XCD gets one contiguous run of the list, eight rows of tiles at a time, columns first within them
  int ti, tj, part;
  {
    const int total = gridDim.x, xcd = blockIdx.x & 7, q = total >> 3, r = total & 7;
    const int lt = xcd * q + (xcd < r ? xcd : r) + (blockIdx.x >> 3);
    int t, tg;
    part = div_known(lt, p.tilesM * p.tilesN, p.inv_tiles, t);
    const int first = div_known(t, 8 * p.tilesN, p.inv_group, tg) * 8;
    if (p.tilesM - first >= 8) {
      ti = first + (tg & 7);
      tj = tg >> 3;
    } else {
      int row;
      tj = div_known(tg, p.tilesM - first, p.inv_tail, row);
      ti = first + row;
    }
    part = __builtin_amdgcn_readfirstlane(part);
    ti = __builtin_amdgcn_readfirstlane(ti);
    tj = __builtin_amdgcn_readfirstlane(tj);
  }
  const int k_first = part * p.slabs * BK;
  const int k_left = p.K - k_first;  // > 0
  const int KT = min((k_left + BK - 1) / BK, p.slabs);

  // ---- global -> LDS: operand X is a tile of BM (BN) rows of 64, or (X K-major) of 64 rows of BM (BN); 16-byte chunk
  // j * NT + tid of it, in LDS order, comes from voff[j].  Rows along the reduction are 128 bytes: chunk c of row r lies at
  // c ^ (r / 2) % 8.  K-major rows: 64-byte group g of row r at g ^ r % 4, its 32-byte halves swapped where r / 8 is odd.
  // (K-major: chunks of the four loads lie 16 rows apart, added when they are issued, which leaves six registers more.)
  uint32_t voffP[PK ? 1 : 4], voffQ[QK ? 1 : 4];
  auto offsets = [&](uint32_t* v, bool kmajor, int width, int ld) {
    if (kmajor) {
      const int cpr = width / 8, row = tid / cpr, c = tid % cpr;
      const int chunk = (((c >> 2) ^ (row & 3)) << 2) | ((c & 3) ^ (((row >> 3) & 1) << 1));
      v[0] = (uint32_t)(row * ld + chunk * 8) * 2u;
    } else {
      const int row = tid >> 3, chunk = (tid & 7) ^ ((row >> 1) & 7);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (uint32_t)((row + j * (NT / 8)) * ld + chunk * 8) * 2u;
    }
  };
  static_assert(NT / (BM / 8) == 16, "a load brings 16 rows of a K-major tile");
  offsets(voffP, PK, BM, p.ldp);
  offsets(voffQ, QK, BN, p.ldq);
  // start of the tile's first slab, and bytes from there to the end of the matrix
  auto begin = [&](const bf16_t* base, bool kmajor, int extent, int at, int ld, const char*& from, int64_t& left) {
    const int64_t skip = kmajor ? (int64_t)k_first * ld + at : (int64_t)at * ld + k_first;
    // (rows are whole chunks)
    const int64_t all = kmajor ? (int64_t)(p.K - 1) * ld + ((extent + 7) & ~7) : (int64_t)(extent - 1) * ld + ((p.K + 7) & ~7);
    from = (const char*)(base + skip);
    left = (all - skip) * 2;
  };
  const char *nextP, *nextQ;
  int64_t leftP, leftQ;
  begin(p.P, PK, p.e.M, ti * BM, p.ldp, nextP, leftP);
  begin(p.Q, QK, p.e.N, tj * BN, p.ldq, nextQ, leftQ);
  const int64_t stepP = PK ? (int64_t)BK * p.ldp * 2 : BK * 2, stepQ = QK ? (int64_t)BK * p.ldq * 2 : BK * 2;
  int nxt = 0;  // the slab that is loaded next
  auto records = [&](int64_t left) -> int {
    // (slabs past the last one are loaded as zeros: the loop is two slabs long, and its waits count on every load)
    const int64_t n = nxt < KT && left > 0 ? (left < 0xfffffff0ll ? left : 0xfffffff0ll) : 0;
    return (int)(uint32_t)n;
  };
  int recsP, recsQ;
  auto prepare = [&]() {
    recsP = records(leftP);
    recsQ = records(leftQ);
    if ((!PK || !QK) && nxt == KT - 1 && (k_left & (BK - 1)) && k_left <= KT * BK) {
      // the reduction ends inside this slab
      const int in = k_left - nxt * BK;
      const int chunk = ((tid & 7) ^ ((tid >> 4) & 7)) * 8;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!PK && chunk >= in) voffP[PK ? 0 : j] = 0xfffffff0u;
        if (!QK && chunk >= in) voffQ[QK ? 0 : j] = 0xfffffff0u;
      }
    }
  };
  auto load = [&](int slot, int j) {
    const int jo = j & 3;
    uint32_t& own = j < 4 ? voffP[PK ? 0 : jo] : voffQ[QK ? 0 : jo];
    asm volatile("" : "+v"(own));  // (the sums below stay here instead of in registers of the whole loop)
    uint32_t v = own;
    if ((j < 4 ? PK : QK) && jo) v += (uint32_t)jo * (uint32_t)(32 * (j < 4 ? p.ldp : p.ldq));
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)(j < 4 ? nextP : nextQ), 0, j < 4 ? recsP : recsQ, 0x00020000);
    char* l = lds + (j < 4 ? 0 : 2 * OPB) + slot * OPB + (j & 3) * (NT * 16) + wave * (64 * 16);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LDS_PTR(l), 16, (int)v, 0, 0, 0);
  };
  auto loaded = [&]() {
    ++nxt;
    nextP += stepP;
    nextQ += stepQ;
    leftP -= stepP;
    leftQ -= stepQ;
    prepare();
  };
  prepare();

  // ---- LDS -> fragments: lane l holds row (column) l % 16 and reduction indices 8 (l / 16) .. + 7 of a 32-deep step
  const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)lds;
  const int l16 = lane & 15, quad = lane >> 4;
  uint32_t aoff[PK ? TM : ST], boff[QK ? TN : ST];
  auto kmajor_off = [&](int base, int width, int at, int f) {
    return lds_base + (uint32_t)(base + (8 * quad + (l16 >> 2)) * (width * 2) + ((((at + f * 16) >> 5) ^ (l16 >> 2)) << 6) +
                                 ((f ^ quad) & 1) * 32 + (l16 & 3) * 8);
  };
  auto row_off = [&](int base, int at, int st) {
    return lds_base + (uint32_t)(base + (at + l16) * (BK * 2) + ((st * 4 + quad) ^ (l16 >> 1)) * 16);
  };
#pragma unroll
  for (int f = 0; f < (PK ? TM : ST); ++f) aoff[f] = PK ? kmajor_off(0, BM, wm * Cfg::WTM, f) : row_off(0, wm * Cfg::WTM, f);
#pragma unroll
  for (int f = 0; f < (QK ? TN : ST); ++f)
    boff[f] = QK ? kmajor_off(2 * OPB, BN, wn * Cfg::WTN, f) : row_off(2 * OPB, wn * Cfg::WTN, f);

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  typedef LinSched<HALVES, ST, PK ? 2 : 1, QK ? 2 : 1> FS;
  typedef std::integral_constant<int, 0> ic0;
  bf16x8 fa[2][4], fb[2][TN];  // A by parity of the half, B by parity of the step
  auto read_a = [&](auto slotc, auto stc, auto setc, auto ic) {
    constexpr int slot = decltype(slotc)::value, st = decltype(stc)::value, i = decltype(ic)::value;
    bf16x8& dst = fa[decltype(setc)::value][i & 3];
    if constexpr (PK) lds_read_tr<slot * OPB + st * (32 * BM * 2), 4 * BM * 2>(dst, aoff[i]);
    else lds_read16<slot * OPB + i * (16 * BK * 2)>(dst, aoff[st]);
  };
  auto read_frag = [&](auto slotc, auto hnc, auto rc) {  // read r of those half hn of a slab needs
    constexpr int slot = decltype(slotc)::value, hn = decltype(hnc)::value, r = decltype(rc)::value;
    constexpr int st = hn / HALVES, part_ = hn % HALVES;
    typedef std::integral_constant<int, st> stc;
    typedef std::integral_constant<int, (hn & 1)> setc;
    if constexpr (part_ != 0) read_a(slotc, stc(), setc(), std::integral_constant<int, 4 + r>());
    else if constexpr (r == 0 || r > 4) read_a(slotc, stc(), setc(), std::integral_constant<int, (r == 0 ? 0 : r - 4)>());
    else if constexpr (QK) lds_read_tr<slot * OPB + st * (32 * BN * 2), 4 * BN * 2>(fb[st & 1][r - 1], boff[r - 1]);
    else lds_read16<slot * OPB + (r - 1) * (16 * BK * 2)>(fb[st & 1][r - 1], boff[st]);
  };

  // ---- slab 0, its first fragments, slab 1
#pragma unroll
  for (int j = 0; j < 8; ++j) load(0, j);
  loaded();
  pipeline_barrier<0>();
  static_for<0, 8>([&](auto rc) { read_frag(ic0(), ic0(), rc); });
#pragma unroll
  for (int j = 0; j < 8; ++j) load(1, j);
  loaded();
  __builtin_amdgcn_sched_barrier(0);
  for (int kt = 0; kt < KT; kt += 2) {
    static_for<0, 2 * HP>([&](auto shc) {
      constexpr int s = decltype(shc)::value / HP, hp = decltype(shc)::value % HP;
      constexpr int st = hp / HALVES, half = hp % HALVES;
      constexpr bool last = hp == HP - 1;
      if constexpr (last) pipeline_barrier<0>();  // the next slab has landed, this one is read: its slot is refilled
      static_for<0, 16>([&](auto qc) {
        constexpr int q = decltype(qc)::value, i = q / 4, j = q % 4;
        frag_wait<FS::allowed(hp, q)>(fa[hp & 1][i], fb[st & 1][j]);
        acc[half * 4 + i][j] =
            __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[st & 1][j], fa[hp & 1][i], acc[half * 4 + i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (FS::read_behind(hp, q) >= 0) {
          typedef std::integral_constant<int, FS::read_behind(hp, q)> rc;
          if constexpr (last) read_frag(std::integral_constant<int, s ^ 1>(), ic0(), rc());
          else read_frag(std::integral_constant<int, s>(), std::integral_constant<int, hp + 1>(), rc());
        }
        if constexpr (last && (q & 1)) load(s, q / 2);
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (last) loaded();
    });
  }
  wait_vmcnt<0>();
  // The reads behind the last half's MFMAs, which nobody uses, land before their registers are let go.
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int f = 0; f < 2; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      asm volatile("" ::"v"(fa[f][i]));
      asm volatile("" ::"v"(fb[f][i]));
    }

  // ---- element e of a lane: row l16, column 4 * quad + e of its 16 x 16 tile
  const int row0 = ti * BM + wm * Cfg::WTM + l16, col0 = tj * BN + wn * Cfg::WTN + 4 * quad;
  if constexpr (SPLIT) {
    float* out = p.part + (int64_t)part * p.e.M * p.e.N;
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
    if constexpr (ACT) {
      // Through the wavefront's eighth (quarter) of the ring, 64 rows at a time: sums [row][column], 16-byte chunk c of row r at
      // c ^ r % 16.  The activation then stands once in a loop of four rows a pass, not once for every accumulator,
      // and C, the addend and the slopes are moved in whole 128-byte lines.
      __syncthreads();  // every wavefront's loads have landed, and every fragment is read
      char* const mine = lds + wave * (64 * 64 * 4);
      static_assert(Cfg::LDS_BYTES >= Cfg::WM * Cfg::WN * 64 * 64 * 4, "staging");
      const int col = tj * BN + wn * Cfg::WTN + 4 * l16;
      const f32x4 b = bias4(p.e, col);
      static_for<0, TM / 4>([&](auto hc) {
        constexpr int h = decltype(hc)::value;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) *(f32x4*)(mine + (i * 16 + l16) * 256 + ((4 * j + quad) ^ l16) * 16) = acc[h * 4 + i][j];
        asm volatile("" ::: "memory");
        const int row_h = ti * BM + wm * Cfg::WTM + h * 64 + quad;
        uint2 r = residual4(p.e, row_h, col);
#pragma unroll 1
        for (int t = 0; t < 16; ++t) {
          const int lr = t * 4 + quad;
          const f32x4 z = *(const f32x4*)(mine + lr * 256 + ((l16 ^ (lr & 15)) * 16));
          const uint2 rn = t < 15 ? residual4(p.e, row_h + t * 4 + 4, col) : make_uint2(0, 0);
          finish4<true>(p.e, row_h + t * 4, col, z, b, r);
          r = rn;
        }
        asm volatile("" ::: "memory");
      });
    } else {
      f32x4 b[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) b[j] = bias4(p.e, col0 + j * 16);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        uint2 r[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) r[j] = residual4(p.e, row0 + i * 16, col0 + j * 16);
#pragma unroll
        for (int j = 0; j < TN; ++j) finish4<false>(p.e, row0 + i * 16, col0 + j * 16, acc[i][j], b[j], r[j]);
        asm volatile("" ::: "memory");
      }
    }
  }
}

// Adds the parts of a split reduction, in their order, and finishes: four elements per thread.
template <bool ACT>
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
    finish4<ACT>(p, row, col, s, bias4(p, col), residual4(p, row, col));
  }
}

// ---------------------------------------------------------------------------------------------- few tokens
// Up to 64 rows of x: the weight is read once and nothing else counts.  A workgroup takes 16 rows of W, its wavefronts an
// equal run of the reduction each; fragments go from memory to registers with no LDS between (a lane's chunk is its MFMA operand
// as it lies), eight loads of W in flight per wavefront.  MFMA row: a row of W; column: a token (past the last one, the
// last one again).  The wavefronts' sums meet in LDS and are added in their order.
template <int TB, int WAVES, bool ACT>
__global__ __launch_bounds__(WAVES * 64) void lin_few_kernel(const LinEpilogue p, const bf16_t* __restrict__ x, int64_t ldx,
                                                             const bf16_t* __restrict__ w, int64_t ldw, int K) {
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
  constexpr int U = 8;
  int s = s0;
  for (; s + U <= s1 && (s + U) * 32 <= K; s += U) {
    bf16x8 fw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) fw[u] = *(const bf16x8*)(wp + (s + u) * 32);
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      bf16x8 fx[U];
#pragma unroll
      for (int u = 0; u < U; ++u) fx[u] = *(const bf16x8*)(xp[b] + (s + u) * 32);
#pragma unroll
      for (int u = 0; u < U; ++u) acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[u], fx[u], acc[b], 0, 0, 0);
    }
  }
  for (; s < s1; ++s) {
    const bool in = s * 32 + quad * 8 < K;
    const bf16x8 zero = {};
    const bf16x8 fw = in ? *(const bf16x8*)(wp + s * 32) : zero;
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      const bf16x8 fx = in ? *(const bf16x8*)(xp[b] + s * 32) : zero;
      acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw, fx, acc[b], 0, 0, 0);
    }
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
    finish4<ACT>(p, row, col, t, bias4(p, col), residual4(p, row, col));
  }
}

// ---------------------------------------------------------------------------------------------- operands and column sums
constexpr int kPrepCols = 256;  // columns of a workgroup: 32 threads of eight, by eight rows

int lin_sum_parts(int rows) {
  const int per = rows <= 8192 ? 64 : (rows + 1023) / 1024 * 8;  // rows of a part, a multiple of eight
  return (rows + per - 1) / per;
}

// SLOPE: src is dy, and dz = dy * act'(z) goes on.  VEC: rows of src, slope and dst are whole 16-byte chunks.
template <bool SLOPE, bool DST, bool SUM, bool VEC>
__global__ __launch_bounds__(256) void lin_prepare_kernel(const bf16_t* __restrict__ src, int64_t ld,
                                                          const uint16_t* __restrict__ slope, int act, int rows, int cols,
                                                          bf16_t* __restrict__ dst, float* __restrict__ partial, int per) {
  __shared__ float sums[8][kPrepCols];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c0 = blockIdx.x * kPrepCols + tx * 8, padded = (cols + 7) & ~7;
  const int r_first = blockIdx.y * per, r_end = r_first + per < rows ? r_first + per : rows;
  float acc[8] = {};
  if (c0 < cols) {
    for (int r = r_first + ty; r < r_end; r += 8) {
      float v[8];
      if constexpr (VEC) {
        st_load8<bf16_t>(src + (int64_t)r * ld + c0, 0, v);
        if constexpr (SLOPE) {
          const u32x4_t s = *(const u32x4_t*)(slope + (int64_t)r * cols + c0);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= slope_unpack(act, (uint16_t)(s[e >> 1] >> (16 * (e & 1))));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = c0 + e < cols ? bf16_to_f32(src[(int64_t)r * ld + c0 + e]) : 0.f;
          if constexpr (SLOPE)
            if (c0 + e < cols) v[e] *= slope_unpack(act, slope[(int64_t)r * cols + c0 + e]);
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

// out[c] = sum of partial[0 .. parts)[c]: 64 columns of a workgroup, four threads a column.
__global__ __launch_bounds__(256) void lin_sum_kernel(const float* __restrict__ partial, int parts, int cols, void* out,
                                                      int out_dtype) {
  __shared__ float sums[4][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), g = threadIdx.x >> 6;
  float s = 0.f;
  if (c < cols)
    for (int k = g; k < parts; k += 4) s += partial[(int64_t)k * cols + c];
  sums[g][threadIdx.x & 63] = s;
  __syncthreads();
  if (g == 0 && c < cols) {
    s = (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
    if (out_dtype) ((float*)out)[c] = s;
    else ((bf16_t*)out)[c] = f32_to_bf16(s);
  }
}

// ---------------------------------------------------------------------------------------------- host
// How a product runs: on which tiles, and in how many parts of the reduction.
struct LinPlan {
  int edge;    // 256, 128, or 0: lin_few_kernel
  int splits, slabs;
};
static LinPlan lin_plan(int M, int N, int K, int p_kmajor, int q_kmajor) {
  if (M <= 64 && !p_kmajor && !q_kmajor) return {0, 1, 0};
  const int KT = (K + 63) / 64;
  LinPlan best{128, 1, KT};
  double least = 1e30;
  for (int edge = 128; edge <= 256; edge += 128) {
    const int64_t tiles = (int64_t)((M + edge - 1) / edge) * ((N + edge - 1) / edge);
    for (int s = 1; s <= 16 && s <= KT; ++s) {
      const int slabs = ((KT + s - 1) / s + 1) & ~1;
      const int parts = (KT + slabs - 1) / slabs;
      if (parts != s) continue;
      const int64_t wgs = tiles * parts;
      double us;
      if (edge == 256) us = (double)((wgs + 255) / 256) * (slabs * 1.3 + 4.0);
      else us = wgs <= 256 ? slabs * 0.4 + 3.0 : (double)((wgs + 511) / 512) * (slabs * 0.65 + 4.0);
      if (parts > 1) us += 3.0 + (double)M * N * parts * 8.0 / 4e6;
      if (us < least) {
        least = us;
        best = {edge, parts, slabs};
      }
    }
  }
  return best;
}

size_t lin_product_scratch(int M, int N, int K, int p_kmajor, int q_kmajor) {
  const LinPlan plan = lin_plan(M, N, K, p_kmajor, q_kmajor);
  return plan.splits > 1 ? (size_t)plan.splits * M * N * sizeof(float) : 0;
}

template <class Cfg, bool PK, bool QK, bool ACT, bool SPLIT>
static hipError_t launch_tile(const LinTileParams& tp, hipStream_t st) {
  static std::atomic<uint64_t> attr_done{0};
  auto kern = lin_tile_kernel<Cfg, PK, QK, ACT, SPLIT>;
  if (hipError_t e = set_max_dynamic_lds_once((const void*)kern, Cfg::LDS_BYTES, attr_done)) return e;
  const int64_t total = (int64_t)tp.tilesM * tp.tilesN * tp.splits;
  if (total > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kern, dim3((unsigned)total), dim3(Cfg::NT), Cfg::LDS_BYTES, st, tp);
  return hipGetLastError();
}

template <class Cfg>
static hipError_t launch_tiles(const LinProduct& p, LinTileParams tp, hipStream_t st) {
  tp.tilesM = (p.M + Cfg::BM - 1) / Cfg::BM;
  tp.tilesN = (p.N + Cfg::BN - 1) / Cfg::BN;
  if ((int64_t)tp.tilesM * tp.tilesN > 0x7fffffff || (int64_t)tp.tilesN * 8 > 0x7fffffff) return hipErrorInvalidValue;
  tp.inv_tiles = (uint32_t)(0xffffffffu / ((int64_t)tp.tilesM * tp.tilesN));
  tp.inv_group = (uint32_t)(0xffffffffu / (8 * (int64_t)tp.tilesN));
  tp.inv_tail = tp.tilesM % 8 ? 0xffffffffu / (tp.tilesM % 8) : 0;
  const bool act = tp.e.act != kActNone, split = tp.splits > 1;
  if (!p.p_kmajor && !p.q_kmajor) {
    if (split) return launch_tile<Cfg, false, false, false, true>(tp, st);
    return act ? launch_tile<Cfg, false, false, true, false>(tp, st) : launch_tile<Cfg, false, false, false, false>(tp, st);
  }
  if (!p.p_kmajor) {
    return split ? launch_tile<Cfg, false, true, false, true>(tp, st) : launch_tile<Cfg, false, true, false, false>(tp, st);
  }
  return split ? launch_tile<Cfg, true, true, false, true>(tp, st) : launch_tile<Cfg, true, true, false, false>(tp, st);
}

template <int TB, int WAVES>
static hipError_t launch_few(const LinProduct& p, const LinEpilogue& e, hipStream_t st) {
  const dim3 grid((unsigned)((p.N + 15) / 16)), block(WAVES * 64);
  if (e.act != kActNone) hipLaunchKernelGGL((lin_few_kernel<TB, WAVES, true>), grid, block, 0, st, e, p.P, p.ldp, p.Q, p.ldq, p.K);
  else hipLaunchKernelGGL((lin_few_kernel<TB, WAVES, false>), grid, block, 0, st, e, p.P, p.ldp, p.Q, p.ldq, p.K);
  return hipGetLastError();
}

hipError_t launch_lin_product(const LinProduct& p, hipStream_t st) {
  if (p.M <= 0 || p.N <= 0 || p.K <= 0) return hipErrorInvalidValue;
  auto whole = [](const void* ptr, int64_t ld, int extent) {
    return ((uint64_t)ptr & 15) == 0 && ld % 8 == 0 && ld >= ((extent + 7) & ~7) && ld <= kLinMaxLd;
  };
  if (!whole(p.P, p.ldp, p.p_kmajor ? p.M : p.K) || !whole(p.Q, p.ldq, p.q_kmajor ? p.N : p.K)) return hipErrorInvalidValue;
  if ((p.p_kmajor && !p.q_kmajor) || (p.act != kActNone && p.q_kmajor)) return hipErrorInvalidValue;
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
  e.vec = p.N % 4 == 0 && (((uint64_t)p.C | (uint64_t)p.slope | (uint64_t)p.R) & 7) == 0 && (!p.R || p.ldr % 4 == 0);
  const LinPlan plan = lin_plan(p.M, p.N, p.K, p.p_kmajor, p.q_kmajor);
  if (plan.edge == 0) {
    // sixteen wavefronts share a reduction where the rows of W alone do not fill the chip
    const bool wide = (p.N + 15) / 16 < 1024;
    if (p.M <= 16) return wide ? launch_few<1, 16>(p, e, st) : launch_few<1, 4>(p, e, st);
    if (p.M <= 32) return wide ? launch_few<2, 16>(p, e, st) : launch_few<2, 4>(p, e, st);
    return wide ? launch_few<4, 8>(p, e, st) : launch_few<4, 4>(p, e, st);
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
  if (hipError_t err = plan.edge == 256 ? launch_tiles<Lin256>(p, tp, st) : launch_tiles<Lin128>(p, tp, st)) return err;
  if (plan.splits > 1) {
    const int64_t wg = ((int64_t)p.M * ((p.N + 3) / 4) + 255) / 256;
    const dim3 grid((unsigned)(wg < 65536 ? wg : 65536));
    if (e.act != kActNone) hipLaunchKernelGGL((lin_join_kernel<true>), grid, dim3(256), 0, st, e, p.scratch, plan.splits);
    else hipLaunchKernelGGL((lin_join_kernel<false>), grid, dim3(256), 0, st, e, p.scratch, plan.splits);
  }
  return hipGetLastError();
}

template <bool SLOPE, bool DST, bool SUM>
static hipError_t launch_prepare(const bf16_t* src, int64_t ld, const uint16_t* slope, int act, int rows, int cols, bf16_t* dst,
                                 float* partial, hipStream_t st) {
  const int parts = lin_sum_parts(rows);
  int per = (rows + parts - 1) / parts;
  per = (per + 7) & ~7;
  const dim3 grid((cols + kPrepCols - 1) / kPrepCols, parts);
  const bool vec = cols % 8 == 0 && ld % 8 == 0 && (((uint64_t)src | (uint64_t)slope | (uint64_t)dst) & 15) == 0;
  if (vec) hipLaunchKernelGGL((lin_prepare_kernel<SLOPE, DST, SUM, true>), grid, dim3(256), 0, st, src, ld, slope, act, rows, cols, dst, partial, per);
  else hipLaunchKernelGGL((lin_prepare_kernel<SLOPE, DST, SUM, false>), grid, dim3(256), 0, st, src, ld, slope, act, rows, cols, dst, partial, per);
  return hipGetLastError();
}

hipError_t launch_lin_prepare(const bf16_t* src, int64_t ld, const uint16_t* slope, int act, int rows, int cols, bf16_t* dst,
                              float* partial, hipStream_t st) {
  if (rows <= 0 || cols <= 0 || (!dst && !partial) || (dst && ((uint64_t)dst & 15))) return hipErrorInvalidValue;
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
  hipLaunchKernelGGL(lin_sum_kernel, dim3((cols + 63) / 64), dim3(256), 0, st, partial, parts, cols, out, out_dtype);
  return hipGetLastError();
}

}  // namespace dion
