// Multi-tensor AdamW whose first and second moments are kept in 8 bits, and the values such codes stand for.
//
// State of a tensor, in blocks of 128 consecutive elements (the last one may be shorter):
//   M  int8 codes c,  one fp32 scale s per block:  m = c s,      s = max |m| / 127
//   V  uint8 codes k, one fp32 scale q per block:  v = (k q)^2,  q = max sqrt(v) / 255
// V's codes are linear in sqrt(v), the quantity the update divides by: the root that the denominator needs is the one
// that is coded, and a block holds second moments down to 1 / 65025 of its largest.  Arithmetic between reading and writing
// the codes is fp32 with fused multiply-adds; root and quotient are the hardware's (1 ulp each).
//
// Rounding to a code is up or down at random, unbiased in m and in v:  c = floor(m / s + u),  k = floor(t) or one more
// with probability (t^2 - floor(t)^2) / (2 floor(t) + 1), t = sqrt(v) / q.  A step without a gradient takes 1 - beta2 off v, and half a
// code is 1 / k of v at code k: rounded to nearest, v would stand still at codes below 1 / (1 - beta2), which is 20 for beta2 = 0.95,
// 100 for 0.99 and all of them from 0.9961 on.  u in [0, 1) comes from a hash of (seed, step counter, element / 8), spread over the eight elements by a
// Weyl sequence: the noise of an element is independent from step to step, and a run repeats bit for bit.
// m / s + u is a sum in fp32, exact for m = 0; beside a code of 64 and more 17 of u's 24 bits count (a mean off by 2^-18 of a code).
// A second moment above zero (the normal numbers of fp32) keeps a code of at least 1, and beside one of zero the first moment is
// dropped: no first moment may be divided by epsilon alone in a later step.  First moments of a block whose largest is below 1e-30
// are dropped too (127 / max would overflow).  A block with a value that is not finite gets a scale of NaN, so that it shows in
// every later step.
//
// Bound by HBM: fp32 parameters, bf16 gradients 14.1 bytes per element (26 with fp32 states): X both ways 8, G 2, codes 4,
// scales 0.125. That leaves about a hundred vector instructions an element (seventy with bf16 parameters), which a plain
// translation of the formulas takes up. us of the update alone, 2 x (50304 x 768) with fp32 parameters and bf16 gradients / 2 x
// (32000 x 4096) in fp32 / 2 x (32003 x 1001) in bf16, cautious: that translation 259 / 885 / 205; half the vector instructions
// (packed conversions, clamps by medians, the hardware's root and quotient) 212 / 810 / 130; two rounds a workgroup past the
// caches 203 / 780 / 129. Codes whose offset is added behind the rounding, and none beside v = 0: 205 / 789 / 130, which is 5.3, 5.4
// and 5.0 TB/s (the third is half in the caches).
#include "elementwise.h"

namespace dion {

constexpr int kA8Round = 2048;  // elements of a round of a workgroup: eight per thread

struct Adam8Tensors {
  uint64_t x[kMtaTensors], g[kMtaTensors], m[kMtaTensors], v[kMtaTensors], ms[kMtaTensors], vs[kMtaTensors],
      step[kMtaTensors];
  int64_t numel[kMtaTensors];
  unsigned wg0[kMtaTensors + 1];  // first workgroup of each tensor; wg0[n] = workgroups of the launch
  int rounds;                     // of kA8Round elements per workgroup
};

struct Adam8Scalars {
  float beta1, beta2, eps, wd_host;
  uint32_t seed;
};

// A 32-bit number from a 32-bit number: shifts and odd multipliers (the first bits behind the point of sqrt 2 and sqrt 3).
static __device__ __forceinline__ uint32_t mix32(uint32_t h) {
  h ^= h >> 16;
  h *= 0x6A09E667u;
  h ^= h >> 15;
  h *= 0xBB67AE85u;
  return h ^ (h >> 16);
}

// step[t] += 1 for every distinct counter of the launch (before the update kernel reads them).
__global__ void adamw8_advance_steps_kernel(Adam8Tensors a, int n) {
  const int t = threadIdx.x;
  const uint64_t mine = t < n ? a.step[t] : 0;
  bool first = t < n;
  for (int u = 0; u + 1 < n; ++u) first = first && (u >= t || a.step[u] != mine);
  if (first) *(float*)mine = *(float*)mine + 1.0f;
}

// Largest over the 16 lanes of a block, in all of them.  Magnitudes as bits: ordered like the values, with infinity and NaN
// above every number.
template <int N>
static __device__ __forceinline__ uint32_t row_ror(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xf, 0xf, false);
}
static __device__ __forceinline__ uint32_t block_max(uint32_t v) {
  v = max(v, row_ror<8>(v));
  v = max(v, row_ror<4>(v));
  v = max(v, row_ror<2>(v));
  return max(v, row_ror<1>(v));
}

// Scale of a block whose largest magnitude is `top` on codes up to LAST, and its inverse.
static __device__ __forceinline__ void block_scale(uint32_t top_bits, float last, float& inv, float& scale) {
  const float top = __uint_as_float(top_bits);
  const bool held = top >= 1e-30f, finite = top_bits < 0x7f800000u;
  inv = held && finite ? last / top : 0.0f;
  scale = !finite ? __uint_as_float(0x7fc00000u) : held ? top / last : 0.0f;
}

// What a thread reads of its eight elements, as it lies in memory.
template <typename T>
struct Raw8 {
  u32x4_t w[sizeof(T) / 2];
};
template <typename T, bool NT>
static __device__ __forceinline__ void raw_load(const T* p, int64_t i, Raw8<T>& r) {
#pragma unroll
  for (int k = 0; k < (int)sizeof(T) / 2; ++k) {
    const u32x4_t* q = (const u32x4_t*)(p + i) + k;
    if constexpr (NT) r.w[k] = __builtin_nontemporal_load(q);
    else r.w[k] = *q;
  }
}
template <typename T>
static __device__ __forceinline__ void raw_values(const Raw8<T>& r, float v[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (sizeof(T) == 4) v[e] = __uint_as_float(r.w[e >> 2][e & 3]);
    else v[e] = __uint_as_float((e & 1) ? (r.w[0][e >> 1] & 0xffff0000u) : (r.w[0][e >> 1] << 16));
  }
}

template <typename GT, typename XT, bool NT, bool CAUTIOUS>
__global__ __launch_bounds__(256) void adamw8_kernel(Adam8Tensors a, int n, const float* __restrict__ lr_dev,
                                                     const float* __restrict__ wd_dev, Adam8Scalars sc) {
  int t = 0;
  for (int hi = n; hi - t > 1;) {  // the tensor of this workgroup
    const int mid = (t + hi) >> 1;
    if (a.wg0[mid] <= blockIdx.x) t = mid;
    else hi = mid;
  }
  const int64_t first = (int64_t)(blockIdx.x - a.wg0[t]) * a.rounds * kA8Round;
  const int64_t numel = a.numel[t];
  XT* __restrict__ x = (XT*)a.x[t];
  const GT* __restrict__ g = (const GT*)a.g[t];
  int8_t* __restrict__ m = (int8_t*)a.m[t];
  uint8_t* __restrict__ v = (uint8_t*)a.v[t];
  float* __restrict__ ms = (float*)a.ms[t];
  float* __restrict__ vs = (float*)a.vs[t];
  const bool vec = (((a.x[t] | a.g[t]) & 15) | ((a.m[t] | a.v[t]) & 7)) == 0;

  Raw8<XT> xr;
  Raw8<GT> gr;
  u32x2_t mr, vr;
  float s_old = 0.f, q_old = 0.f;
  auto fetch = [&](int64_t e0) {
    if (e0 >= numel) {  // (the last round's scales, which may be NaN, are another block's)
      s_old = q_old = 0.f;
      return;
    }
    s_old = ms[e0 >> 7];
    q_old = vs[e0 >> 7];
    if (!vec || e0 + 8 > numel) return;
    raw_load<XT, NT>(x, e0, xr);
    raw_load<GT, NT>(g, e0, gr);
    if constexpr (NT) {
      mr = __builtin_nontemporal_load((const u32x2_t*)(m + e0));
      vr = __builtin_nontemporal_load((const u32x2_t*)(v + e0));
    } else {
      mr = *(const u32x2_t*)(m + e0);
      vr = *(const u32x2_t*)(v + e0);
    }
  };
  int64_t e0 = first + threadIdx.x * 8;
  fetch(e0);
  // the scalars of the step, under the first loads
  const float step = *(const float*)a.step[t];
  const float lr = *lr_dev;
  const float wd = wd_dev ? *wd_dev : sc.wd_host;
  const float inv_bc2_sqrt = 1.0f / sqrtf(1.0f - powf(sc.beta2, step));
  const float adj_lr = lr / (1.0f - powf(sc.beta1, step));
  const float coeff = lr * wd, keep = 1.0f - coeff;
  const uint32_t key = mix32(mix32(sc.seed) + (uint32_t)step);

  const float w1 = 1.0f - sc.beta1, w2 = 1.0f - sc.beta2;
  for (int r = 0; r < a.rounds; ++r, e0 += kA8Round) {
    if (first + (int64_t)r * kA8Round >= numel) break;  // (the same for the whole workgroup)
    const int left = numel - e0 >= 8 ? 8 : numel > e0 ? (int)(numel - e0) : 0;
    const bool whole = vec && left == 8;
    float xv[8], gv[8];
    u32x2_t mb, vb;  // codes, first moments' plus 128
    const float s = s_old, s128 = -128.0f * s_old, q = q_old;
    if (whole) {
      raw_values<XT>(xr, xv);
      raw_values<GT>(gr, gv);
      mb = mr ^ 0x80808080u;
      vb = vr;
    } else {
      // (zeros where the tensor has ended, which change nothing)
      mb = u32x2_t{0x80808080u, 0x80808080u};
      vb = u32x2_t{0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = e < left;
        xv[e] = in ? st_load<XT>(x, e0 + e) : 0.f;
        gv[e] = in ? st_load<GT>(g, e0 + e) : 0.f;
        if (in) {
          mb[e >> 2] ^= (uint32_t)(uint8_t)m[e0 + e] << (8 * (e & 3));
          vb[e >> 2] |= (uint32_t)v[e0 + e] << (8 * (e & 3));
        }
      }
    }
    if (r + 1 < a.rounds) fetch(e0 + kA8Round);
    float mv[8], rt[8];
    uint32_t mtop = 0, rtop = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float m0 = fmaf((float)((mb[e >> 2] >> (8 * (e & 3))) & 0xffu), s, s128);
      const float r0 = (float)((vb[e >> 2] >> (8 * (e & 3))) & 0xffu) * q;
      mv[e] = fmaf(w1, gv[e] - m0, m0);
      rt[e] = __builtin_amdgcn_sqrtf(fmaf(w2 * gv[e], gv[e], r0 * r0 * sc.beta2));
      const float upd = mv[e] * __builtin_amdgcn_rcpf(fmaf(rt[e], inv_bc2_sqrt, sc.eps));
      if constexpr (CAUTIOUS) xv[e] = upd * xv[e] >= 0.0f ? fmaf(-coeff, xv[e], xv[e]) : xv[e];
      else xv[e] *= keep;
      xv[e] = fmaf(-adj_lr, upd, xv[e]);
      mtop = max(mtop, __float_as_uint(mv[e]) & 0x7fffffffu);
      rtop = max(rtop, __float_as_uint(rt[e]));
    }
    float minv, mscale, rinv, rscale;
    block_scale(block_max(mtop), 127.0f, minv, mscale);
    block_scale(block_max(rtop), 255.0f, rinv, rscale);
    const uint32_t h = mix32(key ^ (uint32_t)(e0 >> 3));
    u32x2_t mo = {0, 0}, vo = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = (float)((h + (uint32_t)e * 0x9E3779B9u) >> 8) * 0x1p-24f;
      const float least = __builtin_amdgcn_fmed3f(rt[e] * 0x1p127f, 0.0f, 1.0f);  // 1 where v > 0, else 0
      // (a scale of zero or NaN has an inverse of zero; 128 is added to the code, where it is exact: added to u it would round
      // the last of u's values up to a code of 1 for m = 0)
      const float c = fmaf(floorf(fmaf(mv[e], minv, u)), least, 128.0f);
      mo[e >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_amdgcn_fmed3f(c, 1.0f, 255.0f), e & 3, mo[e >> 2]);
      const float t = rt[e] * rinv, k = floorf(t);
      const float up = fmaf(u, fmaf(2.0f, k, 1.0f), k * k) < t * t ? k + 1.0f : k;
      vo[e >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_amdgcn_fmed3f(up, least, 255.0f), e & 3, vo[e >> 2]);
    }
    mo ^= 0x80808080u;
    if (left > 0 && (threadIdx.x & 15) == 0) {
      ms[e0 >> 7] = mscale;
      vs[e0 >> 7] = rscale;
    }
    if (whole) {
      st_store8<XT, NT>(x + e0, 0, xv);
      if constexpr (NT) {
        __builtin_nontemporal_store(mo, (u32x2_t*)(m + e0));
        __builtin_nontemporal_store(vo, (u32x2_t*)(v + e0));
      } else {
        *(u32x2_t*)(m + e0) = mo;
        *(u32x2_t*)(v + e0) = vo;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e >= left) continue;
        st_store<XT>(x, e0 + e, xv[e]);
        m[e0 + e] = (int8_t)(mo[e >> 2] >> (8 * (e & 3)));
        v[e0 + e] = (uint8_t)(vo[e >> 2] >> (8 * (e & 3)));
      }
    }
  }
}

// The values of codes: eight per thread.  2 x (50304 x 768) to bf16 41 us (5.6 TB/s), 2 x (32000 x 4096) 136 us (5.8).
template <typename OT, bool SQ, bool NT>
__global__ __launch_bounds__(256) void state8_values_kernel(const uint8_t* __restrict__ codes,
                                                            const float* __restrict__ scales, int64_t numel,
                                                            OT* __restrict__ out) {
  const bool vec = (((uint64_t)codes & 7) | ((uint64_t)out & 15)) == 0;
  const int64_t stride = (int64_t)gridDim.x * kA8Round;
  for (int64_t e0 = (int64_t)blockIdx.x * kA8Round + threadIdx.x * 8; e0 < numel; e0 += stride) {
    const float s = scales[e0 >> 7];
    const bool whole = vec && e0 + 8 <= numel;
    u32x2_t raw = {0, 0};
    if (whole) {
      if constexpr (NT) raw = __builtin_nontemporal_load((const u32x2_t*)(codes + e0));
      else raw = *(const u32x2_t*)(codes + e0);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e0 + e < numel) raw[e >> 2] |= (uint32_t)codes[e0 + e] << (8 * (e & 3));
    }
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t b = raw[e >> 2] >> (8 * (e & 3));
      const float w = (SQ ? (float)(uint8_t)b : (float)(int8_t)b) * s;
      o[e] = SQ ? w * w : w;
    }
    if (whole) {
      st_store8<OT, NT>(out + e0, 0, o);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e0 + e < numel) st_store<OT>(out, e0 + e, o[e]);
    }
  }
}

hipError_t launch_adamw8(const uint64_t* X, int x_dtype, const uint64_t* G, int g_dtype, const uint64_t* M,
                         const uint64_t* MS, const uint64_t* V, const uint64_t* VS, const uint64_t* steps,
                         const int64_t* numel, int n, const float* lr_dev, float beta1, float beta2, float eps,
                         const float* wd_dev, float wd_host, int cautious, uint32_t seed, hipStream_t st) {
  Adam8Tensors a;
  int64_t total = 0;
  for (int i = 0; i < n; ++i) total += numel[i];
  const bool nt = exceeds_caches(total * (2 + (x_dtype == 0 ? 2 : 4) + (g_dtype == 0 ? 2 : 4)));
  // us with 1 / 2 / 4 / 8 rounds: past the caches 2 x (50304 x 768) fp32 241 / 205 / 212 / 224, 2 x (32000 x 4096) 837 / 782 / 810 /
  // 845; within them 2 x (32003 x 1001) bf16 146 / 140 / 130 / 133.
  a.rounds = total < (4 << 20) ? 1 : nt ? 2 : 4;
  int64_t wg = 0;
  for (int i = 0; i < kMtaTensors; ++i) {
    const int j = i < n ? i : 0;
    a.x[i] = X[j];
    a.g[i] = G[j];
    a.m[i] = M[j];
    a.v[i] = V[j];
    a.ms[i] = MS[j];
    a.vs[i] = VS[j];
    a.step[i] = steps[j];
    a.numel[i] = i < n ? numel[j] : 0;
    a.wg0[i] = (unsigned)wg;
    if (i < n) wg += (numel[i] + (int64_t)a.rounds * kA8Round - 1) / ((int64_t)a.rounds * kA8Round);
    if (wg > 0x7fffffff) return hipErrorInvalidValue;
  }
  a.wg0[kMtaTensors] = (unsigned)wg;
  hipLaunchKernelGGL(adamw8_advance_steps_kernel, dim3(1), dim3(64), 0, st, a, n);
  if (wg == 0) return hipGetLastError();
  const Adam8Scalars sc{beta1, beta2, eps, wd_host, seed};
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)wg), dim3(256), 0, st, a, n, lr_dev, wd_dev, sc); };
#define A8_LAUNCH(GT, XT)                                                                                              \
  do {                                                                                                                 \
    if (cautious) nt ? launch(adamw8_kernel<GT, XT, true, true>) : launch(adamw8_kernel<GT, XT, false, true>);         \
    else nt ? launch(adamw8_kernel<GT, XT, true, false>) : launch(adamw8_kernel<GT, XT, false, false>);                \
  } while (0)
  if (g_dtype == 0) {
    if (x_dtype == 0) A8_LAUNCH(bf16_t, bf16_t); else A8_LAUNCH(bf16_t, float);
  } else {
    if (x_dtype == 0) A8_LAUNCH(float, bf16_t); else A8_LAUNCH(float, float);
  }
#undef A8_LAUNCH
  return hipGetLastError();
}

hipError_t launch_state8_values(const void* codes, int squared, const float* scales, int64_t numel, void* out,
                                int out_dtype, hipStream_t st) {
  if (numel == 0) return hipSuccess;
  const int64_t wg = (numel + kA8Round - 1) / kA8Round;
  const unsigned grid = (unsigned)(wg < (1 << 20) ? wg : (1 << 20));
  const bool nt = exceeds_caches(numel * (out_dtype == 0 ? 3 : 5));
#define S8_LAUNCH(OT, SQ)                                                                                              \
  do {                                                                                                                 \
    if (nt) hipLaunchKernelGGL((state8_values_kernel<OT, SQ, true>), dim3(grid), dim3(256), 0, st, (const uint8_t*)codes, scales, numel, (OT*)out); \
    else hipLaunchKernelGGL((state8_values_kernel<OT, SQ, false>), dim3(grid), dim3(256), 0, st, (const uint8_t*)codes, scales, numel, (OT*)out);   \
  } while (0)
  if (out_dtype == 0) {
    if (squared) S8_LAUNCH(bf16_t, true); else S8_LAUNCH(bf16_t, false);
  } else {
    if (squared) S8_LAUNCH(float, true); else S8_LAUNCH(float, false);
  }
#undef S8_LAUNCH
  return hipGetLastError();
}

}  // namespace dion
