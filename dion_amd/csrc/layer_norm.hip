// Layer norm of rows of x:  m = mean x,  r = 1 / sqrt(mean (x - m)^2 + eps),  xh = (x - m) r,  y = xh w + b,
// and its gradients, with g = dy w:  dx = r (g - mean g - xh mean(g xh)),  dw = sum over the rows of dy xh,  db = of dy.
// Rows stay in registers between the two sums of a pass (the variance is that of the centred values: no difference of large
// numbers), so x and dy are read once.  Sums fp32, in an order that depends on the sizes alone.  Bound by HBM.  us, bf16: 16384 x 4096
// forward 56 (4.8 TB/s), backward 69 (5.8) and 4 for the sums over the workgroups; 65536 x 768 43 and 53; one row of 768 2.3, a launch
// and one way to memory.  Not at both ends: the backward pass of 8193 to 16384 columns, with sixteen elements of five arrays a thread,
// sends 23 to 97 of its registers through scratch memory (52 to 172 bytes a lane), 4096 x 16384 66 and 109 where its bytes take 56 and 84; and
// rows of 64 or 128 columns leave most of a wavefront idle, 2^20 of 64 286 and 258 where their bytes take 56 and 84.
#include "layers.h"
#include "linear.h"

namespace dion {

constexpr int kNormWide = 16384;  // columns past which a row is read again instead of kept

// Weight or bias of the V columns from c on; `none` without.
template <int V>
static __device__ __forceinline__ void param(const void* p, int dtype, int c, bool in, float none, float* v) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = none;
  } else if (dtype) {
    Piece<float, V> q;
    q.load((const float*)p, c, in);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = q.get(e);
  } else {
    Piece<bf16_t, V> q;
    q.load((const bf16_t*)p, c, in);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = q.get(e);
  }
}

// The sum of v over the G threads of a row; `at`: LDS of the row's wavefronts that nothing else uses before the next barrier but one.
template <int G>
static __device__ __forceinline__ float row_sum(float v, float* at) {
  v = wave_sum(v);
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) at[(threadIdx.x % G) >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int k = 0; k < G / 64; ++k) v += at[k];
  }
  return v;
}

// A row by G threads of E elements each: elements (c G + t) V .. + V - 1 are chunk c of thread t.
template <typename TX, typename TY, int G, int E, int V, bool PAST>
__global__ __launch_bounds__(G < 256 ? 256 : G) void norm_forward_kernel(const NormArgs a) {
  constexpr int NC = E / V, ROWS = (G < 256 ? 256 : G) / G;
  __shared__ float sums[2][G / 64 + 1];
  const int t = threadIdx.x % G;
  const int row = blockIdx.x * ROWS + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / (G / 64);
  if (row >= a.rows) return;  // (whole wavefronts; of a workgroup of one row none)
  const TX* x = (const TX*)a.x + (int64_t)row * a.ldx;
  Piece<TX, V> px[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) px[c].load(x, (c * G + t) * V, (c * G + t) * V < a.width);
  float s = 0.f;  // (E values of x stay as they were read: sixteen bits each, where x is bf16)
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) s += px[c].get(e);
  const float n = 1.f / (float)a.width, mean = row_sum<G>(s, sums[0]) * n;
  s = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = px[c].get(e) - mean;
      s = (c * G + t) * V < a.width ? fmaf(d, d, s) : s;
    }
  const float rstd = 1.f / sqrtf(row_sum<G>(s, sums[1]) * n + a.eps);
  if (t == 0 && a.mean) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  TY* y = (TY*)a.y + (int64_t)row * a.width;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * G + t) * V;
    if (col >= a.width) continue;
    float w[V], b[V];
    param<V>(a.w, a.w_dtype, col, true, 1.f, w);
    param<V>(a.b, a.b_dtype, col, true, 0.f, b);
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = fmaf((px[c].get(e) - mean) * rstd, w[e], b[e]);
    Piece<TY, V>::template store<PAST>(y + col, w);
  }
}

// The same for rows that registers do not hold, by 1024 threads that read them three times.
template <typename TX, typename TY>
__global__ __launch_bounds__(1024) void norm_forward_wide_kernel(const NormArgs a) {
  __shared__ float sums[2][17];
  const int64_t row = blockIdx.x;
  const TX* x = (const TX*)a.x + row * a.ldx;
  TY* y = (TY*)a.y + row * a.width;
  float s = 0.f;
  for (int c = threadIdx.x; c < a.width; c += 1024) s += st_load<TX>(x, c);
  const float n = 1.f / (float)a.width, mean = row_sum<1024>(s, sums[0]) * n;
  s = 0.f;
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    const float d = st_load<TX>(x, c) - mean;
    s += d * d;
  }
  const float rstd = 1.f / sqrtf(row_sum<1024>(s, sums[1]) * n + a.eps);
  if (threadIdx.x == 0 && a.mean) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    float w[1], b[1];
    param<1>(a.w, a.w_dtype, c, true, 1.f, w);
    param<1>(a.b, a.b_dtype, c, true, 0.f, b);
    st_store<TY>(y, c, fmaf((st_load<TX>(x, c) - mean) * rstd, w[0], b[0]));
  }
}

static __device__ __forceinline__ void put(void* p, int dtype, int c, float v) {
  if (dtype) ((float*)p)[c] = v;
  else ((bf16_t*)p)[c] = f32_to_bf16(v);
}

// dw and db of a.lanes (16, 64) columns from all rows, a column a lane: sixteen wavefronts take 1024 / a.lanes rows at a time, eight
// times as many on their way.
template <typename TX, typename TY>
static __device__ __forceinline__ void few_rows_columns(const NormArgs& a, int block, float (*sums)[16][64]) {
  constexpr int AHEAD = 8;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int of = lane & (a.lanes - 1), c = block * a.lanes + of, at = c < a.width ? c : 0, step = 1024 / a.lanes;
  float dw = 0.f, db = 0.f;
  for (int r0 = (int)threadIdx.x / a.lanes; r0 < a.rows; r0 += step * AHEAD) {
    Piece<TX, 1> x[AHEAD];
    Piece<TY, 1> d[AHEAD];
    float mean[AHEAD], rstd[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int64_t r = r0 + step * k < a.rows ? r0 + step * k : r0;
      x[k].load((const TX*)a.x + r * a.ldx, at, true);
      d[k].load((const TY*)a.dy + r * a.lddy, at, true);
      mean[k] = a.mean[r];
      rstd[k] = a.rstd[r];
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const bool in = r0 + step * k < a.rows;
      const float v = d[k].get(0), w = fmaf(v, (x[k].get(0) - mean[k]) * rstd[k], dw);
      dw = in ? w : dw;
      db = in ? db + v : db;
    }
  }
  for (int h = a.lanes; h < 64; h <<= 1) {
    dw += __shfl_xor(dw, h, 64);
    db += __shfl_xor(db, h, 64);
  }
  sums[0][wave][lane] = dw;
  sums[1][wave][lane] = db;
  __syncthreads();
  if (wave > 1 || lane >= a.lanes || c >= a.width) return;
  float s = sums[wave][0][lane];
#pragma unroll
  for (int k = 1; k < 16; ++k) s += sums[wave][k][lane];
  if (wave == 0 && a.dw) put(a.dw, a.w_dtype, c, s);
  if (wave == 1 && a.db) put(a.db, a.b_dtype, c, s);
}

// dx of every row and, in a.partial [workgroups][2][width], this workgroup's sums of dy xh and of dy: sixteen wavefronts take
// 1024 / G rows at a time, the next ones' x and dy on their way meanwhile; a thread's columns are the same in all of them, and one
// workgroup a CU leaves few parts to add.  us, 16384 x 4096: one row ahead of 16 elements a thread 93, two of eight 87, dx around the
// caches 75, loads without branches 67.
template <typename TX, typename TY, int G, int E, int V, bool PAST>
__global__ __launch_bounds__(1024) void norm_backward_kernel(const NormArgs a) {
  constexpr int NC = E / V, ROWS = 1024 / G;
  __shared__ float sums[2][16][2];
  constexpr int HALF = ROWS > 1 ? ROWS / 2 * G * E : 0;
  __shared__ float half[HALF > 2048 ? HALF : 2048];
  if ((int)blockIdx.x >= a.row_wgs) {
    few_rows_columns<TX, TY>(a, blockIdx.x - a.row_wgs, (float(*)[16][64])half);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = wave / (G / 64), t = threadIdx.x % G;
  const int64_t step = (int64_t)a.row_wgs * ROWS;
  int64_t first = (int64_t)blockIdx.x * ROWS;
  const float n = 1.f / (float)a.width;
  // Rows on their way: two of eight elements a thread in one access; one in more; none of sixteen elements.
  constexpr int AHEAD = E > 8 ? 0 : V < 8 ? 1 : 2, SETS = AHEAD > 0 ? AHEAD : 1;
  float w[E], dw[E] = {}, db[E] = {};
#pragma unroll
  for (int c = 0; c < NC; ++c) param<V>(a.w, a.w_dtype, (c * G + t) * V, (c * G + t) * V < a.width, 1.f, w + c * V);
  struct Row {
    Piece<TX, V> px[NC];
    Piece<TY, V> pd[NC];
    float mean, rstd;
  } sets[SETS];
  auto fetch = [&](Row& q, int64_t row) __attribute__((always_inline)) {  // (zeros behind the last row and the last column: they add nothing)
    const bool in = row < a.rows;
    if (!in) row = 0;
    const TX* x = (const TX*)a.x + row * a.ldx;
    const TY* dy = (const TY*)a.dy + row * a.lddy;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * G + t) * V;
      q.px[c].load(x, col, in && col < a.width);
      q.pd[c].load(dy, col, in && col < a.width);
    }
    const float mean = a.mean[row], rstd = a.rstd[row];
    q.mean = in ? mean : 0.f;
    q.rstd = in ? rstd : 0.f;
  };
  auto one = [&](Row& q, int64_t row, int buf) __attribute__((always_inline)) {
    if constexpr (AHEAD == 0) fetch(q, row);
    float xh[E], g[E], s0 = 0.f, s1 = 0.f;
    const float r = q.rstd, mean = q.mean;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int i = c * V + e;
        xh[i] = (c * G + t) * V < a.width ? (q.px[c].get(e) - mean) * r : 0.f;
        const float d = q.pd[c].get(e);
        dw[i] = fmaf(d, xh[i], dw[i]);
        db[i] += d;
        g[i] = d * w[i];
        s0 += g[i];
        s1 = fmaf(g[i], xh[i], s1);
      }
    if constexpr (AHEAD > 0) fetch(q, row + AHEAD * step);
    if (!a.dx) return;
    s0 = wave_sum(s0);
    s1 = wave_sum(s1);
    if constexpr (G > 64) {
      if ((threadIdx.x & 63) == 0) {
        sums[buf][wave][0] = s0;
        sums[buf][wave][1] = s1;
      }
      __syncthreads();
      s0 = s1 = 0.f;
#pragma unroll
      for (int k = 0; k < G / 64; ++k) {
        s0 += sums[buf][group * (G / 64) + k][0];
        s1 += sums[buf][group * (G / 64) + k][1];
      }
    }
    s0 *= n;
    s1 *= n;
    if (row < a.rows) {
      TX* dx = (TX*)a.dx + row * a.width;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = (c * G + t) * V;
        if (col >= a.width) continue;
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = r * (g[c * V + e] - s0 - xh[c * V + e] * s1);
        Piece<TX, V>::template store<PAST>(dx + col, o);
      }
    }
  };
  if constexpr (AHEAD > 0)
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) fetch(sets[k], first + group + k * step);
  for (int buf = 0; first < a.rows;) {  // (the same for the whole workgroup; rows behind the last one are zeros)
#pragma unroll
    for (int k = 0; k < SETS; ++k) {
      one(sets[k], first + group, buf);
      first += step;
      buf ^= 1;
    }
  }
  if (!a.partial) return;
  // The groups' sums meet in LDS, the upper half of them added to the lower one until one is left.
  auto meet = [&](float* v) __attribute__((always_inline)) {
    if constexpr (ROWS > 1) {
#pragma unroll
      for (int h = ROWS / 2; h > 0; h /= 2) {
        __syncthreads();
        if (group >= h && group < 2 * h)
#pragma unroll
          for (int i = 0; i < E; ++i) half[((group - h) * E + i) * G + t] = v[i];
        __syncthreads();
        if (group < h)
#pragma unroll
          for (int i = 0; i < E; ++i) v[i] += half[(group * E + i) * G + t];
      }
    }
  };
  meet(dw);
  meet(db);
  if (group > 0) return;
  float* const out = a.partial + (int64_t)blockIdx.x * 2 * a.width;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * G + t) * V;
    if (col >= a.width) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      out[col + e] = dw[c * V + e];
      out[a.width + col + e] = db[c * V + e];
    }
  }
}

// dx of rows that registers do not hold.
template <typename TX, typename TY>
__global__ __launch_bounds__(1024) void norm_backward_wide_kernel(const NormArgs a) {
  __shared__ float sums[2][17];
  const int64_t row = blockIdx.x;
  const TX* x = (const TX*)a.x + row * a.ldx;
  const TY* dy = (const TY*)a.dy + row * a.lddy;
  const float n = 1.f / (float)a.width, mean = a.mean[row], r = a.rstd[row];
  float s0 = 0.f, s1 = 0.f, w[1];
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    param<1>(a.w, a.w_dtype, c, true, 1.f, w);
    const float g = st_load<TY>(dy, c) * w[0];
    s0 += g;
    s1 = fmaf(g, (st_load<TX>(x, c) - mean) * r, s1);
  }
  s0 = row_sum<1024>(s0, sums[0]) * n;
  s1 = row_sum<1024>(s1, sums[1]) * n;
  TX* dx = (TX*)a.dx + row * a.width;
  for (int c = threadIdx.x; c < a.width; c += 1024) {
    param<1>(a.w, a.w_dtype, c, true, 1.f, w);
    st_store<TX>(dx, c, r * (st_load<TY>(dy, c) * w[0] - s0 - (st_load<TX>(x, c) - mean) * r * s1));
  }
}

// ... and the sums of dy xh and dy over a run of `per` rows, a column a thread.
template <typename TX, typename TY>
__global__ __launch_bounds__(256) void norm_columns_kernel(const NormArgs a, int per) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.width) return;
  const int64_t r0 = (int64_t)blockIdx.y * per, r1 = r0 + per < a.rows ? r0 + per : a.rows;
  float dw = 0.f, db = 0.f;
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r) {
    const float d = st_load<TY>((const TY*)a.dy + r * a.lddy, c);
    dw = fmaf(d, (st_load<TX>((const TX*)a.x + r * a.ldx, c) - a.mean[r]) * a.rstd[r], dw);
    db += d;
  }
  float* out = a.partial + (int64_t)blockIdx.y * 2 * a.width;
  out[c] = dw;
  out[a.width + c] = db;
}

// ---------------------------------------------------------------------------------------------- host
// Threads of a row of the backward pass, eight elements each (sixteen of the widest), and its workgroups: one per CU, or what the rows fill.
static int norm_threads(int width) { return width <= 512 ? 64 : width <= 1024 ? 128 : width <= 2048 ? 256 : width <= 4096 ? 512 : 1024; }
static int norm_parts(int rows, int width) {
  if (width > kNormWide) return rows < 128 ? rows : 128;
  const int at_once = 1024 / norm_threads(width);
  const int wgs = (rows + at_once - 1) / at_once;
  return wgs < 256 ? wgs : 256;
}
// Few rows: dw and db are other workgroups' of the same launch, which read x and dy again, from the caches, instead of parts that a second
// launch adds; 64 columns each where eight loads fetch all rows of them, 16 otherwise.  us, so / in parts and their launch: 16 x 768
// 4.6 / 9.0, 128 x 4096 5.6 / 14, 512 x 768 5.4 / 10, 777 x 1001 fp32 8.3 / 11.3, 1024 x 1024 8.6 / 11; 1024 x 2048 18 / 15.
static bool norm_few(int rows, int width) { return rows <= 1024 && width <= kNormWide && (int64_t)rows * width <= 1 << 20; }
size_t norm_partial_floats(int rows, int width) {
  return rows <= 0 || norm_few(rows, width) ? 0 : (size_t)norm_parts(rows, width) * 2 * width;
}

// Elements that one access can move: 8 (4 with fp32 on either side), 2 or 1, by what every row's start is a multiple of.
static int norm_vec(const NormArgs& a, const void* other, int64_t ldo, int other_dtype) {
  auto fits = [&](int v) {
    auto ok = [&](const void* p, int64_t ld, int dtype) {
      const uint64_t bytes = (uint64_t)v * (dtype ? 4 : 2), line = bytes < 16 ? bytes : 16;
      return !p || (((uint64_t)p % line) == 0 && (uint64_t)ld * (dtype ? 4 : 2) % line == 0);
    };
    return a.width % v == 0 && ok(a.x, a.ldx, a.x_dtype) && ok(other, ldo, other_dtype) && ok(a.w, 0, a.w_dtype) &&
           ok(a.b, 0, a.b_dtype) && ok(a.dx, a.width, a.x_dtype);
  };
  const int most = a.x_dtype || other_dtype ? 4 : 8;
  return fits(most) ? most : fits(2) ? 2 : 1;
}

// go(its arguments) for every run of rows that a launch has threads for, so many a row.
template <typename F>
static void norm_runs(const NormArgs& a, int threads, F&& go) {
  const int64_t at_once = kMostThreads / 1024 * (1024 / threads), x = a.x_dtype ? 4 : 2, y = a.y_dtype ? 4 : 2;
  for (int64_t r = 0; r < a.rows; r += at_once) {
    NormArgs p = a;
    p.rows = (int)(a.rows - r < at_once ? a.rows - r : at_once);
    p.x = (const char*)a.x + r * a.ldx * x;
    if (a.y) p.y = (char*)a.y + r * a.width * y;
    if (a.mean) p.mean += r, p.rstd += r;
    if (a.dy) p.dy = (const char*)a.dy + r * a.lddy * y;
    if (a.dx) p.dx = (char*)a.dx + r * a.width * x;
    go(p);
  }
}

template <typename F>
static hipError_t norm_types(const NormArgs& a, F&& go) {
  if (a.x_dtype) {
    if (a.y_dtype) go((float*)nullptr, (float*)nullptr);
    else go((float*)nullptr, (bf16_t*)nullptr);
  } else {
    if (a.y_dtype) go((bf16_t*)nullptr, (float*)nullptr);
    else go((bf16_t*)nullptr, (bf16_t*)nullptr);
  }
  return hipGetLastError();
}

hipError_t launch_norm_forward(const NormArgs& a, hipStream_t st) {
  if (a.rows <= 0 || a.width <= 0 || !a.x || !a.y || !a.mean != !a.rstd) return hipErrorInvalidValue;
  const bool past = (int64_t)a.rows * a.width * (a.y_dtype ? 4 : 2) > kPast;
  return norm_types(a, [&](auto* tx, auto* ty) {
    typedef std::remove_pointer_t<decltype(tx)> TX;
    typedef std::remove_pointer_t<decltype(ty)> TY;
    if (a.width > 2 * kNormWide) {
      norm_runs(a, 1024, [&](const NormArgs& p) {
        hipLaunchKernelGGL((norm_forward_wide_kernel<TX, TY>), dim3(p.rows), dim3(1024), 0, st, p);
      });
      return;
    }
    auto run = [&](auto gc, auto ec, auto vc) {
      constexpr int G = decltype(gc)::value, E = decltype(ec)::value, V = decltype(vc)::value, T = G < 256 ? 256 : G;
      constexpr bool WIDE = V >= 4;
      auto kernel = WIDE && past ? norm_forward_kernel<TX, TY, G, E, V, WIDE> : norm_forward_kernel<TX, TY, G, E, V, false>;
      norm_runs(a, G, [&](const NormArgs& p) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(((int64_t)p.rows * G + T - 1) / T)), dim3(T), 0, st, p);
      });
    };
    // Up to 64 elements a thread: rows of up to 4096 columns then need no barrier, and wider ones a workgroup of four wavefronts.  Not
    // where they are read one by one, and in the first case not in pairs.  us, 64 / 32 a thread: 16384 x 4096 56 / 66, 4096 x 16384
    // 64 / 87; in pairs 4096 x 4094 28 / 20, 2492 x 14458 47 / 59; one by one 2492 x 2731 33 / 16, 2492 x 14459 149 / 99.
    auto sized = [&](auto vc) {
      constexpr int V = decltype(vc)::value;
      if (a.width <= 512) run(std::integral_constant<int, 64>(), std::integral_constant<int, 8>(), vc);
      else if (a.width <= 1024) run(std::integral_constant<int, 64>(), std::integral_constant<int, 16>(), vc);
      else if (a.width <= 2048) run(std::integral_constant<int, 64>(), std::integral_constant<int, 32>(), vc);
      else if (a.width <= 4096 && V >= 4) run(std::integral_constant<int, 64>(), std::integral_constant<int, V >= 4 ? 64 : 32>(), vc);
      else if (a.width <= 8192) run(std::integral_constant<int, 256>(), std::integral_constant<int, 32>(), vc);
      else if (a.width <= 16384 && V >= 2) run(std::integral_constant<int, 256>(), std::integral_constant<int, V >= 2 ? 64 : 32>(), vc);
      else run(std::integral_constant<int, 1024>(), std::integral_constant<int, 32>(), vc);
    };
    constexpr int W = sizeof(TX) == 2 && sizeof(TY) == 2 ? 8 : 4;
    const int v = norm_vec(a, a.y, a.width, a.y_dtype);
    if (v == W) sized(std::integral_constant<int, W>());
    else if (v == 2) sized(std::integral_constant<int, 2>());
    else sized(std::integral_constant<int, 1>());
  });
}

hipError_t launch_norm_backward(const NormArgs& a, hipStream_t st) {
  if (a.rows <= 0 || a.width <= 0 || !a.x || !a.dy || !a.mean || !a.rstd) return hipErrorInvalidValue;
  NormArgs p = a;
  p.b = nullptr;  // (not read)
  const bool past = (int64_t)a.rows * a.width * (a.x_dtype ? 4 : 2) > kPast;
  const bool sums = a.dw || a.db, joined = sums && norm_partial_floats(a.rows, a.width) > 0;
  if (joined && !a.partial) return hipErrorInvalidValue;
  if (!joined) p.partial = nullptr;
  const int parts = norm_parts(a.rows, a.width);
  hipError_t e = norm_types(p, [&](auto* tx, auto* ty) {
    typedef std::remove_pointer_t<decltype(tx)> TX;
    typedef std::remove_pointer_t<decltype(ty)> TY;
    if (a.width > kNormWide) {
      const int per = (a.rows + parts - 1) / parts;
      if (p.dx)
        norm_runs(p, 1024, [&](const NormArgs& q) {
          hipLaunchKernelGGL((norm_backward_wide_kernel<TX, TY>), dim3(q.rows), dim3(1024), 0, st, q);
        });
      if (p.partial)
        hipLaunchKernelGGL((norm_columns_kernel<TX, TY>), dim3((a.width + 255) / 256, parts), dim3(256), 0, st, p, per);
      return;
    }
    auto run = [&](auto gc, auto ec, auto vc) {
      constexpr int G = decltype(gc)::value, E = decltype(ec)::value, V = decltype(vc)::value;
      constexpr bool WIDE = V >= 4;
      auto kernel = WIDE && past ? norm_backward_kernel<TX, TY, G, E, V, WIDE> : norm_backward_kernel<TX, TY, G, E, V, false>;
      p.row_wgs = p.dx || p.partial ? parts : 0;
      p.lanes = a.rows <= 128 ? 64 : 16;
      const int columns = sums && !joined ? (a.width + p.lanes - 1) / p.lanes : 0;
      hipLaunchKernelGGL(kernel, dim3(p.row_wgs + columns), dim3(1024), 0, st, p);
    };
    auto sized = [&](auto vc) {
      typedef std::integral_constant<int, 8> eight;
      if (a.width <= 512) run(std::integral_constant<int, 64>(), eight(), vc);
      else if (a.width <= 1024) run(std::integral_constant<int, 128>(), eight(), vc);
      else if (a.width <= 2048) run(std::integral_constant<int, 256>(), eight(), vc);
      else if (a.width <= 4096) run(std::integral_constant<int, 512>(), eight(), vc);
      else if (a.width <= 8192) run(std::integral_constant<int, 1024>(), eight(), vc);
      else run(std::integral_constant<int, 1024>(), std::integral_constant<int, 16>(), vc);
    };
    constexpr int W = sizeof(TX) == 2 && sizeof(TY) == 2 ? 8 : 4;
    const int v = norm_vec(p, p.dy, p.lddy, p.y_dtype);
    if (v == W) sized(std::integral_constant<int, W>());
    else if (v == 2) sized(std::integral_constant<int, 2>());
    else sized(std::integral_constant<int, 1>());
  });
  if (e != hipSuccess || !joined) return e;
  return launch_lin_sum(p.partial, parts, a.width, p.dw, p.w_dtype, st, p.db, p.b_dtype);
}

}  // namespace dion
