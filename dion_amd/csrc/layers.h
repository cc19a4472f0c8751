// Launchers of layer_norm.hip and embedding.hip (internal; the public surface is include/dion_hip.h).  dtypes: 0 bf16, 1 fp32.
#pragma once
#include "common.h"

namespace dion {

struct NormArgs {
  const void* x;  // [rows][width], ldx elements between rows
  int64_t ldx;
  const void *w, *b;  // [width] or null
  void* y;            // [rows][width], dense
  float *mean, *rstd;  // [rows], or both null (forward); read by the backward pass
  int rows, width;
  int x_dtype, y_dtype, w_dtype, b_dtype;
  float eps;
  // backward: dy [rows][width] of y_dtype, lddy elements between rows; dx dense, of x_dtype, or null
  const void* dy;
  int64_t lddy;
  void* dx;
  float* partial;  // norm_partial_floats(rows, width), which may be none, where dw or db is asked for
  void *dw, *db;   // of w_dtype, b_dtype, or null
  int row_wgs, lanes;  // set by the launcher: workgroups that take rows, and columns of each of those behind them
};
size_t norm_partial_floats(int rows, int width);
hipError_t launch_norm_forward(const NormArgs& a, hipStream_t st);
hipError_t launch_norm_backward(const NormArgs& a, hipStream_t st);

struct EmbeddingArgs {
  const void* ids;  // [tokens] int32 or int64
  int ids64;
  int tokens, vocab, width;
  int64_t padding;  // an id without a gradient, or -1
  float scale;
  const void* w;  // [vocab][width], ldw elements between rows
  int64_t ldw;
  int w_dtype;
  void* y;  // [tokens][width], dense
  int y_dtype;
  const void* dy;  // of y_dtype, lddy elements between rows
  int64_t lddy;
  void* dw;    // [vocab][width], dense, of w_dtype
  void* space;  // embedding_space_bytes(tokens, vocab, width), 256-byte aligned
};
size_t embedding_space_bytes(int tokens, int vocab, int width);
hipError_t launch_embedding_forward(const EmbeddingArgs& a, hipStream_t st);
hipError_t launch_embedding_backward(const EmbeddingArgs& a, hipStream_t st);

// A result of more bytes than the L2s of the eight XCDs hold is stored non-temporally.  us without / with: layer norm of 8192 x 2048
// 13.9 / 12.2, 16384 x 2048 25.6 / 21.5, 16384 x 4096 53 / 54, forward and backward 146 / 137; rows of a table, 8192 x 4096 18.8 / 17.7,
// 16384 x 4096 36.3 / 32.2.
constexpr int64_t kPast = int64_t(32) << 20;

// V elements as one access moves them.
template <typename T, int V>
struct Piece {
  static constexpr int BYTES = (int)sizeof(T) * V;
  typedef std::conditional_t<BYTES == 32, f32x4, std::conditional_t<BYTES == 16, u32x4_t, std::conditional_t<BYTES == 8, u32x2_t,
          std::conditional_t<BYTES == 4, uint32_t, uint16_t>>>> raw_t;
  typedef std::conditional_t<BYTES == 2, uint32_t, raw_t> held_t;
  held_t r[BYTES == 32 ? 2 : 1];
  // Elements `at` .. of a row, or zeros where `in` is false: then the row's first ones are read.  (A load that is skipped is a branch,
  // into which the compiler takes what follows from a narrow load, and its wait with it.  us, rows of single bf16 elements, branch /
  // none: layer norm of 2492 x 2731, forward 41.5 / 33.4; 6465 tokens of 18573 x 2155, sums 345 / 49.)
  __device__ __forceinline__ void load(const T* row, int at, bool in) {
    const raw_t* p = (const raw_t*)(row + (in ? at : 0));
#pragma unroll
    for (int k = 0; k < (BYTES == 32 ? 2 : 1); ++k) {
      const held_t zero = {}, v = (held_t)p[k];
      r[k] = in ? v : zero;
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (BYTES == 2) return __uint_as_float(r[0] << 16);
    else if constexpr (BYTES == 4 && sizeof(T) == 4) return __uint_as_float(r[0]);
    else if constexpr (BYTES == 4) return __uint_as_float(e ? r[0] & 0xffff0000u : r[0] << 16);
    else if constexpr (BYTES == 32) return r[e >> 2][e & 3];
    else if constexpr (sizeof(T) == 4) return __uint_as_float(r[0][e]);
    else return __uint_as_float((e & 1) ? r[0][e >> 1] & 0xffff0000u : r[0][e >> 1] << 16);
  }
  // PAST: around the caches (kPast).
  template <bool PAST = false>
  static __device__ __forceinline__ void store(T* p, const float* v) {
    if constexpr (V == 8) st_store8<T, PAST>(p, 0, v);
    else if constexpr (V == 4) st_store4<T, PAST>(p, 0, v);
    else if constexpr (V == 2) {
      if constexpr (sizeof(T) == 4) *(uint2*)p = make_uint2(__float_as_uint(v[0]), __float_as_uint(v[1]));
      else *(uint32_t*)p = pack_bf16x2(v[0], v[1]);
    } else st_store<T>(p, 0, v[0]);
  }
};

// The sum over a wavefront, in every lane.
static __device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

}  // namespace dion
