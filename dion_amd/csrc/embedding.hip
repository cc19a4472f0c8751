// Rows of a table, y[t] = scale W[ids[t]], and the table's gradient: dW[v] = scale times the sum of dy[t] over the tokens t with
// ids[t] = v, in the order of t, in fp32, rounded once; zeros where there are none.  A token is then added by whoever holds its
// row, with no atomics on values: a result repeats bit for bit.
//   index  `order`: the tokens grouped by their row, ascending within it; where each row's run of them starts, and its length
//   sums   rows of up to 64 tokens, and the zeros of rows with none; of longer ones a partial sum for every 64 tokens
//   join   the partial sums of a long row, added in order
// An id outside the table reads nothing: its row of y is NaN, and it has no gradient.
// Bound by HBM: the rows, dy, and the whole of dW.  us: 32768 tokens of 32000 x 4096, all bf16, y 72 (3.7 TB/s written, as much read from
// the caches), index 14, sums 104 (5.1 TB/s), join 7; 8192 tokens of 50304 x 768, an fp32 table, y 6 to 7, index 9, sums 28 to 37
// (4.5 to 5.9 TB/s, nine tenths of them zeros), join 4.
#include "layers.h"

namespace dion {

constexpr int kRun = 64;         // tokens of a partial sum
constexpr int kSlice = 512;      // columns: eight a lane of a wavefront
constexpr int kIndexRows = 512;  // rows of a workgroup of the index, at most
constexpr int kIndexWaves = 16;
constexpr int kIndexLds = 144 * 1024;

static int index_groups(int vocab) {  // a power of two, so that a row's workgroup is its lower bits
  int g = 256;
  while ((vocab + g - 1) / g > kIndexRows) g *= 2;
  return g;
}

// ---- y
// A wavefront takes up to SLICES slices of 64 V columns of a token's row.
template <typename TW, typename TY, int V, bool PAST>
__global__ __launch_bounds__(256) void embedding_rows_kernel(const EmbeddingArgs a, uint32_t per_row, uint32_t units) {
  constexpr int SLICES = 4;
  const int lane = threadIdx.x & 63;
  const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int64_t t = unit / per_row;
  const int c0 = (int)(unit - (uint32_t)t * per_row) * (64 * V * SLICES) + lane * V;
  const int64_t id = a.ids64 ? ((const int64_t*)a.ids)[t] : ((const int32_t*)a.ids)[t];
  const bool in = id >= 0 && id < a.vocab;
  const TW* w = (const TW*)a.w + (in ? id * a.ldw : 0);
  TY* y = (TY*)a.y + t * a.width;
  Piece<TW, V> p[SLICES];
#pragma unroll
  for (int s = 0; s < SLICES; ++s) p[s].load(w, c0 + s * 64 * V, in && c0 + s * 64 * V < a.width);
#pragma unroll
  for (int s = 0; s < SLICES; ++s) {
    const int c = c0 + s * 64 * V;
    if (c >= a.width) break;
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = in ? a.scale * p[s].get(e) : __uint_as_float(0x7fc00000u);
    Piece<TY, V>::template store<PAST>(y + c, v);
  }
}

// ---- index
struct IndexArgs {
  const void* ids;
  int tokens, vocab, groups;
  int64_t padding;
  uint32_t *order, *first, *count;  // [tokens], [vocab + 1] (the last one: how many tokens have a gradient), [vocab]
};

// Workgroup g has the rows v with v % groups = g: row v / groups of its own.  Every workgroup reads all ids, and counts its own (by
// wavefront and row) and those of the workgroups before it, which is where its part of `order` starts; then it places its own.  A
// wavefront has a run of consecutive tokens; it lists those of the workgroup's rows in LDS, in order, and counts and places from
// there, 64 at a time, equal ones together; so the tokens of a row stay in order.  Where the list is full it reads the ids again
// instead.  Bound by the instructions that look at an id that is another workgroup's (255 of 256): 8192 tokens 9 us, 32768 14,
// 131072 42.  Without lists, every match counted and placed where it is found, 32768 tokens took 33.  Tables past 131072 rows have more
// workgroups, which all read all ids: 8192 tokens of 300000 rows 28.
template <typename ID>
__global__ __launch_bounds__(kIndexWaves * 64) void embedding_index_kernel(const IndexArgs a, int rows, int capacity) {
  constexpr int AHEAD = 16;  // ids of a lane on their way
  // at [kIndexWaves][rows]: counts, then where a wavefront's next token of the row goes; behind it the lists [kIndexWaves][capacity]:
  // the row, above it how far the token lies behind the wavefront's first one
  extern __shared__ uint32_t at[];
  __shared__ uint32_t sums[kIndexWaves], before;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x, mask = a.groups - 1, shift = __builtin_ctz(a.groups);
  for (int i = threadIdx.x; i < kIndexWaves * rows; i += kIndexWaves * 64) at[i] = 0;
  if (threadIdx.x == 0) before = 0;
  __syncthreads();
  const int batches = (a.tokens + 63) / 64;
  const int b0 = (int)((int64_t)batches * wave / kIndexWaves), b1 = (int)((int64_t)batches * (wave + 1) / kIndexWaves);
  volatile uint32_t* const mine = at + wave * rows;  // (lanes read what others of the wavefront wrote)
  uint32_t* const list = at + kIndexWaves * rows + wave * capacity;
  const uint32_t token0 = (uint32_t)b0 * 64;
  uint32_t lower = 0, listed = 0;  // (both the wavefront's)
  // Every batch of 64 tokens of this wavefront: f(token of the lane, its row or -1, whether the row is this workgroup's).
  auto batches_of = [&](auto&& f) __attribute__((always_inline)) {
    for (int b = b0; b < b1; b += AHEAD) {
      ID ids[AHEAD];
      const int64_t t0 = (int64_t)b * 64 + lane;
      const ID* p = (const ID*)a.ids + t0;
      if (b + AHEAD <= b1 && (int64_t)(b + AHEAD) * 64 <= a.tokens) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) ids[k] = p[k * 64];
      } else {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) ids[k] = b + k < b1 && t0 + k * 64 < a.tokens ? p[k * 64] : (ID)-1;
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        typedef std::make_unsigned_t<ID> U;
        const bool valid = (U)ids[k] < (U)a.vocab && ids[k] != (ID)a.padding;
        const uint32_t id = (uint32_t)ids[k];
        f((uint32_t)t0 + k * 64, id, valid);
      }
    }
  };
  // Tokens of the workgroup's rows, at most one a lane, in the lanes' order: counted, or placed.
  auto take = [&](auto placec, uint32_t token, int row, bool is) __attribute__((always_inline)) {
    constexpr bool PLACE = decltype(placec)::value;
    uint64_t left = __ballot(is);
    while (left) {  // (every turn takes at least one token out)
      const int leader = __builtin_ctzll(left);
      const int r = __builtin_amdgcn_readlane(row, leader);
      const uint64_t same = __ballot(row == r) & left;
      const uint32_t to = mine[r];
      if constexpr (PLACE)
        if ((same >> lane) & 1) a.order[to + __popcll(same & ((1ull << lane) - 1))] = token;
      if (lane == leader) mine[r] = to + __popcll(same);
      left &= ~same;
    }
  };
  auto from_list = [&](auto placec) __attribute__((always_inline)) {
    for (uint32_t i = 0; i < listed; i += 64) {
      const bool is = i + lane < listed;
      const uint32_t e = is ? list[i + lane] : 0;
      take(placec, token0 + e / kIndexRows, (int)(e % kIndexRows), is);
    }
  };
  auto from_ids = [&](auto placec) __attribute__((always_inline)) {
    batches_of([&](uint32_t token, uint32_t id, bool valid) __attribute__((always_inline)) {
      take(placec, token, (int)(id >> shift), valid && (int)(id & mask) == g);
    });
  };
  batches_of([&](uint32_t token, uint32_t id, bool valid) __attribute__((always_inline)) {
    const int group = (int)(id & mask);
    lower += (uint32_t)__popcll(__ballot(valid && group < g));
    const bool is = valid && group == g;
    const uint64_t here = __ballot(is);
    if (here) {
      const uint32_t to = listed + __popcll(here & ((1ull << lane) - 1));
      if (is && to < (uint32_t)capacity) list[to] = (token - token0) * kIndexRows + (id >> shift);
      listed += (uint32_t)__popcll(here);
    }
  });
  const bool fits = listed <= (uint32_t)capacity;
  if (fits) from_list(std::false_type());
  else from_ids(std::false_type());
  if (lane == 0) atomicAdd(&before, lower);
  __syncthreads();
  // Row r is thread r's: its tokens behind those of the rows before it, a wavefront's behind those of the wavefronts before.
  const int r = threadIdx.x;
  uint32_t n = 0;
  if (r < rows)
    for (int w = 0; w < kIndexWaves; ++w) n += at[w * rows + r];
  uint32_t upto = n;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(upto, d, 64);
    if (lane >= d) upto += o;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  uint32_t start = before + upto - n;
  for (int w = 0; w < wave; ++w) start += sums[w];
  if (g == a.groups - 1 && r == kIndexWaves * 64 - 1) a.first[a.vocab] = start + n;
  if (r < rows) {
    const int64_t v = (int64_t)r * a.groups + g;
    if (v < a.vocab) {
      a.first[v] = start;
      a.count[v] = n;
    }
    for (int w = 0; w < kIndexWaves; ++w) {
      const uint32_t k = at[w * rows + r];
      at[w * rows + r] = start;
      start += k;
    }
  }
  __syncthreads();
  if (fits) from_list(std::true_type());
  else from_ids(std::true_type());
}

// ---- sums
struct SumArgs {
  const void* ids;
  const uint32_t *order, *first, *count;
  const void* dy;
  int64_t lddy;
  void* dw;
  float* partial;  // [2 * chunks of 64 of `order`][width]: see slot()
  int tokens, vocab, width, groups;
  uint32_t slices;
  float scale;
};
// Where the partial sum of a long row's tokens from p on lies: of the 64 of `order` that p is in, at most two such runs start
// there -- the last one of a row and the first of the next.
__device__ __forceinline__ int64_t slot(uint32_t p, bool first) { return (int64_t)(p / kRun) * 2 + first; }

// A slice is S times 512 columns: of a lane S times eight, in pieces of V that lie 64 V apart.
// acc += the rows of dy of the tokens that lanes from.. from + U - 1 hold in `token`, of which n are meant, in that order.
template <typename TY, int V, int S, int U>
__device__ __forceinline__ void add_group(const SumArgs& a, int token, int from, int n, int slice, int lane, float* acc) {
  constexpr int NC = 8 * S / V;
  const int col = slice * (kSlice * S) + lane * V;
  Piece<TY, V> q[U][NC];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (u >= n) break;
    const int64_t t = (uint32_t)__builtin_amdgcn_readlane(token, from + u);
    const TY* dy = (const TY*)a.dy + t * a.lddy;
#pragma unroll
    for (int c = 0; c < NC; ++c) q[u][c].load(dy, col + c * 64 * V, col + c * 64 * V < a.width);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u < n)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[c * V + e] += q[u][c].get(e);
}
// ... of the n tokens from lane `from` on.  Pieces of eight are few enough to ask for eight tokens' whatever n is; of single
// elements a row has sixty-four, and what is left of n goes by halves.
template <typename TY, int V, int S>
__device__ __forceinline__ void add_rows(const SumArgs& a, int token, int from, int n, int slice, int lane, float* acc) {
  constexpr int U = 8 / S;
  if constexpr (V == 8) {
    for (int j = 0; j < n; j += U) add_group<TY, V, S, U>(a, token, from + j, n - j < U ? n - j : U, slice, lane, acc);
  } else {
    int j = 0;
    for (; j + 8 <= n; j += 8) add_group<TY, V, S, 8>(a, token, from + j, 8, slice, lane, acc);
    if (n & 4) add_group<TY, V, S, 4>(a, token, from + j, 4, slice, lane, acc), j += 4;
    if (n & 2) add_group<TY, V, S, 2>(a, token, from + j, 2, slice, lane, acc), j += 2;
    if (n & 1) add_group<TY, V, S, 1>(a, token, from + j, 1, slice, lane, acc);
  }
}
// ... of the n <= 64 that `order` lists from p on.
template <typename TY, int V, int S>
__device__ __forceinline__ void add_run(const SumArgs& a, uint32_t p, int n, int slice, int lane, float* acc) {
  add_rows<TY, V, S>(a, lane < n ? (int)a.order[p + lane] : 0, 0, n, slice, lane, acc);
}
template <typename T, int V, int S>
__device__ __forceinline__ void put_slice(T* row, int slice, int lane, int width, const float* v) {
#pragma unroll
  for (int c = 0; c < 8 * S / V; ++c) {
    const int col = slice * (kSlice * S) + c * 64 * V + lane * V;
    if (col < width) Piece<T, V>::store(row + col, v + c * V);
  }
}

constexpr int kUnits = 8;  // rows' slices of a wavefront, far apart: frequent tokens are neighbours in a table

template <typename ID, typename TY, typename TW, int V, int S>
__global__ __launch_bounds__(256) void embedding_sums_kernel(const SumArgs a, uint32_t run_wgs, uint32_t stride) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x < run_wgs) {
    // the runs of long rows that start in 64 entries of `order`
    const uint32_t unit = blockIdx.x * 4 + wave, chunk = unit / a.slices;
    const int slice = (int)(unit - chunk * a.slices);
    const uint32_t p = chunk * kRun + lane;
    uint32_t first = 0, n = 0;
    if (p < a.first[a.vocab]) {  // (`order` ends there)
      const int64_t v = (int64_t)((const ID*)a.ids)[a.order[p]];
      first = a.first[v];
      n = a.count[v];
    }
    uint64_t starts = __ballot(n > kRun && (p - first) % kRun == 0);
    while (starts) {
      const int l = __builtin_ctzll(starts);
      starts &= starts - 1;
      const uint32_t q = chunk * kRun + l, f = __builtin_amdgcn_readlane(first, l), m = __builtin_amdgcn_readlane(n, l);
      const uint32_t left = f + m - q;
      float acc[8 * S] = {};
      add_run<TY, V, S>(a, q, left < kRun ? (int)left : kRun, slice, lane, acc);
      put_slice<float, V, S>(a.partial + slot(q, q == f) * a.width, slice, lane, a.width, acc);
    }
    return;
  }
  const uint32_t w0 = (blockIdx.x - run_wgs) * 4 + wave, units = (uint32_t)a.vocab * a.slices;
  // Lanes 8 k .. 8 k + 7 have the k-th of this wavefront's rows: where its tokens start, how many, and the first eight of them.
  static_assert(kUnits == 8, "eight lanes a row");
  uint32_t first = 0, n = 0, token = 0;
  {
    const uint32_t unit = w0 + (lane >> 3) * stride;
    if (unit < units) {
      first = a.first[unit / a.slices];
      n = a.count[unit / a.slices];
    }
    if ((uint32_t)(lane & 7) < n) token = a.order[first + (lane & 7)];
    asm volatile("" : "+v"(token));  // (waited for here: in the loop that would be a wait for the last row's stores too)
  }
  for (int k = 0; k < kUnits; ++k) {
    const uint32_t unit = w0 + k * stride;
    if (unit >= units) break;
    const uint32_t row = unit / a.slices;
    const int slice = (int)(unit - row * a.slices);
    const uint32_t f = __builtin_amdgcn_readlane(first, 8 * k), m = __builtin_amdgcn_readlane(n, 8 * k);
    if (m > kRun) continue;
    float acc[8 * S] = {};
    if (m > 0) {
      add_rows<TY, V, S>(a, (int)token, 8 * k, m < 8 ? (int)m : 8, slice, lane, acc);
      if (m > 8) add_run<TY, V, S>(a, f + 8, (int)m - 8, slice, lane, acc);
#pragma unroll
      for (int e = 0; e < 8 * S; ++e) acc[e] *= a.scale;
    }
    put_slice<TW, V, S>((TW*)a.dw + (int64_t)row * a.width, slice, lane, a.width, acc);
  }
}

// ---- join
// The long rows of a workgroup of the index, 512 of their columns: eight wavefronts add an eighth of the partial sums each.
constexpr int kJoinWaves = 8;

template <typename TW, int V>
__global__ __launch_bounds__(kJoinWaves * 64) void embedding_join_kernel(const SumArgs a, int rows) {
  __shared__ float others[kJoinWaves - 1][kSlice];
  __shared__ int longs[kIndexRows], n_long;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slice = blockIdx.y;
  if (threadIdx.x == 0) n_long = 0;
  __syncthreads();
  for (int r = threadIdx.x; r < rows; r += kJoinWaves * 64) {
    const int64_t v = (int64_t)r * a.groups + blockIdx.x;
    if (v < a.vocab && a.count[v] > kRun) longs[atomicAdd(&n_long, 1)] = (int)v;  // (in any order: each is a row of its own)
  }
  __syncthreads();
  const int rows_here = n_long;
  for (int i = 0; i < rows_here; ++i) {
    const int64_t v = longs[i];
    const uint32_t first = a.first[v], runs = (a.count[v] + kRun - 1) / kRun;
    const uint32_t k0 = (uint32_t)((uint64_t)runs * wave / kJoinWaves), k1 = (uint32_t)((uint64_t)runs * (wave + 1) / kJoinWaves);
    constexpr int NC = 8 / V;
    const int col = slice * kSlice + lane * V;
    float acc[8] = {};
#pragma unroll 8
    for (uint32_t k = k0; k < k1; ++k) {
      const float* q = a.partial + slot(first + k * kRun, k == 0) * a.width;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        Piece<float, V> p;
        p.load(q, col + c * 64 * V, col + c * 64 * V < a.width);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[c * V + e] += p.get(e);
      }
    }
    if (wave > 0)
#pragma unroll
      for (int e = 0; e < 8; ++e) others[wave - 1][e * 64 + lane] = acc[e];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int w = 0; w < kJoinWaves - 1; ++w) acc[e] += others[w][e * 64 + lane];
        acc[e] *= a.scale;
      }
      put_slice<TW, V, 1>((TW*)a.dw + v * a.width, slice, lane, a.width, acc);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------- host
constexpr int64_t kMostUnits = int64_t(1) << 30;  // of the gradient's rows' slices: room for the strides in 32 bits

struct EmbeddingSpace {
  size_t order, first, count, partial, total;
};
static EmbeddingSpace embedding_space(int tokens, int vocab, int width) {
  EmbeddingSpace s;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  s.order = take((size_t)tokens * 4);
  s.first = take(((size_t)vocab + 1) * 4);
  s.count = take((size_t)vocab * 4);
  s.partial = take(tokens > kRun ? ((size_t)tokens + kRun - 1) / kRun * 2 * width * 4 : 0);
  s.total = at;
  return s;
}
size_t embedding_space_bytes(int tokens, int vocab, int width) { return embedding_space(tokens, vocab, width).total; }

static bool embedding_fits(const void* p, int64_t ld, int dtype, int v) {  // whether V elements of its rows are one access
  const uint64_t size = dtype ? 4 : 2, bytes = v * size, line = bytes < 16 ? bytes : 16;
  return (uint64_t)p % line == 0 && (uint64_t)ld * size % line == 0;
}

hipError_t launch_embedding_forward(const EmbeddingArgs& a, hipStream_t st) {
  const bool past = (int64_t)a.tokens * a.width * (a.y_dtype ? 4 : 2) > kPast;
  if (a.tokens <= 0 || a.vocab <= 0 || a.width <= 0 || !a.ids || !a.w || !a.y) return hipErrorInvalidValue;
  auto go = [&](auto* tw, auto* ty, auto vc) {
    typedef std::remove_pointer_t<decltype(tw)> TW;
    typedef std::remove_pointer_t<decltype(ty)> TY;
    constexpr int V = decltype(vc)::value;
    const int64_t per_row = (a.width + 256 * V - 1) / (256 * V), at_once = kMostThreads / 256 * 4 / per_row;  // (tokens)
    constexpr bool WIDE = V == 8;
    auto kernel = WIDE && past ? embedding_rows_kernel<TW, TY, V, WIDE> : embedding_rows_kernel<TW, TY, V, false>;
    for (int64_t t = 0; t < a.tokens; t += at_once) {
      EmbeddingArgs p = a;
      p.ids = (const char*)a.ids + t * (a.ids64 ? 8 : 4);
      p.y = (TY*)a.y + t * a.width;
      const int64_t units = per_row * (a.tokens - t < at_once ? a.tokens - t : at_once);
      hipLaunchKernelGGL(kernel, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, p, (uint32_t)per_row, (uint32_t)units);
    }
  };
  auto sized = [&](auto* tw, auto* ty) {
    auto fits = [&](int v) {
      return a.width % v == 0 && embedding_fits(a.w, a.ldw, a.w_dtype, v) && embedding_fits(a.y, a.width, a.y_dtype, v);
    };
    if (fits(8)) go(tw, ty, std::integral_constant<int, 8>());
    else if (fits(2)) go(tw, ty, std::integral_constant<int, 2>());
    else go(tw, ty, std::integral_constant<int, 1>());
  };
  if (a.w_dtype) a.y_dtype ? sized((float*)nullptr, (float*)nullptr) : sized((float*)nullptr, (bf16_t*)nullptr);
  else a.y_dtype ? sized((bf16_t*)nullptr, (float*)nullptr) : sized((bf16_t*)nullptr, (bf16_t*)nullptr);
  return hipGetLastError();
}

hipError_t launch_embedding_backward(const EmbeddingArgs& a, hipStream_t st) {
  if (a.tokens < 0 || a.vocab <= 0 || a.width <= 0 || !a.dw || !a.space) return hipErrorInvalidValue;
  const EmbeddingSpace s = embedding_space(a.tokens, a.vocab, a.width);
  char* space = (char*)a.space;
  IndexArgs ix;
  ix.ids = a.ids;
  ix.tokens = a.tokens;
  ix.vocab = a.vocab;
  ix.groups = index_groups(a.vocab);
  ix.padding = a.padding;
  ix.order = (uint32_t*)(space + s.order);
  ix.first = (uint32_t*)(space + s.first);
  ix.count = (uint32_t*)(space + s.count);
  const int rows = (a.vocab + ix.groups - 1) / ix.groups;
  // Lists for all tokens of a wavefront's run, or what LDS has room for; none where a run is too long for an entry's bits.  65536 tokens, of
  // which one is 6 %, 50304 rows: 61 us with lists of 192, which that one's workgroup fills and reads the ids again, 24 with these.
  const int64_t run = ((int64_t)a.tokens + kIndexWaves * 64 - 1) / (kIndexWaves * 64) * 64, room = (kIndexLds / 4 - kIndexWaves * rows) / kIndexWaves;
  const int capacity = run > (int64_t(1) << 32) / kIndexRows ? 0 : (int)(run < room ? run : room);
  const size_t lds = ((size_t)rows + capacity) * kIndexWaves * 4;
  auto index = [&](auto* id) {
    typedef std::remove_pointer_t<decltype(id)> ID;
    static std::atomic<uint64_t> attr_done{0};
    if (hipError_t e = set_max_dynamic_lds_once((const void*)embedding_index_kernel<ID>, kIndexLds, attr_done)) return e;
    hipLaunchKernelGGL((embedding_index_kernel<ID>), dim3(ix.groups), dim3(kIndexWaves * 64), lds, st, ix, rows, capacity);
    return hipGetLastError();
  };
  if (hipError_t e = a.ids64 ? index((int64_t*)nullptr) : index((int32_t*)nullptr)) return e;
  SumArgs p;
  p.ids = a.ids;
  p.order = ix.order;
  p.first = ix.first;
  p.count = ix.count;
  p.dy = a.dy;
  p.lddy = a.lddy;
  p.dw = a.dw;
  p.partial = (float*)(space + s.partial);
  p.tokens = a.tokens;
  p.vocab = a.vocab;
  p.width = a.width;
  p.groups = ix.groups;
  auto fits = [&](int v) {
    return a.width % v == 0 && embedding_fits(a.dy, a.lddy, a.y_dtype, v) && embedding_fits(a.dw, a.width, a.w_dtype, v);
  };
  const bool whole = fits(8);
  const int wide = whole && a.width >= 2 * kSlice ? 2 : 1;  // slices of 1024 columns: half as many ways to memory, one after the other
  p.slices = (a.width + wide * kSlice - 1) / (wide * kSlice);
  p.scale = a.scale;
  const bool longs = a.tokens > kRun;
  const int64_t units = (int64_t)a.vocab * p.slices, run_units = longs ? ((int64_t)a.tokens + kRun - 1) / kRun * p.slices : 0;
  const int64_t run_wgs = (run_units + 3) / 4, row_wgs = (units + 4 * kUnits - 1) / (4 * kUnits);
  if (units > kMostUnits || run_units > kMostUnits || (a.width + kSlice - 1) / kSlice > 65535 ||
      (run_wgs + row_wgs) * 256 > kMostThreads)
    return hipErrorInvalidValue;
  auto go = [&](auto* id, auto* ty, auto* tw, auto vc, auto sc) {
    typedef std::remove_pointer_t<decltype(id)> ID;
    typedef std::remove_pointer_t<decltype(ty)> TY;
    typedef std::remove_pointer_t<decltype(tw)> TW;
    constexpr int V = decltype(vc)::value;
    hipLaunchKernelGGL((embedding_sums_kernel<ID, TY, TW, V, decltype(sc)::value>), dim3((unsigned)(run_wgs + row_wgs)), dim3(256), 0, st, p,
                       (uint32_t)run_wgs, (uint32_t)(row_wgs * 4));
    if (longs)
      hipLaunchKernelGGL((embedding_join_kernel<TW, V>), dim3(ix.groups, (a.width + kSlice - 1) / kSlice), dim3(kJoinWaves * 64), 0, st,
                         p, rows);
  };
  auto sized = [&](auto* id, auto* ty, auto* tw) {
    typedef std::integral_constant<int, 1> one;
    if (wide == 2) go(id, ty, tw, std::integral_constant<int, 8>(), std::integral_constant<int, 2>());
    else if (whole) go(id, ty, tw, std::integral_constant<int, 8>(), one());
    else if (fits(2)) go(id, ty, tw, std::integral_constant<int, 2>(), one());
    else go(id, ty, tw, one(), one());
  };
  auto typed = [&](auto* id) {
    if (a.y_dtype) a.w_dtype ? sized(id, (float*)nullptr, (float*)nullptr) : sized(id, (float*)nullptr, (bf16_t*)nullptr);
    else a.w_dtype ? sized(id, (bf16_t*)nullptr, (float*)nullptr) : sized(id, (bf16_t*)nullptr, (bf16_t*)nullptr);
  };
  if (a.ids64) typed((int64_t*)nullptr);
  else typed((int32_t*)nullptr);
  return hipGetLastError();
}

}  // namespace dion
