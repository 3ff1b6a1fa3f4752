// Embedding lookup y[i] = scale * weight[ids[i]] and its gradient on gfx950.
//
// The gradient sums, for every row of the table, the rows of grad_y at the
// positions that name it. The positions are sorted by id (stable, so each
// id's positions stay in order) and cut at every id; a row with few positions
// is summed by one group of lanes, a row with many (a frequent word, one of
// twenty classes) in chunks of kSegment positions whose partial sums a last
// kernel adds in order. No float atomics: the sums depend on the ids alone.
#include <climits>
#include <type_traits>

#include "row_chunk.hpp"

namespace rhip {
namespace {

constexpr int kEmbThreads = 256;
constexpr int kSegment = kWave; // positions a wave sums by itself, at most
constexpr int kRowsPerWave = 4; // table rows a wave takes one after another, at most
constexpr int64_t kManyRows = 16384; // rows by column tiles of 64 chunks from which on it does
// Table rows per id past which the table is cleared as a whole, its rows search
// their first positions and the sums go by positions. (fp32, 5000 ids in 100000
// rows of 32: 54 us so, 66 the other way; in 60000 of 512: 83 and 75; bf16,
// 40000 in 400000 of 256: 129 and 138, in 200000: 97 and 100.)
constexpr int64_t kSparse = 8;
constexpr int kJoinCols = 16, kJoinLanes = 64; // embed_join_kernel: columns by partial sums

// Lanes per row: the row's chunks rounded up to a power of two, at most a wave.
// Wider rows take several column tiles of 64 chunks.
__host__ __device__ inline int lanes_per_row(int chunks) {
  int g = 4;
  while (g < chunks && g < kWave)
    g *= 2;
  return g;
}

// First column of chunk `chunk` of a row of C; C: past the row. The last chunk of
// a row that ends inside one begins earlier, so that it is whole: its first
// columns are also the chunk's before it, whose lane comes to the same values. (By
// elements, the sums of 3780 ids of 51 classes, 383 wide in bf16, took 55 us; 384
// wide 31.)
template <int V> __device__ __forceinline__ int chunk_column(int chunk, int C) {
  const int c = chunk * V;
  return c >= C ? C : C < V ? c : min(c, C - V);
}

__device__ __forceinline__ int64_t id_at(const void *ids, int is32, int64_t i) {
  return is32 ? static_cast<const int32_t *>(ids)[i] : static_cast<const int64_t *>(ids)[i];
}

// G lanes per row, 256 / G rows per workgroup; blockIdx.y: column tile.
template <typename T>
__global__ __launch_bounds__(kEmbThreads) void embed_forward_kernel(
    const void *__restrict__ ids, int is32, int64_t n, const T *__restrict__ weight,
    int64_t w_row, int64_t vocab, int C, int log_g, float scale, T *__restrict__ y) {
  using R = RowChunk<T>;
  const int lane = threadIdx.x & ((1 << log_g) - 1);
  const int64_t i =
      static_cast<int64_t>(blockIdx.x) * (kEmbThreads >> log_g) + (threadIdx.x >> log_g);
  const int c = chunk_column<R::V>(blockIdx.y * kWave + lane, C);
  if (i >= n || c >= C)
    return;
  const int64_t id = id_at(ids, is32, i);
  float v[R::V];
  R::load(weight + (id >= 0 && id < vocab ? id : 0) * w_row + c,
          id >= 0 && id < vocab ? C - c : 0, v);
#pragma unroll
  for (int e = 0; e < R::V; ++e)
    v[e] *= scale;
  R::store(y + i * C + c, C - c, v);
}

// Sort keys: the id, or `vocab` for an id outside the table.
__global__ __launch_bounds__(kEmbThreads) void embed_keys_kernel(const void *__restrict__ ids,
                                                                 int is32, int64_t n,
                                                                 uint32_t vocab,
                                                                 uint32_t *__restrict__ keys,
                                                                 int32_t *__restrict__ pos) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kEmbThreads + threadIdx.x;
  if (i >= n)
    return;
  const int64_t id = id_at(ids, is32, i);
  keys[i] = id >= 0 && id < vocab ? static_cast<uint32_t>(id) : vocab;
  pos[i] = static_cast<int32_t>(i);
}

// Keys and sort in one workgroup for up to kSmall ids: bitonic in LDS over (key,
// position) words, which are all different, so the order is the stable one.
// (100 ids 7 us, 2000 19 us, against 25 in the keys kernel and the six of a
// radix sort, and six launches less for the host; 4096 would take 33.)
constexpr int kSmall = 2048, kSmallThreads = 1024, kPosBits = 11;
static_assert(kSmall == 1 << kPosBits, "a position fits its bits");
__global__ __launch_bounds__(kSmallThreads) void embed_sort_small_kernel(
    const void *__restrict__ ids, int is32, int n, uint32_t vocab, uint32_t *__restrict__ sorted,
    int32_t *__restrict__ order) {
  __shared__ uint64_t w[kSmall];
  int m = 2; // n rounded up to a power of two; the words behind n sort last
  while (m < n)
    m *= 2;
  for (int i = threadIdx.x; i < m; i += kSmallThreads) {
    uint64_t word = ~0ull;
    if (i < n) {
      const int64_t id = id_at(ids, is32, i);
      word = (id >= 0 && id < vocab ? static_cast<uint64_t>(id) : vocab) << kPosBits | i;
    }
    w[i] = word;
  }
  // A wave's pairs at distances up to 64 lie in 128 words of its own: there no
  // step needs the other waves.
  bool apart = true; // the step before may have crossed waves
  for (int k = 2; k <= m; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      if (apart || j > kWave)
        __syncthreads();
      else
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      apart = j > kWave;
      for (int t = threadIdx.x; t < m / 2; t += kSmallThreads) {
        const int i = 2 * t - (t & (j - 1)); // pairs (i, i + j)
        const uint64_t a = w[i], b = w[i + j];
        if ((a > b) == ((i & k) == 0)) {
          w[i] = b;
          w[i + j] = a;
        }
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kSmallThreads) {
    sorted[i] = static_cast<uint32_t>(w[i] >> kPosBits);
    order[i] = static_cast<int32_t>(w[i] & (kSmall - 1));
  }
}

// start[v] = first sorted position whose key is >= v, v = 0 .. vocab: the rows
// after the key before position i, up to the key at i, start at i. The wave
// fills the gaps between its keys together. For a few ids in a large table that
// would be one wave's work (52 ids, 88325 rows: 50 us): embed_starts_search_kernel.
__global__ __launch_bounds__(kEmbThreads) void embed_starts_kernel(
    const uint32_t *__restrict__ keys, int64_t n, uint32_t vocab, int32_t *__restrict__ start,
    int32_t *__restrict__ runs) {
  if (blockIdx.x == 0 && threadIdx.x == 0)
    *runs = 0;
  constexpr int kShort = 8; // rows a lane fills by itself
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kEmbThreads + threadIdx.x;
  int64_t lo = 0, hi = -1; // rows lo .. hi start at i
  if (i <= n) {
    lo = i == 0 ? 0 : static_cast<int64_t>(keys[i - 1]) + 1;
    hi = i == n ? vocab : keys[i];
  }
  if (hi - lo < kShort)
    for (; lo <= hi; ++lo)
      start[lo] = static_cast<int32_t>(i);
  uint64_t gaps = __ballot(lo <= hi);
  while (gaps) {
    const int l = __ffsll(static_cast<unsigned long long>(gaps)) - 1;
    gaps &= gaps - 1;
    const int64_t first = __shfl(lo, l, kWave), last = __shfl(hi, l, kWave);
    const int32_t at = static_cast<int32_t>(i - lane_id() + l);
    for (int64_t v = first + lane_id(); v <= last; v += kWave)
      start[v] = at;
  }
}

// The same, each table row by a search of its own over the keys, all rows at
// once.
__global__ __launch_bounds__(kEmbThreads) void embed_starts_search_kernel(
    const uint32_t *__restrict__ keys, int64_t n, uint32_t vocab, int32_t *__restrict__ start,
    int32_t *__restrict__ runs) {
  const int64_t v = static_cast<int64_t>(blockIdx.x) * kEmbThreads + threadIdx.x;
  if (v == 0)
    *runs = 0;
  if (v > vocab)
    return;
  int32_t lo = 0, hi = static_cast<int32_t>(n);
  while (lo < hi) {
    const int32_t mid = (lo + hi) >> 1;
    if (keys[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  start[v] = lo;
}

// Sum of grad_y's rows at the sorted positions [p0, p1), at most 64 of them,
// over a lane's NC chunks: the wave's 64 / G position lanes take every (64 /
// G)-th position.
template <typename T, int NC>
__device__ __forceinline__ void sum_rows(const T *__restrict__ gy, int64_t gy_row,
                                         const int32_t *__restrict__ pos, int32_t p0, int32_t p1,
                                         const int (&c)[NC], int C, int log_g,
                                         float (&acc)[NC][RowChunk<T>::V]) {
  using R = RowChunk<T>;
  constexpr int kUnroll = NC == 1 ? 8 : NC == 2 ? 4 : 2; // rows in flight
  const int plane = lane_id() >> log_g, planes = kWave >> log_g, count = p1 - p0;
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int e = 0; e < R::V; ++e)
      acc[i][e] = 0.f;
  const int32_t mine = lane_id() < count ? pos[p0 + lane_id()] : 0;
  // every lane goes every turn: lanes hand each other the positions
  for (int p = 0; p < count; p += kUnroll * planes) {
    float v[kUnroll][NC][R::V];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int q = p + plane + u * planes;
      const T *row = gy + static_cast<int64_t>(__shfl(mine, q, kWave)) * gy_row;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        R::load(row + c[i], q < count ? C - c[i] : 0, v[u][i]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < R::V; ++e)
          acc[i][e] += v[u][i][e];
  }
  for (int off = 1 << log_g; off < kWave; off <<= 1)
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int e = 0; e < R::V; ++e)
        acc[i][e] += __shfl_xor(acc[i][e], off, kWave);
}

// Zeros, for a table most of whose rows no id names.
__global__ __launch_bounds__(kEmbThreads) void embed_clear_kernel(char *__restrict__ p,
                                                                  int64_t bytes) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kEmbThreads * 16;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kEmbThreads + threadIdx.x) * 16; i < bytes;
       i += step) {
    if (i + 16 <= bytes) {
      __builtin_nontemporal_store(v4u{0u, 0u, 0u, 0u}, reinterpret_cast<v4u_any *>(p + i));
    } else {
      for (int64_t e = i; e < bytes; e += 2) // elements of two bytes at least
        *reinterpret_cast<uint16_t *>(p + e) = 0;
    }
  }
}

// One wave per work item and column tile of 64 NC chunks. The first items, the
// longest: chunk j of the sorted positions, for the parts of long runs in it.
// A chunk meets at most two of those: one from before it (partial sum 2 j) and
// one that starts in it (2 j + 1), which then goes on the list of runs to join
// (in any order: each is joined by itself). The others: some table rows, each
// with at most kSegment positions, summed (or zeroed) and written; most rows
// of a large table are in no batch, so a wave takes up to four. SPARSE: the table
// has been cleared, and a wave takes the rows that begin at some positions.
template <typename T, int NC, bool SPARSE>
__global__ __launch_bounds__(kEmbThreads) void embed_backward_kernel(
    const T *__restrict__ gy, int64_t gy_row, const uint32_t *__restrict__ keys,
    const int32_t *__restrict__ pos, const int32_t *__restrict__ start, int64_t n, int64_t vocab,
    int C, int log_g, float scale, T *__restrict__ gw, float *__restrict__ part,
    int32_t *__restrict__ runs, int64_t item0, int rows_per_wave) {
  using R = RowChunk<T>;
  const int64_t item = item0 + static_cast<int64_t>(blockIdx.x) * (kEmbThreads / kWave) +
                       __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = lane_id() & ((1 << log_g) - 1);
  const bool writer = (lane_id() >> log_g) == 0;
  int c[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) // chunks past the row: nothing to load or write
    c[i] = chunk_column<R::V>((blockIdx.y * NC + i) * kWave + lane, C);
  float acc[NC][R::V];
  const int64_t segments = (n + kSegment - 1) / kSegment;
  if (item >= segments) {
    const int64_t first = (item - segments) * rows_per_wave;
    if (first >= (SPARSE ? n : vocab))
      return;
    int32_t at[kRowsPerWave + 1], end[kRowsPerWave];
    int64_t row[kRowsPerWave];
#pragma unroll
    for (int r = 0; r < kRowsPerWave; ++r)
      row[r] = SPARSE ? keys[min(first + r, n - 1)] : min(first + r, vocab);
#pragma unroll
    for (int r = 0; r < kRowsPerWave; ++r)
      at[r] = start[row[r]];
    at[kRowsPerWave] = SPARSE ? 0 : start[min(first + kRowsPerWave, vocab)];
#pragma unroll
    for (int r = 0; r < kRowsPerWave; ++r)
      end[r] = SPARSE ? start[min(row[r] + 1, vocab)] : at[r + 1];
#pragma unroll
    for (int r = 0; r < kRowsPerWave; ++r) {
      const int64_t v = row[r];
      if (r >= rows_per_wave)
        break;
      if (v >= vocab || end[r] - at[r] > kSegment || (SPARSE && at[r] != first + r))
        continue;
      sum_rows<T, NC>(gy, gy_row, pos, at[r], end[r], c, C, log_g, acc);
      if (writer) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
#pragma unroll
          for (int e = 0; e < R::V; ++e)
            acc[i][e] *= scale;
          R::store(gw + v * C + c[i], C - c[i], acc[i]);
        }
      }
    }
    return;
  }
  const int64_t j = item, s0 = j * kSegment, s1 = min(n, s0 + kSegment);
  for (int k = 0; k < 2; ++k) {
    // the run at the chunk's first position, if it began before it, and the
    // run at the last position, if it began inside
    const uint32_t v = keys[k == 0 ? s0 : s1 - 1];
    if (v >= vocab)
      continue;
    const int32_t p0 = start[v], p1 = start[v + 1];
    const bool before = p0 < s0;
    if (p1 - p0 <= kSegment || before != (k == 0))
      continue;
    if (!before && blockIdx.y == 0 && lane_id() == 0)
      runs[1 + atomicAdd(runs, 1)] = static_cast<int32_t>(j);
    sum_rows<T, NC>(gy, gy_row, pos, max(p0, static_cast<int32_t>(s0)),
                    min(p1, static_cast<int32_t>(s1)), c, C, log_g, acc);
    if (writer) {
      float *dst = part + (2 * j + k) * C;
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < R::V; ++e)
          if (c[i] + e < C)
            dst[c[i] + e] = acc[i][e];
    }
  }
}

// The table rows of the long runs: for each on the list the partial sums of
// its chunks, 64 lanes over the chunks by 16 columns, then a tree. The order of
// the sums depends on the chunks alone.
template <typename T>
__global__ __launch_bounds__(kJoinCols *kJoinLanes) void embed_join_kernel(
    const uint32_t *__restrict__ keys, const int32_t *__restrict__ start, int64_t n, int C,
    float scale, const float *__restrict__ part, const int32_t *__restrict__ runs,
    T *__restrict__ gw) {
  __shared__ float lds[kJoinLanes][kJoinCols];
  const int col = threadIdx.x % kJoinCols, r = threadIdx.x / kJoinCols;
  const int32_t count = runs[0];
  for (int32_t k = blockIdx.x; k < count; k += gridDim.x) {
    const int64_t j = runs[1 + k];
    const uint32_t v = keys[min(n, (j + 1) * kSegment) - 1];
    const int64_t last = (start[v + 1] - 1) / kSegment;
    for (int c0 = blockIdx.y * kJoinCols; c0 < C; c0 += gridDim.y * kJoinCols) {
      const int c = min(c0 + col, C - 1);
      float s = 0.f;
#pragma unroll 4
      for (int64_t q = j + r; q <= last; q += kJoinLanes)
        s += part[(2 * q + (q == j)) * C + c];
      __syncthreads(); // the previous columns' sums have been read
      lds[r][col] = s;
#pragma unroll
      for (int off = kJoinLanes / 2; off; off >>= 1) {
        __syncthreads();
        if (r < off)
          lds[r][col] += lds[r + off][col];
      }
      if (r == 0 && c0 + col < C)
        gw[static_cast<int64_t>(v) * C + c] = from_f32<T>(lds[0][col] * scale);
    }
  }
}

// ------------------------------------------------------------------ host

void check_embed(int64_t n, int64_t vocab, int32_t C) {
  RHIP_CHECK_ARG(n >= 0 && vocab >= 0 && C >= 1, "bad sizes");
  if (n > INT32_MAX - kSegment || vocab > INT32_MAX - 1)
    throw Error(RHIP_ERR_UNSUPPORTED, "ids and table rows must stay below 2^31 - 64");
}
void check_embed_type(int32_t dtype, int32_t C) {
  if (dtype != RHIP_F32 && dtype != RHIP_BF16)
    throw Error(RHIP_ERR_UNSUPPORTED, "dtype must be RHIP_F32 or RHIP_BF16");
  // column tiles of 64 chunks along the grid's second axis
  if (ceil_div(C, kWave * (dtype == RHIP_F32 ? RowChunk<float>::V : RowChunk<__bf16>::V)) > 65535)
    throw Error(RHIP_ERR_UNSUPPORTED, "an embedding takes at most 65535 x 64 chunks of 16 bytes");
}

struct EmbedWs {
  uint32_t *keys, *sorted;
  int32_t *pos, *order, *start;
  int32_t *runs; // how many long runs there are, then the chunk each starts in
  float *part;
  void *sort;
  size_t sort_bytes;
};
EmbedWs carve_embed(Carve &cv, int64_t n, int64_t vocab, int32_t C) {
  EmbedWs w{};
  const int64_t m = std::max<int64_t>(n, 1);
  w.keys = cv.take<uint32_t>(m);
  w.sorted = cv.take<uint32_t>(m);
  w.pos = cv.take<int32_t>(m);
  w.order = cv.take<int32_t>(m);
  w.start = cv.take<int32_t>(vocab + 2);
  w.runs = cv.take<int32_t>(1 + ceil_div(m, kSegment));
  w.part = cv.take<float>(2 * static_cast<size_t>(ceil_div(m, kSegment)) * C);
  w.sort_bytes = sort_pairs_u32_bytes(m);
  w.sort = cv.take<char>(w.sort_bytes);
  return w;
}

int log2_of(int v) { return 31 - __builtin_clz(static_cast<unsigned>(v)); }
int bits_of(uint64_t v) { return 64 - __builtin_clzll(v | 1); }

template <typename F> void with_embed_type(int32_t dtype, F &&f) {
  if (dtype == RHIP_F32)
    f(float{});
  else
    f(__bf16{});
}

} // namespace
} // namespace rhip

using namespace rhip;

extern "C" int rhip_embed_forward(const void *ids, int32_t ids_int32, int64_t n,
                                  const void *weight, int64_t weight_row, int64_t vocabulary,
                                  int32_t C, float scale, void *y, int32_t dtype,
                                  hipStream_t stream) {
  return guarded([&] {
    check_embed_type(dtype, C);
    check_embed(n, vocabulary, C);
    if (n == 0)
      return;
    RHIP_CHECK_ARG(ids && y, "ids and y are required");
    RHIP_CHECK_ARG(vocabulary == 0 || weight, "weight is required");
    with_embed_type(dtype, [&](auto t) {
      using T = decltype(t);
      const int chunks = static_cast<int>(ceil_div(C, RowChunk<T>::V));
      const int g = lanes_per_row(chunks);
      const int64_t most = max_groups(kEmbThreads) * (kEmbThreads / g);
      for (int64_t i = 0; i < n; i += most) { // more rows than one launch takes
        const int64_t rows = std::min(n - i, most);
        hipLaunchKernelGGL((embed_forward_kernel<T>),
                           dim3(static_cast<unsigned>(ceil_div(rows, kEmbThreads / g)),
                                static_cast<unsigned>(ceil_div(chunks, kWave))),
                           dim3(kEmbThreads), 0, stream,
                           static_cast<const char *>(ids) + i * (ids_int32 ? 4 : 8), ids_int32,
                           rows, static_cast<const T *>(weight), weight_row, vocabulary, C,
                           log2_of(g), scale, static_cast<T *>(y) + i * C);
        RHIP_LAUNCH_CHECK();
      }
    });
  });
}

extern "C" int rhip_embed_workspace_bytes(int64_t n, int64_t vocabulary, int32_t C,
                                          size_t *bytes) {
  return guarded([&] {
    RHIP_CHECK_ARG(bytes != nullptr, "bytes is null");
    check_embed(n, vocabulary, C);
    Carve cv(nullptr, 0);
    carve_embed(cv, n, vocabulary, C);
    *bytes = cv.used + 256;
  });
}

extern "C" int rhip_embed_backward(const void *grad_y, int64_t grad_y_row, const void *ids,
                                   int32_t ids_int32, int64_t n, int64_t vocabulary, int32_t C,
                                   float scale, void *grad_weight, int32_t dtype,
                                   void *workspace, size_t ws_bytes, hipStream_t stream) {
  return guarded([&] {
    check_embed_type(dtype, C);
    check_embed(n, vocabulary, C);
    if (vocabulary == 0)
      return;
    RHIP_CHECK_ARG(grad_weight && workspace, "grad_weight and workspace are required");
    RHIP_CHECK_ARG(n == 0 || (grad_y && ids), "grad_y and ids are required");
    Carve cv(workspace, ws_bytes);
    const EmbedWs w = carve_embed(cv, n, vocabulary, C);
    if (n > 0 && n <= kSmall) {
      hipLaunchKernelGGL(embed_sort_small_kernel, dim3(1), dim3(kSmallThreads), 0, stream, ids,
                         ids_int32, static_cast<int>(n), static_cast<uint32_t>(vocabulary),
                         w.sorted, w.order);
      RHIP_LAUNCH_CHECK();
    } else if (n > 0) {
      hipLaunchKernelGGL(embed_keys_kernel, dim3(static_cast<unsigned>(ceil_div(n, kEmbThreads))),
                         dim3(kEmbThreads), 0, stream, ids, ids_int32, n,
                         static_cast<uint32_t>(vocabulary), w.keys, w.pos);
      RHIP_LAUNCH_CHECK();
      sort_pairs_u32(w.sort, w.sort_bytes, w.keys, w.sorted, w.pos, w.order, n,
                     bits_of(static_cast<uint64_t>(vocabulary)), stream);
    }
    const bool sparse = vocabulary > kSparse * n;
    if (sparse)
      hipLaunchKernelGGL(embed_starts_search_kernel,
                         dim3(static_cast<unsigned>(ceil_div(vocabulary + 1, kEmbThreads))),
                         dim3(kEmbThreads), 0, stream, w.sorted, n,
                         static_cast<uint32_t>(vocabulary), w.start, w.runs);
    else
      hipLaunchKernelGGL(embed_starts_kernel,
                         dim3(static_cast<unsigned>(ceil_div(n + 1, kEmbThreads))),
                         dim3(kEmbThreads), 0, stream, w.sorted, n,
                         static_cast<uint32_t>(vocabulary), w.start, w.runs);
    RHIP_LAUNCH_CHECK();
    with_embed_type(dtype, [&](auto t) {
      using T = decltype(t);
      const int chunks = static_cast<int>(ceil_div(C, RowChunk<T>::V));
      const int64_t segments = ceil_div(n, kSegment);
      // chunks per lane: whole rows in one wave as far as registers go, unless
      // that leaves too few waves (8340 labels of 3 classes, 986 wide: 53 us
      // with two chunks per lane, 41 with one)
      // rows one after another only where waves are many: few rows with 64
      // positions each would leave the chip to some waves. (1047 ids of 16 classes,
      // 1973 wide in bf16, this kernel: 103 us four to a wave, 45 one; 40000 ids of
      // 200000 rows, 256 wide, the whole gradient: 100 us and 127.)
      const int64_t units = sparse ? n : vocabulary;
      const int rows = units * ceil_div(chunks, kWave) >= kManyRows ? kRowsPerWave : 1;
      const int64_t items = ceil_div(units, rows) + segments;
      if (sparse) {
        const int64_t bytes = vocabulary * C * static_cast<int64_t>(sizeof(T));
        hipLaunchKernelGGL(embed_clear_kernel,
                           dim3(static_cast<unsigned>(
                               std::min<int64_t>(ceil_div(bytes, kEmbThreads * 16), 8192))),
                           dim3(kEmbThreads), 0, stream, static_cast<char *>(grad_weight), bytes);
        RHIP_LAUNCH_CHECK();
        if (n == 0)
          return;
      }
      const int64_t fill = 4096 / items; // column tiles that fill the chip
      auto launch_rows = [&](auto nc, auto s) {
        constexpr int NC = decltype(nc)::value;
        constexpr bool SPARSE = decltype(s)::value;
        const int64_t most = max_groups(kEmbThreads) * (kEmbThreads / kWave);
        for (int64_t i = 0; i < items; i += most) {
          hipLaunchKernelGGL((embed_backward_kernel<T, NC, SPARSE>),
                             dim3(static_cast<unsigned>(ceil_div(std::min(items - i, most),
                                                                 kEmbThreads / kWave)),
                                  static_cast<unsigned>(ceil_div(chunks, kWave * NC))),
                             dim3(kEmbThreads), 0, stream, static_cast<const T *>(grad_y),
                             grad_y_row, w.sorted, w.order, w.start, n, vocabulary, C,
                             log2_of(lanes_per_row(chunks)), scale,
                             static_cast<T *>(grad_weight), w.part, w.runs, i, rows);
          RHIP_LAUNCH_CHECK();
        }
      };
      auto launch = [&](auto nc) {
        if (sparse)
          launch_rows(nc, std::true_type{});
        else
          launch_rows(nc, std::false_type{});
      };
      if (chunks <= kWave || fill >= ceil_div(chunks, kWave))
        launch(std::integral_constant<int, 1>{});
      else if (chunks <= 2 * kWave || fill >= ceil_div(chunks, 2 * kWave))
        launch(std::integral_constant<int, 2>{});
      else
        launch(std::integral_constant<int, 4>{});
      if (segments > 0) {
        // about 512 workgroups over the runs (no more than table rows) and columns
        const int64_t runs = std::min<int64_t>({segments, vocabulary, 64});
        const int64_t tiles =
            std::min<int64_t>(ceil_div(C, kJoinCols), std::max<int64_t>(1, 512 / runs));
        hipLaunchKernelGGL((embed_join_kernel<T>),
                           dim3(static_cast<unsigned>(runs), static_cast<unsigned>(tiles)),
                           dim3(kJoinCols * kJoinLanes), 0, stream, w.sorted, w.start, n, C,
                           scale, w.part, w.runs, static_cast<T *>(grad_weight));
        RHIP_LAUNCH_CHECK();
      }
    });
  });
}
