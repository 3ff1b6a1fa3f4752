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
constexpr int kSegment = 64; // positions a group of lanes sums by itself, at most
constexpr int kJoinLanes = 16; // partial sums added side by side by embed_join_kernel

// Lanes per row: the row's chunks rounded up to a power of two, at most a wave.
// Wider rows take several column tiles of 64 chunks.
__host__ __device__ inline int lanes_per_row(int chunks) {
  int g = 4;
  while (g < chunks && g < kWave)
    g *= 2;
  return g;
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
  const int c = (blockIdx.y * kWave + lane) * R::V;
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

// start[v] = first sorted position whose key is >= v, v = 0 .. vocab: the rows
// after the key before position i, up to the key at i, start at i. The wave
// fills the gaps between its keys together, so a few tokens in a large table
// cost no more than many.
__global__ __launch_bounds__(kEmbThreads) void embed_starts_kernel(
    const uint32_t *__restrict__ keys, int64_t n, uint32_t vocab, int32_t *__restrict__ start) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kEmbThreads + threadIdx.x;
  int64_t lo = 0, hi = -1; // rows lo .. hi start at i
  if (i <= n) {
    lo = i == 0 ? 0 : static_cast<int64_t>(keys[i - 1]) + 1;
    hi = i == n ? vocab : keys[i];
  }
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

// Sum of grad_y's rows at sorted positions [p0, p1) over one chunk column:
// the wave's 64 / G position lanes take every (64 / G)-th position.
template <typename T>
__device__ __forceinline__ void sum_rows(const T *__restrict__ gy, int64_t gy_row,
                                         const int32_t *__restrict__ pos, int32_t p0, int32_t p1,
                                         int c, int C, int log_g,
                                         float (&acc)[RowChunk<T>::V]) {
  using R = RowChunk<T>;
  constexpr int kUnroll = 4;
  const int plane = lane_id() >> log_g, planes = kWave >> log_g;
#pragma unroll
  for (int e = 0; e < R::V; ++e)
    acc[e] = 0.f;
  for (int32_t p = p0 + plane; p < p1; p += kUnroll * planes) {
    float v[kUnroll][R::V];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int32_t q = p + u * planes;
      R::load(gy + static_cast<int64_t>(pos[min(q, p1 - 1)]) * gy_row + c, q < p1 ? C - c : 0,
              v[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int e = 0; e < R::V; ++e)
        acc[e] += v[u][e];
  }
  for (int off = 1 << log_g; off < kWave; off <<= 1)
#pragma unroll
    for (int e = 0; e < R::V; ++e)
      acc[e] += __shfl_xor(acc[e], off, kWave);
}

// One wave per work item and column tile. Items [0, vocab): a table row with
// at most kSegment positions, summed (or zeroed) and written. Items vocab + j:
// chunk j of the sorted positions, for the parts of longer runs in it. A chunk
// meets at most two of those: one from before it (partial sum 2 j) and one
// that starts in it (2 j + 1).
template <typename T>
__global__ __launch_bounds__(kEmbThreads) void embed_backward_kernel(
    const T *__restrict__ gy, int64_t gy_row, const uint32_t *__restrict__ keys,
    const int32_t *__restrict__ pos, const int32_t *__restrict__ start, int64_t n, int64_t vocab,
    int C, int log_g, float scale, T *__restrict__ gw, float *__restrict__ part) {
  using R = RowChunk<T>;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kEmbThreads / kWave) +
                       threadIdx.x / kWave;
  const int lane = lane_id() & ((1 << log_g) - 1);
  const int c = (blockIdx.y * kWave + lane) * R::V;
  const bool writer = (lane_id() >> log_g) == 0 && c < C;
  const int cc = min(c, C - 1), left = c < C ? C : cc; // lanes past the row load nothing
  float acc[R::V];
  if (item < vocab) {
    const int32_t p0 = start[item], p1 = start[item + 1];
    if (p1 - p0 > kSegment)
      return;
    sum_rows(gy, gy_row, pos, p0, p1, cc, left, log_g, acc);
    if (writer) {
#pragma unroll
      for (int e = 0; e < R::V; ++e)
        acc[e] *= scale;
      R::store(gw + item * C + c, C - c, acc);
    }
    return;
  }
  const int64_t j = item - vocab;
  const int64_t s0 = j * kSegment, s1 = min(n, s0 + kSegment);
  if (s0 >= n)
    return;
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
    sum_rows(gy, gy_row, pos, max(p0, static_cast<int32_t>(s0)),
             min(p1, static_cast<int32_t>(s1)), cc, left, log_g, acc);
    if (writer) {
      float *dst = part + (2 * j + k) * C + c;
#pragma unroll
      for (int e = 0; e < R::V; ++e)
        if (c + e < C)
          dst[e] = acc[e];
    }
  }
}

// The table row of the run that starts in chunk j, if it is a long one: its
// chunks' partial sums, 16 lanes over the chunks by 16 columns, then in lane
// order.
template <typename T>
__global__ __launch_bounds__(kEmbThreads) void embed_join_kernel(
    const uint32_t *__restrict__ keys, const int32_t *__restrict__ start, int64_t n,
    int64_t vocab, int C, float scale, const float *__restrict__ part, T *__restrict__ gw) {
  constexpr int kCols = kEmbThreads / kJoinLanes;
  __shared__ float lds[kJoinLanes][kCols];
  const int64_t j = blockIdx.x, s0 = j * kSegment, s1 = min(n, s0 + kSegment);
  const uint32_t v = keys[s1 - 1];
  if (v >= vocab)
    return;
  const int32_t p0 = start[v], p1 = start[v + 1];
  if (p1 - p0 <= kSegment || p0 < s0)
    return;
  const int64_t last = (p1 - 1) / kSegment;
  const int col = threadIdx.x % kCols, r = threadIdx.x / kCols;
  for (int c0 = blockIdx.y * kCols; c0 < C; c0 += gridDim.y * kCols) {
    const int c = c0 + col;
    float s = 0.f;
    if (c < C)
      for (int64_t q = j + r; q <= last; q += kJoinLanes)
        s += part[(2 * q + (q == j)) * C + c];
    __syncthreads(); // the previous tile's sums have been read
    lds[r][col] = s;
    __syncthreads();
    if (r == 0 && c < C) {
#pragma unroll
      for (int k = 1; k < kJoinLanes; ++k)
        s += lds[k][col];
      gw[static_cast<int64_t>(v) * C + c] = from_f32<T>(s * scale);
    }
  }
}

// ------------------------------------------------------------------ host

void check_embed(int64_t n, int64_t vocab, int32_t C) {
  RHIP_CHECK_ARG(n >= 0 && vocab >= 0 && C >= 1, "bad sizes");
  if (n > INT32_MAX - kSegment || vocab > INT32_MAX - 1)
    throw Error(RHIP_ERR_UNSUPPORTED, "ids and table rows must stay below 2^31 - 64");
}
void check_embed_type(int32_t dtype) {
  if (dtype != RHIP_F32 && dtype != RHIP_BF16)
    throw Error(RHIP_ERR_UNSUPPORTED, "dtype must be RHIP_F32 or RHIP_BF16");
}

struct EmbedWs {
  uint32_t *keys, *sorted;
  int32_t *pos, *order, *start;
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
    check_embed_type(dtype);
    check_embed(n, vocabulary, C);
    if (n == 0)
      return;
    RHIP_CHECK_ARG(ids && y, "ids and y are required");
    RHIP_CHECK_ARG(vocabulary == 0 || weight, "weight is required");
    with_embed_type(dtype, [&](auto t) {
      using T = decltype(t);
      const int chunks = static_cast<int>(ceil_div(C, RowChunk<T>::V));
      const int g = lanes_per_row(chunks);
      hipLaunchKernelGGL((embed_forward_kernel<T>),
                         dim3(static_cast<unsigned>(ceil_div(n, kEmbThreads / g)),
                              static_cast<unsigned>(ceil_div(chunks, kWave))),
                         dim3(kEmbThreads), 0, stream, ids, ids_int32, n,
                         static_cast<const T *>(weight), weight_row, vocabulary, C, log2_of(g),
                         scale, static_cast<T *>(y));
      RHIP_LAUNCH_CHECK();
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
    check_embed_type(dtype);
    check_embed(n, vocabulary, C);
    if (vocabulary == 0)
      return;
    RHIP_CHECK_ARG(grad_weight && workspace, "grad_weight and workspace are required");
    RHIP_CHECK_ARG(n == 0 || (grad_y && ids), "grad_y and ids are required");
    Carve cv(workspace, ws_bytes);
    const EmbedWs w = carve_embed(cv, n, vocabulary, C);
    if (n > 0) {
      hipLaunchKernelGGL(embed_keys_kernel, dim3(static_cast<unsigned>(ceil_div(n, kEmbThreads))),
                         dim3(kEmbThreads), 0, stream, ids, ids_int32, n,
                         static_cast<uint32_t>(vocabulary), w.keys, w.pos);
      RHIP_LAUNCH_CHECK();
      sort_pairs_u32(w.sort, w.sort_bytes, w.keys, w.sorted, w.pos, w.order, n,
                     bits_of(static_cast<uint64_t>(vocabulary)), stream);
    }
    hipLaunchKernelGGL(embed_starts_kernel,
                       dim3(static_cast<unsigned>(ceil_div(n + 1, kEmbThreads))),
                       dim3(kEmbThreads), 0, stream, w.sorted, n,
                       static_cast<uint32_t>(vocabulary), w.start);
    RHIP_LAUNCH_CHECK();
    with_embed_type(dtype, [&](auto t) {
      using T = decltype(t);
      const int chunks = static_cast<int>(ceil_div(C, RowChunk<T>::V));
      const int64_t segments = ceil_div(n, kSegment);
      hipLaunchKernelGGL((embed_backward_kernel<T>),
                         dim3(static_cast<unsigned>(
                                  ceil_div(vocabulary + segments, kEmbThreads / kWave)),
                              static_cast<unsigned>(ceil_div(chunks, kWave))),
                         dim3(kEmbThreads), 0, stream, static_cast<const T *>(grad_y),
                         grad_y_row, w.sorted, w.order, w.start, n, vocabulary, C,
                         log2_of(lanes_per_row(chunks)), scale, static_cast<T *>(grad_weight),
                         w.part);
      RHIP_LAUNCH_CHECK();
      if (segments > 0) {
        const unsigned tiles = static_cast<unsigned>(
            std::min<int64_t>(ceil_div(C, kEmbThreads / kJoinLanes), 64));
        hipLaunchKernelGGL((embed_join_kernel<T>), dim3(static_cast<unsigned>(segments), tiles),
                           dim3(kEmbThreads), 0, stream, w.sorted, w.start, n, vocabulary, C,
                           scale, w.part, static_cast<T *>(grad_weight));
        RHIP_LAUNCH_CHECK();
      }
    });
  });
}
