// Gated feed-forward block on gfx950, forward and backward:
//   g = x gate^T, u = x up^T, h = act(g) u, y = h down^T.
// One kernel makes both projections of a tile, the activation and the product:
// its workgroups' tiles hold the same columns of g and u, so h (and for the
// backward g and u) leave from registers. Backward, with dh = dy down:
//   dg = dh u act'(g), du = dh act(g)      in the epilogue of that product,
//   dx = dg gate + du up                   one product over 2 H,
//   dgate = dg^T x, dup = du^T x           one launch,
//   ddown = dy^T h.
//
// All are tiles of gemm_device.hpp's product, bound by the matrix cores. Where
// tiles leave part of the chip idle their k is shared by workgroups, whose fp32
// sums a second kernel adds in order and finishes. The forward of few rows (single
// tokens) goes to a kernel that streams the weights through registers, bound by
// their bytes.
//
// Operands that do not hold aligned, whole 16-byte chunks (odd widths,
// unaligned views) are laid out once per call in the workspace, zeros behind
// their rows' ends.
//
// bf16: h, dg and du are rounded to bf16, as operands of the matrix cores. g and
// u are kept for the backward to 16 significant bits (a bf16 plane each, the
// next eight bits of both in a third), so that they add nothing to that.
#include <climits>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "gemm_device.hpp"

namespace rhip {
namespace {

constexpr int kGatedThreads = 256; // of the kernels that join and pack
using LargeTiles = GemmShape<2, 4, 4, 2>; // 256 x 256, eight waves, one workgroup to a CU
using SmallTiles = GemmShape<2, 2, 2, 2>; // 128 x 128, four waves, two workgroups
using TinyTiles = GemmShape<2, 2, 1, 1>;  // 64 x 64, four
using TinyPairs = GemmShape<2, 2, 1, 2>;  // 64 x 64 of both projections

// ------------------------------------------------------------- activation

__device__ __forceinline__ float act_exp(float v, __bf16) { return exp2_fast(v * kLog2e); }
__device__ __forceinline__ float act_exp(float v, float) { return expf(v); }
__device__ __forceinline__ float act_inv(float v, __bf16) { return __builtin_amdgcn_rcpf(v); }
__device__ __forceinline__ float act_inv(float v, float) { return 1.f / v; }

// The activation and its derivative at g, as exact as T's results need.
template <typename T>
__device__ __forceinline__ float activation(int32_t kind, float g, float &derivative) {
  if (kind == RHIP_ACT_SILU) {
    const float s = act_inv(1.f + act_exp(-g, T{}), T{});
    derivative = s * fmaf(g, 1.f - s, 1.f);
    return g * s;
  }
  const float half = 0.5f * erfcf(g * -0.70710678118654752f);
  derivative = fmaf(g * 0.39894228040143268f, act_exp(-0.5f * g * g, T{}), half);
  return g * half;
}

// g and u for the backward: fp32 as they are; bf16 the upper 24 bits, rounded.
__device__ __forceinline__ uint32_t upper24(float v) {
  const uint32_t b = __float_as_uint(v);
  return (v != v ? b : b + 0x80u) >> 8;
}

struct GatedSaved { // planes [n, pitch]
  void *h, *g, *u;
  uint16_t *low; // bf16: the eight bits behind g's and u's planes
};

// E values of 32 bits from one 16-byte chunk (fp32) or of 16 bits (bf16's planes).
template <typename T> struct SavedChunk {
  static constexpr int E = 16 / sizeof(T);
  // whole 16-byte chunks of the planes at `at`
  __device__ static __forceinline__ void load(const GatedSaved &s, int64_t at, float (&g)[E],
                                              float (&u)[E]) {
    if constexpr (sizeof(T) == 4) {
      const v4f a = *reinterpret_cast<const v4f *>(static_cast<const float *>(s.g) + at);
      const v4f b = *reinterpret_cast<const v4f *>(static_cast<const float *>(s.u) + at);
#pragma unroll
      for (int i = 0; i < E; ++i)
        g[i] = a[i], u[i] = b[i];
    } else {
      const v4u a = *reinterpret_cast<const v4u *>(static_cast<const uint16_t *>(s.g) + at);
      const v4u b = *reinterpret_cast<const v4u *>(static_cast<const uint16_t *>(s.u) + at);
      const v4u c = *reinterpret_cast<const v4u *>(s.low + at);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int sh = 16 * (i % 2);
        g[i] = __uint_as_float(a[i / 2] >> sh << 16 | ((c[i / 2] >> sh) & 0xffu) << 8);
        u[i] = __uint_as_float(b[i / 2] >> sh << 16 | ((c[i / 2] >> sh) & 0xff00u));
      }
    }
  }
  __device__ static __forceinline__ void store(const GatedSaved &s, int64_t at,
                                               const float (&g)[E], const float (&u)[E]) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<v4f *>(static_cast<float *>(s.g) + at) = v4f{g[0], g[1], g[2], g[3]};
      *reinterpret_cast<v4f *>(static_cast<float *>(s.u) + at) = v4f{u[0], u[1], u[2], u[3]};
    } else {
      v4u a, b, c;
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const uint32_t g0 = upper24(g[i]), g1 = upper24(g[i + 1]);
        const uint32_t u0 = upper24(u[i]), u1 = upper24(u[i + 1]);
        a[i / 2] = g0 >> 8 | (g1 >> 8) << 16;
        b[i / 2] = u0 >> 8 | (u1 >> 8) << 16;
        c[i / 2] = (g0 & 0xffu) | (u0 & 0xffu) << 8 | (g1 & 0xffu) << 16 | (u1 & 0xffu) << 24;
      }
      *reinterpret_cast<v4u *>(static_cast<uint16_t *>(s.g) + at) = a;
      *reinterpret_cast<v4u *>(static_cast<uint16_t *>(s.u) + at) = b;
      *reinterpret_cast<v4u *>(s.low + at) = c;
    }
  }
};

template <typename T, int E> __device__ __forceinline__ void put_chunk(T *p, const float (&v)[E]) {
  T e[E];
#pragma unroll
  for (int i = 0; i < E; ++i)
    e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<v4u *>(p) = __builtin_bit_cast(v4u, e);
}

// ---------------------------------------------------------------- products

// Tiles of whose sums a workgroup may have a part: in bf16 tiles are cut evenly, so
// its own; fp32's parts begin and end anywhere, so a last one beside the first.
constexpr int part_tiles(bool f32) { return f32 ? 2 : 1; }
template <typename T> constexpr int kPartTiles = part_tiles(sizeof(T) == 4);

enum GatedStage {
  kProject, // h (and the saved planes) from x, gate, up
  kPlain,   // one matrix of results
  kHidden   // dg, du from dy, down and the saved planes
};

struct GatedArgs {
  GemmSide y, x;
  int32_t tiles_i, tiles_j, k_tiles;
  int32_t outs;       // results, each with its own y matrix
  int32_t parts;      // workgroups that share the work
  int32_t rows, cols; // of the results
  void *out[2];
  int64_t out_row;
  float *part; // fp32 sums of tiles that several workgroups share: kPartTiles for each
  GatedSaved saved;
  int64_t pitch; // of h's, dg's, du's and the saved planes' rows
  void *dg, *du;
  int32_t keep; // kProject: whether to write the saved planes
  int32_t kind; // activation
};

// One 16-byte chunk (of T) of the results' rows: h and the saved planes from g
// and u (v[0], v[1]), or dg and du from dh (v[0]). The columns behind the last,
// `left` away, which fill the rows to whole chunks, are zeros.
template <typename T, GatedStage STAGE>
__device__ __forceinline__ void finish_chunk(const GatedArgs &a, int64_t at, int32_t left,
                                             float (&v)[2][16 / sizeof(T)]) {
  constexpr int E = 16 / sizeof(T);
  float g[E], u[E], o[E];
  if constexpr (STAGE == kProject) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      g[i] = i < left ? v[0][i] : 0.f;
      u[i] = i < left ? v[1][i] : 0.f;
      float d;
      o[i] = activation<T>(a.kind, g[i], d) * u[i];
    }
    put_chunk(static_cast<T *>(a.saved.h) + at, o);
    if (a.keep)
      SavedChunk<T>::store(a.saved, at, g, u);
  } else {
    SavedChunk<T>::load(a.saved, at, g, u);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float dh = i < left ? v[0][i] : 0.f;
      float d;
      const float act = activation<T>(a.kind, g[i], d);
      o[i] = dh * u[i] * d;
      u[i] = dh * act;
    }
    put_chunk(static_cast<T *>(a.dg) + at, o);
    put_chunk(static_cast<T *>(a.du) + at, u);
  }
}

// E fp32 values of a strip's row.
template <typename S, int E>
__device__ __forceinline__ void strip_values(const char *strip, int r, int c, float (&v)[E]) {
#pragma unroll
  for (int i = 0; i < E; i += 4) {
    const v4u u = S::chunk(strip, r, c + i);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[i + e] = __uint_as_float(u[e]);
  }
}

// A tile's results from the waves' sums.
template <typename T, typename P, GatedStage STAGE>
__device__ __forceinline__ void finish_tile(const GatedArgs &a, char *lds, int32_t which,
                                            int32_t i0, int32_t j0,
                                            v16f (&acc)[P::NJ][P::NI]) {
  constexpr int E = 16 / sizeof(T), kHalf = P::kHalves;
  constexpr int NB = P::NJ / kHalf; // blocks of columns of a wave
  const int w = wave_uniform(threadIdx.x / kWave);
  const int32_t col0 = j0 + (w % P::WJ) * NB * 32;
  char *strip = lds + w * P::kStrip;
#pragma unroll
  for (int b = 0; b < P::NI; ++b) {
    const int32_t row0 = i0 + ((w / P::WJ) * P::NI + b) * 32;
    const int32_t rows = a.rows - row0;
    if constexpr (STAGE == kPlain) {
      using S = GemmStrip<T, NB>;
      S::put(strip, [&](int c, int r) { return from_f32<T>(acc[c][b][r]); });
      __builtin_amdgcn_wave_barrier();
      T *to = static_cast<T *>(a.out[which]) + row0 * a.out_row + col0;
      S::template walk<E>([&](int r, int c) {
        if (r < rows)
          store_chunk(to + r * a.out_row + c, S::chunk(strip, r, c), a.cols - col0 - c);
      });
    } else {
      using S = GemmStrip<float, NB>;
      static_assert(kHalf * S::kBytes <= P::kStrip, "a wave's strips fit its LDS");
      S::put(strip, [&](int c, int r) { return acc[c][b][r]; });
      if constexpr (STAGE == kProject)
        S::put(strip + S::kBytes, [&](int c, int r) { return acc[c + NB][b][r]; });
      __builtin_amdgcn_wave_barrier();
      S::template walk<E>([&](int r, int c) {
        if (r < rows && col0 + c < a.pitch) {
          float v[2][E];
          strip_values<S, E>(strip, r, c, v[0]);
          if constexpr (STAGE == kProject)
            strip_values<S, E>(strip + S::kBytes, r, c, v[1]);
          finish_chunk<T, STAGE>(a, (row0 + static_cast<int64_t>(r)) * a.pitch + col0 + c,
                                 a.cols - col0 - c, v);
        }
      });
    }
    __builtin_amdgcn_wave_barrier(); // the strip is free
  }
}

// The waves' sums as they are: [halves][BI, BJ / halves] at `to`.
template <typename P>
__device__ __forceinline__ void keep_tile(char *lds, float *to, v16f (&acc)[P::NJ][P::NI]) {
  constexpr int kHalf = P::kHalves, NB = P::NJ / kHalf, kRow = P::BJ / kHalf;
  using S = GemmStrip<float, NB>;
  const int w = wave_uniform(threadIdx.x / kWave);
  char *strip = lds + w * P::kStrip;
#pragma unroll
  for (int h = 0; h < kHalf; ++h)
#pragma unroll
    for (int b = 0; b < P::NI; ++b) {
      S::put(strip, [&](int c, int r) { return acc[c + h * NB][b][r]; });
      __builtin_amdgcn_wave_barrier();
      float *at = to + (h * P::BI + ((w / P::WJ) * P::NI + b) * 32) * kRow + (w % P::WJ) * NB * 32;
      S::template walk<4>([&](int r, int c) {
        *reinterpret_cast<v4u *>(at + r * kRow + c) = S::chunk(strip, r, c);
      });
      __builtin_amdgcn_wave_barrier();
    }
}

// SHARED: the work is one line of tiles of k, of which every workgroup has an
// equal part: whole tiles, and at its ends parts of tiles, whose sums the join
// adds. Otherwise a workgroup has a tile.
//
// 8192 rows, 2048 channels, 5504 hidden, bf16: g, u and h 400 us (920 TFLOP/s: the
// activation and what it saves follow the sums), y 169 (1090), dg and du 270 (their
// bytes alone 94), dx 310 (1190), dgate and dup 380, ddown 206; the library's
// products alone reach 1300 to 1390. 8320 rows, 256 channels, 683 hidden, fp32: g,
// u and h 70 us (84 TFLOP/s), y 36 and a join of 8, dg and du 45, dx 61 and 8,
// dgate and dup 62 and 5, ddown 35 and 6; a tile to every workgroup, or each
// tile's k in two or four, took 407 us in all where this takes 345.
template <typename T, typename SHAPE, bool YACROSS, bool XACROSS, GemmPair PAIR, GatedStage STAGE,
          bool SHARED>
__global__ __launch_bounds__(SHAPE::kThreads, 2) void gated_product_kernel(GatedArgs a) {
  using P = Gemm<T, SHAPE, YACROSS, XACROSS, PAIR>;
  __shared__ alignas(16) char lds[P::kLds];
  uint32_t place;
  if (!gemm_place(a.parts, place))
    return;
  int32_t ti, tj, which;
  v16f acc[P::NJ][P::NI];
  auto sum = [&](uint32_t t, int32_t kt0, int32_t kt1) {
    gemm_tile(a.tiles_i, a.tiles_j, t, ti, tj, which);
    P::run(lds, a.y, static_cast<const T *>(a.y.p[which]), a.x, ti * P::BI,
           tj * (P::BJ / P::kHalves), kt0, kt1, acc);
  };
  auto finish = [&] {
    finish_tile<T, P, STAGE>(a, lds, which, ti * P::BI, tj * (P::BJ / P::kHalves), acc);
  };
  if constexpr (!SHARED) {
    sum(place, 0, a.k_tiles);
    finish();
  } else {
    const uint32_t tiles = static_cast<uint32_t>(a.tiles_i) * a.tiles_j * a.outs;
    const int64_t units = static_cast<int64_t>(tiles) * a.k_tiles;
    // tiles cut evenly: those of one slice of k follow one another, as they
    // share what they load
    if (a.parts % tiles == 0)
      place = place % tiles * (a.parts / tiles) + place / tiles;
    const int64_t first = gemm_cut(units, a.parts, place);
    const int64_t end = gemm_cut(units, a.parts, place + 1);
    for (int64_t u = first; u < end;) {
      const uint32_t t = static_cast<uint32_t>(u / a.k_tiles);
      const int32_t kt0 = static_cast<int32_t>(u - static_cast<int64_t>(t) * a.k_tiles);
      const int32_t kt1 =
          static_cast<int32_t>(min<int64_t>(a.k_tiles, kt0 + (end - u)));
      sum(t, kt0, kt1);
      if (kt0 == 0 && kt1 == a.k_tiles)
        finish();
      else
        keep_tile<P>(lds,
                     a.part + (static_cast<int64_t>(place) * kPartTiles<T> +
                               (kPartTiles<T> == 1 || u == first ? 0 : 1)) *
                                  P::BI * P::BJ,
                     acc);
      u += kt1 - kt0;
      __syncthreads(); // the strips are free for the next tile
    }
  }
}

// Adds the sums of tiles that several workgroups share, in their order, and
// finishes them as the products' own epilogues do: a 16-byte chunk (of T) for
// PARTS threads, which take every PARTS-th sum each and add up in LDS.
template <typename T, typename SHAPE, GemmPair PAIR, GatedStage STAGE, int PARTS>
__global__ __launch_bounds__(kGatedThreads) void gated_join_kernel(GatedArgs a) {
  constexpr int E = STAGE == kPlain ? 4 : 16 / sizeof(T);
  constexpr int kHalf = PAIR == kGemmHalves ? 2 : 1, kSums = kHalf * E;
  constexpr int BI = SHAPE::BI, kRow = SHAPE::BJ / kHalf, kChunks = kRow / E; // of a tile's row
  constexpr int kOwn = kGatedThreads / PARTS;             // chunks of a workgroup
  constexpr int kGroups = BI * kChunks / kOwn;            // workgroups of a tile
  const uint32_t tiles = static_cast<uint32_t>(a.tiles_i) * a.tiles_j * a.outs;
  const int64_t units = static_cast<int64_t>(tiles) * a.k_tiles;
  uint32_t t = blockIdx.x / kGroups;
  int32_t w0, w1; // the first and last workgroup with a part of it
  if (tiles <= static_cast<uint32_t>(a.parts)) {
    w0 = wave_uniform(gemm_part(units, a.parts, static_cast<int64_t>(t) * a.k_tiles));
    w1 = wave_uniform(gemm_part(units, a.parts, static_cast<int64_t>(t + 1) * a.k_tiles - 1));
  } else { // the tile that workgroup t and its neighbour share
    w0 = t, w1 = w0 + 1;
    const int64_t cut = gemm_cut(units, a.parts, w1);
    t = static_cast<uint32_t>(cut / a.k_tiles);
    if (cut == static_cast<int64_t>(t) * a.k_tiles)
      return;
  }
  if (w0 == w1)
    return; // one workgroup had it whole
  const int64_t u0 = static_cast<int64_t>(t) * a.k_tiles;
  int32_t ti, tj, which;
  gemm_tile(a.tiles_i, a.tiles_j, t, ti, tj, which);
  const int own = threadIdx.x % kOwn, part = threadIdx.x / kOwn;
  const int q = static_cast<int>(blockIdx.x % kGroups) * kOwn + own;
  const int r = q / kChunks, c = q % kChunks * E;
  float v[2][E];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < E; ++i)
      v[h][i] = 0.f;
  for (int32_t w = w0 + part; w <= w1; w += PARTS) {
    // a workgroup whose part begins in this tile has its sums in its first place
    const int slot = kPartTiles<T> > 1 && gemm_begins(units, a.parts, w, u0 - 1) ? 1 : 0;
    const float *at = a.part + (static_cast<int64_t>(w) * kPartTiles<T> + slot) * BI * SHAPE::BJ +
                      r * kRow + c;
#pragma unroll
    for (int h = 0; h < kHalf; ++h)
#pragma unroll
      for (int i = 0; i < E; i += 4) {
        const v4f f = *reinterpret_cast<const v4f *>(at + h * BI * kRow + i);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[h][i + e] += f[e];
      }
  }
  if constexpr (PARTS > 1) {
    __shared__ float sums[PARTS][kSums][kOwn];
#pragma unroll
    for (int i = 0; i < kSums; ++i)
      sums[part][i][own] = v[i / E][i % E];
    __syncthreads();
    if (part > 0)
      return;
#pragma unroll
    for (int i = 0; i < kSums; ++i)
#pragma unroll
      for (int p = 1; p < PARTS; ++p)
        v[i / E][i % E] += sums[p][i][own];
  }
  const int32_t row = ti * BI + r, col = tj * kRow + c, left = a.cols - col;
  if (row >= a.rows)
    return;
  if constexpr (STAGE == kPlain) {
    T *to = static_cast<T *>(a.out[which]) + row * a.out_row + col;
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < left)
        to[i] = from_f32<T>(v[0][i]);
  } else if (col < a.pitch) {
    finish_chunk<T, STAGE>(a, row * a.pitch + col, left, v);
  }
}

// Matrices laid out anew, all of a pass in one launch: rows of `cols` elements at
// p, row stride `row`, as rows of `chunks` whole 16-byte chunks, zeros behind
// `cols`. first: the matrix' first chunk in the launch.
constexpr int kPackMost = 5;
struct PackJobs {
  struct Job {
    const void *p;
    void *out;
    int64_t row, first;
    int32_t cols, chunks;
  } job[kPackMost];
  int32_t n;
  int64_t total;
};
template <typename T>
__global__ __launch_bounds__(kGatedThreads) void gated_pack_kernel(PackJobs jobs) {
  using K = RowChunk<T>;
  for (int64_t q = static_cast<int64_t>(blockIdx.x) * kGatedThreads + threadIdx.x; q < jobs.total;
       q += static_cast<int64_t>(gridDim.x) * kGatedThreads) {
    int k = 0;
    while (k + 1 < jobs.n && q >= jobs.job[k + 1].first)
      ++k;
    const PackJobs::Job &job = jobs.job[k];
    const int64_t at = q - job.first;
    const int64_t r = at >> 32 ? at / job.chunks
                               : static_cast<uint32_t>(at) / static_cast<uint32_t>(job.chunks);
    const int32_t c = static_cast<int32_t>(at - r * job.chunks) * K::V;
    static_cast<v4u *>(job.out)[at] =
        K::fetch(static_cast<const T *>(job.p) + r * job.row + c, job.cols - c, false);
  }
}

// ---------------------------------------------------------------- few rows

// 16 TB rows each: a workgroup's waves share 16 columns (of g and u, or of y) and
// part k among them; weights go from memory to registers and the matrix cores as
// they come, 64 bytes of 16 rows to a load. The waves' sums are added in LDS in
// order.
//
// Bound by memory: 32 rows, 4096 channels, 11008 hidden, bf16: g and u 40 us (4.5
// TB/s), y 27. (In the operands' own order of lanes the loads alone took 55 and
// 37; with each wave's k in one piece 44 and 29; without a turn ahead 52.)
struct FewArgs {
  const void *y, *x[2]; // rows [n, k] and weights [cols, k]
  int64_t y_row, x_row[2];
  int32_t n, k, cols;
  void *out; // kPlain: [n, cols]
  int64_t out_row;
  GatedSaved saved;
  int64_t pitch;
  int32_t keep, kind;
};

template <typename T, int TB, bool GATE, int WAVES>
__global__ __launch_bounds__(WAVES *kWave) void gated_few_kernel(FewArgs a) {
  using M = Mfma<T>;
  using K = RowChunk<T>;
  constexpr int N = GATE ? 2 : 1, E = K::V;
  constexpr int kOuts = 256 * TB * N; // results of a workgroup
  __shared__ float sums[WAVES][kOuts];
  const int lane = lane_id(), w = wave_uniform(threadIdx.x / kWave);
  const int32_t col0 = blockIdx.x * 16, row0 = blockIdx.y * 16 * TB;
  const int32_t steps = (a.k + M::kCh - 1) / M::kCh;
  // a quad of lanes loads 64 bytes of one row, which then go to the lanes that
  // hold them as operands: in those lanes' own order each would cost an access
  const int r = lane & 15, lr = lane >> 2, at = (lane & 3) * E, src = quad_src(lane);
  const T *xp[N], *yp[TB];
#pragma unroll
  for (int i = 0; i < N; ++i)
    xp[i] = static_cast<const T *>(a.x[i]) + min(col0 + lr, a.cols - 1) * a.x_row[i] + at;
#pragma unroll
  for (int b = 0; b < TB; ++b)
    yp[b] = static_cast<const T *>(a.y) + min(row0 + 16 * b + lr, a.n - 1) * a.y_row + at;
  v4f acc[N][TB];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int b = 0; b < TB; ++b)
      acc[i][b] = v4f{0.f, 0.f, 0.f, 0.f};
  // the waves take turns of two steps, so that the workgroup reads a row's bytes in
  // order, and hold the next turn's while they multiply one's
  constexpr int kTurn = 2;
  struct Turn {
    v4u x[kTurn][N], y[kTurn][TB];
  };
  const int32_t full = a.k / M::kCh, whole = full / kTurn * kTurn; // steps of whole chunks
  auto load = [&](Turn &c, int32_t s) {
    if (s >= whole)
      return;
#pragma unroll
    for (int t = 0; t < kTurn; ++t) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        c.x[t][i] = K::raw(xp[i] + (s + t) * M::kCh);
#pragma unroll
      for (int b = 0; b < TB; ++b)
        c.y[t][b] = K::raw(yp[b] + (s + t) * M::kCh);
    }
  };
  auto multiply = [&](const v4u (&x)[N], const v4u (&y)[TB]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int b = 0; b < TB; ++b)
        M::mma(__builtin_bit_cast(typename M::Frag, quad_to_mfma(x[i], src)),
               __builtin_bit_cast(typename M::Frag, quad_to_mfma(y[b], src)), acc[i][b]);
  };
  constexpr int32_t kStride = kTurn * WAVES;
  Turn turns[2];
  int32_t s = w * kTurn;
  load(turns[0], s);
  load(turns[1], s + kStride);
  for (; s < whole; s += 2 * kStride)
#pragma unroll
    for (int d = 0; d < 2; ++d)
      if (s + d * kStride < whole) {
#pragma unroll
        for (int t = 0; t < kTurn; ++t)
          multiply(turns[d].x[t], turns[d].y[t]);
        load(turns[d], s + (d + 2) * kStride);
      }
  for (s = whole + w; s < steps; s += WAVES) { // what no turn holds, and a partial chunk
    v4u x[N], y[TB];
    const int32_t k = s * M::kCh;
#pragma unroll
    for (int i = 0; i < N; ++i)
      x[i] = K::fetch(xp[i] + k, a.k - k - at, false);
#pragma unroll
    for (int b = 0; b < TB; ++b)
      y[b] = K::fetch(yp[b] + k, a.k - k - at, false);
    multiply(x, y);
  }
  // entry e: column 4 (lane / 16) + e, row lane % 16 of block b
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sums[w][((b * 16 + r) * N + i) * 16 + 4 * (lane >> 4) + e] = acc[i][b][e];
  __syncthreads();
  for (int o = threadIdx.x; o < 256 * TB; o += WAVES * kWave) {
    const int32_t r = o / 16, c = o % 16, row = row0 + r, col = col0 + c;
    if (row >= a.n)
      break;
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int p = 0; p < WAVES; ++p)
        v[i] += sums[p][(r * N + i) * 16 + c];
    }
    if constexpr (GATE) {
      if (col >= a.pitch)
        continue;
      if (col >= a.cols) // the columns behind the last are zeros
        v[0] = v[N - 1] = 0.f;
      const int64_t to = row * a.pitch + col;
      float d;
      static_cast<T *>(a.saved.h)[to] = from_f32<T>(activation<T>(a.kind, v[0], d) * v[N - 1]);
      if (a.keep) {
        if constexpr (sizeof(T) == 4) {
          static_cast<float *>(a.saved.g)[to] = v[0];
          static_cast<float *>(a.saved.u)[to] = v[N - 1];
        } else {
          const uint32_t g = upper24(v[0]), u = upper24(v[N - 1]);
          static_cast<uint16_t *>(a.saved.g)[to] = g >> 8;
          static_cast<uint16_t *>(a.saved.u)[to] = u >> 8;
          a.saved.low[to] = (g & 0xff) | (u & 0xff) << 8;
        }
      }
    } else if (col < a.cols) {
      static_cast<T *>(a.out)[row * a.out_row + col] = from_f32<T>(v[0]);
    }
  }
}

// ------------------------------------------------------------------ host

void check_gated_sizes(const rhip_gated *d) {
  RHIP_CHECK_ARG(d != nullptr, "descriptor is null");
  if (d->dtype != RHIP_F32 && d->dtype != RHIP_BF16)
    throw Error(RHIP_ERR_UNSUPPORTED, "dtype must be RHIP_F32 or RHIP_BF16");
  RHIP_CHECK_ARG(d->n >= 0 && d->channels >= 1 && d->hidden >= 1 && d->outputs >= 1, "bad sizes");
  if (d->n > INT32_MAX - 256 || d->channels > kGemmMaxRow || d->hidden > kGemmMaxRow ||
      d->outputs > kGemmMaxRow)
    throw Error(RHIP_ERR_UNSUPPORTED,
                "at most 2^31 - 257 rows and 2^20 channels, hidden channels and outputs");
  RHIP_CHECK_ARG(d->activation == RHIP_ACT_SILU || d->activation == RHIP_ACT_GELU,
                 "activation must be one of RHIP_ACT_");
}
void check_gated(const rhip_gated *d) {
  check_gated_sizes(d);
  RHIP_CHECK_ARG((d->n == 0 || d->x) && d->gate && d->up && d->down,
                 "x, gate, up and down are required");
}

int64_t chunk_elements(int32_t dtype) { return dtype == RHIP_F32 ? 4 : 8; }
int64_t whole_chunks(int64_t n, int32_t dtype) {
  return static_cast<int64_t>(align_up(static_cast<size_t>(n), chunk_elements(dtype)));
}
size_t element_bytes(int32_t dtype) { return dtype == RHIP_F32 ? 4 : 2; }

// A matrix as the products take it: itself, or a copy in the workspace.
struct Packed {
  const void *src;
  int64_t src_row;
  int32_t rows, cols;
  bool copied;
  void *copy;
  const void *p;
  int64_t row; // of p
};
Packed plan_pack(Carve &cv, const void *p, int64_t row, int64_t rows, int64_t cols,
                 int32_t dtype) {
  const int64_t e = chunk_elements(dtype);
  Packed m{p, row, static_cast<int32_t>(rows), static_cast<int32_t>(cols), false, nullptr, p, row};
  // (a single row's stride does not matter, and may be anything)
  if (!aligned16(p) || cols % e != 0 || (rows > 1 && (row % e != 0 || row < cols || row > kGemmMaxRow))) {
    m.copied = true;
    m.row = whole_chunks(cols, dtype);
    m.copy = cv.take<char>(static_cast<size_t>(std::max<int64_t>(rows, 1)) * m.row *
                           element_bytes(dtype));
    m.p = m.copy;
  } else if (rows <= 1) {
    m.row = cols;
  }
  return m;
}
template <typename T>
void run_packs(std::initializer_list<const Packed *> matrices, hipStream_t stream) {
  PackJobs jobs{};
  for (const Packed *m : matrices) {
    if (!m->copied || m->rows == 0)
      continue;
    const int32_t chunks = static_cast<int32_t>(m->row / RowChunk<T>::V);
    jobs.job[jobs.n++] = {m->src, m->copy, m->src_row, jobs.total, m->cols, chunks};
    jobs.total += static_cast<int64_t>(m->rows) * chunks;
  }
  if (jobs.n == 0)
    return;
  hipLaunchKernelGGL((gated_pack_kernel<T>),
                     dim3(static_cast<unsigned>(
                         std::min<int64_t>(ceil_div(jobs.total, kGatedThreads), 1 << 20))),
                     dim3(kGatedThreads), 0, stream, jobs);
  RHIP_LAUNCH_CHECK();
}

enum ProductTiles : int32_t { kLargeTiles, kSmallTiles, kTinyTiles };
struct ProductPlan {
  ProductTiles tiles;
  int32_t parts; // workgroups that share the tiles; 0: one has each
  size_t part;   // fp32 values of the parts' sums
};

// A product's results, their tiles of k, and whether a tile holds both projections.
struct ProductSize {
  int64_t rows, cols, k_tiles, outs;
  bool halves;
};
ProductSize product_size(const rhip_gated &d, int32_t product) {
  const int64_t bk = kGemmTileBytes / static_cast<int64_t>(element_bytes(d.dtype));
  const int64_t pitch = whole_chunks(d.hidden, d.dtype), kn = ceil_div(d.n, bk);
  switch (product) {
  case RHIP_GATED_HIDDEN: return {d.n, pitch, ceil_div(d.channels, bk), 1, true};
  case RHIP_GATED_OUTPUT: return {d.n, d.outputs, ceil_div(pitch, bk), 1, false};
  case RHIP_GATED_GRAD_HIDDEN: return {d.n, pitch, ceil_div(d.outputs, bk), 1, false};
  case RHIP_GATED_GRAD_X: return {d.n, d.channels, 2 * ceil_div(d.hidden, bk), 1, false};
  case RHIP_GATED_GRAD_GATES: return {d.hidden, d.channels, kn, 2, false};
  default: return {d.outputs, d.hidden, kn, 1, false};
  }
}

// How a product's work is shared, by estimated time in microseconds: 256x256 tiles,
// one workgroup to a CU (bf16), 128x128 ones, two, or 64x64 ones, four; a
// workgroup to every tile, or k shared: in fp32 by as many workgroups as the chip
// holds at once, or a half or a quarter of them, an equal part of all tiles of k
// each; in bf16 every tile by 2, 4 .. of them (parts that begin inside a tile
// load other slices of k than their neighbours, which share what an XCD's L2
// holds: 12000 rows, 300 channels, 700 hidden 206 us, 166 even; 16000, 512, 1024
// 298 and 255). A tile of k takes `alone` however few workgroups there are; more
// of them on a CU share its matrix cores (fp32) or its way to memory (bf16, up to
// `full`). (bf16, 4000 rows, 1024 channels, 4096 hidden: the weights' gradients 97
// us in 256x256 tiles, which fill half the chip, 71 in 128x128. fp32, 2000 rows,
// 300 channels, 4000 hidden, a pass: 565 us with tiles cut evenly, 488.)
ProductPlan plan_product(const ProductSize &size, int32_t dtype) {
  const int64_t rows = size.rows, cols = size.cols, k_tiles = size.k_tiles, outs = size.outs;
  const bool halves = size.halves;
  struct Cost {
    int64_t side;
    double slots, start, alone, full;
  };
  static constexpr Cost kCosts[2][3] = {
      {{256, 256, 6.0, 9.0, 9.0}, {128, 512, 4.0, 2.2, 2.2}, {64, 1024, 3.0, 0.82, 0.64}},
      {{256, 256, 12.0, 1.65, 1.9}, {128, 512, 6.0, 0.9, 1.15}, {64, 1024, 3.0, 0.5, 0.9}}};
  const bool f32 = dtype == RHIP_F32;
  ProductPlan best{};
  double least = 0.0;
  for (int shape = f32 ? kSmallTiles : kLargeTiles; shape <= kTinyTiles; ++shape) {
    const Cost &c = kCosts[f32 ? 0 : 1][shape];
    // the pair of a 64x64 tile is twice a tile's work
    const bool pair = halves && shape == kTinyTiles;
    const double twice = pair ? 2.0 : 1.0;
    const int64_t wide = c.side / (halves && !pair ? 2 : 1);
    const int64_t tiles = ceil_div(rows, c.side) * ceil_div(cols, wide) * outs;
    const double n = static_cast<double>(tiles), k = static_cast<double>(k_tiles);
    // a tile of k, with so many workgroups there: in bf16 the loads are waited
    // for, in fp32 the fullest CU's matrix cores
    auto turn = [&](double groups) {
      return twice * std::max(c.alone, f32 ? c.full * std::ceil(groups / 256.0)
                                           : c.full * std::sqrt(std::min(1.0, groups / c.slots)));
    };
    auto consider = [&](double t, int64_t parts) {
      if (least != 0.0 && t >= least)
        return;
      least = t;
      best = {static_cast<ProductTiles>(shape), static_cast<int32_t>(parts),
              static_cast<size_t>(parts * part_tiles(f32) * c.side * c.side) * (pair ? 2 : 1)};
    };
    // `each` of a tile's turns for a workgroup, `starts` of tiles
    auto shared = [&](int64_t parts, double starts, double each) {
      const double p = static_cast<double>(parts);
      const double sums = (p + std::min(p, n)) * c.side * c.side * 4.0 * twice;
      consider(starts * c.start + each * turn(p) + 5.0 + sums / 4.0e6, parts);
    };
    if (f32) {
      consider((std::floor(n / c.slots) + 1.0) * c.start + k * turn(n), 0);
      for (const double share : {1.0, 0.5, 0.25}) {
        const int64_t parts =
            std::min<int64_t>(static_cast<int64_t>(c.slots * share), tiles * k_tiles / 4);
        if (parts >= 2 && parts != tiles)
          shared(parts, std::ceil(n / parts) + 1.0, n * k / parts);
      }
      continue;
    }
    for (int64_t s = 1; s == 1 || (s <= 64 && 4 * s <= k_tiles && tiles * s <= 2 * c.slots);
         s *= 2) {
      const double rounds = std::ceil(n * s / c.slots);
      if (s == 1)
        consider(rounds * (c.start + k * turn(n)), 0);
      else
        shared(tiles * s, rounds, rounds * std::ceil(k / s));
    }
  }
  return best;
}

// Threads of the join for each of a product's chunks: few chunks leave most of the
// chip idle unless several threads share one.
int32_t join_threads(int64_t parts, int64_t tiles, int64_t tile_chunks) {
  return parts >= 8 * tiles && tiles * tile_chunks < 256 * 1024 ? 8 : 1;
}

// Launches a product of the given stage, and what joins its shared tiles.
template <typename T, bool YACROSS, bool XACROSS, GemmPair PAIR, GatedStage STAGE>
void run_product(GatedArgs a, const ProductPlan &plan, float *part, hipStream_t stream) {
  if (a.rows == 0)
    return;
  constexpr int kHalf = PAIR == kGemmHalves ? 2 : 1;
  a.part = part;
  auto launch = [&](auto shape) {
    using SHAPE = decltype(shape);
    a.tiles_i = static_cast<int32_t>(ceil_div(a.rows, SHAPE::BI));
    a.tiles_j = static_cast<int32_t>(ceil_div(a.cols, SHAPE::BJ / kHalf));
    const int64_t tiles = static_cast<int64_t>(a.tiles_i) * a.tiles_j * a.outs;
    if (gemm_grid(tiles) > max_groups(SHAPE::kThreads))
      throw Error(RHIP_ERR_UNSUPPORTED, "too many tiles");
    const dim3 threads(SHAPE::kThreads);
    if (plan.parts == 0) {
      a.parts = static_cast<int32_t>(tiles);
      hipLaunchKernelGGL((gated_product_kernel<T, SHAPE, YACROSS, XACROSS, PAIR, STAGE, false>),
                         dim3(static_cast<unsigned>(gemm_grid(tiles))), threads, 0, stream, a);
      RHIP_LAUNCH_CHECK();
      return;
    }
    a.parts = plan.parts;
    hipLaunchKernelGGL((gated_product_kernel<T, SHAPE, YACROSS, XACROSS, PAIR, STAGE, true>),
                       dim3(static_cast<unsigned>(gemm_grid(a.parts))), threads, 0, stream, a);
    RHIP_LAUNCH_CHECK();
    constexpr int E = STAGE == kPlain ? 4 : 16 / static_cast<int>(sizeof(T));
    auto join = [&](auto n) {
      constexpr int PARTS = decltype(n)::value;
      constexpr int64_t kGroups = int64_t(SHAPE::BI) * (SHAPE::BJ / kHalf) / E /
                                  (kGatedThreads / PARTS);
      const int64_t shared = tiles <= a.parts ? tiles : a.parts - 1; // at most
      hipLaunchKernelGGL((gated_join_kernel<T, SHAPE, PAIR, STAGE, PARTS>),
                         dim3(static_cast<unsigned>(shared * kGroups)), dim3(kGatedThreads), 0,
                         stream, a);
      RHIP_LAUNCH_CHECK();
    };
    if (join_threads(a.parts, tiles, SHAPE::BI * (SHAPE::BJ / kHalf) / E) > 1)
      join(std::integral_constant<int, 8>{});
    else
      join(std::integral_constant<int, 1>{});
  };
  if constexpr (sizeof(T) == 2) // in fp32 no faster than 128x128 tiles
    if (plan.tiles == kLargeTiles)
      return launch(LargeTiles{});
  if (plan.tiles == kSmallTiles)
    return launch(SmallTiles{});
  launch(std::conditional_t<PAIR == kGemmHalves, TinyPairs, TinyTiles>{});
}

GemmSide side(const Packed &m, bool across, const Packed *second = nullptr) {
  GemmSide s{};
  s.p[0] = m.p, s.p[1] = second ? second->p : m.p;
  s.row = m.row;
  // along its rows a matrix is whole chunks
  const int32_t wide = m.copied ? static_cast<int32_t>(m.row) : m.cols;
  s.idx = across ? wide : m.rows;
  s.k = across ? m.rows : wide;
  return s;
}
GemmSide side(const void *p, const void *second, int32_t rows, int64_t pitch, bool across) {
  GemmSide s{};
  s.p[0] = p, s.p[1] = second;
  s.row = pitch;
  s.idx = across ? static_cast<int32_t>(pitch) : rows;
  s.k = across ? rows : static_cast<int32_t>(pitch);
  return s;
}

// gate and up as one pair of matrices with one row stride
void pack_pair(Carve &cv, const rhip_gated *d, Packed &gate, Packed &up) {
  Carve dry(nullptr, 0);
  gate = plan_pack(dry, d->gate, d->gate_row, d->hidden, d->channels, d->dtype);
  up = plan_pack(dry, d->up, d->up_row, d->hidden, d->channels, d->dtype);
  const bool copy = gate.copied || up.copied || gate.row != up.row;
  for (auto *m : {&gate, &up}) {
    if (copy) {
      m->copied = true;
      m->row = whole_chunks(d->channels, d->dtype);
      m->copy = cv.take<char>(static_cast<size_t>(d->hidden) * m->row * element_bytes(d->dtype));
      m->p = m->copy;
    }
  }
}

GatedSaved carve_saved(Carve &cv, const rhip_gated *d, int64_t pitch, bool keep) {
  GatedSaved s{};
  const size_t n = static_cast<size_t>(std::max<int64_t>(d->n, 1)) * pitch;
  s.h = cv.take<char>(n * element_bytes(d->dtype));
  if (keep) {
    s.g = cv.take<char>(n * element_bytes(d->dtype));
    s.u = cv.take<char>(n * element_bytes(d->dtype));
    if (d->dtype == RHIP_BF16)
      s.low = cv.take<uint16_t>(n);
  }
  return s;
}

struct GatedForward {
  Packed x, gate, up, down;
  GatedSaved saved; // without a saved buffer: h alone
  ProductPlan project, out;
  float *part;
};
// Whether the kernel for few rows takes the forward: up to 64 rows, which it takes
// at once (4096 channels, 11008 hidden, bf16, 64 rows: 89 us, in tiles 91 at 65),
// and up to 256 where reading the weights again for every 64 rows, mostly from the
// caches, costs less than the tiles' few workgroups and further launches. 65, 128
// and 256 rows of so many channels and hidden ones, few rows / tiles, us:
//   bf16  512, 1376   12/18  13/18  18/18    fp32  20/28  20/28  28/34
//         1024, 2816  21/27  22/27  29/27          42/42  43/43  56/63
//         1536, 4096  28/30  29/30  51/35          62/62  64/62  114/103
//         2048, 5504  47/42  50/43  86/59          99/95  102/96  186/163
// Between 200 and 400 million products of fp32 the tiles, which then run, are up to
// a quarter behind (768, 2048, 128 rows: 26/32) or level.
bool few_rows(const rhip_gated *d) {
  if (d->n <= 64)
    return true;
  const int64_t products =
      d->n * (2 * static_cast<int64_t>(d->channels) + d->outputs) / 3 * d->hidden;
  return d->n <= 256 && products <= (d->dtype == RHIP_F32 ? 200'000'000 : 600'000'000);
}
GatedForward plan_forward(Carve &cv, const rhip_gated *d, bool keep) {
  GatedForward f{};
  const int64_t pitch = whole_chunks(d->hidden, d->dtype);
  if (!keep)
    f.saved = carve_saved(cv, d, pitch, false);
  if (few_rows(d))
    return f;
  f.x = plan_pack(cv, d->x, d->x_row, d->n, d->channels, d->dtype);
  pack_pair(cv, d, f.gate, f.up);
  f.down = plan_pack(cv, d->down, d->down_row, d->outputs, d->hidden, d->dtype);
  f.project = plan_product(product_size(*d, RHIP_GATED_HIDDEN), d->dtype);
  f.out = plan_product(product_size(*d, RHIP_GATED_OUTPUT), d->dtype);
  f.part = cv.take<float>(std::max(f.project.part, f.out.part));
  return f;
}

struct GatedBackward {
  Packed x, gate, up, down, gy;
  void *dg, *du;
  ProductPlan hidden, gx, gw, gd;
  float *part;
};
GatedBackward plan_backward(Carve &cv, const rhip_gated *d) {
  GatedBackward b{};
  const int64_t pitch = whole_chunks(d->hidden, d->dtype);
  b.x = plan_pack(cv, d->x, d->x_row, d->n, d->channels, d->dtype);
  pack_pair(cv, d, b.gate, b.up);
  b.down = plan_pack(cv, d->down, d->down_row, d->outputs, d->hidden, d->dtype);
  b.gy = plan_pack(cv, d->grad_y, d->grad_y_row, d->n, d->outputs, d->dtype);
  const size_t n = static_cast<size_t>(std::max<int64_t>(d->n, 1)) * pitch;
  b.dg = cv.take<char>(n * element_bytes(d->dtype));
  b.du = cv.take<char>(n * element_bytes(d->dtype));
  b.hidden = plan_product(product_size(*d, RHIP_GATED_GRAD_HIDDEN), d->dtype);
  b.gx = plan_product(product_size(*d, RHIP_GATED_GRAD_X), d->dtype);
  b.gw = plan_product(product_size(*d, RHIP_GATED_GRAD_GATES), d->dtype);
  b.gd = plan_product(product_size(*d, RHIP_GATED_GRAD_DOWN), d->dtype);
  b.part = cv.take<float>(std::max({b.hidden.part, b.gx.part, b.gw.part, b.gd.part}));
  return b;
}

template <typename F> void with_type(int32_t dtype, F &&f) {
  if (dtype == RHIP_F32)
    f(float{});
  else
    f(__bf16{});
}

GatedArgs gated_args(const rhip_gated *d, const GatedSaved &saved) {
  GatedArgs a{};
  a.outs = 1;
  a.saved = saved;
  a.pitch = whole_chunks(d->hidden, d->dtype);
  a.kind = d->activation;
  return a;
}

template <typename T, bool GATE> void run_few(const FewArgs &f, hipStream_t stream) {
  const int64_t cols = GATE ? f.pitch : f.cols;
  auto launch = [&](auto tb) {
    const int64_t groups = ceil_div(cols, 16);
    auto waves = [&](auto n) {
      constexpr int kWaves = decltype(n)::value;
      hipLaunchKernelGGL((gated_few_kernel<T, decltype(tb)::value, GATE, kWaves>),
                         dim3(static_cast<unsigned>(groups),
                              static_cast<unsigned>(ceil_div(f.n, 16 * decltype(tb)::value))),
                         dim3(kWaves * kWave), 0, stream, f);
    };
    // two workgroups for each CU: four waves are enough (11008 hidden: 40 us, with
    // eight 42), else eight (4096 columns: 27 and 28)
    if (groups >= 512)
      waves(std::integral_constant<int, 4>{});
    else
      waves(std::integral_constant<int, 8>{});
    RHIP_LAUNCH_CHECK();
  };
  if (f.n <= 16)
    launch(std::integral_constant<int, 1>{});
  else if (f.n <= 32)
    launch(std::integral_constant<int, 2>{});
  else
    launch(std::integral_constant<int, 4>{});
}

} // namespace
} // namespace rhip

using namespace rhip;

extern "C" int rhip_gated_saved_bytes(const rhip_gated *gated, size_t *bytes) {
  return guarded([&] {
    check_gated(gated);
    RHIP_CHECK_ARG(bytes != nullptr, "bytes is null");
    Carve cv(nullptr, 0);
    carve_saved(cv, gated, whole_chunks(gated->hidden, gated->dtype), true);
    *bytes = cv.used + 256;
  });
}

extern "C" int rhip_gated_workspace_bytes(const rhip_gated *gated, int32_t pass, size_t *bytes) {
  return guarded([&] {
    check_gated(gated);
    RHIP_CHECK_ARG(bytes != nullptr, "bytes is null");
    RHIP_CHECK_ARG(pass >= RHIP_GATED_INFERENCE && pass <= RHIP_GATED_BACKWARD,
                   "pass must be one of RHIP_GATED_");
    Carve cv(nullptr, 0);
    if (pass == RHIP_GATED_BACKWARD)
      plan_backward(cv, gated);
    else
      plan_forward(cv, gated, pass == RHIP_GATED_FORWARD);
    *bytes = cv.used + 256;
  });
}

extern "C" int rhip_gated_plan(const rhip_gated *gated, int32_t product, rhip_gated_launch *launch) {
  return guarded([&] {
    check_gated_sizes(gated);
    RHIP_CHECK_ARG(launch != nullptr, "launch is null");
    RHIP_CHECK_ARG(product >= RHIP_GATED_HIDDEN && product <= RHIP_GATED_GRAD_DOWN,
                   "product must be one of RHIP_GATED_");
    *launch = rhip_gated_launch{};
    const rhip_gated &d = *gated;
    const bool forward = product <= RHIP_GATED_OUTPUT;
    if (d.n == 0 && product <= RHIP_GATED_GRAD_X)
      return;
    if (forward && few_rows(gated))
      return;
    const ProductSize s = product_size(d, product);
    const ProductPlan p = plan_product(s, d.dtype);
    const bool halves = s.halves, tiny = p.tiles == kTinyTiles;
    launch->side = p.tiles == kLargeTiles ? 256 : p.tiles == kSmallTiles ? 128 : 64;
    const int64_t wide = launch->side / (halves && !tiny ? 2 : 1);
    launch->tiles = ceil_div(s.rows, launch->side) * ceil_div(s.cols, wide) * s.outs;
    launch->k_tiles = static_cast<int32_t>(s.k_tiles);
    launch->parts = p.parts;
    const bool chunks = product == RHIP_GATED_HIDDEN || product == RHIP_GATED_GRAD_HIDDEN;
    if (p.parts > 0)
      launch->join = join_threads(p.parts, launch->tiles,
                                  launch->side * wide / (chunks ? chunk_elements(d.dtype) : 4));
  });
}

extern "C" int rhip_gated_forward(const rhip_gated *gated, void *y, void *saved,
                                  size_t saved_bytes, void *workspace, size_t ws_bytes,
                                  hipStream_t stream) {
  return guarded([&] {
    const rhip_gated *d = gated;
    check_gated(d);
    if (d->n == 0)
      return;
    RHIP_CHECK_ARG(y != nullptr, "y is required");
    RHIP_CHECK_ARG(workspace != nullptr, "workspace is required");
    RHIP_CHECK_ARG(aligned16(saved) && aligned16(workspace),
                   "saved and workspace must be aligned to 16 bytes");
    Carve cv(workspace, ws_bytes);
    GatedForward f = plan_forward(cv, d, saved != nullptr);
    if (saved) {
      Carve keep(saved, saved_bytes);
      f.saved = carve_saved(keep, d, whole_chunks(d->hidden, d->dtype), true);
    }
    with_type(d->dtype, [&](auto t) {
      using T = decltype(t);
      GatedArgs a = gated_args(d, f.saved);
      if (few_rows(d)) {
        FewArgs w{};
        w.y = d->x, w.y_row = d->x_row;
        w.x[0] = d->gate, w.x[1] = d->up;
        w.x_row[0] = d->gate_row, w.x_row[1] = d->up_row;
        w.n = static_cast<int32_t>(d->n), w.k = d->channels, w.cols = d->hidden;
        w.saved = f.saved, w.pitch = a.pitch, w.keep = saved != nullptr, w.kind = d->activation;
        run_few<T, true>(w, stream);
        w.y = f.saved.h, w.y_row = a.pitch;
        w.x[0] = d->down, w.x_row[0] = d->down_row;
        w.k = d->hidden, w.cols = d->outputs;
        w.out = y, w.out_row = d->outputs;
        run_few<T, false>(w, stream);
        return;
      }
      run_packs<T>({&f.x, &f.gate, &f.up, &f.down}, stream);
      a.y = side(f.x, false);
      a.x = side(f.gate, false, &f.up);
      a.k_tiles = static_cast<int32_t>(ceil_div(a.x.k, gemm_bk<T>()));
      a.rows = static_cast<int32_t>(d->n), a.cols = d->hidden;
      a.keep = saved != nullptr;
      run_product<T, false, false, kGemmHalves, kProject>(a, f.project, f.part, stream);
      a.y = side(f.saved.h, f.saved.h, a.rows, a.pitch, false);
      a.x = side(f.down, false);
      a.k_tiles = static_cast<int32_t>(ceil_div(a.x.k, gemm_bk<T>()));
      a.cols = d->outputs;
      a.out[0] = y, a.out_row = d->outputs;
      run_product<T, false, false, kGemmOne, kPlain>(a, f.out, f.part, stream);
    });
  });
}

extern "C" int rhip_gated_backward(const rhip_gated *gated, const void *saved,
                                   size_t saved_bytes, void *grad_x, void *grad_gate,
                                   void *grad_up, void *grad_down, void *workspace,
                                   size_t ws_bytes, hipStream_t stream) {
  return guarded([&] {
    const rhip_gated *d = gated;
    check_gated(d);
    RHIP_CHECK_ARG((grad_gate == nullptr) == (grad_up == nullptr),
                   "grad_gate and grad_up go together");
    if (!(grad_x && d->n > 0) && !grad_gate && !grad_down)
      return;
    RHIP_CHECK_ARG(d->n == 0 || (d->grad_y && saved), "grad_y and saved are required");
    RHIP_CHECK_ARG(workspace != nullptr, "workspace is required");
    RHIP_CHECK_ARG(aligned16(saved) && aligned16(workspace),
                   "saved and workspace must be aligned to 16 bytes");
    Carve cv(workspace, ws_bytes);
    const GatedBackward b = plan_backward(cv, d);
    GatedSaved s{};
    if (saved) {
      Carve keep(const_cast<void *>(saved), saved_bytes);
      s = carve_saved(keep, d, whole_chunks(d->hidden, d->dtype), true);
    }
    with_type(d->dtype, [&](auto t) {
      using T = decltype(t);
      const GatedArgs base = gated_args(d, s);
      const int32_t n = static_cast<int32_t>(d->n);
      const Packed none{};
      run_packs<T>({&b.gy, grad_x || grad_gate ? &b.down : &none, grad_x ? &b.gate : &none,
                    grad_x ? &b.up : &none, grad_gate ? &b.x : &none},
                   stream);
      if (grad_x || grad_gate) {
        GatedArgs a = base;
        a.y = side(b.gy, false);
        a.x = side(b.down, true);
        a.k_tiles = static_cast<int32_t>(ceil_div(a.x.k, gemm_bk<T>()));
        a.rows = n, a.cols = d->hidden;
        a.dg = b.dg, a.du = b.du;
        run_product<T, false, true, kGemmOne, kHidden>(a, b.hidden, b.part, stream);
      }
      if (grad_x) {
        GatedArgs a = base;
        a.y = side(b.dg, b.du, n, a.pitch, false);
        a.x = side(b.gate, true, &b.up);
        a.k_tiles = 2 * static_cast<int32_t>(ceil_div(a.x.k, gemm_bk<T>()));
        a.rows = n, a.cols = d->channels;
        a.out[0] = grad_x, a.out_row = d->channels;
        run_product<T, false, true, kGemmBehind, kPlain>(a, b.gx, b.part, stream);
      }
      if (grad_gate) {
        GatedArgs a = base;
        a.y = side(b.dg, b.du, n, a.pitch, true);
        a.x = side(b.x, true);
        a.outs = 2;
        a.k_tiles = static_cast<int32_t>(ceil_div(n, gemm_bk<T>()));
        a.rows = d->hidden, a.cols = d->channels;
        a.out[0] = grad_gate, a.out[1] = grad_up, a.out_row = d->channels;
        run_product<T, true, true, kGemmOne, kPlain>(a, b.gw, b.part, stream);
      }
      if (grad_down) {
        GatedArgs a = base;
        a.y = side(b.gy, true);
        a.x = side(s.h, s.h, n, a.pitch, true);
        a.k_tiles = static_cast<int32_t>(ceil_div(n, gemm_bk<T>()));
        a.rows = d->outputs, a.cols = d->hidden;
        a.out[0] = grad_down, a.out_row = d->hidden;
        run_product<T, true, true, kGemmOne, kPlain>(a, b.gd, b.part, stream);
      }
    });
  });
}
