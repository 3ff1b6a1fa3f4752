// Matrix products out[i, j] = sum over k of Y(i, k) X(j, k) of rows in device
// memory on gfx950: LDS tiles streamed by direct loads, their operands for the
// 32x32 matrix instructions, and the loop over k with one barrier a tile.
//
// Either operand lies with k along its rows (a row holds one index's values) or
// across them (a row holds all indices' values of one k). A tile is B indices
// by 128 bytes of k (64 bf16, 32 fp32):
//   k along:  row r at 128 r, its 16-byte chunk c at (c ^ (r / 2 % 8)) * 16, so
//             16 consecutive rows hold one chunk column in 16 bank groups;
//   k across: row k at B * sizeof(T) * k; bf16: chunk c at c ^ (k % 4 * 4) (rows of
//             128 bytes: c ^ (k / 2 % 2 * 4)), so four rows' pieces of a transpose
//             read lie in four bank groups; fp32: c ^ (k / 4 % 2 * 8), for the
//             lanes' two halves.
// The first operand of a matrix instruction is X, the second Y: a lane then
// holds, of one i, runs of four consecutive j, which is the order of the
// results in memory.
#pragma once

#include <type_traits>

#include "attn_device.hpp"
#include "row_chunk.hpp"

namespace rhip {

constexpr int kGemmTileBytes = 128; // of k in a tile
constexpr int64_t kGemmMaxRow = int64_t(1) << 20; // row stride in elements

template <typename T> constexpr int gemm_bk() { return kGemmTileBytes / sizeof(T); }

// One side of a product in memory: up to two matrices of the same shape, `idx`
// indices by `k`, row stride `row` elements. Rows hold whole 16-byte chunks, so
// of two sides one may have its k rounded up, to values of zero.
struct GemmSide {
  const void *p[2];
  int64_t row;
  int32_t idx, k;
};

template <typename T, int B, bool ACROSS, int THREADS> struct GemmTile {
  static constexpr int E = 16 / sizeof(T);
  static constexpr int kBytes = B * kGemmTileBytes;
  static constexpr int kSteps = 4; // of two chunks of k
  static constexpr int kRowBytes = ACROSS ? B * static_cast<int>(sizeof(T)) : kGemmTileBytes;
  static constexpr int kRowChunks = kRowBytes / 16;
  static constexpr int kLoads = kBytes / 16 / THREADS;
  static constexpr int kRowsPerLoad = THREADS / kRowChunks;
  // the 64-byte piece of a row across, in units of four chunks, that row k % 4 swaps
  __device__ static __forceinline__ int turn(int k) {
    return kRowChunks >= 16 ? k & 3 : (k >> 1) & 1;
  }
  using Frag = typename Mfma<T>::Frag;

  // A lane's read addresses: k along, of the four steps; across, of up to four
  // 32-index blocks from block0 on.
  struct Lane {
    uint32_t at[4];
  };
  __device__ static __forceinline__ Lane lane(uint32_t lds, int block0) {
    const int l = lane_id(), half = l >> 5;
    Lane a;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (!ACROSS) {
        a.at[i] = lds + (block0 * 32 + (l & 31)) * kRowBytes +
                  (((2 * i + half) ^ ((l >> 1) & 7)) * 16);
      } else if constexpr (sizeof(T) == 2) {
        const int j = (l & 15) >> 2, q = 2 * ((l >> 4) & 1) + ((l & 3) >> 1);
        a.at[i] = lds + (8 * half + j) * kRowBytes + (((block0 + i) ^ turn(j)) * 4 + q) * 16 +
                  (l & 1) * 8;
      } else {
        a.at[i] = lds + 4 * half * kRowBytes + ((block0 + i) ^ half) * 128 + (l & 31) * 4;
      }
    }
    return a;
  }
  // The operand of block `block` (of the wave's), two chunks of k at `step`.
  __device__ static __forceinline__ Frag read(const Lane &a, int bytes, int block, int step) {
    if constexpr (!ACROSS) {
      return lds_read<Frag>(a.at[step] + (bytes + block * 32 * kRowBytes));
    } else if constexpr (sizeof(T) == 2) {
      const uint32_t at = a.at[block] + (bytes + 16 * step * kRowBytes);
      const v4s lo = lds_read_tr16(at), hi = lds_read_tr16(at + 4 * kRowBytes);
      return __builtin_bit_cast(v8bf, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      Frag f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        f[i] = lds_read<float>(a.at[block] + (bytes + (8 * step + i) * kRowBytes));
      return f;
    }
  }

  // A thread's loads: its byte offset in the tile's first rows (for fp32 with
  // rows of 64 chunks, of the even and the odd ones), and its chunk of k.
  static constexpr int kOffs = ACROSS && sizeof(T) == 4 && kRowsPerLoad == 4 ? 2 : 1;
  uint32_t off[kOffs];
  int32_t chunk;
  // idx_left: indices from the tile's first on
  __device__ __forceinline__ void init(int64_t row, int32_t idx_left) {
    const int t = threadIdx.x, r = t / kRowChunks, slot = t % kRowChunks;
    if constexpr (!ACROSS) {
      chunk = slot ^ ((r >> 1) & 7);
      off[0] = static_cast<uint32_t>(r * row * sizeof(T)) + chunk * 16;
    } else {
#pragma unroll
      for (int i = 0; i < kOffs; ++i) {
        const int rr = r + i * kRowsPerLoad;
        const int c = sizeof(T) == 2 ? slot ^ (turn(rr) << 2) : slot ^ (((rr >> 2) & 1) << 3);
        off[i] = c * E < idx_left ? static_cast<uint32_t>(r * row * sizeof(T)) + c * 16 : kBufOob;
      }
      chunk = 0;
    }
  }
  // The tile at p (its first index and k), idx_left and k_left from there on
  // (k_left above zero; both whole chunks along the rows), into LDS; loads
  // FIRST .. LAST - 1 of the rows, p being load FIRST's. What lies outside
  // arrives as zeros.
  template <int FIRST = 0, int LAST = kLoads>
  __device__ __forceinline__ void issue(uint32_t lds, const T *p, int64_t row, int32_t idx_left,
                                        int32_t k_left) const {
    constexpr int kRows = (LAST - FIRST) * kRowsPerLoad;
    const int32_t rows = min(ACROSS ? k_left : idx_left, kRows);
    const int32_t wide = ACROSS ? idx_left : k_left;
    const int64_t bytes =
        rows > 0 ? ((rows - 1) * row + wide) * static_cast<int64_t>(sizeof(T)) : 0;
    const __amdgpu_buffer_rsrc_t rsrc = wave_rsrc(p, bytes);
    const uint32_t to = lds + wave_uniform(static_cast<int32_t>(threadIdx.x / kWave * kWave * 16));
    const uint32_t step = static_cast<uint32_t>(kRowsPerLoad * row * sizeof(T));
    uint32_t first[kOffs];
#pragma unroll
    for (int i = 0; i < kOffs; ++i)
      first[i] = opaque(!ACROSS && chunk * E >= k_left ? kBufOob : off[i]);
#pragma unroll
    for (int i = FIRST; i < LAST; ++i)
      dma16(rsrc, to + i * THREADS * 16, first[i % kOffs] + (i - FIRST) * step);
  }
};

// Workgroup -> its place among `groups`, so that each XCD, to which they are dealt
// round-robin, gets consecutive ones; false for those that fill the grid up.
__device__ __forceinline__ bool gemm_place(uint32_t groups, uint32_t &place) {
  const uint32_t per = (groups + kXcds - 1) / kXcds, m = blockIdx.x / kXcds;
  place = blockIdx.x % kXcds * per + m;
  return m < per && place < groups;
}
inline int64_t gemm_grid(int64_t groups) { return ceil_div(groups, kXcds) * kXcds; }

// Tile t of `outs` results of tiles_i x tiles_j tiles: in bands of eight rows of
// tiles, column by column, so what runs at once on an XCD shares an L2's worth of
// both sides.
__device__ __forceinline__ void gemm_tile(uint32_t tiles_i, uint32_t tiles_j, uint32_t t,
                                          int32_t &ti, int32_t &tj, int32_t &out) {
  constexpr uint32_t kBand = 8;
  const uint32_t plane = tiles_i * tiles_j;
  out = t / plane;
  const uint32_t rem = t - out * plane, band = rem / (kBand * tiles_j);
  const uint32_t in = rem - band * kBand * tiles_j;
  const uint32_t high = min(kBand, tiles_i - band * kBand);
  ti = band * kBand + in % high;
  tj = in / high;
}

// The work of a product as one line of `units`, tiles of k tile by tile, in equal
// parts of the line: part w's first unit.
__device__ __forceinline__ int64_t gemm_cut(int64_t units, int32_t parts, int64_t w) {
  return units * w / parts;
}
// Whether part w begins at unit u or before it: gemm_cut(w) <= u, with no division.
__device__ __forceinline__ bool gemm_begins(int64_t units, int32_t parts, int64_t w, int64_t u) {
  return units * w < (u + 1) * parts;
}
// The part that holds unit u.
__device__ __forceinline__ int32_t gemm_part(int64_t units, int32_t parts, int64_t u) {
  int32_t w = static_cast<int32_t>(static_cast<double>(u) * parts / static_cast<double>(units));
  while (w + 1 < parts && gemm_begins(units, parts, w + 1, u))
    ++w;
  while (w > 0 && !gemm_begins(units, parts, w, u))
    --w;
  return w;
}

// A workgroup's waves and each wave's blocks.
template <int WI_, int WJ_, int NI_, int NJ_> struct GemmShape {
  static constexpr int WI = WI_, WJ = WJ_, NI = NI_, NJ = NJ_;
  static constexpr int BI = 32 * WI * NI, BJ = 32 * WJ * NJ;
  static constexpr int kWaves = WI * WJ, kThreads = kWaves * kWave;
};

// What the rows of X in a tile are: one matrix', the halves of two matrices'
// tiles (the same indices of both), or the second matrix behind the first along
// k (both sides).
enum GemmPair { kGemmOne, kGemmHalves, kGemmBehind };

// The sums of a workgroup's tile of results over its tiles of k: WI x WJ waves,
// each with NI x NJ blocks of 32 by 32. acc[b][a]: X block b, Y block a. With
// kGemmHalves a wave's first NJ / 2 blocks are the first matrix', the others the
// second's.
//
// Two LDS buffers and one barrier a tile: at the last of its four steps every
// wave has read the whole tile and the next one has landed; the loads of the
// one after it then go where this one lay, and the last step's products run
// while the next tile's first operands arrive.
template <typename T, typename SHAPE, bool YACROSS, bool XACROSS, GemmPair PAIR> struct Gemm {
  static constexpr int NI = SHAPE::NI, NJ = SHAPE::NJ, WI = SHAPE::WI, WJ = SHAPE::WJ;
  static constexpr int BI = SHAPE::BI, BJ = SHAPE::BJ, BK = gemm_bk<T>();
  using YTile = GemmTile<T, BI, YACROSS, SHAPE::kThreads>;
  using XTile = GemmTile<T, BJ, XACROSS, SHAPE::kThreads>;
  using Frag = typename Mfma<T>::Frag;
  static constexpr int kLds = 2 * (YTile::kBytes + XTile::kBytes);
  static constexpr int kStrip = kLds / SHAPE::kWaves; // a wave's share once the sums are done
  static constexpr int kHalves = PAIR == kGemmHalves ? 2 : 1;
  static_assert(PAIR != kGemmHalves || (!XACROSS && NJ % 2 == 0), "halves: k along the rows");
  static_assert(YTile::kRowsPerLoad % 4 == 0 && XTile::kRowsPerLoad % 4 == 0,
                "a thread's loads share their chunk's turn");

  // y, x: the sides; i0, j0: the tile's first indices; tiles [kt0, kt1) of k
  // (with kGemmBehind those of both matrices one after another)
  __device__ static __forceinline__ void run(char *lds, const GemmSide &y, const T *yp,
                                             const GemmSide &x, int32_t i0, int32_t j0,
                                             int32_t kt0, int32_t kt1, v16f (&acc)[NJ][NI]) {
    const int w = wave_uniform(threadIdx.x / kWave), wi = w / WJ, wj = w % WJ;
    const uint32_t base = lds_address(lds);
    constexpr int kXAt = 2 * YTile::kBytes;
    const typename YTile::Lane ya = YTile::lane(base, wi * NI);
    constexpr int kHalf = PAIR == kGemmHalves ? NJ / 2 : NJ; // a wave's blocks in a row
    const typename XTile::Lane xa = XTile::lane(base + kXAt, wj * kHalf);
    YTile yt;
    XTile xt;
    yt.init(y.row, y.idx - i0);
    xt.init(x.row, x.idx - j0);
    const int32_t per = (x.k + BK - 1) / BK; // tiles of one matrix
    auto issue = [&](int32_t kt, int buf) {
      const int which = PAIR == kGemmBehind && kt >= per ? 1 : 0;
      const int32_t k0 = (kt - which * per) * BK, left = x.k - k0;
      const T *yq = PAIR == kGemmBehind ? static_cast<const T *>(y.p[which]) : yp;
      const T *xq = static_cast<const T *>(x.p[which]);
      yt.issue(base + buf * YTile::kBytes,
               yq + (YACROSS ? k0 * y.row + i0 : i0 * y.row + k0), y.row, y.idx - i0, y.k - k0);
      const int64_t at = XACROSS ? k0 * x.row + j0 : j0 * x.row + k0;
      const uint32_t to = base + kXAt + buf * XTile::kBytes;
      if constexpr (PAIR == kGemmHalves) {
        constexpr int kMid = XTile::kLoads / 2;
        xt.template issue<0, kMid>(to, xq + at, x.row, x.idx - j0, left);
        xt.template issue<kMid, XTile::kLoads>(to, static_cast<const T *>(x.p[1]) + at, x.row,
                                               x.idx - j0, left);
      } else {
        xt.issue(to, xq + at, x.row, x.idx - j0, left);
      }
    };
#pragma unroll
    for (int b = 0; b < NJ; ++b)
#pragma unroll
      for (int a = 0; a < NI; ++a)
        acc[b][a] = v16f{};
    if (kt0 >= kt1)
      return;
    Frag fy[2][NI], fx[2][NJ];
    auto fetch = [&](int set, int buf, int step) {
#pragma unroll
      for (int a = 0; a < NI; ++a)
        fy[set][a] = YTile::read(ya, buf * YTile::kBytes, a, step);
#pragma unroll
      for (int b = 0; b < NJ; ++b)
        fx[set][b] = XTile::read(xa, buf * XTile::kBytes,
                                 b < kHalf ? b : b - kHalf + WJ * kHalf, step);
    };
    auto multiply = [&](int set) {
#pragma unroll
      for (int b = 0; b < NJ; ++b)
#pragma unroll
        for (int a = 0; a < NI; ++a)
          AttnTile<T, 32>::mma(fx[set][b], fy[set][a], acc[b][a]);
    };
    issue(kt0, 0);
    wait_stream();
    __syncthreads();
    if (kt0 + 1 < kt1)
      issue(kt0 + 1, 1);
    fetch(0, 0, 0);
    auto turn = [&](int32_t kt, auto buf_) {
      constexpr int buf = decltype(buf_)::value;
#pragma unroll
      for (int s = 0; s < 3; ++s) {
        fetch((s + 1) & 1, buf, s + 1);
        multiply(s & 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (kt + 1 < kt1) {
        wait_stream();
        __syncthreads();
        if (kt + 2 < kt1)
          issue(kt + 2, buf);
        fetch(0, buf ^ 1, 0);
      }
      multiply(1);
      __builtin_amdgcn_sched_barrier(0);
    };
    for (int32_t kt = kt0; kt < kt1; kt += 2) {
      turn(kt, std::integral_constant<int, 0>{});
      if (kt + 1 < kt1)
        turn(kt + 1, std::integral_constant<int, 1>{});
    }
    __syncthreads(); // the tiles' LDS is free
  }
};

// A wave's 32 rows (one a lane's two halves share) of 32 N columns from blocks as
// the products leave them, through LDS: 16 bytes a lane of the rows' values as
// O, neighbouring lanes neighbouring bytes.
template <typename O, int N> struct GemmStrip {
  static constexpr int E = 16 / sizeof(O);
  static constexpr int kPitch = 32 * N * static_cast<int>(sizeof(O)) + 16;
  static constexpr int kBytes = 32 * kPitch;
  // f(block, r): the value of entry r
  template <typename F> __device__ static __forceinline__ void put(char *lds, F &&f) {
    const int l = lane_id(), half = l >> 5;
    char *mine = lds + (l & 31) * kPitch;
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        O e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          e[i] = f(b, 4 * g + i);
        __builtin_memcpy(__builtin_assume_aligned(mine + (32 * b + 8 * g + 4 * half) * sizeof(O),
                                                  4 * sizeof(O)),
                         e, sizeof(e));
      }
  }
  // each(row, column) for the lanes' shares of LEN values of the rows at a time
  template <int LEN, typename F> __device__ static __forceinline__ void walk(F &&each) {
    constexpr int kChunks = 32 * N / LEN;
#pragma unroll 1
    for (int q = lane_id(); q < 32 * kChunks; q += kWave)
      each(q / kChunks, q % kChunks * LEN);
  }
  __device__ static __forceinline__ v4u chunk(const char *lds, int r, int c) {
    return *reinterpret_cast<const v4u *>(lds + r * kPitch + c * sizeof(O));
  }
};

// The first `left` of a 16-byte chunk's values to p, at any alignment.
template <typename O> __device__ __forceinline__ void store_chunk(O *p, const v4u &u, int left) {
  constexpr int E = 16 / sizeof(O);
  if (left >= E) {
    *reinterpret_cast<v4u_any *>(p) = u;
  } else {
    O e[E];
    __builtin_memcpy(e, &u, 16);
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < left)
        p[i] = e[i];
  }
}

} // namespace rhip
