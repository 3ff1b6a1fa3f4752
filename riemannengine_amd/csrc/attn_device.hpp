// Device helpers shared by the attention kernels: sequences and tiles of
// packed rows, 32-row LDS tiles and the two matrix products over them.
//
// Every kernel works on 32x32 score blocks with the 32x32 matrix
// instructions (bf16 32x32x16, fp32 32x32x2): lane l holds, of a block's
// column l % 32, the 16 rows 8 (r / 4) + 4 (l / 32) + r % 4, r = 0 .. 15.
// Scores are computed transposed to the product that follows, so a lane
// holds 16 entries of one softmax row (or of one key) and the block goes into
// the next product as it lies: the sum over its rows may run in any order, so
// the other operand is read in the order the lanes hold (no exchange between
// lanes, no trip through LDS).
#pragma once

#include <type_traits>

#include "conv_device.hpp"

namespace rhip {

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kAttnMaxDim = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// The kernels' arguments: rhip_attn's fields (strides in elements), scale
// times log2(e) and the buffers.
struct AttnArgs {
  const void *q, *k, *v, *go;
  const int32_t *q_off, *k_off, *k_len;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, go_row, go_head;
  int32_t n_q, n_k, n_seq, heads, kv_heads, group, dim, causal;
  int32_t tiles, splits; // of the pass
  int32_t tile0, launched; // the tiles of this launch: launched of them from tile0 on
  float scale, c;        // c = scale * log2(e)
  void *o, *rest;        // out, and bf16 out's rounding error (training)
  float *lse;            // [heads, n_q], natural logarithm
  float *part_o, *part_ml; // [splits, n_q * heads, dim], [splits, n_q * heads, 2]
  float2 *stat;          // [heads, n_q]: log2 of the denominator, -rowsum(grad_out * out)
  float *part_k, *part_v; // [splits, n_k * kv_heads, dim]
  void *gq, *gk, *gv;
};

// One sequence of the packed rows, clamped to the buffers whatever the
// offsets hold.
struct AttnSeq {
  int32_t s, tile; // sequence, tile within it
  int32_t q0, lq, k0, lk;
};

// A value that all lanes share, in a scalar register whatever the compiler can
// prove: as vector registers the loops' bounds alone would cost a dozen.
__device__ __forceinline__ int32_t wave_uniform(int32_t v) {
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ AttnSeq wave_uniform(AttnSeq q) {
  q.s = wave_uniform(q.s), q.tile = wave_uniform(q.tile);
  q.q0 = wave_uniform(q.q0), q.lq = wave_uniform(q.lq);
  q.k0 = wave_uniform(q.k0), q.lk = wave_uniform(q.lk);
  return q;
}

__device__ __forceinline__ int32_t clamp_off(int32_t v, int32_t lo, int32_t hi) {
  return v < lo ? lo : (v > hi ? hi : v);
}

// Tile t of packed rows cut into tiles of `bm` rows at every sequence.
// Sequence s starts at tile floor(off[s] * mul / bm) + s: no two sequences
// share a tile, the tiles between one's last and the next's first are empty,
// and n * mul / bm + n_seq + 1 tiles cover them all, so neither the host nor
// another kernel has to count tiles. Rows behind the last sequence count as
// one more, without keys. mul: rows of a tile per packed row (grouped heads).
__device__ __forceinline__ void find_tile(const int32_t *off, int32_t n_seq, int32_t n, int bm,
                                          int mul, int32_t t, int32_t &seq, int32_t &tile,
                                          int32_t &r0, int32_t &len) {
  int lo = 0, hi = n_seq; // largest s with base(s) <= t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    const int64_t b =
        static_cast<int64_t>(clamp_off(off[mid], 0, n)) * mul / bm + mid;
    if (b <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  seq = lo;
  r0 = lo == 0 ? 0 : clamp_off(off[lo], 0, n);
  const int32_t r1 = lo == n_seq ? n : clamp_off(off[lo + 1], r0, n);
  len = r1 - r0;
  tile = t - static_cast<int32_t>(static_cast<int64_t>(r0) * mul / bm + lo);
}

// The keys of q.s in use.
__device__ __forceinline__ void key_range(const AttnArgs &a, AttnSeq &q) {
  q.k0 = q.lk = 0;
  if (q.s < a.n_seq) {
    q.k0 = q.s == 0 ? 0 : clamp_off(a.k_off[q.s], 0, a.n_k);
    q.lk = clamp_off(a.k_off[q.s + 1], q.k0, a.n_k) - q.k0;
    if (a.k_len)
      q.lk = clamp_off(a.k_len[q.s], 0, q.lk);
  }
}

__device__ __forceinline__ AttnSeq query_tile(const AttnArgs &a, int bm, int mul, int32_t t) {
  AttnSeq q;
  find_tile(a.q_off, a.n_seq, a.n_q, bm, mul, t, q.s, q.tile, q.q0, q.lq);
  key_range(a, q);
  return wave_uniform(q);
}

// The keys in use and the query rows of q.s, whose region holds `room` keys.
__device__ __forceinline__ void query_range(const AttnArgs &a, AttnSeq &q, int32_t room) {
  q.q0 = q.lq = q.lk = 0;
  if (q.s < a.n_seq) {
    q.lk = a.k_len ? clamp_off(a.k_len[q.s], 0, room) : room;
    q.q0 = q.s == 0 ? 0 : clamp_off(a.q_off[q.s], 0, a.n_q);
    q.lq = clamp_off(a.q_off[q.s + 1], q.q0, a.n_q) - q.q0;
  }
}

// The same over the key rows (backward of k and v): lk counts the rows in
// use, `room` all rows of the region.
__device__ __forceinline__ AttnSeq key_tile(const AttnArgs &a, int bm, int32_t t, int32_t &room) {
  AttnSeq q;
  find_tile(a.k_off, a.n_seq, a.n_k, bm, 1, t, q.s, q.tile, q.k0, room);
  query_range(a, q, room);
  room = wave_uniform(room);
  return wave_uniform(q);
}

// Workgroup -> (tile, key head, split) of a launch over tiles x key heads x
// splits. Workgroups are dealt to the 8 XCDs round-robin, and what reads the
// same keys should share an L2: each XCD gets whole heads where there are
// enough, or every second (fourth, eighth) tile of one head where 8 is a
// multiple of the heads, else all of everything. Tiles come in order on every
// XCD, so with the heaviest first (under a causal mask) their work evens out.
__device__ __forceinline__ bool attn_item(const AttnArgs &a, int32_t &tile, int32_t &kv,
                                          int32_t &split) {
  const uint32_t x = blockIdx.x % kXcds, i = blockIdx.x / kXcds;
  const uint32_t heads = a.kv_heads, units = static_cast<uint32_t>(a.launched) * a.splits;
  uint32_t unit;
  if (heads % kXcds == 0) {
    const uint32_t mine = heads / kXcds;
    unit = i / mine;
    kv = x * mine + i % mine;
  } else if (kXcds % heads == 0) {
    const uint32_t share = kXcds / heads;
    unit = i * share + x % share;
    kv = x / share;
  } else {
    unit = blockIdx.x / heads;
    kv = blockIdx.x % heads;
  }
  tile = a.tile0 + unit / a.splits;
  split = unit % a.splits;
  return unit < units;
}
// Workgroups of such a launch.
inline int64_t attn_grid(int64_t tiles, int64_t heads, int64_t splits) {
  const int64_t units = tiles * splits;
  if (kXcds % heads == 0)
    return ceil_div(units, kXcds / heads) * kXcds;
  return units * heads;
}

// LDS reads by byte address (wave instructions' immediate offsets hold what is
// constant, so a kernel keeps a handful of addresses per lane).
template <typename V> __device__ __forceinline__ V lds_read(uint32_t addr) {
  return *reinterpret_cast<const __attribute__((address_space(3))) V *>(addr);
}
__device__ __forceinline__ v4s lds_read_tr16(uint32_t addr) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s *>(addr));
}

// Keeps a branch a branch: what it guards is rare, and as selects it would
// cost every pass.
__device__ __forceinline__ void rare_path() { asm volatile(""); }

// Rows of `DP` elements (the head width padded to 32, 64, 96 or 128) as 16-byte
// chunks in LDS, in groups of four rows: chunk c of row r lies at
//   (r / 4) * 64 C + (c / 4) * 256 + (r % 4) * 64 + ((c % 4) ^ (r / 4 % 4)) * 16.
// Then 16 consecutive rows hold one chunk column in 16 different bank groups
// (row reads), so do 4 consecutive chunks of 4 consecutive rows (transpose
// reads), and a quad of lanes that loads four chunks fetches 64 consecutive
// bytes. Both kinds of read step by constants but for one bit, so each needs
// two addresses per lane.
template <typename T, int DP> struct AttnTile {
  static constexpr int E = 16 / sizeof(T);  // elements per chunk
  static constexpr int C = DP / E;          // chunks per row
  static constexpr int kDBlocks = DP / 32;  // 32-wide blocks of the head width
  static constexpr int kSteps = C / 2;      // row_product steps (two chunks each)
  static constexpr int kGroup = 64 * C;     // bytes of four rows
  using Frag = typename Mfma<T>::Frag;      // one chunk

  // Row and chunk of the 16 bytes at position `pos` (in 16-byte units).
  __device__ static __forceinline__ void place(int pos, int &row, int &c) {
    const int group = pos / (4 * C), rem = pos % (4 * C);
    row = 4 * group + (rem >> 2) % 4;
    c = (rem >> 4) * 4 + ((rem & 3) ^ (group & 3));
  }

  // A lane's addresses within a tile: of its row (l % 32) for the even and odd
  // steps of row_product, and for the two reads of a col_product step.
  struct Lane {
    uint32_t row[2], col[2];
    // the same in the tile at `lds`; opaque, so that what is constant stays an
    // immediate offset of the reads instead of an addition for each
    __device__ __forceinline__ Lane in(uint32_t lds) const {
      Lane a;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        a.row[u] = opaque(row[u] + lds);
        a.col[u] = opaque(col[u] + lds);
      }
      return a;
    }
  };
  __device__ static __forceinline__ Lane lane_addresses() {
    const int lane = lane_id(), half = lane >> 5, r = lane & 31;
    Lane a;
    const uint32_t row = (r >> 2) * kGroup + (r & 3) * 64;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      a.row[u] = row + (((2 * u + half) ^ ((r >> 2) & 3)) * 16);
    if constexpr (sizeof(T) == 2) {
      const int i = lane & 15, g = (lane >> 4) & 1;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        a.col[u] = (half + 2 * u) * kGroup + (i >> 2) * 64 +
                   ((2 * g + ((i & 3) >> 1)) ^ (half + 2 * u)) * 16 + (i & 1) * 8;
    } else { // element l % 32 of a block: chunk l % 32 / 4; row parity in u
      const int q = r >> 2;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        a.col[u] = half * kGroup + (q >> 2) * 256 + ((q & 3) ^ (half + 2 * u)) * 16 + (r & 3) * 4;
    }
    return a;
  }

  // Chunk c of a global row (E elements from p + c * E), zero past dim.
  template <bool VEC>
  __device__ static __forceinline__ uint4 chunk(const T *p, int c, int dim, bool row_ok) {
    if constexpr (VEC) { // dim is a multiple of E and rows are 16-byte aligned
      if (row_ok && c * E < dim)
        return *reinterpret_cast<const uint4 *>(p + c * E);
      return uint4{0u, 0u, 0u, 0u};
    } else {
      T e[E];
#pragma unroll
      for (int i = 0; i < E; ++i)
        e[i] = row_ok && c * E + i < dim ? p[c * E + i] : static_cast<T>(0.f);
      return __builtin_bit_cast(uint4, e);
    }
  }

  // acc += A[32 rows x dim] B[dim x 32 columns], kSteps steps: A's rows row0 ..
  // row0 + 31 of the LDS tile (plus `bytes`: of one a constant further on), B
  // the chunks a lane holds of its column. A step's left operand:
  __device__ static __forceinline__ Frag row_operand(const Lane &at, int bytes, int row0,
                                                     int step) {
    return lds_read<Frag>(at.row[step & 1] + (bytes + row0 / 4 * kGroup + (step >> 1) * 256));
  }

  // The product of one chunk pair: lane half h holds elements (2 s + h) E ..
  __device__ static __forceinline__ void mma(const Frag &a, const Frag &b, v16f &acc) {
    if constexpr (sizeof(T) == 2) {
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], acc, 0, 0, 0);
    }
  }

  // A 32x32 block as the right operand of col_product: bf16 rounds here (the
  // products' operands are 16 bits wide; their sums stay fp32).
  struct Block {
    v8bf lo, hi;
    v16f f;
  };
  __device__ static __forceinline__ void pack(const v16f &p, Block &b) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        b.lo[i] = static_cast<__bf16>(p[i]);
        b.hi[i] = static_cast<__bf16>(p[8 + i]);
      }
    } else {
      b.f = p;
    }
  }

  // acc[db] += X^T[dim x 32 rows] B[32 rows x 32 columns], kColSteps steps: X's
  // rows row0 .. row0 + 31 of the LDS tile, B the block the lanes hold. bf16:
  // slot j of half h in step (s, db) stands for row 16 s + 8 (j / 4) + 4 h + j %
  // 4, B's own order; a transpose read gives four consecutive rows of a lane's
  // element column. fp32: two rows a step.
  static constexpr int kColSteps = sizeof(T) == 2 ? 2 * kDBlocks : 16 * kDBlocks;
  using ColOperand = std::conditional_t<sizeof(T) == 2, v8bf, float>;
  __device__ static __forceinline__ ColOperand col_operand(const Lane &at, int bytes, int row0,
                                                           int step) {
    if constexpr (sizeof(T) == 2) {
      const int s = step / kDBlocks, db = step % kDBlocks;
      const int off = bytes + (row0 + 16 * s) / 4 * kGroup + db * 256;
      const v4s lo = lds_read_tr16(at.col[0] + off), hi = lds_read_tr16(at.col[1] + off);
      return __builtin_bit_cast(v8bf,
                                __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int e = step / kDBlocks, db = step % kDBlocks;
      return lds_read<float>(at.col[(e >> 2) & 1] +
                             (bytes + (row0 + 8 * (e >> 2)) / 4 * kGroup + db * 512 +
                              (e & 3) * 64));
    }
  }
  __device__ static __forceinline__ void col_step(const ColOperand &x, int step, const Block &b,
                                                  v16f (&acc)[kDBlocks]) {
    const int db = step % kDBlocks;
    if constexpr (sizeof(T) == 2)
      acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, step / kDBlocks ? b.hi : b.lo, acc[db],
                                                        0, 0, 0);
    else
      acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, b.f[step / kDBlocks], acc[db], 0, 0, 0);
  }
  __device__ static __forceinline__ void col_product(const Lane &at, int bytes, int row0,
                                                     const Block &b, v16f (&acc)[kDBlocks]) {
#pragma unroll
    for (int i = 0; i < kColSteps; ++i)
      col_step(col_operand(at, bytes, row0, i), i, b, acc);
  }

  // Zeroes what is not finite in the ROWS rows of the LDS tile at `tile`: the
  // values, or with WHOLE the rows that hold one. WAVES waves share the rows;
  // returns whether this one (`wave`) found any.
  template <bool WHOLE, int ROWS, int WAVES>
  __device__ static __forceinline__ bool zero_not_finite(uint32_t tile, int wave) {
    constexpr int P = C <= 4 ? 4 : C <= 8 ? 8 : C <= 16 ? 16 : 32; // lanes to a row
    constexpr int kTurn = kWave / P;                              // rows of a turn
    static_assert(ROWS % (kTurn * WAVES) == 0, "every lane takes part in every turn");
    const int lane = opaque(lane_id()); // nothing of this is kept in registers meanwhile
    const int c = lane % P, r0 = wave * kTurn + lane / P;
    auto address = [&](int r) {
      return tile + (r >> 2) * kGroup + (c >> 2) * 256 + (r & 3) * 64 +
             ((c & 3) ^ ((r >> 2) & 3)) * 16;
    };
    if (!__any(c < C && holds_not_finite<ROWS / (kTurn * WAVES), WAVES * kTurn>(r0, address)))
      return false;
    rare_path();
    constexpr uint32_t kLow = sizeof(T) == 2 ? 0x7f80u : 0x7f800000u, kHigh = 0x7f800000u;
    constexpr uint32_t kKeepHigh = sizeof(T) == 2 ? 0xffff0000u : 0u;
    constexpr uint32_t kKeepLow = sizeof(T) == 2 ? 0x0000ffffu : 0u;
#pragma unroll 1
    for (int r = r0; r < ROWS; r += WAVES * kTurn) {
      v4u u{0u, 0u, 0u, 0u}, clean;
      if (c < C)
        u = lds_read<v4u>(address(r));
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) { // an exponent of ones
        clean[e] = (u[e] & kLow) == kLow ? u[e] & kKeepHigh : u[e];
        clean[e] = (u[e] & kHigh) == kHigh ? clean[e] & kKeepLow : clean[e];
        bad |= clean[e] != u[e];
      }
      if constexpr (WHOLE) {
        const uint64_t row = __ballot(bad) >> (lane / P * P);
        bad = (row & ((uint64_t(1) << P) - 1)) != 0u;
        clean = v4u{0u, 0u, 0u, 0u};
      }
      if (bad && c < C)
        *reinterpret_cast<__attribute__((address_space(3))) v4u *>(address(r)) = clean;
    }
    return true;
  }
  // Whether the chunks at address(r), r = r0, r0 + STEP .. (N of them), hold a
  // value that is not finite.
  template <int N, int STEP, typename A>
  __device__ static __forceinline__ bool holds_not_finite(int r0, A &&address) {
    if constexpr (sizeof(T) == 2) {
      typedef uint16_t v2us __attribute__((ext_vector_type(2)));
      v2us top{};
#pragma unroll 4
      for (int i = 0; i < N; ++i) {
        const v4u u = lds_read<v4u>(address(r0 + i * STEP));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          top = __builtin_elementwise_max(top, __builtin_bit_cast(v2us, u[e] & 0x7fff7fffu));
      }
      return top[0] >= 0x7f80 || top[1] >= 0x7f80;
    } else {
      uint32_t top = 0;
#pragma unroll 4
      for (int i = 0; i < N; ++i) {
        const v4u u = lds_read<v4u>(address(r0 + i * STEP));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          top = max(top, u[e] & 0x7fffffffu);
      }
      return top >= 0x7f800000u;
    }
  }

  // Adds what zero_not_finite took off rows r0 .. r1 - 1 at p to the columns
  // whose lanes say sees(row): infinities and NaN as they are (an entry that a
  // column sees has a weight above zero in out and grad_v), or NaN.
  template <bool AS_NAN, typename S>
  __device__ static void add_not_finite(const T *p, int64_t stride, int dim, int32_t r0,
                                        int32_t r1, S &&sees, v16f (&acc)[kDBlocks]) {
    const int lane = lane_id(), half = lane >> 5;
#pragma unroll 1
    for (int32_t r = r0; r < r1; ++r) {
      const T *row = p + r * stride;
      const float x[2] = {lane < dim ? to_f32(row[lane]) : 0.f,
                          lane + kWave < dim ? to_f32(row[lane + kWave]) : 0.f};
      const uint64_t bad[2] = {__ballot(!isfinite(x[0])), __ballot(!isfinite(x[1]))};
      if (!(bad[0] | bad[1]))
        continue;
      const uint64_t none[2] = {__ballot(isnan(x[0])), __ballot(isnan(x[1]))};
      const uint64_t negative[2] = {__ballot(x[0] < 0.f), __ballot(x[1] < 0.f)};
      if (!sees(r))
        continue;
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db) {
        // the row's elements 32 db + 4 half .. as bits from 0 on
        auto bits = [&](const uint64_t (&m)[2]) {
          return static_cast<uint32_t>(m[db / 2] >> (32 * (db % 2))) >> (4 * half);
        };
        const uint32_t b = bits(bad), n = AS_NAN ? b : bits(none), s = bits(negative);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t d = 1u << (8 * (e >> 2) + (e & 3));
          const float v = n & d ? NAN : s & d ? -INFINITY : INFINITY;
          acc[db][e] += b & d ? v : 0.f;
          __builtin_amdgcn_sched_barrier(0); // registers, not speed
        }
      }
    }
  }

  // One lane's column of a [32 DB x 32] result, scaled, as a row of dim
  // elements at p; store_rest: what its rounding left over.
  template <bool VEC>
  __device__ static __forceinline__ void store_column(T *p, int dim, float mul,
                                                      const v16f (&acc)[kDBlocks]) {
    store<VEC>(p, dim, [&](float v) { return from_f32<T>(v * mul); }, acc);
  }
  template <bool VEC>
  __device__ static __forceinline__ void store_rest(T *p, int dim, float mul,
                                                    const v16f (&acc)[kDBlocks]) {
    store<VEC>(p, dim,
               [&](float v) { return from_f32<T>(v * mul - to_f32(from_f32<T>(v * mul))); }, acc);
  }

  template <bool VEC, typename F>
  __device__ static __forceinline__ void store(T *p, int dim, F &&f,
                                               const v16f (&acc)[kDBlocks]) {
    const int half = lane_id() >> 5;
#pragma unroll
    for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * db + 8 * g + 4 * half;
        T e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          e[i] = f(acc[db][4 * g + i]);
        if constexpr (VEC) { // dim is a multiple of E, so of 4
          if (d < dim) {
            if constexpr (sizeof(T) == 2)
              *reinterpret_cast<uint2 *>(p + d) = __builtin_bit_cast(uint2, e);
            else
              *reinterpret_cast<uint4 *>(p + d) = __builtin_bit_cast(uint4, e);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (d + i < dim)
              p[d + i] = e[i];
        }
      }
  }
};

// 16 (or 4) bytes per lane from a buffer straight into LDS, lane l's at lds +
// l * 16 (* 4); offsets outside the buffer write zeros. The caller waits
// (wait_stream) and keeps LDS reads of the target behind it.
__device__ __forceinline__ void dma16(const __amdgpu_buffer_rsrc_t &rsrc, uint32_t lds,
                                      uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(off), "s"(rsrc)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(const __amdgpu_buffer_rsrc_t &rsrc, uint32_t lds,
                                     uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(off), "s"(rsrc)
               : "memory", "m0");
}
// This wave's loads into LDS have landed, and its LDS reads have returned.
__device__ __forceinline__ void wait_stream() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void *p) { // wave-uniform
  return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)));
}

// A buffer whose pointer and size are the same in every lane, in scalar
// registers whatever the compiler can prove.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t wave_rsrc(const void *p, int64_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32));
  return buf_rsrc(reinterpret_cast<const void *>(static_cast<uint64_t>(hi) << 32 | lo),
                  __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(bytes)));
}

// Tiles of ROWS rows streamed from global memory into swizzled LDS tiles by
// THREADS threads (a workgroup, or a wave on its own). With VEC the loads go
// straight to LDS and stay in flight until wait_stream: no registers, no LDS
// writes. Lanes fill LDS in order, so each fetches what belongs at its place;
// rows past `valid` and chunks past dim become zeros.
template <typename T, int DP, int ROWS, int THREADS, bool VEC> struct TileStream {
  using Tile = AttnTile<T, DP>;
  static constexpr int kBytes = ROWS * Tile::C * 16;
  static constexpr int kPer = ROWS * Tile::C / THREADS;
  // Where a thread's loads step by whole swizzle periods (16 rows) they have
  // one chunk column, and rows a constant apart: one offset and a step for all.
  static constexpr bool kStep = THREADS / Tile::C % 16 == 0;
  static constexpr int kOffs = kStep ? 1 : kPer;
  uint32_t off[kOffs];

  __device__ __forceinline__ void init(int64_t row_stride, int dim) {
    const int t = threadIdx.x % THREADS;
#pragma unroll
    for (int i = 0; i < kOffs; ++i) {
      int r, c;
      Tile::place(t + i * THREADS, r, c);
      off[i] = c * Tile::E < dim ? static_cast<uint32_t>(r * row_stride * sizeof(T) + c * 16)
                                 : kBufOob;
    }
  }
  // base: the tile's first row; valid: rows from there on (may be 0 or less)
  __device__ __forceinline__ void issue(char *lds, const T *base, int64_t row_stride,
                                        int32_t valid, int dim) const {
    const int t = threadIdx.x % THREADS;
    const int32_t rows = min(valid, ROWS);
    if constexpr (VEC) {
      const int64_t bytes =
          rows > 0 ? ((rows - 1) * row_stride + dim) * static_cast<int64_t>(sizeof(T)) : 0;
      const __amdgpu_buffer_rsrc_t rsrc = wave_rsrc(base, bytes);
      const uint32_t to = lds_address(lds) + lds_address_of_wave(t);
      const uint32_t step = static_cast<uint32_t>(row_stride * sizeof(T)); // a row's bytes
      const uint32_t first = opaque(off[0]); // one register, not one for each step
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        dma16(rsrc, to + i * THREADS * 16,
              kStep ? first + i * (THREADS / Tile::C) * step : off[i % kOffs]);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        int r, c;
        Tile::place(t + i * THREADS, r, c);
        *reinterpret_cast<uint4 *>(lds + (t + i * THREADS) * 16) =
            Tile::template chunk<false>(base + r * row_stride, c, dim, r < rows);
      }
    }
  }

private:
  __device__ static __forceinline__ uint32_t lds_address_of_wave(int t) {
    return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(t / kWave * kWave * 16));
  }
};

// N matrix steps whose operands come from LDS: load(i) fetches step i's, A
// steps before use(i, operand) needs it. Left to itself the compiler, short of
// registers, reads each operand right before its product and waits out the
// read's latency there (the keys' kernel, 128 wide: 940 TFLOP/s so, 1058 ahead).
// `before`: what to do once the first operands are on their way.
// A = 0 leaves the order to it.
template <int N, int A, typename L, typename U, typename B>
__device__ __forceinline__ void ahead(L &&load, U &&use, B &&before) {
  if constexpr (A == 0) {
    before();
#pragma unroll
    for (int i = 0; i < N; ++i)
      use(i, load(i));
  } else {
    decltype(load(0)) f[A];
#pragma unroll
    for (int i = 0; i < A && i < N; ++i)
      f[i] = load(i);
    __builtin_amdgcn_sched_barrier(0);
    before();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      use(i, f[i % A]);
      if (i + A < N)
        f[i % A] = load(i + A);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}
template <int N, int A, typename L, typename U>
__device__ __forceinline__ void ahead(L &&load, U &&use) {
  ahead<N, A>(load, use, [] {});
}

// Entry r of a lane's 16 of a 32x32 block is row block_row(r) + 4 (lane / 32).
constexpr int block_row(int r) { return 8 * (r >> 2) + (r & 3); }

// Maximum and sum over the lane pair l, l ^ 32 (a column's two halves).
__device__ __forceinline__ float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

} // namespace rhip
