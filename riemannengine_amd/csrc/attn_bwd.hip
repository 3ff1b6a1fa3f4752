// Attention over packed sequences on gfx950, backward. With p = softmax rows
// (recomputed from lse), dp = do v^T and delta = rowsum(do o):
//   ds = p (dp - delta),  dq = scale ds k,  dk = scale ds^T q,  dv = p^T do.
// Two kernels: one over query rows (dq, and each row's statistics for the
// other), one over keys (dk and dv, summed over the query heads of a group
// inside the workgroup). Each gradient row is summed by one workgroup in a
// fixed order, so results do not change from run to run; the price is that
// scores and dp are computed twice (7 products instead of 5).
//
// Both have the forward's shapes: W blocks of 32 rows (keys) per workgroup,
// whose four waves read the same tiles of the other side (W = 4; 2: two waves
// share a block, each with half of every tile) or tiles of their own (W = 1),
// and add what they share at the end. With W = 1 the keys' kernel may also be
// split over workgroups, whose partial sums a last kernel adds.
#include "attn.hpp"

namespace rhip {
namespace {

constexpr int kBwdThreads = 256;
constexpr int kBwdWaves = kBwdThreads / kWave;
template <typename T, int DP, int W, bool KEYS> struct BwdShape {
  static constexpr int kRows = 32 * W;
  static constexpr int kParts = kBwdWaves / W; // waves that share a block of rows
  // The keys' kernel in bf16 at full width holds 192 registers of keys, values
  // and sums, which leaves none to read ahead with: its values stay in LDS,
  // where they fit beside 32-row tiles. (W = 1, 4 heads, one causal sequence of
  // 1000: 30 us from registers, which spill, 23 from LDS.)
  static constexpr bool kOwnInLds = KEYS && W != 2 && sizeof(T) == 2 && DP == 128;
  // Rows of the other side per LDS tile: 64 where they fit, 128 of narrow heads
  // in bf16 (32 wide, four sequences of 4096, 16 heads: 278 and 379 us in 64,
  // 264 and 352 in 128).
  static constexpr int kBN =
      W == 1 || (W == 4 && sizeof(T) == 4 && DP == 128) || kOwnInLds ? 32
      : sizeof(T) == 2 && DP == 32                                   ? 128
                                                                     : 64;
  // Registers let two workgroups into a CU. Two buffers where they leave LDS for
  // as many: two workgroups cover each other's waits better than a second
  // buffer does. (W = 1, two buffers and one workgroup, then one buffer and two:
  // fp32, 64 wide, 6 over 2 heads, three of 1100: dq 80 us, 71; bf16, 128 wide, 16
  // over 2 heads, one of 1500: keys' kernel 71 us, 40.)
  static constexpr bool kSlim = sizeof(T) == 2 || DP <= (KEYS && W == 4 ? 32 : 64);
  static constexpr int kStreams = W == 1 ? kBwdWaves : 1;
  static constexpr int kTileBytes = kBN * DP * sizeof(T);
  static constexpr int kStatBytes = kBN * 8; // (lse2, -delta) of a tile's rows
  static constexpr int kBufBytes = 2 * kTileBytes + kStatBytes;
  static constexpr int kBuffers = kStreams * 2 * kBufBytes <= (kSlim ? 80 : 160) * 1024 ? 2 : 1;
  static constexpr int kJoinRow = DP + 4; // floats per row of the joined sums
  static constexpr int kJoinBytes =
      W < 4 ? kBwdWaves * 32 * kJoinRow * static_cast<int>(sizeof(float)) : 0;
  static constexpr int kOwnBytes = kOwnInLds ? kRows * DP * static_cast<int>(sizeof(T)) : 0;
  static constexpr int kStageBytes = kStreams * kBuffers * kBufBytes + kOwnBytes;
  static constexpr int kLds = kStageBytes > kJoinBytes ? kStageBytes : kJoinBytes;
  // Waves per SIMD: two workgroups' where their LDS and registers fit; 64 wide in
  // bf16 three, within 168 registers, which the compiler would pass by two.
  static constexpr int kOccupancy = !kSlim || kLds > 80 * 1024                      ? 1
                                    : sizeof(T) == 2 && DP == 64 && kLds < 53 * 1024 ? 3
                                                                                     : 2;
};

// The first query row that sees key j, and the keys that row i sees.
__device__ __forceinline__ int32_t first_row(const AttnArgs &a, const AttnSeq &sq, int64_t j) {
  const int64_t i = a.causal ? j - (static_cast<int64_t>(sq.lk) - sq.lq) : 0;
  return static_cast<int32_t>(i < 0 ? 0 : (i > sq.lq ? sq.lq : i));
}
__device__ __forceinline__ int32_t keys_seen(const AttnArgs &a, const AttnSeq &sq, int64_t i) {
  const int64_t n =
      a.causal ? min<int64_t>(sq.lk, i + static_cast<int64_t>(sq.lk) - sq.lq + 1) : sq.lk;
  return static_cast<int32_t>(n < 0 ? 0 : n);
}

template <typename T>
__device__ __forceinline__ void put2(T *p, int dim, float v0, float v1, float mul) {
  const int lane = lane_id();
  if (lane < dim)
    p[lane] = from_f32<T>(v0 * mul);
  if (lane + kWave < dim)
    p[lane + kWave] = from_f32<T>(v1 * mul);
}

// One wave writes a row of dq, or of dk and dv; lane l holds elements l and
// l + 64 of its sum.
template <typename T>
__device__ void finish_dq(const AttnArgs &a, int64_t row, int head, float g0, float g1) {
  put2(static_cast<T *>(a.gq) + (row * a.heads + head) * a.dim, a.dim, g0, g1, a.scale);
}
template <typename T>
__device__ void finish_dkv(const AttnArgs &a, int64_t key, int kv, const float (&gk)[2],
                           const float (&gv)[2]) {
  const int64_t at = (key * a.kv_heads + kv) * a.dim;
  put2(static_cast<T *>(a.gk) + at, a.dim, gk[0], gk[1], a.scale);
  put2(static_cast<T *>(a.gv) + at, a.dim, gv[0], gv[1], 1.f);
}

// The columns a wave's lanes hold, as 32 rows of floats in LDS.
template <int DB>
__device__ __forceinline__ void spill_columns(float *rows, int row_floats, const v16f (&acc)[DB]) {
  const int lane = lane_id(), half = lane >> 5;
  float *mine = rows + (lane & 31) * row_floats;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<v4f *>(mine + 32 * db + 8 * g + 4 * half) =
          v4f{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
}
// Elements lane and lane + 64 of row r of the workgroup's, summed over the
// PARTS waves that share it in order.
template <int DP, int PARTS>
__device__ __forceinline__ void join_row(const float *rows, int row_floats, int r, float &v0,
                                         float &v1) {
  const int lane = lane_id();
  v0 = v1 = 0.f;
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const float *src = rows + ((r / 32 * PARTS + i) * 32 + r % 32) * row_floats;
    if (lane < DP)
      v0 += src[lane];
    if (lane + kWave < DP)
      v1 += src[lane + kWave];
  }
}

// dq of 128 (32) packed query rows of one key head's group over the keys;
// also the rows' statistics. Blocks are transposed as in the forward (S^T = K
// Q^T, dP^T = V dO^T), so dS^T is the right operand of dQ^T = K^T dS^T as it
// lies. dP's sums start at -delta.
//
// Bound by the matrix cores (four causal prompts of 4096, 16 over 4 heads, 128
// wide, bf16: 398 us, 1035 TFLOP/s), by the vector instructions at 32 wide (890).
//
// LOCAL: inside a window, as in the forward (causal, 16 over 4 heads of 128, four
// texts of up to 4096, window 1024: 132 us; both sides, 8 heads of 32, window 256:
// 32).
template <typename T, int DP, bool VEC, int W, bool LOCAL>
__global__ __launch_bounds__(kBwdThreads, (BwdShape<T, DP, W, false>::kOccupancy)) void
attn_dq_kernel(AttnArgs a) {
  using Shape = BwdShape<T, DP, W, false>;
  using Tile = AttnTile<T, DP>;
  using Frag = typename Tile::Frag;
  constexpr int kBN = Shape::kBN;
  constexpr int kAhead = sizeof(T) == 2 ? 4 : 0; // LDS operands on their way to the products
  constexpr int kB = kBN / 32 / (W == 2 ? 2 : 1); // blocks of a tile that are a wave's
  using Stream = TileStream<T, DP, kBN, W == 1 ? kWave : kBwdThreads, VEC>;
  __shared__ alignas(16) char lds[Shape::kLds];
  __shared__ int any_left_out;

  int32_t t, kv, split;
  if (!attn_item(a, t, kv, split))
    return;
  t = a.tiles - 1 - t; // as in the forward; the first keys have the most rows below
  const AttnSeq sq = query_tile(a, Shape::kRows, a.group, t);
  const int32_t n_rows = sq.lq * a.group, row0 = sq.tile * Shape::kRows;
  if (row0 >= n_rows)
    return;
  const int lane = lane_id(), half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int32_t wave0 = row0 + w / Shape::kParts * 32;
  const int b0 = W == 2 ? w % 2 * kB : 0; // the wave's first block of a tile
  const int32_t row = wave0 + (lane & 31);
  const bool row_ok = row < n_rows;
  const int32_t rc = min(row, n_rows - 1);
  const int32_t qi = rc / a.group;
  const int head = kv * a.group + rc % a.group;
  auto sees = [&](int32_t r) { return keys_seen(a, sq, r / a.group); };
  const int32_t lim = row_ok ? sees(row) : 0;
  const int32_t wg_lim = wave_uniform(sees(min(row0 + Shape::kRows, n_rows) - 1));
  const int32_t wg_full = wave_uniform(sees(row0));
  const int32_t wave_lim =
      wave_uniform(wave0 < n_rows ? sees(min(wave0 + 32, n_rows) - 1) : 0);
  const int32_t wave_full = wave_uniform(wave0 < n_rows ? sees(wave0) : 0);
  using Tiles = LocalTiles<kBN>;
  auto local = [&](int32_t r) {
    return LOCAL && r >= 0 ? local_keys(a, sq, r / a.group) : LocalKeys{0, 0, 0};
  };
  const LocalKeys mine = local(row_ok ? row : -1);
  const Tiles wg(local(row0), local(min(row0 + Shape::kRows, n_rows) - 1));
  const bool any_row = wave0 < n_rows;
  const Tiles wave(local(any_row ? wave0 : -1), local(any_row ? min(wave0 + 32, n_rows) - 1 : -1));
  auto cut = [&](int32_t kt) { // a tile of which some rows see a part
    return LOCAL ? !wg.all(kt * kBN, min((kt + 1) * kBN, sq.lk))
                 : wg_full < wg_lim && (kt + 1) * kBN > wg_full;
  };
  const int32_t kt1 = !a.gq ? 0 : LOCAL ? wg.count : (wg_lim + kBN - 1) / kBN; // 0: statistics alone
  const int32_t first = W == 1 ? w : 0, step = W == 1 ? kBwdWaves : 1;

  const T *kp = static_cast<const T *>(a.k) + sq.k0 * a.k_row + kv * a.k_head;
  const T *vp = static_cast<const T *>(a.v) + sq.k0 * a.v_row + kv * a.v_head;
  Stream ks, vs;
  ks.init(a.k_row, a.dim);
  vs.init(a.v_row, a.dim);
  char *stage = lds + (W == 1 ? w : 0) * Shape::kBuffers * Shape::kBufBytes;
  auto issue = [&](int32_t n, int buf) {
    const int32_t kt = LOCAL ? wg.tile(n) : n;
    char *to = stage + buf * Shape::kBufBytes;
    ks.issue(to, kp + static_cast<int64_t>(kt) * kBN * a.k_row, a.k_row, sq.lk - kt * kBN,
             a.dim);
    vs.issue(to + Shape::kTileBytes, vp + static_cast<int64_t>(kt) * kBN * a.v_row, a.v_row,
             sq.lk - kt * kBN, a.dim);
  };
  if (first < kt1)
    issue(first, 0);

  const int64_t gr = sq.q0 + static_cast<int64_t>(qi);
  const T *qp = static_cast<const T *>(a.q) + gr * a.q_row + head * a.q_head;
  const T *gp = static_cast<const T *>(a.go) + gr * a.go_row + head * a.go_head;
  const T *op = static_cast<const T *>(a.o) + (gr * a.heads + head) * a.dim;
  const T *rp = static_cast<const T *>(a.rest) + (gr * a.heads + head) * a.dim;
  Frag qf[Tile::kSteps], gf[Tile::kSteps];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < Tile::kSteps; ++s) {
    const int c = 2 * s + half;
    qf[s] = __builtin_bit_cast(Frag, Tile::template chunk<VEC>(qp, c, a.dim, row_ok));
    gf[s] = __builtin_bit_cast(Frag, Tile::template chunk<VEC>(gp, c, a.dim, row_ok));
    const Frag of = __builtin_bit_cast(Frag, Tile::template chunk<VEC>(op, c, a.dim, row_ok));
#pragma unroll
    for (int e = 0; e < Tile::E; ++e)
      delta = fmaf(static_cast<float>(gf[s][e]), static_cast<float>(of[e]), delta);
    if (sizeof(T) == 2 && a.rest) {
      const Frag rf = __builtin_bit_cast(Frag, Tile::template chunk<VEC>(rp, c, a.dim, row_ok));
#pragma unroll
      for (int e = 0; e < Tile::E; ++e)
        delta = fmaf(static_cast<float>(gf[s][e]), static_cast<float>(rf[e]), delta);
    }
  }
  delta = pair_sum(delta);
  float lse2 = 0.f; // log2 of the softmax's denominator
  if (row_ok) {
    const int64_t li = static_cast<int64_t>(head) * a.n_q + gr;
    lse2 = a.lse[li] * kLog2e;
    if (lse2 == INFINITY) // an infinite score: the row's probabilities are NaN
      lse2 = NAN;
    if (half == 0 && w % Shape::kParts == 0)
      a.stat[li] = make_float2(lse2, -delta);
  }

  // As in the forward, but for whole keys: where the row's statistics are finite, a
  // key that is not has probability zero and adds nothing but NaN at the places
  // that are not finite (its score counts as 0, so a row of scores all below -88,
  // where that weight overflows, gets NaN throughout). Where the statistics are
  // not finite, all of the row's sums are NaN.
  bool left_out = false;
  if (W > 1 && threadIdx.x == 0)
    any_left_out = 0;
  v16f dq[Tile::kDBlocks], dp0;
#pragma unroll
  for (int db = 0; db < Tile::kDBlocks; ++db)
    dq[db] = v16f{};
#pragma unroll
  for (int r = 0; r < 16; ++r)
    dp0[r] = -delta;

  const typename Tile::Lane lane_at = Tile::lane_addresses();
  const uint32_t stage_at = lds_address(stage);
  int buf = 0;
  for (int32_t n = first; n < kt1; n += step) {
    const int32_t kt = LOCAL ? wg.tile(n) : n;
    wait_stream(); // as in the forward
    if constexpr (W > 1)
      __syncthreads();
    if (cut(kt)) {
      rare_path();
      const bool found = Tile::template zero_not_finite<true, kBN, W == 1 ? 1 : kBwdWaves>(
          stage_at + buf * Shape::kBufBytes, W == 1 ? 0 : w);
      if constexpr (W > 1) {
        if (found)
          any_left_out = 1;
        __syncthreads();
        left_out = wave_uniform(any_left_out) != 0;
      } else {
        left_out |= found;
      }
    }
    const typename Tile::Lane at =
        lane_at.in(stage_at + buf * Shape::kBufBytes + b0 * (32 / 4) * Tile::kGroup);
    if (Shape::kBuffers == 2 && n + step < kt1)
      issue(n + step, buf ^ 1);
    const int32_t j0 = kt * kBN + 32 * b0;
    if (W == 1 || (LOCAL ? wave.some(j0, j0 + 32 * kB) : j0 < wave_lim)) {
      const bool masked = LOCAL ? !wave.all(j0, j0 + 32 * kB) : j0 + 32 * kB > wave_full;
#pragma unroll
      for (int b = 0; b < kB; ++b) {
        v16f s{}, dp = dp0;
        ahead<2 * Tile::kSteps, kAhead>(
            [&](int i) {
              return Tile::row_operand(at, i % 2 * Shape::kTileBytes, 32 * b, i / 2);
            },
            [&](int i, const Frag &x) {
              if (i % 2)
                Tile::mma(x, gf[i / 2], dp);
              else
                Tile::mma(x, qf[i / 2], s);
            });
        typename Tile::Block ds;
        ahead<Tile::kColSteps, kAhead>(
            [&](int i) { return Tile::col_operand(at, 0, 32 * b, i); },
            [&](int i, const typename Tile::ColOperand &x) { Tile::col_step(x, i, ds, dq); },
            [&] {
#pragma unroll
              for (int r = 0; r < 16; ++r)
                s[r] = exp2_fast(fmaf(s[r], a.c, -lse2)) * dp[r];
              if (masked) {
                rare_path();
                const int32_t at0 = j0 + 32 * b + 4 * half;
                const int32_t seen = lim - at0;
                const int32_t lo = mine.lo - at0, hi = mine.hi - at0, sinks = mine.first - at0;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                  const int j = block_row(r);
                  s[r] = (LOCAL ? (j >= lo && j < hi) || j < sinks : j < seen) ? s[r] : 0.f;
                }
              }
              Tile::pack(s, ds);
            });
      }
    }
    if (Shape::kBuffers == 2) {
      buf ^= 1;
    } else if (n + step < kt1) {
      wait_stream();
      if constexpr (W > 1)
        __syncthreads();
      issue(n + step, 0);
    }
  }
  if (!a.gq)
    return;
  if (LOCAL) {
    if (left_out)
#pragma unroll 1
      for (int32_t n = 0; n < kt1; ++n) {
        const int32_t kt = wg.tile(n);
        if (cut(kt))
          Tile::template add_not_finite<true>(
              kp, a.k_row, a.dim, kt * kBN, min((kt + 1) * kBN, sq.lk),
              [&](int32_t j) { return (j >= mine.lo && j < mine.hi) || j < mine.first; }, dq);
      }
  } else if (left_out)
    Tile::template add_not_finite<true>(kp, a.k_row, a.dim, max(wg_full - kBN, 0), wave_lim,
                                        [&](int32_t j) { return j < lim; }, dq);
  if constexpr (W == 4) {
    const int32_t my_row = wave0 + (opaque(lane) & 31); // not kept through the loop
    if (my_row < n_rows) {
      const int64_t place = (sq.q0 + static_cast<int64_t>(my_row / a.group)) * a.heads +
                            kv * a.group + my_row % a.group;
      Tile::template store_column<VEC>(static_cast<T *>(a.gq) + place * a.dim, a.dim, a.scale, dq);
    }
  } else {
    __syncthreads(); // every wave is past its tiles
    float *join = reinterpret_cast<float *>(lds);
    spill_columns(join + w * 32 * Shape::kJoinRow, Shape::kJoinRow, dq);
    __syncthreads();
    for (int r = w; r < Shape::kRows && row0 + r < n_rows; r += kBwdWaves) {
      float g0, g1;
      join_row<DP, Shape::kParts>(join, Shape::kJoinRow, r, g0, g1);
      finish_dq<T>(a, sq.q0 + static_cast<int64_t>((row0 + r) / a.group),
                   kv * a.group + (row0 + r) % a.group, g0, g1);
    }
  }
}

// The launch over the keys apart: tile t of their sequences, `apart` keys each.
__device__ __forceinline__ AttnSeq apart_tile(const AttnArgs &a, int bm, int32_t t,
                                              int32_t &room) {
  const int32_t per = a.apart / bm;
  AttnSeq q;
  q.s = t / per, q.tile = t - q.s * per;
  room = 0, q.k0 = 0;
  if (q.s < a.n_seq) {
    q.k0 = q.s == 0 ? 0 : clamp_off(a.k_off[q.s], 0, a.n_k);
    room = clamp_off(a.k_off[q.s + 1], q.k0, a.n_k) - q.k0;
  }
  query_range(a, q, room);
  room = wave_uniform(room);
  return wave_uniform(q);
}
// Rows of a split's partial sums, and where key j of a sequence stands there.
__device__ __forceinline__ int64_t partial_rows(const AttnArgs &a, bool apart) {
  return apart ? static_cast<int64_t>(a.n_seq) * a.apart : a.n_k;
}
__device__ __forceinline__ int64_t partial_row(const AttnArgs &a, const AttnSeq &sq, bool apart,
                                               int32_t j) {
  return (apart ? static_cast<int64_t>(sq.s) * a.apart : sq.k0) + j;
}

// dk and dv of 128 (32) keys of one key head over the query rows of every
// head of its group. A lane holds one key's column (S = Q K^T, dP = dO V^T),
// so P and dS are the right operands of dV^T = dO^T P and dK^T = Q^T dS as
// they lie.
//
// Bound by the matrix cores and by the tiles' reads from LDS (same prompts: 613
// us, 897 TFLOP/s, four products a block against the other kernel's three).
//
// LOCAL: inside a window (LocalRows). The keys of the tiles that hold sinks, which
// rows of the whole sequence see, are a launch of their own (apart_pass), whose
// workgroups split those rows; partial sums then lie by sequence. (Four causal
// texts of up to 4096, 16 over 4 heads of 128, window 1024, 4 sinks: 151 to 158 us, 29
// for the keys apart, joins of 16 and 8; in one launch the sinks' workgroups alone
// would go through every row.)
template <typename T, int DP, bool VEC, int W, bool LOCAL>
__global__ __launch_bounds__(kBwdThreads, (BwdShape<T, DP, W, true>::kOccupancy)) void
attn_dkv_kernel(AttnArgs a) {
  using Shape = BwdShape<T, DP, W, true>;
  using Tile = AttnTile<T, DP>;
  using Frag = typename Tile::Frag;
  constexpr int kBM = Shape::kBN;
  constexpr bool kVLds = Shape::kOwnBytes > 0;
  // LDS operands on their way to the products (96 wide: 490 us for 558 left to the
  // compiler, four causal texts of 4096, 16 over 4 heads)
  constexpr int kAhead = kVLds || (sizeof(T) == 2 && DP == 96) ? 3 : 0;
  constexpr int kB = kBM / 32 / (W == 2 ? 2 : 1);
  using Stream = TileStream<T, DP, kBM, W == 1 ? kWave : kBwdThreads, VEC>;
  __shared__ alignas(16) char lds[Shape::kLds];
  __shared__ int any_left_out;

  int32_t t, kv, split;
  if (!attn_item(a, t, kv, split))
    return;
  int32_t room;
  const bool apart = LOCAL && a.apart_pass;
  const AttnSeq sq = apart ? apart_tile(a, Shape::kRows, t, room)
                           : key_tile(a, Shape::kRows, t, room);
  const int32_t key0 = sq.tile * Shape::kRows;
  // keys below `other` are the other launch's (whole waves; those behind the last
  // sequence are in none)
  const int32_t other = LOCAL && !apart && sq.s < a.n_seq ? a.apart : 0;
  if (key0 >= room || key0 + Shape::kRows <= other)
    return;
  const int lane = lane_id(), half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int32_t wave0 = key0 + w / Shape::kParts * 32;
  const int b0 = W == 2 ? w % 2 * kB : 0;
  const int32_t key = wave0 + (lane & 31);
  const bool key_ok = key < sq.lk;
  const int32_t lo = first_row(a, sq, key);
  // no earlier row sees any key of the wave's; every later row sees all
  const int32_t wave_lo = wave_uniform(first_row(a, sq, wave0));
  const int32_t wave_full = wave_uniform(first_row(a, sq, wave0 + 31));
  const int32_t wg_full =
      wave_uniform(first_row(a, sq, min(key0 + Shape::kRows, sq.lk) - 1));
  // LOCAL: the rows that see some key of the workgroup's (wave's), and those
  // that see all of them; the lane's
  auto rows_of = [&](int32_t from, int32_t to, LocalRows &some, LocalRows &all) {
    const int32_t last = max(min(to, sq.lk) - 1, from);
    const LocalRows x = local_rows(a, sq, from), y = local_rows(a, sq, last);
    some = {wave_uniform(x.lo), wave_uniform(from < a.sinks ? sq.lq : y.hi)};
    all = {wave_uniform(y.lo), wave_uniform(last < a.sinks
                                                ? sq.lq
                                                : local_rows(a, sq, max(from, a.sinks)).hi)};
  };
  LocalRows wg_some{}, wg_all{}, wave_some{}, wave_all{}, mine{};
  if constexpr (LOCAL) {
    rows_of(max(key0, other), key0 + Shape::kRows, wg_some, wg_all);
    if (wave0 >= other) {
      rows_of(wave0, wave0 + 32, wave_some, wave_all);
      mine = local_rows(a, sq, key);
    }
  }
  const int32_t it0 = (LOCAL ? wg_some.lo : wave_uniform(first_row(a, sq, key0))) / kBM;
  const int32_t rows_end = LOCAL ? wg_some.hi : sq.lq;
  auto cut = [&](int32_t i) { // a tile of rows from i on, some of which do not see all keys
    return LOCAL ? !(i >= wg_all.lo && min(i + kBM, sq.lq) <= wg_all.hi) : i < wg_full;
  };
  // tiles of query rows from the first that sees a key, for each head; this
  // workgroup's part of them
  const int32_t per_head = key0 < sq.lk ? max((rows_end + kBM - 1) / kBM - it0, 0) : 0;
  int32_t n0 = 0, n1 = per_head * a.group;
  if (a.splits > 1) {
    const int32_t per = (n1 + a.splits - 1) / a.splits;
    n0 = min(split * per, n1);
    n1 = min(n0 + per, n1);
  }
  const int32_t first = n0 + (W == 1 ? w : 0), step = W == 1 ? kBwdWaves : 1;

  Stream qs, gs;
  qs.init(a.q_row, a.dim);
  gs.init(a.go_row, a.dim);
  char *stage = lds + (W == 1 ? w : 0) * Shape::kBuffers * Shape::kBufBytes;
  auto issue = [&](int32_t n, int buf) {
    const int h = n / per_head, head = kv * a.group + h;
    const int32_t i0 = (it0 + n - h * per_head) * kBM;
    const int64_t r0 = sq.q0 + static_cast<int64_t>(i0);
    char *to = stage + buf * Shape::kBufBytes;
    qs.issue(to, static_cast<const T *>(a.q) + r0 * a.q_row + head * a.q_head, a.q_row,
             sq.lq - i0, a.dim);
    gs.issue(to + Shape::kTileBytes,
             static_cast<const T *>(a.go) + r0 * a.go_row + head * a.go_head, a.go_row,
             sq.lq - i0, a.dim);
    // (lse2, -delta) of the tile's rows, parted: for every 32 rows 32 of each
    const __amdgpu_buffer_rsrc_t rsrc =
        wave_rsrc(a.stat + static_cast<int64_t>(head) * a.n_q + r0,
                  static_cast<int64_t>(min(sq.lq - i0, kBM)) * 8);
    const int block = W == 1 ? 0 : w;
    if (block * 32 < kBM)
      dma4(rsrc, lds_address(to + 2 * Shape::kTileBytes + block * 256),
           (block * 32 + (lane & 31)) * 8 + half * 4);
  };
  char *own = lds + Shape::kStreams * Shape::kBuffers * Shape::kBufBytes;
  if (first < n1)
    issue(first, 0);
  if (kVLds && n0 < n1) { // waited for in the first turn; without one it may not start
    TileStream<T, DP, Shape::kRows, kBwdThreads, VEC> os;
    os.init(a.v_row, a.dim);
    os.issue(own,
             static_cast<const T *>(a.v) + (sq.k0 + static_cast<int64_t>(key0)) * a.v_row +
                 kv * a.v_head,
             a.v_row, sq.lk - key0, a.dim);
  }

  const int64_t gk = sq.k0 + static_cast<int64_t>(key);
  const T *kp = static_cast<const T *>(a.k) + gk * a.k_row + kv * a.k_head;
  const T *vp = static_cast<const T *>(a.v) + gk * a.v_row + kv * a.v_head;
  Frag kf[Tile::kSteps], vf[kVLds ? 1 : Tile::kSteps];
#pragma unroll
  for (int s = 0; s < Tile::kSteps; ++s) {
    const int c = 2 * s + half;
    kf[s] = __builtin_bit_cast(Frag, Tile::template chunk<VEC>(kp, c, a.dim, key_ok));
    if constexpr (!kVLds)
      vf[s] = __builtin_bit_cast(Frag, Tile::template chunk<VEC>(vp, c, a.dim, key_ok));
  }
  // As in the forward: values of grad_out that are not finite, and whole query
  // rows that hold one, in tiles of which some keys are not seen. Such a query
  // row's statistics are not finite, so what it adds is NaN without its values.
  bool left_out = false;
  if (W > 1 && threadIdx.x == 0)
    any_left_out = 0;
  v16f dk[Tile::kDBlocks], dv[Tile::kDBlocks];
#pragma unroll
  for (int db = 0; db < Tile::kDBlocks; ++db)
    dk[db] = dv[db] = v16f{};

  const typename Tile::Lane lane_at = Tile::lane_addresses();
  const uint32_t stage_at = lds_address(stage);
  typename Tile::Lane own_at{}; // this wave's keys in `own`
  if constexpr (kVLds)
    own_at = lane_at.in(lds_address(own) + w / Shape::kParts * (32 / 4) * Tile::kGroup);
  if constexpr (kVLds && W == 1) { // waves take turns of their own
    wait_stream();
    __syncthreads();
  }
  int buf = 0;
  for (int32_t n = first; n < n1; n += step) {
    wait_stream();
    if constexpr (W > 1)
      __syncthreads();
    if (cut((it0 + n % per_head) * kBM)) {
      rare_path();
      const uint32_t tile = stage_at + buf * Shape::kBufBytes;
      constexpr int kShare = W == 1 ? 1 : kBwdWaves;
      Tile::template zero_not_finite<true, kBM, kShare>(tile, W == 1 ? 0 : w);
      const bool found = Tile::template zero_not_finite<false, kBM, kShare>(
          tile + Shape::kTileBytes, W == 1 ? 0 : w);
      if constexpr (W > 1) {
        if (found)
          any_left_out = 1;
        __syncthreads();
        left_out = wave_uniform(any_left_out) != 0;
      } else {
        left_out |= found;
      }
    }
    const typename Tile::Lane at =
        lane_at.in(stage_at + buf * Shape::kBufBytes + b0 * (32 / 4) * Tile::kGroup);
    const uint32_t stat = opaque(stage_at + buf * Shape::kBufBytes + 2 * Shape::kTileBytes +
                                 b0 * 256 + half * 16);
    if (Shape::kBuffers == 2 && n + step < n1)
      issue(n + step, buf ^ 1);
    const int32_t i0 = (it0 + n % per_head) * kBM + 32 * b0;
    if (LOCAL ? i0 + 32 * kB > wave_some.lo && i0 < wave_some.hi : i0 + 32 * kB > wave_lo) {
      const bool masked = LOCAL ? i0 < wave_all.lo || i0 + 32 * kB > wave_all.hi
                                : i0 < wave_full || i0 + 32 * kB > sq.lq;
#pragma unroll
      for (int b = 0; b < kB; ++b) {
        v16f s{}, dp;
        // this lane's rows: 8 g + 4 half + e
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const v4f d = lds_read<v4f>(stat + b * 256 + 128 + g * 32);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            dp[4 * g + e] = d[e];
        }
        // dP, then S
        struct Pair {
          Frag x, v;
        };
        ahead<2 * Tile::kSteps, kAhead>(
            [&](int i) {
              Pair f{};
              f.x = Tile::row_operand(at, i < Tile::kSteps ? Shape::kTileBytes : 0, 32 * b,
                                      i % Tile::kSteps);
              if (kVLds && i < Tile::kSteps)
                f.v = Tile::row_operand(own_at, 0, 0, i);
              return f;
            },
            [&](int i, const Pair &f) {
              if (i >= Tile::kSteps)
                Tile::mma(f.x, kf[i - Tile::kSteps], s);
              else
                Tile::mma(f.x, kVLds ? f.v : vf[kVLds ? 0 : i], dp);
            });
        typename Tile::Block p, ds;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const v4f l = lds_read<v4f>(stat + b * 256 + g * 32);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[4 * g + e] = exp2_fast(fmaf(s[4 * g + e], a.c, -l[e]));
            dp[4 * g + e] *= s[4 * g + e];
          }
        }
        if (masked) {
          rare_path();
          const int32_t at0 = i0 + 32 * b + 4 * half;
          const int32_t from = (LOCAL ? mine.lo : lo) - at0, to = (LOCAL ? mine.hi : sq.lq) - at0;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const bool sees = block_row(r) >= from && block_row(r) < to;
            s[r] = sees ? s[r] : 0.f;
            dp[r] = sees ? dp[r] : 0.f;
          }
        }
        Tile::pack(s, p);
        Tile::col_product(at, Shape::kTileBytes, 32 * b, p, dv);
        Tile::pack(dp, ds);
        Tile::col_product(at, 0, 32 * b, ds, dk);
      }
    }
    if (Shape::kBuffers == 2) {
      buf ^= 1;
    } else if (n + step < n1) {
      wait_stream();
      if constexpr (W > 1)
        __syncthreads();
      issue(n + step, 0);
    }
  }

  if (left_out)
    for (int head = kv * a.group; head < (kv + 1) * a.group; ++head) {
      const T *gp = static_cast<const T *>(a.go) + sq.q0 * a.go_row + head * a.go_head;
      if (LOCAL) {
#pragma unroll 1
        for (int32_t i = it0 * kBM; i < rows_end; i += kBM)
          if (cut(i))
            Tile::template add_not_finite<false>(
                gp, a.go_row, a.dim, i, min(i + kBM, sq.lq),
                [&](int32_t r) { return r >= mine.lo && r < mine.hi; }, dv);
      } else {
        Tile::template add_not_finite<false>(gp, a.go_row, a.dim, wave_lo,
                                             min(wg_full + kBM, sq.lq),
                                             [&](int32_t i) { return i >= lo; }, dv);
      }
    }
  // Rows of the region behind the keys in use get zeros: where their lanes
  // share a wave with keys in use, those met them as a key of zeros, with a
  // probability of exp(-lse).
  const int32_t my_key = wave0 + (opaque(lane_id()) & 31); // not kept through the loop
  if (my_key >= sq.lk) {
#pragma unroll
    for (int db = 0; db < Tile::kDBlocks; ++db)
      dk[db] = dv[db] = v16f{};
  }
  if constexpr (W == 4) {
    if (a.splits > 1) {
      if (my_key < room && (!LOCAL || my_key >= other)) {
        const int64_t place =
            ((split * partial_rows(a, apart) + partial_row(a, sq, apart, my_key)) * a.kv_heads +
             kv) * a.dim;
        using Sum = AttnTile<float, DP>;
        if (a.dim % 4 == 0) {
          Sum::template store_column<true>(a.part_k + place, a.dim, 1.f, dk);
          Sum::template store_column<true>(a.part_v + place, a.dim, 1.f, dv);
        } else {
          Sum::template store_column<false>(a.part_k + place, a.dim, 1.f, dk);
          Sum::template store_column<false>(a.part_v + place, a.dim, 1.f, dv);
        }
      }
      return;
    }
    if (my_key < room && (!LOCAL || my_key >= other)) {
      const int64_t place =
          ((sq.k0 + static_cast<int64_t>(my_key)) * a.kv_heads + kv) * a.dim;
      Tile::template store_column<VEC>(static_cast<T *>(a.gk) + place, a.dim, a.scale, dk);
      Tile::template store_column<VEC>(static_cast<T *>(a.gv) + place, a.dim, 1.f, dv);
    }
  } else {
    // add the waves' sums, dk then dv through the same LDS; a wave ends with
    // rows w, w + 4, .. of both
    float *join = reinterpret_cast<float *>(lds);
    constexpr int kMine = Shape::kRows / kBwdWaves;
    float rk[kMine][2], rv[kMine][2];
    __syncthreads();
    spill_columns(join + w * 32 * Shape::kJoinRow, Shape::kJoinRow, dk);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMine; ++u)
      join_row<DP, Shape::kParts>(join, Shape::kJoinRow, w + u * kBwdWaves, rk[u][0], rk[u][1]);
    __syncthreads();
    spill_columns(join + w * 32 * Shape::kJoinRow, Shape::kJoinRow, dv);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMine; ++u)
      join_row<DP, Shape::kParts>(join, Shape::kJoinRow, w + u * kBwdWaves, rv[u][0], rv[u][1]);
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      const int32_t j = key0 + w + u * kBwdWaves;
      if (j >= room)
        break;
      if (LOCAL && j < other)
        continue;
      if (a.splits == 1) {
        finish_dkv<T>(a, sq.k0 + static_cast<int64_t>(j), kv, rk[u], rv[u]);
      } else {
        const int64_t place =
            ((split * partial_rows(a, apart) + partial_row(a, sq, apart, j)) * a.kv_heads + kv) *
            a.dim;
        put2(a.part_k + place, a.dim, rk[u][0], rk[u][1], 1.f);
        put2(a.part_v + place, a.dim, rv[u][0], rv[u][1], 1.f);
      }
    }
  }
}

// Adds the splits' partial sums of dk and dv, TURN of them at a time: one wave per
// key and key head, WIDE: of more than 64 elements. Few splits of many keys are
// bound by memory (two of 8191 keys, 4 heads of 128: 17 us), many of few keys by the
// loads' latency (32 of 128 keys: 8 us; with branches around the lanes' loads 22 and
// 21). Six splits of 3301 keys, 2 heads of 40: 5.1 us; in turns of four, with the
// second half of a wide head's loads, 5.5; in turns of 16 8.9.
template <typename T, int TURN, bool WIDE>
__global__ __launch_bounds__(kBwdThreads) void attn_dkv_join_kernel(AttnArgs a) {
  constexpr int U = WIDE ? 2 : 1;
  const int64_t rows = partial_rows(a, a.apart_pass) * a.kv_heads;
  const int lane = lane_id();
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * kBwdWaves + threadIdx.x / kWave; at < rows;
       at += static_cast<int64_t>(gridDim.x) * kBwdWaves) {
    int64_t key = at / a.kv_heads;
    if (a.apart_pass) { // key j of a sequence, if its region holds it
      const int32_t seq = static_cast<int32_t>(key / a.apart);
      const int32_t j = static_cast<int32_t>(key - static_cast<int64_t>(seq) * a.apart);
      const int32_t k0 = seq == 0 ? 0 : clamp_off(a.k_off[seq], 0, a.n_k);
      if (j >= clamp_off(a.k_off[seq + 1], k0, a.n_k) - k0)
        continue;
      key = k0 + static_cast<int64_t>(j);
    }
    float gk[2] = {0.f, 0.f}, gv[2] = {0.f, 0.f};
    // lanes behind the head's width read its last element, places behind the last
    // split that split's: with no branch around them all loads of a turn are under
    // way at once
    const int c[2] = {min(lane, a.dim - 1), min(lane + kWave, a.dim - 1)};
    for (int s0 = 0; s0 < a.splits; s0 += TURN) {
      float k[TURN][U], v[TURN][U];
#pragma unroll
      for (int i = 0; i < TURN; ++i) {
        const int64_t p = (min(s0 + i, a.splits - 1) * rows + at) * a.dim;
#pragma unroll
        for (int u = 0; u < U; ++u)
          k[i][u] = a.part_k[p + c[u]], v[i][u] = a.part_v[p + c[u]];
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < TURN; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          gk[u] += s0 + i < a.splits ? k[i][u] : 0.f;
          gv[u] += s0 + i < a.splits ? v[i][u] : 0.f;
        }
    }
    finish_dkv<T>(a, key, static_cast<int>(at % a.kv_heads), gk, gv);
  }
}

AttnPlan plan_queries(int64_t rows, int32_t n_seq, int32_t kv_heads, int32_t dtype) {
  AttnPlan p{attn_waves(rows, kv_heads, dtype), 0, 1};
  p.tiles = rows / (32 * p.waves) + n_seq + 1;
  return p;
}

// The keys' kernel: W and the splits by estimated time, in microseconds. A
// 32x32 block takes a SIMD `block` when two waves keep it busy (measured over
// whole launches: 128-wide bf16 1.14 us, narrower ones in
// proportion; fp32 at 125 TFLOP/s) and a wave on its own 1.5 times that. The
// launch takes the larger of all blocks over 1024 SIMDs and the longest
// workgroup's blocks one after another (under a causal mask the first keys'
// have twice the mean; sequences of unlike lengths a quarter more). W = 2 and
// 1 cost 1.3 and 1.7 times the blocks (less shared per tile); every round of
// workgroups 10 us to start and finish; splits write and read fp32 partial
// sums at 4.5 TB/s. (16 over 4 heads, 128 wide, four causal texts of 4096: 912
// us with one split, 686 with three, joining included; 8 heads, eight of
// 1024: 70 us with one, 113 with two.)
AttnPlan plan_keys(int64_t n_q, int64_t n_k, int32_t n_seq, int32_t heads, int32_t kv_heads,
                   int32_t dim, int32_t causal, int32_t dtype, const AttnWindow &window) {
  const int64_t seqs = std::max<int64_t>(1, std::min<int64_t>(n_seq, n_k));
  double rows = static_cast<double>(n_q) * (heads / kv_heads) / seqs; // per key
  // a window's rows, and no mask's half of them (unless sinks are most of the keys)
  if (window.window > 0 && window.sinks <= n_k / seqs + 128) {
    const double seen =
        (static_cast<double>(window.window) * (causal ? 1 : 2) + 64) * (heads / kv_heads);
    causal = causal && seen > rows;
    rows = std::min(rows, seen);
  }
  const double block =
      1.14 * (dim <= 32 ? 0.25 : dim <= 64 ? 0.5 : dim <= 96 ? 0.8 : 1.0) * (dtype == RHIP_F32 ? 7.5 : 1.0);
  const double all = static_cast<double>(n_k) * kv_heads * rows * (causal ? 0.5 : 1.0) / 1024.0;
  const double traffic = static_cast<double>(n_k) * kv_heads * dim * 16 / 4.5e6;
  AttnPlan best{};
  double least = 0.0;
  for (int32_t w = 4; w >= 1; w /= 2) {
    const double wgs = static_cast<double>(n_k / (32 * w) + seqs) * kv_heads;
    for (int32_t s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
      // a split gets four 32-row tiles for each wave, at least
      if (s > 1 && rows < 512.0 * s)
        break;
      const double spread = all / 1024.0 * block * (w == 4 ? 1.0 : w == 2 ? 1.3 : 1.7);
      const double longest = 1.25 * rows / 32.0 * w / 4.0 / s * block * 1.5;
      const double t = std::max(spread, longest) + (wgs * s / 512.0 + 1.0) * 10.0 +
                       (s > 1 ? 4.0 + s * traffic : 0.0);
      if (best.waves == 0 || t < least) {
        least = t;
        best = {w, n_k / (32 * w) + n_seq + 1, s};
      }
    }
  }
  return best;
}

} // namespace

AttnPlan attn_queries_plan(const rhip_attn &d) {
  return plan_queries(d.n_q * (d.heads / d.kv_heads), d.n_seq, d.kv_heads, d.dtype);
}
AttnPlan attn_keys_plan(const rhip_attn &d, const AttnWindow &window) {
  return plan_keys(d.n_q, d.n_k, d.n_seq, d.heads, d.kv_heads, d.dim, d.causal, d.dtype, window);
}

// Tiles of 32 keys (W = 1), each over all rows of its sequence in as many parts
// as fill the chip twice, each part of 128 rows (a tile a wave) of the mean sequence
// at least. (Four causal texts to 4096, 16 over 4 heads of 128, 4 sinks: 38 us in
// 16 parts, 55 in four.)
AttnApart attn_apart_plan(const rhip_attn &d, const AttnWindow &window) {
  if (window.window == 0 || window.sinks == 0 || d.n_seq == 0 || d.n_k == 0)
    return {};
  AttnApart p{};
  // Whole blocks. Where they would be more than the keys there are, sinks are
  // most of every sequence, and all keys stay in one launch.
  const int64_t keys = align_up(window.sinks, 32);
  if (keys > d.n_k / d.n_seq + 128)
    return p;
  p.keys = static_cast<int32_t>(keys);
  p.plan.waves = 1;
  p.plan.tiles = d.n_seq * (keys / 32);
  const int64_t rows = d.n_q / d.n_seq * (d.heads / d.kv_heads);
  const int64_t busy = p.plan.tiles * d.kv_heads;
  p.plan.splits = 1;
  while (p.plan.splits < 64 && busy * p.plan.splits < 512 && rows >= 256 * p.plan.splits)
    p.plan.splits *= 2;
  return p;
}

void attn_backward_run(const AttnArgs &args, const AttnApart &apart, int32_t dtype, bool vec,
                       hipStream_t stream) {
  const AttnPlan pq =
      plan_queries(static_cast<int64_t>(args.n_q) * args.group, args.n_seq, args.kv_heads, dtype);
  const AttnPlan pk = plan_keys(args.n_q, args.n_k, args.n_seq, args.heads, args.kv_heads,
                                args.dim, args.causal, dtype, {args.window, args.sinks});
  with_attn(dtype, args.dim, vec, [&](auto t, auto dp, auto v) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    constexpr bool VEC = decltype(v)::value;
    const dim3 b(kBwdThreads);
    if (args.n_q > 0) {
      with_waves(pq.waves, [&](auto w) {
        constexpr int W = decltype(w)::value;
        const unsigned spread = spread_lds<W>(args, BwdShape<T, DP, W, false>::kLds);
        attn_launches(args, pq, kBwdThreads, [&](const AttnArgs &part, unsigned groups) {
          if (args.window > 0)
            hipLaunchKernelGGL((attn_dq_kernel<T, DP, VEC, W, true>), dim3(groups), b, spread,
                               stream, part);
          else
            hipLaunchKernelGGL((attn_dq_kernel<T, DP, VEC, W, false>), dim3(groups), b, spread,
                               stream, part);
        });
      });
    }
    if (!args.gk || args.n_k == 0)
      return;
    auto join = [&](AttnArgs a, int64_t keys, int32_t splits) {
      const int64_t rows = keys * args.kv_heads;
      a.splits = splits;
      const dim3 groups(
          static_cast<unsigned>(std::min(ceil_div(rows, kBwdWaves), max_groups(kBwdThreads))));
      auto launch = [&](auto turn) {
        constexpr int TURN = decltype(turn)::value;
        if (args.dim > kWave)
          hipLaunchKernelGGL((attn_dkv_join_kernel<T, TURN, true>), groups, b, 0, stream, a);
        else
          hipLaunchKernelGGL((attn_dkv_join_kernel<T, TURN, false>), groups, b, 0, stream, a);
      };
      if (splits > 8)
        launch(std::integral_constant<int, 16>{});
      else if (splits == 6)
        launch(std::integral_constant<int, 6>{});
      else if (splits > 3)
        launch(std::integral_constant<int, 4>{});
      else
        launch(std::integral_constant<int, 2>{});
      RHIP_LAUNCH_CHECK();
    };
    with_waves(pk.waves, [&](auto w) {
      constexpr int W = decltype(w)::value;
      attn_launches(args, pk, kBwdThreads, [&](const AttnArgs &part, unsigned groups) {
        if (args.window > 0)
          hipLaunchKernelGGL((attn_dkv_kernel<T, DP, VEC, W, true>), dim3(groups), b, 0, stream,
                             part);
        else
          hipLaunchKernelGGL((attn_dkv_kernel<T, DP, VEC, W, false>), dim3(groups), b, 0, stream,
                             part);
      });
    });
    if (pk.splits > 1)
      join(args, args.n_k, pk.splits);
    if (apart.keys > 0) {
      AttnArgs a = args;
      a.apart_pass = 1;
      a.part_k = args.apart_k, a.part_v = args.apart_v;
      attn_launches(a, apart.plan, kBwdThreads, [&](const AttnArgs &part, unsigned groups) {
        hipLaunchKernelGGL((attn_dkv_kernel<T, DP, VEC, 1, true>), dim3(groups), b, 0, stream,
                           part);
      });
      if (apart.plan.splits > 1)
        join(a, static_cast<int64_t>(a.n_seq) * a.apart, apart.plan.splits);
    }
  });
}

} // namespace rhip
