// Attention over packed sequences on gfx950, forward: softmax(scale q k^T) v
// for every sequence and head by itself, in one pass over the keys with the
// running maximum and sum of the softmax.
//
// The heads of a group are packed: row r of a key head's sequence is query
// row r / group, head r % group, so all rows that read the same keys stand in
// the same tiles. A workgroup's four waves hold W blocks of 32 rows:
//   W = 4  each wave has a block; all read the same LDS tiles of keys;
//   W = 2  two waves share a block, each with half of every tile's keys;
//   W = 1  all share one, each with every fourth tile of 32 keys, through LDS
//          tiles of its own (no barrier until the end).
// Waves that share rows join their sums in LDS at the end. With W = 1 the
// keys may further be split over workgroups, joined by a second kernel: for
// single tokens, and wherever larger tiles leave the chip empty.
#include <cmath>

#include "attn.hpp"

namespace rhip {
namespace {

constexpr int kFwdThreads = 256;
constexpr int kFwdWaves = kFwdThreads / kWave;
constexpr int kMinSplitKeys = 128; // a tile for each wave of every split

template <typename T, int DP, int W> struct FwdShape {
  static constexpr int kRows = 32 * W;
  static constexpr int kParts = kFwdWaves / W; // waves that share a block of rows
  // Keys per LDS tile: two 32-key blocks where they fit, four of narrow heads
  // in bf16 (32 wide, four sequences of 2048, 8 heads: 53 us in two, 49 in four).
  static constexpr int kBN = W == 1 || (W == 4 && sizeof(T) == 4 && DP == 128) ? 32
                             : sizeof(T) == 2 && DP == 32                       ? 128
                                                                                : 64;
  static constexpr int kStreams = W == 1 ? kFwdWaves : 1;
  static constexpr int kTileBytes = kBN * DP * sizeof(T);
  // Registers let two workgroups into a CU.
  static constexpr bool kSlim = sizeof(T) == 2 || DP <= 64;
  // Two buffers where they fit; in fp32 up to 64 wide only where they leave LDS
  // for a second workgroup, which covers the first one's waits better (6 over 2
  // heads, three causal sequences of 1100: two buffers and one workgroup 72 us, one
  // buffer and two workgroups 57). bf16's W = 1 serves single tokens too, whose
  // stream of keys is better held by two buffers (32 over caches of 1 to 16384, 8
  // key heads, 128 wide: 156 us, and 172 with two workgroups); other launches of
  // few rows pay for that (16 rows a sequence over 3000 keys: 50 us, and 37).
  static constexpr int kBuffers =
      kStreams * 4 * kTileBytes <= (sizeof(T) == 4 && DP <= 64 ? 80 : 160) * 1024 ? 2 : 1;
  static constexpr int kJoinRow = DP + 4; // floats per row of the joined results
  static constexpr int kJoinBytes =
      W < 4 ? kFwdWaves * 32 * (kJoinRow + 2) * static_cast<int>(sizeof(float)) : 0;
  static constexpr int kStageBytes = kStreams * kBuffers * 2 * kTileBytes;
  static constexpr int kLds = kStageBytes > kJoinBytes ? kStageBytes : kJoinBytes;
  // waves per SIMD: two workgroups' where their LDS and registers fit
  static constexpr int kOccupancy = kSlim && kLds <= 80 * 1024 ? 2 : 1;
};

// A row's result from one wave: lane l holds elements l and l + 64 of the
// unnormalised sum.
template <typename T>
__device__ void finish_row(const AttnArgs &a, int64_t row, int32_t head, float o0, float o1,
                           float m, float sum) {
  const int lane = lane_id();
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t at = (row * a.heads + head) * a.dim;
  auto put = [&](int d, float v) {
    if (d < a.dim) {
      const T t = from_f32<T>(v * inv);
      static_cast<T *>(a.o)[at + d] = t;
      if (sizeof(T) == 2 && a.rest)
        static_cast<T *>(a.rest)[at + d] = from_f32<T>(v * inv - to_f32(t));
    }
  };
  put(lane, o0);
  put(lane + kWave, o1);
  if (a.lse && lane == 0)
    a.lse[static_cast<int64_t>(head) * a.n_q + row] =
        sum == 0.f ? -INFINITY : m * a.scale + logf(sum);
}

// Scores are S^T = K Q^T (a lane holds 16 keys of one query row's block, the
// other half of the pair l, l + 32 the other 16), so maximum and sum are
// in-lane but for one exchange, and P^T is the right operand of O^T = V^T P^T
// as it lies. The next tile's loads are in flight while this one is
// multiplied.
//
// Bounds: the matrix cores at width 128 (four causal prompts of 4096, 16 over 4
// heads, bf16: 327 us, 840 TFLOP/s; the cores busy for 38% of the cycles, the
// softmax's vector instructions beside them); the vector instructions at 32 and
// 64 (630 and 900: a score costs one exponential whatever the width); memory
// for single tokens (32 over caches of 1 to 16384, 8 key heads of 128: 4.7 TB/s).
// Taken back as no faster: the next tile's scores computed beside this one's
// softmax, row sums as a product with ones, priorities of waves.
template <typename T, int DP, bool VEC, int W>
__global__ __launch_bounds__(kFwdThreads, (FwdShape<T, DP, W>::kOccupancy)) void
attn_fwd_kernel(AttnArgs a) {
  using Shape = FwdShape<T, DP, W>;
  using Tile = AttnTile<T, DP>;
  using Frag = typename Tile::Frag;
  constexpr int kBN = Shape::kBN;
  constexpr int kAhead = sizeof(T) == 2 ? 4 : 0; // LDS operands on their way to the products
  constexpr int kB = kBN / 32 / (W == 2 ? 2 : 1); // blocks of a tile that are a wave's
  using Stream = TileStream<T, DP, kBN, W == 1 ? kWave : kFwdThreads, VEC>;
  __shared__ alignas(16) char lds[Shape::kLds];
  __shared__ int any_left_out; // of the workgroup

  int32_t t, kv, split;
  if (!attn_item(a, t, kv, split))
    return;
  t = a.tiles - 1 - t; // the last tiles first: under a causal mask they see the most keys
  const AttnSeq sq = query_tile(a, Shape::kRows, a.group, t);
  const int32_t n_rows = sq.lq * a.group, row0 = sq.tile * Shape::kRows;
  if (row0 >= n_rows)
    return;
  const int lane = lane_id(), half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int32_t wave0 = row0 + w / Shape::kParts * 32;
  const int b0 = W == 2 ? w % 2 * kB : 0; // the wave's first block of a tile
  const int32_t row = wave0 + (lane & 31); // this lane's packed row
  const bool row_ok = row < n_rows;
  const int32_t rc = min(row, n_rows - 1);
  const int32_t qi = rc / a.group;
  const int head = kv * a.group + rc % a.group;
  const int64_t shift = static_cast<int64_t>(sq.lk) - sq.lq;
  // keys a packed row sees (causal: query row i sees keys j <= i + shift)
  auto sees = [&](int32_t r) {
    const int64_t n = a.causal ? min<int64_t>(sq.lk, r / a.group + shift + 1) : sq.lk;
    return static_cast<int32_t>(n < 0 ? 0 : n);
  };
  const int32_t lim = row_ok ? sees(row) : 0;
  const int32_t wg_lim = wave_uniform(sees(min(row0 + Shape::kRows, n_rows) - 1));
  const int32_t wg_full = wave_uniform(sees(row0)); // seen by all its rows
  const int32_t wave_lim =
      wave_uniform(wave0 < n_rows ? sees(min(wave0 + 32, n_rows) - 1) : 0);
  const int32_t wave_full = wave_uniform(wave0 < n_rows ? sees(wave0) : 0);
  // this workgroup's tiles [kt0, kt1) of keys; a wave's first and step
  int32_t kt0 = 0, kt1 = (wg_lim + kBN - 1) / kBN;
  if (W == 1 && a.splits > 1) {
    const int32_t per = (kt1 + a.splits - 1) / a.splits;
    kt0 = min(split * per, kt1);
    kt1 = min(kt0 + per, kt1);
  }
  const int32_t first = kt0 + (W == 1 ? w : 0), step = W == 1 ? kFwdWaves : 1;

  const T *kp = static_cast<const T *>(a.k) + sq.k0 * a.k_row + kv * a.k_head;
  const T *vp = static_cast<const T *>(a.v) + sq.k0 * a.v_row + kv * a.v_head;
  Stream ks, vs;
  ks.init(a.k_row, a.dim);
  vs.init(a.v_row, a.dim);
  char *stage = lds + (W == 1 ? w : 0) * Shape::kBuffers * 2 * Shape::kTileBytes;
  auto issue = [&](int32_t kt, int buf) {
    char *to = stage + buf * 2 * Shape::kTileBytes;
    ks.issue(to, kp + static_cast<int64_t>(kt) * kBN * a.k_row, a.k_row, sq.lk - kt * kBN,
             a.dim);
    vs.issue(to + Shape::kTileBytes, vp + static_cast<int64_t>(kt) * kBN * a.v_row, a.v_row,
             sq.lk - kt * kBN, a.dim);
  };
  if (first < kt1)
    issue(first, 0);

  const T *qp = static_cast<const T *>(a.q) + (sq.q0 + static_cast<int64_t>(qi)) * a.q_row +
                head * a.q_head;
  Frag qf[Tile::kSteps];
#pragma unroll
  for (int s = 0; s < Tile::kSteps; ++s)
    qf[s] = __builtin_bit_cast(Frag, Tile::template chunk<VEC>(qp, 2 * s + half, a.dim, row_ok));

  v16f o[Tile::kDBlocks];
#pragma unroll
  for (int db = 0; db < Tile::kDBlocks; ++db)
    o[db] = v16f{};
  float m = -INFINITY, sum = 0.f; // of this lane's row; sum over its half of the keys
  // Values that are not finite, in tiles of which some rows see a part: a masked
  // entry's zero times one would be NaN, so they are zeroed in LDS, and the rows
  // that see them get them at the end.
  bool left_out = false;
  if (W > 1 && threadIdx.x == 0)
    any_left_out = 0; // behind the barrier of the first turn

  const typename Tile::Lane lane_at = Tile::lane_addresses();
  const uint32_t stage_at = lds_address(stage);
  int buf = 0;
  for (int32_t kt = first; kt < kt1; kt += step) {
    // this tile has landed; then every wave is past its reads of the other
    // buffer, which the next tile's loads overwrite
    wait_stream();
    if constexpr (W > 1)
      __syncthreads();
    if (wg_full < wg_lim && (kt + 1) * kBN > wg_full) {
      rare_path();
      const bool found = Tile::template zero_not_finite<false, kBN, W == 1 ? 1 : kFwdWaves>(
          stage_at + buf * 2 * Shape::kTileBytes + Shape::kTileBytes, W == 1 ? 0 : w);
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
        lane_at.in(stage_at + buf * 2 * Shape::kTileBytes + b0 * (32 / 4) * Tile::kGroup);
    if (Shape::kBuffers == 2 && kt + step < kt1)
      issue(kt + step, buf ^ 1);
    const int32_t j0 = kt * kBN + 32 * b0;
    if (W == 1 || j0 < wave_lim) {
      v16f s[kB];
#pragma unroll
      for (int b = 0; b < kB; ++b)
        s[b] = v16f{};
      // the blocks take turns: two sums to add to
      ahead<kB * Tile::kSteps, kAhead>(
          [&](int i) { return Tile::row_operand(at, 0, 32 * (i % kB), i / kB); },
          [&](int i, const Frag &x) { Tile::mma(x, qf[i / kB], s[i % kB]); });
      if (j0 + 32 * kB > wave_full) {
        rare_path();
#pragma unroll
        for (int b = 0; b < kB; ++b) {
          const int32_t seen = lim - j0 - 32 * b - 4 * half; // of the lane's rows of the block
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[b][r] = block_row(r) < seen ? s[b][r] : -INFINITY;
        }
      }
      float top = m;
#pragma unroll
      for (int b = 0; b < kB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          top = fmaxf(top, s[b][r]);
      top = pair_max(top);
      const float base = (top == -INFINITY ? 0.f : top) * a.c;
      if (__any(top > m)) { // otherwise every factor is 1
        const float f = exp2_fast(m * a.c - base);
        sum *= f;
#pragma unroll
        for (int db = 0; db < Tile::kDBlocks; ++db)
          o[db] *= f;
        m = top;
      }
#pragma unroll
      for (int b = 0; b < kB; ++b) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[b][r] = exp2_fast(fmaf(s[b][r], a.c, -base));
          sum += s[b][r];
        }
        typename Tile::Block p;
        Tile::pack(s[b], p);
        Tile::col_product(at, Shape::kTileBytes, 32 * b, p, o);
      }
    }
    if (Shape::kBuffers == 2) {
      buf ^= 1;
    } else if (kt + step < kt1) {
      wait_stream();
      if constexpr (W > 1)
        __syncthreads();
      issue(kt + step, 0);
    }
  }
  sum = pair_sum(sum);
  if (left_out)
    Tile::template add_not_finite<false>(vp, a.v_row, a.dim, max(wg_full - kBN, 0), wave_lim,
                                         [&](int32_t j) { return j < lim; }, o);

  if constexpr (W == 4) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t place = (sq.q0 + static_cast<int64_t>(qi)) * a.heads + head;
    if (row_ok) {
      Tile::template store_column<VEC>(static_cast<T *>(a.o) + place * a.dim, a.dim, inv, o);
      if (sizeof(T) == 2 && a.rest)
        Tile::template store_rest<VEC>(static_cast<T *>(a.rest) + place * a.dim, a.dim, inv, o);
      if (a.lse && half == 0)
        a.lse[static_cast<int64_t>(head) * a.n_q + sq.q0 + qi] =
            sum == 0.f ? -INFINITY : m * a.scale + logf(sum);
    }
  } else {
    // join the waves: [wave][row][DP] sums, then each row's maximum and sum
    __syncthreads(); // every wave is past its tiles
    float *jo = reinterpret_cast<float *>(lds);
    float *jm = jo + kFwdWaves * 32 * Shape::kJoinRow;
    float *mine = jo + (w * 32 + (lane & 31)) * Shape::kJoinRow;
#pragma unroll
    for (int db = 0; db < Tile::kDBlocks; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<v4f *>(mine + 32 * db + 8 * g + 4 * half) =
            v4f{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
    if (half == 0) {
      jm[(w * 32 + lane) * 2] = m;
      jm[(w * 32 + lane) * 2 + 1] = sum;
    }
    __syncthreads();
    for (int r = w; r < Shape::kRows && row0 + r < n_rows; r += kFwdWaves) {
      // the row in the first of its waves' results
      const int first_at = r / 32 * Shape::kParts * 32 + r % 32;
      float mr = -INFINITY;
#pragma unroll
      for (int i = 0; i < Shape::kParts; ++i)
        mr = fmaxf(mr, jm[(i * 32 + first_at) * 2]);
      const float base = (mr == -INFINITY ? 0.f : mr) * a.c;
      float o0 = 0.f, o1 = 0.f, sr = 0.f;
#pragma unroll
      for (int i = 0; i < Shape::kParts; ++i) {
        const float f = exp2_fast(jm[(i * 32 + first_at) * 2] * a.c - base);
        sr = fmaf(jm[(i * 32 + first_at) * 2 + 1], f, sr);
        const float *src = jo + (i * 32 + first_at) * Shape::kJoinRow;
        if (lane < DP)
          o0 = fmaf(src[lane], f, o0);
        if (lane + kWave < DP)
          o1 = fmaf(src[lane + kWave], f, o1);
      }
      const int32_t i = (row0 + r) / a.group;
      const int h = kv * a.group + (row0 + r) % a.group;
      if (a.splits == 1) {
        finish_row<T>(a, sq.q0 + static_cast<int64_t>(i), h, o0, o1, mr, sr);
      } else {
        const int64_t place = split * static_cast<int64_t>(a.n_q) * a.heads +
                           (sq.q0 + static_cast<int64_t>(i)) * a.heads + h;
        if (lane < a.dim)
          a.part_o[place * a.dim + lane] = o0;
        if (lane + kWave < a.dim)
          a.part_o[place * a.dim + lane + kWave] = o1;
        if (lane == 0) {
          a.part_ml[2 * place] = mr;
          a.part_ml[2 * place + 1] = sr;
        }
      }
    }
  }
}

// Joins the splits' partial sums, a workgroup per row and head: each wave
// weighs every fourth split (its loads all independent), the sums are added in
// wave order.
template <typename T>
__global__ __launch_bounds__(kFwdThreads) void attn_join_kernel(AttnArgs a) {
  __shared__ float2 sums[kFwdWaves][kWave];
  __shared__ float totals[kFwdWaves];
  const int64_t rows = static_cast<int64_t>(a.n_q) * a.heads, at = blockIdx.x;
  const int lane = lane_id(), w = threadIdx.x / kWave;
  const int32_t row = static_cast<int32_t>(at / a.heads), head = static_cast<int32_t>(at % a.heads);
  // lane s: split s (at most 64 of them)
  const bool mine = lane < a.splits;
  const float m = mine ? a.part_ml[2 * (lane * rows + at)] : -INFINITY;
  const float l = mine ? a.part_ml[2 * (lane * rows + at) + 1] : 0.f;
  float mr = m;
#pragma unroll
  for (int off = 32; off; off >>= 1)
    mr = fmaxf(mr, __shfl_xor(mr, off, kWave));
  const float base = (mr == -INFINITY ? 0.f : mr) * a.c;
  const float f = mine ? exp2_fast(m * a.c - base) : 0.f;
  float o0 = 0.f, o1 = 0.f, sr = 0.f;
#pragma unroll 4
  for (int s = w; s < a.splits; s += kFwdWaves) {
    const float fs = __shfl(f, s, kWave);
    const float *src = a.part_o + (s * rows + at) * a.dim;
    sr = fmaf(__shfl(l, s, kWave), fs, sr);
    o0 = fmaf(lane < a.dim ? src[lane] : 0.f, fs, o0);
    o1 = fmaf(lane + kWave < a.dim ? src[lane + kWave] : 0.f, fs, o1);
  }
  sums[w][lane] = make_float2(o0, o1);
  if (lane == 0)
    totals[w] = sr;
  __syncthreads();
  if (w > 0)
    return;
#pragma unroll
  for (int i = 1; i < kFwdWaves; ++i) {
    o0 += sums[i][lane].x;
    o1 += sums[i][lane].y;
    sr += totals[i];
  }
  finish_row<T>(a, row, head, o0, o1, mr, sr);
}

// W by attn_waves; with W = 1 the splits by estimated time, in microseconds: a
// round of workgroups (two per CU with narrow rows, one with wide) takes 8 to start
// and finish and `tile` for every four 32-key tiles (one to a wave) of the mean
// sequence; no less than the longest sequence alone, taken as 1.5 times the
// mean, or 3 times for single tokens, whose caches differ most; joining takes
// another 8. (32 tokens over caches of 1 to 16384 keys, 8 key heads, 128 wide:
// four splits 172 us, one 390. Three causal sequences of 1000, 2 heads of 96:
// one split 26 us, three 32 and 7 to join.)
AttnPlan plan_forward(int64_t n_q, int64_t n_k, int32_t n_seq, int32_t heads, int32_t kv_heads,
                      int32_t dim, int32_t causal, int32_t dtype) {
  const int64_t rows = n_q * (heads / kv_heads);
  AttnPlan p{attn_waves(rows, kv_heads, dtype), 0, 1};
  p.tiles = rows / (32 * p.waves) + n_seq + 1;
  if (p.waves > 1 || n_seq == 0)
    return p;
  const bool f32 = dtype == RHIP_F32;
  const double width = dim <= 32 ? 0.25 : dim <= 64 ? 0.5 : dim <= 96 ? 0.75 : 1.0;
  const double tile = std::max(1.2, (f32 ? 5.0 : 3.0) * width);
  // workgroups with rows: a tile of every 32 rows, and one per sequence
  const double busy = static_cast<double>(rows / 32 + std::min<int64_t>(n_seq, rows)) * kv_heads;
  const bool tokens = rows <= 32 * static_cast<int64_t>(n_seq);
  const double slots = width * (f32 ? 2 : 1) <= 0.5 ? 512.0 : 256.0;
  const double tiles =
      static_cast<double>(n_k) / n_seq / (32 * kFwdWaves) * (causal && !tokens ? 0.5 : 1.0);
  double least = 0.0;
  for (int32_t s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
    if (s > 1 && n_k / n_seq < static_cast<int64_t>(kMinSplitKeys) * s)
      break;
    const double turn = std::ceil(tiles / s) * tile;
    const double all = std::ceil(busy * s / slots) * (8.0 + turn);
    const double longest = 8.0 + turn * (tokens ? 3.0 : 1.5);
    const double t = std::max(all, longest) + (s > 1 ? 8.0 : 0.0);
    if (s == 1 || t < least) {
      least = t;
      p.splits = s;
    }
  }
  return p;
}

} // namespace

AttnPlan attn_forward_plan(const rhip_attn &d) {
  return plan_forward(d.n_q, d.n_k, d.n_seq, d.heads, d.kv_heads, d.dim, d.causal, d.dtype);
}

void attn_forward_run(const AttnArgs &args, int32_t dtype, bool vec, hipStream_t stream) {
  AttnArgs a = args;
  const AttnPlan plan = plan_forward(a.n_q, a.n_k, a.n_seq, a.heads, a.kv_heads, a.dim,
                                     a.causal, dtype);
  const int64_t rows = static_cast<int64_t>(a.n_q) * a.heads;
  a.splits = plan.splits;
  with_attn(dtype, a.dim, vec, [&](auto t, auto dp, auto v) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    constexpr bool VEC = decltype(v)::value;
    const dim3 b(kFwdThreads);
    with_waves(plan.waves, [&](auto w) {
      constexpr int W = decltype(w)::value;
      const unsigned spread = spread_lds<W>(a, FwdShape<T, DP, W>::kLds);
      attn_launches(a, plan, kFwdThreads, [&](const AttnArgs &part, unsigned groups) {
        hipLaunchKernelGGL((attn_fwd_kernel<T, DP, VEC, W>), dim3(groups), b, spread, stream,
                           part);
      });
    });
    if (a.splits > 1) { // with W = 1, so rows for a few hundred workgroups at most
      hipLaunchKernelGGL((attn_join_kernel<T>),
                         dim3(static_cast<unsigned>(rows)), b, 0, stream, a);
      RHIP_LAUNCH_CHECK();
    }
  });
}

} // namespace rhip
