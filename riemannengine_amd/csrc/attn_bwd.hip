// Attention over packed sequences on gfx950, backward. With p = softmax rows
// (recomputed from lse), dp = do v^T and delta = rowsum(do o):
//   ds = p (dp - delta),  dq = scale ds k,  dk = scale ds^T q,  dv = p^T do.
// Two kernels: one over query rows (dq, and delta for the other), one over
// keys (dk and dv, summed over the query heads of a group inside the
// workgroup). Each gradient row is summed by one wave in a fixed order, so
// results do not change from run to run; the price is that scores and dp are
// computed twice (7 products instead of 5).
#include "attn.hpp"

namespace rhip {
namespace {

constexpr int kBwdThreads = 256;
constexpr int kBwdRows = 128; // query rows (dq) or keys (dk, dv) per workgroup

// Tile size over the other axis. fp32 at full width holds 32-row tiles.
template <typename T> constexpr int kBwdTile = sizeof(T) == 2 ? 64 : 32;

// Workgroup -> (tile, head) as in the forward: head-major runs per XCD.
// `last_first`: the tiles with the most work come first under a causal mask.
__device__ __forceinline__ bool bwd_item(int32_t tiles, int32_t heads, bool last_first,
                                         int32_t &tile, int32_t &head) {
  const uint32_t total = static_cast<uint32_t>(tiles) * heads;
  const uint32_t per = (total + kXcds - 1) / kXcds;
  const uint32_t i = (blockIdx.x % kXcds) * per + blockIdx.x / kXcds;
  if (i >= total || blockIdx.x / kXcds >= per)
    return false;
  head = i / tiles;
  tile = i % tiles;
  if (last_first)
    tile = tiles - 1 - tile;
  return true;
}

// dq of 128 query rows of one head, 32 per wave, over the keys; also delta.
// Blocks are transposed as in the forward (S^T = K Q^T, dP^T = V dO^T), so
// dS^T is the right operand of dQ^T = K^T dS^T as it lies.
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(kBwdThreads, sizeof(T) == 4 && DP == 128 ? 1 : 2) void
attn_dq_kernel(AttnArgs a) {
  using Tile = AttnTile<T, DP>;
  using Frag = typename Tile::Frag;
  constexpr int kBN = kBwdTile<T>, kB = kBN / 32;
  constexpr int kBytes = kBN * Tile::C * 16;
  constexpr int kPer = kBN * Tile::C / kBwdThreads;
  __shared__ alignas(16) char lds[2][2][kBytes];

  int32_t t, head;
  if (!bwd_item(a.tiles, a.heads, true, t, head))
    return;
  const AttnSeq sq = query_tile(a, kBwdRows, 1, t);
  const int32_t row0 = sq.tile * kBwdRows;
  if (row0 >= sq.lq)
    return;
  const int lane = lane_id(), w = threadIdx.x / kWave, half = lane >> 5;
  const int32_t row = row0 + w * 32 + (lane & 31);
  const bool row_ok = row < sq.lq;
  const int64_t shift = sq.lk - sq.lq;
  auto sees = [&](int64_t r) {
    const int64_t n = a.causal ? min<int64_t>(sq.lk, r + shift + 1) : sq.lk;
    return static_cast<int32_t>(n < 0 ? 0 : n);
  };
  const int32_t lim = row_ok ? sees(row) : 0;
  const int32_t wg_lim = sees(min(row0 + kBwdRows, sq.lq) - 1);
  const int32_t wave_lim = row0 + w * 32 < sq.lq ? sees(min(row0 + w * 32 + 32, sq.lq) - 1) : 0;
  const int32_t wave_full = row0 + w * 32 < sq.lq ? sees(row0 + w * 32) : 0;
  const int32_t n_tiles = a.gq ? (wg_lim + kBN - 1) / kBN : 0; // else delta alone

  const int kv = head / a.group;
  const T *kp = static_cast<const T *>(a.k) + sq.k0 * a.k_row + kv * a.k_head;
  const T *vp = static_cast<const T *>(a.v) + sq.k0 * a.v_row + kv * a.v_head;
  const int64_t gr = sq.q0 + static_cast<int64_t>(row);
  const T *qp = static_cast<const T *>(a.q) + gr * a.q_row + head * a.q_head;
  const T *gp = static_cast<const T *>(a.go) + gr * a.go_row + head * a.go_head;
  const T *op = static_cast<const T *>(a.o) + (gr * a.heads + head) * a.dim;

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
  }
  delta = pair_sum(delta);
  const int64_t li = static_cast<int64_t>(head) * a.n_q + gr;
  float lse2 = 0.f; // log2 of the softmax's denominator
  if (row_ok) {
    lse2 = a.lse[li] * kLog2e;
    if (half == 0)
      a.delta[li] = delta;
  }

  uint4 rk[kPer], rv[kPer];
  auto load_tile = [&](int32_t kt) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int idx = threadIdx.x + i * kBwdThreads, r = idx / Tile::C, c = idx % Tile::C;
      const int32_t j = kt * kBN + r;
      const bool ok = j < sq.lk;
      rk[i] = Tile::template chunk<VEC>(kp + j * a.k_row, c, a.dim, ok);
      rv[i] = Tile::template chunk<VEC>(vp + j * a.v_row, c, a.dim, ok);
    }
  };
  v16f dq[Tile::kDBlocks];
#pragma unroll
  for (int db = 0; db < Tile::kDBlocks; ++db)
    dq[db] = v16f{};

  if (n_tiles > 0)
    load_tile(0);
  for (int32_t kt = 0; kt < n_tiles; ++kt) {
    char *lk = lds[kt & 1][0], *lv = lds[kt & 1][1];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int idx = threadIdx.x + i * kBwdThreads, r = idx / Tile::C, c = idx % Tile::C;
      *reinterpret_cast<uint4 *>(Tile::at(lk, r, c)) = rk[i];
      *reinterpret_cast<uint4 *>(Tile::at(lv, r, c)) = rv[i];
    }
    if (kt + 1 < n_tiles)
      load_tile(kt + 1);
    __syncthreads(); // one per tile, as in the forward
    const int32_t j0 = kt * kBN;
    if (j0 >= wave_lim)
      continue;
    const bool masked = j0 + kBN > wave_full;
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      v16f s{}, dp{};
      Tile::row_product(lk, 32 * b, qf, s);
      Tile::row_product(lv, 32 * b, gf, dp);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[r] = exp2_fast(fmaf(s[r], a.c, -lse2)) * (dp[r] - delta);
      if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[r] = j0 + 32 * b + block_row(r) < lim ? s[r] : 0.f;
      }
      typename Tile::Block ds;
      Tile::pack(s, ds);
      Tile::col_product(lk, 32 * b, ds, dq);
    }
  }
  if (row_ok && a.gq)
    Tile::template store_column<VEC>(
        static_cast<T *>(a.gq) + (gr * a.heads + head) * a.dim, a.dim, a.scale, dq);
}

// dk and dv of 128 keys of one key head, 32 per wave, over the query rows of
// every head of its group. A lane holds one key's column (S = Q K^T, dP = dO
// V^T), so P and dS are the right operands of dV^T = dO^T P and dK^T = Q^T dS
// as they lie.
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(kBwdThreads, DP == 128 ? 1 : 2) void
attn_dkv_kernel(AttnArgs a) {
  using Tile = AttnTile<T, DP>;
  using Frag = typename Tile::Frag;
  constexpr int kBM = kBwdTile<T>, kB = kBM / 32;
  constexpr int kBytes = kBM * Tile::C * 16;
  constexpr int kPer = kBM * Tile::C / kBwdThreads;
  __shared__ alignas(16) char lds[2][2][kBytes];
  __shared__ alignas(16) float rows[2][2][kBM]; // lse2 and delta of the tile's rows

  int32_t t, kv;
  if (!bwd_item(a.tiles, a.kv_heads, false, t, kv))
    return;
  int32_t room;
  const AttnSeq sq = key_tile(a, kBwdRows, t, room);
  const int32_t key0 = sq.tile * kBwdRows;
  if (key0 >= room)
    return;
  const int lane = lane_id(), w = threadIdx.x / kWave, half = lane >> 5;
  const int32_t key = key0 + w * 32 + (lane & 31);
  const bool key_ok = key < sq.lk;
  const int64_t shift = sq.lk - sq.lq;
  // the first row that sees a key
  auto first_row = [&](int64_t j) {
    const int64_t i = a.causal ? j - shift : 0;
    return static_cast<int32_t>(i < 0 ? 0 : (i > sq.lq ? sq.lq : i));
  };
  const int32_t lo = first_row(key);
  const int32_t wave_lo = first_row(key0 + w * 32);         // no earlier row sees any
  const int32_t wave_full = first_row(key0 + w * 32 + 31);  // every later row sees all
  const int32_t it0 = first_row(key0) / kBM;
  // tiles of query rows from the first that sees a key, for each head
  const int32_t per_head = key0 < sq.lk ? max((sq.lq + kBM - 1) / kBM - it0, 0) : 0;
  const int32_t n_tiles = per_head * a.group;

  const int64_t gk = sq.k0 + static_cast<int64_t>(key);
  const T *kp = static_cast<const T *>(a.k) + gk * a.k_row + kv * a.k_head;
  const T *vp = static_cast<const T *>(a.v) + gk * a.v_row + kv * a.v_head;
  Frag kf[Tile::kSteps], vf[Tile::kSteps];
#pragma unroll
  for (int s = 0; s < Tile::kSteps; ++s) {
    const int c = 2 * s + half;
    kf[s] = __builtin_bit_cast(Frag, Tile::template chunk<VEC>(kp, c, a.dim, key_ok));
    vf[s] = __builtin_bit_cast(Frag, Tile::template chunk<VEC>(vp, c, a.dim, key_ok));
  }

  uint4 rq[kPer], rg[kPer];
  float rs = 0.f;
  auto load_tile = [&](int32_t n) {
    const int head = kv * a.group + n / per_head;
    const int32_t i0 = (it0 + n % per_head) * kBM;
    const T *qp = static_cast<const T *>(a.q) + sq.q0 * a.q_row + head * a.q_head;
    const T *gp = static_cast<const T *>(a.go) + sq.q0 * a.go_row + head * a.go_head;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int idx = threadIdx.x + i * kBwdThreads, r = idx / Tile::C, c = idx % Tile::C;
      const int32_t qi = i0 + r;
      rq[i] = Tile::template chunk<VEC>(qp + qi * a.q_row, c, a.dim, qi < sq.lq);
      rg[i] = Tile::template chunk<VEC>(gp + qi * a.go_row, c, a.dim, qi < sq.lq);
    }
    if (threadIdx.x < 2 * kBM) {
      const int r = threadIdx.x % kBM;
      const float *src = threadIdx.x < kBM ? a.lse : a.delta;
      rs = i0 + r < sq.lq ? src[static_cast<int64_t>(head) * a.n_q + sq.q0 + i0 + r] : 0.f;
      if (threadIdx.x < kBM)
        rs *= kLog2e;
    }
  };

  v16f dk[Tile::kDBlocks], dv[Tile::kDBlocks];
#pragma unroll
  for (int db = 0; db < Tile::kDBlocks; ++db)
    dk[db] = dv[db] = v16f{};

  if (n_tiles > 0)
    load_tile(0);
  for (int32_t n = 0; n < n_tiles; ++n) {
    char *lq = lds[n & 1][0], *lg = lds[n & 1][1];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int idx = threadIdx.x + i * kBwdThreads, r = idx / Tile::C, c = idx % Tile::C;
      *reinterpret_cast<uint4 *>(Tile::at(lq, r, c)) = rq[i];
      *reinterpret_cast<uint4 *>(Tile::at(lg, r, c)) = rg[i];
    }
    if (threadIdx.x < 2 * kBM)
      rows[n & 1][threadIdx.x / kBM][threadIdx.x % kBM] = rs;
    if (n + 1 < n_tiles)
      load_tile(n + 1);
    __syncthreads();
    const int32_t i0 = (it0 + n % per_head) * kBM;
    if (i0 + kBM <= wave_lo)
      continue;
    const bool masked = i0 < wave_full || i0 + kBM > sq.lq;
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      v16f s{}, dp{};
      Tile::row_product(lq, 32 * b, kf, s);
      Tile::row_product(lg, 32 * b, vf, dp);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int r = 32 * b + 8 * g + 4 * half;
        const v4f l = *reinterpret_cast<const v4f *>(&rows[n & 1][0][r]);
        const v4f d = *reinterpret_cast<const v4f *>(&rows[n & 1][1][r]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[4 * g + e] = exp2_fast(fmaf(s[4 * g + e], a.c, -l[e]));
          if (masked) {
            const int32_t i = i0 + r + e;
            s[4 * g + e] = i >= lo && i < sq.lq ? s[4 * g + e] : 0.f;
            dp[4 * g + e] = i >= lo && i < sq.lq ? dp[4 * g + e] : d[e];
          }
          dp[4 * g + e] = s[4 * g + e] * (dp[4 * g + e] - d[e]);
        }
      }
      typename Tile::Block p, ds;
      Tile::pack(s, p);
      Tile::col_product(lg, 32 * b, p, dv);
      Tile::pack(dp, ds);
      Tile::col_product(lq, 32 * b, ds, dk);
    }
  }
  if (key < room) { // rows behind the keys in use get zeros
    const int64_t at = (gk * a.kv_heads + kv) * a.dim;
    Tile::template store_column<VEC>(static_cast<T *>(a.gk) + at, a.dim, a.scale, dk);
    Tile::template store_column<VEC>(static_cast<T *>(a.gv) + at, a.dim, 1.f, dv);
  }
}

unsigned bwd_grid(int64_t tiles, int64_t heads) {
  const int64_t grid = ceil_div(tiles * heads, kXcds) * kXcds;
  if (grid > INT32_MAX)
    throw Error(RHIP_ERR_UNSUPPORTED, "too many tiles for one launch");
  return static_cast<unsigned>(grid);
}

} // namespace

void attn_backward_run(const AttnArgs &args, int32_t dtype, bool vec, hipStream_t stream) {
  AttnArgs aq = args, ak = args;
  aq.tiles = args.n_q / kBwdRows + args.n_seq + 1;
  ak.tiles = args.n_k / kBwdRows + args.n_seq + 1;
  const unsigned gq = bwd_grid(aq.tiles, args.heads), gk = bwd_grid(ak.tiles, args.kv_heads);
  with_attn(dtype, args.dim, vec, [&](auto t, auto dp, auto v) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    constexpr bool VEC = decltype(v)::value;
    hipLaunchKernelGGL((attn_dq_kernel<T, DP, VEC>), dim3(gq), dim3(kBwdThreads), 0, stream, aq);
    RHIP_LAUNCH_CHECK();
    if (!args.gk)
      return;
    hipLaunchKernelGGL((attn_dkv_kernel<T, DP, VEC>), dim3(gk), dim3(kBwdThreads), 0, stream, ak);
    RHIP_LAUNCH_CHECK();
  });
}

} // namespace rhip
