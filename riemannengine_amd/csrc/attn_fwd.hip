// Attention over packed sequences on gfx950, forward: softmax(scale q k^T) v
// for every sequence and head by itself, in one pass over the keys with the
// running maximum and sum of the softmax.
#include "attn_device.hpp"
#include "attn.hpp"

namespace rhip {
namespace {

constexpr int kFwdThreads = 256;
constexpr int kFwdRows = 128; // query rows per workgroup, 32 per wave
template <typename T> constexpr int kFwdKeys = sizeof(T) == 2 ? 64 : 32; // keys per LDS tile

// Workgroup -> (tile, head). Workgroups go to the XCDs round-robin; each XCD
// takes a contiguous run of the head-major list, so the tiles that read one
// head's keys share an L2. Within a head the last tiles come first: under a
// causal mask those have the most keys.
__device__ __forceinline__ bool fwd_item(const AttnArgs &a, int32_t &tile, int32_t &head) {
  const uint32_t total = static_cast<uint32_t>(a.tiles) * a.heads;
  const uint32_t per = (total + kXcds - 1) / kXcds;
  const uint32_t i = (blockIdx.x % kXcds) * per + blockIdx.x / kXcds;
  if (i >= total || blockIdx.x / kXcds >= per)
    return false;
  head = i / a.tiles;
  tile = a.tiles - 1 - i % a.tiles;
  return true;
}

// One row by its definition, for rows whose sums came out not finite under a
// causal mask: there a product with a masked key's probability 0 and a value
// that is not finite is not 0. Only keys the row sees are read. All 64 lanes
// of the wave work on the row; lane l returns elements l and l + 64.
template <typename T>
__device__ void exact_row(const T *q, const T *k, int64_t k_row, const T *v, int64_t v_row,
                          int32_t lim, int32_t dim, float c, float &o0, float &o1, float &m,
                          float &sum) {
  const int lane = lane_id();
  auto score = [&](int32_t j) {
    float s = 0.f;
    for (int d = 0; d < dim; ++d)
      s += to_f32(q[d]) * to_f32(k[j * k_row + d]);
    return s;
  };
  m = -INFINITY;
  for (int32_t j = lane; j < lim; j += kWave)
    m = fmaxf(m, score(j));
  for (int off = 32; off; off >>= 1)
    m = fmaxf(m, __shfl_xor(m, off, kWave));
  const float base = (m == -INFINITY ? 0.f : m) * c;
  o0 = o1 = sum = 0.f;
  for (int32_t j0 = 0; j0 < lim; j0 += kWave) {
    const float p = j0 + lane < lim ? exp2_fast(score(j0 + lane) * c - base) : 0.f;
    sum += p;
    const int cnt = min(kWave, lim - j0);
    for (int e = 0; e < cnt; ++e) {
      const float pe = __shfl(p, e, kWave);
      const T *row = v + (j0 + e) * v_row;
      if (lane < dim)
        o0 += pe * to_f32(row[lane]);
      if (lane + kWave < dim)
        o1 += pe * to_f32(row[lane + kWave]);
    }
  }
  for (int off = 32; off; off >>= 1)
    sum += __shfl_xor(sum, off, kWave);
}

// o = softmax(scale q k^T) v and lse for 128 query rows of one head, 32 per
// wave. Scores are S^T = K Q^T (a lane holds 16 keys of one query row's block,
// the other half of the pair l, l + 32 the other 16), so maximum and sum are
// in-lane but for one exchange, and P^T is the right operand of O^T = V^T P^T
// as it lies. K and V tiles go through LDS, double-buffered: the next tile's
// loads are in flight while this one is multiplied.
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(kFwdThreads, 2) void attn_fwd_kernel(AttnArgs a) {
  using Tile = AttnTile<T, DP>;
  using Frag = typename Tile::Frag;
  constexpr int kBN = kFwdKeys<T>, kB = kBN / 32;
  constexpr int kBytes = kBN * Tile::C * 16;
  constexpr int kPer = kBN * Tile::C / kFwdThreads; // chunks per thread of a tile
  __shared__ alignas(16) char lds[2][2][kBytes];

  int32_t t, head;
  if (!fwd_item(a, t, head))
    return;
  const AttnSeq sq = query_tile(a, kFwdRows, 1, t);
  const int32_t row0 = sq.tile * kFwdRows;
  if (row0 >= sq.lq)
    return;
  const int lane = lane_id(), w = threadIdx.x / kWave, half = lane >> 5;
  const int32_t row = row0 + w * 32 + (lane & 31); // this lane's query row
  const bool row_ok = row < sq.lq;
  const int64_t shift = sq.lk - sq.lq; // causal: row i sees keys j <= i + shift
  // keys this lane's row sees, and how far the workgroup's and this wave's go
  auto sees = [&](int64_t r) {
    const int64_t n = a.causal ? min<int64_t>(sq.lk, r + shift + 1) : sq.lk;
    return static_cast<int32_t>(n < 0 ? 0 : n);
  };
  const int32_t lim = row_ok ? sees(row) : 0;
  const int32_t wg_lim = sees(min(row0 + kFwdRows, sq.lq) - 1);
  const int32_t wave_lim = row0 + w * 32 < sq.lq ? sees(min(row0 + w * 32 + 32, sq.lq) - 1) : 0;
  const int32_t wave_full = row0 + w * 32 < sq.lq ? sees(row0 + w * 32) : 0; // seen by all rows
  const int32_t n_tiles = (wg_lim + kBN - 1) / kBN;

  const int kv = head / a.group;
  const T *kp = static_cast<const T *>(a.k) + sq.k0 * a.k_row + kv * a.k_head;
  const T *vp = static_cast<const T *>(a.v) + sq.k0 * a.v_row + kv * a.v_head;

  const T *qp = static_cast<const T *>(a.q) + (sq.q0 + static_cast<int64_t>(row)) * a.q_row +
                head * a.q_head;
  Frag qf[Tile::kSteps];
#pragma unroll
  for (int s = 0; s < Tile::kSteps; ++s)
    qf[s] = __builtin_bit_cast(Frag, Tile::template chunk<VEC>(qp, 2 * s + half, a.dim, row_ok));

  uint4 rk[kPer], rv[kPer];
  auto load_tile = [&](int32_t kt) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int idx = threadIdx.x + i * kFwdThreads, r = idx / Tile::C, c = idx % Tile::C;
      const int32_t j = kt * kBN + r;
      const bool ok = j < sq.lk;
      rk[i] = Tile::template chunk<VEC>(kp + j * a.k_row, c, a.dim, ok);
      rv[i] = Tile::template chunk<VEC>(vp + j * a.v_row, c, a.dim, ok);
    }
  };

  v16f o[Tile::kDBlocks];
#pragma unroll
  for (int db = 0; db < Tile::kDBlocks; ++db)
    o[db] = v16f{};
  float m = -INFINITY, sum = 0.f; // of this lane's row; sum over its half of the keys

  if (n_tiles > 0)
    load_tile(0);
  for (int32_t kt = 0; kt < n_tiles; ++kt) {
    char *lk = lds[kt & 1][0], *lv = lds[kt & 1][1];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int idx = threadIdx.x + i * kFwdThreads, r = idx / Tile::C, c = idx % Tile::C;
      *reinterpret_cast<uint4 *>(Tile::at(lk, r, c)) = rk[i];
      *reinterpret_cast<uint4 *>(Tile::at(lv, r, c)) = rv[i];
    }
    if (kt + 1 < n_tiles)
      load_tile(kt + 1);
    // one barrier per tile: the buffer written next was last read before the
    // barrier of the tile between
    __syncthreads();
    const int32_t j0 = kt * kBN;
    if (j0 >= wave_lim)
      continue;
    v16f s[kB];
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      s[b] = v16f{};
      Tile::row_product(lk, 32 * b, qf, s[b]);
    }
    if (j0 + kBN > wave_full) {
#pragma unroll
      for (int b = 0; b < kB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[b][r] = j0 + 32 * b + block_row(r) < lim ? s[b][r] : -INFINITY;
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
      Tile::col_product(lv, 32 * b, p, o);
    }
  }

  sum = pair_sum(sum);
  float lse = sum == 0.f ? -INFINITY : m * a.scale + logf(sum);
  float inv = sum == 0.f ? 0.f : 1.f / sum;
  T *op = static_cast<T *>(a.o) +
          ((sq.q0 + static_cast<int64_t>(row)) * a.heads + head) * a.dim;
  bool bad = false;
  if (a.causal) {
#pragma unroll
    for (int db = 0; db < Tile::kDBlocks; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        bad |= !isfinite(o[db][r]);
    bad = (bad || !isfinite(sum)) && row_ok;
  }
  uint64_t redo = __ballot(bad);
  redo = (redo | redo >> 32) & 0xffffffffull;
  if (row_ok && !((redo >> (lane & 31)) & 1)) {
    Tile::template store_column<VEC>(op, a.dim, inv, o);
    if (a.lse && half == 0)
      a.lse[static_cast<int64_t>(head) * a.n_q + sq.q0 + row] = lse;
  }
  while (redo) {
    const int i = __ffsll(static_cast<unsigned long long>(redo)) - 1;
    redo &= redo - 1;
    const int64_t r = sq.q0 + static_cast<int64_t>(row0) + w * 32 + i;
    float o0, o1, mr, sr;
    exact_row<T>(static_cast<const T *>(a.q) + r * a.q_row + head * a.q_head, kp, a.k_row, vp,
                 a.v_row, sees(row0 + w * 32 + i), a.dim, a.c, o0, o1, mr, sr);
    T *p = static_cast<T *>(a.o) + (r * a.heads + head) * a.dim;
    const float iv = sr == 0.f ? 0.f : 1.f / sr;
    if (lane < a.dim)
      p[lane] = from_f32<T>(o0 * iv);
    if (lane + kWave < a.dim)
      p[lane + kWave] = from_f32<T>(o1 * iv);
    if (a.lse && lane == 0)
      a.lse[static_cast<int64_t>(head) * a.n_q + r] = mr * a.scale + logf(sr);
  }
}

} // namespace

void attn_forward_run(const AttnArgs &args, int32_t dtype, bool vec, hipStream_t stream) {
  AttnArgs a = args;
  a.tiles = a.n_q / kFwdRows + a.n_seq + 1;
  const int64_t grid = ceil_div(static_cast<int64_t>(a.tiles) * a.heads, kXcds) * kXcds;
  if (grid > INT32_MAX)
    throw Error(RHIP_ERR_UNSUPPORTED, "too many query tiles for one launch");
  with_attn(dtype, a.dim, vec, [&](auto t, auto dp, auto v) {
    using T = decltype(t);
    hipLaunchKernelGGL((attn_fwd_kernel<T, decltype(dp)::value, decltype(v)::value>),
                       dim3(static_cast<unsigned>(grid)), dim3(kFwdThreads), 0, stream, a);
    RHIP_LAUNCH_CHECK();
  });
}

} // namespace rhip
