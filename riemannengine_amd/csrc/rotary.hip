// Rotation of the heads of queries and keys by positions of several axes on
// gfx950, with the heads' RMS norm before it, forward and backward. A head of
// D elements has P pairs (a, b), elements (p, P + p) or (2 p, 2 p + 1), each
// turned by angle t = position[axis of p] * frequency[p]:
//   (a cos t - b sin t, a sin t + b cos t);
// elements 2 P .. D - 1 stay. With the norm, z = x r w is turned, r = 1 /
// sqrt(mean x^2 + eps). Backward: d = grad_y turned back,
//   grad_w = sum over rows and heads of d x r,
//   grad_x = r (d w - x r^2 mean(d w x)).
//
// A workgroup takes a tile of rows: it makes their cosines and sines in LDS,
// once for all heads of queries and keys, and its groups of G lanes then go
// through the (row, head) pairs, each lane with two chunks of 16 bytes that
// hold its pairs. A head's values stay in registers between its norm and its
// rotation, so x (and grad_y) are read once and y (grad_x) is written once.
// Angles are products of fp64, reduced to a part of a turn by 1 / (2 pi) in two
// fp64 parts: up to 2^53 radians the reduction is off by less than 2^-50 turns, so
// a far angle is as exact as its product (half an fp64 step of it).
//
// Bound by memory: 16384 rows of 32 + 8 heads of 128, bf16, with the norm: 71 us
// forward (4.7 TB/s), 96 backward (5.2) and 6 for the weights' sums; by the angles
// beside it for narrow heads (100003 rows of 8 heads of 32: 28 and 30 us, 3.6
// TB/s). 32 rows: one launch, 6 us.
#include <climits>
#include <type_traits>

#include "row_chunk.hpp"

namespace rhip {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotMaxDim = 256;
constexpr int kRotTable = 512;   // pairs of a tile's table (4 KB)
constexpr int kRotMaxRows = 256; // rows of a tile
// Backward workgroups that sum the weights' gradients, three to a CU; each writes a
// row of sums (16384 rows of 40 heads of 128: 96 us, with 1024 or 512 of them
// a sixth more).
constexpr int kRotBlocks = 768;

struct RotHeads {
  const void *x, *gy;
  int64_t x_row, x_head, gy_row, gy_head;
  const float *weight;
  void *y; // forward: y, backward: grad_x; dense
  int32_t heads;
  uint32_t inverse; // of heads, 2^32 / heads rounded up; 0: too many heads for it
};

struct RotArgs {
  RotHeads t[2];
  const void *positions;
  const double *frequencies;
  int64_t position_row;
  int32_t position_type;
  int32_t axes, ends[RHIP_ROTARY_MAX_AXES]; // pairs of the axes up to and with this one
  int32_t n, dim, pairs, turning, passing;   // lanes of a group with pairs that turn, that stay
  int32_t rows, tiles;                       // rows of a tile; tiles
  int32_t interleaved;
  float eps;
  float *part; // backward: [workgroups][2][dim] sums of the weights' gradients
};

// What a lane of a group holds of a head: two chunks of V elements, from a and
// b on, of which the first na and nb lie within its part of the head. A last,
// partial chunk starts earlier, so that it is whole: its first skip_a and
// skip_b elements are another lane's too and count there. pair: its first pair
// in the tile's table, below 0 where nothing turns.
struct RotLane {
  int32_t a, b, na, nb, skip_a, skip_b, pair;
};

template <int V> __device__ __forceinline__ RotLane rot_lane(const RotArgs &p, int lane) {
  RotLane l{0, 0, 0, 0, 0, 0, -1};
  const bool turns = lane < p.turning;
  if (!turns && lane >= p.turning + p.passing)
    return l;
  if (turns) {
    const int want = lane * V, first = max(0, min(want, p.pairs - V));
    const int count = min(V, p.pairs - first), skip = want - first;
    l.pair = lane * V;
    if (p.interleaved) {
      l.a = 2 * first, l.b = 2 * first + V;
      l.na = min(V, 2 * count), l.nb = max(0, 2 * count - V);
      l.skip_a = min(V, 2 * skip), l.skip_b = max(0, 2 * skip - V);
    } else {
      l.a = first, l.b = p.pairs + first;
      l.na = l.nb = count;
      l.skip_a = l.skip_b = skip;
    }
  } else {
    const int from = 2 * p.pairs, want = from + (lane - p.turning) * 2 * V;
    const int first = max(from, min(want, p.dim - 2 * V));
    const int count = min(2 * V, p.dim - first), skip = want - first;
    l.a = first, l.b = first + V;
    l.na = min(V, count), l.nb = max(0, count - V);
    l.skip_a = min(V, skip), l.skip_b = max(0, skip - V);
  }
  return l;
}

// The table's pair at `slot` of a row: lane slot / V's (slot % V)-th pair.
template <int V> __device__ __forceinline__ int rot_pair(const RotArgs &p, int slot) {
  const int first = max(0, min(slot / V * V, p.pairs - V));
  return min(first + slot % V, p.pairs - 1);
}

__device__ __forceinline__ double rot_position(const RotArgs &p, int64_t row, int axis) {
  const int64_t at = row * p.position_row + axis;
  if (p.position_type == RHIP_POSITION_I32)
    return static_cast<double>(static_cast<const int32_t *>(p.positions)[at]);
  if (p.position_type == RHIP_POSITION_I64)
    return static_cast<double>(static_cast<const int64_t *>(p.positions)[at]);
  return static_cast<double>(static_cast<const float *>(p.positions)[at]);
}

// Angle t as turns, without the whole ones. t times the first part of 1 / (2 pi) less
// its nearest whole number is exact, at any size; what it leaves with the second part
// has whole turns again from 2^53 on. (One product and its difference
// to the nearest whole number: off by up to 2^-24 of a turn at t = 2^31, by any part
// of one from 2^53 on; in the same time.)
__device__ __forceinline__ float rot_part(double t) {
  constexpr double kTurn = 0.15915494309189535, kRest = -9.839338337591243e-18;
  const double part = fma(t, kRest, fma(t, kTurn, -rint(t * kTurn)));
  return static_cast<float>(part - rint(part));
}

// Cosines and sines of the tile's rows: [row][slot], slots = turning * V.
template <int V>
__device__ __forceinline__ void rot_table(const RotArgs &p, int32_t row0, int32_t rows,
                                          float *cosines, float *sines) {
  const int slots = p.turning * V;
  for (int i = threadIdx.x; i < rows * slots; i += kRotThreads) {
    const int r = i / slots, pair = rot_pair<V>(p, i - r * slots);
    int axis = 0;
    while (axis < p.axes - 1 && pair >= p.ends[axis])
      ++axis;
    const double t =
        rot_position(p, static_cast<int64_t>(row0) + r, axis) * p.frequencies[pair];
    sincospif(2.f * rot_part(t), &sines[i], &cosines[i]);
  }
}

// Turns a lane's pairs by the angles at `at` of the table (`back`: the other way).
template <int V>
__device__ __forceinline__ void rot_turn(const RotArgs &p, bool back, const float *cosines,
                                         const float *sines, int at, float (&a)[V],
                                         float (&b)[V]) {
  float c[V], s[V];
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const v4f x = *reinterpret_cast<const v4f *>(cosines + at + i);
    const v4f y = *reinterpret_cast<const v4f *>(sines + at + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[i + e] = x[e];
      s[i + e] = back ? -y[e] : y[e];
    }
  }
  auto turn = [&](float &x, float &y, int i) {
    const float u = x * c[i] - y * s[i];
    y = fmaf(x, s[i], y * c[i]);
    x = u;
  };
  if (p.interleaved) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      turn(a[i], a[i + 1], i / 2);
      turn(b[i], b[i + 1], V / 2 + i / 2);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      turn(a[i], b[i], i);
  }
}

template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int off = 1; off < G; off <<= 1)
    v += __shfl_xor(v, off, kWave);
  return v;
}

template <int V>
__device__ __forceinline__ void rot_weight(const float *w, const RotLane &l, float (&wa)[V],
                                           float (&wb)[V]) {
  load_params<V>(w ? w + l.a : nullptr, 0, l.na, 1.f, wa);
  load_params<V>(w ? w + l.b : nullptr, 0, l.nb, 1.f, wb);
}

// The row (of the tile) of item i of a tensor, heads fastest.
__device__ __forceinline__ int32_t rot_row(const RotHeads &t, int32_t i) {
  return t.inverse ? static_cast<int32_t>(__umulhi(static_cast<uint32_t>(i), t.inverse))
                   : i / t.heads;
}

template <typename T, int G, bool NORM>
__global__ __launch_bounds__(kRotThreads) void rot_forward_kernel(RotArgs p) {
  using K = RowChunk<T>;
  constexpr int V = K::V, kGroups = kRotThreads / G;
  __shared__ alignas(16) float cosines[kRotTable], sines[kRotTable];
  const RotLane l = rot_lane<V>(p, threadIdx.x % G);
  const float inv = 1.f / static_cast<float>(p.dim);
  for (int32_t tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
    const int32_t row0 = tile * p.rows, rows = min(p.rows, p.n - row0);
    __syncthreads(); // the last tile's table is free
    rot_table<V>(p, row0, rows, cosines, sines);
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const RotHeads &t = p.t[which];
      float wa[V], wb[V];
      if constexpr (NORM)
        rot_weight<V>(t.weight, l, wa, wb);
      const int32_t step = gridDim.y * kGroups;
      for (int32_t i = blockIdx.y * kGroups + threadIdx.x / G; i < rows * t.heads; i += step) {
        const int32_t r = rot_row(t, i), head = i - r * t.heads;
        const int64_t row = static_cast<int64_t>(row0) + r;
        const T *x = static_cast<const T *>(t.x) + row * t.x_row + head * t.x_head;
        // both loads before the first use
        const v4u ra = K::fetch(x + l.a, l.na, false), rb = K::fetch(x + l.b, l.nb, false);
        float a[V], b[V];
        K::unpack(ra, a);
        K::unpack(rb, b);
        if constexpr (NORM) {
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            sum = fmaf(e >= l.skip_a ? a[e] : 0.f, a[e], sum);
            sum = fmaf(e >= l.skip_b ? b[e] : 0.f, b[e], sum);
          }
          const float rs = 1.f / sqrtf(group_sum<G>(sum) * inv + p.eps);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            a[e] *= rs * wa[e];
            b[e] *= rs * wb[e];
          }
        }
        if (l.pair >= 0)
          rot_turn<V>(p, false, cosines, sines, r * p.turning * V + l.pair, a, b);
        T *y = static_cast<T *>(t.y) + (row * t.heads + head) * p.dim;
        K::store(y + l.a, l.na, a);
        K::store(y + l.b, l.nb, b);
      }
    }
  }
}

template <typename T, int G, bool NORM>
__global__ __launch_bounds__(kRotThreads) void rot_backward_kernel(RotArgs p) {
  using K = RowChunk<T>;
  constexpr int V = K::V, kGroups = kRotThreads / G;
  __shared__ alignas(16) float cosines[kRotTable], sines[kRotTable];
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const RotLane l = rot_lane<V>(p, lane);
  const float inv = 1.f / static_cast<float>(p.dim);
  float sa[2][V], sb[2][V]; // sums of d x r, of both tensors
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int e = 0; e < V; ++e)
      sa[which][e] = sb[which][e] = 0.f;
  for (int32_t tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
    const int32_t row0 = tile * p.rows, rows = min(p.rows, p.n - row0);
    __syncthreads(); // the last tile's table is free
    rot_table<V>(p, row0, rows, cosines, sines);
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const RotHeads &t = p.t[which];
      float wa[V], wb[V];
      if constexpr (NORM)
        rot_weight<V>(t.weight, l, wa, wb);
      for (int32_t i = group; i < rows * t.heads; i += kGroups) {
        const int32_t r = rot_row(t, i), head = i - r * t.heads;
        const int64_t row = static_cast<int64_t>(row0) + r;
        const T *gy = static_cast<const T *>(t.gy) + row * t.gy_row + head * t.gy_head;
        // all loads before the first use
        const v4u ra = K::fetch(gy + l.a, l.na, false), rb = K::fetch(gy + l.b, l.nb, false);
        v4u rxa{}, rxb{};
        if constexpr (NORM) {
          const T *x = static_cast<const T *>(t.x) + row * t.x_row + head * t.x_head;
          rxa = K::fetch(x + l.a, l.na, false);
          rxb = K::fetch(x + l.b, l.nb, false);
        }
        float a[V], b[V];
        K::unpack(ra, a);
        K::unpack(rb, b);
        if (l.pair >= 0)
          rot_turn<V>(p, true, cosines, sines, r * p.turning * V + l.pair, a, b);
        if constexpr (NORM) {
          float xa[V], xb[V], sq = 0.f, dot = 0.f;
          K::unpack(rxa, xa);
          K::unpack(rxb, xb);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float ya = e >= l.skip_a ? xa[e] : 0.f, yb = e >= l.skip_b ? xb[e] : 0.f;
            sq = fmaf(ya, xa[e], sq);
            sq = fmaf(yb, xb[e], sq);
            dot = fmaf(ya, a[e] * wa[e], dot);
            dot = fmaf(yb, b[e] * wb[e], dot);
          }
          const float rs = 1.f / sqrtf(group_sum<G>(sq) * inv + p.eps);
          const float mean = group_sum<G>(dot) * inv * rs * rs;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            sa[which][e] = fmaf(a[e], xa[e] * rs, sa[which][e]);
            sb[which][e] = fmaf(b[e], xb[e] * rs, sb[which][e]);
            a[e] = rs * (a[e] * wa[e] - xa[e] * mean);
            b[e] = rs * (b[e] * wb[e] - xb[e] * mean);
          }
        }
        if (t.y) {
          T *y = static_cast<T *>(t.y) + (row * t.heads + head) * p.dim;
          K::store(y + l.a, l.na, a);
          K::store(y + l.b, l.nb, b);
        }
      }
    }
  }
  if constexpr (NORM) {
    if (!p.part)
      return;
    // the groups' sums, added in group order
    __shared__ float sums[kRotThreads][2 * V + 1];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) {
        sums[threadIdx.x][e] = sa[which][e];
        sums[threadIdx.x][V + e] = sb[which][e];
      }
      __syncthreads();
      if (group == 0) {
#pragma unroll 1
        for (int k = 1; k < kGroups; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            sa[which][e] += sums[k * G + lane][e];
            sb[which][e] += sums[k * G + lane][V + e];
          }
        float *dst = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + which) * p.dim;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (e >= l.skip_a && e < l.na)
            dst[l.a + e] = sa[which][e];
          if (e >= l.skip_b && e < l.nb)
            dst[l.b + e] = sb[which][e];
        }
      }
    }
  }
}

// The weights' gradients from the workgroups' sums: a wave per element, fp64,
// fixed order.
__global__ __launch_bounds__(kWave) void rot_sums_kernel(const float *__restrict__ part,
                                                         int blocks, int dim, float *gq,
                                                         float *gk) {
  const int c = blockIdx.x;
  float *dst = c < dim ? gq : gk;
  if (!dst)
    return;
  double s = 0.0;
  for (int b = threadIdx.x; b < blocks; b += kWave)
    s += part[static_cast<int64_t>(b) * 2 * dim + c];
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1)
    s += __shfl_xor(s, off, kWave);
  if (threadIdx.x == 0)
    dst[c < dim ? c : c - dim] = static_cast<float>(s);
}

// ------------------------------------------------------------------ host

void check_rotary(const rhip_rotary *r) {
  RHIP_CHECK_ARG(r != nullptr, "descriptor is null");
  if (r->dtype != RHIP_F32 && r->dtype != RHIP_BF16)
    throw Error(RHIP_ERR_UNSUPPORTED, "dtype must be RHIP_F32 or RHIP_BF16");
  RHIP_CHECK_ARG(r->n >= 0, "bad row count");
  if (r->n > INT32_MAX - kRotMaxRows)
    throw Error(RHIP_ERR_UNSUPPORTED, "too many rows");
  RHIP_CHECK_ARG(r->dim >= 1, "head width must be positive");
  if (r->dim > kRotMaxDim)
    throw Error(RHIP_ERR_UNSUPPORTED, "head width must not exceed 256");
  RHIP_CHECK_ARG(r->axes >= 1 && r->axes <= RHIP_ROTARY_MAX_AXES,
                 "positions must have 1 to 8 axes");
  int64_t pairs = 0;
  for (int i = 0; i < r->axes; ++i) {
    RHIP_CHECK_ARG(r->sections[i] >= 0, "sections must not be negative");
    pairs += r->sections[i];
  }
  RHIP_CHECK_ARG(pairs >= 1 && 2 * pairs <= r->dim,
                 "sections must hold at least one pair and no more than the head width");
  RHIP_CHECK_ARG(r->position_type >= RHIP_POSITION_I32 && r->position_type <= RHIP_POSITION_F32,
                 "position_type must be one of RHIP_POSITION_");
  RHIP_CHECK_ARG(!r->norm || static_cast<float>(r->eps) > 0.f, "eps must be positive in fp32");
  RHIP_CHECK_ARG(r->n == 0 || (r->positions && r->frequencies),
                 "positions and frequencies are required");
}

void check_rotary_heads(const rhip_rotary *r, const rhip_rotary_heads *h, bool backward) {
  RHIP_CHECK_ARG(h->heads >= 1, "a tensor needs at least one head");
  if (h->heads > (1 << 20))
    throw Error(RHIP_ERR_UNSUPPORTED, "at most 2^20 heads");
  if (r->n == 0)
    return;
  RHIP_CHECK_ARG(backward ? h->grad_y != nullptr && (!r->norm || h->x) : h->x && h->y,
                 "a tensor's operands are required");
}

int rot_v(int32_t dtype) { return dtype == RHIP_F32 ? 4 : 8; }
struct RotShape {
  int32_t turning, passing, group;
};
RotShape rot_shape(const rhip_rotary *r) {
  const int v = rot_v(r->dtype);
  int32_t pairs = 0;
  for (int i = 0; i < r->axes; ++i)
    pairs += r->sections[i];
  RotShape s;
  s.turning = static_cast<int32_t>(ceil_div(pairs, v));
  s.passing = static_cast<int32_t>(ceil_div(r->dim - 2 * pairs, 2 * v));
  s.group = 1;
  while (s.group < s.turning + s.passing)
    s.group *= 2;
  return s;
}

// Rows per tile: at most sixteen heads for each group of a workgroup, and two
// pairs of the table for each thread with the norm, one without (more make a
// start that the others wait for: rotation of 100003 rows of 8 heads of 32 27 us,
// with four 37), while that leaves two workgroups for each CU.
int32_t rot_rows(const rhip_rotary *r, const RotShape &s, int64_t heads) {
  const int64_t groups = kRotThreads / s.group;
  const int64_t slots = static_cast<int64_t>(s.turning) * rot_v(r->dtype);
  const int64_t rows = std::min<int64_t>({16 * groups / heads,
                                          kRotTable / (r->norm ? 1 : 2) / slots, kRotMaxRows,
                                          r->n / 512});
  return static_cast<int32_t>(std::max<int64_t>(rows, 1));
}

RotArgs rot_args(const rhip_rotary *r, const rhip_rotary_heads *q, const rhip_rotary_heads *k) {
  RotArgs p{};
  const RotShape s = rot_shape(r);
  for (const auto *h : {q, k}) {
    RotHeads &t = p.t[h == q ? 0 : 1];
    if (!h)
      continue;
    t.x = h->x, t.x_row = h->x_row, t.x_head = h->x_head;
    t.weight = h->weight, t.heads = h->heads;
    // exact for items below 2^32 / heads; a tile has at most kRotMaxRows * heads
    t.inverse = h->heads <= 4096 && h->heads > 1
                    ? static_cast<uint32_t>(((uint64_t(1) << 32) + h->heads - 1) / h->heads)
                    : 0u;
  }
  p.positions = r->positions, p.position_row = r->position_row;
  p.position_type = r->position_type, p.frequencies = r->frequencies;
  p.axes = r->axes;
  for (int i = 0; i < r->axes; ++i) {
    p.pairs += r->sections[i];
    p.ends[i] = p.pairs;
  }
  p.n = static_cast<int32_t>(r->n), p.dim = r->dim;
  p.turning = s.turning, p.passing = s.passing;
  p.rows = rot_rows(r, s, q->heads + (k ? k->heads : 0));
  p.tiles = static_cast<int32_t>(ceil_div(r->n, p.rows));
  p.interleaved = r->interleaved ? 1 : 0;
  p.eps = static_cast<float>(r->eps);
  return p;
}

// f(T{}, lanes of a group, whether the heads are normed)
template <typename F> void with_rotary(const rhip_rotary *r, F &&f) {
  auto grouped = [&](auto t, auto norm) {
    switch (rot_shape(r).group) {
    case 1: return f(t, std::integral_constant<int, 1>{}, norm);
    case 2: return f(t, std::integral_constant<int, 2>{}, norm);
    case 4: return f(t, std::integral_constant<int, 4>{}, norm);
    case 8: return f(t, std::integral_constant<int, 8>{}, norm);
    case 16: return f(t, std::integral_constant<int, 16>{}, norm);
    case 32: return f(t, std::integral_constant<int, 32>{}, norm);
    default: return f(t, std::integral_constant<int, 64>{}, norm);
    }
  };
  auto typed = [&](auto t) {
    if (r->norm)
      grouped(t, std::true_type{});
    else
      grouped(t, std::false_type{});
  };
  if (r->dtype == RHIP_F32)
    typed(float{});
  else
    typed(__bf16{});
}

constexpr int64_t kRotMaxGrid = 1 << 20; // tiles beyond it go in further turns

int64_t rot_backward_blocks(const rhip_rotary *r, int32_t tiles) {
  return std::max<int64_t>(1, std::min<int64_t>(tiles, r->norm ? kRotBlocks : kRotMaxGrid));
}

} // namespace
} // namespace rhip

using namespace rhip;

extern "C" int rhip_rotary_forward(const rhip_rotary *rotary, const rhip_rotary_heads *q,
                                   const rhip_rotary_heads *k, hipStream_t stream) {
  return guarded([&] {
    check_rotary(rotary);
    RHIP_CHECK_ARG(q != nullptr, "the first tensor is required");
    check_rotary_heads(rotary, q, false);
    if (k)
      check_rotary_heads(rotary, k, false);
    if (rotary->n == 0)
      return;
    RotArgs p = rot_args(rotary, q, k);
    p.t[0].y = q->y;
    if (k)
      p.t[1].y = k->y;
    with_rotary(rotary, [&](auto t, auto g, auto norm) {
      constexpr int G = decltype(g)::value;
      // few rows: their heads over several workgroups, one for each group
      const int64_t items = static_cast<int64_t>(p.rows) * std::max(p.t[0].heads, p.t[1].heads);
      const int64_t share = std::min<int64_t>(ceil_div(items, kRotThreads / G),
                                              std::max<int64_t>(1, 1024 / p.tiles));
      const dim3 grid(static_cast<unsigned>(std::min<int64_t>(p.tiles, kRotMaxGrid)),
                      static_cast<unsigned>(share));
      hipLaunchKernelGGL((rot_forward_kernel<decltype(t), G, decltype(norm)::value>), grid,
                         dim3(kRotThreads), 0, stream, p);
      RHIP_LAUNCH_CHECK();
    });
  });
}

extern "C" int rhip_rotary_workspace_bytes(const rhip_rotary *rotary, size_t *bytes) {
  return guarded([&] {
    check_rotary(rotary);
    RHIP_CHECK_ARG(bytes != nullptr, "bytes is null");
    Carve cv(nullptr, 0);
    if (rotary->norm)
      cv.take<float>(static_cast<size_t>(kRotBlocks) * 2 * rotary->dim);
    *bytes = cv.used + 256;
  });
}

extern "C" int rhip_rotary_backward(const rhip_rotary *rotary, const rhip_rotary_heads *q,
                                    const rhip_rotary_heads *k, void *workspace,
                                    size_t ws_bytes, hipStream_t stream) {
  return guarded([&] {
    check_rotary(rotary);
    RHIP_CHECK_ARG(q != nullptr, "the first tensor is required");
    check_rotary_heads(rotary, q, true);
    if (k)
      check_rotary_heads(rotary, k, true);
    float *gq = rotary->norm ? q->grad_weight : nullptr;
    float *gk = rotary->norm && k ? k->grad_weight : nullptr;
    if (!gq && !gk && (rotary->n == 0 || (!q->grad_x && !(k && k->grad_x))))
      return;
    RHIP_CHECK_ARG(workspace != nullptr || !(gq || gk), "workspace is required");
    RotArgs p = rot_args(rotary, q, k);
    int64_t blocks = 0;
    if (gq || gk) {
      Carve cv(workspace, ws_bytes);
      p.part = cv.take<float>(static_cast<size_t>(kRotBlocks) * 2 * p.dim);
    }
    for (const auto *h : {q, k}) {
      if (!h)
        continue;
      RotHeads &t = p.t[h == q ? 0 : 1];
      t.gy = h->grad_y, t.gy_row = h->grad_y_row, t.gy_head = h->grad_y_head;
      t.y = h->grad_x;
    }
    if (rotary->n > 0) {
      blocks = rot_backward_blocks(rotary, p.tiles);
      with_rotary(rotary, [&](auto t, auto g, auto norm) {
        hipLaunchKernelGGL(
            (rot_backward_kernel<decltype(t), decltype(g)::value, decltype(norm)::value>),
            dim3(static_cast<unsigned>(blocks)), dim3(kRotThreads), 0, stream, p);
        RHIP_LAUNCH_CHECK();
      });
    }
    if (p.part) {
      hipLaunchKernelGGL(rot_sums_kernel, dim3(2 * static_cast<unsigned>(p.dim)), dim3(kWave), 0,
                         stream, p.part, static_cast<int>(blocks), p.dim, gq, gk);
      RHIP_LAUNCH_CHECK();
    }
  });
}
