// Layer normalisation of feature rows on gfx950, forward and backward with
// the parameters' gradients.
//
// A row belongs to G lanes (8 .. 64 of a wave, or the workgroup's 256), which
// keep it in registers between its statistics and its output: x is read once
// in the forward, x and grad_y once in the backward. The variance is summed
// around the mean from the registers, so no cancellation: fp32 is enough.
// Rows too wide for the registers are streamed again from the caches.
//
// The parameters' gradients are sums over rows. A backward workgroup walks
// many rows and keeps its sums in registers next to the rows' own, writes
// them once, and a second kernel adds the workgroups' sums (fp64, fixed
// order).
//
// Bound by memory: 16384 rows of 4096 in bf16 take 46 us forward (5.8 TB/s), and
// 77 us backward with the second kernel (5.2 TB/s); 100k rows of 96, 11 and 24 us.
// One row is one launch, about 6 us.
#include <climits>
#include <type_traits>

#include "row_chunk.hpp"

namespace rhip {
namespace {

constexpr int kLnThreads = 256;
// Backward workgroups, two per CU: each writes 2 C fp32 sums, so more of them
// move more bytes (1024 of them on 16384 rows of 4096: 66 MB beside 402).
constexpr int kLnBlocks = 512;
constexpr int kSumCols = 16, kSumRows = 64; // ln_sums_kernel's columns and row lanes
constexpr int32_t kLnMaxC = 1 << 30; // a workgroup's steps along a row stay below 2^31
// ln_sums_kernel's launch: 2 C columns, 64 threads each
constexpr int32_t kLnMaxParams = (1 << 25) - kSumCols;

// N sums over a row's G lanes, in every lane; G = 256: the workgroup, through
// LDS (buf is free again after the next barrier but one).
template <int G, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*buf)[4]) {
#pragma unroll
  for (int off = 1; off < (G < kWave ? G : kWave); off <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] += __shfl_xor(v[i], off, kWave);
  if constexpr (G > kWave) {
    if (lane_id() == 0)
#pragma unroll
      for (int i = 0; i < N; ++i)
        buf[i][threadIdx.x / kWave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = (buf[i][0] + buf[i][1]) + (buf[i][2] + buf[i][3]);
  }
}

// y = (x - mean) rstd w + b: R rows at a time per group of G lanes, NC chunks
// of each per lane.
template <typename T, int G, int NC, int R>
__global__ __launch_bounds__(kLnThreads) void ln_forward_kernel(
    const T *__restrict__ x, int64_t x_row, int64_t n, int C, const float *__restrict__ weight,
    const float *__restrict__ bias, float eps, T *__restrict__ y, float *__restrict__ mean_out,
    float *__restrict__ rstd_out) {
  using K = RowChunk<T>;
  __shared__ float buf[2][R][4];
  const int lane = threadIdx.x % G;
  // rows row0 + r * groups: neighbouring groups stay neighbours in memory
  constexpr int kGroups = kLnThreads / G;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kGroups * R + threadIdx.x / G;
  float v[R][NC][K::V], mean[R], rstd[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = row0 + r * kGroups;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (lane + i * G) * K::V;
      K::load(x + row * x_row + c, row < n ? C - c : 0, v[r][i]);
    }
  }
  const float inv_c = 1.f / static_cast<float>(C);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mean[r] = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int e = 0; e < K::V; ++e)
        mean[r] += v[r][i][e];
  }
  row_sums<G>(mean, buf[0]);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mean[r] *= inv_c;
    rstd[r] = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = (lane + i * G) * K::V;
#pragma unroll
      for (int e = 0; e < K::V; ++e) {
        v[r][i][e] = c + e < C ? v[r][i][e] - mean[r] : 0.f;
        rstd[r] = fmaf(v[r][i][e], v[r][i][e], rstd[r]);
      }
    }
  }
  row_sums<G>(rstd, buf[1]);
#pragma unroll
  for (int r = 0; r < R; ++r)
    rstd[r] = 1.f / sqrtf(rstd[r] * inv_c + eps);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = (lane + i * G) * K::V;
    if (c >= C)
      continue;
    float w[K::V], b[K::V];
    load_params<K::V>(weight, c, C, 1.f, w);
    load_params<K::V>(bias, c, C, 0.f, b);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * kGroups;
      if (row < n) {
#pragma unroll
        for (int e = 0; e < K::V; ++e)
          v[r][i][e] = fmaf(v[r][i][e] * rstd[r], w[e], b[e]);
        K::store(y + row * C + c, C - c, v[r][i]);
      }
    }
  }
  if (mean_out && lane == 0)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * kGroups;
      if (row < n) {
        mean_out[row] = mean[r];
        rstd_out[row] = rstd[r];
      }
    }
}

// Rows wider than the registers: three passes over the row, the later two
// from the caches. One workgroup per row.
template <typename T>
__global__ __launch_bounds__(kLnThreads) void ln_forward_wide_kernel(
    const T *__restrict__ x, int64_t x_row, int64_t n, int C, const float *__restrict__ weight,
    const float *__restrict__ bias, float eps, T *__restrict__ y, float *__restrict__ mean_out,
    float *__restrict__ rstd_out) {
  using R = RowChunk<T>;
  __shared__ float buf[2][4];
  const int64_t row = blockIdx.x;
  const T *xr = x + row * x_row;
  const int c0 = threadIdx.x * R::V, step = kLnThreads * R::V;
  float v[R::V], s = 0.f;
  for (int c = c0; c < C; c += step) {
    R::load(xr + c, C - c, v);
#pragma unroll
    for (int e = 0; e < R::V; ++e)
      s += v[e];
  }
  float one[1] = {s};
  row_sums<kLnThreads>(one, &buf[0]);
  const float mean = one[0] / static_cast<float>(C);
  s = 0.f;
  for (int c = c0; c < C; c += step) {
    R::load(xr + c, C - c, v);
#pragma unroll
    for (int e = 0; e < R::V; ++e) {
      const float d = c + e < C ? v[e] - mean : 0.f;
      s = fmaf(d, d, s);
    }
  }
  one[0] = s;
  row_sums<kLnThreads>(one, &buf[1]);
  const float rstd = 1.f / sqrtf(one[0] / static_cast<float>(C) + eps);
  for (int c = c0; c < C; c += step) {
    float w[R::V], b[R::V];
    R::load(xr + c, C - c, v);
    load_params<R::V>(weight, c, C, 1.f, w);
    load_params<R::V>(bias, c, C, 0.f, b);
#pragma unroll
    for (int e = 0; e < R::V; ++e)
      v[e] = fmaf((v[e] - mean) * rstd, w[e], b[e]);
    R::store(y + row * C + c, C - c, v);
  }
  if (mean_out && threadIdx.x == 0) {
    mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
}

// grad_x of the workgroup's rows, R at a time per group of G lanes, and its
// sums of grad_y and grad_y xhat over them into part[b] = [2][C]. The next
// rows' loads are in flight while these are worked on.
template <typename T, int G, int NC, int R>
__global__ __launch_bounds__(kLnThreads, 2) void ln_backward_kernel(
    const T *__restrict__ gy, int64_t gy_row, const T *__restrict__ x, int64_t x_row, int64_t n,
    int C, const float *__restrict__ mean, const float *__restrict__ rstd,
    const float *__restrict__ weight, T *__restrict__ gx, float *__restrict__ part) {
  using K = RowChunk<T>;
  constexpr int kGroups = kLnThreads / G;
  __shared__ float buf[2][2 * R][4];
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const bool whole = C % K::V == 0; // no partial chunk: rows load as they lie
  float w[NC][K::V], sb[NC][K::V], sw[NC][K::V];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    load_params<K::V>(weight, (lane + i * G) * K::V, C, 1.f, w[i]);
#pragma unroll
    for (int e = 0; e < K::V; ++e)
      sb[i][e] = sw[i][e] = 0.f;
  }
  const float inv_c = 1.f / static_cast<float>(C);
  v4u ng[R][NC], nx[R][NC]; // the next rows
  float nm[R], nr[R];
  auto fetch = [&](int64_t r0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = r0 + r * kGroups + group;
      const bool ok = row < n;
      nm[r] = ok ? mean[row] : 0.f;
      nr[r] = ok ? rstd[row] : 0.f;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = (lane + i * G) * K::V;
        ng[r][i] = K::fetch(gy + row * gy_row + c, ok ? C - c : 0, whole);
        nx[r][i] = K::fetch(x + row * x_row + c, ok ? C - c : 0, whole);
      }
    }
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups * R;
  int64_t r0 = static_cast<int64_t>(blockIdx.x) * kGroups * R;
  if (r0 < n)
    fetch(r0);
  int turn = 0;
  // the workgroup's groups go through the loop together (its barriers)
  for (; r0 < n; r0 += step) {
    float g[R][NC][K::V], h[R][NC][K::V], rs[R], s[2 * R]; // grad_y, xhat
#pragma unroll
    for (int r = 0; r < R; ++r) {
      rs[r] = nr[r];
      s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = (lane + i * G) * K::V;
        K::unpack(ng[r][i], g[r][i]);
        K::unpack(nx[r][i], h[r][i]);
#pragma unroll
        for (int e = 0; e < K::V; ++e) {
          h[r][i][e] = (whole ? c : c + e) < C ? (h[r][i][e] - nm[r]) * rs[r] : 0.f;
          const float gw = g[r][i][e] * w[i][e];
          s[2 * r] += gw;
          s[2 * r + 1] = fmaf(gw, h[r][i][e], s[2 * r + 1]);
          sb[i][e] += g[r][i][e];
          sw[i][e] = fmaf(g[r][i][e], h[r][i][e], sw[i][e]);
        }
      }
    }
    if (r0 + step < n)
      fetch(r0 + step);
    if (gx) {
      row_sums<G>(s, buf[turn]);
      turn ^= 1;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t row = r0 + r * kGroups + group;
        const float s1 = s[2 * r] * inv_c, s2 = s[2 * r + 1] * inv_c;
        if (row < n) {
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            const int c = (lane + i * G) * K::V;
            if (c < C) {
              float o[K::V];
#pragma unroll
              for (int e = 0; e < K::V; ++e)
                o[e] = rs[r] * (g[r][i][e] * w[i][e] - s1 - h[r][i][e] * s2);
              K::store(gx + row * C + c, C - c, o);
            }
          }
        }
      }
    }
  }
  if (!part)
    return;
  float *dst = part + static_cast<int64_t>(blockIdx.x) * 2 * C;
  auto put = [&](int i, const float (&b)[K::V], const float (&s)[K::V]) {
    const int c = (lane + i * G) * K::V;
#pragma unroll
    for (int e = 0; e < K::V; ++e)
      if (c + e < C) {
        dst[c + e] = b[e];
        dst[C + c + e] = s[e];
      }
  };
  if constexpr (kGroups == 1) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      put(i, sb[i], sw[i]);
  } else {
    // the groups' sums, added in group order
    __shared__ float lds[kLnThreads][2 * K::V + 1];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < K::V; ++e) {
        lds[threadIdx.x][e] = sb[i][e];
        lds[threadIdx.x][K::V + e] = sw[i][e];
      }
      __syncthreads();
      if (group == 0) {
#pragma unroll 1
        for (int k = 1; k < kGroups; ++k)
#pragma unroll
          for (int e = 0; e < K::V; ++e) {
            sb[i][e] += lds[k * G + lane][e];
            sw[i][e] += lds[k * G + lane][K::V + e];
          }
        put(i, sb[i], sw[i]);
      }
    }
  }
}

// Wide rows: grad_x alone, a workgroup per row, reading the row twice.
template <typename T>
__global__ __launch_bounds__(kLnThreads) void ln_backward_wide_kernel(
    const T *__restrict__ gy, int64_t gy_row, const T *__restrict__ x, int64_t x_row, int C,
    const float *__restrict__ mean, const float *__restrict__ rstd,
    const float *__restrict__ weight, T *__restrict__ gx) {
  using R = RowChunk<T>;
  __shared__ float buf[2][4];
  const int64_t row = blockIdx.x;
  const T *xr = x + row * x_row, *gr = gy + row * gy_row;
  const float mu = mean[row], rs = rstd[row], inv_c = 1.f / static_cast<float>(C);
  const int c0 = threadIdx.x * R::V, step = kLnThreads * R::V;
  float g[R::V], h[R::V], w[R::V], s1 = 0.f, s2 = 0.f;
  auto load = [&](int c) {
    R::load(gr + c, C - c, g);
    R::load(xr + c, C - c, h);
    load_params<R::V>(weight, c, C, 1.f, w);
#pragma unroll
    for (int e = 0; e < R::V; ++e) {
      h[e] = c + e < C ? (h[e] - mu) * rs : 0.f;
      g[e] *= w[e];
    }
  };
  for (int c = c0; c < C; c += step) {
    load(c);
#pragma unroll
    for (int e = 0; e < R::V; ++e) {
      s1 += g[e];
      s2 = fmaf(g[e], h[e], s2);
    }
  }
  float both[2] = {s1, s2};
  row_sums<kLnThreads>(both, buf);
  s1 = both[0] * inv_c, s2 = both[1] * inv_c;
  for (int c = c0; c < C; c += step) {
    load(c);
#pragma unroll
    for (int e = 0; e < R::V; ++e)
      g[e] = rs * (g[e] - s1 - h[e] * s2);
    R::store(gx + row * C + c, C - c, g);
  }
}

// Wide rows: the parameters' sums of the rows b, b + blocks, .. over one tile
// of 256 chunks (blockIdx.y).
template <typename T>
__global__ __launch_bounds__(kLnThreads) void ln_param_wide_kernel(
    const T *__restrict__ gy, int64_t gy_row, const T *__restrict__ x, int64_t x_row, int64_t n,
    int C, const float *__restrict__ mean, const float *__restrict__ rstd,
    float *__restrict__ part) {
  using R = RowChunk<T>;
  const int c = (blockIdx.y * kLnThreads + threadIdx.x) * R::V;
  if (c >= C)
    return;
  float sb[R::V], sw[R::V];
#pragma unroll
  for (int e = 0; e < R::V; ++e)
    sb[e] = sw[e] = 0.f;
  for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
    const float mu = mean[row], rs = rstd[row];
    float g[R::V], h[R::V];
    R::load(gy + row * gy_row + c, C - c, g);
    R::load(x + row * x_row + c, C - c, h);
#pragma unroll
    for (int e = 0; e < R::V; ++e) {
      sb[e] += g[e];
      sw[e] = fmaf(g[e], (h[e] - mu) * rs, sw[e]);
    }
  }
  float *dst = part + static_cast<int64_t>(blockIdx.x) * 2 * C;
#pragma unroll
  for (int e = 0; e < R::V; ++e)
    if (c + e < C) {
      dst[c + e] = sb[e];
      dst[C + c + e] = sw[e];
    }
}

// grad_bias = sum over b of part[b][0], grad_weight of part[b][1]: 16 columns
// by 64 row lanes per workgroup, then a tree in LDS.
__global__ __launch_bounds__(kSumCols *kSumRows) void ln_sums_kernel(
    const float *__restrict__ part, int blocks, int C, float *__restrict__ gw,
    float *__restrict__ gb) {
  __shared__ double lds[kSumRows][kSumCols];
  const int col = threadIdx.x % kSumCols, r = threadIdx.x / kSumCols;
  const int c = blockIdx.x * kSumCols + col;
  double s = 0.0;
  if (c < 2 * C)
    for (int b = r; b < blocks; b += kSumRows)
      s += part[static_cast<int64_t>(b) * 2 * C + c];
  lds[r][col] = s;
#pragma unroll
  for (int off = kSumRows / 2; off; off >>= 1) {
    __syncthreads();
    if (r < off)
      lds[r][col] += lds[r + off][col];
  }
  if (r == 0 && c < 2 * C) {
    float *dst = c < C ? gb : gw;
    if (dst)
      dst[c < C ? c : c - C] = static_cast<float>(lds[0][col]);
  }
}

// ------------------------------------------------------------------ host

// f(T{}, lanes per row, chunks per lane, rows at a time); lanes 0: wider than
// the registers. Two chunks per lane until a wave is full, then up to four,
// then the workgroup shares the row; several narrow rows at a time, so that
// enough loads are in flight.
template <typename F> void with_row(int32_t dtype, int C, F &&f) {
  auto typed = [&](auto t) {
    const int chunks = static_cast<int>(ceil_div(C, RowChunk<decltype(t)>::V));
    auto go = [&](auto g, auto nc, auto r) { f(t, g, nc, r); };
    using std::integral_constant;
    if (chunks <= 16)
      go(integral_constant<int, 8>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
    else if (chunks <= 32)
      go(integral_constant<int, 16>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
    else if (chunks <= 64)
      go(integral_constant<int, 32>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
    else if (chunks <= 128)
      go(integral_constant<int, 64>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
    else if (chunks <= 256)
      go(integral_constant<int, 64>{}, integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else if (chunks <= 512)
      go(integral_constant<int, 256>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
    else if (chunks <= 1024)
      go(integral_constant<int, 256>{}, integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else
      go(integral_constant<int, 0>{}, integral_constant<int, 0>{}, integral_constant<int, 0>{});
  };
  if (dtype == RHIP_F32)
    typed(float{});
  else
    typed(__bf16{});
}

void check_rows(int32_t dtype, int64_t n, int32_t C) {
  if (dtype != RHIP_F32 && dtype != RHIP_BF16)
    throw Error(RHIP_ERR_UNSUPPORTED, "dtype must be RHIP_F32 or RHIP_BF16");
  RHIP_CHECK_ARG(n >= 0 && C >= 1, "bad sizes");
  if (n > INT32_MAX)
    throw Error(RHIP_ERR_UNSUPPORTED, "too many rows");
  if (C > kLnMaxC)
    throw Error(RHIP_ERR_UNSUPPORTED, "layer norm takes at most 2^30 channels");
}

// Workgroups of the backward: no more than row groups, at most kLnBlocks.
int64_t ln_blocks(int64_t n) { return std::max<int64_t>(1, std::min<int64_t>(n, kLnBlocks)); }

} // namespace
} // namespace rhip

using namespace rhip;

extern "C" int rhip_ln_workspace_bytes(int64_t n, int32_t C, size_t *bytes) {
  return guarded([&] {
    RHIP_CHECK_ARG(bytes != nullptr, "bytes is null");
    RHIP_CHECK_ARG(n >= 0 && C >= 1, "bad sizes");
    Carve cv(nullptr, 0);
    cv.take<float>(ln_blocks(n) * 2 * static_cast<size_t>(C));
    *bytes = cv.used + 256;
  });
}

extern "C" int rhip_ln_forward(const void *x, int64_t x_row, int64_t n, int32_t C,
                               const float *weight, const float *bias, double eps, void *y,
                               float *mean, float *rstd, int32_t dtype, hipStream_t stream) {
  return guarded([&] {
    check_rows(dtype, n, C);
    RHIP_CHECK_ARG(static_cast<float>(eps) > 0.f, "eps must be positive in fp32");
    RHIP_CHECK_ARG((mean == nullptr) == (rstd == nullptr), "mean and rstd go together");
    if (n == 0)
      return;
    RHIP_CHECK_ARG(x && y, "x and y are required");
    with_row(dtype, C, [&](auto t, auto g, auto nc, auto r) {
      using T = decltype(t);
      constexpr int G = decltype(g)::value, NC = decltype(nc)::value, R = decltype(r)::value;
      const T *xp = static_cast<const T *>(x);
      T *yp = static_cast<T *>(y);
      const float e = static_cast<float>(eps);
      constexpr int64_t kRows = G == 0 ? 1 : kLnThreads / (G == 0 ? 1 : G) * R; // of a workgroup
      const int64_t most = max_groups(kLnThreads) * kRows;
      for (int64_t r = 0; r < n; r += most) { // more rows than one launch takes: some narrow ones
        const int64_t rows = std::min(n - r, most);
        const dim3 g(static_cast<unsigned>(ceil_div(rows, kRows)));
        const T *xr = xp + r * x_row;
        T *yr = yp + r * C;
        float *mr = mean ? mean + r : nullptr, *sr = rstd ? rstd + r : nullptr;
        if constexpr (G == 0)
          hipLaunchKernelGGL((ln_forward_wide_kernel<T>), g, dim3(kLnThreads), 0, stream, xr, x_row,
                             rows, C, weight, bias, e, yr, mr, sr);
        else
          hipLaunchKernelGGL((ln_forward_kernel<T, G, NC, R>), g, dim3(kLnThreads), 0, stream, xr,
                             x_row, rows, C, weight, bias, e, yr, mr, sr);
        RHIP_LAUNCH_CHECK();
      }
    });
  });
}

extern "C" int rhip_ln_backward(const void *grad_y, int64_t grad_y_row, const void *x,
                                int64_t x_row, int64_t n, int32_t C, const float *mean,
                                const float *rstd, const float *weight, void *grad_x,
                                float *grad_weight, float *grad_bias, int32_t dtype,
                                void *workspace, size_t ws_bytes, hipStream_t stream) {
  return guarded([&] {
    check_rows(dtype, n, C);
    RHIP_CHECK_ARG(n == 0 || (grad_y && x && mean && rstd),
                   "grad_y, x, mean and rstd are required");
    const bool params = grad_weight || grad_bias;
    RHIP_CHECK_ARG(!params || workspace, "workspace is required");
    if (params && C > kLnMaxParams)
      throw Error(RHIP_ERR_UNSUPPORTED, "the parameters' gradients take fewer than 2^25 channels");
    int64_t blocks = ln_blocks(n);
    float *part = nullptr;
    if (params) {
      Carve cv(workspace, ws_bytes);
      part = cv.take<float>(blocks * 2 * static_cast<size_t>(C));
    }
    if (!params && (!grad_x || n == 0))
      return;
    with_row(dtype, C, [&](auto t, auto g, auto nc, auto r) {
      using T = decltype(t);
      constexpr int G = decltype(g)::value, NC = decltype(nc)::value, R = decltype(r)::value;
      const T *gp = static_cast<const T *>(grad_y), *xp = static_cast<const T *>(x);
      T *gxp = static_cast<T *>(grad_x);
      if constexpr (G == 0) {
        const int64_t most = max_groups(kLnThreads);
        for (int64_t r = 0; gxp && r < n; r += most) {
          hipLaunchKernelGGL((ln_backward_wide_kernel<T>),
                             dim3(static_cast<unsigned>(std::min(n - r, most))), dim3(kLnThreads),
                             0, stream, gp + r * grad_y_row, grad_y_row, xp + r * x_row, x_row, C,
                             mean + r, rstd + r, weight, gxp + r * C);
          RHIP_LAUNCH_CHECK();
        }
        if (part) {
          const unsigned tiles =
              static_cast<unsigned>(ceil_div(C, kLnThreads * RowChunk<T>::V));
          hipLaunchKernelGGL((ln_param_wide_kernel<T>), dim3(static_cast<unsigned>(blocks), tiles),
                             dim3(kLnThreads), 0, stream, gp, grad_y_row, xp, x_row, n, C, mean,
                             rstd, part);
          RHIP_LAUNCH_CHECK();
        }
      } else {
        blocks = std::max<int64_t>(1, std::min(blocks, ceil_div(n, kLnThreads / G * R)));
        hipLaunchKernelGGL((ln_backward_kernel<T, G, NC, R>), dim3(static_cast<unsigned>(blocks)),
                           dim3(kLnThreads), 0, stream, gp, grad_y_row, xp, x_row, n, C, mean,
                           rstd, weight, n > 0 ? gxp : nullptr, part);
        RHIP_LAUNCH_CHECK();
      }
    });
    if (part) {
      hipLaunchKernelGGL(ln_sums_kernel, dim3(static_cast<unsigned>(ceil_div(2 * C, kSumCols))),
                         dim3(kSumCols * kSumRows), 0, stream, part, static_cast<int>(blocks), C,
                         grad_weight, grad_bias);
      RHIP_LAUNCH_CHECK();
    }
  });
}
