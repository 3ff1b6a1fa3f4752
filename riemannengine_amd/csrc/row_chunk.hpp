// Rows in 16-byte chunks at any alignment, for the kernels that stream whole
// rows (layer norm, embedding). Global loads and stores of 16 bytes need only
// the element's own alignment on gfx950, so rows of odd widths, strides and
// offsets move as fast as aligned ones. A row's last, partial chunk goes element
// by element here; the embedding moves it back to be whole.
#pragma once

#include "conv_device.hpp"

namespace rhip {

typedef v4u v4u_any __attribute__((aligned(2)));

template <typename T> struct RowChunk {
  static constexpr int V = 16 / sizeof(T); // elements per chunk

  // v[e] = p[e], 0 from element `left` on
  __device__ static __forceinline__ void load(const T *p, int left, float (&v)[V]) {
    if (left >= V) {
      unpack(raw(p), v);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        v[e] = e < left ? to_f32(p[e]) : 0.f;
    }
  }
  // Stores bypass the caches' write allocation: the rows are written once and
  // not read again here (16384 rows of 4096 bf16, layer norm forward: 75 us
  // with ordinary stores, 46 with these).
  __device__ static __forceinline__ void store(T *p, int left, const float (&v)[V]) {
    T t[V];
#pragma unroll
    for (int e = 0; e < V; ++e)
      t[e] = from_f32<T>(v[e]);
    if (left >= V) {
      __builtin_nontemporal_store(__builtin_bit_cast(v4u, t), reinterpret_cast<v4u_any *>(p));
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < left)
          p[e] = t[e];
    }
  }
  // The chunk as it lies, zeros from element `left` on; `whole`: rows hold
  // whole chunks, so left is a multiple of V (or negative) in every lane.
  __device__ static __forceinline__ v4u fetch(const T *p, int left, bool whole) {
    if (left >= V)
      return raw(p);
    v4u u{0u, 0u, 0u, 0u};
    if (!whole && left > 0) {
      T t[V];
#pragma unroll
      for (int e = 0; e < V; ++e)
        t[e] = e < left ? p[e] : static_cast<T>(0.f);
      __builtin_memcpy(&u, t, 16);
    }
    return u;
  }
  // the 16 bytes at p (all of them inside the row)
  __device__ static __forceinline__ v4u raw(const T *p) {
    return *reinterpret_cast<const v4u_any *>(p);
  }
  __device__ static __forceinline__ void unpack(const v4u &u, float (&v)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        v[e] = __uint_as_float(u[e]);
    } else {
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        v[2 * e] = __uint_as_float(u[e] << 16);
        v[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
      }
    }
  }
};

// V fp32 parameters from element c on, `dflt` past C or without a pointer.
template <int V>
__device__ __forceinline__ void load_params(const float *p, int c, int C, float dflt,
                                            float (&v)[V]) {
  if (p && c + V <= C) {
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      v4f f;
      __builtin_memcpy(&f, p + c + e, 16);
      v[e] = f[0], v[e + 1] = f[1], v[e + 2] = f[2], v[e + 3] = f[3];
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      v[e] = p && c + e < C ? p[c + e] : dflt;
  }
}

} // namespace rhip
