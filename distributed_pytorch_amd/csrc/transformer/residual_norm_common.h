// Row layout shared by the two directions of residual_norm: which lanes own a row and how its chunks are moved.
//
// A row of C channels is cut into chunks of 16 bytes.  Up to 64 chunks: G lanes of one wave own the row (G the power of
// two >= chunks, at least 4; 64 / G rows side by side); up to 128: a wave with two chunks a lane; wider: the workgroup's
// 256 lanes with 1, 2, 4 or 8 chunks each (a sum then takes two barriers, but the per-channel sums of backward stay
// few enough for registers).  Rows whose length or base is not a multiple of 16 bytes move element by element (VEC =
// false), in the same layout.
#pragma once
#include "../common.h"
#include "transformer.h"

namespace dpa {
namespace rn {

template <typename T> constexpr int kV = 16 / (int)sizeof(T);

struct Plan {
  int G, maxch;
  bool wide;
  int rows_per_trip;      // of a workgroup, with one row per lane group
};
inline Plan plan(int C, int vec) {
  Plan p;
  const int chunks = (C + vec - 1) / vec;
  p.wide = chunks > 128;
  if (!p.wide) {
    p.G = 4;
    while (p.G < chunks && p.G < 64) p.G <<= 1;
    p.maxch = chunks <= 64 ? 1 : 2;
    p.rows_per_trip = 4 * (64 / p.G);
  } else {
    p.G = 256;
    p.maxch = chunks <= 256 ? 1 : (chunks <= 512 ? 2 : (chunks <= 1024 ? 4 : 8));
    p.rows_per_trip = 1;
  }
  return p;
}

// sum over the lanes that own a row; R sums at once.  WIDE: `red` is [2][R][4] floats of LDS; consecutive calls
// alternate between its halves, so one barrier per call separates a write from the read of the call before the last
template <bool WIDE, int R> struct GroupSum {
  float* red;
  int flip = 0;
  __device__ __forceinline__ void run(float (&v)[R], int G) {
    if constexpr (!WIDE) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        for (int off = G >> 1; off > 0; off >>= 1) v[r] += __shfl_xor(v[r], off, 64);
    } else {
      float* half = red + flip * R * 4;
      flip ^= 1;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        v[r] = wave_sum(v[r]);
        if ((threadIdx.x & 63) == 0) half[r * 4 + (threadIdx.x >> 6)] = v[r];
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r) v[r] = (half[r * 4] + half[r * 4 + 1]) + (half[r * 4 + 2] + half[r * 4 + 3]);
    }
  }
};

// one chunk of a row; elements behind the row's end read as zero and are not written
template <typename T, bool VEC> __device__ __forceinline__ Vec16<T> load_chunk(const T* row, int ch, int C) {
  Vec16<T> v;
  v.raw = make_uint4(0u, 0u, 0u, 0u);
  const int c0 = ch * kV<T>;
  if constexpr (VEC) {
    if (c0 < C) v.load(row + c0);
  } else {
#pragma unroll
    for (int j = 0; j < kV<T>; ++j)
      if (c0 + j < C) __builtin_memcpy(reinterpret_cast<char*>(&v.raw) + j * sizeof(T), row + c0 + j, sizeof(T));
  }
  return v;
}
template <typename T, bool VEC> __device__ __forceinline__ void store_chunk(const Vec16<T>& v, T* row, int ch, int C) {
  const int c0 = ch * kV<T>;
  if constexpr (VEC) {
    if (c0 < C) v.store(row + c0);
  } else {
#pragma unroll
    for (int j = 0; j < kV<T>; ++j)
      if (c0 + j < C) __builtin_memcpy(row + c0 + j, reinterpret_cast<const char*>(&v.raw) + j * sizeof(T), sizeof(T));
  }
}
// the chunk's kV floats of a per-channel vector (`absent` where there is none)
template <int V, bool VEC> __device__ __forceinline__ void load_vec(const float* p, int ch, int C, float absent, float (&r)[V]) {
  const int c0 = ch * V;
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = absent;
    return;
  }
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const float4 a = c0 < C ? reinterpret_cast<const float4*>(p + c0)[q] : make_float4(0.f, 0.f, 0.f, 0.f);
      r[4 * q] = a.x; r[4 * q + 1] = a.y; r[4 * q + 2] = a.z; r[4 * q + 3] = a.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = c0 + j < C ? p[c0 + j] : 0.f;
  }
}

}  // namespace rn
}  // namespace dpa
