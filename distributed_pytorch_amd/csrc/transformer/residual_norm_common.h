// Row layout shared by the two directions of residual_norm: which lanes own a row and how its chunks are moved.
//
// A row of C channels is cut into chunks of 16 bytes.  Up to 64 chunks: G lanes of one wave own the row (G the power of
// two >= chunks, at least 4; 64 / G rows side by side); up to 128: a wave with two chunks a lane; wider: a workgroup of
// just the waves that the row fills, with 1 (up to 512 chunks), 2 or 4 chunks a lane (a sum then takes a barrier, but the
// per-channel sums of backward stay few enough for registers, and 320 chunks do not idle half of 2 x 256 lanes).  Rows whose length or base is not a multiple of 16 bytes move element by element (VEC =
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
  int threads;
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
    p.threads = 256;
  } else {
    p.maxch = chunks <= 512 ? 1 : (chunks <= 1024 ? 2 : 4);
    p.threads = ((chunks + p.maxch - 1) / p.maxch + 63) / 64 * 64;
    p.G = p.threads;
    p.rows_per_trip = 1;
  }
  return p;
}

// sum over groups of G (4 .. 64, a power of two) neighbouring lanes, the same in every lane of a group.  Lane exchange in
// the VALU (DPP inside rows of 16 lanes, the permlane swaps across them): a butterfly of LDS shuffles waits for LDS six
// times, and two sums per row and norm are the longest chain of these kernels
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_sum(float v, int G) {
  v += dpp<0xB1>(v);                       // quad_perm 1 0 3 2
  v += dpp<0x4E>(v);                       // quad_perm 2 3 0 1
  if (G >= 8) v += dpp<0x141>(v);          // row_half_mirror
  if (G >= 16) v += dpp<0x140>(v);         // row_mirror
  if (G >= 32) {
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  if (G >= 64) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  return v;
}

// sum over the lanes that own a row; R sums at once.  WIDE: `red` is [2][R][8] floats of LDS, cleared at the start (clear());
// consecutive calls alternate between its halves, so one barrier per call separates a write from the read of the call
// before the last
constexpr int kMaxWaves = 8;
template <bool WIDE, int R> struct GroupSum {
  float* red;
  int flip = 0;
  __device__ __forceinline__ void clear() {
    if constexpr (WIDE) {
      if (threadIdx.x < 2 * R * kMaxWaves) red[threadIdx.x] = 0.f;
      __syncthreads();
    }
  }
  __device__ __forceinline__ void run(float (&v)[R], int G) {
    if constexpr (!WIDE) {
#pragma unroll
      for (int r = 0; r < R; ++r) v[r] = lane_sum(v[r], G);
    } else {
      float* half = red + flip * R * kMaxWaves;
      flip ^= 1;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        v[r] = lane_sum(v[r], 64);
        if ((threadIdx.x & 63) == 0) half[r * kMaxWaves + (threadIdx.x >> 6)] = v[r];
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 a = reinterpret_cast<const float4*>(half + r * kMaxWaves)[0], b = reinterpret_cast<const float4*>(half + r * kMaxWaves)[1];
        v[r] = ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
      }
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
