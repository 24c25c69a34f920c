// Forward of the fused residual sum with its norms (gfx950):
//
//     z = post(y)         LayerNorm ((v - mean) / sqrt(var + eps) * w + b), RMSNorm (v / sqrt(mean(v^2) + eps) * w) or y
//     s = x + scale[n] * gate * z        gate: none, [C] (layer scale) or [N][C]; scale: [N] (stochastic depth)
//     h = pre(s)          the norm in front of the next block
//
// One pass: x and y are read once, s and h written once; s stays in registers in 32 bits between the sum and the
// statistics of `pre` (which therefore see the unrounded sum), statistics are a true two-pass mean / variance.  Bound by
// memory bandwidth (the layout of a row is in residual_norm_common.h): 64 x 197 x 1024 bf16 with `pre` 24 us, 4.3 TB/s; 64 x
// 3136 x 96 bf16 with `post` 32 us, 3.6 TB/s; 24 x 257 x 1280 fp32 with both and a gate 31 us, 4.1 TB/s, behind the writes
// of a backward pass (21, 26 and 24 us with inputs in the last-level cache).  Rows that are no whole 16-byte chunks move element
// by element: 64 x 197 x 1023 bf16 with `pre` 113 us, backward 119.
#include "residual_norm_common.h"

namespace dpa {
namespace {
using namespace rn;

// statistics of R rows held as floats (zeros behind the row's end)
template <typename T, int MAXCH, int R, bool WIDE, bool VEC>
__device__ __forceinline__ void row_stats(const float (&v)[R][MAXCH][kV<T>], int kind, float eps, float invC, int gl, int G,
                                          int C, GroupSum<WIDE, R>& gs, float (&mean)[R], float (&rstd)[R]) {
  constexpr int V = kV<T>;
#pragma unroll
  for (int r = 0; r < R; ++r) mean[r] = 0.f;
  if (kind == kNormLayer) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < MAXCH; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) mean[r] += v[r][k][j];
    gs.run(mean, G);
#pragma unroll
    for (int r = 0; r < R; ++r) mean[r] *= invC;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    rstd[r] = 0.f;
#pragma unroll
    for (int k = 0; k < MAXCH; ++k) {
      const int c0 = (gl + k * G) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = v[r][k][j] - mean[r];
        rstd[r] += (VEC ? c0 < C : c0 + j < C) ? d * d : 0.f;
      }
    }
  }
  gs.run(rstd, G);
#pragma unroll
  for (int r = 0; r < R; ++r) rstd[r] = rsqrtf(rstd[r] * invC + eps);
}

template <typename T, int MAXCH, int R, bool WIDE, bool VEC>
__global__ __launch_bounds__(WIDE ? 512 : 256) void residual_norm_fwd_kernel(const ResidualNormFwd p, const int G,
                                                                const FastDiv by_sample) {
  constexpr int V = kV<T>;
  __shared__ __attribute__((aligned(16))) float red[WIDE ? 2 * R * kMaxWaves : 4];
  GroupSum<WIDE, R> gs{red};
  gs.clear();
  const int lane = threadIdx.x & 63;
  const int gl = WIDE ? threadIdx.x : (lane & (G - 1));
  const int rpw = WIDE ? 1 : 64 / G;
  const int groups = WIDE ? 1 : 4;                       // row groups of a workgroup that walk on their own
  const int grp = WIDE ? 0 : threadIdx.x >> 6;
  const int C = p.C;
  const float invC = 1.f / (float)C;
  const T* x = reinterpret_cast<const T*>(p.x);
  const T* y = reinterpret_cast<const T*>(p.y);
  T* s_out = reinterpret_cast<T*>(p.s);
  T* h_out = reinterpret_cast<T*>(p.h);
  const long stride = (long)gridDim.x * groups * rpw * R;
  // uniform trip count per wave (workgroup): lanes whose row is past the end are masked
  for (long base = ((long)blockIdx.x * groups + grp) * rpw * R; base < p.rows; base += stride) {
    long row[R];
    bool live[R];
    Vec16<T> xv[R][MAXCH], yv[R][MAXCH];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      row[r] = base + r * rpw + (WIDE ? 0 : lane / G);
      live[r] = row[r] < p.rows;
      const int Cr = live[r] ? C : 0;                    // a dead row has no elements
      const long at = live[r] ? row[r] * C : 0;
#pragma unroll
      for (int k = 0; k < MAXCH; ++k) {
        xv[r][k] = load_chunk<T, VEC>(x + at, gl + k * G, Cr);
        if (y != nullptr) yv[r][k] = load_chunk<T, VEC>(y + at, gl + k * G, Cr);
      }
    }
    float s[R][MAXCH][V];
    if (y == nullptr) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < MAXCH; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) s[r][k][j] = xv[r][k].get(j);
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < MAXCH; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) s[r][k][j] = yv[r][k].get(j);
      if (p.post != kNormNone) {
        float mean[R], rstd[R];
        row_stats<T, MAXCH, R, WIDE, VEC>(s, p.post, p.post_eps, invC, gl, G, C, gs, mean, rstd);
#pragma unroll
        for (int k = 0; k < MAXCH; ++k) {
          float w[V], b[V];
          load_vec<V, VEC>(p.post_w, gl + k * G, C, 1.f, w);
          load_vec<V, VEC>(p.post_b, gl + k * G, C, 0.f, b);
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < V; ++j) s[r][k][j] = (s[r][k][j] - mean[r]) * rstd[r] * w[j] + b[j];
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (live[r] && gl == 0 && p.post_stat != nullptr) {
            p.post_stat[row[r]] = mean[r];
            p.post_stat[p.rows + row[r]] = rstd[r];
          }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const long n = p.scale != nullptr || p.gate_kind == kGateSample ? fdiv((uint32_t)(live[r] ? row[r] : 0), by_sample) : 0;
        const float sc = p.scale != nullptr ? p.scale[n] : 1.f;
        const float* gate = p.gate_kind == kGateSample ? p.gate + n * C : p.gate;
#pragma unroll
        for (int k = 0; k < MAXCH; ++k) {
          float g[V];
          load_vec<V, VEC>(gate, gl + k * G, C, 1.f, g);
          Vec16<T> o;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            s[r][k][j] = xv[r][k].get(j) + sc * g[j] * s[r][k][j];
            o.set(j, s[r][k][j]);
          }
          if (live[r]) store_chunk<T, VEC>(o, s_out + row[r] * C, gl + k * G, C);
        }
      }
    }
    if (p.pre != kNormNone) {
      // post(0) of a chunk behind the row's end is not zero: take it out of the sums
#pragma unroll
      for (int k = 0; k < MAXCH; ++k) {
        const int c0 = (gl + k * G) * V;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (!(VEC ? c0 < C : c0 + j < C))
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][k][j] = 0.f;
      }
      float mean[R], rstd[R];
      row_stats<T, MAXCH, R, WIDE, VEC>(s, p.pre, p.pre_eps, invC, gl, G, C, gs, mean, rstd);
#pragma unroll
      for (int k = 0; k < MAXCH; ++k) {
        float w[V], b[V];
        load_vec<V, VEC>(p.pre_w, gl + k * G, C, 1.f, w);
        load_vec<V, VEC>(p.pre_b, gl + k * G, C, 0.f, b);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          Vec16<T> o;
#pragma unroll
          for (int j = 0; j < V; ++j) o.set(j, (s[r][k][j] - mean[r]) * rstd[r] * w[j] + b[j]);
          if (live[r]) store_chunk<T, VEC>(o, h_out + row[r] * C, gl + k * G, C);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (live[r] && gl == 0 && p.pre_stat != nullptr) {
          p.pre_stat[row[r]] = mean[r];
          p.pre_stat[p.rows + row[r]] = rstd[r];
        }
    }
  }
}

template <typename T, int MAXCH, int R, bool WIDE>
void launch(const ResidualNormFwd& p, const Plan& pl, bool vec, hipStream_t s) {
  const long trips = (p.rows + (long)pl.rows_per_trip * R - 1) / ((long)pl.rows_per_trip * R);
  const unsigned blocks = (unsigned)(trips < 2048 ? trips : 2048);
  const FastDiv by_sample = make_fastdiv((uint32_t)p.per_sample);
  if (vec)
    hipLaunchKernelGGL((residual_norm_fwd_kernel<T, MAXCH, R, WIDE, true>), dim3(blocks), dim3(pl.threads), 0, s, p, pl.G, by_sample);
  else
    hipLaunchKernelGGL((residual_norm_fwd_kernel<T, MAXCH, R, WIDE, false>), dim3(blocks), dim3(pl.threads), 0, s, p, pl.G, by_sample);
}

}  // namespace

void residual_norm_fwd_launch(const ResidualNormFwd& p, int dtype, hipStream_t s) {
  if (p.rows <= 0) return;
  if (p.rows >= (1l << 31)) throw std::invalid_argument("residual_norm: at most 2^31 - 1 rows");
  const int vecn = dtype == kF32 ? 4 : 8;
  if (p.C <= 0 || (p.C + vecn - 1) / vecn > kResidualNormMaxChunks)
    throw std::invalid_argument("residual_norm: C must be 1 .. 2048 16-byte chunks");
  const Plan pl = plan(p.C, vecn);
  auto off16 = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) != 0; };
  const bool vec = p.C % vecn == 0 && !(off16(p.x) || off16(p.y) || off16(p.s) || off16(p.h) || off16(p.post_w) ||
                                        off16(p.post_b) || off16(p.pre_w) || off16(p.pre_b) || off16(p.gate));
  DPA_DISPATCH_DTYPE(dtype, {
    if (!pl.wide && pl.maxch == 1) launch<T, 1, 2, false>(p, pl, vec, s);
    else if (!pl.wide) launch<T, 2, 1, false>(p, pl, vec, s);
    else if (pl.maxch == 1) launch<T, 1, 1, true>(p, pl, vec, s);
    else if (pl.maxch == 2) launch<T, 2, 1, true>(p, pl, vec, s);
    else launch<T, 4, 1, true>(p, pl, vec, s);
  });
  DPA_CHECK_HIP(hipGetLastError());
}

}  // namespace dpa
