// Backward of residual_norm (gfx950).  With sh = (s - mean) / dev and yh likewise:
//
//     gs = ds + dpre,  dpre = (g - [layer] mean(g) - sh * mean(g sh)) / dev,  g = dh * w_pre
//     dx = gs,  dz = scale * gate * gs,  dgate = sum scale * gs * z,  dw_pre = sum dh * sh,  db_pre = sum dh
//     dy = dz, or the same formula of `post` applied to it;  dw_post = sum dz * yh,  db_post = sum dz
//
// One pass: ds, dh, x, y are read once, dx and dy written once (64 x 197 x 1024 bf16 with `pre` 24 us, 5.3 TB/s; 64 x 3136 x
// 96 bf16 with `post` 28 us, 4.1 TB/s, with `pre` and a scale 51; 24 x 257 x 1280 fp32 with both and a per-sample gate 42 us, 4.5 TB/s; the fold 4 us, a
// launch and a wait for memory).  s is formed again from x and y in 32 bits: the s of
// the forward pass is rounded to T, and 1 / deviation and the sums over rows magnify that (dw_pre of bf16 rows is off by
// 2e-3 from it, by 2e-7 from this), for one more tensor to read where there is no `post` (5 in place of 4).  The per-channel sums stay with the lane across all rows
// that it visits (its channels never change), meet across the row groups of a wave with shuffles and across waves in
// LDS, and every workgroup writes one partial row; residual_norm_fold_kernel adds those in a fixed order, straight into
// the gradients' buffers.  A per-sample gate's sums are flushed at the end of every unit, a part of one sample's rows.
#include "residual_norm_common.h"
#include <atomic>

namespace dpa {
namespace {
using namespace rn;

constexpr int kCompute = 256;       // compute units
constexpr int kMaxParts = 1024;     // workgroups of the pass = partial rows of the fold, at most

// what a kernel is made for: s = x + y, s = x + scale * post(y) without `pre`, or everything
enum Mode : int { kPreOnly = 0, kPostOnly = 1, kAll = 2 };

// v[k][j] of every wave (row group) of the workgroup added up and written to out[C]; the lanes of the first group write
template <typename T, int MAXCH, bool WIDE, bool VEC>
__device__ __forceinline__ void merge_out(float (&v)[MAXCH][kV<T>], float* out, float* lds, int gl, int G, int C) {
  constexpr int V = kV<T>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if constexpr (!WIDE) {
#pragma unroll
    for (int k = 0; k < MAXCH; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j)
        for (int off = 32; off >= G; off >>= 1) v[k][j] += __shfl_xor(v[k][j], off, 64);
    __syncthreads();                                   // the buffer's last readers are done
    if (lane < G)
#pragma unroll
      for (int k = 0; k < MAXCH; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) lds[(wave * MAXCH * 64 + gl + k * G) * V + j] = v[k][j];
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += 256) {
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) a += lds[w * MAXCH * 64 * V + c];
      out[c] = a;
    }
  } else {
#pragma unroll
    for (int k = 0; k < MAXCH; ++k) {
      const int c0 = (gl + k * G) * V;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c0 + j < C) out[c0 + j] = v[k][j];
    }
  }
}

template <typename T, int MAXCH, bool WIDE, bool VEC, int MODE>
__global__ __launch_bounds__(WIDE ? 512 : 256) void residual_norm_bwd_kernel(const ResidualNormBwd p, const int G, const long units,
                                                                const long unit_rows, const int splits,
                                                                const FastDiv by_sample) {
  constexpr int V = kV<T>;
  constexpr bool PRE = MODE != kPostOnly, POST = MODE != kPreOnly;
  __shared__ __attribute__((aligned(16))) float red[WIDE ? 4 * kMaxWaves : 4];
  __shared__ float lds[WIDE ? 1 : 4 * MAXCH * 64 * V];
  GroupSum<WIDE, 2> gsum{red};
  gsum.clear();
  const int lane = threadIdx.x & 63;
  const int gl = WIDE ? threadIdx.x : (lane & (G - 1));
  const int rpw = WIDE ? 1 : 64 / G;
  const int groups = WIDE ? 1 : 4;
  const int grp = WIDE ? 0 : threadIdx.x >> 6;
  const int C = p.C;
  const float invC = 1.f / (float)C;
  const T* ds_in = reinterpret_cast<const T*>(p.ds);
  const T* dh_in = reinterpret_cast<const T*>(p.dh);
  const T* x_in = reinterpret_cast<const T*>(p.x);
  const T* y_in = reinterpret_cast<const T*>(p.y);
  T* dx = reinterpret_cast<T*>(p.dx);
  T* dy = reinterpret_cast<T*>(p.dy);
  const bool has_pre = PRE && p.pre != kNormNone && dh_in != nullptr;
  const bool has_post = POST && p.post != kNormNone;
  const bool has_gate = MODE == kAll && p.gate_kind != kGateNone;

  float a_prew[PRE ? MAXCH : 1][V], a_preb[PRE ? MAXCH : 1][V], a_postw[POST ? MAXCH : 1][V], a_postb[POST ? MAXCH : 1][V],
      a_gate[MODE == kAll ? MAXCH : 1][V];
  auto clear = [&](auto& a) {
    for (auto& ak : a)
#pragma unroll
      for (int j = 0; j < V; ++j) ak[j] = 0.f;
  };
  clear(a_prew); clear(a_preb); clear(a_postw); clear(a_postb); clear(a_gate);

  // the lane's channels never change: their parameters stay in registers (chunks of a wide lane are read again per row)
  constexpr bool HOIST = MAXCH <= 2;
  constexpr int HM = HOIST ? MAXCH : 1;
  float pre_w[PRE ? HM : 1][V], post_w[POST ? HM : 1][V], post_b[MODE == kAll ? HM : 1][V], gate_v[MODE == kAll ? HM : 1][V];
  if constexpr (HOIST)
#pragma unroll
    for (int k = 0; k < MAXCH; ++k) {
      if constexpr (PRE) load_vec<V, VEC>(p.pre_w, gl + k * G, C, 1.f, pre_w[k]);
      if constexpr (POST) load_vec<V, VEC>(p.post_w, gl + k * G, C, 1.f, post_w[k]);
      if constexpr (MODE == kAll) load_vec<V, VEC>(p.post_b, gl + k * G, C, 0.f, post_b[k]);
      if constexpr (MODE == kAll) load_vec<V, VEC>(p.gate_kind == kGateChannel ? p.gate : nullptr, gl + k * G, C, 1.f, gate_v[k]);
    }
  struct Row {
    Vec16<T> ds[MAXCH], dh[PRE ? MAXCH : 1], x[PRE ? MAXCH : 1], y[MAXCH];
    float mean, rstd, ymean, yrstd, sc;
  };
  const auto request = [&](Row& r, long base, long hi) {
    const long row = base + (WIDE ? 0 : lane / G);
    const bool live = row < hi;
    const int Cr = live ? C : 0;                         // a dead row has no elements
    const long at = live ? row * C : 0;
    r.mean = r.rstd = r.ymean = r.yrstd = 0.f;
    r.sc = 1.f;
    if (live) {
      if (has_pre) { r.mean = p.pre_stat[row]; r.rstd = p.pre_stat[p.rows + row]; }
      if (has_post) { r.ymean = p.post_stat[row]; r.yrstd = p.post_stat[p.rows + row]; }
      if (MODE != kPreOnly && p.scale != nullptr) r.sc = p.scale[fdiv((uint32_t)row, by_sample)];
    }
#pragma unroll
    for (int k = 0; k < MAXCH; ++k) {
      if (ds_in != nullptr) r.ds[k] = load_chunk<T, VEC>(ds_in + at, gl + k * G, Cr);
      else r.ds[k].raw = make_uint4(0u, 0u, 0u, 0u);
      if constexpr (PRE)
        if (has_pre) {
          r.dh[k] = load_chunk<T, VEC>(dh_in + at, gl + k * G, Cr);
          r.x[k] = load_chunk<T, VEC>(x_in + at, gl + k * G, Cr);
        }
      if (y_in != nullptr) r.y[k] = load_chunk<T, VEC>(y_in + at, gl + k * G, Cr);
      else r.y[k].raw = make_uint4(0u, 0u, 0u, 0u);
    }
  };

  for (long u = blockIdx.x; u < units; u += gridDim.x) {
    // rows of this unit: a part of one sample where the gate is per sample, else a part of all rows
    long lo, hi;
    if (MODE == kAll && p.gate_kind == kGateSample) {
      const long n = u / splits, part = u - n * splits;
      lo = n * p.per_sample + part * unit_rows;
      hi = min(lo + unit_rows, (n + 1) * p.per_sample);
      if constexpr (HOIST && MODE == kAll)
#pragma unroll
        for (int k = 0; k < MAXCH; ++k) load_vec<V, VEC>(p.gate + n * C, gl + k * G, C, 1.f, gate_v[k]);
    } else {
      lo = u * unit_rows;
      hi = min(lo + unit_rows, p.rows);
    }
    // the next row is requested before this one is worked on: a workgroup waits for memory and for its sums in turn otherwise
    // (24 x 257 x 1280 fp32: 57 us against 42), where registers hold two rows without giving up residency
    constexpr bool AHEAD = MAXCH == 1 || (MAXCH == 2 && MODE != kAll);
    Row cur;
    if (AHEAD && lo + grp * rpw < hi) request(cur, lo + grp * rpw, hi);
    // (vmcnt(0): the compiler would otherwise place this wait in the loop, behind the next row's requests)
    if constexpr (AHEAD) __builtin_amdgcn_s_waitcnt(0x0f70);
    for (long base = lo + grp * rpw; base < hi; base += groups * rpw) {
      const long row = base + (WIDE ? 0 : lane / G);
      const bool live = row < hi;
      if constexpr (!AHEAD) request(cur, base, hi);
      Row next;
      if (AHEAD && base + groups * rpw < hi) request(next, base + groups * rpw, hi);
      const float sc = cur.sc, ymean = cur.ymean, yrstd = cur.yrstd;
      const float* gate = p.gate;
      if (!HOIST && p.gate_kind == kGateSample) gate += (long)fdiv((uint32_t)(live ? row : 0), by_sample) * C;
      // parameters of chunk k
      const auto param = [&](const float* from, const float (&kept)[V], int k, float absent, float (&r)[V]) {
        if constexpr (HOIST) {
#pragma unroll
          for (int j = 0; j < V; ++j) r[j] = kept[j];
        } else {
          load_vec<V, VEC>(from, gl + k * G, C, absent, r);
        }
      };
      float g[MAXCH][V];
#pragma unroll
      for (int k = 0; k < MAXCH; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) g[k][j] = cur.ds[k].get(j);
      if constexpr (PRE)
      if (has_pre) {
        const float mean = cur.mean, rstd = cur.rstd;
        float m[2] = {0.f, 0.f};
        float sh[MAXCH][V];
#pragma unroll
        for (int k = 0; k < MAXCH; ++k) {
          float w[V], f[V], pw[V], pb[V];
          param(p.pre_w, pre_w[HOIST ? k : 0], k, 1.f, w);
          if constexpr (MODE == kAll) {
            param(gate, gate_v[HOIST ? k : 0], k, 1.f, f);
            if (has_post) {
              param(p.post_w, post_w[HOIST ? k : 0], k, 1.f, pw);
              param(p.post_b, post_b[HOIST ? k : 0], k, 0.f, pb);
            }
          }
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float z = cur.y[k].get(j);
            if (MODE == kAll) {
              if (has_post) z = (z - ymean) * yrstd * pw[j] + pb[j];
              z *= sc * f[j];
            }
            const float d = cur.dh[k].get(j), gw = d * w[j];      // absent: d = 0
            sh[k][j] = (cur.x[k].get(j) + z - mean) * rstd;
            m[0] += gw;
            m[1] += gw * sh[k][j];
            a_prew[k][j] += d * sh[k][j];
            a_preb[k][j] += d;
          }
        }
        gsum.run(m, G);
        const float m0 = p.pre == kNormLayer ? m[0] * invC : 0.f, m1 = m[1] * invC;
#pragma unroll
        for (int k = 0; k < MAXCH; ++k) {
          float w[V];
          param(p.pre_w, pre_w[HOIST ? k : 0], k, 1.f, w);
#pragma unroll
          for (int j = 0; j < V; ++j) g[k][j] += rstd * (cur.dh[k].get(j) * w[j] - m0 - sh[k][j] * m1);
        }
      }
      // the results are stored at the end of the row's work, behind the wait for the next row (stores count in it)
      Vec16<T> odx[MAXCH], ody[MAXCH];
#pragma unroll
      for (int k = 0; k < MAXCH; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) odx[k].set(j, g[k][j]);
      if (dy != nullptr) {
        float m[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < MAXCH; ++k) {
          const int c0 = (gl + k * G) * V;
          float gt[V], w[V], b[V];
          if constexpr (MODE == kAll) param(gate, gate_v[HOIST ? k : 0], k, 1.f, gt);
          if constexpr (POST)
            if (has_post) param(p.post_w, post_w[HOIST ? k : 0], k, 1.f, w);
          if constexpr (MODE == kAll)
            if (has_post && has_gate) param(p.post_b, post_b[HOIST ? k : 0], k, 0.f, b);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const bool ok = live && (VEC ? c0 < C : c0 + j < C);
            const float dzs = ok ? sc * g[k][j] : 0.f;
            const float yj = cur.y[k].get(j);
            const float yh = has_post ? (yj - ymean) * yrstd : yj;
            if constexpr (MODE == kAll)
              if (has_gate && ok) a_gate[k][j] += dzs * (has_post ? yh * w[j] + b[j] : yh);
            float dz = MODE == kAll && has_gate ? dzs * gt[j] : dzs;
            if constexpr (POST)
              if (has_post) {
                if (ok) {
                  a_postw[k][j] += dz * yh;
                  a_postb[k][j] += dz;
                }
                dz *= w[j];
                m[0] += dz;
                m[1] += dz * yh;
              }
            g[k][j] = dz;
          }
        }
        if (has_post) {
          gsum.run(m, G);
          const float m0 = p.post == kNormLayer ? m[0] * invC : 0.f, m1 = m[1] * invC;
#pragma unroll
          for (int k = 0; k < MAXCH; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j)
              g[k][j] = yrstd * (g[k][j] - m0 - (cur.y[k].get(j) - ymean) * yrstd * m1);
        }
#pragma unroll
        for (int k = 0; k < MAXCH; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) ody[k].set(j, g[k][j]);
      }
      if constexpr (AHEAD) {
        __builtin_amdgcn_s_waitcnt(0x0f70);
        cur = next;
      }
      if (live) {
        if (dx != nullptr)
#pragma unroll
          for (int k = 0; k < MAXCH; ++k) store_chunk<T, VEC>(odx[k], dx + row * C, gl + k * G, C);
        if (dy != nullptr)
#pragma unroll
          for (int k = 0; k < MAXCH; ++k) store_chunk<T, VEC>(ody[k], dy + row * C, gl + k * G, C);
      }
    }
    if constexpr (MODE == kAll)
      if (p.gate_kind == kGateSample && p.gate_partial != nullptr) {
        merge_out<T, MAXCH, WIDE, VEC>(a_gate, p.gate_partial + u * C, lds, gl, G, C);
        clear(a_gate);
      }
  }
  if (p.partial == nullptr) return;
  float* part = p.partial + (long)blockIdx.x * 5 * C;
  if constexpr (PRE) {
    if (p.out[0] != nullptr) merge_out<T, MAXCH, WIDE, VEC>(a_prew, part, lds, gl, G, C);
    if (p.out[1] != nullptr) merge_out<T, MAXCH, WIDE, VEC>(a_preb, part + C, lds, gl, G, C);
  }
  if constexpr (POST) {
    if (p.out[2] != nullptr) merge_out<T, MAXCH, WIDE, VEC>(a_postw, part + 2 * C, lds, gl, G, C);
    if (p.out[3] != nullptr) merge_out<T, MAXCH, WIDE, VEC>(a_postb, part + 3 * C, lds, gl, G, C);
  }
  if constexpr (MODE == kAll)
    if (p.out[4] != nullptr) merge_out<T, MAXCH, WIDE, VEC>(a_gate, part + 4 * C, lds, gl, G, C);
}

// out[v][c] = beta * out + sum over the partial rows, in a fixed order: workgroups of 16 columns x 64 part lanes, all reads of
// a lane in flight; behind them, for the samples' gates, the sum over the few splits of a sample: 64 columns x 16 lanes
struct FoldArgs {
  const float* partial; long nparts, part_stride;
  float* out[5]; float beta[5];
  const float* gate_partial; float* dgate; int splits;
  int C, which[5], of_vector, of_sample;      // workgroups of one vector, of one sample's gate
  long vectors;                               // workgroups of all vectors
};
template <int COLS> __device__ __forceinline__ void fold(const FoldArgs& a, long part, long tile, bool vector, float* red) {
  constexpr int LANES = 1024 / COLS, S = COLS + 1;
  const int cl = threadIdx.x % COLS, pl = threadIdx.x / COLS;
  const long c = tile * COLS + cl;
  const int v = vector ? a.which[part] : 0;
  const float* src = vector ? a.partial + (long)v * a.C + c : a.gate_partial + part * a.splits * a.C + c;
  const long stride = vector ? a.part_stride : a.C, parts = vector ? a.nparts : a.splits;
  float t = 0.f;
  if (c < a.C)
    for (long q = pl; q < parts; q += 8 * LANES) {
      float r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = q + i * LANES < parts ? src[(q + i * LANES) * stride] : 0.f;
      t += ((r[0] + r[1]) + (r[2] + r[3])) + ((r[4] + r[5]) + (r[6] + r[7]));
    }
  red[pl * S + cl] = t;
  __syncthreads();
  if (pl < 8) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < LANES / 8; ++i) t += red[(pl * (LANES / 8) + i) * S + cl];
  }
  __syncthreads();
  if (pl < 8) red[pl * S + cl] = t;
  __syncthreads();
  if (pl == 0 && c < a.C) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += red[i * S + cl];
    float* out = vector ? a.out[v] + c : a.dgate + part * a.C + c;
    *out = vector && a.beta[v] != 0.f ? sum + a.beta[v] * *out : sum;
  }
}
__global__ __launch_bounds__(1024) void residual_norm_fold_kernel(const FoldArgs a) {
  __shared__ float red[64 * 17];
  const long b = blockIdx.x;
  if (b < a.vectors) fold<16>(a, b / a.of_vector, b % a.of_vector, true, red);
  else fold<64>(a, (b - a.vectors) / a.of_sample, (b - a.vectors) % a.of_sample, false, red);
}

struct Units {
  long units, unit_rows;
  int splits;
  unsigned blocks;
};
// `parts`: how many workgroups the card holds at once.  With that many, 256 and 768, the pass with its fold, us: 64 x 197 x 1024
// bf16 (512 fit) 27 : 28 : 32, 64 x 3136 x 96 bf16 29 : 52 : 30, 24 x 257 x 1280 fp32 47 : 75 : 47
Units units_of(long rows, long per_sample, const Plan& pl, long parts, int gate_kind) {
  Units u;
  const long trip = pl.rows_per_trip;
  if (gate_kind == kGateSample) {
    const long samples = rows / per_sample;
    long splits = (parts + samples - 1) / samples;
    const long most = (per_sample + trip - 1) / trip;
    if (splits > most) splits = most;
    u.unit_rows = (per_sample + splits - 1) / splits;
    u.unit_rows = (u.unit_rows + trip - 1) / trip * trip;
    u.splits = (int)((per_sample + u.unit_rows - 1) / u.unit_rows);
    u.units = samples * u.splits;
    u.blocks = (unsigned)(u.units < parts ? u.units : parts);
  } else {
    long blocks = (rows + trip - 1) / trip;
    if (blocks > parts) blocks = parts;
    u.unit_rows = (rows + blocks - 1) / blocks;
    u.unit_rows = (u.unit_rows + trip - 1) / trip * trip;
    u.units = (rows + u.unit_rows - 1) / u.unit_rows;
    u.splits = 1;
    u.blocks = (unsigned)u.units;
  }
  return u;
}

template <typename T, int MAXCH, bool WIDE> using Kernel = void (*)(ResidualNormBwd, int, long, long, int, FastDiv);
template <typename T, int MAXCH, bool WIDE> Kernel<T, MAXCH, WIDE> kernel_of(bool vec, int mode) {
  if (!vec) return residual_norm_bwd_kernel<T, MAXCH, WIDE, false, kAll>;
  if (mode == kPreOnly) return residual_norm_bwd_kernel<T, MAXCH, WIDE, true, kPreOnly>;
  if (mode == kPostOnly) return residual_norm_bwd_kernel<T, MAXCH, WIDE, true, kPostOnly>;
  return residual_norm_bwd_kernel<T, MAXCH, WIDE, true, kAll>;
}
// workgroups that the card holds at once; asked for once for each kernel and size of workgroup
template <typename T, int MAXCH, bool WIDE> long resident(bool vec, int mode, int threads) {
  static std::atomic<int> known[4][9];
  std::atomic<int>& k = known[vec ? mode : 3][threads / 64];
  int n = k.load(std::memory_order_relaxed);
  if (n == 0) {
    DPA_CHECK_HIP(hipOccupancyMaxActiveBlocksPerMultiprocessor(
        &n, reinterpret_cast<const void*>(kernel_of<T, MAXCH, WIDE>(vec, mode)), threads, 0));
    if (n < 1) n = 1;
    k.store(n, std::memory_order_relaxed);
  }
  const long all = (long)n * kCompute;
  return all < kMaxParts ? all : kMaxParts;
}

// f(type, chunks a lane, wide) for the row's layout
#define DPA_RN_LAYOUT(pl, dtype, ...)                                                                              \
  DPA_DISPATCH_DTYPE(dtype, {                                                                                      \
    if (!(pl).wide && (pl).maxch == 1) { constexpr int MAXCH = 1; constexpr bool WIDE = false; __VA_ARGS__; }      \
    else if (!(pl).wide) { constexpr int MAXCH = 2; constexpr bool WIDE = false; __VA_ARGS__; }                    \
    else if ((pl).maxch == 1) { constexpr int MAXCH = 1; constexpr bool WIDE = true; __VA_ARGS__; }                \
    else if ((pl).maxch == 2) { constexpr int MAXCH = 2; constexpr bool WIDE = true; __VA_ARGS__; }                \
    else { constexpr int MAXCH = 4; constexpr bool WIDE = true; __VA_ARGS__; }                                     \
  })

struct Pick {
  Plan pl;
  bool vec;
  int mode;
  Units u;
};
Pick pick(const ResidualNormBwd& p, int dtype) {
  if (p.rows <= 0 || p.per_sample <= 0) throw std::invalid_argument("residual_norm: empty shape");
  if (p.rows >= (1l << 31)) throw std::invalid_argument("residual_norm: at most 2^31 - 1 rows");
  const int vecn = dtype == kF32 ? 4 : 8;
  if (p.C <= 0 || (p.C + vecn - 1) / vecn > kResidualNormMaxChunks)
    throw std::invalid_argument("residual_norm: C must be 1 .. 2048 16-byte chunks");
  Pick k;
  k.pl = plan(p.C, vecn);
  auto off16 = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) != 0; };
  k.vec = p.C % vecn == 0 && !(off16(p.ds) || off16(p.dh) || off16(p.x) || off16(p.y) || off16(p.dx) || off16(p.dy) ||
                               off16(p.post_w) || off16(p.post_b) || off16(p.pre_w) || off16(p.gate));
  const bool plain = p.post == kNormNone && p.gate_kind == kGateNone && p.scale == nullptr;
  k.mode = plain ? kPreOnly : (p.pre == kNormNone && p.gate_kind == kGateNone && p.post != kNormNone ? kPostOnly : kAll);
  if (plain && p.dy != nullptr) throw std::invalid_argument("residual_norm: without a branch of its own dy is dx");
  long parts = 0;
  DPA_RN_LAYOUT(k.pl, dtype, (parts = resident<T, MAXCH, WIDE>(k.vec, k.mode, k.pl.threads)));
  k.u = units_of(p.rows, p.per_sample, k.pl, parts, p.gate_kind);
  return k;
}

}  // namespace

long residual_norm_parts(const ResidualNormBwd& p, int dtype, long* splits) {
  const Pick k = pick(p, dtype);
  *splits = k.u.splits;
  return k.u.blocks;
}

void residual_norm_bwd_launch(const ResidualNormBwd& p, int dtype, hipStream_t s) {
  if (p.rows <= 0) return;
  const Pick k = pick(p, dtype);
  const Units& u = k.u;
  const FastDiv by_sample = make_fastdiv((uint32_t)p.per_sample);
  DPA_RN_LAYOUT(k.pl, dtype, hipLaunchKernelGGL((kernel_of<T, MAXCH, WIDE>(k.vec, k.mode)), dim3(u.blocks), dim3(k.pl.threads), 0, s, p,
                                                k.pl.G, u.units, u.unit_rows, u.splits, by_sample));
  DPA_CHECK_HIP(hipGetLastError());
  FoldArgs f{};
  f.partial = p.partial;
  f.nparts = u.blocks;
  f.part_stride = 5l * p.C;
  f.C = p.C;
  f.of_vector = (p.C + 15) / 16;
  f.of_sample = (p.C + 63) / 64;
  for (int v = 0; v < 5; ++v) {
    f.out[v] = p.out[v];
    f.beta[v] = p.beta[v];
    if (p.out[v] != nullptr) f.which[f.vectors++] = v;
  }
  f.vectors *= f.of_vector;
  f.gate_partial = p.gate_partial;
  f.dgate = p.dgate_sample;
  f.splits = u.splits;
  const bool gates = p.gate_kind == kGateSample && p.dgate_sample != nullptr;
  const long all = f.vectors + (gates ? p.rows / p.per_sample * f.of_sample : 0);
  if (all >= (1l << 31)) throw std::invalid_argument("residual_norm: too many gates");
  if (all == 0) return;
  hipLaunchKernelGGL(residual_norm_fold_kernel, dim3((unsigned)all), dim3(1024), 0, s, f);
  DPA_CHECK_HIP(hipGetLastError());
}

}  // namespace dpa
