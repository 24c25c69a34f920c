// Log probability of one given class (token) per row of logits, the entropy of the row, its k most probable classes, and
// their joint gradient (gfx950).  With m = max z, S = sum e^(z - m), U = sum (z - m) e^(z - m):
//
//     logprob = (z_t - m) - log S,   H = log S - U / S,   top_j = (z_(j) - m) - log S
//     dz_v = p_v (-g_lp - sum_j g_top_j - g_H (log p_v + H)) + [v = t] g_lp + sum_j [v = idx_j] g_top_j
//
// A masked class (-inf) has probability zero and adds nothing; a row that is masked altogether has entropy 0, log
// probabilities -inf and no gradient.  A target outside the row is ignored (log probability 0).  S and U come from ONE pass with a running maximum per
// lane.  The k largest: every lane knows the largest element that it saw; the k-th largest of those lane maxima is a bound
// that at least k elements of the row reach, and few more do; a second look at the row (from cache) collects them into LDS,
// and a count of larger ones ranks them.  Elements are compared as 64-bit keys (order-preserving value bits, then the
// lower index), so ties go to the lowest index and the result does not depend on the order of collection.  If more than the
// list's capacity reach the bound (many large elements with one lane), the k-th largest collected becomes the new bound
// and the row is looked at again.  Few long rows are split over workgroups and joined.  Bound by memory bandwidth.
#include "../common.h"
#include "transformer.h"

namespace dpa {
namespace {

constexpr int kCap = 1024;         // candidates of one look

// order-preserving bits of a float as unsigned (-0 as +0); > 0 for everything but a NaN with the sign bit
__device__ __forceinline__ uint32_t order_bits(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
// larger value first, then lower index; 0 is no key
__device__ __forceinline__ uint64_t make_key(float z, long i) {
  return ((uint64_t)order_bits(z) << 32) | (uint64_t)(0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ long key_index(uint64_t k) { return (long)(0xffffffffu - (uint32_t)k); }

struct RunSums {                    // running maximum m, S and U relative to it
  float m, s, u;
  __device__ __forceinline__ void clear() { m = -INFINITY; s = u = 0.f; }
  __device__ __forceinline__ void raise(float to) {
    if (to > m) {
      const float d = m - to;
      if (s != 0.f) {               // also where s is NaN
        const float f = __expf(d);
        u = f == 0.f ? 0.f : (u + d * s) * f;        // (d * s may have left the range where f is 0)
        s *= f;
      }
      m = to;
    }
  }
  __device__ __forceinline__ void add(float z) {
    const float d = z - m, e = z == -INFINITY ? 0.f : __expf(d);
    s += e;
    u += z == -INFINITY ? 0.f : d * e;
  }
  __device__ __forceinline__ void join(float m2, float s2, float u2) {
    raise(m2);
    if (s2 != 0.f) {
      const float d = m2 - m, f = d == 0.f ? 1.f : __expf(d);
      s += s2 * f;
      u += f == 0.f ? 0.f : (d == 0.f ? u2 : (u2 + d * s2)) * f;
    }
  }
};

// 16 bytes at any element boundary (a row of an odd number of classes starts anywhere; the hardware takes unaligned vectors)
template <typename T> __device__ __forceinline__ Vec16<T> load_any(const T* p) {
  Vec16<T> v;
  __builtin_memcpy(&v.raw, p, 16);
  return v;
}
template <typename T> __device__ __forceinline__ void store_any(const Vec16<T>& v, T* p) { __builtin_memcpy(p, &v.raw, 16); }

// elements [lo, hi) of a row, lo a multiple of a chunk: a lane takes every 256th chunk of 16 bytes, whatever the row's
// alignment (results do not depend on it).  F(z, i) sees one element, M(largest of the next few) comes before them
template <typename T, typename F, typename M>
__device__ __forceinline__ void scan_row(const T* z, long lo, long hi, F f, M before) {
  constexpr int V = 16 / (int)sizeof(T);
  for (long c = lo + (long)threadIdx.x * V; c < hi; c += (long)blockDim.x * V) {
    if (c + V <= hi) {
      const Vec16<T> v = load_any(z + c);
      float mx = v.get(0);
#pragma unroll
      for (int j = 1; j < V; ++j) mx = fmaxf(mx, v.get(j));
      before(mx);
#pragma unroll
      for (int j = 0; j < V; ++j) f(v.get(j), c + j);
    } else {
      for (long i = c; i < hi; ++i) {
        const float v = to_float(z[i]);
        before(v);
        f(v, i);
      }
    }
  }
}

struct TopShared {
  uint64_t best[256];
  uint64_t cand[kCap];
  uint64_t bound;
  int count;
};

// the k largest of the candidates, by the count of larger ones, to out[0 .. k) (0 where there are fewer)
__device__ __forceinline__ void rank_out(const TopShared& sh, int n, int k, uint64_t* out) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const uint64_t mine = sh.cand[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += sh.cand[j] > mine ? 1 : 0;
    if (r < k) out[r] = mine;
  }
  for (int i = n + threadIdx.x; i < k; i += blockDim.x) out[i] = 0;
}

// the k largest keys of [lo, hi) in descending order to out (LDS or global); `best`: this lane's largest key
template <typename T>
__device__ __forceinline__ void top_of(const T* z, long lo, long hi, int k, uint64_t best, TopShared& sh, uint64_t* out) {
  sh.best[threadIdx.x] = best;
  if (threadIdx.x == 0) { sh.bound = 0; sh.count = 0; }
  __syncthreads();
  {
    int r = 0;
    for (int j = 0; j < 256; ++j) r += sh.best[j] > best ? 1 : 0;
    // with fewer than k lanes that saw anything the bound stays 0 and every element is a candidate (few, then)
    if (best != 0 && r == k - 1) sh.bound = best;
  }
  __syncthreads();
  for (;;) {
    const uint64_t bound = sh.bound;
    scan_row(z, lo, hi, [&](float v, long i) {
      const uint64_t key = make_key(v, i);
      if (key >= bound) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kCap) sh.cand[at] = key;
      }
    }, [](float) {});
    __syncthreads();
    const int n = sh.count;
    if (n <= kCap) {
      rank_out(sh, n, k, out);
      return;
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    for (int i = threadIdx.x; i < kCap; i += blockDim.x) {
      const uint64_t mine = sh.cand[i];
      int r = 0;
      for (int j = 0; j < kCap; ++j) r += sh.cand[j] > mine ? 1 : 0;
      if (r == k - 1) sh.bound = mine;
    }
    __syncthreads();
  }
}

__device__ __forceinline__ void write_row(const TokenLogprobs& p, long row, const RunSums& a, float zt, bool valid) {
  const float ls = logf(a.s);
  const bool empty = a.s == 0.f;                   // every class is masked
  p.norm[2 * row] = a.m;
  p.norm[2 * row + 1] = ls;
  p.logprob[row] = valid ? (empty ? -INFINITY : (zt - a.m) - ls) : 0.f;
  p.entropy[row] = empty ? 0.f : ls - a.u / a.s;
}

template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_kernel(const TokenLogprobs p) {
  __shared__ float wm[4], ws[4], wu[4];
  __shared__ TopShared sh;
  __shared__ uint64_t top[kTokenTopMax];
  const long row = blockIdx.x / p.splits;
  const int part = (int)(blockIdx.x - row * p.splits);
  const T* z = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  const long each = ((p.C + p.splits - 1) / p.splits + 7) & ~7l;
  const long lo = min(part * each, p.C), hi = min(lo + each, p.C);
  RunSums a;
  a.clear();
  uint64_t best = 0;
  scan_row(z, lo, hi,
           [&](float v, long i) {
             a.add(v);
             const uint64_t key = make_key(v, i);
             best = key > best ? key : best;
           },
           [&](float mx) { a.raise(mx); });
  // lanes, then waves, in a fixed order
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(a.m, o, 64), s2 = __shfl_xor(a.s, o, 64), u2 = __shfl_xor(a.u, o, 64);
    a.join(m2, s2, u2);
  }
  if ((threadIdx.x & 63) == 0) { const int w = threadIdx.x >> 6; wm[w] = a.m; ws[w] = a.s; wu[w] = a.u; }
  __syncthreads();
  a.clear();
  for (int w = 0; w < 4; ++w) a.join(wm[w], ws[w], wu[w]);
  if (p.k > 0) top_of(z, lo, hi, p.k, best, sh, p.splits == 1 ? top : p.keys + (long)blockIdx.x * p.k);
  if (p.splits > 1) {
    if (threadIdx.x == 0) {
      float* st = p.stat + (long)blockIdx.x * 3;
      st[0] = a.m; st[1] = a.s; st[2] = a.u;
    }
    return;
  }
  __syncthreads();
  const long t = p.target[row];
  const bool valid = t >= 0 && t < p.C;
  if (threadIdx.x == 0) write_row(p, row, a, valid ? to_float(z[t]) : 0.f, valid);
  const float ls = logf(a.s);
  if ((int)threadIdx.x < p.k) {
    const uint64_t key = top[threadIdx.x];
    p.index[row * p.k + threadIdx.x] = key_index(key);
    p.top[row * p.k + threadIdx.x] = a.s == 0.f ? -INFINITY : (order_value((uint32_t)(key >> 32)) - a.m) - ls;
  }
}

// joins the parts of a row: one workgroup per row
template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_join_kernel(const TokenLogprobs p) {
  __shared__ TopShared sh;
  __shared__ uint64_t top[kTokenTopMax];
  const long row = blockIdx.x;
  const T* z = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  RunSums a;
  a.clear();
  for (int q = 0; q < p.splits; ++q) {
    const float* st = p.stat + (row * p.splits + q) * 3;
    a.join(st[0], st[1], st[2]);
  }
  if (p.k > 0) {
    // splits * k keys, at most kCap (token_logprobs_splits)
    const int n = p.splits * p.k;
    for (int i = threadIdx.x; i < n; i += 256) sh.cand[i] = p.keys[row * n + i];
    __syncthreads();
    // an absent key (0) is below all others and never among the first k of C >= k elements
    for (int i = threadIdx.x; i < n; i += 256) {
      const uint64_t mine = sh.cand[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += sh.cand[j] > mine ? 1 : 0;
      if (mine != 0 && r < p.k) top[r] = mine;
    }
    __syncthreads();
  }
  const long t = p.target[row];
  const bool valid = t >= 0 && t < p.C;
  if (threadIdx.x == 0) write_row(p, row, a, valid ? to_float(z[t]) : 0.f, valid);
  const float ls = logf(a.s);
  if ((int)threadIdx.x < p.k) {
    const uint64_t key = top[threadIdx.x];
    p.index[row * p.k + threadIdx.x] = key_index(key);
    p.top[row * p.k + threadIdx.x] = a.s == 0.f ? -INFINITY : (order_value((uint32_t)(key >> 32)) - a.m) - ls;
  }
}

// one part of a row; elements that carry a gradient of their own are found through a bit per 8 columns
template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(const TokenLogprobsBwd p, const int splits) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ uint32_t marked[1024];
  __shared__ long idx[kTokenTopMax + 1];
  __shared__ float gx[kTokenTopMax + 1];
  const long row = blockIdx.x / splits;
  const int part = (int)(blockIdx.x - row * splits);
  const T* z = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  T* dz = reinterpret_cast<T*>(p.dlogits) + row * p.C;
  const long each = ((p.C + splits - 1) / splits + 7) & ~7l;
  const long lo = min(part * each, p.C), hi = min(lo + each, p.C);
  for (int i = threadIdx.x; i < 1024; i += 256) marked[i] = 0;
  const long t = p.target[row];
  const bool valid = t >= 0 && t < p.C;
  const float glp = p.d_logprob != nullptr && valid ? p.d_logprob[row] : 0.f;
  const float ge = p.d_entropy != nullptr ? p.d_entropy[row] : 0.f;
  const int k = p.d_top != nullptr ? p.k : 0;
  if ((int)threadIdx.x < k) {
    idx[threadIdx.x] = p.index[row * p.k + threadIdx.x];
    gx[threadIdx.x] = p.d_top[row * p.k + threadIdx.x];
  }
  if (threadIdx.x == 255) { idx[k] = valid ? t : -1; gx[k] = glp; }
  __syncthreads();
  float gsum = glp;
  for (int j = 0; j < k; ++j) gsum += gx[j];
  if ((int)threadIdx.x <= k && idx[threadIdx.x] >= 0) {
    const uint32_t bit = (uint32_t)((idx[threadIdx.x] >> 3) & 32767);
    atomicOr(&marked[bit >> 5], 1u << (bit & 31));
  }
  __syncthreads();
  const float m = p.norm[2 * row], ls = p.norm[2 * row + 1], H = p.entropy[row];
  const bool empty = ls == -INFINITY;
  auto grad = [&](float v, long i) {
    if (empty) return 0.f;
    const float logp = (v - m) - ls, pr = __expf(logp);
    float g = -pr * gsum;
    if (ge != 0.f) g -= v == -INFINITY ? 0.f : ge * pr * (logp + H);
    const uint32_t bit = (uint32_t)((i >> 3) & 32767);
    if ((marked[bit >> 5] >> (bit & 31)) & 1u)
      for (int j = 0; j <= k; ++j) g += idx[j] == i ? gx[j] : 0.f;
    return g;
  };
  for (long c = lo + (long)threadIdx.x * V; c < hi; c += 256 * V) {
    if (c + V <= hi) {
      const Vec16<T> v = load_any(z + c);
      Vec16<T> o;
#pragma unroll
      for (int j = 0; j < V; ++j) o.set(j, grad(v.get(j), c + j));
      store_any(o, dz + c);
    } else {
      for (long i = c; i < hi; ++i) dz[i] = from_float<T>(grad(to_float(z[i]), i));
    }
  }
}

void check(long N, long C, int k) {
  if (N < 0 || C <= 0 || C >= (1l << 31)) throw std::invalid_argument("token_logprobs: 1 .. 2^31 - 1 classes");
  if (k < 0 || k > kTokenTopMax || k > C) throw std::invalid_argument("token_logprobs: k must be 0 .. min(64, classes)");
}

}  // namespace

// workgroups per row: enough of them for the card, at least 4096 elements each, and (with k <= 64) kCap keys to join
int token_logprobs_splits(long N, long C, int) {
  long s = N <= 0 ? 1 : 512 / N;
  if (s > C / 4096) s = C / 4096;
  if (s > kCap / kTokenTopMax) s = kCap / kTokenTopMax;
  return (int)(s < 1 ? 1 : s);
}

void token_logprobs_launch(const TokenLogprobs& p, int dtype, hipStream_t s) {
  check(p.N, p.C, p.k);
  if (p.N == 0) return;
  if (p.splits < 1 || p.splits * p.k > kCap || p.N * p.splits >= (1l << 31))
    throw std::invalid_argument("token_logprobs: splits");
  DPA_DISPATCH_DTYPE(dtype, {
    hipLaunchKernelGGL(token_logprobs_kernel<T>, dim3((unsigned)(p.N * p.splits)), dim3(256), 0, s, p);
    if (p.splits > 1) hipLaunchKernelGGL(token_logprobs_join_kernel<T>, dim3((unsigned)p.N), dim3(256), 0, s, p);
  });
  DPA_CHECK_HIP(hipGetLastError());
}

void token_logprobs_bwd_launch(const TokenLogprobsBwd& p, int dtype, hipStream_t s) {
  check(p.N, p.C, p.k);
  if (p.N == 0) return;
  long splits = 2048 / p.N;
  if (splits > p.C / 4096) splits = p.C / 4096;
  if (splits < 1) splits = 1;
  if (p.N * splits >= (1l << 31)) throw std::invalid_argument("token_logprobs: too many rows");
  DPA_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL(token_logprobs_bwd_kernel<T>, dim3((unsigned)(p.N * splits)), dim3(256), 0, s, p,
                                               (int)splits));
  DPA_CHECK_HIP(hipGetLastError());
}

}  // namespace dpa
