// Log probability of one given class (token) per row of logits, the entropy of the row, its k most probable classes, and
// their joint gradient (gfx950).  With m = max z, S = sum e^(z - m), U = sum (z - m) e^(z - m):
//
//     logprob = (z_t - m) - log S,   H = log S - U / S,   top_j = (z_(j) - m) - log S
//     dz_v = p_v (-g_lp - sum_j g_top_j - g_H (log p_v + H)) + [v = t] g_lp + sum_j [v = idx_j] g_top_j
//
// A masked class (-inf) has probability zero and adds nothing; a row that is masked altogether has entropy 0, log
// probabilities -inf and no gradient.  A target outside the row is ignored (log probability 0).  S and U come from ONE pass
// with a running maximum per lane.  The k largest: every lane knows the largest element that it saw; the k-th largest of
// those lane maxima is a bound that at least k elements of the row reach, and few more do; a second look at the row (from
// cache) collects them into LDS, and a count of larger ones ranks them.  Elements are compared as 64-bit keys
// (order-preserving value bits, then the lower index), so ties go to the lowest index and the result does not depend on the
// order of collection.  If more than the list's capacity reach the bound (many large elements with one lane), the k-th
// largest collected becomes the new bound and the row is looked at again.  Few long rows are split over workgroups and
// joined.  Bound by memory bandwidth and the exponentials' issue rate together: 2048 x 50257 bf16 with k = 20 63 us with inputs
// from memory (3.3 TB/s), 84 behind a backward pass's writes; backward 80 us (5.2 TB/s); 1024 x 1000 fp32 9 + 6 us; one row of
// 128000 fp32 10 us and 5 to join, bound by latency.
#include "../common.h"
#include "transformer.h"

namespace dpa {
namespace {

constexpr int kCap = 1024;         // candidates of one look

// elements of one part of a row, whole chunks
__host__ __device__ __forceinline__ long part_of(long C, int splits) { return ((C + splits - 1) / splits + 7) & ~7l; }

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

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// running maximum m, S and U relative to it.  m starts at the lowest finite value: a masked class is then exp(-inf) = 0
// without a case of its own
constexpr float kLowest = -3.402823466e38f;
struct RunSums {
  float m, s, u;
  __device__ __forceinline__ void clear() { m = kLowest; s = u = 0.f; }
  __device__ __forceinline__ void raise(float to) {
    if (to > m) {
      if (s != 0.f) {               // also where s is NaN
        const float d = m - to, f = exp_of(d);
        u = f == 0.f ? 0.f : (u + d * s) * f;        // (d * s may have left the range where f is 0)
        s *= f;
      }
      m = to;
    }
  }
  __device__ __forceinline__ void add(float z) {
    const float d = z - m, e = exp_of(d);
    s += e;
    u += fmaxf(d, kLowest) * e;     // (-inf times 0 would be NaN; a NaN comes through e)
  }
  __device__ __forceinline__ void join(float m2, float s2, float u2) {
    raise(m2);
    if (s2 != 0.f) {
      const float d = m2 - m, f = d == 0.f ? 1.f : exp_of(d);
      s += s2 * f;
      u += f == 0.f ? 0.f : (d == 0.f ? u2 : (u2 + d * s2)) * f;
    }
  }
  // all 64 lanes' sums, the same in every lane
  __device__ __forceinline__ void join_wave() {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64), u2 = __shfl_xor(u, o, 64);
      join(m2, s2, u2);
    }
  }
};

// 16 bytes at any element boundary (a row of an odd number of classes starts anywhere; the hardware takes unaligned vectors)
template <typename T> __device__ __forceinline__ Vec16<T> load_any(const T* p) {
  Vec16<T> v;
  __builtin_memcpy(&v.raw, p, 16);
  return v;
}
typedef uint32_t any128 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> __device__ __forceinline__ void store_any(const Vec16<T>& v, T* p) {
  const any128 x = {v.raw.x, v.raw.y, v.raw.z, v.raw.w};
  *reinterpret_cast<any128*>(p) = x;
}

template <typename T> __device__ __forceinline__ float chunk_max(const Vec16<T>& v) {
  float mx = v.get(0);
#pragma unroll
  for (int j = 1; j < Vec16<T>::N; ++j) mx = fmaxf(mx, v.get(j));
  return mx;
}
// chunk q of a row's elements [lo, hi), lo a multiple of a chunk; -inf behind the end.  A lane takes every blockDim-th chunk
// whatever the row's alignment: results do not depend on it
template <typename T> __device__ __forceinline__ Vec16<T> load_chunk(const T* z, int c, int hi) {
  if (c + Vec16<T>::N <= hi) return load_any(z + c);
  Vec16<T> v;
#pragma unroll
  for (int j = 0; j < Vec16<T>::N; ++j) v.set(j, c + j < hi ? to_float(z[c + j]) : -INFINITY);
  return v;
}

// f(chunk, first column) for the lane's chunks of [lo, hi), four requested at a time
template <typename T, int TH, typename F>
__device__ __forceinline__ void walk(const T* z, int lo, int hi, F f) {
  constexpr int V = Vec16<T>::N, U = 4, kStep = TH * V;
  int c = lo + (int)threadIdx.x * V;
  for (; c + (U - 1) * kStep + V <= hi; c += U * kStep) {
    Vec16<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load_any(z + c + u * kStep);
#pragma unroll
    for (int u = 0; u < U; ++u) f(v[u], c + u * kStep);
  }
  for (; c < hi; c += kStep) f(load_chunk(z, c, hi), c);
}

template <int TH> struct TopShared {
  uint64_t best[TH];
  uint64_t cand[kCap];
  uint64_t bound;
  int count;
  int lanes, lane[8];              // lanes whose chunks are all looked at again
};

// how many of keys[0 .. n) are larger than `mine`: sixteen reads in flight (one after the other, each waits for LDS: a count
// over 256 keys took 3.6 us); keys has whole sixteens of room
__device__ __forceinline__ int count_larger(const uint64_t* keys, int n, uint64_t mine) {
  int r = 0, j = 0;
  for (; j + 16 <= n; j += 16) {
    uint64_t v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) v[u] = keys[j + u];
#pragma unroll
    for (int u = 0; u < 16; ++u) r += v[u] > mine ? 1 : 0;
  }
  if (j < n) {
    uint64_t v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) v[u] = keys[j + u];
#pragma unroll
    for (int u = 0; u < 16; ++u) r += (v[u] > mine) & (j + u < n) ? 1 : 0;
  }
  return r;
}

// A bound that at least k of the TH keys reach, and kSlack more at most; 0 if fewer than k are there.  One wave builds it
// bit by bit from ballots, the value's bits, then (among equal values) the index's, until few enough keys reach it
constexpr int kSlack = 16;
template <int TH> __device__ __forceinline__ void kth_bound(const uint64_t* keys, int k, uint64_t* bound) {
  constexpr int U = TH / 64;
  uint32_t hi[U], lo[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t key = keys[threadIdx.x + 64 * u];
    hi[u] = (uint32_t)(key >> 32);
    lo[u] = (uint32_t)key;
  }
  // a word that `need` of the words reach, and kSlack more at most (`enough`), else the largest such
  const auto search = [&](const uint32_t (&w)[U], int need, bool& enough) {
    uint32_t at = 0;
    enough = false;
    for (uint32_t bit = 0x80000000u; bit != 0 && !enough; bit >>= 1) {
      const uint32_t t = at | bit;
      int reach = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) reach += __popcll(__ballot(w[u] >= t));
      if (reach >= need) {
        at = t;
        enough = reach <= need + kSlack;
      }
    }
    return at;
  };
  bool enough;
  const uint32_t value = search(hi, k, enough);
  uint32_t index = 0;
  if (value != 0 && !enough) {
    int larger = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      larger += __popcll(__ballot(hi[u] > value));
      lo[u] = hi[u] == value ? lo[u] : 0;
    }
    index = search(lo, k - larger, enough);
  }
  if (threadIdx.x == 0) *bound = (uint64_t)value << 32 | index;
}

// keys of the candidates in descending order: out[r] for r < k (0 where there are fewer)
__device__ __forceinline__ void rank_out(const uint64_t* cand, int n, int k, uint64_t* out) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const uint64_t mine = cand[i];
    const int r = count_larger(cand, n, mine);
    if (r < k) out[r] = mine;
  }
  for (int i = n + threadIdx.x; i < k; i += blockDim.x) out[i] = 0;
}

// The k largest keys in descending order to out (LDS or global).  `best`: the largest key that this lane has seen;
// `each(least, f)`, called by the whole workgroup, calls f(chunk, first column) for all chunks with an element that is not below
// `least`, and others at will; `hi`: end of the row.  `plain`: there is no NaN, so a chunk whose largest element is below the
// bound has nothing to offer (fmaxf passes over NaN)
template <typename T, int TH, typename E>
__device__ __forceinline__ void top_of(int k, int hi, uint64_t best, bool plain, TopShared<TH>& sh, uint64_t* out, E each) {
  sh.best[threadIdx.x] = best;
  if (threadIdx.x == 0) {
    sh.bound = 0;
    sh.count = sh.lanes = 0;
  }
  __syncthreads();
  // with fewer than k lanes that saw anything the bound is 0 and every element is a candidate (few, then)
  if constexpr (TH == 64) {
    if (best != 0 && count_larger(sh.best, TH, best) == k - 1) sh.bound = best;
  } else {
    if (threadIdx.x < 64) kth_bound<TH>(sh.best, k, &sh.bound);
  }
  __syncthreads();
  for (;;) {
    const uint64_t bound = sh.bound;
    const float least = plain && bound != 0 ? order_value((uint32_t)(bound >> 32)) : -INFINITY;
    each(least, [&](const Vec16<T>& v, int c) {
      if (chunk_max(v) < least) return;
      uint32_t take = 0;
#pragma unroll
      for (int j = 0; j < Vec16<T>::N; ++j)
        if (make_key(v.get(j), c + j) >= bound && c + j < hi) take |= 1u << j;
      if (take == 0) return;
      int at = atomicAdd(&sh.count, __popc(take));       // (one wait for LDS in place of one per element)
#pragma unroll
      for (int j = 0; j < Vec16<T>::N; ++j)
        if (take >> j & 1u) {
          if (at < kCap) sh.cand[at] = make_key(v.get(j), c + j);
          ++at;
        }
    });
    __syncthreads();
    const int n = sh.count;
    if (n <= kCap) {
      rank_out(sh.cand, n, k, out);
      return;
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.count = sh.lanes = 0;
    for (int i = threadIdx.x; i < kCap; i += TH) {
      const uint64_t mine = sh.cand[i];
      if (count_larger(sh.cand, kCap, mine) == k - 1) sh.bound = mine;
    }
    __syncthreads();
  }
}

// the row's results from its sums and (k > 0) its first keys
template <typename T>
__device__ __forceinline__ void write_row(const TokenLogprobs& p, long row, bool valid, float zt, const RunSums& a,
                                          const uint64_t* top) {
  const float ls = logf(a.s);
  const bool empty = a.s == 0.f;                   // every class is masked
  if (threadIdx.x == 0) {
    p.norm[2 * row] = a.m;
    p.norm[2 * row + 1] = ls;
    p.logprob[row] = valid ? (empty ? -INFINITY : (zt - a.m) - ls) : 0.f;
    p.entropy[row] = empty ? 0.f : ls - a.u / a.s;
  }
  for (int i = threadIdx.x; i < p.k; i += blockDim.x) {
    const uint64_t key = top[i];
    p.index[row * p.k + i] = key_index(key);
    p.top[row * p.k + i] = empty ? -INFINITY : (order_value((uint32_t)(key >> 32)) - a.m) - ls;
  }
}

// One workgroup of TH lanes per row, or per part of a row; a second look comes from cache.  (Keeping a row's chunks in registers
// from the first look cost more residency than it saved: 4457 x 15054 bf16 with k = 5 233 us against 67.)
template <typename T, int TH>
__global__ __launch_bounds__(TH) void token_logprobs_kernel(const TokenLogprobs p) {
  constexpr int V = Vec16<T>::N;
  __shared__ float wm[TH / 64], ws[TH / 64], wu[TH / 64];
  __shared__ TopShared<TH> sh;
  __shared__ uint64_t top[kTokenTopMax];
  const long row = blockIdx.x / p.splits;
  const int part = (int)(blockIdx.x - row * p.splits);
  const T* z = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  const long each = part_of(p.C, p.splits);
  const int lo = (int)min(part * each, p.C), hi = (int)min(lo + each, p.C);
  const int c0 = (int)lo + (int)threadIdx.x * V;
  const long t = p.target[row];                    // (early: two loads that follow each other)
  const bool valid = t >= 0 && t < p.C;
  const float zt = valid ? to_float(z[t]) : 0.f;
  RunSums a;
  a.clear();
  int where = c0;                                 // chunk with this lane's largest element
  // the lane's two largest chunk maxima, where they are, and the largest of its other chunks: the second look needs
  // two chunks of a lane at most, unless a third one reaches the bound as well
  float first = -INFINITY, second = -INFINITY, third = -INFINITY;
  int where2 = c0;
  walk<T, TH>(z, (int)lo, (int)hi, [&](const Vec16<T>& x, int c) {
    const float mx = chunk_max(x);
    if (mx > first) {
      third = second;
      second = first;
      where2 = where;
      first = mx;
      where = c;
    } else if (mx > second) {
      third = second;
      second = mx;
      where2 = c;
    } else {
      third = fmaxf(third, mx);
    }
    a.raise(mx);
#pragma unroll
    for (int j = 0; j < V; ++j) a.add(x.get(j));
  });
  // the lane's largest chunks again, on their way while the sums meet
  Vec16<T> b1, b2;
  if (p.k > 0 && c0 < hi) {
    b1 = load_chunk(z, where, hi);
    b2 = load_chunk(z, where2, hi);
  }
  // lanes, then waves, in a fixed order
  a.join_wave();
  if constexpr (TH > 64) {
    if ((threadIdx.x & 63) == 0) { const int w = threadIdx.x >> 6; wm[w] = a.m; ws[w] = a.s; wu[w] = a.u; }
    __syncthreads();
    a.clear();
    for (int w = 0; w < TH / 64; ++w) a.join(wm[w], ws[w], wu[w]);
  }
  if (p.k > 0) {
    uint64_t best = 0;
    if (c0 < hi) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (where + j < hi) {
          const uint64_t key = make_key(b1.get(j), where + j);
          best = key > best ? key : best;
        }
    }
    const bool plain = a.s == a.s;
    uint64_t* out = p.splits == 1 ? top : p.keys + (long)blockIdx.x * p.k;
    top_of<T, TH>(p.k, hi, best, plain, sh, out, [&](float least, auto f) {
      if (least == -INFINITY) {
        walk<T, TH>(z, (int)lo, (int)hi, f);
        return;
      }
      // a lane that walks its chunks alone keeps the workgroup waiting for all of their latencies: a few such lanes are
      // shared out, a chunk a lane
      const bool all = third >= least;
      if (all) {
        const int at = atomicAdd(&sh.lanes, 1);
        if (at < 8) sh.lane[at] = threadIdx.x;
      } else {
        if (first >= least) f(b1, where);
        if (second >= least) f(b2, where2);
      }
      __syncthreads();
      const int lanes = sh.lanes;
      if (lanes <= 8) {
        for (int i = 0; i < lanes; ++i)
          for (int c = lo + (sh.lane[i] + (int)threadIdx.x * TH) * V; c < hi; c += TH * TH * V) f(load_chunk(z, c, hi), c);
      } else if (all) {
        walk<T, TH>(z, (int)lo, (int)hi, f);
      }
    });
  }
  if (p.splits > 1) {
    if (threadIdx.x == 0) {
      float* st = p.stat + (long)blockIdx.x * 3;
      st[0] = a.m; st[1] = a.s; st[2] = a.u;
    }
    return;
  }
  __syncthreads();
  write_row<T>(p, row, valid, zt, a, top);
}

// joins the parts of a row: one workgroup per row.  The parts' lists are in descending order, so where m of them have a t-th
// key that reaches a bound, m t keys do: with m t >= k the m-th largest of the t-th keys is one.  Few more than k keys reach
// it, and only those are ranked.
constexpr int kJoin = 512, kParts = 32;
template <typename T>
__global__ __launch_bounds__(kJoin) void token_logprobs_join_kernel(const TokenLogprobs p) {
  __shared__ uint64_t keys[kParts * kTokenTopMax], cand[kParts * kTokenTopMax], bound;
  __shared__ uint64_t top[kTokenTopMax];
  __shared__ int count;
  const long row = blockIdx.x;
  const long t = p.target[row];                    // (early: two loads that follow each other)
  const bool valid = t >= 0 && t < p.C;
  const float zt = valid ? to_float(reinterpret_cast<const T*>(p.logits)[row * p.ld + t]) : 0.f;
  const int n = p.splits * p.k;
  for (int i = threadIdx.x; i < n; i += kJoin) keys[i] = p.keys[row * n + i];
  if (threadIdx.x == 0) count = 0;
  RunSums a;
  a.clear();
  const int lane = threadIdx.x & 63;               // (one part a lane)
  if (lane < p.splits) {
    const float* st = p.stat + (row * p.splits + lane) * 3;
    a.m = st[0]; a.s = st[1]; a.u = st[2];
  }
  a.join_wave();
  __syncthreads();
  // (an absent key, 0, is below all others and never among the first k of C >= k elements)
  if (p.k > 0) {
    const int depth = (p.k + p.splits - 1) / p.splits, m = (p.k + depth - 1) / depth;
    if ((int)threadIdx.x < p.splits) {
      const uint64_t mine = keys[threadIdx.x * p.k + depth - 1];
      int r = 0;                                   // (absent keys are equal: the lower part comes first)
#pragma unroll 8
      for (int q = 0; q < p.splits; ++q) {
        const uint64_t other = keys[q * p.k + depth - 1];
        r += other > mine || (other == mine && q < (int)threadIdx.x) ? 1 : 0;
      }
      if (r == m - 1) bound = mine;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kJoin)
      if (keys[i] >= bound) cand[atomicAdd(&count, 1)] = keys[i];
    __syncthreads();
    rank_out(cand, count, p.k, top);
  }
  __syncthreads();
  write_row<T>(p, row, valid, zt, a, top);
}

// One part of a row.  The elements that carry a gradient of their own (the target and the k listed ones) are few: the pass
// writes all elements without them, and a lane each then writes those again.  (Looking for them in the pass, by a bit per 8
// columns, made it a fifth longer for 2048 x 50257 bf16 with k = 20: nearly every row has waves that stop for them.)
template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(const TokenLogprobsBwd p, const int splits) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ long idx[kTokenTopMax + 1];
  __shared__ float gx[kTokenTopMax + 1];
  const long row = blockIdx.x / splits;
  const int part = (int)(blockIdx.x - row * splits);
  const T* z = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  T* dz = reinterpret_cast<T*>(p.dlogits) + row * p.C;
  const long each = part_of(p.C, splits);
  const int lo = (int)min(part * each, p.C), hi = (int)min(lo + each, p.C);
  const float m = p.norm[2 * row], ls = p.norm[2 * row + 1], H = p.entropy[row];
  const long t = p.target[row];
  const bool valid = t >= 0 && t < p.C;
  const float glp = p.d_logprob != nullptr && valid ? p.d_logprob[row] : 0.f;
  const float ge = p.d_entropy != nullptr ? p.d_entropy[row] : 0.f;
  const int k = p.d_top != nullptr ? p.k : 0, tid = threadIdx.x;
  long at = -1;                                    // this lane's own element
  if (tid <= k) {
    at = tid < k ? p.index[row * p.k + tid] : (valid ? t : -1);
    idx[tid] = at;
    gx[tid] = tid < k ? p.d_top[row * p.k + tid] : glp;
  }
  if (at < lo || at >= hi) at = -1;
  const float own = at >= 0 ? to_float(z[at]) : 0.f;
  __syncthreads();
  float gsum = glp;
  for (int j = 0; j < k; ++j) gsum += gx[j];
  const bool empty = ls == -INFINITY;              // a row that is masked altogether
  if (empty) {
    for (int i = lo + tid; i < hi; i += 256) dz[i] = from_float<T>(0.f);
    return;
  }
  // p (-gsum - ge (log p + H)) with log p = d - ls, d = z - m.  Below -128 p is 0 (ls >= 0, and e^-104 is under the smallest
  // float): d stops there, so that its product with ge does not overflow beside a p of 0
  const float c0 = -gsum - ge * H + ge * ls, shift = -ls * kLog2e;
  const auto grad = [&](float v) {
    const float d = v - m;
    return __builtin_amdgcn_exp2f(fmaf(d, kLog2e, shift)) * fmaf(-ge, fmaxf(d, -128.f), c0);
  };
  const auto chunk = [&](const Vec16<T>& v) {
    Vec16<T> o;
#pragma unroll
    for (int j = 0; j < V; ++j) o.set(j, grad(v.get(j)));
    return o;
  };
  constexpr int U = 4, kStep = 256 * V;            // chunks in flight per lane
  int c = lo + tid * V;
  for (; c + (U - 1) * kStep + V <= hi; c += U * kStep) {
    Vec16<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load_any(z + c + u * kStep);
#pragma unroll
    for (int u = 0; u < U; ++u) store_any(chunk(v[u]), dz + c + u * kStep);
  }
  for (; c < hi; c += kStep) {
    const Vec16<T> o = chunk(load_chunk(z, c, hi));
    if (c + V <= hi) {
      store_any(o, dz + c);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < hi) dz[c + j] = from_float<T>(o.get(j));
    }
  }
  float g = grad(own);
  if (at >= 0)
    for (int j = 0; j <= k; ++j) {
      if (idx[j] != at) continue;
      g += gx[j];
      if (j < tid) at = -2;                        // (an element listed twice is written by the first lane that has it)
    }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the pass has written
  __syncthreads();
  if (at >= 0) dz[at] = from_float<T>(g);
}

void check(long N, long C, int k) {
  if (N < 0 || C <= 0 || C > (1l << 30)) throw std::invalid_argument("token_logprobs: 1 .. 2^30 classes");
  if (k < 0 || k > kTokenTopMax || k > C) throw std::invalid_argument("token_logprobs: k must be 0 .. min(64, classes)");
}

}  // namespace

// workgroups per row: enough of them for the card, of at least 2048 elements each.  A row below 8192 stays whole: the join costs
// more than the shorter parts save (one row of 4200 bf16, k = 5: 9.5 us whole, 12.0 in two; of 128000, k = 20: 18.7 in 16
// parts, 15.8 in 32)
int token_logprobs_splits(long N, long C) {
  long s = N <= 0 || C < 8192 ? 1 : 512 / N;
  if (s > C / 2048) s = C / 2048;
  if (s > kParts) s = kParts;
  return (int)(s < 1 ? 1 : s);
}

void token_logprobs_launch(const TokenLogprobs& p, int dtype, hipStream_t s) {
  check(p.N, p.C, p.k);
  if (p.N == 0) return;
  if (p.splits < 1 || p.splits > kParts || p.N * p.splits >= (1l << 31))
    throw std::invalid_argument("token_logprobs: splits");
  const long part = part_of(p.C, p.splits) < p.C ? part_of(p.C, p.splits) : p.C;
  const dim3 grid((unsigned)(p.N * p.splits));
  DPA_DISPATCH_DTYPE(dtype, {
    // as few waves a row as fill the card (4096 are resident), since a row's waves wait for each other at the end of each pass;
    // with 1, 2 or 4 waves, k = 5, us: 8192 x 4000 bf16 32 : 47 : 72, 2048 x 50257 bf16 50 : 47 : 53, 1024 x 16000 fp32
    // 22 : 19 : 19, 300 x 16000 fp32 19 : 16 : 13; 64 x 1000 bf16 7.1 : 7.5 : 7.9
    const long rows = p.N * p.splits, chunks = (part + Vec16<T>::N - 1) / Vec16<T>::N;
    if (rows >= 4096 || chunks <= 256) hipLaunchKernelGGL((token_logprobs_kernel<T, 64>), grid, dim3(64), 0, s, p);
    else if (rows >= 2048) hipLaunchKernelGGL((token_logprobs_kernel<T, 128>), grid, dim3(128), 0, s, p);
    else hipLaunchKernelGGL((token_logprobs_kernel<T, 256>), grid, dim3(256), 0, s, p);
    if (p.splits > 1) hipLaunchKernelGGL(token_logprobs_join_kernel<T>, dim3((unsigned)p.N), dim3(kJoin), 0, s, p);
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
