// Newton-Schulz orthogonalisation of a batch of matrices (gfx950):  X = G / (|G|_F + eps) (transposed where it has more
// rows than columns), then `steps` times
//
//     A = X X^T,   B = b A + c A A,   X = a X + B X
//
// on the fp16 matrix cores.  Values are held times 2^10 (singular values stay below ~4, so nothing leaves the fp16 range,
// and the scale keeps small entries clear of the subnormals) in fp16 planes: `hi`, and `lo` with what hi leaves, together
// 22 significant bits.
//
//  * PAIR (whatever the caller's type): every operand is hi + lo and a product is hi hi + hi lo + lo hi in fp32
//    accumulators, 32-bit products at three times the cost of one fp16 product; fp32's own matrix rate is 1 / 16 of fp16's.
//    A bf16 result is the 32-bit one, rounded once.
//  * single (bf16 results of a caller who asks for it, `fast`): products take the hi planes alone, a third of the cost, and
//    11 significant bits.  What keeps the error (2e-4 .. 7e-4 of the result's norm, 2e-3 where a few directions are 100
//    times the rest) below the rounding of the result (1.7e-3): X itself stays hi + lo (with one plane: 5e-3 to 2e-2 there),
//    and the diagonals of A and B, which are near 1 and -2.7 and would be rounded as such (1.4e-3 to 1.8e-3 by
//    themselves), are kept apart in fp32; with A = Ao + Da,
//        A A = Ao Ao + (Da_i + Da_j) Ao_ij + Da^2,   a X + B X = (a + Db_i) X_ij + Bo X.
//
// A and B are symmetric: only tiles on and below the diagonal are computed.  X is also kept transposed, because B X needs
// it with m contiguous.  Dimensions are padded to whole tiles with zeros, which every product preserves.
//
// Two product kernels (ns_use_large has the rule and its measurements):
//  * 256 x 256 tiles, 8 waves: the half-tile ring of the framework's large GEMM (gemm8.hip has the ordering argument),
//    bound by the matrix cores; the epilogue moves whole 128-byte row pieces through the free ring.  24 x 1024 x 4096, a
//    step: A 322 us (0.96 PFLOP/s of fp16 products), B 105 us, X 681 us (0.91 PFLOP/s beside 1.6 GB of planes); `fast`:
//    A 120 us (0.86 PFLOP/s), B 47 us, X 360 us (0.57 PFLOP/s beside 1.2 GB).
//  * 64 x 64 and 128 x 128 tiles: for matrices too small or too few to fill the card with the large ones; bound by latency
//    and by the L2's rate.  6 x 256 x 2304 fp32, a step: A 10 + 5 us (parts and their join), B 8 us, X 18 us.
#include "../common.h"
#include "transformer.h"
#include <type_traits>

namespace dpa {
namespace {

typedef __attribute__((address_space(3))) void* lds_void_ptr;
typedef const __attribute__((address_space(1))) void* gbl_void_ptr;

constexpr float kScale = 1024.f, kInvScale = 1.f / 1024.f;
constexpr int kNormParts = 64;

struct Half2 { _Float16 hi, lo; };
__device__ __forceinline__ Half2 split(float x) {
  Half2 h;
  h.hi = (_Float16)x;
  h.lo = (_Float16)(x - (float)h.hi);
  return h;
}
__device__ __forceinline__ uint32_t pack(_Float16 a, _Float16 b) {
  uint16_t x, y;
  __builtin_memcpy(&x, &a, 2);
  __builtin_memcpy(&y, &b, 2);
  return (uint32_t)x | ((uint32_t)y << 16);
}

// Two registers' 16-bit halves (r in the low half, r + 1 in the high one) of neighbouring lanes, traded so that an even lane
// has register r of itself and its neighbour and an odd lane register r + 1 of both
__device__ __forceinline__ uint32_t trade_pair(uint32_t both, bool odd) {
  const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)both, 0xB1, 0xf, 0xf, true);      // lanes 1 0 3 2
  return odd ? (other >> 16) | (both & 0xffff0000u) : (both & 0xffffu) | (other << 16);
}

// ---- |G|_F^2 in 64 bits: kNormParts partial sums a matrix
template <typename T>
__global__ __launch_bounds__(256) void ns_norm_kernel(const T* __restrict__ g, long elems, double* __restrict__ parts) {
  __shared__ double red[4];
  const T* p = g + blockIdx.y * elems;
  const long each = (elems + kNormParts - 1) / kNormParts;
  const long lo = min((long)blockIdx.x * each, elems), hi = min(lo + each, elems);
  double t = 0.0;
  constexpr int V = Vec16<T>::N;
  if (((elems * sizeof(T)) & 15) == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0) {      // whole chunks everywhere
    const long chunks = elems / V, mine = (chunks + kNormParts - 1) / kNormParts;
    const long c0 = min((long)blockIdx.x * mine, chunks), c1 = min(c0 + mine, chunks);
    for (long c = c0 + threadIdx.x; c < c1; c += 256) {
      Vec16<T> v;
      v.load(p + c * V);
      // (eight squares in 32 bits would overflow or vanish where 64 do not)
#pragma unroll
      for (int j = 0; j < V; ++j) t += (double)v.get(j) * (double)v.get(j);
    }
  } else {
    for (long i = lo + threadIdx.x; i < hi; i += 256) {
      const double v = (double)to_float(p[i]);
      t += v * v;
    }
  }
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) parts[(long)blockIdx.y * kNormParts + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// a matrix of fp16 planes: rows of ld elements, `next` elements from one matrix of the batch to the next
struct Planes {
  _Float16* hi; _Float16* lo;
  long ld, next;
};

// ---- planes of X and X^T, 64 x 64 elements of the normalised matrix (zeros in the padding)
template <typename T>
__global__ __launch_bounds__(256) void ns_split_kernel(const T* __restrict__ g, long rows, long cols, int turned, double eps,
                                                       const double* __restrict__ parts, const Planes x, const Planes xt) {
  __shared__ float tile[64][65];
  __shared__ float inv_s;
  const long b = blockIdx.z;
  if (threadIdx.x < kNormParts) {            // one wave
    double t = parts[b * kNormParts + threadIdx.x];
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
    if (threadIdx.x == 0) inv_s = (float)(1.0 / (sqrt(t) + eps));
  }
  __syncthreads();
  const float inv = inv_s;
  const long i0 = (long)blockIdx.y * 64, j0 = (long)blockIdx.x * 64;     // in X
  const T* p = g + b * rows * cols;
  constexpr int V = Vec16<T>::N;
  if (cols % V == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0) {     // rows of whole chunks
    for (int e = threadIdx.x; e < 4096 / V; e += 256) {
      const int r = e / (64 / V), c = e % (64 / V) * V;
      const long gr = (turned ? j0 : i0) + r, gc = (turned ? i0 : j0) + c;
      Vec16<T> v;
      v.raw = make_uint4(0u, 0u, 0u, 0u);
      if (gr < rows && gc < cols) v.load(p + gr * cols + gc);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        const float f = v.get(q) * inv * kScale;
        if (turned) tile[c + q][r] = f;
        else tile[r][c + q] = f;
      }
    }
  } else
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int r = e >> 6, c = e & 63;                                    // of G's tile
    const long gr = (turned ? j0 : i0) + r, gc = (turned ? i0 : j0) + c;
    const float v = gr < rows && gc < cols ? to_float(p[gr * cols + gc]) * inv * kScale : 0.f;
    if (turned) tile[c][r] = v;
    else tile[r][c] = v;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 512; e += 256) {
    const int r = e >> 3, u = (e & 7) * 8;
    f16x8_t h, l;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const Half2 v = split(tile[r][u + q]);
      h[q] = v.hi; l[q] = v.lo;
    }
    long o = b * x.next + (i0 + r) * x.ld + j0 + u;
    *reinterpret_cast<f16x8_t*>(x.hi + o) = h;
    *reinterpret_cast<f16x8_t*>(x.lo + o) = l;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const Half2 v = split(tile[u + q][r]);
      h[q] = v.hi; l[q] = v.lo;
    }
    o = b * xt.next + (j0 + r) * xt.ld + i0 + u;
    *reinterpret_cast<f16x8_t*>(xt.hi + o) = h;
    if (xt.lo != nullptr) *reinterpret_cast<f16x8_t*>(xt.lo + o) = l;
  }
}

// ---- products: P Q^T on planes with the contraction contiguous, and what becomes of it
enum Op : int { kGram = 0, kPoly = 1, kApply = 2, kFinal = 3 };
struct Product {
  Planes P, Q, R, out, out_t;               // R: added term; out: result, out_t: its transpose (lo may be null)
  float* diag;                              // kGram: Da (written), kPoly and kApply: read (Da, Db)
  float* diag_out;                          // kPoly: Db
  void* fin;                                // kFinal: the result in the caller's type and orientation
  long diag_next, fin_next;
  int mt, nt, ktiles, turned;               // tiles; slices of 128 bytes of a row
  long rows, cols;                          // of the caller's matrix
  float c0, c1;                             // kPoly: b, c; kApply, kFinal: a, -
  int splits; float* partial;               // kGram on 64 x 64 tiles: the contraction split over workgroups,
};                                          // [tile][split][4096] sums

// which tile of which matrix
struct Place { long b; int ti, tj; };
template <int OP> __device__ __forceinline__ Place place_of(const Product& p, uint32_t per_matrix, uint32_t lid) {
  Place q;
  q.b = lid / per_matrix;
  const uint32_t t = lid - (uint32_t)q.b * per_matrix;
  if constexpr (OP == kGram || OP == kPoly) {                 // on and below the diagonal
    q.ti = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((uint32_t)(q.ti + 1) * (q.ti + 2) / 2 <= t) ++q.ti;
    while ((uint32_t)q.ti * (q.ti + 1) / 2 > t) --q.ti;
    q.tj = (int)(t - (uint32_t)q.ti * (q.ti + 1) / 2);
  } else {
    q.ti = (int)(t % (uint32_t)p.mt);
    q.tj = (int)(t / (uint32_t)p.mt);
  }
  return q;
}

// element (i, j) of the result from the accumulated product, in the scale of the planes; r = R(i, j)
template <int OP> __device__ __forceinline__ float combine(float acc, float r, float di, float dj, float c0, float c1) {
  if constexpr (OP == kGram) return acc * kInvScale;
  else if constexpr (OP == kPoly) return c0 * r + c1 * (acc * kInvScale + (di + dj) * r);
  else return (c0 + di) * r + acc * kInvScale;
}
// the diagonal element's true value
template <int OP> __device__ __forceinline__ float on_diagonal(float acc, float di, float c0, float c1) {
  if constexpr (OP == kGram) return acc * kInvScale * kInvScale;
  else return c0 * di + c1 * (acc * kInvScale * kInvScale + di * di);
}

// ================================================================================ 64 x 64 tiles
constexpr int kSmall = 64;

// products of one 32 x 32 block over one K slice.  The terms go to accumulators of their own: a chain on one of them
// would wait for each product's full latency, and few waves are there to fill in
template <bool PAIR> __device__ __forceinline__ void slice_mma(f32x16_t (&acc)[2], const f16x8_t (&q)[4], const f16x8_t (&f)[4]) {
  if constexpr (PAIR) {                     // [k16 step * 2 + plane]
    acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q[0], f[0], acc[0], 0, 0, 0);
    acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q[1], f[0], acc[1], 0, 0, 0);
    acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q[2], f[2], acc[0], 0, 0, 0);
    acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q[0], f[1], acc[1], 0, 0, 0);
    acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q[3], f[2], acc[0], 0, 0, 0);
    acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q[2], f[3], acc[1], 0, 0, 0);
  } else {
#pragma unroll
    for (int s = 0; s < 4; ++s) acc[s & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q[s], f[s], acc[s & 1], 0, 0, 0);
  }
}

// what becomes of four neighbouring sums, elements (i, j .. j + 3); `diag_tile`: on the diagonal of a symmetric result
template <int OP, typename T>
__device__ __forceinline__ void quad_epilogue(const Product& p, long b, long i, long j, bool diag_tile, float di,
                                              const float (&sum)[4]) {
  constexpr bool SYM = OP == kGram || OP == kPoly;
  float v[4];
  float r[4] = {0.f, 0.f, 0.f, 0.f};
  if constexpr (OP != kGram) {
    const long o = b * p.R.next + i * p.R.ld + j;
    _Float16 h[4];
    uint2 raw = *reinterpret_cast<const uint2*>(p.R.hi + o);
    __builtin_memcpy(h, &raw, 8);
#pragma unroll
    for (int q = 0; q < 4; ++q) r[q] = (float)h[q];
    if (p.R.lo != nullptr) {
      raw = *reinterpret_cast<const uint2*>(p.R.lo + o);
      __builtin_memcpy(h, &raw, 8);
#pragma unroll
      for (int q = 0; q < 4; ++q) r[q] += (float)h[q];
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float dj = OP == kPoly ? p.diag[b * p.diag_next + j + q] : 0.f;
    v[q] = combine<OP>(sum[q], r[q], di, dj, p.c0, p.c1);
    if constexpr (SYM)
      if (i == j + q) {
        (OP == kGram ? p.diag : p.diag_out)[b * p.diag_next + i] = on_diagonal<OP>(sum[q], di, p.c0, p.c1);
        v[q] = 0.f;
      }
  }
  if constexpr (OP == kFinal) {
    T* f = reinterpret_cast<T*>(p.fin) + b * p.fin_next;
    T t[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) t[q] = from_float<T>(v[q] * kInvScale);
    if (!p.turned && p.cols % 4 == 0 && (reinterpret_cast<uintptr_t>(p.fin) & 15) == 0) {      // four columns at once
      if (i < p.rows && j < p.cols) __builtin_memcpy(__builtin_assume_aligned(f + i * p.cols + j, 4 * sizeof(T)), t, 4 * sizeof(T));
      return;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const long row = p.turned ? j + q : i, col = p.turned ? i : j + q;
      if (row < p.rows && col < p.cols) f[row * p.cols + col] = t[q];
    }
  } else {
    Half2 h[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) h[q] = split(v[q]);
    const long o = b * p.out.next + i * p.out.ld + j;
    *reinterpret_cast<uint2*>(p.out.hi + o) = make_uint2(pack(h[0].hi, h[1].hi), pack(h[2].hi, h[3].hi));
    if (p.out.lo != nullptr) *reinterpret_cast<uint2*>(p.out.lo + o) = make_uint2(pack(h[0].lo, h[1].lo), pack(h[2].lo, h[3].lo));
    if (!SYM || !diag_tile) {
      const long t = b * p.out_t.next + j * p.out_t.ld + i;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        p.out_t.hi[t + q * p.out_t.ld] = h[q].hi;
        if (p.out_t.lo != nullptr) p.out_t.lo[t + q * p.out_t.ld] = h[q].lo;
      }
    }
  }
}

// a wave's sums on a 64 x 64 tile: half of the registers of its 32 x 32 quarter
template <int OP, typename T>
__device__ __forceinline__ void small_epilogue(const Product& p, const Place& at, int wave, int lane, const float (&sum)[8]) {
  const int kg = wave >> 2, wr = (wave >> 1) & 1, wc = wave & 1, l31 = lane & 31, lh = lane >> 5;
  const long i = (long)at.ti * kSmall + wr * 32 + l31;
  const float di = OP == kGram ? 0.f : p.diag[at.b * p.diag_next + i];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float four[4] = {sum[g * 4], sum[g * 4 + 1], sum[g * 4 + 2], sum[g * 4 + 3]};
    quad_epilogue<OP, T>(p, at.b, i, (long)at.tj * kSmall + wc * 32 + 16 * kg + 8 * g + 4 * lh, at.ti == at.tj, di, four);
  }
}

// 8 waves: two groups of four take turns at the K slices (a wave's reads, waits and products follow each other; the other
// group's fill in), each wave a 32 x 32 quarter of the tile.  RING slices of LDS, RING - 2 in flight.
template <bool PAIR, int OP, typename T, int RING>
__global__ __launch_bounds__(512) void ns_small_kernel(const Product p, const uint32_t per_matrix) {
  constexpr int kSlice = 2 * kSmall * 128;  // bytes
  __shared__ __attribute__((aligned(16))) unsigned char smem[RING * kSlice];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = wave >> 2, wr = (wave >> 1) & 1, wc = wave & 1, l31 = lane & 31, lh = lane >> 5;
  uint32_t lid = xcd_remap(blockIdx.x, gridDim.x);           // a matrix's tiles share an XCD's L2
  int first = 0, nk = p.ktiles, part = 0;
  if constexpr (OP == kGram)
    if (p.splits > 1) {
      part = (int)(lid % (uint32_t)p.splits);
      lid /= (uint32_t)p.splits;
      const int each = (p.ktiles + p.splits - 1) / p.splits;
      first = part * each;
      nk = max(min(first + each, p.ktiles) - first, 0);       // (the last parts can be empty: they stage a slice, unused)
      first = min(first, p.ktiles - 1);
    }
  const Place at = place_of<OP>(p, per_matrix, lid);
  const long b = at.b, i0 = (long)at.ti * kSmall, j0 = (long)at.tj * kSmall;
  // staging, two slices a round: instruction q of wave w of a group covers rows (w * 2 + q) * 8 + lane / 8 of the group's
  // slice; LDS chunk lane % 8 holds source chunk (lane % 8) ^ ((row >> 1) & 7), so that 16 rows of a fragment read touch 16
  // different 16-byte columns.  PAIR: chunks 0 .. 3 are 32 elements of hi, 4 .. 7 the same of lo
  const _Float16* src[2][2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int row = ((wave & 3) * 2 + q) * 8 + (lane >> 3);
    const int ch = (lane & 7) ^ ((row >> 1) & 7);
    const _Float16* hp = PAIR && ch >= 4 ? p.P.lo : p.P.hi;
    const _Float16* hq = PAIR && ch >= 4 ? p.Q.lo : p.Q.hi;
    const int k = (PAIR ? ch & 3 : ch) * 8 + first * (PAIR ? 32 : 64);
    src[0][q] = hp + b * p.P.next + (i0 + row) * p.P.ld + k;
    src[1][q] = hq + b * p.Q.next + (j0 + row) * p.Q.ld + k;
  }
  auto stage = [&](int k) {                 // this group's slice; always four loads, behind the last slice of the last one
    unsigned char* dst = smem + (k % RING) * kSlice + (wave & 3) * 2048;
    const long o = (long)max(min(k, nk - 1), 0) * (PAIR ? 32 : 64);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      __builtin_amdgcn_global_load_lds((gbl_void_ptr)(src[0][q] + o), (lds_void_ptr)(dst + q * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((gbl_void_ptr)(src[1][q] + o), (lds_void_ptr)(dst + kSmall * 128 + q * 1024), 16, 0, 0);
    }
  };
  f32x16_t acc[2];
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[0][r] = acc[1][r] = 0.f;
  // a wave requests RING / 2 - 1 of its group's slices ahead, four loads each, and one more per round: when round k is
  // waited for, the newer ones may stay in flight
  const int rounds = (nk + 1) / 2;
#pragma unroll
  for (int r = 0; r < RING / 2 - 1; ++r) stage(2 * r + kg);
  for (int r = 0; r < rounds; ++r) {
    if constexpr (RING == 8) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();           // round r has landed for every wave; round r - 1 has been read by all ...
    asm volatile("" ::: "memory");
    stage(2 * (r + RING / 2 - 1) + kg);     // ... and its slots are free
    const int k = 2 * r + kg;
    const unsigned char* base = smem + (k % RING) * kSlice;
    if (k < nk) {
      f16x8_t fp[4], fq[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        // PAIR: c = k16 step * 2 + plane, else the k16 step
        const int ch = (PAIR ? (c & 1) * 4 + (c >> 1) * 2 + lh : c * 2 + lh) ^ ((l31 >> 1) & 7);
        fp[c] = *reinterpret_cast<const f16x8_t*>(base + (wr * 32 + l31) * 128 + ch * 16);
        fq[c] = *reinterpret_cast<const f16x8_t*>(base + kSmall * 128 + (wc * 32 + l31) * 128 + ch * 16);
      }
      slice_mma<PAIR>(acc, fq, fp);
    }
  }
  // the groups' sums meet: each finishes half of the registers (8 of 16) of its quarter
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      // (the requests behind the last slice, too)
  __syncthreads();
  float* swap = reinterpret_cast<float*>(smem);                     // [wave][8][64]
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    swap[(wave * 8 + r) * 64 + lane] = kg == 0 ? acc[0][8 + r] + acc[1][8 + r] : acc[0][r] + acc[1][r];
  }
  __syncthreads();
  float sum[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const float mine = kg == 0 ? acc[0][r] + acc[1][r] : acc[0][8 + r] + acc[1][8 + r];
    const float other = swap[((wave ^ 4) * 8 + r) * 64 + lane];
    sum[r] = kg == 0 ? mine + other : other + mine;
  }
  if constexpr (OP == kGram)
    if (p.splits > 1) {                     // ns_join_kernel goes on from here
      float* to = p.partial + ((long)lid * p.splits + part) * 4096 + wave * 512 + lane;
#pragma unroll
      for (int r = 0; r < 8; ++r) to[r * 64] = sum[r];
      return;
    }
  small_epilogue<OP, T>(p, at, wave, lane, sum);
}

// adds the parts of a tile in their order
template <typename T>
__global__ __launch_bounds__(512) void ns_join_kernel(const Product p, const uint32_t per_matrix) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at = place_of<kGram>(p, per_matrix, blockIdx.x);
  const float* from = p.partial + (long)blockIdx.x * p.splits * 4096 + wave * 512 + lane;
  float sum[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) sum[r] = from[r * 64];
  for (int q = 1; q < p.splits; ++q)
#pragma unroll
    for (int r = 0; r < 8; ++r) sum[r] += from[(long)q * 4096 + r * 64];
  small_epilogue<kGram, T>(p, at, wave, lane, sum);
}

// ================================================================================ 128 x 128 tiles
// X = a X + B X of small matrices: a contraction of a few slices over many tiles, bound by the traffic into LDS, of which
// a 64 x 64 tile takes twice as much.  8 waves of 64 x 32, a ring of four slices, three in flight.
constexpr int kMid = 128;

template <bool PAIR, int OP, typename T>
__global__ __launch_bounds__(512) void ns_mid_kernel(const Product p, const uint32_t per_matrix) {
  constexpr int kSlice = 2 * kMid * 128;
  __shared__ __attribute__((aligned(16))) unsigned char smem[4 * kSlice];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave >> 2, wc = wave & 3, l31 = lane & 31, lh = lane >> 5;
  const Place at = place_of<OP>(p, per_matrix, xcd_remap(blockIdx.x, gridDim.x));
  const long b = at.b, i0 = (long)at.ti * kMid, j0 = (long)at.tj * kMid;
  const _Float16* src[2][2];                 // instruction q of a wave: rows (wave * 2 + q) * 8 + lane / 8
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int row = (wave * 2 + q) * 8 + (lane >> 3);
    const int ch = (lane & 7) ^ ((row >> 1) & 7);
    const int k = (PAIR ? ch & 3 : ch) * 8;
    src[0][q] = (PAIR && ch >= 4 ? p.P.lo : p.P.hi) + b * p.P.next + (i0 + row) * p.P.ld + k;
    src[1][q] = (PAIR && ch >= 4 ? p.Q.lo : p.Q.hi) + b * p.Q.next + (j0 + row) * p.Q.ld + k;
  }
  const int nk = p.ktiles;
  auto stage = [&](int k) {                  // four loads a wave; behind the last slice the last one again
    unsigned char* dst = smem + (k & 3) * kSlice + wave * 2048;
    const long o = (long)min(k, nk - 1) * (PAIR ? 32 : 64);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      __builtin_amdgcn_global_load_lds((gbl_void_ptr)(src[0][q] + o), (lds_void_ptr)(dst + q * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((gbl_void_ptr)(src[1][q] + o), (lds_void_ptr)(dst + kMid * 128 + q * 1024), 16, 0, 0);
    }
  };
  f32x16_t acc[2][2];                        // [32-row block][accumulator]
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[x >> 1][x & 1][r] = 0.f;
  stage(0);
  stage(1);
  stage(2);
  for (int k = 0; k < nk; ++k) {
    // slices k .. k + 2 are requested: eight newer loads than slice k's may stay in flight
    asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();            // slice k has landed for every wave; slice k - 1 has been read by all ...
    asm volatile("" ::: "memory");
    stage(k + 3);                            // ... and its slot is free
    const unsigned char* base = smem + (k & 3) * kSlice;
    f16x8_t fp[2][4], fq[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int ch = (PAIR ? (c & 1) * 4 + (c >> 1) * 2 + lh : c * 2 + lh) ^ ((l31 >> 1) & 7);
      fq[c] = *reinterpret_cast<const f16x8_t*>(base + kMid * 128 + (wc * 32 + l31) * 128 + ch * 16);
#pragma unroll
      for (int m = 0; m < 2; ++m) fp[m][c] = *reinterpret_cast<const f16x8_t*>(base + (wr * 64 + m * 32 + l31) * 128 + ch * 16);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) slice_mma<PAIR>(acc[m], fq, fp[m]);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");       // (the requests behind the last slice, too)
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[m][0][r] += acc[m][1][r];
  if constexpr (OP == kFinal) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const long i = i0 + wr * 64 + m * 32 + l31;
      const float di = p.diag[b * p.diag_next + i];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float four[4] = {acc[m][0][g * 4], acc[m][0][g * 4 + 1], acc[m][0][g * 4 + 2], acc[m][0][g * 4 + 3]};
        quad_epilogue<OP, T>(p, b, i, j0 + wc * 32 + 8 * g + 4 * lh, false, di, four);
      }
    }
  } else {
    // whole row pieces through LDS, as in the large kernel: straight from registers a wave's 64 x 32 results are 16-byte
    // pieces of rows and 2-byte pieces of columns (22 us in place of 17 for 6 x 256 x 2304).  A wave's own 16 KiB: 64 rows of 64
    // bytes, or 32 rows of 128 for the transpose, 16-byte chunks swizzled
    __syncthreads();                         // every wave is past its last read of the ring
    unsigned char* my = smem + wave * 16384;
    const long mw = i0 + wr * 64, nw = j0 + wc * 32;
    const auto row_at = [](int row, int col) { return row * 64 + (((col >> 3) ^ ((row >> 1) & 3)) * 16) + (col & 7) * 2; };
    float di[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) di[m] = p.c0 + p.diag[b * p.diag_next + mw + m * 32 + l31];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[m][0][r] *= kInvScale;
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      const _Float16* R = (plane ? p.R.lo : p.R.hi) + b * p.R.next + mw * p.R.ld + nw;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int row = q * 16 + (lane >> 2);
        __builtin_amdgcn_global_load_lds((gbl_void_ptr)(R + row * p.R.ld + ((lane & 3) ^ ((row >> 1) & 3)) * 8),
                                         (lds_void_ptr)(my + plane * 4096 + q * 1024), 16, 0, 0);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int o = row_at(m * 32 + l31, 8 * g + 4 * lh);
        _Float16 h[4], l[4];
        __builtin_memcpy(h, my + o, 8);
        __builtin_memcpy(l, my + 4096 + o, 8);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[m][0][g * 4 + q] += di[m] * ((float)h[q] + (float)l[q]);
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    // hi rows, lo rows, hi of the transpose, lo of it: 4 KiB each
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const Half2 s0 = split(acc[m][0][r]), s1 = split(acc[m][0][r + 1]);
        const uint32_t hi = pack(s0.hi, s1.hi), lo = pack(s0.lo, s1.lo);
        const int row = m * 32 + l31, o = row_at(row, (r & 3) + 8 * (r >> 2) + 4 * lh);
        *reinterpret_cast<uint32_t*>(my + o) = hi;
        *reinterpret_cast<uint32_t*>(my + 4096 + o) = lo;
        const bool odd = lane & 1;
        const int n = ((r + (odd ? 1 : 0)) & 3) + 8 * (r >> 2) + 4 * lh, c = row & ~1;
        const int t = n * 128 + (((c >> 3) ^ (n & 7)) * 16) + (c & 7) * 2;
        *reinterpret_cast<uint32_t*>(my + 8192 + t) = trade_pair(hi, odd);
        if (PAIR) *reinterpret_cast<uint32_t*>(my + 12288 + t) = trade_pair(lo, odd);
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      _Float16* out = (plane ? p.out.lo : p.out.hi) + b * p.out.next + mw * p.out.ld + nw;
      _Float16* out_t = plane ? p.out_t.lo : p.out_t.hi;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int row = q * 16 + (lane >> 2), ck = lane & 3;
        *reinterpret_cast<uint4*>(out + row * p.out.ld + ck * 8) =
            *reinterpret_cast<const uint4*>(my + plane * 4096 + row * 64 + ((ck ^ ((row >> 1) & 3)) * 16));
        if (!PAIR && plane) continue;
        const int n = q * 8 + (lane >> 3), ct = lane & 7;
        *reinterpret_cast<uint4*>(out_t + b * p.out_t.next + (nw + n) * p.out_t.ld + mw + ct * 8) =
            *reinterpret_cast<const uint4*>(my + 8192 + plane * 4096 + n * 128 + ((ct ^ (n & 7)) * 16));
      }
    }
  }
}

// ================================================================================ 256 x 256 tiles
constexpr int kLarge = 256;
constexpr int kHalf = 128 * 128;            // bytes of a half-tile: 128 rows of a 128-byte slice
constexpr int kRing = 8 * kHalf;            // two K slices of P and Q

template <int OFF> __device__ __forceinline__ f16x8_t lds_read16(uint32_t addr) {
  uint4 r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(OFF));
  f16x8_t v;
  __builtin_memcpy(&v, &r, 16);
  return v;
}
// Makes the accumulators new values to the compiler: it would otherwise keep what one pass of the epilogue derived from
// them for the next one, and spill thousands of registers.
__device__ __forceinline__ void forget(f32x16_t (&acc)[2][2][2]) {
#pragma unroll
  for (int x = 0; x < 8; ++x) asm volatile("" : "+v"(acc[x >> 2][(x >> 1) & 1][x & 1]));
}
// where element (row, col) of a wave's 128 x 64 16-bit results lies in its 16 KiB
__device__ __forceinline__ int row_place(int row, int col) { return row * 128 + (((col >> 3) ^ (row & 7)) * 16) + (col & 7) * 2; }
// Puts registers r and r + 1 (16 bits each, the two halves of `both`) of lane row m into the transposed 64 x 128 layout:
// neighbouring lanes hold neighbouring columns of it and trade, so that each has two columns of one row (an even lane the
// row of register r, its neighbour that of r + 1)
__device__ __forceinline__ void to_transpose(unsigned char* my, uint32_t both, int m, int nq, int r, int lh) {
  const bool odd = m & 1;
  const uint32_t v = trade_pair(both, odd);
  const int n = nq * 32 + ((r + (odd ? 1 : 0)) & 3) + 8 * (r >> 2) + 4 * lh;
  *reinterpret_cast<uint32_t*>(my + n * 256 + ((((m & ~1) >> 3) ^ (n & 15)) * 16) + ((m & ~1) & 7) * 2) = v;
}
// products of one 32 x 32 block over one K slice
template <bool PAIR> __device__ __forceinline__ void block_mma(f32x16_t& acc, const f16x8_t (&q)[4], const f16x8_t (&f)[4]) {
  if constexpr (PAIR) {                     // [k16 step * 2 + plane]
#pragma unroll
    for (int s = 0; s < 4; s += 2) {
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(q[s], f[s], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(q[s + 1], f[s], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(q[s], f[s + 1], acc, 0, 0, 0);
    }
  } else {
#pragma unroll
    for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(q[s], f[s], acc, 0, 0, 0);
  }
}

template <bool PAIR, int OP, typename T>
__global__ __launch_bounds__(512, 1) void ns_large_kernel(const Product p, const uint32_t per_matrix) {
  __shared__ __attribute__((aligned(16))) unsigned char smem[kRing];
  constexpr bool SYM = OP == kGram || OP == kPoly;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave >> 2, wc = wave & 3;
  const int l31 = lane & 31, lh = lane >> 5;
  const Place at = place_of<OP>(p, per_matrix, xcd_remap(blockIdx.x, gridDim.x));
  const long b = at.b, m0 = (long)at.ti * kLarge, n0 = (long)at.tj * kLarge;
  const int nk = p.ktiles, nhalf = 4 * nk;

  // staging: wave-instruction i of this wave covers rows (wave * 2 + i) * 8 + lane / 8 of a half-tile; chunks swizzled as
  // in the small kernel.  Half-tile kinds: Q rows 0 .. 127, 128 .. 255, P rows 0 .. 127, 128 .. 255
  const _Float16* src[4][2];
#pragma unroll
  for (int h = 0; h < 4; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = (wave * 2 + i) * 8 + (lane >> 3);
      const int ch = (lane & 7) ^ ((row >> 1) & 7);
      const Planes& m = h >= 2 ? p.P : p.Q;
      const _Float16* base = PAIR && ch >= 4 ? m.lo : m.hi;
      src[h][i] = base + b * m.next + ((h >= 2 ? m0 : n0) + (h & 1) * 128 + row) * m.ld + (PAIR ? ch & 3 : ch) * 8;
    }
  auto stage = [&](int g, auto kind_c) {
    constexpr int h = decltype(kind_c)::value;
    unsigned char* dst = smem + (g & 7) * kHalf + wave * 2048;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      __builtin_amdgcn_global_load_lds((gbl_void_ptr)src[h][i], (lds_void_ptr)(dst + i * 1024), 16, 0, 0);
      src[h][i] += PAIR ? 32 : 64;
    }
  };
  constexpr std::integral_constant<int, 0> kB0{};
  constexpr std::integral_constant<int, 1> kB1{};
  constexpr std::integral_constant<int, 2> kA0{};
  constexpr std::integral_constant<int, 3> kA1{};

  const uint32_t lds0 = (uint32_t)(uintptr_t)((__attribute__((address_space(3))) unsigned char*)smem);
  uint32_t cA[4], cB[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int ch = PAIR ? (c & 1) * 4 + (c >> 1) * 2 + lh : c * 2 + lh;
    const uint32_t o = (uint32_t)((ch ^ ((l31 >> 1) & 7)) * 16) + (uint32_t)l31 * 128;
    cA[c] = lds0 + (2 + wr) * kHalf + o;
    cB[c] = lds0 + (wc >> 1) * kHalf + (wc & 1) * 8192 + o;
  }
  f32x16_t acc[2][2][2];                    // [mq][mt][nq]
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[x][y][z][r] = 0.f;

  // prologue: half-tiles 0 .. 4, K slice 0 complete (one half-tile may stay in flight)
  stage(0, kB0);
  stage(1, kB1);
  stage(2, kA0);
  stage(3, kA1);
  if (4 < nhalf) {
    stage(4, kB0);
    asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  __builtin_amdgcn_s_barrier();
  if (wr == 1) __builtin_amdgcn_s_barrier();          // this group runs one barrier behind

  f16x8_t fa[2][4], fb[2][4];               // P fragments of the current mq [mt], Q fragments [nq]
  for (int t = 0; t < nk; ++t) {
    const uint32_t tb = (uint32_t)(t & 1) * (4 * kHalf);
    const int g = 4 * t + 5;                // half-tile requested in phase 0 of this K slice
    // ---- phase 0: quadrant (m 0, n 0)
#pragma unroll
    for (int c = 0; c < 4; ++c) fb[0][c] = lds_read16<0>(cB[c] + tb);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      fa[0][c] = lds_read16<0>(cA[c] + tb);
      fa[1][c] = lds_read16<4096>(cA[c] + tb);
    }
    if (g < nhalf) stage(g, kB1);
    __builtin_amdgcn_s_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    block_mma<PAIR>(acc[0][0][0], fb[0], fa[0]);
    block_mma<PAIR>(acc[0][1][0], fb[0], fa[1]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_s_barrier();
    // ---- phase 1: quadrant (m 0, n 1)
#pragma unroll
    for (int c = 0; c < 4; ++c) fb[1][c] = lds_read16<4096>(cB[c] + tb);
    if (g + 1 < nhalf) stage(g + 1, kA0);
    __builtin_amdgcn_s_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    block_mma<PAIR>(acc[0][0][1], fb[1], fa[0]);
    block_mma<PAIR>(acc[0][1][1], fb[1], fa[1]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_s_barrier();
    // ---- phase 2: quadrant (m 1, n 1)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      fa[0][c] = lds_read16<8192>(cA[c] + tb);
      fa[1][c] = lds_read16<12288>(cA[c] + tb);
    }
    if (g + 2 < nhalf) stage(g + 2, kA1);
    __builtin_amdgcn_s_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    block_mma<PAIR>(acc[1][0][1], fb[1], fa[0]);
    block_mma<PAIR>(acc[1][1][1], fb[1], fa[1]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_s_barrier();
    // ---- phase 3: quadrant (m 1, n 0): operands are in registers; K slice t + 1 must have landed
    if (g + 3 < nhalf) {
      stage(g + 3, kB0);
      asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    block_mma<PAIR>(acc[1][0][0], fb[0], fa[0]);
    block_mma<PAIR>(acc[1][1][0], fb[0], fa[1]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_s_barrier();
  }
  if (wr == 0) __builtin_amdgcn_s_barrier();          // balance the stagger

  // ---- epilogue.  acc[mq][mt][nq][r] is element (m0 + wr*128 + mq*64 + mt*32 + l31,
  // n0 + wc*64 + nq*32 + (r & 3) + 8 * (r >> 2) + 4 * lh).  Every wave is past its last read of the ring, and owns 16 KiB
  // of it: 128 rows of 64 elements ([row][8 chunks of 16 bytes], chunk ^ (row & 7)), or 64 rows of 128 for the transpose.
  // Only the wave itself touches them, so a wait for its own LDS traffic orders everything.
  unsigned char* my = smem + wave * 16384;
  const long mw = m0 + wr * 128, nw = n0 + wc * 64;
  const float* diag = p.diag + b * p.diag_next;
  float di[2][2];
#pragma unroll
  for (int mq = 0; mq < 2; ++mq)
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) di[mq][mt] = OP == kGram ? 0.f : diag[mw + mq * 64 + mt * 32 + l31];

  if constexpr (SYM) {                      // the diagonal, before the off-diagonal terms are added
    if (at.ti == at.tj)
#pragma unroll
      for (int mq = 0; mq < 2; ++mq)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nq = 0; nq < 2; ++nq)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const long i = mw + mq * 64 + mt * 32 + l31, j = nw + nq * 32 + (r & 3) + 8 * (r >> 2) + 4 * lh;
              if (i == j)
                (OP == kGram ? p.diag : p.diag_out)[b * p.diag_next + i] =
                    on_diagonal<OP>(acc[mq][mt][nq][r], di[mq][mt], p.c0, p.c1);
            }
  }
  // acc <- result: one plane of R at a time through LDS (lo alone first, so that r = hi + lo is added up term by term)
  if constexpr (OP == kGram) {
#pragma unroll
    for (int x = 0; x < 8; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x >> 2][(x >> 1) & 1][x & 1][r] *= kInvScale;
  } else {
    const float scale = OP == kPoly ? p.c1 * kInvScale : kInvScale;
#pragma unroll
    for (int x = 0; x < 8; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x >> 2][(x >> 1) & 1][x & 1][r] *= scale;
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      const _Float16* R = plane ? p.R.lo : p.R.hi;
      if (R == nullptr) continue;
      forget(acc);
      R += b * p.R.next + mw * p.R.ld + nw;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int row = i * 8 + (lane >> 3);
        __builtin_amdgcn_global_load_lds((gbl_void_ptr)(R + row * p.R.ld + ((lane & 7) ^ (row & 7)) * 8),
                                         (lds_void_ptr)(my + i * 1024), 16, 0, 0);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int mq = 0; mq < 2; ++mq)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nq = 0; nq < 2; ++nq)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int row = mq * 64 + mt * 32 + l31, col = nq * 32 + 8 * g + 4 * lh;
              const uint2 raw = *reinterpret_cast<const uint2*>(my + row * 128 + (((col >> 3) ^ (row & 7)) * 16) + (col & 7) * 2);
              _Float16 h[4];
              __builtin_memcpy(h, &raw, 8);
              float4 dj = make_float4(0.f, 0.f, 0.f, 0.f);
              if constexpr (OP == kPoly) dj = *reinterpret_cast<const float4*>(diag + nw + col);
              const float djs[4] = {dj.x, dj.y, dj.z, dj.w};
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float f = OP == kPoly ? p.c0 + p.c1 * (di[mq][mt] + djs[q]) : p.c0 + di[mq][mt];
                acc[mq][mt][nq][g * 4 + q] += f * (float)h[q];
              }
              __builtin_amdgcn_sched_barrier(0);      // (left to itself the compiler reads ahead until it spills)
            }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
  if constexpr (SYM) {
    if (at.ti == at.tj)
#pragma unroll
      for (int mq = 0; mq < 2; ++mq)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nq = 0; nq < 2; ++nq)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (mw + mq * 64 + mt * 32 + l31 == nw + nq * 32 + (r & 3) + 8 * (r >> 2) + 4 * lh) acc[mq][mt][nq][r] = 0.f;
  }

  if constexpr (OP == kFinal) {
    T* f = reinterpret_cast<T*>(p.fin) + b * p.fin_next;
    if constexpr (sizeof(T) == 2) {
      // 16-bit results whose rows are whole chunks leave like the planes below
      if (p.cols % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.fin) | (uintptr_t)(p.fin_next * 2)) & 15) == 0) {
#pragma unroll
        for (int mq = 0; mq < 2; ++mq)
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int nq = 0; nq < 2; ++nq)
#pragma unroll
              for (int r = 0; r < 16; r += 2) {
                uint16_t h[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  const T v = from_float<T>(acc[mq][mt][nq][r + q] * kInvScale);
                  __builtin_memcpy(&h[q], &v, 2);
                }
                const uint32_t both = (uint32_t)h[0] | ((uint32_t)h[1] << 16);
                if (p.turned) to_transpose(my, both, mq * 64 + mt * 32 + l31, nq, r, lh);
                else *reinterpret_cast<uint32_t*>(my + row_place(mq * 64 + mt * 32 + l31, nq * 32 + (r & 3) + 8 * (r >> 2) + 4 * lh)) = both;
              }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          long row, col;
          uint4 v;
          if (p.turned) {
            const int n = i * 4 + (lane >> 4), ck = lane & 15;
            v = *reinterpret_cast<const uint4*>(my + n * 256 + ((ck ^ (n & 15)) * 16));
            row = nw + n; col = mw + ck * 8;
          } else {
            const int m = i * 8 + (lane >> 3), ck = lane & 7;
            v = *reinterpret_cast<const uint4*>(my + m * 128 + ((ck ^ (m & 7)) * 16));
            row = mw + m; col = nw + ck * 8;
          }
          if (row < p.rows && col < p.cols) *reinterpret_cast<uint4*>(f + row * p.cols + col) = v;
        }
        return;
      }
    }
    // else its type and orientation straight from registers: rows may start anywhere
#pragma unroll
    for (int mq = 0; mq < 2; ++mq)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int nq = 0; nq < 2; ++nq)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const long i = mw + mq * 64 + mt * 32 + l31, j = nw + nq * 32 + (r & 3) + 8 * (r >> 2) + 4 * lh;
            const long row = p.turned ? j : i, col = p.turned ? i : j;
            if (row < p.rows && col < p.cols) f[row * p.cols + col] = from_float<T>(acc[mq][mt][nq][r] * kInvScale);
          }
    return;
  } else {
    // rows of the result: hi, then lo
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      _Float16* out = plane ? p.out.lo : p.out.hi;
      if (out == nullptr) continue;
      forget(acc);
      out += b * p.out.next + mw * p.out.ld + nw;
#pragma unroll
      for (int mq = 0; mq < 2; ++mq)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nq = 0; nq < 2; ++nq)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int row = mq * 64 + mt * 32 + l31, col = nq * 32 + 8 * g + 4 * lh;
              _Float16 h[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const Half2 s = split(acc[mq][mt][nq][g * 4 + q]);
                h[q] = plane ? s.lo : s.hi;
              }
              *reinterpret_cast<uint2*>(my + row * 128 + (((col >> 3) ^ (row & 7)) * 16) + (col & 7) * 2) =
                  make_uint2(pack(h[0], h[1]), pack(h[2], h[3]));
              __builtin_amdgcn_sched_barrier(0);
            }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int row = i * 8 + (lane >> 3), ck = lane & 7;
        const uint4 v = *reinterpret_cast<const uint4*>(my + row * 128 + ((ck ^ (row & 7)) * 16));
        *reinterpret_cast<uint4*>(out + row * p.out.ld + ck * 8) = v;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    // rows of the transpose
    if (SYM && at.ti == at.tj) return;
#pragma unroll
    for (int plane = 0; plane < 2; ++plane) {
      _Float16* out = plane ? p.out_t.lo : p.out_t.hi;
      if (out == nullptr) continue;
      forget(acc);
      out += b * p.out_t.next + nw * p.out_t.ld + mw;
#pragma unroll
      for (int mq = 0; mq < 2; ++mq)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nq = 0; nq < 2; ++nq)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
              const Half2 s0 = split(acc[mq][mt][nq][r]), s1 = split(acc[mq][mt][nq][r + 1]);
              to_transpose(my, plane ? pack(s0.lo, s1.lo) : pack(s0.hi, s1.hi), mq * 64 + mt * 32 + l31, nq, r, lh);
              if ((r & 3) == 2) __builtin_amdgcn_sched_barrier(0);
            }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int n = i * 4 + (lane >> 4), ck = lane & 15;
        const uint4 v = *reinterpret_cast<const uint4*>(my + n * 256 + ((ck ^ (n & 15)) * 16));
        *reinterpret_cast<uint4*>(out + n * p.out_t.ld + ck * 8) = v;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
}

// Tile of the products, and with it the padding: 256 x 256 where A has enough of those tiles that are not padding.  Five
// steps, small tiles against large ones, us (tiles of A; volume: what the larger padding multiplies the products by):
//     fast  7 x 1024 x 4096 (70 tiles)   1170 : 1170      fp32  2492 : 2628
//          10 x 1024 x 4096 (100)        1753 : 1463            3574 : 3185
//          22 x 1024 x 4096 (220)        3768 : 2573            7884 : 5724
//           5 x 1024 x 1024 (50)          388 :  534             756 : 1137
//          64 x 448 x 1792  (192, 1.3)   1903 : 1302            3051 : 2544
//          64 x 384 x 1536  (192, 1.8)   1073 : 1149            1897 : 2175
//          64 x 300 x 1000  (192, 2.7)    640 :  762            1127 : 1553
// Between volumes of 1.5 and 1.9 either side won by up to a fifth.
bool ns_use_large(long batch, long m, long n) {
  const long mt = (m + kLarge - 1) / kLarge;
  const auto volume = [&](long tile) {
    const double mp = (double)((m + tile - 1) / tile * tile), np = (double)((n + tile - 1) / tile * tile);
    return mp * mp * (3.0 * np + mp);
  };
  const double waste = volume(kLarge) / volume(kSmall);
  return waste <= 1.6 && (double)(batch * mt * (mt + 1) / 2) >= 96.0 * waste;
}

template <bool PAIR, int OP, typename T>
void product(const Product& p, long batch, bool large, bool mid, hipStream_t s) {
  const uint32_t per = OP == kGram || OP == kPoly ? (uint32_t)p.mt * (p.mt + 1) / 2 : (uint32_t)p.mt * p.nt;
  const long blocks = (long)per * batch * (OP == kGram && !large ? p.splits : 1);
  if (blocks >= (1l << 31)) throw std::invalid_argument("newton_schulz: batch too large");
  if constexpr (OP == kApply || OP == kFinal)
    if (mid) {
      hipLaunchKernelGGL((ns_mid_kernel<PAIR, OP, T>), dim3((unsigned)blocks), dim3(512), 0, s, p, per);
      return;
    }
  if (large) hipLaunchKernelGGL((ns_large_kernel<PAIR, OP, T>), dim3((unsigned)blocks), dim3(512), 0, s, p, per);
  else hipLaunchKernelGGL((ns_small_kernel<PAIR, OP, T, OP == kGram || OP == kPoly ? 8 : 4>), dim3((unsigned)blocks), dim3(512), 0, s,
                          p, per);
  if constexpr (OP == kGram)
    if (!large && p.splits > 1) hipLaunchKernelGGL(ns_join_kernel<T>, dim3((unsigned)(per * batch)), dim3(512), 0, s, p, per);
}

struct Sizes {
  long m, n, mp, np;                        // X: m <= n, padded
  bool large, mid;                          // 256 x 256 tiles; else 128 x 128 ones for the products with X
  int splits;                               // of the contraction over n
  size_t x, sq, diag, norm;                 // bytes of one plane of X, of A, of a diagonal, of the partial norms
  size_t partial;                           // ... of the split sums
};
Sizes sizes(long batch, long rows, long cols) {
  Sizes z;
  z.m = rows < cols ? rows : cols;
  z.n = rows < cols ? cols : rows;
  z.large = ns_use_large(batch, z.m, z.n);
  const long tile = z.large ? kLarge : kSmall;
  z.mp = (z.m + tile - 1) / tile * tile;
  z.np = (z.n + tile - 1) / tile * tile;
  // enough 64 x 64 tiles for two rounds of workgroups, and rows that fill 128-row tiles.  Five steps with 64 x 64 tiles against
  // 128 x 128 ones, us: 256 x 2304 fp32, 3 matrices (432 tiles) 195 : 202, 4 (576) 216 : 201, 6 (864) 238 : 217; 768 x 768
  // fast, 3 (432) 162 : 169, 4 (576) 242 : 225; 1024 x 1024 fast, 2 (512) 234 : 246, 3 (768) 279 : 259
  z.mid = !z.large && z.mp % kMid == 0 && batch * (z.mp / kSmall) * (z.np / kSmall) > 512;
  if (z.mid) z.np = (z.np + kMid - 1) / kMid * kMid;
  z.x = (size_t)batch * z.mp * z.np * 2;
  z.sq = (size_t)batch * z.mp * z.mp * 2;
  z.diag = (size_t)batch * z.mp * 4;
  z.norm = (size_t)batch * kNormParts * 8;
  // a few dozen tiles of a long contraction see one memory latency after the other (60 tiles, 2304 elements: 22 us):
  // split it until the card has a workgroup per compute unit, 8 slices each at least
  const long tiles = batch * (z.mp / kSmall) * (z.mp / kSmall + 1) / 2, slices = z.np / 32;
  z.splits = 1;
  if (!z.large)
    while (z.splits < 8 && tiles * (z.splits + 1) <= 256 && slices / (z.splits + 1) >= 8) ++z.splits;
  z.partial = z.splits > 1 ? (size_t)tiles * z.splits * 4096 * 4 : 0;
  return z;
}

template <bool PAIR, typename T>
void run(const NewtonSchulz& q, hipStream_t s) {
  const Sizes z = sizes(q.batch, q.rows, q.cols);
  const int turned = q.rows > q.cols;
  char* w = reinterpret_cast<char*>(q.work);
  auto take = [&](size_t bytes) { char* r = w; w += bytes; return r; };
  auto planes = [&](size_t bytes, long ld, long next, bool lo) {
    Planes p{reinterpret_cast<_Float16*>(take(bytes)), nullptr, ld, next};
    if (lo) p.lo = reinterpret_cast<_Float16*>(take(bytes));
    return p;
  };
  const long bx = z.mp * z.np, ba = z.mp * z.mp;
  const Planes X = planes(z.x, z.np, bx, true);
  const Planes XT[2] = {planes(z.x, z.mp, bx, PAIR), planes(z.x, z.mp, bx, PAIR)};
  const Planes A = planes(z.sq, z.mp, ba, PAIR), B = planes(z.sq, z.mp, ba, PAIR);
  float* Da = reinterpret_cast<float*>(take(z.diag));
  float* Db = reinterpret_cast<float*>(take(z.diag));
  double* norm = reinterpret_cast<double*>(take(z.norm));
  float* partial = reinterpret_cast<float*>(take(z.partial));
  const T* g = reinterpret_cast<const T*>(q.g);
  hipLaunchKernelGGL(ns_norm_kernel<T>, dim3(kNormParts, (unsigned)q.batch), dim3(256), 0, s, g, q.rows * q.cols, norm);
  hipLaunchKernelGGL(ns_split_kernel<T>, dim3((unsigned)(z.np / 64), (unsigned)(z.mp / 64), (unsigned)q.batch), dim3(256), 0, s,
                     g, q.rows, q.cols, turned, q.eps, norm, X, XT[0]);
  const long tile = z.large ? kLarge : kSmall, slice = PAIR ? 32 : 64;
  for (int it = 0; it < q.steps; ++it) {
    Product a{};                            // A = X X^T
    a.P = a.Q = X;
    a.out = a.out_t = A;
    a.diag = Da; a.diag_next = z.mp;
    a.mt = a.nt = (int)(z.mp / tile); a.ktiles = (int)(z.np / slice);
    a.splits = z.splits; a.partial = partial;
    product<PAIR, kGram, T>(a, q.batch, z.large, false, s);
    Product b{};                            // B = b A + c A A
    b.P = b.Q = b.R = A;
    b.out = b.out_t = B;
    b.diag = Da; b.diag_out = Db; b.diag_next = z.mp;
    b.mt = b.nt = (int)(z.mp / tile); b.ktiles = (int)(z.mp / slice);
    b.c0 = q.b; b.c1 = q.c;
    product<PAIR, kPoly, T>(b, q.batch, z.large, false, s);
    Product c{};                            // X = a X + B X
    c.P = B; c.Q = XT[it & 1]; c.R = X;
    c.diag = Db; c.diag_next = z.mp;
    const long apply = z.mid ? kMid : tile;
    c.mt = (int)(z.mp / apply); c.nt = (int)(z.np / apply); c.ktiles = (int)(z.mp / slice);
    c.c0 = q.a;
    if (it + 1 == q.steps) {
      c.fin = q.out; c.fin_next = q.rows * q.cols; c.rows = q.rows; c.cols = q.cols; c.turned = turned;
      product<PAIR, kFinal, T>(c, q.batch, z.large, z.mid, s);
    } else {
      c.out = X; c.out_t = XT[(it + 1) & 1];
      product<PAIR, kApply, T>(c, q.batch, z.large, z.mid, s);
    }
  }
}

}  // namespace

size_t newton_schulz_workspace(long batch, long rows, long cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) throw std::invalid_argument("newton_schulz: empty shape");
  const Sizes z = sizes(batch, rows, cols);
  return 6 * z.x + 4 * z.sq + 2 * z.diag + z.norm + z.partial;
}

void newton_schulz_launch(const NewtonSchulz& q, int dtype, hipStream_t s) {
  if (q.batch <= 0 || q.rows <= 0 || q.cols <= 0 || q.steps <= 0) throw std::invalid_argument("newton_schulz: empty shape or no steps");
  const Sizes z = sizes(q.batch, q.rows, q.cols);
  if (q.batch > 65535 || z.mp / 64 > 65535) throw std::invalid_argument("newton_schulz: too many matrices");
  if (q.fast && dtype != kBF16) throw std::invalid_argument("newton_schulz: fast products are for bfloat16");
  switch (dtype) {
    case kF32: run<true, float>(q, s); break;
    case kF16: run<true, f16_t>(q, s); break;
    case kBF16:
      if (q.fast) run<false, bf16_t>(q, s);
      else run<true, bf16_t>(q, s);
      break;
    default: throw std::invalid_argument("unsupported dtype");
  }
  DPA_CHECK_HIP(hipGetLastError());
}

}  // namespace dpa
