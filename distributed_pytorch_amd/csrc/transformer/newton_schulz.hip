// Newton-Schulz orthogonalisation of a batch of matrices (gfx950):  X = G / (|G|_F + eps) (transposed where it has more
// rows than columns), then `steps` times
//
//     A = X X^T,   B = b A + c A A,   X = a X + B X
//
// 32-bit products on the 16-bit matrix cores.  Every matrix is held as two fp16 planes, x * 2^10 = hi + lo with 22
// significant bits (singular values stay below ~4, so nothing leaves the fp16 range, and the scale keeps `lo` clear of the
// subnormals), and a product is hi hi + hi lo + lo hi in fp32 accumulators: three MFMAs in place of one fp32 product at
// a sixteenth of the rate, with an error near that of fp32 (one fp16 or bf16 plane loses 3 to 6 bits over five steps,
// more than the rounding of a bf16 result).  Planes are interleaved by 8 elements ([row][k / 8][hi 8][lo 8]), so a
// K slice of 32 is one 128-byte row piece.  All dimensions are padded to whole tiles with zeros, which every product
// preserves; A and B are symmetric, and only their tiles on and below the diagonal are computed.
// X is also kept transposed, because B X needs it with m contiguous.
#include "../common.h"
#include "transformer.h"
#include <type_traits>

namespace dpa {
namespace {

typedef __attribute__((address_space(3))) void* lds_void_ptr;
typedef const __attribute__((address_space(1))) void* gbl_void_ptr;

constexpr int kTile = 128;
constexpr float kScale = 1024.f, kInvScale = 1.f / 1024.f;
constexpr int kNormParts = 64;

struct Half2 { _Float16 hi, lo; };
__device__ __forceinline__ Half2 split(float x) {
  Half2 h;
  h.hi = (_Float16)x;
  h.lo = (_Float16)(x - (float)h.hi);
  return h;
}
// element (r, k) of a plane pair
__device__ __forceinline__ long at(long r, long k, long ld) { return r * ld + ((k >> 3) << 4) + (k & 7); }

// ---- |G|_F^2 in 64 bits: kNormParts partial sums a matrix
template <typename T>
__global__ __launch_bounds__(256) void ns_norm_kernel(const T* __restrict__ g, long elems, double* __restrict__ parts) {
  __shared__ double red[4];
  const T* p = g + blockIdx.y * elems;
  const long each = (elems + kNormParts - 1) / kNormParts;
  const long lo = min((long)blockIdx.x * each, elems), hi = min(lo + each, elems);
  double t = 0.0;
  for (long i = lo + threadIdx.x; i < hi; i += 256) {
    const double v = (double)to_float(p[i]);
    t += v * v;
  }
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) parts[(long)blockIdx.y * kNormParts + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- X and X^T planes of 64 x 64 elements of the normalised matrix (zeros in the padding)
template <typename T>
__global__ __launch_bounds__(256) void ns_split_kernel(const T* __restrict__ g, long rows, long cols, int turned, double eps,
                                                       const double* __restrict__ parts, _Float16* __restrict__ x,
                                                       _Float16* __restrict__ xt, long mp, long np) {
  __shared__ float tile[64][65];
  __shared__ float inv_s;
  const long b = blockIdx.z;
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < kNormParts; ++i) t += parts[b * kNormParts + i];
    inv_s = (float)(1.0 / (sqrt(t) + eps));
  }
  __syncthreads();
  const float inv = inv_s;
  const long i0 = (long)blockIdx.y * 64, j0 = (long)blockIdx.x * 64;     // in X
  const T* p = g + b * rows * cols;
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int r = e >> 6, c = e & 63;                                    // of G's tile
    const long gr = (turned ? j0 : i0) + r, gc = (turned ? i0 : j0) + c;
    const float v = gr < rows && gc < cols ? to_float(p[gr * cols + gc]) * inv * kScale : 0.f;
    if (turned) tile[c][r] = v;
    else tile[r][c] = v;
  }
  __syncthreads();
  _Float16* xb = x + b * mp * np * 2;
  _Float16* xtb = xt + b * mp * np * 2;
  for (int e = threadIdx.x; e < 512; e += 256) {
    const int r = e >> 3, u = e & 7;
    f16x8_t h, l;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const Half2 v = split(tile[r][u * 8 + q]);
      h[q] = v.hi; l[q] = v.lo;
    }
    f16x8_t* d = reinterpret_cast<f16x8_t*>(xb + at(i0 + r, j0 + u * 8, 2 * np));
    d[0] = h; d[1] = l;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const Half2 v = split(tile[u * 8 + q][r]);
      h[q] = v.hi; l[q] = v.lo;
    }
    d = reinterpret_cast<f16x8_t*>(xtb + at(j0 + r, i0 + u * 8, 2 * mp));
    d[0] = h; d[1] = l;
  }
}

// ---- out = alpha * R + beta * P Q^T on plane pairs
struct Product {
  const _Float16* P; const _Float16* Q; const _Float16* R;
  _Float16* out; _Float16* out_t;            // planes of the result and of its transpose (each may be null)
  void* fin;                                 // the last step: the result in the caller's type and orientation
  long ldp, ldq, ldr, ldo, ldt;              // in fp16 elements: twice the padded row length
  long bp, bq, br, bo, bt, bfin;             // from one matrix of the batch to the next
  int mt, nt, ksteps, sym, turned;
  long rows, cols;                           // of the caller's matrix
  float alpha, beta, fin_scale;
};

template <typename T>
__global__ __launch_bounds__(256, 2) void ns_product_kernel(const Product p, const uint32_t per_matrix) {
  __shared__ __attribute__((aligned(16))) unsigned char smem[4 * kTile * 128];     // two stages of P and Q slices
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave >> 1, wc = wave & 1, l31 = lane & 31, lh = lane >> 5;
  const uint32_t lid = xcd_remap(blockIdx.x, gridDim.x);
  const long b = lid / per_matrix;
  uint32_t t = lid - (uint32_t)b * per_matrix;
  int ti, tj;
  if (p.sym) {                               // tiles on and below the diagonal
    ti = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((uint32_t)(ti + 1) * (ti + 2) / 2 <= t) ++ti;
    while ((uint32_t)ti * (ti + 1) / 2 > t) --ti;
    tj = (int)(t - (uint32_t)ti * (ti + 1) / 2);
  } else {
    ti = (int)(t % (uint32_t)p.mt);
    tj = (int)(t / (uint32_t)p.mt);
  }
  const long i0 = (long)ti * kTile, j0 = (long)tj * kTile;
  // staging: instruction q of a wave covers rows (wave * 4 + q) * 8 + lane / 8; LDS chunk lane % 8 holds source chunk
  // (lane % 8) ^ ((row >> 1) & 7), so that 16 rows of a fragment read touch 16 different 16-byte columns
  const _Float16* srcp[4];
  const _Float16* srcq[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int row = (wave * 4 + q) * 8 + (lane >> 3);
    const int ch = (lane & 7) ^ ((row >> 1) & 7);
    srcp[q] = p.P + b * p.bp + (i0 + row) * p.ldp + ch * 8;
    srcq[q] = p.Q + b * p.bq + (j0 + row) * p.ldq + ch * 8;
  }
  auto stage = [&](int k) {
    unsigned char* dst = smem + (k & 1) * (2 * kTile * 128) + wave * 4096;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      __builtin_amdgcn_global_load_lds((gbl_void_ptr)(srcp[q] + (long)k * 64), (lds_void_ptr)(dst + q * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((gbl_void_ptr)(srcq[q] + (long)k * 64), (lds_void_ptr)(dst + kTile * 128 + q * 1024), 16,
                                       0, 0);
    }
  };
  f32x16_t acc[2][2];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][c][r] = 0.f;
  stage(0);
  for (int k = 0; k < p.ksteps; ++k) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();                         // slice k has landed for every wave, and slice k - 1 has been read
    if (k + 1 < p.ksteps) stage(k + 1);
    const unsigned char* base = smem + (k & 1) * (2 * kTile * 128);
    f16x8_t fp[2][2][2], fq[2][2][2];        // [32-row block][k16][hi, lo]
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int ch = ((s * 2 + lh) * 2 + h) ^ ((l31 >> 1) & 7);
          fp[m][s][h] = *reinterpret_cast<const f16x8_t*>(base + (wr * 64 + m * 32 + l31) * 128 + ch * 16);
          fq[m][s][h] = *reinterpret_cast<const f16x8_t*>(base + kTile * 128 + (wc * 64 + m * 32 + l31) * 128 + ch * 16);
        }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int x = 0; x < 3; ++x)            // hi hi, hi lo, lo hi
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n)
            acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fq[n][s][x == 1], fp[m][s][x == 2], acc[m][n], 0, 0, 0);
  }
  // acc[m][n][r] is element (i0 + wr * 64 + m * 32 + l31, j0 + wc * 64 + n * 32 + (r & 3) + 8 * (r >> 2) + 4 * lh)
  const bool mirror = p.out_t != nullptr && !(p.sym && ti == tj);
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const long i = i0 + wr * 64 + m * 32 + l31;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const long j = j0 + wc * 64 + n * 32 + 8 * g + 4 * lh;
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = p.beta * acc[m][n][g * 4 + q];
        if (p.R != nullptr) {
          const _Float16* r = p.R + b * p.br + at(i, j, p.ldr);
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] += p.alpha * ((float)r[q] + (float)r[q + 8]);
        }
        if (p.fin != nullptr) {
          T* f = reinterpret_cast<T*>(p.fin) + b * p.bfin;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const long r = p.turned ? j + q : i, c = p.turned ? i : j + q;
            if (r < p.rows && c < p.cols) f[r * p.cols + c] = from_float<T>(v[q] * p.fin_scale);
          }
        }
        if (p.out != nullptr || mirror) {
          Half2 h[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) h[q] = split(v[q]);
          if (p.out != nullptr) {
            _Float16* o = p.out + b * p.bo + at(i, j, p.ldo);
#pragma unroll
            for (int q = 0; q < 4; ++q) { o[q] = h[q].hi; o[q + 8] = h[q].lo; }
          }
          if (mirror)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              _Float16* o = p.out_t + b * p.bt + at(j + q, i, p.ldt);
              o[0] = h[q].hi;
              o[8] = h[q].lo;
            }
        }
      }
  }
}

template <typename T>
void product(const Product& p, long batch, hipStream_t s) {
  const uint32_t per = p.sym ? (uint32_t)p.mt * (p.mt + 1) / 2 : (uint32_t)p.mt * p.nt;
  const long blocks = (long)per * batch;
  if (blocks >= (1l << 31)) throw std::invalid_argument("newton_schulz: batch too large");
  hipLaunchKernelGGL(ns_product_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, p, per);
}

struct Sizes {
  long m, n, mp, np;                         // X: m <= n, padded
  size_t x, sq, norm;                        // bytes of the X planes, of A and of the partial norms
};
Sizes sizes(long batch, long rows, long cols) {
  Sizes z;
  z.m = rows < cols ? rows : cols;
  z.n = rows < cols ? cols : rows;
  z.mp = (z.m + kTile - 1) / kTile * kTile;
  z.np = (z.n + kTile - 1) / kTile * kTile;
  z.x = (size_t)batch * z.mp * z.np * 4;
  z.sq = (size_t)batch * z.mp * z.mp * 4;
  z.norm = (size_t)batch * kNormParts * 8;
  return z;
}

template <typename T>
void run(const NewtonSchulz& q, hipStream_t s) {
  const Sizes z = sizes(q.batch, q.rows, q.cols);
  const int turned = q.rows > q.cols;
  char* w = reinterpret_cast<char*>(q.work);
  auto take = [&](size_t bytes) { char* r = w; w += bytes; return r; };
  _Float16* X = reinterpret_cast<_Float16*>(take(z.x));
  _Float16* XT[2];
  XT[0] = reinterpret_cast<_Float16*>(take(z.x));
  XT[1] = reinterpret_cast<_Float16*>(take(z.x));
  _Float16* A = reinterpret_cast<_Float16*>(take(z.sq));
  _Float16* B = reinterpret_cast<_Float16*>(take(z.sq));
  double* norm = reinterpret_cast<double*>(take(z.norm));
  const T* g = reinterpret_cast<const T*>(q.g);
  hipLaunchKernelGGL(ns_norm_kernel<T>, dim3(kNormParts, (unsigned)q.batch), dim3(256), 0, s, g, q.rows * q.cols, norm);
  hipLaunchKernelGGL(ns_split_kernel<T>, dim3((unsigned)(z.np / 64), (unsigned)(z.mp / 64), (unsigned)q.batch), dim3(256), 0, s,
                     g, q.rows, q.cols, turned, q.eps, norm, X, XT[0], z.mp, z.np);
  const long bx = z.mp * z.np * 2, ba = z.mp * z.mp * 2;
  for (int it = 0; it < q.steps; ++it) {
    const bool last = it + 1 == q.steps;
    Product a{};                             // A = X X^T
    a.P = a.Q = X; a.ldp = a.ldq = 2 * z.np; a.bp = a.bq = bx;
    a.out = a.out_t = A; a.ldo = a.ldt = 2 * z.mp; a.bo = a.bt = ba;
    a.mt = a.nt = (int)(z.mp / kTile); a.ksteps = (int)(z.np / 32); a.sym = 1;
    a.beta = kInvScale;
    product<T>(a, q.batch, s);
    Product b{};                             // B = b A + c A A
    b.P = b.Q = b.R = A; b.ldp = b.ldq = b.ldr = 2 * z.mp; b.bp = b.bq = b.br = ba;
    b.out = b.out_t = B; b.ldo = b.ldt = 2 * z.mp; b.bo = b.bt = ba;
    b.mt = b.nt = (int)(z.mp / kTile); b.ksteps = (int)(z.mp / 32); b.sym = 1;
    b.alpha = q.b; b.beta = q.c * kInvScale;
    product<T>(b, q.batch, s);
    Product c{};                             // X = a X + B X
    c.P = B; c.ldp = 2 * z.mp; c.bp = ba;
    c.Q = XT[it & 1]; c.ldq = 2 * z.mp; c.bq = bx;
    c.R = X; c.ldr = 2 * z.np; c.br = bx;
    if (last) {
      c.fin = q.out; c.bfin = q.rows * q.cols; c.rows = q.rows; c.cols = q.cols; c.turned = turned; c.fin_scale = kInvScale;
    } else {
      c.out = X; c.ldo = 2 * z.np; c.bo = bx;
      c.out_t = XT[(it + 1) & 1]; c.ldt = 2 * z.mp; c.bt = bx;
    }
    c.mt = (int)(z.mp / kTile); c.nt = (int)(z.np / kTile); c.ksteps = (int)(z.mp / 32);
    c.alpha = q.a; c.beta = kInvScale;
    product<T>(c, q.batch, s);
  }
}

}  // namespace

size_t newton_schulz_workspace(long batch, long rows, long cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) throw std::invalid_argument("newton_schulz: empty shape");
  const Sizes z = sizes(batch, rows, cols);
  return 3 * z.x + 2 * z.sq + z.norm;
}

void newton_schulz_launch(const NewtonSchulz& q, int dtype, hipStream_t s) {
  if (q.batch <= 0 || q.rows <= 0 || q.cols <= 0 || q.steps <= 0) throw std::invalid_argument("newton_schulz: empty shape or no steps");
  const Sizes z = sizes(q.batch, q.rows, q.cols);
  if (q.batch > 65535 || z.mp / 64 > 65535) throw std::invalid_argument("newton_schulz: too many matrices");
  DPA_DISPATCH_DTYPE(dtype, run<T>(q, s));
  DPA_CHECK_HIP(hipGetLastError());
}

}  // namespace dpa
