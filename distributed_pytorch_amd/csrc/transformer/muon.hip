// The two elementwise ends of the Muon step (gfx950), each ONE launch over a device-resident table of matrices:
//
//     begin:  buf = mu * buf + g / loss_scale,   u = nesterov ? g / loss_scale + mu * buf : buf
//     (newton_schulz.hip turns every u into O, in place)
//     end:    p = p * (1 - lr * wd) - lr * scale * O,   and the low-precision copy of p
//
// Hyper-parameters live in a device array (a schedule needs no re-capture) and both are predicated on the loss scaler's
// overflow flag without a host sync.  Bound by memory bandwidth: a workgroup owns a chunk of 2048 elements (28 million of them,
// 12 x 2304 x 768 and 12 x 768 x 768, fp32: begin 72 us, 6.3 TB/s, end 58 us, 5.8 TB/s, parts of both in the last-level cache).
#include "../common.h"
#include "transformer.h"

namespace dpa {
namespace {

constexpr int kChunk = 2048;

__device__ __forceinline__ const MuonTensor& find(const MuonTensor* table, int n, long chunk) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table[mid].chunk0 <= chunk) lo = mid; else hi = mid - 1;
  }
  return table[lo];
}

template <typename TG>
__global__ __launch_bounds__(256) void muon_begin_kernel(const MuonTensor* __restrict__ table, int n,
                                                         const float* __restrict__ hyper, const float* __restrict__ inv_scale,
                                                         const float* __restrict__ found_inf, float* __restrict__ update) {
  if (found_inf != nullptr && found_inf[0] > 0.f) return;
  const long chunk = blockIdx.x;
  const MuonTensor t = find(table, n, chunk);
  const long base = (chunk - t.chunk0) * kChunk;
  const float mu = hyper[1], gs = inv_scale != nullptr ? inv_scale[0] : 1.f;
  const bool nesterov = hyper[3] != 0.f;
  const TG* g = reinterpret_cast<const TG*>(t.g);
#pragma unroll
  for (int k = 0; k < kChunk / 256; ++k) {
    const long i = base + k * 256 + threadIdx.x;
    if (i >= t.n) break;
    const float gr = to_float(g[i]) * gs;
    const float b = mu * t.buf[i] + gr;
    t.buf[i] = b;
    update[t.at + i] = nesterov ? gr + mu * b : b;
  }
}

template <typename TL>
__global__ __launch_bounds__(256) void muon_end_kernel(const MuonTensor* __restrict__ table, int n,
                                                       const float* __restrict__ hyper, const float* __restrict__ found_inf,
                                                       const float* __restrict__ update) {
  if (found_inf != nullptr && found_inf[0] > 0.f) return;
  const long chunk = blockIdx.x;
  const MuonTensor t = find(table, n, chunk);
  const long base = (chunk - t.chunk0) * kChunk;
  const float lr = hyper[0], keep = 1.f - lr * hyper[2], step = lr * hyper[4] * t.scale;
  TL* lp = reinterpret_cast<TL*>(t.lp);
#pragma unroll
  for (int k = 0; k < kChunk / 256; ++k) {
    const long i = base + k * 256 + threadIdx.x;
    if (i >= t.n) break;
    const float p = t.p[i] * keep - step * update[t.at + i];
    t.p[i] = p;
    if (lp != nullptr) lp[i] = from_float<TL>(p);
  }
}

}  // namespace

int muon_chunk_elems() { return kChunk; }

void muon_begin_launch(const MuonTensor* table, int n, long chunks, int g_dtype, const float* hyper, const float* inv_scale,
                       const float* found_inf, float* update, hipStream_t s) {
  if (n <= 0 || chunks <= 0) return;
  if (chunks >= (1l << 31)) throw std::invalid_argument("muon: too many elements");
  DPA_DISPATCH_DTYPE(g_dtype, hipLaunchKernelGGL(muon_begin_kernel<T>, dim3((unsigned)chunks), dim3(256), 0, s, table, n, hyper,
                                                 inv_scale, found_inf, update));
  DPA_CHECK_HIP(hipGetLastError());
}

void muon_end_launch(const MuonTensor* table, int n, long chunks, int lp_dtype, const float* hyper, const float* found_inf,
                     const float* update, hipStream_t s) {
  if (n <= 0 || chunks <= 0) return;
  if (chunks >= (1l << 31)) throw std::invalid_argument("muon: too many elements");
  DPA_DISPATCH_DTYPE(lp_dtype, hipLaunchKernelGGL(muon_end_kernel<T>, dim3((unsigned)chunks), dim3(256), 0, s, table, n, hyper,
                                                  found_inf, update));
  DPA_CHECK_HIP(hipGetLastError());
}

}  // namespace dpa
