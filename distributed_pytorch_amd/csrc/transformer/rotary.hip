// Rotary positions of several axes on the packed projection [B][S][3][H][D] (gfx950): pair j of every query and key head
// is turned by the angle pos[token][axis[j]] * freq[j],
//
//     (a, b) -> (a cos - b sin, a sin + b cos),
//
// pairs (2j, 2j + 1) or (j, j + P); the values and what lies behind the P pairs are copied.  The gradient is the same
// with the angles negated.  The angle is formed in 64 bits and reduced to a fraction of a turn there (32 bits lose it for
// far positions), sine and cosine of the fraction in 32: they are computed once per token and pair into LDS and serve
// the 2 H heads.  Bound by memory bandwidth: 32 x 257 tokens of 3 x 16 x 80 bf16 27 us (4.7 TB/s), 4 x 3137 tokens of 3 x 16 x 64
// fp16 35 us (4.4 TB/s).
#include "../common.h"
#include "transformer.h"

namespace dpa {
namespace {

__device__ __forceinline__ double position(const void* p, long i, int kind) {
  switch (kind) {
    case kPosI64: return (double)reinterpret_cast<const long*>(p)[i];
    case kPosI32: return (double)reinterpret_cast<const int*>(p)[i];
    case kPosF32: return (double)reinterpret_cast<const float*>(p)[i];
    default: return reinterpret_cast<const double*>(p)[i];
  }
}

// VEC: D, P (not INTER) and every row are whole 16-byte chunks; else element by element.  ANY (not INTER, not in place): P may
// be anything, a chunk's partners come from wherever they start (33 x 1765 tokens of 3 x 6 x 48 bf16, P = 15: 68 us, element
// by element 115; in place they still move so: 38 us, 24 pairs in whole chunks 25)
template <typename T, bool VEC, bool INTER, bool ANY>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p, const int tt, const FastDiv by_items,
                                                     const FastDiv by_chunks, const FastDiv by_rest) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  extern __shared__ float2 turn[];                 // [tt][P]: cos, sin
  const int P = p.pairs, D = p.D, H = p.H;
  const long first = (long)blockIdx.x * tt;
  const int count = (int)min((long)tt, p.tokens - first);
  for (int i = threadIdx.x; i < count * P; i += 256) {
    const int t = i / P, j = i - t * P;
    const long tok = first + t;
    const long b = tok / p.S, s = tok - b * p.S;
    const int axis = p.axis[j];
    if (axis < 0 || axis >= p.axes) {              // no such position: seen in the result, never read
      turn[i] = make_float2(NAN, NAN);
      continue;
    }
    const long at = (p.pos_batched ? tok : s) * p.axes + axis;
    const double f = p.freq_f64 ? reinterpret_cast<const double*>(p.freq)[j] : (double)reinterpret_cast<const float*>(p.freq)[j];
    double turns = position(p.pos, at, p.pos_kind) * f * 0.15915494309189535;       // 1 / (2 pi)
    turns -= rint(turns);
    float sn, cs;
    sincospif((float)(2.0 * turns), &sn, &cs);
    turn[i] = make_float2(cs, p.negate ? -sn : sn);
  }
  __syncthreads();
  const T* in = reinterpret_cast<const T*>(p.in);
  T* out = reinterpret_cast<T*>(p.out);
  const bool copy = p.in != p.out;
  // items of one token: the chunks (pairs of chunks) that turn, then the ones that are copied
  // per head; INTER: the last one may hold pairs that stay; not INTER: with a partner P further on
  const int chunks = ANY ? D / V : ((INTER ? 2 * P : P) + V - 1) / V;
  const int rest = ANY ? 0 : (INTER ? D / V - chunks : (D - 2 * P) / V);
  const int n_turn = 2 * H * chunks;
  const int n_rest = copy ? 2 * H * rest : 0;
  const int items = n_turn + n_rest + (copy ? H * D / V : 0);
  for (int i = threadIdx.x; i < count * items; i += 256) {
    const int t = (int)fdiv((uint32_t)i, by_items);
    int it = i - t * items;
    const long tok = first + t;
    const long b = tok / p.S, s = tok - b * p.S;
    const T* src = in + b * p.in_batch + s * p.in_token;
    T* dst = out + b * p.out_batch + s * p.out_token;
    if (it < n_turn) {
      const int head = (int)fdiv((uint32_t)it, by_chunks);
      const int j0 = (it - head * chunks) * V;
      const float2* cs = turn + t * P;
      const long o = (long)head * D + j0;
      if constexpr (VEC) {
        if constexpr (INTER) {
          Vec16<T> v;
          v.load(src + o);
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            if (j0 + j >= 2 * P) break;
            const float2 c = cs[(j0 + j) / 2];
            const float a = v.get(j), b2 = v.get(j + 1);
            v.set(j, a * c.x - b2 * c.y);
            v.set(j + 1, a * c.y + b2 * c.x);
          }
          v.store(dst + o);
        } else if constexpr (ANY) {
          // (behind the last key head lie the values: a read of up to V - 1 elements too many stays in the token's row)
          Vec16<T> v, above, below;
          v.load(src + o);
          if (j0 < P) __builtin_memcpy(&above.raw, src + o + P, 16);
          if (j0 >= P && j0 < 2 * P) __builtin_memcpy(&below.raw, src + o - P, 16);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int e = j0 + j;
            if (e < P) {
              const float2 c = cs[e];
              const float a = v.get(j), b2 = above.get(j);
              v.set(j, a * c.x - b2 * c.y);
            } else if (e < 2 * P) {
              const float2 c = cs[e - P];
              const float a = j0 >= P ? below.get(j) : to_float(src[o + j - P]), b2 = v.get(j);
              v.set(j, a * c.y + b2 * c.x);
            }
          }
          v.store(dst + o);
        } else {
          Vec16<T> v, w;
          v.load(src + o);
          w.load(src + o + P);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float2 c = cs[j0 + j];
            const float a = v.get(j), b2 = w.get(j);
            v.set(j, a * c.x - b2 * c.y);
            w.set(j, a * c.y + b2 * c.x);
          }
          v.store(dst + o);
          w.store(dst + o + P);
        }
      } else if constexpr (INTER) {
        if ((j0 & 1) == 0) {                         // the even element of a pair does both
          const float2 c = cs[j0 / 2];
          const float a = to_float(src[o]), b2 = to_float(src[o + 1]);
          dst[o] = from_float<T>(a * c.x - b2 * c.y);
          dst[o + 1] = from_float<T>(a * c.y + b2 * c.x);
        }
      } else {
        const float2 c = cs[j0];
        const float a = to_float(src[o]), b2 = to_float(src[o + P]);
        dst[o] = from_float<T>(a * c.x - b2 * c.y);
        dst[o + P] = from_float<T>(a * c.y + b2 * c.x);
      }
    } else {
      it -= n_turn;
      long o;
      if (it < n_rest) {
        const int head = (int)fdiv((uint32_t)it, by_rest);
        o = (long)head * D + (INTER ? chunks * V : 2 * P) + (it - head * rest) * V;
      } else {
        o = 2l * H * D + (long)(it - n_rest) * V;
      }
      if constexpr (VEC) {
        Vec16<T> v;
        v.load(src + o);
        v.store(dst + o);
      } else {
        dst[o] = src[o];
      }
    }
  }
}

template <typename T>
void launch(const RotaryParams& p, hipStream_t s) {
  const int V = 16 / (int)sizeof(T);
  auto off16 = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) != 0; };
  const bool copy = p.in != p.out;
  const bool any = !p.interleaved && p.pairs % V != 0 && copy;
  const bool vec = p.D % V == 0 && (p.interleaved || p.pairs % V == 0 || any) &&
                   !off16(p.in) && !off16(p.out) && p.in_batch % V == 0 && p.in_token % V == 0 && p.out_batch % V == 0 &&
                   p.out_token % V == 0;
  const int v = vec ? V : 1;
  const int chunks = vec && any ? p.D / v : ((p.interleaved ? 2 * p.pairs : p.pairs) + v - 1) / v;
  const int rest = vec && any ? 0 : (p.interleaved ? p.D / v - chunks : (p.D - 2 * p.pairs) / v);
  const int items = 2 * p.H * chunks + (copy ? 2 * p.H * rest + p.H * p.D / v : 0);
  if (items <= 0) return;
  // many short workgroups, whose angles and copies overlap, one token each for short calls (4 x 3137 tokens of 3 x 16 x 64
  // fp16: 45 us with 2048 workgroups, 36 with 8192; a copy of the same bytes takes 32)
  long tt = p.tokens / 8192;
  tt = tt < 1 ? 1 : (tt > 8 ? 8 : tt);
  while (tt > 1 && (tt * p.pairs * 8 > 32768 || tt * items >= (1l << 30))) tt >>= 1;
  const long blocks = (p.tokens + tt - 1) / tt;
  if (blocks >= (1l << 31)) throw std::invalid_argument("rotary: too many tokens");
  const size_t lds = (size_t)(tt * p.pairs * 8 + 8);
  const FastDiv bi = make_fastdiv((uint32_t)items), bc = make_fastdiv((uint32_t)(chunks > 0 ? chunks : 1)),
                br = make_fastdiv((uint32_t)(rest > 0 ? rest : 1));
#define DPA_ROTARY(VECB, INTERB, ANYB) \
  hipLaunchKernelGGL((rotary_kernel<T, VECB, INTERB, ANYB>), dim3((unsigned)blocks), dim3(256), lds, s, p, (int)tt, bi, bc, br)
  if (vec) {
    if (p.interleaved) DPA_ROTARY(true, true, false);
    else if (any) DPA_ROTARY(true, false, true);
    else DPA_ROTARY(true, false, false);
  } else {
    if (p.interleaved) DPA_ROTARY(false, true, false);
    else DPA_ROTARY(false, false, false);
  }
#undef DPA_ROTARY
  DPA_CHECK_HIP(hipGetLastError());
}

}  // namespace

void rotary_launch(const RotaryParams& p, int dtype, hipStream_t s) {
  if (p.tokens <= 0) return;
  if (p.H <= 0 || p.D <= 0 || p.pairs < 0 || 2 * p.pairs > p.D || p.pairs > 4096 || (long)3 * p.H * p.D >= (1l << 28))
    throw std::invalid_argument("rotary: head layout");
  DPA_DISPATCH_DTYPE(dtype, launch<T>(p, s));
}

}  // namespace dpa
