// Host entry points of the transformer-block kernels: residual_norm*.hip, rotary.hip, token_logprobs.hip,
// newton_schulz.hip, muon.hip.
#pragma once
#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include "../dtype.h"

namespace dpa {

// ---- s = x + scale[n] * gate * post(y), h = pre(s) on rows of C channels --------------------------------------------
enum NormKind : int { kNormNone = 0, kNormLayer = 1, kNormRms = 2 };
enum GateKind : int { kGateNone = 0, kGateChannel = 1, kGateSample = 2 };

struct ResidualNormFwd {
  const void* x = nullptr; const void* y = nullptr;      // y null: only h = pre(x)
  void* s = nullptr; void* h = nullptr;
  const float* post_w = nullptr; const float* post_b = nullptr;
  const float* pre_w = nullptr; const float* pre_b = nullptr;      // b null: no shift
  const float* gate = nullptr; const float* scale = nullptr;
  float* post_stat = nullptr; float* pre_stat = nullptr;           // [2][rows]: mean, 1 / deviation
  long rows = 0, per_sample = 1;
  int C = 0, post = 0, pre = 0, gate_kind = 0;
  float post_eps = 0.f, pre_eps = 0.f;
};
struct ResidualNormBwd {
  const void* ds = nullptr; const void* dh = nullptr;              // either may be null
  const void* x = nullptr; const void* y = nullptr;                // x: with `pre`; y null: none (pre of x alone)
  void* dx = nullptr; void* dy = nullptr;                          // dy null: the same as dx
  const float* post_w = nullptr; const float* post_b = nullptr; const float* pre_w = nullptr;
  const float* gate = nullptr; const float* scale = nullptr;
  const float* post_stat = nullptr; const float* pre_stat = nullptr;
  float* partial = nullptr;                                        // [residual_norm_parts()][vectors][C]
  float* gate_partial = nullptr;                                   // per-sample gate: [samples * splits][C]
  // vectors: pre_w, pre_b, post_w, post_b, gate (per channel); null where there is none.  beta 1 accumulates
  float* out[5] = {nullptr, nullptr, nullptr, nullptr, nullptr};
  float beta[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  float* dgate_sample = nullptr;                                   // [samples][C]
  long rows = 0, per_sample = 1;
  int C = 0, post = 0, pre = 0, gate_kind = 0;
};
constexpr int kResidualNormMaxChunks = 2048;                       // 16-byte chunks of one row
long residual_norm_parts(const ResidualNormBwd& p, int dtype, long* splits);
void residual_norm_fwd_launch(const ResidualNormFwd& p, int dtype, hipStream_t s);
void residual_norm_bwd_launch(const ResidualNormBwd& p, int dtype, hipStream_t s);

// ---- rotary positions of several axes on the packed projection [B][S][3][H][D] ---------------------------------------
enum PosKind : int { kPosI64 = 0, kPosI32 = 1, kPosF32 = 2, kPosF64 = 3 };
struct RotaryParams {
  const void* in = nullptr; void* out = nullptr;                   // out == in: in place
  const void* pos = nullptr; const void* freq = nullptr; const int* axis = nullptr;
  long tokens = 0, S = 1, in_batch = 0, in_token = 0, out_batch = 0, out_token = 0;      // strides in elements
  int H = 0, D = 0, pairs = 0, axes = 1, pos_kind = 0, pos_batched = 0, freq_f64 = 0, interleaved = 0, negate = 0;
};
void rotary_launch(const RotaryParams& p, int dtype, hipStream_t s);

// ---- log probability of a given class, entropy, k most probable classes of [N][C] logits ------------------------------
struct TokenLogprobs {
  const void* logits = nullptr; const long* target = nullptr;
  long N = 0, C = 0, ld = 0;
  int k = 0, splits = 1;
  float* logprob = nullptr; float* entropy = nullptr; float* norm = nullptr;     // norm: [N][2], m and log S
  float* top = nullptr; long* index = nullptr;                     // [N][k]
  float* stat = nullptr; uint64_t* keys = nullptr;                 // splits > 1: [N][splits][3], [N][splits][k]
};
struct TokenLogprobsBwd {
  const void* logits = nullptr; const long* target = nullptr;
  const float* norm = nullptr; const float* entropy = nullptr; const long* index = nullptr;
  const float* d_logprob = nullptr; const float* d_entropy = nullptr; const float* d_top = nullptr;   // each may be null
  void* dlogits = nullptr;                                         // [N][C], contiguous
  long N = 0, C = 0, ld = 0;
  int k = 0;
};
constexpr int kTokenTopMax = 64;
int token_logprobs_splits(long N, long C);
void token_logprobs_launch(const TokenLogprobs& p, int dtype, hipStream_t s);
void token_logprobs_bwd_launch(const TokenLogprobsBwd& p, int dtype, hipStream_t s);

// ---- Newton-Schulz orthogonalisation of a batch of matrices -----------------------------------------------------------
struct NewtonSchulz {
  const void* g = nullptr; void* out = nullptr;                    // [batch][rows][cols], contiguous
  void* work = nullptr;                                            // newton_schulz_workspace() bytes
  long batch = 0, rows = 0, cols = 0;
  int steps = 0;
  float a = 0.f, b = 0.f, c = 0.f;
  double eps = 0.0;
  bool fast = false;                                               // bf16 alone: products of single fp16 planes
};
size_t newton_schulz_workspace(long batch, long rows, long cols);
void newton_schulz_launch(const NewtonSchulz& p, int dtype, hipStream_t s);      // out may be g

// ---- Muon: momentum into the update, the update into the parameter; hyper: lr, momentum, weight decay, nesterov, step
// scale
struct MuonTensor {
  float* p; const void* g; float* buf; void* lp;                   // lp: low-precision copy of p, may be null
  long n, chunk0, at;                                              // elements, first chunk, place in the update buffer
  float scale; int pad;
};
int muon_chunk_elems();
void muon_begin_launch(const MuonTensor* table, int n, long chunks, int g_dtype, const float* hyper, const float* inv_scale,
                       const float* found_inf, float* update, hipStream_t s);
void muon_end_launch(const MuonTensor* table, int n, long chunks, int lp_dtype, const float* hyper, const float* found_inf,
                     const float* update, hipStream_t s);

}  // namespace dpa
