// pybind11 surface of the transformer-block kernels (kernels/transformer.h): addresses and streams as integers.
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include "kernels/transformer.h"

namespace py = pybind11;

namespace dpa {
namespace {
template <typename T> T* ptr(uintptr_t p) { return reinterpret_cast<T*>(p); }
hipStream_t st(uintptr_t s) { return reinterpret_cast<hipStream_t>(s); }
}  // namespace

void bind_transformer(py::module_& m) {
  m.attr("RESIDUAL_NORM_MAX_CHUNKS") = kResidualNormMaxChunks;
  m.attr("TOKEN_TOP_MAX") = kTokenTopMax;

  m.def("residual_norm_fwd",
        [](uintptr_t x, uintptr_t y, uintptr_t s, uintptr_t h, uintptr_t post_w, uintptr_t post_b, uintptr_t pre_w,
           uintptr_t pre_b, uintptr_t gate, uintptr_t scale, uintptr_t post_stat, uintptr_t pre_stat, long rows,
           long per_sample, int C, int post, int pre, int gate_kind, float post_eps, float pre_eps, int dtype,
           uintptr_t stream) {
          ResidualNormFwd p;
          p.x = ptr<const void>(x); p.y = ptr<const void>(y); p.s = ptr<void>(s); p.h = ptr<void>(h);
          p.post_w = ptr<const float>(post_w); p.post_b = ptr<const float>(post_b);
          p.pre_w = ptr<const float>(pre_w); p.pre_b = ptr<const float>(pre_b);
          p.gate = ptr<const float>(gate); p.scale = ptr<const float>(scale);
          p.post_stat = ptr<float>(post_stat); p.pre_stat = ptr<float>(pre_stat);
          p.rows = rows; p.per_sample = per_sample; p.C = C; p.post = post; p.pre = pre; p.gate_kind = gate_kind;
          p.post_eps = post_eps; p.pre_eps = pre_eps;
          residual_norm_fwd_launch(p, dtype, st(stream));
        });
  m.def("residual_norm_parts", [](long rows, long per_sample, int C, int dtype, int gate_kind) {
    long splits = 1;
    const long parts = residual_norm_parts(rows, per_sample, C, dtype, gate_kind, &splits);
    return std::make_pair(parts, splits);
  });
  m.def("residual_norm_bwd",
        [](uintptr_t ds, uintptr_t dh, uintptr_t x, uintptr_t y, uintptr_t dx, uintptr_t dy, uintptr_t post_w,
           uintptr_t post_b, uintptr_t pre_w, uintptr_t gate, uintptr_t scale, uintptr_t post_stat, uintptr_t pre_stat,
           uintptr_t partial, uintptr_t gate_partial, const std::vector<uintptr_t>& out, const std::vector<float>& beta,
           uintptr_t dgate_sample, long rows, long per_sample, int C, int post, int pre, int gate_kind, int dtype,
           uintptr_t stream) {
          if (out.size() != 5 || beta.size() != 5) throw std::invalid_argument("residual_norm_bwd: five outputs");
          ResidualNormBwd p;
          p.ds = ptr<const void>(ds); p.dh = ptr<const void>(dh); p.x = ptr<const void>(x); p.y = ptr<const void>(y);
          p.dx = ptr<void>(dx); p.dy = ptr<void>(dy);
          p.post_w = ptr<const float>(post_w); p.post_b = ptr<const float>(post_b); p.pre_w = ptr<const float>(pre_w);
          p.gate = ptr<const float>(gate); p.scale = ptr<const float>(scale);
          p.post_stat = ptr<const float>(post_stat); p.pre_stat = ptr<const float>(pre_stat);
          p.partial = ptr<float>(partial); p.gate_partial = ptr<float>(gate_partial);
          for (int i = 0; i < 5; ++i) { p.out[i] = ptr<float>(out[i]); p.beta[i] = beta[i]; }
          p.dgate_sample = ptr<float>(dgate_sample);
          p.rows = rows; p.per_sample = per_sample; p.C = C; p.post = post; p.pre = pre; p.gate_kind = gate_kind;
          residual_norm_bwd_launch(p, dtype, st(stream));
        });
  m.def("rotary",
        [](uintptr_t in, uintptr_t out, uintptr_t pos, uintptr_t freq, uintptr_t axis, long tokens, long S, long in_batch,
           long in_token, long out_batch, long out_token, int H, int D, int pairs, int axes, int pos_kind, int pos_batched,
           int freq_f64, int interleaved, int negate, int dtype, uintptr_t stream) {
          RotaryParams p;
          p.in = ptr<const void>(in); p.out = ptr<void>(out); p.pos = ptr<const void>(pos); p.freq = ptr<const void>(freq);
          p.axis = ptr<const int>(axis);
          p.tokens = tokens; p.S = S; p.in_batch = in_batch; p.in_token = in_token; p.out_batch = out_batch;
          p.out_token = out_token; p.H = H; p.D = D; p.pairs = pairs; p.axes = axes; p.pos_kind = pos_kind;
          p.pos_batched = pos_batched; p.freq_f64 = freq_f64; p.interleaved = interleaved; p.negate = negate;
          rotary_launch(p, dtype, st(stream));
        });
  m.def("token_logprobs_splits", &token_logprobs_splits);
  m.def("token_logprobs",
        [](uintptr_t logits, uintptr_t target, long N, long C, long ld, int k, int splits, uintptr_t logprob,
           uintptr_t entropy, uintptr_t norm, uintptr_t top, uintptr_t index, uintptr_t stat, uintptr_t keys, int dtype,
           uintptr_t stream) {
          TokenLogprobs p;
          p.logits = ptr<const void>(logits); p.target = ptr<const long>(target);
          p.N = N; p.C = C; p.ld = ld; p.k = k; p.splits = splits;
          p.logprob = ptr<float>(logprob); p.entropy = ptr<float>(entropy); p.norm = ptr<float>(norm);
          p.top = ptr<float>(top); p.index = ptr<long>(index); p.stat = ptr<float>(stat); p.keys = ptr<uint64_t>(keys);
          token_logprobs_launch(p, dtype, st(stream));
        });
  m.def("token_logprobs_bwd",
        [](uintptr_t logits, uintptr_t target, uintptr_t norm, uintptr_t entropy, uintptr_t index, uintptr_t d_logprob,
           uintptr_t d_entropy, uintptr_t d_top, uintptr_t dlogits, long N, long C, long ld, int k, int dtype,
           uintptr_t stream) {
          TokenLogprobsBwd p;
          p.logits = ptr<const void>(logits); p.target = ptr<const long>(target); p.norm = ptr<const float>(norm);
          p.entropy = ptr<const float>(entropy); p.index = ptr<const long>(index);
          p.d_logprob = ptr<const float>(d_logprob); p.d_entropy = ptr<const float>(d_entropy);
          p.d_top = ptr<const float>(d_top); p.dlogits = ptr<void>(dlogits);
          p.N = N; p.C = C; p.ld = ld; p.k = k;
          token_logprobs_bwd_launch(p, dtype, st(stream));
        });
  m.def("newton_schulz_workspace", &newton_schulz_workspace);
  m.def("newton_schulz",
        [](uintptr_t g, uintptr_t out, uintptr_t work, long batch, long rows, long cols, int steps, float a, float b, float c,
           double eps, int dtype, uintptr_t stream) {
          NewtonSchulz p;
          p.g = ptr<const void>(g); p.out = ptr<void>(out); p.work = ptr<void>(work);
          p.batch = batch; p.rows = rows; p.cols = cols; p.steps = steps; p.a = a; p.b = b; p.c = c; p.eps = eps;
          newton_schulz_launch(p, dtype, st(stream));
        });
  m.def("muon_chunk_elems", &muon_chunk_elems);
  m.def("muon_table_entry_bytes", []() { return sizeof(MuonTensor); });
  m.def("muon_begin", [](uintptr_t table, int n, long chunks, int g_dtype, uintptr_t hyper, uintptr_t inv_scale,
                         uintptr_t found_inf, uintptr_t update, uintptr_t stream) {
    muon_begin_launch(ptr<const MuonTensor>(table), n, chunks, g_dtype, ptr<const float>(hyper), ptr<const float>(inv_scale),
                      ptr<const float>(found_inf), ptr<float>(update), st(stream));
  });
  m.def("muon_end", [](uintptr_t table, int n, long chunks, int lp_dtype, uintptr_t hyper, uintptr_t found_inf,
                       uintptr_t update, uintptr_t stream) {
    muon_end_launch(ptr<const MuonTensor>(table), n, chunks, lp_dtype, ptr<const float>(hyper), ptr<const float>(found_inf),
                    ptr<const float>(update), st(stream));
  });
}

}  // namespace dpa
