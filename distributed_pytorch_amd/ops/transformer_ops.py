"""GPU implementations of the transformer-block operators: autograd wrappers over ``csrc/kernels/residual_norm*.hip``,
``rotary.hip``, ``token_logprobs.hip`` and ``newton_schulz.hip``.

Like ``hip_ops``: outputs and workspaces come from ``torch.empty`` per call (stream-ordered, safe to capture, nothing is
shared between two calls or two graphs), launches go to torch's current stream of the tensors' device, nothing
synchronises with the host.  Arguments are checked in ``functional``.
"""
from __future__ import annotations

import contextlib
import struct

import torch

from . import grad_sink
from .hip_ops import C, _deliver, _dense, _dt, _f32, _lp_copy_of, _p, _same_layout, _stamp, _stream

_KINDS = {None: 0, "layer": 1, "rms": 2}
_POS_KINDS = {torch.int64: 0, torch.int32: 1, torch.float32: 2, torch.float64: 3}


def _on(t: torch.Tensor):
    """The tensor's device as the current one while a kernel is launched (a launch goes to the current device's stream)."""
    if t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _contig(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _vec32(t):
    return None if t is None else _contig(_f32(t.detach()))


def _tracked(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ------------------------------------------------------------------------------------------
# residual sum with its norms
# ------------------------------------------------------------------------------------------
def _rn_shape(x):
    Cc = x.shape[-1]
    rows = x.numel() // Cc if x.numel() else 0
    return Cc, rows, max(1, rows // max(1, x.shape[0]))


def _rn_forward(x, y, post_w, post_b, pre_w, pre_b, gate, scale, cfg, want_stats):
    """-> (x, y, s, h, post_stat, pre_stat, fp32 vectors); y None: h = pre(x) alone."""
    post, post_eps, pre, pre_eps = cfg
    x, y = _contig(x), _contig(y)
    vecs = [_vec32(t) for t in (post_w, post_b, pre_w, pre_b, gate, scale)]
    Cc, rows, per = _rn_shape(x)
    s = torch.empty_like(x) if y is not None else None
    h = torch.empty_like(x) if pre else None
    post_stat = torch.empty((2, rows), dtype=torch.float32, device=x.device) if post and want_stats else None
    pre_stat = torch.empty((2, rows), dtype=torch.float32, device=x.device) if pre and want_stats else None
    with _on(x):
        C().residual_norm_fwd(x.data_ptr(), _p(y), _p(s), _p(h), _p(vecs[0]), _p(vecs[1]), _p(vecs[2]), _p(vecs[3]),
                              _p(vecs[4]), _p(vecs[5]), _p(post_stat), _p(pre_stat), rows, per, Cc, _KINDS[post],
                              _KINDS[pre], 0 if gate is None else gate.dim(), post_eps, pre_eps, _dt(x), _stream())
    return x, y, s, h, post_stat, pre_stat, vecs


def _rn_backward(ds, dh, x, y, post_stat, pre_stat, vecs, cfg, params, needs, need_x, need_y):
    """``params``: the caller's pre_w, pre_b, post_w, post_b, gate; ``needs``: which of them get a gradient.
    -> (dx, dy, their gradients: None where delivered to a sink)."""
    post, _, pre, _ = cfg
    post_w, post_b, pre_w, _, gate, scale = vecs
    ref = ds if ds is not None else dh
    Cc, rows, per = _rn_shape(ref)
    dev, code = ref.device, _dt(ref)
    ds, dh = _contig(ds), _contig(dh)
    gate_kind = 0 if gate is None else gate.dim()
    # without a norm, gate or scale of its own the block's gradient is that of the sum
    plain = post is None and gate is None and scale is None
    branch = need_y and not plain
    grads = any(needs)
    dx = torch.empty_like(ref, memory_format=torch.contiguous_format) if need_x or (need_y and not branch) else None
    want_branch = branch or any(needs[2:])
    dy = torch.empty_like(ref, memory_format=torch.contiguous_format) if want_branch else None
    out, beta, own, sinks = [0] * 5, [0.0] * 5, [None] * 5, []
    per_sample = gate_kind == 2
    taken = set()
    for i, (p, need) in enumerate(zip(params, needs)):
        if not need or (i == 4 and per_sample):
            continue
        sink = grad_sink.sink_of(p)
        # (a parameter used twice in one call: its second sum goes through a buffer of its own)
        if sink is not None and sink.view.is_contiguous() and id(sink) not in taken:
            taken.add(id(sink))
            sinks.append(sink)
            out[i], beta[i] = sink.view.data_ptr(), sink.beta()
        else:
            own[i] = torch.empty(Cc, dtype=torch.float32, device=dev)
            out[i] = own[i].data_ptr()
    partial = gate_partial = dgate = None
    with _on(ref):
        if rows:
            parts, splits = C().residual_norm_parts(rows, per, Cc, code, gate_kind)
            if any(out):
                partial = torch.empty((parts, 5, Cc), dtype=torch.float32, device=dev)
            if per_sample and needs[4]:
                gate_partial = torch.empty((rows // per * splits, Cc), dtype=torch.float32, device=dev)
                dgate = torch.empty((rows // per, Cc), dtype=torch.float32, device=dev)
            C().residual_norm_bwd(_p(ds), _p(dh), _p(x), _p(y), _p(dx), _p(dy), _p(post_w), _p(post_b), _p(pre_w), _p(gate),
                                  _p(scale), _p(post_stat), _p(pre_stat), _p(partial), _p(gate_partial), out, beta, _p(dgate),
                                  rows, per, Cc, _KINDS[post], _KINDS[pre], gate_kind, code, _stream())
        elif grads:                        # no rows: every sum is zero
            for i, t in enumerate(own):
                if t is not None:
                    t.zero_()
            for sk in sinks:
                if sk.beta() == 0.0:
                    sk.view.zero_()
            if per_sample and needs[4]:
                dgate = torch.zeros_like(gate)
        for sk in sinks:
            sk.delivered()
        got = []
        for i, (p, need) in enumerate(zip(params, needs)):
            g = own[i] if not (i == 4 and per_sample) else dgate
            got.append(None if not need or g is None else _deliver(p, g.to(p.dtype).reshape(p.shape)))
    if need_y and not branch:
        dy = dx
    return dx if need_x else None, dy if need_y else None, got


class _ResidualNormFn(torch.autograd.Function):
    """s = x + scale * gate * post(y) and h = pre(s) in one pass; one pass backward (+ the fold of the parameter sums)."""

    @staticmethod
    def forward(ctx, x, y, post_w, post_b, pre_w, pre_b, gate, scale, cfg):
        x, y, s, h, post_stat, pre_stat, vecs = _rn_forward(x, y, post_w, post_b, pre_w, pre_b, gate, scale, cfg, True)
        ctx.save_for_backward(x if cfg[2] else None, y if cfg[0] or cfg[2] or gate is not None else None, post_stat, pre_stat,
                              *vecs)
        ctx.refs, ctx.cfg = (pre_w, pre_b, post_w, post_b, gate), cfg
        ctx.set_materialize_grads(False)
        return (s, h) if h is not None else s

    @staticmethod
    def backward(ctx, ds, dh=None):
        x, y, post_stat, pre_stat, *vecs = ctx.saved_tensors
        n = ctx.needs_input_grad
        needs = (n[4], n[5], n[2], n[3], n[6])
        if ds is None and dh is None:
            return (None,) * 9
        dx, dy, (g_pw, g_pb, g_qw, g_qb, g_gate) = _rn_backward(ds, dh, x, y, post_stat, pre_stat, vecs, ctx.cfg, ctx.refs,
                                                                needs, n[0], n[1])
        return dx, dy, g_qw, g_qb, g_pw, g_pb, g_gate, None, None


def residual_norm(x, y, post, gate, scale, pre):
    cfg = (None if post is None else post.kind, 0.0 if post is None else float(post.eps),
           None if pre is None else pre.kind, 0.0 if pre is None else float(pre.eps))
    pw, pb = (None, None) if post is None else (post.weight, post.bias)
    qw, qb = (None, None) if pre is None else (pre.weight, pre.bias)
    if not _tracked(x, y, pw, pb, qw, qb, gate):
        _, _, s, h, *_ = _rn_forward(x, y, pw, pb, qw, qb, gate, scale, cfg, False)
        return (s, h) if pre is not None else s
    grad_sink.note_use(pw, pb, qw, qb, gate)
    return _ResidualNormFn.apply(x, y, pw, pb, qw, qb, gate, scale, cfg)


class _NormFn(torch.autograd.Function):
    """h = pre(x) alone (the norm in front of a first block)."""

    @staticmethod
    def forward(ctx, x, w, b, cfg):
        x, _, _, h, _, stat, vecs = _rn_forward(x, None, None, None, w, b, None, None, cfg, True)
        ctx.save_for_backward(x, stat, *vecs)
        ctx.refs, ctx.cfg = (w, b, None, None, None), cfg
        return h

    @staticmethod
    def backward(ctx, dh):
        x, stat, *vecs = ctx.saved_tensors
        n = ctx.needs_input_grad
        dx, _, got = _rn_backward(None, dh, x, None, None, stat, vecs, ctx.cfg, ctx.refs,
                                  (n[1], n[2], False, False, False), n[0], False)
        return dx, got[0], got[1], None


def rms_norm(x, weight, eps):
    cfg = (None, 0.0, "rms", float(eps))
    if not _tracked(x, weight):
        return _rn_forward(x, None, None, None, weight, None, None, None, cfg, False)[3]
    grad_sink.note_use(weight)
    return _NormFn.apply(x, weight, None, cfg)


# ------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------
def _rotary_launch(src, out, pos, freqs, axis, H, interleaved, negate):
    B, S, W3 = src.shape
    with _on(src):
        C().rotary(src.data_ptr(), out.data_ptr(), pos.data_ptr(), freqs.data_ptr(), axis.data_ptr(), B * S, max(S, 1),
                   src.stride(0), src.stride(1), out.stride(0), out.stride(1), H, W3 // (3 * H), freqs.numel(),
                   pos.shape[-1], _POS_KINDS[pos.dtype], int(pos.dim() == 3), int(freqs.dtype == torch.float64),
                   int(interleaved), int(negate), _dt(src), _stream())
    return out


def _rotary_src(t):
    return t if t.stride(-1) == 1 else t.contiguous()


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, pos, freqs, axis, H, interleaved):
        src = _rotary_src(qkv)
        out = torch.empty(src.shape, dtype=src.dtype, device=src.device)
        _rotary_launch(src, out, pos, freqs, axis, H, interleaved, False)
        ctx.save_for_backward(pos, freqs, axis)
        ctx.cfg = (H, interleaved)
        return out

    @staticmethod
    def backward(ctx, dout):
        pos, freqs, axis = ctx.saved_tensors
        src = _rotary_src(dout)
        d = torch.empty(src.shape, dtype=src.dtype, device=src.device)
        return _rotary_launch(src, d, pos, freqs, axis, ctx.cfg[0], ctx.cfg[1], True), None, None, None, None, None


def rotary(qkv, positions, freqs, axis, num_heads, interleaved, inplace):
    pos, freqs = _contig(positions), _contig(freqs)
    axis = _contig(axis if axis.dtype == torch.int32 else axis.to(torch.int32))
    if inplace:
        return _rotary_launch(qkv, qkv, pos, freqs, axis, num_heads, interleaved, False)
    if not _tracked(qkv):
        src = _rotary_src(qkv.detach())
        out = torch.empty(src.shape, dtype=src.dtype, device=src.device)
        return _rotary_launch(src, out, pos, freqs, axis, num_heads, interleaved, False)
    return _RotaryFn.apply(qkv, pos, freqs, axis, int(num_heads), bool(interleaved))


# ------------------------------------------------------------------------------------------
# log probabilities of given classes
# ------------------------------------------------------------------------------------------
def _logprobs_forward(logits, target, k):
    z = logits if logits.stride(1) == 1 else logits.contiguous()
    N, V = z.shape
    dev = z.device
    t = target if target.dtype == torch.int64 and target.is_contiguous() else target.long().contiguous()
    lp, ent = (torch.empty(N, dtype=torch.float32, device=dev) for _ in range(2))
    norm = torch.empty((N, 2), dtype=torch.float32, device=dev)
    top = torch.empty((N, k), dtype=torch.float32, device=dev)
    idx = torch.empty((N, k), dtype=torch.int64, device=dev)
    with _on(z):
        splits = C().token_logprobs_splits(N, V, _dt(z))
        stat = keys = None
        if splits > 1:
            stat = torch.empty((N, splits, 3), dtype=torch.float32, device=dev)
            keys = torch.empty((N, splits, k), dtype=torch.int64, device=dev)
        C().token_logprobs(z.data_ptr(), t.data_ptr(), N, V, z.stride(0), k, splits, lp.data_ptr(), ent.data_ptr(),
                           norm.data_ptr(), top.data_ptr(), idx.data_ptr(), _p(stat), _p(keys), _dt(z), _stream())
    return z, t, lp, ent, norm, top, idx


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, k):
        z, t, lp, ent, norm, top, idx = _logprobs_forward(logits, target, k)
        ctx.save_for_backward(z, t, norm, ent, idx)
        ctx.k = k
        ctx.mark_non_differentiable(idx)
        ctx.set_materialize_grads(False)
        return lp, ent, top, idx

    @staticmethod
    def backward(ctx, d_lp, d_ent, d_top, _):
        z, t, norm, ent, idx = ctx.saved_tensors
        if d_lp is None and d_ent is None and d_top is None:
            return None, None, None
        N, V = z.shape
        d_lp, d_ent, d_top = (None if g is None else _contig(_f32(g)) for g in (d_lp, d_ent, d_top))
        dz = torch.empty((N, V), dtype=z.dtype, device=z.device)
        with _on(z):
            C().token_logprobs_bwd(z.data_ptr(), t.data_ptr(), norm.data_ptr(), ent.data_ptr(), idx.data_ptr(),
                                   _p(d_lp), _p(d_ent), _p(d_top), dz.data_ptr(), N, V, z.stride(0), ctx.k, _dt(z), _stream())
        return dz, None, None


def token_logprobs(logits, target, k):
    if not _tracked(logits):
        _, _, lp, ent, _, top, idx = _logprobs_forward(logits.detach(), target, k)
        return lp, ent, top, idx
    return _TokenLogprobsFn.apply(logits, target, k)


# ------------------------------------------------------------------------------------------
# Newton-Schulz
# ------------------------------------------------------------------------------------------
def newton_schulz(g, steps, coefficients, eps):
    src = _contig(g.detach())
    out = torch.empty_like(src)
    with _on(src):
        _schulz_launch(src, out, steps, coefficients, eps)
    return out


def _schulz_launch(src, out, steps, coefficients, eps) -> None:
    rows, cols = src.shape[-2:]
    batch = src.numel() // (rows * cols)
    a, b, c = (float(v) for v in coefficients)
    work = torch.empty(C().newton_schulz_workspace(batch, rows, cols), dtype=torch.uint8, device=src.device)
    C().newton_schulz(src.data_ptr(), out.data_ptr(), work.data_ptr(), batch, rows, cols, int(steps), a, b, c, float(eps),
                      _dt(src), _stream())


def matrix_shape(p):
    """(rows, columns) of a parameter as Muon sees it: a convolution's filters are rows of C * R * S elements, in the order
    of their memory (a permutation of the columns turns with the result)."""
    return p.shape[0], p.numel() // p.shape[0]


class MuonPlan:
    """Device-resident tables of the matrices of the ``orthogonal`` groups (cf. ``hip_ops.SgdPlan``): per group one launch
    that forms every update, ``newton_schulz`` in place for each shape, one launch that applies them.  The update buffer
    is allocated per step (a captured step holds one of its own)."""

    def __init__(self, opt):
        chunk = C().muon_chunk_elems()
        self.groups = []
        for group in opt.param_groups:
            if not group.get("orthogonal"):
                continue
            members = [p for p in group["params"] if p.grad is not None]
            if not members:
                continue
            shapes = {}
            for p in members:
                if p.dtype != torch.float32:
                    raise TypeError("FusedMuon HIP path needs fp32 parameters, got %s" % p.dtype)
                if not _dense(p):
                    raise ValueError("FusedMuon: parameter is not densely laid out")
                if not _same_layout(p, p.grad):
                    p.grad = torch.empty_like(p).copy_(p.grad)
                shapes.setdefault(matrix_shape(p), []).append(p)
            if len({p.grad.dtype for p in members}) != 1 or len({p.device for p in members}) != 1:
                raise TypeError("FusedMuon: one gradient dtype and device per group")
            lps = [_lp_copy_of(p) for p in members]
            lp_dtype = next((lp.dtype for lp in lps if lp is not None), torch.float32)
            raw, keep, plist, buckets, nchunks, place = [], [], [], [], 0, 0
            for (rows, cols), ps in shapes.items():
                buckets.append((place, len(ps), rows, cols))
                for p in ps:
                    buf = opt._momentum_buffer(p)
                    if not _same_layout(p, buf):
                        buf = torch.empty_like(p).copy_(buf)
                        opt.state[p]["momentum_buffer"] = buf
                    lp = _lp_copy_of(p)
                    lp = lp if lp is not None and lp.dtype == lp_dtype else None
                    raw.append(struct.pack("<QQQQqqqfi", p.data_ptr(), p.grad.data_ptr(), buf.data_ptr(), _p(lp), p.numel(),
                                           nchunks, place, max(1.0, rows / cols) ** 0.5, 0))
                    keep.extend([p, p.grad, buf, lp])
                    plist.append((p, lp))
                    nchunks += -(-p.numel() // chunk)
                    place += p.numel()
            raw = b"".join(raw)
            assert len(raw) == len(members) * C().muon_table_entry_bytes()
            device = members[0].device
            self.groups.append(dict(group=group, table=torch.frombuffer(bytearray(raw), dtype=torch.uint8).to(device),
                                    n=len(members), chunks=nchunks, elems=place, buckets=buckets, device=device,
                                    g_dtype=_dt(members[0].grad), lp_dtype=_dt(lp_dtype), plist=plist, keep=keep,
                                    hyper=torch.zeros(5, dtype=torch.float32, device=device), hyper_host=None))
        self.sig = self.signature(opt)

    @staticmethod
    def signature(opt):
        return tuple((p.data_ptr(), p.grad.data_ptr(), _p(_lp_copy_of(p)), _p(opt.state[p].get("momentum_buffer")))
                     for g in opt.param_groups if g.get("orthogonal") for p in g["params"] if p.grad is not None)

    def matches(self, opt) -> bool:
        return self.sig == self.signature(opt)

    def sync_hyper(self, opt) -> None:
        for gt in self.groups:
            g = gt["group"]
            host = (float(g["lr"]), float(g["momentum"]), float(g["weight_decay"]), 1.0 if g["nesterov"] else 0.0,
                    float(g["matrix_scale"]))
            if gt["hyper_host"] != host:
                gt["hyper"].copy_(torch.tensor(host, dtype=torch.float32), non_blocking=True)
                gt["hyper_host"] = host

    def launch(self, opt, scaler) -> None:
        if not torch.cuda.is_current_stream_capturing():
            self.sync_hyper(opt)
        inv = found = 0
        if scaler is not None and not scaler.is_identity:
            inv, found = scaler.inv_scale.data_ptr(), scaler.found_inf.data_ptr()
        for gt in self.groups:
            g = gt["group"]
            with _on(gt["table"]):
                u = torch.empty(gt["elems"], dtype=torch.float32, device=gt["device"])
                C().muon_begin(gt["table"].data_ptr(), gt["n"], gt["chunks"], gt["g_dtype"], gt["hyper"].data_ptr(), inv, found,
                               u.data_ptr(), _stream())
                for at, count, rows, cols in gt["buckets"]:
                    m = u[at:at + count * rows * cols].view(count, rows, cols)
                    _schulz_launch(m, m, g["ns_steps"], g["ns_coefficients"], g["ns_eps"])
                C().muon_end(gt["table"].data_ptr(), gt["n"], gt["chunks"], gt["lp_dtype"], gt["hyper"].data_ptr(), found,
                             u.data_ptr(), _stream())

    def stamp_copies(self) -> None:
        """After ``bump_generation``: the copies that the last launch wrote are current."""
        for gt in self.groups:
            for p, lp in gt["plist"]:
                if lp is not None:
                    p._dpa_wcache.wc_stamp = _stamp(p)
