"""GPU side of the transformer-block operators: ``csrc/transformer`` does allocation, launches and autograd in C++ (module
``_T``); here are the calls into it and the device tables of the Muon step.  ``_T`` checks arguments and returns None for
what it does not take; ``functional`` then raises the error that names it."""
from __future__ import annotations

import struct

import torch

from .. import backend
from . import grad_sink
from .hip_ops import _dense, _dt, _lp_copy_of, _p, _same_layout, _stamp

_T = None
_KINDS = {"layer": 1, "rms": 2}


def T():
    global _T
    if _T is None:
        _T = backend.require_transformer()
    return _T


def residual_norm(x, y, post, gate, scale, pre):
    pw, pb, pe, pk = (None, None, 0.0, 0) if post is None else (post[0], post[1], post[2], _KINDS.get(post[3], -1))
    qw, qb, qe, qk = (None, None, 0.0, 0) if pre is None else (pre[0], pre[1], pre[2], _KINDS.get(pre[3], -1))
    if y is None:
        return None
    sinks = grad_sink.any_sinks
    out = (_T or T()).residual_norm(x, y, pw, pb, pk, pe, qw, qb, qk, qe, gate, scale, sinks)
    if out is None:
        return None
    if sinks:
        grad_sink.note_use(pw, pb, qw, qb, gate)
    return out[0] if qk == 0 else out


def rms_norm(x, weight, eps):
    sinks = grad_sink.any_sinks
    out = (_T or T()).residual_norm(x, None, None, None, 0, 0.0, weight, None, _KINDS["rms"], eps, None, None, sinks)
    if out is None:
        return None
    if sinks:
        grad_sink.note_use(weight)
    return out[1]


def rotary(qkv, positions, freqs, axis, num_heads, interleaved, inplace):
    return (_T or T()).rotary(qkv, positions, freqs, axis, num_heads, interleaved, inplace)


def token_logprobs(logits, target, k):
    return (_T or T()).token_logprobs(logits, target, k)


def newton_schulz(g, steps, coefficients, eps, fast):
    a, b, c = coefficients
    return T().newton_schulz(g.detach(), None, steps, a, b, c, eps, fast)


def matrix_shape(p):
    """(rows, columns) of a parameter as Muon sees it: a convolution's filters are rows of C * R * S elements, in the order
    of their memory (a permutation of the columns turns with the result)."""
    return p.shape[0], p.numel() // p.shape[0]


class MuonPlan:
    """Device-resident tables of the matrices of the ``orthogonal`` groups (cf. ``hip_ops.SgdPlan``): per group one launch
    that forms every update, ``newton_schulz`` in place for each shape, one launch that applies them.  The update buffer
    is allocated per step (a captured step holds one of its own)."""

    def __init__(self, opt):
        chunk = T().muon_chunk_elems()
        self.groups = []
        for group in opt.param_groups:
            if not group.get("orthogonal"):
                continue
            members = [p for p in group["params"] if p.grad is not None]
            if not members:
                continue
            shapes = {}
            for p in members:
                if not p.is_cuda:
                    raise ValueError("FusedMuon: parameters on the CPU beside others on the GPU")
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
            assert len(raw) == len(members) * T().muon_table_entry_bytes()
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
        inv = found = None
        if scaler is not None and not scaler.is_identity:
            inv, found = scaler.inv_scale, scaler.found_inf
        for gt in self.groups:
            g = gt["group"]
            a, b, c = g["ns_coefficients"]
            u = torch.empty(gt["elems"], dtype=torch.float32, device=gt["device"])
            T().muon_begin(gt["table"], gt["n"], gt["chunks"], gt["g_dtype"], gt["hyper"], inv, found, u)
            for at, count, rows, cols in gt["buckets"]:
                m = u[at:at + count * rows * cols].view(count, rows, cols)
                T().newton_schulz(m, m, g["ns_steps"], a, b, c, g["ns_eps"], False)
            T().muon_end(gt["table"], gt["n"], gt["chunks"], gt["lp_dtype"], gt["hyper"], found, u)

    def stamp_copies(self) -> None:
        """After ``bump_generation``: the copies that the last launch wrote are current."""
        for gt in self.groups:
            for p, lp in gt["plist"]:
                if lp is not None:
                    p._dpa_wcache.wc_stamp = _stamp(p)
