"""The transformer-block operators on the CPU backend: results, gradients and refusals."""
import math

import pytest
import torch

import _transformer_ref as ref
from distributed_pytorch_amd.ops import functional as F


def test_residual_norm_reference():
    g = torch.Generator().manual_seed(0)
    for post, pre, gk, sc in (("layer", "rms", "channel", True), (None, "layer", None, False), ("rms", None, "sample", True)):
        x, y, ds, dh = (torch.randn(3, 5, 24, generator=g) for _ in range(4))
        mk = lambda kind: None if kind is None else F.Norm(torch.rand(24, generator=g) + 0.5,
                                                           torch.randn(24, generator=g) if kind == "layer" else None, 1e-5, kind)
        p, q = mk(post), mk(pre)
        gate = None if gk is None else torch.randn((24,) if gk == "channel" else (3, 24), generator=g)
        scale = torch.tensor([0.0, 1.25, 1.25]) if sc else None
        want = ref.residual_norm(x, y, p, gate, scale, q, ds, dh if q is not None else None)
        leaves = [t for t in (x, y, gate) if t is not None]
        for t in leaves:
            t.requires_grad_()
        out = F.residual_norm(x, y, post=p, gate=gate, scale=scale, pre=q)
        s, h = out if q is not None else (out, None)
        ref.within(s, *want["s"], "s")
        outs, grads = ([s, h], [ds, dh]) if q is not None else ([s], [ds])
        if q is not None:
            ref.within(h, *want["h"], "h")
        got = torch.autograd.grad(outs, leaves, grads)
        for name, t in zip([n for n, v in (("d_x", x), ("d_y", y), ("d_gate", gate)) if v is not None], got):
            ref.within(t, want[name][0], 4 * want[name][1], name)      # torch's own sums, another order


def test_rotary_reference():
    g = torch.Generator().manual_seed(0)
    for inter in (False, True):
        for P in (0, 3, 8):
            qkv = torch.randn(2, 7, 3 * 2 * 16, generator=g)
            pos = torch.randint(0, 1000, (2, 7, 2), generator=g)
            freqs, axis = torch.rand(P, generator=g), torch.randint(0, 2, (P,), generator=g)
            out = F.rotary(qkv, pos, freqs, axis, 2, interleaved=inter)
            ref.within(out, *ref.rotary(qkv, pos, freqs, axis, 2, inter), "out")
            same = qkv.clone()
            assert F.rotary(same, pos, freqs, axis, 2, interleaved=inter, inplace=True) is same and torch.equal(same, out)


def test_token_logprobs_reference():
    g = torch.Generator().manual_seed(0)
    z = torch.randn(6, 50, generator=g)
    z[1, ::3] = -math.inf
    z[2] = -math.inf
    z[3] = 1.0
    t = torch.tensor([3, 1, 0, 4, -1, 50])
    z.requires_grad_()
    d_lp, d_ent = torch.randn(6, generator=g), torch.randn(6, generator=g)
    lp, ent, top, idx = F.token_logprobs(z, t, 4)
    want = ref.token_logprobs(z, t, 4, d_lp, d_ent)
    assert torch.equal(idx, want["index"][0])
    for name, got in (("logprob", lp), ("entropy", ent), ("top", top)):
        ref.within(got, *want[name], name)
    (d,) = torch.autograd.grad([lp, ent], [z], [d_lp, d_ent])
    ref.within(d, want["d_logits"][0], 4 * want["d_logits"][1], "d_logits")


def test_newton_schulz_reference():
    g = torch.randn(2, 20, 33, generator=torch.Generator().manual_seed(0))
    for m in (g, g.mT):
        got = F.newton_schulz(m)
        value, rel = ref.newton_schulz(m)
        assert float((got.double() - value).norm() / value.norm()) <= rel
        s = torch.linalg.svdvals(got.double())
        assert float(s.max()) < 1.3 and float(s.min()) > 0.3


def _raises(kind, f, *a, **k):
    with pytest.raises(kind):
        f(*a, **k)


def test_residual_norm_refusals():
    x = torch.randn(2, 3, 8)
    w, b = torch.ones(8), torch.zeros(8)
    r = F.residual_norm
    _raises(ValueError, r, x, x[:, :2])
    _raises(ValueError, r, x, x.bfloat16())
    _raises(TypeError, r, x.double(), x.double())
    _raises(TypeError, r, x.int(), x.int())
    _raises(ValueError, r, x[0, 0], x[0, 0])
    _raises(ValueError, r, torch.zeros(2, 0), torch.zeros(2, 0))
    _raises(ValueError, r, torch.zeros(1, 8193), torch.zeros(1, 8193))
    _raises(ValueError, r, x, x, pre=F.Norm(w[:7], b))
    _raises(ValueError, r, x, x, pre=F.Norm(w, b[:7]))
    _raises(ValueError, r, x, x, post=F.Norm(w, b, 1e-5, "batch"))
    _raises(ValueError, r, x, x, post=F.Norm(w, b, 1e-5, "rms"))
    _raises(ValueError, r, x, x, post=F.Norm(w, b, -1.0))
    _raises(ValueError, r, x, x, post=F.Norm(w, b, math.nan))
    _raises(ValueError, r, x, x, gate=torch.ones(3))
    _raises(ValueError, r, x, x, gate=torch.ones(3, 8))
    _raises(ValueError, r, x, x, scale=torch.ones(3))
    _raises(ValueError, r, x, x, scale=torch.ones(2, requires_grad=True))
    _raises(ValueError, F.rms_norm, x, w[:5])


def test_rotary_refusals():
    qkv, pos, fr, ax = torch.randn(2, 5, 3 * 2 * 8), torch.zeros(5, 2), torch.ones(4), torch.zeros(4, dtype=torch.int32)
    r = F.rotary
    assert r(qkv, pos, fr, ax, 2).shape == qkv.shape
    _raises(ValueError, r, qkv[0], pos, fr, ax, 2)
    _raises(ValueError, r, qkv, pos, fr, ax, 5)
    _raises(ValueError, r, qkv, pos, fr, ax, 0)
    _raises(ValueError, r, qkv, pos[:4], fr, ax, 2)
    _raises(ValueError, r, qkv, pos.expand(3, 5, 2), fr, ax, 2)
    _raises(ValueError, r, qkv, pos[:, :0], fr, ax, 2)
    _raises(TypeError, r, qkv, pos.half(), fr, ax, 2)
    _raises(TypeError, r, qkv, pos, fr.half(), ax, 2)
    _raises(TypeError, r, qkv, pos, fr, ax.float(), 2)
    _raises(ValueError, r, qkv, pos, torch.ones(5), torch.zeros(5, dtype=torch.int32), 2)
    _raises(ValueError, r, qkv, pos, fr, ax[:3], 2)
    _raises(ValueError, r, qkv, pos, fr.clone().requires_grad_(), ax, 2)
    _raises(TypeError, r, qkv.double(), pos, fr, ax, 2)
    _raises(ValueError, r, qkv.clone().requires_grad_(), pos, fr, ax, 2, inplace=True)
    _raises(ValueError, r, qkv[:, :1].expand(2, 5, 48), pos, fr, ax, 2, inplace=True)
    _raises(ValueError, r, torch.randn(2, 5, 96)[..., ::2], pos, fr, ax, 2, inplace=True)
    # tokens (0, 1) and (1, 0) in the same place
    _raises(ValueError, r, torch.randn(6 * 48).as_strided((2, 5, 48), (48, 48, 1)), pos, fr, ax, 2, inplace=True)
    crossed = torch.randn(5, 2, 48).transpose(0, 1)
    assert r(crossed, pos, fr, ax, 2, inplace=True) is crossed


def test_token_logprobs_refusals():
    z, t = torch.randn(3, 10), torch.zeros(3, dtype=torch.int64)
    r = F.token_logprobs
    _raises(ValueError, r, z, t[:2])
    _raises(ValueError, r, z, t, 11)
    _raises(ValueError, r, z, t, -1)
    _raises(ValueError, r, torch.randn(3, 100), t, 65)
    _raises(ValueError, r, torch.randn(3, 0), t)
    _raises(TypeError, r, z.double(), t)
    _raises(TypeError, r, z, t.float())


def test_newton_schulz_refusals():
    g = torch.randn(4, 5)
    r = F.newton_schulz
    _raises(ValueError, r, g[0])
    _raises(ValueError, r, torch.zeros(0, 4, 4))
    _raises(TypeError, r, g.double())
    _raises(ValueError, r, g, steps=0)
    _raises(ValueError, r, g, eps=0.0)
    _raises(ValueError, r, g, coefficients=(1.0, 2.0))
    _raises(ValueError, r, g, coefficients=(1.0, math.inf, 0.0))
    _raises(ValueError, r, g, coefficients=(4.0, 1.0, 1.0))
    _raises(ValueError, r, g.clone().requires_grad_())
