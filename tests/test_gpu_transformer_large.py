"""The transformer-block operators on tensors of more than 2^31 elements: the last rows (whose offsets do not fit 32 bits)
have to equal a call on those rows alone, bit for bit where both add up in one order."""
import pytest
import torch

import _transformer_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _free(request):
    print(request.node.name, flush=True)
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def _normal(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=g)


def F():
    from distributed_pytorch_amd.ops import functional

    return functional


def test_residual_norm():
    T, C, tail = 2200000, 1024, 64
    assert T * C > 1 << 31
    x, y = _normal((1, T, C), 0).requires_grad_(), _normal((1, T, C), 1).requires_grad_()
    w, b = torch.rand(C, device="cuda") + 0.5, torch.rand(C, device="cuda")
    pre = F().Norm(w, b, 1e-5, "layer")
    s, h = F().residual_norm(x, y, pre=pre)
    g = _normal((1, T, C), 2)
    (dx,) = torch.autograd.grad(h, [x], g)
    for lo in (0, T - tail):
        xs = x.detach()[:, lo:lo + tail].clone().requires_grad_()
        s2, h2 = F().residual_norm(xs, y.detach()[:, lo:lo + tail], pre=pre)
        (d2,) = torch.autograd.grad(h2, [xs], g[:, lo:lo + tail].contiguous())
        for a, c in ((s, s2), (h, h2), (dx, d2)):
            assert torch.equal(a[:, lo:lo + tail], c)


def test_rotary():
    S, H, D = 940000, 12, 64
    assert S * 3 * H * D > 1 << 31
    qkv = _normal((1, S, 3 * H * D), 0)
    pos = torch.arange(S, device="cuda").view(S, 1)
    freqs = 10000.0 ** (-torch.arange(32, device="cuda", dtype=torch.float64) / 32)
    axis = torch.zeros(32, dtype=torch.int32, device="cuda")
    out = F().rotary(qkv, pos, freqs, axis, H)
    for lo in (0, S - 100):
        part = F().rotary(qkv[:, lo:lo + 100].contiguous(), pos[lo:lo + 100], freqs, axis, H)
        assert torch.equal(out[:, lo:lo + 100], part)


def test_token_logprobs():
    N, V = 46000, 50257
    assert N * V > 1 << 31
    z = _normal((N, V), 0).requires_grad_()
    t = torch.arange(N, device="cuda") % V
    lp, ent, top, idx = F().token_logprobs(z, t, 8)
    (d,) = torch.autograd.grad(lp.sum() + ent.sum(), z)
    for lo in (0, N - 1100):
        zs = z.detach()[lo:lo + 1100].clone().requires_grad_()
        part = F().token_logprobs(zs, t[lo:lo + 1100], 8)
        (d2,) = torch.autograd.grad(part[0].sum() + part[1].sum(), zs)
        assert torch.equal(idx[lo:lo + 1100], part[3])
        # a call of few rows gives a row more waves, so its sums are added up in another order: both are within the bound
        # that _transformer_ref derives for any order, and so within twice it of each other
        rows = slice(0, 4) if lo == 0 else slice(1096, 1100)
        ones = torch.ones(4, device="cuda")
        want = ref.token_logprobs(zs.detach()[rows], t[lo:lo + 1100][rows], 8, ones, ones, torch.zeros(4, 8, device="cuda"))
        for name, a, c in (("logprob", lp, part[0]), ("entropy", ent, part[1]), ("top", top, part[2]), ("d_logits", d, d2)):
            ref.within(a[lo:lo + 1100][rows], *want[name], name)
            ref.within(c[rows], *want[name], name)
            # (all rows: a rounding to bf16 each, 2 * 2^-8; the 32-bit sums are off by 220 * 2^-24 * 12 < 2^-12)
            assert torch.allclose(a[lo:lo + 1100].float(), c.float(), rtol=2.0 ** -7, atol=2.0 ** -12)
