"""The transformer operators' refusals, modules and optimizer at their edges, on the CPU backend."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from distributed_pytorch_amd import models
from distributed_pytorch_amd.ops import functional as F


def test_newton_schulz_fast_is_for_bf16():
    g = torch.randn(6, 9)
    for dtype in (torch.float32, torch.float16):
        with pytest.raises(ValueError, match="bfloat16"):
            F.newton_schulz(g.to(dtype), fast=True)
    assert torch.equal(F.newton_schulz(g.bfloat16(), fast=True), F.newton_schulz(g.bfloat16()))     # (32 bits here either way)


def _native_calls():
    """{name: (call of the native module with one floating-point argument, that argument)}: what it refuses, it refuses before it
    looks at the device."""
    from distributed_pytorch_amd.ops.transformer_ops import T

    x, y, w = torch.randn(2, 3, 16), torch.randn(2, 3, 16), torch.randn(16)
    qkv, pos, freqs, axis = torch.randn(1, 4, 48), torch.zeros(4, 2), torch.ones(8), torch.zeros(8, dtype=torch.int32)

    def rn(**kw):
        a = dict(x=x, y=y, post_w=None, post_b=None, post=0, post_eps=0.0, pre_w=None, pre_b=None, pre=0, pre_eps=0.0, gate=None,
                 scale=None)
        a.update(kw)
        return T().residual_norm(*a.values(), False)

    calls = {k: (lambda v, k=k: rn(**{k: v}), v) for k, v in (
        ("x", x), ("y", y), ("post_w", w), ("post_b", w), ("pre_w", w), ("pre_b", w), ("gate", w), ("scale", torch.ones(2)))}
    calls["qkv"] = (lambda v: T().rotary(v, pos, freqs, axis, 1, False, False), qkv)
    calls["inplace"] = (lambda v: T().rotary(v, pos, freqs, axis, 1, False, True), qkv)
    calls["positions"] = (lambda v: T().rotary(qkv, v, freqs, axis, 1, False, False), pos)
    calls["freqs"] = (lambda v: T().rotary(qkv, pos, v, axis, 1, False, False), freqs)
    calls["logits"] = (lambda v: T().token_logprobs(v, torch.zeros(2, dtype=torch.int64), 3), torch.randn(2, 9))
    return calls


def test_native_module_refuses_tangents():
    for name, (call, v) in _native_calls().items():
        assert call(v) is None, name                # (not a GPU tensor: not taken, and no error)
        with fwd.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(fwd.make_dual(v, torch.ones_like(v)))


def test_native_module_refuses_what_records_it():
    """Traces, fake tensors, functional wrappers, tensor subclasses: the results would be buffers that nothing fills, and the
    arguments have no memory to read."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    class Watched(torch.Tensor):
        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            return NotImplemented

    for name, (call, v) in _native_calls().items():
        with pytest.raises((NotImplementedError, RuntimeError), match="traced"):
            torch.jit.trace(call, (v,), check_trace=False)
        with pytest.raises(NotImplementedError, match="traced|subclasses"):
            make_fx(lambda u: call(u))(v)
        mode = FakeTensorMode(allow_non_fake_inputs=True)
        fake = mode.from_tensor(v)
        with pytest.raises(NotImplementedError, match="subclasses"):
            call(fake)
        with mode, pytest.raises(NotImplementedError, match="traced"):
            call(v)
        with pytest.raises(NotImplementedError, match="subclasses"):
            call(torch._to_functional_tensor(v))
        with pytest.raises(NotImplementedError, match="subclasses"):
            call(torch.Tensor._make_subclass(Watched, v))
        with pytest.raises(NotImplementedError, match="subclasses"):
            torch.func.vmap(lambda u: call(u), in_dims=0)(torch.stack([v, v]))
        assert call(v) is None and call(torch.nn.Parameter(v) if v.is_floating_point() and name not in ("scale", "positions", "freqs")
                                        else v) is None


def test_newton_schulz_refuses_tangents():
    with fwd.dual_level():
        F.newton_schulz(torch.ones(3, 4))
        with pytest.raises(ValueError, match="no gradient"):
            F.newton_schulz(fwd.make_dual(torch.ones(3, 4), torch.ones(3, 4)))


def _tiny_vit(rotary=False):
    torch.manual_seed(0)
    m = models.vit.VisionTransformer(32, 8, 2, 2, 32, 64, num_classes=5, rotary=rotary)
    torch.nn.init.normal_(m.heads.head.weight)
    return m


class _Renamed(torch.nn.Module):
    """A module in place of another that takes one argument, as checkpointing wrappers are."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return self.inner(x)


@pytest.mark.parametrize("rotary", [False, True])
def test_hooks_of_the_encoder(rotary):
    """Hooks on the sequence of blocks, the blocks, their norms and attention fire, with the activations alone as arguments
    where there are no rotary positions."""
    m, x, seen = _tiny_vit(rotary), torch.randn(2, 3, 32, 32), []
    want = m(x)
    block = m.encoder.layers[1]
    for name, mod in (("layers", m.encoder.layers), ("block", block), ("ln_1", block.ln_1), ("attention", block.self_attention),
                      ("ln_2", block.ln_2), ("ln", m.encoder.ln)):
        mod.register_forward_hook(lambda mod, args, out, name=name: seen.append((name, len(args))))
    assert torch.equal(m(x), want)
    more = 2 if rotary else 1
    assert sorted(seen) == sorted([("layers", more), ("block", more), ("ln_1", 1), ("attention", more), ("ln_2", 1), ("ln", 1)])
    assert isinstance(m.encoder.layers, torch.nn.Sequential) and len(m.encoder.layers[:1]) == 1


def test_blocks_that_take_the_activations_alone():
    m, x = _tiny_vit(), torch.randn(2, 3, 32, 32)
    want = m(x)
    m.encoder.layers[0] = _Renamed(m.encoder.layers[0])
    m.encoder.layers[1].self_attention = _Renamed(m.encoder.layers[1].self_attention)
    assert torch.equal(m(x), want)


def _block_of(arch, **kw):
    """(model, input, a block of it, what the fused pass of that block stands in for)"""
    from distributed_pytorch_amd.models import convnext, swin

    torch.manual_seed(0)
    if arch == "vit":
        m = _tiny_vit()
        b = m.encoder.layers[0]
        return m, torch.randn(2, 3, 32, 32), [m.encoder.layers, b, b.ln_1, b.ln_2, m.encoder.ln]
    if arch == "convnext":
        b = convnext.CNBlock(16, 0.5, 0.5)
        return b, torch.randn(2, 8, 8, 16), [b.stochastic_depth]
    kind = swin.SwinTransformerBlock if arch == "swin" else swin.SwinTransformerBlockV2
    b = kind(32, 2, [4, 4], [0, 0], stochastic_depth_prob=0.5)
    return b, torch.randn(2, 8, 8, 32), [b.norm1, b.norm2, b.stochastic_depth]


@pytest.mark.parametrize("arch", ["vit", "swin", "swin_v2", "convnext"])
def test_fused_passes_step_aside_for_hooks(arch, monkeypatch):
    """A hook on anything that the fused pass would stand in for is called, and may change what its module returns."""
    monkeypatch.setattr(F, "_FUSE_RESIDUAL_NORM", True)
    m, x, inside = _block_of(arch)
    m.train()
    for mod in inside:
        seen = []
        for hook in (mod.register_forward_hook(lambda *a: seen.append(0)), mod.register_forward_pre_hook(lambda *a: seen.append(0)),
                     mod.register_full_backward_hook(lambda *a: seen.append(0))):
            del seen[:]
            m(x.clone().requires_grad_()).sum().backward()
            assert seen, (mod, hook)
            hook.remove()
    seen = []
    hook = torch.nn.modules.module.register_module_forward_hook(lambda mod, *a: seen.append(mod))
    try:
        m(x)
    finally:
        hook.remove()
    assert all(any(mod is s for s in seen) for mod in inside)


@pytest.mark.parametrize("arch", ["vit", "swin", "swin_v2", "convnext"])
def test_fused_passes_step_aside_for_other_modules(arch, monkeypatch):
    """A norm or stochastic depth that is another module, or whose forward was replaced, is the one that runs."""
    monkeypatch.setattr(F, "_FUSE_RESIDUAL_NORM", True)
    m, x, inside = _block_of(arch)
    m.eval()
    mod = inside[-1]                     # the last norm, or stochastic depth
    mod.forward = lambda v: torch.zeros_like(v)
    out = m(x)
    if arch == "vit":
        assert torch.equal(out, m.heads.head.bias.expand_as(out))
    else:
        monkeypatch.setattr(F, "_FUSE_RESIDUAL_NORM", False)
        assert torch.equal(m(x), out)
    del mod.forward
    if arch == "vit":
        m.encoder.layers[0] = _Renamed(m.encoder.layers[0])
        m(x)


@pytest.mark.parametrize("arch", ["swin", "swin_v2", "convnext"])
def test_fused_stochastic_depth_follows_its_own_mode(arch, monkeypatch):
    """Stochastic depth in evaluation mode inside a block that trains drops nothing."""
    m, x, inside = _block_of(arch)
    m.train()
    inside[-1].eval()
    got = []
    for fused in (False, True):
        monkeypatch.setattr(F, "_FUSE_RESIDUAL_NORM", fused)
        got.append(m(x))
    # 32 bits either way, additions in another order: 2^-24 each, some hundreds deep at most
    assert float((got[0] - got[1]).abs().max()) <= 1e-4 * float(got[0].abs().max())


def test_fused_encoder_without_blocks(monkeypatch):
    monkeypatch.setattr(F, "_FUSE_RESIDUAL_NORM", True)
    m = models.vit.VisionTransformer(32, 8, 0, 2, 32, 64, num_classes=5)
    assert m(torch.randn(1, 3, 32, 32)).shape == (1, 5)


# ------------------------------------------------------------------------------------------ FusedMuon
def _matrices(seed):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(6, 10, generator=g)), torch.nn.Parameter(torch.randn(7, generator=g))]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g)
    return ps


def test_muon_nesterov_of_a_group():
    """A group's own choice stands; the constructor's is for groups without one."""
    from distributed_pytorch_amd.optim import FusedMuon

    a, b = _matrices(0), _matrices(1)
    for of_all in (True, False):
        opt = FusedMuon([dict(params=a[:1], orthogonal=True, nesterov=not of_all), dict(params=b[:1], orthogonal=True),
                         dict(params=a[1:])], nesterov=of_all)
        assert [g["nesterov"] for g in opt.param_groups] == [not of_all, of_all, False]
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.ones(3, 4))], orthogonal=True))
        assert opt.param_groups[-1]["nesterov"] is of_all


@pytest.mark.parametrize("saved", [True, False])
def test_muon_resumes_with_the_checkpoints_nesterov(saved):
    """Whatever the new optimizer was built with: the steps after a resume are those of the run that was saved."""
    import copy

    from distributed_pytorch_amd.optim import FusedMuon

    a, b = _matrices(2), _matrices(2)
    x, y = FusedMuon(a, lr=0.1, nesterov=saved), FusedMuon(b, lr=0.1, nesterov=not saved)
    x.step()
    y.load_state_dict(copy.deepcopy(x.state_dict()))
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    for _ in range(2):
        x.step()
        y.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_muon_from_a_checkpoint_of_sgd_and_back():
    """The momentum goes over; which groups are orthogonalised stays the optimizer's own, and SGD updates every group."""
    import copy

    from distributed_pytorch_amd.optim import FusedMuon, FusedSGD

    a, b, c, d = (_matrices(4) for _ in range(4))
    sgd, muon = FusedSGD(a[:1], lr=0.1, momentum=0.9), FusedMuon([dict(params=b[:1], orthogonal=True)], lr=0.2, matrix_scale=0.5)
    sgd.step()
    muon.load_state_dict(copy.deepcopy(sgd.state_dict()))
    group = muon.param_groups[0]
    assert group["orthogonal"] is True and group["nesterov"] is True and group["matrix_scale"] == 0.5 and group["lr"] == 0.1
    with torch.no_grad():
        b[0].copy_(c[0])
    muon.step()
    buf = 0.9 * a[0].grad + a[0].grad
    want = c[0] - 0.1 * 0.5 * F.newton_schulz((a[0].grad + 0.9 * buf).detach())
    assert torch.allclose(b[0], want, rtol=0, atol=1e-5)

    back = FusedSGD(d[:1], lr=0.1, momentum=0.9)
    back.load_state_dict(copy.deepcopy(muon.state_dict()))
    before = d[0].detach().clone()
    assert back.sgd_groups() == back.param_groups and len(back.param_groups) == 1
    back.step()
    assert not torch.equal(before, d[0])
