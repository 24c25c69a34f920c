"""Calls at the edge of what the transformer operators take: who watches a call (tangents, traces, tensor subclasses), every
size of workgroup, vectors, sinks of gates, extreme gradients.  Bounds are those of tests/_transformer_ref.py."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

import _transformer_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _named(request):
    print(request.node.name, flush=True)
    yield
    torch.cuda.synchronize()


def F():
    from distributed_pytorch_amd.ops import functional

    return functional


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)


def _calls():
    """{name: (call of one tensor, that tensor)}; every floating-point argument of every operator once."""
    g = gen(0)
    x, y, w, b = normal(g, (2, 3, 16)), normal(g, (2, 3, 16)), normal(g, (16,)), normal(g, (16,))
    pos = torch.arange(4, device="cuda")[:, None].expand(4, 2).contiguous()
    qkv, freqs, axis = normal(g, (1, 4, 48)), normal(g, (8,)).double(), torch.zeros(8, dtype=torch.int32, device="cuda")
    z, t = normal(g, (3, 20)), torch.zeros(3, dtype=torch.int64, device="cuda")
    norm = lambda v, q: F().Norm(v, q, 1e-5, "layer")                                                       # noqa: E731
    return {
        "x": (lambda v: F().residual_norm(v, y, pre=norm(w, b))[1], x),
        "y": (lambda v: F().residual_norm(x, v), y),
        "post.weight": (lambda v: F().residual_norm(x, y, post=norm(v, b)), w),
        "post.bias": (lambda v: F().residual_norm(x, y, post=norm(w, v)), b),
        "pre.weight": (lambda v: F().residual_norm(x, y, pre=norm(v, b))[1], w),
        "pre.bias": (lambda v: F().residual_norm(x, y, pre=norm(w, v))[1], b),
        "gate": (lambda v: F().residual_norm(x, y, gate=v), w),
        "scale": (lambda v: F().residual_norm(x, y, scale=v), torch.ones(2, device="cuda")),
        "rms_norm": (lambda v: F().rms_norm(v, w), x),
        "rms_norm.weight": (lambda v: F().rms_norm(x, v), w),
        "rotary": (lambda v: F().rotary(v, pos, freqs, axis, 1), qkv),
        "rotary.inplace": (lambda v: F().rotary(v, pos, freqs, axis, 1, inplace=True), qkv.clone()),
        "rotary.positions": (lambda v: F().rotary(qkv, v, freqs, axis, 1), pos.double()),
        "rotary.freqs": (lambda v: F().rotary(qkv, pos, v, axis, 1), freqs),
        "token_logprobs": (lambda v: F().token_logprobs(v, t, 3)[0], z),
        "newton_schulz": (lambda v: F().newton_schulz(v), normal(g, (12, 20))),
    }


CALLS = ["x", "y", "post.weight", "post.bias", "pre.weight", "pre.bias", "gate", "scale", "rms_norm", "rms_norm.weight", "rotary",
         "rotary.inplace", "rotary.positions", "rotary.freqs", "token_logprobs", "newton_schulz"]


# ------------------------------------------------------------------------------------------ Newton-Schulz of bf16 updates
@pytest.mark.parametrize("shape", [(7, 5), (2, 130, 33), (6, 256, 520), (40, 260, 300), (10, 1024, 1030), (20, 128, 1000)])
def test_newton_schulz_of_bf16_is_the_32_bit_result_rounded(shape):
    """The products of a bf16 update carry what those of the same update in float32 do: one rounding at the end apart the
    results are the same, on every kind of tile, upright and turned."""
    for s in (shape, shape[:-2] + (shape[-1], shape[-2])):
        g = normal(gen(sum(s)), s, torch.bfloat16)
        assert torch.equal(F().newton_schulz(g), F().newton_schulz(g.float()).to(torch.bfloat16))


@pytest.mark.parametrize("shape", [(64, 64), (130, 33), (3, 100, 257), (6, 256, 2304), (33, 300, 513), (10, 1024, 1030)])
def test_newton_schulz_fast_products(shape):
    """Single-plane products, asked for: within the bound of a bf16 result (a rounding of 2^-8, in the quadratic mean
    2^-8 / sqrt(3) at most, beside 7e-4 of the products), also with directions 100 times the rest."""
    g = gen(sum(shape))
    u, v = normal(g, shape[:-1] + (4,)), normal(g, shape[:-2] + (4, shape[-1]))
    for m in (normal(g, shape, torch.bfloat16), (normal(g, shape) + 50.0 * torch.matmul(u, v)).to(torch.bfloat16)):
        got = F().newton_schulz(m, fast=True)
        value, rel = ref.newton_schulz(m)
        assert got.dtype == torch.bfloat16
        off = torch.linalg.vector_norm(got.double().cpu() - value, dim=(-2, -1)) / torch.linalg.vector_norm(value, dim=(-2, -1))
        assert bool((off <= rel).all()), (off.max(), rel)


def test_newton_schulz_fast_is_for_bf16():
    for dtype in (torch.float32, torch.float16):
        with pytest.raises(ValueError, match="bfloat16"):
            F().newton_schulz(torch.ones(4, 8, dtype=dtype, device="cuda"), fast=True)


# ------------------------------------------------------------------------------------------ tangents, traces, tensor subclasses
@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name):
    """A forward-mode derivative is refused, not left out, with and without requires_grad, and in-place data stays as it is."""
    call, v = _calls()[name]
    before = v.clone()
    with fwd.dual_level():
        dual = fwd.make_dual(v, torch.ones_like(v))
        with pytest.raises((NotImplementedError, ValueError), match="forward-mode|no gradient"):
            call(dual)
    torch.cuda.synchronize()
    assert torch.equal(v, before)
    call(v)                                        # (and no tangent, no refusal)
    with fwd.dual_level():
        call(v)


@pytest.mark.parametrize("name", CALLS)
def test_tracing_is_refused(name):
    """A trace would hold the allocation of the result and nothing that fills it."""
    call, v = _calls()[name]
    with pytest.raises((NotImplementedError, RuntimeError), match="trac"):
        torch.jit.trace(call, (v,), check_trace=False)


@pytest.mark.parametrize("name", CALLS)
def test_fake_tensors_and_graph_tracing_are_refused(name):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    call, v = _calls()[name]
    mode = FakeTensorMode(allow_non_fake_inputs=True)
    with pytest.raises(NotImplementedError, match="traced|subclasses"):
        call(mode.from_tensor(v))
    with mode, pytest.raises(NotImplementedError, match="traced|subclasses"):
        call(v)
    with pytest.raises(NotImplementedError, match="traced|subclasses"):
        make_fx(call)(v)


def test_backward_is_not_traced_either():
    x = normal(gen(0), (2, 3, 16)).requires_grad_()
    h = F().rms_norm(x, torch.ones(16, device="cuda"))
    from torch.fx.experimental.proxy_tensor import make_fx

    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(lambda v: torch.autograd.grad(h, x, v, retain_graph=True)[0])(torch.ones_like(h))


def test_modes_that_watch_are_welcome():
    """A mode that only watches what torch allocates changes nothing."""
    from torch.utils.flop_counter import FlopCounterMode

    x, w = normal(gen(0), (2, 3, 16)), torch.ones(16, device="cuda")
    want = F().rms_norm(x, w)
    with FlopCounterMode(display=False):
        assert torch.equal(F().rms_norm(x, w), want)


# ------------------------------------------------------------------------------------------ saved tensors
def _with_gradients(seed=0):
    """[(results, leaves, gradients)] of every operator that has a backward pass."""
    g = gen(seed)
    leaf = lambda *shape, dtype=torch.float32: normal(g, shape, dtype).requires_grad_()                        # noqa: E731
    x, y, w, b, v, gate = leaf(3, 5, 24), leaf(3, 5, 24), leaf(24), leaf(24), leaf(24), leaf(3, 24)
    scale = torch.tensor([0.0, 1.0, 2.0], device="cuda")
    s, h = F().residual_norm(x, y, post=F().Norm(w, b, 1e-5, "layer"), gate=gate, scale=scale, pre=F().Norm(v, None, 1e-5, "rms"))
    qkv, z = leaf(2, 4, 48, dtype=torch.bfloat16), leaf(3, 20)
    wide = normal(g, (3, 30)).requires_grad_()
    pos = torch.arange(8, device="cuda").view(2, 4, 1)
    r = F().rotary(qkv, pos, torch.ones(8, device="cuda"), torch.zeros(8, dtype=torch.int64, device="cuda"), 1)
    t = torch.tensor([1, 5, -1], device="cuda")
    lp = F().token_logprobs(z, t, 4)[:3] + F().token_logprobs(wide[:, 3:23], t, 4)[:3]
    return [([s, h], [x, y, w, b, v, gate], None), ([r], [qkv], None), (list(lp), [z, wide], None)]


def _gradients(cases):
    return [torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs]) for outs, leaves, _ in cases]


def test_saved_tensors_may_go_elsewhere_and_come_back():
    want = _gradients(_with_gradients())
    with torch.autograd.graph.save_on_cpu():
        cases = _with_gradients()
    for a, b in zip(_gradients(cases), want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_recomputed_calls_give_the_same_gradients():
    from torch.utils.checkpoint import checkpoint

    x, y, w = (normal(gen(i), s).requires_grad_() for i, s in enumerate([(3, 5, 24), (3, 5, 24), (24,)]))
    call = lambda x, y, w: F().residual_norm(x, y * 2.0, pre=F().Norm(w, None, 1e-5, "rms"))[1]              # noqa: E731
    want = torch.autograd.grad(call(x, y, w).sum(), [x, y, w])
    for reentrant in (False, True):
        got = torch.autograd.grad(checkpoint(call, x, y, w, use_reentrant=False).sum(), [x, y, w]) if not reentrant else None
        if reentrant:
            checkpoint(call, x, y, w, use_reentrant=True).sum().backward()
            got = [t.grad for t in (x, y, w)]
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("unpack", ["shorter", "narrower", "elsewhere", "fake"])
def test_saved_tensors_that_come_back_changed_are_refused(unpack):
    """... before a kernel reads past their ends."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    changed = {"shorter": lambda v: v.flatten()[:1], "narrower": lambda v: v.to(torch.float16 if v.is_floating_point() else torch.int32), "elsewhere": lambda v: v.cpu(),
               "fake": lambda v: FakeTensorMode(allow_non_fake_inputs=True).from_tensor(v)}[unpack]
    for which in range(3):
        with torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: changed(v.detach())):
            case = _with_gradients()[which]
        with pytest.raises(RuntimeError, match="saved tensor came back|subclass|Type"):
            _gradients([case])


def test_gradients_that_are_wrappers_are_refused():
    for outs, leaves, _ in _with_gradients():
        with pytest.raises(RuntimeError):
            torch.autograd.grad(outs[:1], leaves[:1], [torch.stack([torch.ones_like(outs[0])] * 2)], is_grads_batched=True)


# ------------------------------------------------------------------------------------------ residual norm
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [1, 8, 33, 768, 4099])
def test_rms_norm_of_a_vector(C, dtype):
    g = gen(C)
    x, w, dh = normal(g, (C,), dtype, 2.0), normal(g, (C,), std=0.2, mean=1.0), normal(g, (C,), dtype)
    want = ref.residual_norm(x[None], torch.zeros_like(x)[None], None, None, None, F().Norm(w, None, 1e-6, "rms"), None, dh[None])
    x.requires_grad_()
    w.requires_grad_()
    h = F().rms_norm(x, w, 1e-6)
    dx, dw = torch.autograd.grad(h, [x, w], dh)
    for name, got in (("h", h), ("d_x", dx)):
        ref.within(got, want[name][0][0], want[name][1][0], name)
    ref.within(dw, *want["d_pre_w"], "dw")
    with torch.no_grad():
        assert torch.equal(h, F().rms_norm(x, w, 1e-6))


def test_gate_of_samples_with_a_sink():
    """A per-sample gate that is a parameter of a gradient arena: delivered like any other, over two uses, and nothing is owed
    to its sink afterwards."""
    from distributed_pytorch_amd.parallel.distributed import GradArena

    g = gen(3)
    x, y, ds = normal(g, (4, 5, 24)), normal(g, (4, 5, 24)), normal(g, (4, 5, 24))
    gate, flat = torch.nn.Parameter(normal(g, (4, 24))), torch.nn.Parameter(normal(g, (24,)))
    ready = []
    arena = GradArena([gate, flat], on_ready=lambda s: ready.append(s.param))
    arena.begin_step()
    total = 0.0
    for _ in range(2):
        total = total + (F().residual_norm(x, y, gate=gate) * ds).sum() + (F().residual_norm(x, y, gate=flat) * ds).sum()
    total.backward()
    assert [sum(p is q for q in ready) for p in (gate, flat)] == [1, 1]
    arena.finish_step()
    for p in (gate, flat):
        assert p.grad is p._dpa_sink.view and p._dpa_sink.uses == 0
        value, bound = ref.residual_norm(x, y, None, p, None, None, ds)["d_gate"]
        ref.within(p.grad, 2 * value, 2 * bound + 8 * ref.E32 * value.abs(), "gate")


def test_an_error_on_delivery_is_the_callers():
    """Who is told of a finished gradient may raise (a collective that failed): the call to backward raises it, and the process
    goes on."""
    from distributed_pytorch_amd.parallel.distributed import GradArena

    g = gen(3)
    x, y = normal(g, (4, 5, 24)), normal(g, (4, 5, 24))
    w, gate = torch.nn.Parameter(normal(g, (24,))), torch.nn.Parameter(normal(g, (4, 24)))
    fail = [True]

    def ready(sink):
        if fail[0]:
            raise ValueError("not delivered")

    arena = GradArena([w, gate], on_ready=ready)

    def step():
        arena.begin_step()
        s, h = F().residual_norm(x, y, gate=gate, pre=F().Norm(w, None, 1e-5, "rms"))
        (s.sum() + h.sum()).backward()

    for _ in range(3):
        with pytest.raises(Exception, match="not delivered"):
            step()
        arena.end_step()
    fail[0] = False
    step()
    arena.finish_step()
    assert w.grad.isfinite().all() and gate.grad.isfinite().all()


# ------------------------------------------------------------------------------------------ log probabilities
# rows that select 64, 128 and 256 lanes a row where rows are long
ROWS = [520, 2100, 4200]


def _lanes(rows):
    return 64 if rows >= 4096 else 128 if rows >= 2048 else 256


def _check_rows(z, t, k, rows, seed=0):
    """Every row's results and gradients are computed, `rows` of them are compared."""
    g = gen(seed)
    N = z.shape[0]
    d_lp, d_ent, d_top = normal(g, (N,)), normal(g, (N,)), normal(g, (N, k))
    z = z.detach().requires_grad_()
    out = F().token_logprobs(z, t, k)
    (d,) = torch.autograd.grad(out[:3], [z], [d_lp, d_ent, d_top])
    at = torch.tensor(rows, device="cuda")
    want = ref.token_logprobs(z[at], t[at], k, d_lp[at], d_ent[at], d_top[at])
    assert torch.equal(out[3][at].cpu(), want["index"][0]), "indices"
    # (the reference's bounds count V / 256 additions in a row for a lane; fewer lanes add more of them)
    V = z.shape[1]
    more = (V / _lanes(N) + 24) / (V / 256 + 24)
    for name, got in zip(("logprob", "entropy", "top"), out):
        ref.within(got[at], want[name][0], more * want[name][1], name)
    value, bound = want["d_logits"]
    rounding = ref.U[z.dtype] * value.abs()
    ref.within(d[at], value, rounding + more * (bound - rounding), "d_logits")


@pytest.mark.parametrize("N", ROWS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("few,k", [(1, 40), (12, 64), (64, 64)])
def test_token_logprobs_crowded_lanes_of_every_workgroup(few, k, dtype, N):
    """Long rows whose largest values lie in the chunks of a few lanes, several chunks each, for each size of workgroup."""
    V, g = 9001, gen(few)
    lanes, step = _lanes(N), 16 // (torch.finfo(dtype).bits // 8)
    assert -(-V // step) > 256
    lane = torch.arange(V, device="cuda") // step % lanes
    z = normal(g, (N, V))
    crowd = (lane >= 5) & (lane < 5 + few)
    z[1] += torch.where(crowd, 9.0, 0.0)
    z[N - 1] += torch.where(crowd, 3.0, 0.0)
    z[N // 2] = torch.where(crowd, 2.0, 0.0)                  # equal values alone: more than the list holds
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    _check_rows(z.to(dtype), t, k, [0, 1, N // 2, N - 1])


@pytest.mark.parametrize("N", ROWS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_ties_and_masks_of_every_workgroup(dtype, N):
    V, k, g = 9001, 64, gen(N)
    base = torch.arange(V, device="cuda")
    z = normal(g, (N, V), dtype, 2.0)
    z[0] = 0.0                                                # every class the same: looked at again and again
    z[1] = (base % 3).to(dtype)
    z[2] = (base / V).to(dtype)
    z[3] = (-base / V).to(dtype)
    z[4] = torch.finfo(dtype).min
    z[5, 70:] = -math.inf
    z[6, ::2] = -math.inf
    t = torch.randint(0, 64, (N,), generator=g, device="cuda") | 1
    _check_rows(z, t, k, [0, 1, 2, 3, 4, 5, 6, 7, N - 1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e9, 1e30])
def test_token_logprobs_large_entropy_gradients_beside_masked_classes(size, dtype):
    """A masked class has no gradient however large the entropy's is (a loss scale on top of a large weight)."""
    g = gen(5)
    z = normal(g, (3, 300))
    z[0, ::3] = -math.inf
    z[1, 1:] = torch.finfo(dtype).min
    z[2] = z[2] * 10
    z = z.to(dtype).requires_grad_()
    t = torch.zeros(3, dtype=torch.int64, device="cuda") + 1
    _, ent, _, _ = F().token_logprobs(z, t)
    d_ent = normal(g, (3,)) * size
    (d,) = torch.autograd.grad(ent, z, d_ent)
    assert not d[0, ::3].any()
    value, bound = ref.token_logprobs(z, t, 0, torch.zeros(3), d_ent)["d_logits"]
    if dtype == torch.float16:                                # (values past its range are infinite)
        assert not d.isnan().any()
    else:
        ref.within(d, value, bound, "d_logits")


# ------------------------------------------------------------------------------------------ rotary
def test_rotary_axis_far_outside():
    """An entry that does not fit 32 bits is outside like any other."""
    qkv, pos = normal(gen(0), (1, 4, 48)), torch.arange(8, device="cuda").view(4, 2)
    freqs, axis = torch.ones(8, device="cuda"), torch.tensor([0, 1, 2 ** 32, 0, -2 ** 32 + 1, 1, 2 ** 33 + 1, 0], device="cuda")
    out = F().rotary(qkv, pos, freqs, axis, 1).view(4, 3, 2, 8)
    outside = torch.tensor([False, False, True, False, True, False, True, False], device="cuda")
    assert out[:, :2][..., outside].isnan().all() and out[..., ~outside].isfinite().all() and out[:, 2].isfinite().all()


def test_rotary_in_place_of_an_inference_tensor():
    """Refused outside inference mode before anything is written, taken inside."""
    with torch.inference_mode():
        qkv = normal(gen(0), (1, 4, 48))
        kept = qkv.clone()
    pos = torch.arange(4, device="cuda")[:, None]
    freqs, axis = torch.ones(8, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    with torch.no_grad(), pytest.raises(RuntimeError, match="[Ii]nference"):
        F().rotary(qkv, pos, freqs, axis, 1, inplace=True)
    with torch.inference_mode():
        assert torch.equal(qkv, kept)
        want = F().rotary(qkv, pos, freqs, axis, 1)
        assert torch.equal(F().rotary(qkv, pos, freqs, axis, 1, inplace=True), want)


# ------------------------------------------------------------------------------------------ FusedMuon
def test_sgd_with_the_groups_of_a_muon_checkpoint():
    """FusedSGD updates every parameter, also in groups that a checkpoint of FusedMuon marks as matrices; FusedMuon takes the
    momentum of an SGD checkpoint and goes on with its matrices."""
    import copy

    from distributed_pytorch_amd.optim import FusedMuon, FusedSGD

    def params():
        ps = [torch.nn.Parameter(normal(gen(1), (24, 40)))]
        ps[0].grad = normal(gen(2), (24, 40))
        return ps

    a, b, c = params(), params(), params()
    muon = FusedMuon([dict(params=a, orthogonal=True)], lr=0.1, momentum=0.9)
    muon.step()
    sgd = FusedSGD(b, lr=0.1, momentum=0.9)
    sgd.load_state_dict(copy.deepcopy(muon.state_dict()))
    before, grad, buf = b[0].detach().clone(), b[0].grad.clone(), sgd.state[b[0]]["momentum_buffer"].clone()
    sgd.step()
    buf = 0.9 * buf + grad
    step = grad + 0.9 * buf if sgd.param_groups[0]["nesterov"] else buf
    assert torch.allclose(b[0], before - 0.1 * step, rtol=0, atol=1e-5)
    again = FusedMuon([dict(params=c, orthogonal=True)], lr=0.1, momentum=0.9)
    again.load_state_dict(copy.deepcopy(FusedSGD(params(), lr=0.1, momentum=0.9).state_dict()))
    before = c[0].detach().clone()
    again.step()
    assert again.param_groups[0]["orthogonal"] is True and 0.0 < float((c[0] - before).norm()) < 0.1 * 0.2 * 1.3 * 24 ** 0.5


@pytest.mark.parametrize("cpu", ["matrix", "vector"])
def test_optimizers_refuse_parameters_of_the_cpu_beside_the_gpus(cpu):
    """... whose addresses no kernel may read."""
    from distributed_pytorch_amd.optim import FusedMuon, FusedSGD

    def params():
        ps = [torch.nn.Parameter(torch.ones(s, device="cpu" if (len(s) == 2) == (cpu == "matrix") else "cuda")) for s in ((4, 6), (5,))]
        for p in ps:
            p.grad = torch.ones_like(p)
        return ps

    a, b = params(), params()
    for opt in (FusedMuon([dict(params=a[:1], orthogonal=True), dict(params=a[1:])], lr=0.1),
                FusedSGD([dict(params=b[:1]), dict(params=b[1:])], lr=0.1)):
        with pytest.raises(ValueError, match="CPU"):
            opt.step()
    for p in a + b:
        assert bool((p == 1.0).all())
