"""The transformer-block kernels against 64-bit references (tests/_transformer_ref.py: bounds are derived there)."""
import math

import pytest
import torch

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


# ------------------------------------------------------------------------------------------ residual norm
def _residual_case(shape, dtype, post, pre, gate, scale, seed=0, train=True):
    g = gen(seed)
    C, N = shape[-1], shape[0]
    x, y = normal(g, shape, dtype, 1.5), normal(g, shape, dtype, 0.7, 0.1)
    norms = {}
    for side, kind in (("post", post), ("pre", pre)):
        w, b = normal(g, (C,), std=0.2, mean=1.0), normal(g, (C,), std=0.2)
        norms[side] = None if kind is None else F().Norm(w, b if kind == "layer" else None, 1e-5, kind)
    gt = None if gate is None else normal(g, (C,) if gate == "channel" else (N, C), std=0.3, mean=0.5)
    sc = None
    if scale:
        sc = (torch.rand((N,), generator=g, device="cuda") < 0.6).float() / 0.6
    ds = normal(g, shape, dtype)
    dh = normal(g, shape, dtype) if pre else None
    return x, y, norms["post"], gt, sc, norms["pre"], ds, dh


def _residual_run(x, y, post, gate, scale, pre, ds, dh):
    leaves = {"d_x": x, "d_y": y, "d_gate": gate}
    for side, n in (("post", post), ("pre", pre)):
        if n is not None:
            leaves["d_%s_w" % side], leaves["d_%s_b" % side] = n.weight, n.bias
    leaves = {k: v for k, v in leaves.items() if v is not None}
    for v in leaves.values():
        v.requires_grad_()
    out = F().residual_norm(x, y, post=post, gate=gate, scale=scale, pre=pre)
    s, h = out if pre is not None else (out, None)
    outs = [(o, g) for o, g in ((s, ds), (h, dh)) if g is not None]
    got = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)
    res = dict(zip(leaves, got), s=s)
    if h is not None:
        res["h"] = h
    return res


def _residual_check(case):
    x, y, post, gate, scale, pre, ds, dh = case
    want = ref.residual_norm(x, y, post, gate, scale, pre, ds, dh)
    got = _residual_run(*case)
    for name, (value, bound) in want.items():
        assert got[name].dtype == (x.dtype if name in ("s", "h", "d_x", "d_y") else torch.float32)
        ref.within(got[name], value, bound, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("post,pre,gate,scale", [
    (None, "layer", None, False), (None, "rms", None, False), ("layer", None, None, True), ("rms", "rms", "sample", False),
    ("layer", "layer", "channel", True), (None, None, "channel", True), (None, "layer", "sample", True),
    ("rms", None, None, False), (None, None, None, False)])
@pytest.mark.parametrize("shape", [(1, 1, 8), (3, 5, 7), (2, 197, 96), (5, 3, 640), (2, 9, 1032)])
def test_residual_norm(shape, dtype, post, pre, gate, scale):
    _residual_check(_residual_case(shape, dtype, post, pre, gate, scale))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 2, 3, 2056), (3, 1, 4096), (1, 3, 4099), (2, 3, 8192), (1, 2, 16384), (4, 1),
                                   (300, 40), (7, 2, 3, 5, 24)])
def test_residual_norm_wide_and_odd(shape, dtype):
    if shape[-1] * (4 if dtype == torch.float32 else 2) > 2048 * 16:
        with pytest.raises(ValueError):
            _residual_check(_residual_case(shape, dtype, None, "layer", None, False))
        return
    _residual_check(_residual_case(shape, dtype, "layer", "rms", "channel", True, seed=1))
    _residual_check(_residual_case(shape, dtype, None, "layer", None, False, seed=2))


def test_residual_norm_many_rows():
    """More rows than one round of workgroups, and samples of unlike shares."""
    _residual_check(_residual_case((37, 211, 96), torch.bfloat16, "layer", "layer", "sample", True, seed=3))
    _residual_check(_residual_case((1000, 1, 64), torch.float16, "rms", None, "sample", False, seed=4))


def test_residual_norm_strides_and_offsets():
    x, y, post, gate, scale, pre, ds, dh = _residual_case((4, 6, 64), torch.bfloat16, "layer", "rms", "channel", True)
    xt = x.transpose(0, 1).contiguous().transpose(0, 1)               # other strides
    buf = torch.empty(4 * 6 * 64 + 3, dtype=torch.bfloat16, device="cuda")
    yo = buf[3:].view(4, 6, 64)                                       # rows that start off a 16-byte boundary
    yo.copy_(y)
    assert not xt.is_contiguous() and yo.data_ptr() % 16
    want = ref.residual_norm(x, y, post, gate, scale, pre, ds, dh)
    got = _residual_run(xt.detach(), yo.detach(), post, gate, scale, pre, ds.transpose(0, 1).contiguous().transpose(0, 1), dh)
    for name, (value, bound) in want.items():
        ref.within(got[name], value, bound, name)


@pytest.mark.parametrize("used", ["s", "h"])
def test_residual_norm_one_result_used(used):
    case = list(_residual_case((3, 4, 40), torch.float32, "rms", "layer", "channel", False))
    case[7 if used == "s" else 6] = None
    want = ref.residual_norm(*case)
    got = _residual_run(*case)
    for name, (value, bound) in want.items():
        if got[name] is None or name in ("s", "h"):
            continue
        ref.within(got[name], value, bound, name)


def test_residual_norm_no_rows():
    x, y, post, gate, scale, pre, ds, dh = _residual_case((0, 5, 32), torch.bfloat16, "layer", "layer", "sample", True)
    got = _residual_run(x, y, post, gate, scale, pre, ds, dh)
    assert got["s"].shape == (0, 5, 32) and got["d_gate"].shape == (0, 32)
    assert not got["d_pre_w"].any() and not got["d_post_b"].any()


def test_residual_norm_dropped_samples_get_no_gradient():
    x, y, post, gate, _, pre, ds, dh = _residual_case((4, 3, 32), torch.float32, "layer", "layer", "channel", False)
    scale = torch.tensor([0.0, 2.0, 0.0, 1.0], device="cuda")
    got = _residual_run(x, y, post, gate, scale, pre, ds, dh)
    assert not got["d_y"][0].any() and not got["d_y"][2].any() and got["d_y"][1].any()
    assert torch.equal(got["s"][0], x[0])


def test_residual_norm_differences():
    """Central differences of sum(s * ds + h * dh) along a random direction of every leaf at once.  The function is
    smooth with third derivatives of order 10 here: h = 2^-6 leaves h^2 * 10 / 6 = 4e-4 of it, and 32-bit results
    (2^-24 each, independent) 2^-24 sqrt(n) * |.| / h, far below; 2e-3 of the sum of magnitudes holds both."""
    case = _residual_case((3, 7, 48), torch.float32, "layer", "rms", "sample", True, seed=9)
    x, y, post, gate, scale, pre, ds, dh = case
    got = _residual_run(*case)
    leaves = {"d_x": x, "d_y": y, "d_gate": gate, "d_post_w": post.weight, "d_post_b": post.bias, "d_pre_w": pre.weight}
    g = gen(5)
    for name, leaf in leaves.items():
        v = normal(g, leaf.shape)
        v = v / v.norm()
        vals = []
        with torch.no_grad():
            for sign in (1.0, -1.0):
                leaf.add_(v, alpha=sign / 64)
                s, h = F().residual_norm(x, y, post=post, gate=gate, scale=scale, pre=pre)
                leaf.add_(v, alpha=-sign / 64)
                vals.append((s.double() * ds.double()).sum() + (h.double() * dh.double()).sum())
        diff = float(vals[0] - vals[1]) * 32
        want = float((got[name].double() * v.double()).sum())
        assert abs(diff - want) <= 2e-3 * float(got[name].double().norm()) + 1e-3, (name, diff, want)


def test_residual_norm_gradient_sinks():
    """Parameters of a gradient arena: written in place, accumulated over two uses, also where one parameter serves
    both norms of a call."""
    from distributed_pytorch_amd.parallel.distributed import GradArena

    x, y, post, gate, scale, pre, ds, dh = _residual_case((2, 9, 64), torch.float32, "layer", "layer", "channel", True)
    w, b, gt = (torch.nn.Parameter(t.detach().clone()) for t in (pre.weight, pre.bias, gate))
    both = F().Norm(w, b, 1e-5, "layer")
    arena = GradArena([w, b, gt])
    arena.begin_step()

    def loss():
        total = 0.0
        for _ in range(2):
            s, h = F().residual_norm(x, y, post=both, gate=gt, scale=scale, pre=both)
            total = total + (s * ds).sum() + (h * dh).sum()
        return total

    loss().backward()
    arena.finish_step()
    want = ref.residual_norm(x, y, both, gt, scale, both, ds, dh)
    for p, names in ((w, ("d_pre_w", "d_post_w")), (b, ("d_pre_b", "d_post_b")), (gt, ("d_gate",))):
        assert p.grad is p._dpa_sink.view
        value = 2 * sum(want[n][0] for n in names)
        ref.within(p.grad, value, 2 * sum(want[n][1] for n in names) + 8 * ref.E32 * value.abs(), str(names))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(5, 33), (2, 3, 768), (1, 4096)])
def test_rms_norm(dtype, shape):
    g = gen(0)
    x, w, dh = normal(g, shape, dtype, 2.0), normal(g, shape[-1:], std=0.2, mean=1.0), normal(g, shape, dtype)
    norm = F().Norm(w, None, 1e-6, "rms")
    zero = torch.zeros_like(x)
    want = ref.residual_norm(x, zero, None, None, None, norm, None, dh)
    x.requires_grad_()
    w.requires_grad_()
    h = F().rms_norm(x, w, 1e-6)
    dx, dw = torch.autograd.grad(h, [x, w], dh)
    ref.within(h, *want["h"], "h")
    ref.within(dx, *want["d_x"], "dx")
    ref.within(dw, *want["d_pre_w"], "dw")
    with torch.no_grad():
        assert torch.equal(h, F().rms_norm(x, w, 1e-6))


# ------------------------------------------------------------------------------------------ rotary
def _rotary_case(B, S, H, D, P, A, dtype, span=50, seed=0, batched=True, kind=torch.int64):
    g = gen(seed)
    qkv = normal(g, (B, S, 3 * H * D), dtype)
    pos = torch.rand((B, S, A) if batched else (S, A), generator=g, device="cuda", dtype=torch.float64) * span
    pos = pos.floor().to(kind) if not kind.is_floating_point else pos.to(kind)
    freqs = 100.0 ** (-torch.rand((P,), generator=g, device="cuda", dtype=torch.float64))
    axis = torch.randint(0, A, (P,), generator=g, device="cuda", dtype=torch.int32)
    return qkv, pos, freqs, axis


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,H,D,P,A,batched", [
    (1, 1, 1, 2, 1, 1, True), (2, 5, 3, 8, 4, 2, True), (2, 17, 2, 64, 32, 2, False), (1, 197, 12, 64, 32, 2, False),
    (3, 33, 4, 80, 40, 3, True), (2, 7, 3, 10, 4, 3, True), (2, 9, 2, 96, 24, 3, True), (1, 50, 1, 130, 65, 1, False),
    (1, 3, 2, 16, 0, 1, False), (1, 6, 5, 33, 16, 2, True), (3, 2700, 2, 16, 8, 2, True)])
def test_rotary(B, S, H, D, P, A, batched, dtype, interleaved):
    qkv, pos, freqs, axis = _rotary_case(B, S, H, D, P, A, dtype, batched=batched)
    dout = normal(gen(1), qkv.shape, dtype)
    qkv.requires_grad_()
    out = F().rotary(qkv, pos, freqs, axis, H, interleaved=interleaved)
    ref.within(out, *ref.rotary(qkv, pos, freqs, axis, H, interleaved), "out")
    (d,) = torch.autograd.grad(out, qkv, dout)
    ref.within(d, *ref.rotary(dout, pos, freqs, axis, H, interleaved, -1.0), "gradient")
    with torch.no_grad():
        assert torch.equal(F().rotary(qkv, pos, freqs, axis, H, interleaved=interleaved), out)
        same = qkv.detach().clone()
        back = F().rotary(same, pos, freqs, axis, H, interleaved=interleaved, inplace=True)
        assert back is same and torch.equal(same, out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,P", [(48, 15), (48, 9), (24, 1), (16, 7), (40, 20), (32, 13)])
def test_rotary_pairs_end_inside_a_chunk(D, P, interleaved, dtype):
    """What lies behind the pairs is copied as it is, infinities and NaN too, out of place and in place."""
    qkv, pos, freqs, axis = _rotary_case(2, 9, 3, D, P, 2, dtype)
    value, bound = ref.rotary(qkv, pos, freqs, axis, 3, interleaved)
    ref.within(F().rotary(qkv, pos, freqs, axis, 3, interleaved=interleaved), value, bound, "out")
    special = qkv.clone().view(2, 9, 3, 3, D)
    special[..., 2 * P:] = torch.tensor([math.inf, -math.inf, math.nan, 1.5], device="cuda").to(dtype).repeat(D)[:D - 2 * P]
    flat = special.view(2, 9, -1)
    out = F().rotary(flat, pos, freqs, axis, 3, interleaved=interleaved)
    again = F().rotary(flat.clone(), pos, freqs, axis, 3, interleaved=interleaved, inplace=True)
    assert torch.equal(out.view(torch.uint8), again.view(torch.uint8))
    tail = out.view(2, 9, 3, 3, D)[..., 2 * P:].contiguous()
    assert torch.equal(tail.view(torch.uint8), special[..., 2 * P:].contiguous().view(torch.uint8))


@pytest.mark.parametrize("kind", [torch.int64, torch.int32, torch.float32, torch.float64])
def test_rotary_far_positions(kind):
    """Angles of 10^6 and more turns' worth: 32 bits would be off by a tenth of a radian."""
    qkv, pos, freqs, axis = _rotary_case(2, 40, 2, 32, 16, 2, torch.float32, span=3e6, kind=kind)
    out = F().rotary(qkv, pos, freqs, axis, 2)
    value, bound = ref.rotary(qkv, pos, freqs, axis, 2, False)
    # the product in 64 bits is off by 2^-53 of 3e6, and so is its reduction: 1e-9, within the slack
    ref.within(out, value, bound, "far")


def test_rotary_strides():
    qkv, pos, freqs, axis = _rotary_case(3, 10, 2, 32, 16, 2, torch.bfloat16)
    wide = torch.empty((3, 12, 3 * 64 + 5), dtype=torch.bfloat16, device="cuda").fill_(7.0)
    part = wide[:, 1:11, 5:]
    part.copy_(qkv)
    want = F().rotary(qkv, pos, freqs, axis, 2)
    assert torch.equal(F().rotary(part, pos, freqs, axis, 2), want)
    assert torch.equal(F().rotary(qkv.transpose(0, 1).contiguous().transpose(0, 1), pos, freqs, axis, 2), want)
    F().rotary(part, pos, freqs, axis, 2, inplace=True)
    assert torch.equal(part, want)
    wide[:, 1:11, 5:] = 7.0
    assert bool((wide == 7.0).all())                                  # nothing beside the tokens was written


def test_rotary_axis_outside():
    qkv, pos, freqs, axis = _rotary_case(1, 4, 1, 16, 8, 2, torch.float32)
    good = F().rotary(qkv, pos, freqs, axis, 1)
    axis[3] = 2
    axis[5] = -1
    out = F().rotary(qkv, pos, freqs, axis, 1).view(1, 4, 3, 2, 8)
    bad = torch.zeros(8, dtype=torch.bool)
    bad[3] = bad[5] = True
    assert out[:, :, :2][..., bad.cuda()].isnan().all()
    assert torch.equal(out[..., ~bad.cuda()], good.view(1, 4, 3, 2, 8)[..., ~bad.cuda()])


def test_rotary_relative():
    """Queries against keys depend on the difference of positions alone: what rotary positions are for.  32-bit results
    of 64 products: 64 * 10 * 2^-24 of the magnitude."""
    g = gen(3)
    H, D, P = 1, 64, 32
    qkv = normal(g, (1, 1, 3 * D)).expand(1, 6, 3 * D).contiguous()
    freqs = 100.0 ** (-torch.arange(P, device="cuda", dtype=torch.float64) / P)
    axis = torch.arange(P, device="cuda", dtype=torch.int32) % 2
    pos = torch.tensor([[0, 0], [3, 1], [100, 7], [103, 8], [5000, 20], [5003, 21]], device="cuda")
    q, k, _ = F().rotary(qkv, pos, freqs, axis, H)[0].double().chunk(3, -1)
    scores = [(q[i] * k[i + 1]).sum() for i in (0, 2, 4)]
    slack = 64 * 10 * ref.E32 * float((q[0].abs() * k[0].abs()).sum() + 1)
    assert max(scores) - min(scores) <= slack


# ------------------------------------------------------------------------------------------ log probabilities
def _logprobs_check(z, t, k, train=True, seed=0):
    g = gen(seed)
    N, V = z.shape
    d_lp, d_ent, d_top = normal(g, (N,)), normal(g, (N,)), normal(g, (N, k))
    if train:
        z = z.detach().requires_grad_()
    lp, ent, top, idx = F().token_logprobs(z, t, k)
    want = ref.token_logprobs(z, t, k, *((d_lp, d_ent, d_top) if train else ()))
    assert torch.equal(idx.cpu(), want["index"][0]), "indices"
    for name, got in (("logprob", lp), ("entropy", ent), ("top", top)):
        assert got.dtype == torch.float32
        ref.within(got, *want[name], name)
    if train:
        (d,) = torch.autograd.grad([lp, ent, top], [z], [d_lp, d_ent, d_top])
        assert d.dtype == z.dtype
        ref.within(d, *want["d_logits"], "d_logits")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (1, 2, 0), (3, 7, 7), (5, 63, 5), (4, 64, 64), (33, 1000, 5), (2, 1023, 20),
                                   (3, 4099, 64), (1, 8192, 3), (2, 50257, 20), (1, 131075, 64), (600, 10, 2)])
def test_token_logprobs(N, V, k, dtype):
    g = gen(N + V)
    z = normal(g, (N, V), dtype, 3.0)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    _logprobs_check(z, t, k)
    with torch.no_grad():
        _logprobs_check(z, t, k, train=False)


@pytest.mark.parametrize("V,k", [(6, 6), (1000, 5), (20000, 64), (70001, 40)])
def test_token_logprobs_ties_and_orders(V, k):
    """Ties go to the lowest index; values that crowd one lane's share of the row; sorted rows."""
    base = torch.arange(V, device="cuda")
    rows = [torch.zeros(V, device="cuda"), (base % 3).float(), base.float() / V, -base.float() / V,
            torch.where(base % 2048 < 8, 5.0, 0.0) + (base % 7) * 0.25, torch.where(base % 2 == 0, -0.0, 0.0)]
    z = torch.stack(rows)
    t = torch.zeros(len(rows), dtype=torch.int64, device="cuda") + V // 2
    _logprobs_check(z, t, k)
    _logprobs_check(z.to(torch.bfloat16), t, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("crowd", [(0,), (255,), (3, 64, 65, 66, 67, 68, 69, 250), tuple(range(100, 112)), tuple(range(256))])
def test_token_logprobs_crowded_lanes(crowd, dtype):
    """Whole rows of a workgroup (many rows), the largest values in chunks that few lanes visit, several chunks each."""
    N, V, k = 520, 34001, 40
    g = gen(len(crowd))
    step = 16 // (torch.finfo(dtype).bits // 8)
    lane = torch.arange(V, device="cuda") // step % 256
    z = normal(g, (N, V), torch.float32)
    z[1] += torch.where(torch.isin(lane, torch.tensor(crowd, device="cuda")), 9.0, 0.0)
    z[N - 1] += torch.where(torch.isin(lane, torch.tensor(crowd, device="cuda")), 3.0, 0.0)
    z = z.to(dtype)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    out = F().token_logprobs(z, t, k)
    rows = torch.tensor([0, 1, N - 1], device="cuda")
    want = ref.token_logprobs(z[rows], t[rows], k)
    assert torch.equal(out[3][rows].cpu(), want["index"][0])
    for name, got in zip(("logprob", "entropy", "top"), out):
        ref.within(got[rows], *want[name], name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [9, 3000, 40000])
def test_token_logprobs_masks(V, dtype):
    g = gen(V)
    z = normal(g, (7, V), dtype, 2.0)
    z[0, ::2] = -math.inf                      # half of the classes
    z[1] = -math.inf                           # all of them
    z[2] = -math.inf
    z[2, V - 1] = 1.0                          # all but one
    z[3] = torch.finfo(dtype).min              # the type's lowest value everywhere
    z[4, 1:] = torch.finfo(dtype).min
    z[5, : V // 2] = -math.inf
    t = torch.tensor([1, 0, V - 1, 2, 0, V - 1, 0], device="cuda")
    k = min(V, 5)
    z.requires_grad_()
    lp, ent, top, idx = F().token_logprobs(z, t, k)
    # (a masked class's own log probability is -inf and has no useful gradient: none is asked for here)
    d_lp, d_ent = normal(g, (7,)), normal(g, (7,))
    want = ref.token_logprobs(z, t, k, d_lp, d_ent, None)
    assert torch.equal(idx.cpu(), want["index"][0])
    for name, got in (("logprob", lp), ("entropy", ent), ("top", top)):
        ref.within(got, *want[name], name)
    (d,) = torch.autograd.grad([lp, ent], [z], [d_lp, d_ent])
    ref.within(d, *want["d_logits"], "d_logits")
    assert not d[1].any()


def test_token_logprobs_ignored_targets():
    g = gen(0)
    z = normal(g, (4, 100)).requires_grad_()
    t = torch.tensor([-100, 5, 100, -1], device="cuda")
    lp, ent, top, idx = F().token_logprobs(z, t, 3)
    assert lp[0] == 0 and lp[2] == 0 and lp[3] == 0 and lp[1] < 0
    (d,) = torch.autograd.grad(lp.sum(), z)
    assert not d[0].any() and not d[2].any() and not d[3].any() and d[1].any()


def test_token_logprobs_not_finite():
    g = gen(0)
    for V in (50, 20000):
        z = normal(g, (4, V))
        z[0, 3] = math.nan
        z[1, 7] = math.inf
        z[2, 0] = z[2, V - 1] = math.inf
        t = torch.zeros(4, dtype=torch.int64, device="cuda")
        lp, ent, top, idx = F().token_logprobs(z, t, 4)
        assert lp[:3].isnan().all() and ent[:3].isnan().all() and top[:3].isnan().all() and lp[3].isfinite()
        assert bool(((idx >= 0) & (idx < V)).all()) and all(len(set(r)) == 4 for r in idx.tolist())


def test_token_logprobs_strides_and_shapes():
    g = gen(2)
    wide = normal(g, (6, 1005), torch.bfloat16)
    z = wide[:, 3:1003]
    t = torch.randint(0, 1000, (6,), generator=g, device="cuda", dtype=torch.int32)
    want = F().token_logprobs(z.contiguous(), t, 5)
    for a, b in zip(F().token_logprobs(z, t, 5), want):
        assert torch.equal(a, b)
    for a, b in zip(F().token_logprobs(z.t().contiguous().t(), t, 5), want):
        assert torch.equal(a, b)
    got = F().token_logprobs(z.contiguous().view(2, 3, 1000), t.view(2, 3), 5)
    assert got[0].shape == (2, 3) and got[3].shape == (2, 3, 5)
    for a, b in zip(got, want):
        assert torch.equal(a.reshape(b.shape), b)
    lp, ent, top, idx = F().token_logprobs(z[0], t[0], 2)
    assert lp.shape == () and top.shape == (2,)
    none = F().token_logprobs(z[:0], t[:0], 2)
    assert none[0].shape == (0,) and none[3].shape == (0, 2)


def test_token_logprobs_agrees_with_cross_entropy():
    """The mean of -logprob is F.cross_entropy: two 32-bit evaluations of 1000 terms, 2^-24 * (1000 / 256 + 40) each."""
    g = gen(7)
    z = normal(g, (64, 1000), std=3.0).requires_grad_()
    t = torch.randint(0, 1000, (64,), generator=g, device="cuda")
    a = -F().token_logprobs(z, t)[0].mean()
    b = F().cross_entropy(z, t)
    assert abs(float(a) - float(b)) <= 2 * 44 * ref.E32 * (float(b) + 8)
    (da,) = torch.autograd.grad(a, z)
    (db,) = torch.autograd.grad(b, z)
    assert float((da - db).abs().max()) <= 4 * 44 * ref.E32 / 64


# ------------------------------------------------------------------------------------------ Newton-Schulz
def _ns_check(g, steps=5, coef=ref.COEF):
    got = F().newton_schulz(g, steps=steps, coefficients=coef)
    assert got.dtype == g.dtype and got.shape == g.shape and got.is_contiguous()
    value, rel = ref.newton_schulz(g, steps, coef)
    got = got.double().cpu()
    off = torch.linalg.vector_norm(got - value, dim=(-2, -1)) / torch.linalg.vector_norm(value, dim=(-2, -1)).clamp_min(1e-30)
    assert bool((off <= rel).all()), (off.max(), rel)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (7, 5), (64, 64), (33, 130), (130, 33), (2, 128, 128), (3, 100, 257),
                                   (2, 300, 129), (2, 2, 65, 64), (1, 384, 640), (640, 384)])
def test_newton_schulz(shape, dtype):
    # values around 1: fp16's own range does not cut them
    _ns_check(normal(gen(sum(shape)), shape, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(96, 40, 72), (97, 256, 130), (33, 300, 513), (10, 1024, 1030), (34, 264, 136),
                                   (33, 520, 264), (9, 1032, 1040), (6, 256, 2304), (6, 2304, 256), (20, 128, 1000), (5, 380, 1500),
                                   (150, 250, 300), (110, 500, 250), (1, 128, 2112)])
def test_newton_schulz_many_matrices(shape, dtype):
    """Enough tiles for the larger product kernels, upright and turned, rows of whole chunks and not."""
    _ns_check(normal(gen(sum(shape)), shape, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,m,n", [(1, 64, 200), (2, 200, 64), (40, 260, 300)])
def test_newton_schulz_strong_directions(batch, m, n, dtype):
    """A few directions 100 times the rest: the rest's singular values start near 10^-3 of the norm.  A result rounded
    to bf16 is off by 2^-8 / sqrt(3) in the quadratic mean at most, so the bound leaves 2^-8 * sqrt(2 / 3) = 3e-3 to the
    single-plane products, whose X keeps 22 bits."""
    g = gen(batch)
    u, v = normal(g, (batch, m, 4)), normal(g, (batch, 4, n))
    _ns_check((normal(g, (batch, m, n)) + 50.0 * torch.matmul(u, v)).to(dtype))


@pytest.mark.parametrize("steps", [1, 2, 5, 7])
def test_newton_schulz_steps_and_coefficients(steps):
    g = normal(gen(steps), (2, 96, 160))
    _ns_check(g, steps)
    # the classical cubic step: slope at most 1.5 on [0, 1], within the bound for slopes up to 4
    _ns_check(g, steps, (1.5, -0.5, 0.0))


def test_newton_schulz_scales():
    """The result does not depend on the scale of the update (in 64-bit norms: 1e-30 and 1e30 are fine)."""
    g = normal(gen(0), (48, 80))
    want = F().newton_schulz(g)
    for s in (2.0 ** -90, 2.0 ** 90):
        # eps = 1e-7 is felt only where the norm is near it: a norm of 62 * 2^-90 is all eps
        got = F().newton_schulz(g * s, eps=1e-38 if s < 1 else 1e-7)
        assert torch.allclose(got, want, rtol=0, atol=2e-4)


def test_newton_schulz_special_values():
    g = normal(gen(0), (4, 40, 24))
    g[1] = 0.0
    g[2, 3, 4] = math.nan
    g[3, 0, 0] = math.inf
    out = F().newton_schulz(g)
    assert not out[1].any() and out[0].isfinite().all()
    assert out[2].isnan().any() and not out[3].isfinite().all()
    one = F().newton_schulz(g[0])
    assert torch.equal(one, out[0])               # a matrix does not depend on its neighbours


def test_newton_schulz_strides():
    g = normal(gen(4), (3, 40, 56))
    want = F().newton_schulz(g)
    assert torch.equal(F().newton_schulz(g.transpose(0, 1).contiguous().transpose(0, 1)), want)
    assert torch.equal(F().newton_schulz(g.mT.contiguous().mT), want)


# ------------------------------------------------------------------------------------------ streams and graphs
def _everything(x, y, w, b, qkv, pos, freqs, axis, z, t, m):
    s, h = F().residual_norm(x, y, pre=F().Norm(w, b, 1e-5, "layer"))
    r = F().rotary(qkv, pos, freqs, axis, 2)
    lp, ent, top, idx = F().token_logprobs(z, t, 5)
    return [s, h, r, lp, ent, top, idx, F().newton_schulz(m)]


def _everything_inputs(seed):
    g = gen(seed)
    qkv, pos, freqs, axis = _rotary_case(2, 30, 2, 32, 16, 2, torch.bfloat16, seed=seed)
    return [normal(g, (4, 50, 128), torch.bfloat16), normal(g, (4, 50, 128), torch.bfloat16), normal(g, (128,)), normal(g, (128,)),
            qkv, pos, freqs, axis, normal(g, (2, 40000)), torch.randint(0, 40000, (2,), generator=g, device="cuda"),
            normal(g, (2, 100, 70))]


def test_other_stream():
    ins = _everything_inputs(0)
    want = _everything(*ins)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _everything(*ins)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_graph_replays_match_eager():
    """Two captured calls, replayed in turn with eager work and synchronisations between, on new inputs each time."""
    static = [_everything_inputs(0), _everything_inputs(1)]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for ins in static:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _everything(*ins)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(_everything(*ins))
        graphs.append(g)
    for rnd in range(3):
        want = []
        for q in range(2):
            new = _everything_inputs(10 + 2 * rnd + q)
            for a, b in zip(static[q], new):
                a.copy_(b)
            want.append([o.clone() for o in _everything(*new)])
        if rnd == 1:
            torch.cuda.synchronize()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for q in range(2):
            for a, b in zip(outs[q], want[q]):
                assert torch.equal(a, b)


def test_graph_of_forward_and_backward():
    case = _residual_case((4, 20, 96), torch.bfloat16, "layer", "rms", "sample", True)
    x, y, post, gate, scale, pre, ds, dh = case
    g = gen(1)
    z, t = normal(g, (8, 1000)), torch.randint(0, 1000, (8,), generator=g, device="cuda")
    qkv, pos, freqs, axis = _rotary_case(2, 30, 2, 32, 16, 2, torch.bfloat16)
    dq = normal(g, qkv.shape, torch.bfloat16)

    def step():
        # leaves of this call's own: a graph must not meet the gradient nodes of an eager call
        leaf = [v.detach().requires_grad_() for v in (x, y, gate, post.weight, post.bias, pre.weight, z, qkv)]
        s, h = F().residual_norm(leaf[0], leaf[1], post=F().Norm(leaf[3], leaf[4], 1e-5, "layer"), gate=leaf[2], scale=scale,
                                 pre=F().Norm(leaf[5], None, 1e-5, "rms"))
        lp, ent, top, _ = F().token_logprobs(leaf[6], t, 5)
        r = F().rotary(leaf[7], pos, freqs, axis, 2)
        return torch.autograd.grad([s, h, lp, ent, top, r], leaf, [ds, dh, lp.detach(), ent.detach(), top.detach(), dq])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for _ in range(3):
        want = [v.clone() for v in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        with torch.no_grad():
            x.add_(0.25)
            z.mul_(0.5)


def test_no_second_derivative():
    """A gradient of a gradient is refused, not left out."""
    case = _residual_case((2, 3, 16), torch.float32, None, "layer", None, False)
    x = case[0].requires_grad_()
    s, h = F().residual_norm(x, case[1], pre=case[5])
    qkv, pos, freqs, axis = _rotary_case(1, 4, 1, 16, 8, 2, torch.float32)
    z = normal(gen(0), (3, 20)).requires_grad_()
    for out, leaf in ((h, x), (F().rotary(qkv.requires_grad_(), pos, freqs, axis, 1), qkv),
                      (F().token_logprobs(z, torch.zeros(3, dtype=torch.int64, device="cuda"))[0], z)):
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(out.sum(), leaf, create_graph=True)


def test_same_tensor_twice_and_other_leaves():
    """x as both operands, one vector for both norms and the gate, an expanded gate, a gradient that is one number."""
    g = gen(4)
    x = normal(g, (3, 5, 24)).requires_grad_()
    w = normal(g, (24,), std=0.2, mean=1.0).requires_grad_()
    n = F().Norm(w, None, 1e-5, "rms")
    s, h = F().residual_norm(x, x, post=n, gate=w, pre=n)
    dx, dw = torch.autograd.grad(s.sum() + 2 * h.sum(), [x, w])
    ones = torch.ones_like(x)
    want = ref.residual_norm(x, x, n, w, None, n, ones, 2 * ones)
    ref.within(dx, want["d_x"][0] + want["d_y"][0], want["d_x"][1] + want["d_y"][1] + 4 * ref.E32 * want["d_x"][0].abs(), "dx")
    total = sum(want[k][0] for k in ("d_pre_w", "d_post_w", "d_gate"))
    ref.within(dw, total, sum(want[k][1] for k in ("d_pre_w", "d_post_w", "d_gate")) + 8 * ref.E32 * total.abs(), "dw")
    v = normal(g, (24,)).requires_grad_()
    s = F().residual_norm(x, x.detach(), gate=v.expand(3, 24))
    (dv,) = torch.autograd.grad(s.sum(), v)
    want = ref.residual_norm(x, x.detach(), None, v, None, None, ones)
    ref.within(dv, want["d_gate"][0], 4 * want["d_gate"][1], "expanded gate")


@pytest.mark.parametrize("dtype", DTYPES)
def test_parameters_in_16_bits(dtype):
    """Parameters of the activations' type (opt level O3): read in 32 bits, gradients rounded to their type."""
    if dtype == torch.float32:
        return
    x, y, post, gate, scale, pre, ds, dh = _residual_case((3, 6, 40), dtype, "layer", "rms", "channel", True)
    lo = lambda n: F().Norm(n.weight.to(dtype), None if n.bias is None else n.bias.to(dtype), n.eps, n.kind)  # noqa: E731
    case = (x, y, lo(post), gate.to(dtype), scale, lo(pre), ds, dh)
    want = ref.residual_norm(*case)
    got = _residual_run(*case)
    for name, (value, bound) in want.items():
        assert got[name].dtype == dtype
        ref.within(got[name], value, bound + ref.U[dtype] * value.abs(), name)


def test_results_repeat():
    ins = _everything_inputs(3)
    first = [o.clone() for o in _everything(*ins)]
    for _ in range(3):
        for a, b in zip(_everything(*ins), first):
            assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["residual_norm", "rotary", "token_logprobs", "newton_schulz"])
def test_refusals_on_the_device(name):
    """What the CPU backend refuses is refused here, with the same error, before anything is launched."""
    import test_transformer_ops_cpu as cpu

    with torch.device("cuda"):
        getattr(cpu, "test_%s_refusals" % name)()


def test_refuses_mixed_devices():
    x, w = torch.randn(2, 3, 8, device="cuda"), torch.ones(8)
    for call in (lambda: F().residual_norm(x, x.cpu()), lambda: F().residual_norm(x, x, pre=F().Norm(w)),
                 lambda: F().residual_norm(x, x, post=F().Norm(w.cuda(), w)), lambda: F().residual_norm(x, x, gate=w),
                 lambda: F().residual_norm(x, x, scale=torch.ones(2)), lambda: F().rms_norm(x, w),
                 lambda: F().token_logprobs(x, torch.zeros(2, 3, dtype=torch.int64)),
                 lambda: F().token_logprobs(x[0], torch.zeros(3, dtype=torch.int64)),
                 lambda: F().rotary(torch.randn(1, 3, 48, device="cuda"), torch.zeros(3, 1), torch.ones(4),
                                    torch.zeros(4, dtype=torch.int32), 2)):
        with pytest.raises(ValueError):
            call()


def test_second_backward():
    """A kept graph gives the same gradients again; a released one says so."""
    case = _residual_case((2, 3, 16), torch.float32, None, "layer", None, False)
    x = case[0].requires_grad_()
    s, h = F().residual_norm(x, case[1], pre=case[5])
    qkv, pos, freqs, axis = _rotary_case(1, 4, 1, 16, 8, 2, torch.float32)
    z = normal(gen(0), (3, 20)).requires_grad_()
    lp, ent, top, _ = F().token_logprobs(z, torch.zeros(3, dtype=torch.int64, device="cuda"), 4)
    for out, leaf in ((s.sum() + h.square().sum(), x), (F().rotary(qkv.requires_grad_(), pos, freqs, axis, 1).square().sum(), qkv),
                      (lp.sum() + (ent * ent).sum() + top.sum(), z)):
        a, = torch.autograd.grad(out, leaf, retain_graph=True)
        b, = torch.autograd.grad(out, leaf)
        assert torch.equal(a, b)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, leaf)


def test_saved_values_changed_in_place():
    """A value that backward needs and that was overwritten is noticed."""
    z = normal(gen(0), (3, 20)).requires_grad_()
    y = z * 1.0
    lp, ent, _, _ = F().token_logprobs(y, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lp.sum().backward()
