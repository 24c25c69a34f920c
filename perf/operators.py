"""The transformer operators of the framework as a user's program calls them, over the sizes they are used at.

``own = False`` computes each operator in its plain form (elementary torch operations in 32 bits, 64 where 32 lose what
matters), ``own = True`` calls the framework.  Four operators:

* ``residual_norm``   s = x + scale * gate * post(y), h = pre(s), with its gradients
* ``rotary``          queries and keys of a packed projection turned by positions of several axes, with its gradient
* ``logprobs``        log probability of a given class / token, entropy and the k most probable ones, with gradients
* ``newton_schulz``   the orthogonalised update of a batch of matrices
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_COEF = (3.4445, -4.7750, 2.0315)


def listed():
    return [
        # one image through a ViT-B/16 block while serving: the residual sum and the next LayerNorm, latency counts
        dict(name="residual_serve", op="residual_norm", n=1, t=197, c=768, dtype="bf16", post="none", pre="layer",
             gate="none", scale=False, train=False),
        # ViT-L/16 training, 64 images: residual sum + LayerNorm, forward and backward
        dict(name="residual_vit_l_train", op="residual_norm", n=64, t=197, c=1024, dtype="bf16", post="none", pre="layer",
             gate="none", scale=False, train=True),
        # Swin V2-T stage 1, 64 images: LayerNorm AFTER the block, stochastic depth, residual sum
        dict(name="residual_swin_v2_train", op="residual_norm", n=64, t=56 * 56, c=96, dtype="bf16", post="layer",
             pre="none", gate="none", scale=True, train=True),
        # a conditioned block of ViT-H/14 width: RMSNorm on both sides and a gate for each sample, 32 bits
        dict(name="residual_gated_train", op="residual_norm", n=24, t=257, c=1280, dtype="f32", post="rms", pre="rms",
             gate="sample", scale=False, train=True),
        # one image of a ViT-B/16 while serving: 14 x 14 patches and the class token
        dict(name="rotary_serve", op="rotary", b=1, s=197, h=12, d=64, axes=2, rotated=64, interleaved=False,
             span=14, dtype="bf16", train=False),
        # ViT-H/14 training: 16 x 16 patches and the class token, heads of 80
        dict(name="rotary_vit_h_train", op="rotary", b=32, s=257, h=16, d=80, axes=2, rotated=80, interleaved=True,
             span=16, dtype="bf16", train=True),
        # video clips: time, height and width, a time stamp that runs far, a part of the head left as it is
        dict(name="rotary_video_train", op="rotary", b=4, s=3137, h=16, d=64, axes=3, rotated=48, interleaved=False,
             span=100000, dtype="f16", train=True),
        # the classifier's head: 1000 classes, the logits that F.linear(out_dtype=float32) gives, top 5
        dict(name="logprobs_classes_train", op="logprobs", n=1024, v=1000, k=5, dtype="f32", masked=0.0, train=True),
        # a language head: an odd number of tokens, some of them masked out
        dict(name="logprobs_tokens_train", op="logprobs", n=2048, v=50257, k=20, dtype="bf16", masked=0.1, train=True),
        # one new token over a long list: the row has to be split over the card
        dict(name="logprobs_one_token", op="logprobs", n=1, v=128000, k=20, dtype="f32", masked=0.0, train=False),
        # the 3x3 convolutions of a ResNet-50 stage as matrices of 256 x 2304
        dict(name="newton_schulz_conv", op="newton_schulz", b=6, m=256, n=2304, steps=5, dtype="f32"),
        # the second MLP product of every block of a ViT-L/16
        dict(name="newton_schulz_vit_l", op="newton_schulz", b=24, m=1024, n=4096, steps=5, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["residual_norm", "rotary", "logprobs", "newton_schulz"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "residual_norm":
        c = _log(rng, 48, 4096)
        if rng.random() < 0.7:
            c = -(-c // 8) * 8
        n = _log(rng, 1, 128)
        t = max(1, min(_log(rng, 1, 4096), (1 << 24) // (n * c)))
        post, pre = rng.choice(["none", "layer", "rms"]), rng.choice(["none", "layer", "rms"])
        return dict(op=op, n=n, t=t, c=c, dtype=dtype, post=post, pre=pre, gate=rng.choice(["none", "channel", "sample"]),
                    scale=rng.random() < 0.5, train=rng.random() < 0.7)
    if op == "rotary":
        h, d = rng.choice([1, 3, 6, 8, 12, 16, 24]), rng.choice([32, 48, 64, 80, 96, 128])
        axes = rng.choice([1, 2, 3])
        b = _log(rng, 1, 64)
        s = max(1, min(_log(rng, 1, 8192), (1 << 24) // (b * h * d)))
        rotated = d if rng.random() < 0.6 else 2 * rng.randint(axes, d // 2)
        return dict(op=op, b=b, s=s, h=h, d=d, axes=axes, rotated=rotated, interleaved=rng.random() < 0.5,
                    span=_log(rng, 4, 1000000), dtype=dtype, train=rng.random() < 0.7)
    if op == "logprobs":
        v = _log(rng, 2, 150000)
        n = max(1, min(_log(rng, 1, 8192), (1 << 26) // v))
        return dict(op=op, n=n, v=v, k=rng.randint(0, min(32, v)), dtype=dtype, masked=rng.choice([0.0, 0.0, 0.3]),
                    train=rng.random() < 0.6)
    m, n = _log(rng, 16, 2048), _log(rng, 16, 4096)
    if rng.random() < 0.5:
        m, n = -(-m // 32) * 32, -(-n // 32) * 32
    side = min(m, n)
    b = max(1, min(_log(rng, 1, 24), int(6e10 / (6.0 * side * m * n))))
    return dict(op=op, b=b, m=m, n=n, steps=rng.choice([3, 5, 5, 6]), dtype=rng.choice(["f32", "bf16"]))


def _normal(g, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std + mean).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"case": case, **_PREPARE[case["op"]](case, g)}


def _prepare_residual(c, g):
    dt = _DT[c["dtype"]]
    shape = (c["n"], c["t"], c["c"])
    st = dict(x=_normal(g, shape, dt, 1.5), y=_normal(g, shape, dt, 0.7, 0.1), gate=None, scale=None)
    for side in ("post", "pre"):
        if c[side] != "none":
            st[side + "_w"] = _normal(g, (c["c"],), std=0.2, mean=1.0)
            st[side + "_b"] = _normal(g, (c["c"],), std=0.2) if c[side] == "layer" else None
    if c["gate"] != "none":
        st["gate"] = _normal(g, (c["c"],) if c["gate"] == "channel" else (c["n"], c["c"]), std=0.3, mean=0.5)
    if c["scale"]:        # stochastic depth: a sample's branch is dropped or scaled up
        keep = torch.rand((c["n"],), generator=g, device="cuda") < 0.8
        st["scale"] = keep.float() / 0.8
    if c["train"]:
        st["ds"] = _normal(g, shape, dt)
        st["dh"] = _normal(g, shape, dt) if c["pre"] != "none" else None
        st["leaves"] = [k for k in ("x", "y", "gate", "post_w", "post_b", "pre_w", "pre_b") if st.get(k) is not None]
        for k in st["leaves"]:
            st[k].requires_grad_()
    return st


def _prepare_rotary(c, g):
    dt = _DT[c["dtype"]]
    st = dict(qkv=_normal(g, (c["b"], c["s"], 3 * c["h"] * c["d"]), dt))
    # whole positions of every axis, those of the first axis up to `span`
    pos = torch.rand((c["b"], c["s"], c["axes"]), generator=g, device="cuda", dtype=torch.float64)
    reach = torch.tensor([c["span"]] + [64] * (c["axes"] - 1), device="cuda", dtype=torch.float64)
    st["pos"] = (pos * reach).floor().to(torch.int64)
    pairs = c["rotated"] // 2
    each = [pairs // c["axes"] + (1 if a < pairs % c["axes"] else 0) for a in range(c["axes"])]
    freqs = torch.cat([10000.0 ** (-torch.arange(p, dtype=torch.float64) / max(p, 1)) for p in each])
    st["freqs"] = freqs.cuda()
    st["axis"] = torch.cat([torch.full((p,), a, dtype=torch.int32) for a, p in enumerate(each)]).cuda()
    if c["train"]:
        st["qkv"].requires_grad_()
        st["dout"] = _normal(g, st["qkv"].shape, dt)
    return st


def _prepare_logprobs(c, g):
    dt = _DT[c["dtype"]]
    z = _normal(g, (c["n"], c["v"]), std=2.0)
    target = torch.randint(0, c["v"], (c["n"],), generator=g, device="cuda")
    # a trained head knows something: the target's logit stands out in most rows
    rows = torch.arange(c["n"], device="cuda")
    z[rows, target] += 6.0
    if c["masked"]:
        drop = torch.rand((c["n"], c["v"]), generator=g, device="cuda") < c["masked"]
        drop[rows, target] = False
        z.masked_fill_(drop, -math.inf)
    st = dict(logits=z.to(dt), target=target)
    if c["train"]:
        st["logits"].requires_grad_()
        st["d_lp"] = _normal(g, (c["n"],))
        st["d_ent"] = _normal(g, (c["n"],))
        st["d_top"] = _normal(g, (c["n"], c["k"])) if not c["masked"] else torch.zeros((c["n"], c["k"]), device="cuda")
    return st


def _prepare_newton_schulz(c, g):
    # a momentum buffer: a few strong directions over noise
    b, m, n = c["b"], c["m"], c["n"]
    r = min(8, m, n)
    u, v = _normal(g, (b, m, r)), _normal(g, (b, r, n), std=1.0 / math.sqrt(r))
    return dict(g=(1e-3 * (_normal(g, (b, m, n)) + 0.5 * torch.matmul(u, v))).to(_DT[c["dtype"]]))


_PREPARE = {"residual_norm": _prepare_residual, "rotary": _prepare_rotary, "logprobs": _prepare_logprobs,
            "newton_schulz": _prepare_newton_schulz}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return _RUN[state["case"]["op"]](state, state["case"])


def _norm_plain(v, kind, w, b, eps):
    if kind == "layer":
        d = v - v.mean(-1, keepdim=True)
        return d * (d.square().mean(-1, keepdim=True) + eps).rsqrt() * w + b
    return v * (v.square().mean(-1, keepdim=True) + eps).rsqrt() * w


def _run_residual(st, c):
    if own:
        from distributed_pytorch_amd.ops import functional as F

        side = {k: None if c[k] == "none" else F.Norm(st[k + "_w"], st.get(k + "_b"), 1e-6, c[k]) for k in ("post", "pre")}
        out = F.residual_norm(st["x"], st["y"], gate=st["gate"], scale=st["scale"], **side)
        s, h = out if side["pre"] is not None else (out, None)
    else:
        z = st["y"].float()
        if c["post"] != "none":
            z = _norm_plain(z, c["post"], st["post_w"], st.get("post_b"), 1e-6)
        if c["gate"] != "none":
            z = z * (st["gate"] if c["gate"] == "channel" else st["gate"][:, None, :])
        if c["scale"]:
            z = z * st["scale"][:, None, None]
        s = st["x"].float() + z
        h = None if c["pre"] == "none" else _norm_plain(s, c["pre"], st["pre_w"], st.get("pre_b"), 1e-6).to(st["x"].dtype)
        s = s.to(st["x"].dtype)
    if not c["train"]:
        return dict(s=s, h=h)
    outs, grads = ([s], [st["ds"]]) if h is None else ([s, h], [st["ds"], st["dh"]])
    got = torch.autograd.grad(outs, [st[k] for k in st["leaves"]], grads)
    return dict(s=s, h=h, **{"d_" + k: v for k, v in zip(st["leaves"], got)})


def _run_rotary(st, c):
    if own:
        from distributed_pytorch_amd.ops import functional as F

        out = F.rotary(st["qkv"], st["pos"], st["freqs"], st["axis"], c["h"], interleaved=c["interleaved"])
    else:
        pairs = c["rotated"] // 2
        angle = st["pos"].double()[..., st["axis"].long()] * st["freqs"]                  # [B, S, pairs]
        cos, sin = angle.cos().float()[:, :, None, None, :], angle.sin().float()[:, :, None, None, :]
        v = st["qkv"].float().reshape(c["b"], c["s"], 3, c["h"], c["d"])
        qk, rest = v[:, :, :2], v[:, :, :2, :, c["rotated"]:]
        if c["interleaved"]:
            a, b = qk[..., 0:c["rotated"]:2], qk[..., 1:c["rotated"]:2]
            turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
        else:
            a, b = qk[..., :pairs], qk[..., pairs:2 * pairs]
            turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
        out = torch.cat([torch.cat([turned, rest], dim=-1), v[:, :, 2:]], dim=2).reshape(st["qkv"].shape).to(st["qkv"].dtype)
    if not c["train"]:
        return dict(out=out)
    (d,) = torch.autograd.grad([out], [st["qkv"]], [st["dout"]])
    return dict(out=out, d_qkv=d)


def _top_plain(z, k):
    """Indices of the k largest of every row, ties to the lowest index: one whole number per entry that orders both."""
    bits = (z.detach() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    column = torch.arange(z.shape[1], device=z.device)
    return torch.topk(order * (1 << 20) + (z.shape[1] - 1 - column), k, dim=1).indices


def _run_logprobs(st, c):
    if own:
        from distributed_pytorch_amd.ops import functional as F

        lp, ent, top, idx = F.token_logprobs(st["logits"], st["target"], c["k"])
    else:
        z = st["logits"].float()
        shifted = z - z.detach().amax(1, keepdim=True)
        logp = shifted - shifted.exp().sum(1, keepdim=True).log()
        lp = logp.gather(1, st["target"][:, None])[:, 0]
        # a masked class has probability zero and adds nothing
        ent = -(logp.exp() * torch.where(logp == -math.inf, 0.0, logp)).sum(1)
        idx = _top_plain(z, c["k"])
        top = logp.gather(1, idx)
    if not c["train"]:
        return dict(logprob=lp, entropy=ent, top=top, index=idx)
    (d,) = torch.autograd.grad([lp, ent, top], [st["logits"]], [st["d_lp"], st["d_ent"], st["d_top"]])
    return dict(logprob=lp, entropy=ent, top=top, index=idx, d_logits=d)


def _run_newton_schulz(st, c):
    if own:
        from distributed_pytorch_amd.ops import functional as F

        return dict(update=F.newton_schulz(st["g"], steps=c["steps"], coefficients=_COEF))
    a, b, k = _COEF
    x = st["g"].float()
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt().float() + 1e-7)
    turned = c["m"] > c["n"]
    x = x.mT.contiguous() if turned else x
    for _ in range(c["steps"]):
        gram = torch.matmul(x, x.mT.contiguous())
        x = a * x + torch.matmul(b * gram + k * torch.matmul(gram, gram), x)
    return dict(update=(x.mT if turned else x).to(st["g"].dtype).contiguous())


_RUN = {"residual_norm": _run_residual, "rotary": _run_rotary, "logprobs": _run_logprobs,
        "newton_schulz": _run_newton_schulz}


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    c, size = case, _BYTES[case["dtype"]]
    if c["op"] == "residual_norm":
        e = c["n"] * c["t"] * c["c"]
        has_h = c["pre"] != "none"
        tensors = 3 + has_h                                       # x, y -> s (, h)
        if c["train"]:                                            # ds (, dh) -> dx (, dy where it is not dx)
            apart = c["post"] != "none" or c["gate"] != "none" or c["scale"]
            tensors += 2 + has_h + apart
        return {"bytes": e * size * tensors, "flops": e * (30 if c["train"] else 10)}
    if c["op"] == "rotary":
        e = c["b"] * c["s"] * 3 * c["h"] * c["d"]
        passes = 2 if c["train"] else 1
        return {"bytes": passes * 2 * e * size + c["b"] * c["s"] * c["axes"] * 8,
                "flops": passes * 6 * c["b"] * c["s"] * 2 * c["h"] * c["rotated"] // 2}
    if c["op"] == "logprobs":
        e = c["n"] * c["v"]
        return {"bytes": e * size * (2 if c["train"] else 1) + c["n"] * (16 + 12 * c["k"]), "flops": e * (12 if c["train"] else 6)}
    m, n = min(c["m"], c["n"]), max(c["m"], c["n"])
    # the two products with a symmetric result need half of their entries
    return {"bytes": 2 * c["b"] * m * n * size, "flops": c["b"] * c["steps"] * (m * m * n + m ** 3 + 2 * m * m * n)}


# ------------------------------------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    with torch.no_grad():
        return _EXACT[case["op"]](prepare(case, seed), case)


def _norm64(v, kind, w, b):
    """(normalised and weighted, normalised, 1 / deviation)"""
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    dev = 1.0 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + 1e-6)
    unit = (v - mean) * dev
    return unit * w.double() + (0.0 if b is None else b.double()), unit, dev


def _norm64_back(g, kind, w, unit, dev):
    """gradients of (input, weight, bias)"""
    gw = g * w.double()
    gx = gw - unit * (gw * unit).mean(-1, keepdim=True)
    if kind == "layer":
        gx = gx - gw.mean(-1, keepdim=True)
    return gx * dev, (g * unit).sum((0, 1)), g.sum((0, 1))


def _exact_residual(st, c):
    x, y = st["x"].double(), st["y"].double()
    post = pre = None
    z = y
    if c["post"] != "none":
        post = _norm64(y, c["post"], st["post_w"], st.get("post_b"))
        z = post[0]
    row = st["scale"].double()[:, None, None] if c["scale"] else 1.0
    gate = 1.0
    if c["gate"] != "none":
        gate = st["gate"].double()
        gate = gate[:, None, :] if c["gate"] == "sample" else gate
    s = x + row * gate * z
    out = dict(s=s, h=None)
    if c["pre"] != "none":
        pre = _norm64(s, c["pre"], st["pre_w"], st.get("pre_b"))
        out["h"] = pre[0]
    if not c["train"]:
        return out
    ds = st["ds"].double()
    if pre is not None:
        g, out["d_pre_w"], db = _norm64_back(st["dh"].double(), c["pre"], st["pre_w"], pre[1], pre[2])
        ds = ds + g
        if c["pre"] == "layer":
            out["d_pre_b"] = db
    out["d_x"] = ds
    ds = ds * row
    if c["gate"] != "none":
        out["d_gate"] = (ds * z).sum(1) if c["gate"] == "sample" else (ds * z).sum((0, 1))
    dz = ds * gate
    if post is not None:
        dz, out["d_post_w"], db = _norm64_back(dz, c["post"], st["post_w"], post[1], post[2])
        if c["post"] == "layer":
            out["d_post_b"] = db
    out["d_y"] = dz
    return out


def _turn64(v, st, c, sign):
    """Every pair as a complex number times e^(i angle)."""
    pairs = c["rotated"] // 2
    angle = sign * torch.stack([st["pos"][..., int(a)].double() * f for a, f in zip(st["axis"].tolist(), st["freqs"])], -1)
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if c["interleaved"] else (slice(0, pairs), slice(pairs, 2 * pairs))
    out = v.double().reshape(c["b"], c["s"], 3, c["h"], c["d"]).clone()
    w = torch.polar(torch.ones_like(angle), angle)[:, :, None, :]
    for which in range(2):
        turned = torch.complex(out[:, :, which, :, first].contiguous(), out[:, :, which, :, second].contiguous()) * w
        out[:, :, which, :, first], out[:, :, which, :, second] = turned.real, turned.imag
    return out.reshape(v.shape)


def _exact_rotary(st, c):
    out = dict(out=_turn64(st["qkv"], st, c, 1.0))
    if c["train"]:
        out["d_qkv"] = _turn64(st["dout"], st, c, -1.0)
    return out


def _exact_logprobs(st, c):
    z, t, k = st["logits"], st["target"], c["k"]
    outs = []
    for i in range(0, c["n"], 256):                     # rows in parts: 64 bits of them all are large
        rows = z[i:i + 256].double()
        logp = rows - torch.logsumexp(rows, 1, keepdim=True)
        p = logp.exp()
        fin = torch.where(logp == -math.inf, 0.0, logp)
        ent = -(p * fin).sum(1)
        idx = torch.sort(rows, dim=1, descending=True, stable=True).indices[:, :k]
        part = dict(logprob=logp.gather(1, t[i:i + 256, None])[:, 0], entropy=ent, top=logp.gather(1, idx), index=idx)
        if c["train"]:
            glp, ge, gt = (st[n][i:i + 256].double() for n in ("d_lp", "d_ent", "d_top"))
            d = -p * (glp + gt.sum(1))[:, None] - ge[:, None] * p * (fin + ent[:, None])
            d.scatter_add_(1, t[i:i + 256, None], glp[:, None])
            d.scatter_add_(1, idx, gt)
            part["d_logits"] = d
        outs.append(part)
    return {n: torch.cat([o[n] for o in outs]) for n in outs[0]}


def _exact_newton_schulz(st, c):
    """With products on the other side: X (a + b M + c M M), M = X^T X."""
    if c["b"] * c["steps"] * 4.0 * c["n"] * c["n"] * (c["m"] + c["n"]) > 4e14:
        return None
    a, b, k = _COEF
    outs = []
    for one in st["g"]:
        x = one.double()
        x = x / (torch.linalg.vector_norm(x) + 1e-7)
        for _ in range(c["steps"]):
            gram = x.t().contiguous() @ x
            poly = b * gram + k * (gram @ gram)
            poly.diagonal().add_(a)
            x = x @ poly
        outs.append(x)
    return dict(update=torch.stack(outs))


_EXACT = {"residual_norm": _exact_residual, "rotary": _exact_rotary, "logprobs": _exact_logprobs,
          "newton_schulz": _exact_newton_schulz}
