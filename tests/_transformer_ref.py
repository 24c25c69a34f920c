"""64-bit references of the transformer-block operators, with bounds on how far a kernel may be from them.

A result of type T that is computed in 32 bits and rounded once is off by at most U[T] * |value| (half a step of T) plus
the 32-bit error, a small multiple of 2^-24 times the magnitude of the terms that were summed."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E32 = 2.0 ** -24
# below a type's normal range its steps no longer shrink with the value: half of the smallest one (fp16: values under
# 2^-14 are multiples of 2^-24, so rounding is off by up to 2^-25 there, whatever the value)
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def within(got, ref, bound, what):
    bound = bound.double().cpu() + TINY.get(got.dtype, 0.0)
    got, ref = got.detach().double().cpu(), ref.double().cpu()
    assert got.shape == ref.shape, "%s: shape %s, reference %s" % (what, tuple(got.shape), tuple(ref.shape))
    same = torch.isfinite(ref)
    assert torch.equal(same, torch.isfinite(got)), "%s: not finite in other places" % what
    assert torch.equal(ref[~same].nan_to_num(7.0), got[~same].nan_to_num(7.0)), "%s: other infinities" % what
    err = torch.where(same, got - ref, 0.0).abs()
    over = err - torch.where(same, bound, 0.0).expand_as(err)
    if (over > 0).any():
        i = int(over.argmax())
        raise AssertionError("%s: %d of %d too far off; worst %g, reference %g, off by %g, bound %g" % (
            what, int((over > 0).sum()), err.numel(), got.flatten()[i], ref.flatten()[i], err.flatten()[i],
            bound.expand_as(err).flatten()[i]))


# ------------------------------------------------------------------------------------------ residual norm
def _unit(v, norm):
    mean = v.mean(-1, keepdim=True) if norm.kind == "layer" else torch.zeros_like(v[..., :1])
    rstd = 1.0 / ((v - mean).square().mean(-1, keepdim=True) + norm.eps).sqrt()
    return (v - mean) * rstd, mean, rstd


def _unit_error(v, mean, rstd, rel):
    """Bound on the error of (v - mean) * rstd where v is off by rel * |v| and the arithmetic is 32-bit: the mean's and
    the deviation's sums run over at most 64 lanes x 8 chunks x 8 elements, a depth of some 32 additions each way."""
    d, k = (v - mean).abs(), 48 * E32
    dv = rel * v.abs() + k * (v.abs() + v.abs().mean(-1, keepdim=True)) + rel * v.abs().mean(-1, keepdim=True)
    # deviation: relative error of the mean square is at most 2 dv / d in the quadratic mean
    rr = rstd * (dv.square().mean(-1, keepdim=True).sqrt()) + k
    return rstd * dv + d * rstd * rr


def residual_norm(x, y, post=None, gate=None, scale=None, pre=None, ds=None, dh=None):
    """-> {name: (value, bound)} for s, h and, with ds / dh, the gradients of x, y, gate, post.*, pre.*"""
    T = x.dtype
    u = U[T]
    X, Y = x.detach().double(), y.detach().double()
    N, C = X.shape[0], X.shape[-1]
    out = {}
    z, ez = Y, torch.zeros_like(Y)
    if post is not None:
        yh, ym, yr = _unit(Y, post)
        eyh = _unit_error(Y, ym, yr, 0.0)
        w = post.weight.detach().double()
        b = torch.zeros_like(w) if post.bias is None else post.bias.detach().double()
        z, ez = yh * w + b, eyh * w.abs() + 4 * E32 * (yh * w).abs() + 4 * E32 * b.abs()
    f = torch.ones_like(X[..., :1])
    if scale is not None:
        f = scale.detach().double().reshape((N,) + (1,) * (X.dim() - 1))
    g = torch.ones((1,) * X.dim(), dtype=torch.float64, device=X.device)
    if gate is not None:
        g = gate.detach().double()
        g = g.reshape((1,) * (X.dim() - 1) + (C,)) if gate.dim() == 1 else g.reshape((N,) + (1,) * (X.dim() - 2) + (C,))
    fg = f * g
    s = X + fg * z
    es = fg.abs() * ez + 8 * E32 * (X.abs() + (fg * z).abs())
    out["s"] = (s, u * s.abs() + 1.01 * es)
    if pre is not None:
        sh, sm, sr = _unit(s, pre)
        w = pre.weight.detach().double()
        b = torch.zeros_like(w) if pre.bias is None else pre.bias.detach().double()
        h = sh * w + b
        rel_s = 0.0
        esh = _unit_error(s, sm, sr, rel_s) + sr * (es + es.mean(-1, keepdim=True)) + sh.abs() * sr * es.square().mean(-1, keepdim=True).sqrt()
        out["h"] = (h, u * h.abs() + 1.01 * (esh * w.abs() + 4 * E32 * ((sh * w).abs() + b.abs())))
    if ds is None and dh is None:
        return out
    rows = tuple(range(X.dim() - 1))
    n_rows = X.numel() // C
    depth = (n_rows ** 0.5 + 64) * E32        # sums over rows: long ones split over workgroups, lanes and a fold
    D = torch.zeros_like(X) if ds is None else ds.double()
    eD = torch.zeros_like(X)
    if pre is not None:
        G = torch.zeros_like(X) if dh is None else dh.double()
        gw = G * w
        m0 = gw.mean(-1, keepdim=True) if pre.kind == "layer" else 0.0
        m1 = (gw * sh).mean(-1, keepdim=True)
        # (backward forms s again in 32 bits)
        exh = esh
        D = D + sr * (gw - m0 - sh * m1)
        am = gw.abs().mean(-1, keepdim=True)
        em1 = (gw.abs() * exh).mean(-1, keepdim=True) + 48 * E32 * (gw * sh).abs().mean(-1, keepdim=True)
        eD = sr * (48 * E32 * (gw.abs() + am + (sh * m1).abs()) + sh.abs() * em1 + exh * m1.abs())
        rr = sr * es.square().mean(-1, keepdim=True).sqrt() + 64 * E32
        eD = eD + rr * (sr * (gw - m0 - sh * m1)).abs()
        out["d_pre_w"] = ((G * sh).sum(rows), (G.abs() * exh).sum(rows) + depth * (G * sh).abs().sum(rows))
        if pre.bias is not None:
            out["d_pre_b"] = (G.sum(rows), depth * G.abs().sum(rows))
    out["d_x"] = (D, u * D.abs() + 1.01 * (eD + 4 * E32 * D.abs()))
    dzs, edzs = f * D, f.abs() * (eD + 4 * E32 * D.abs())
    if gate is not None:
        v, e = dzs * z, edzs * z.abs() + dzs.abs() * ez + 4 * E32 * (dzs * z).abs()
        over = rows if gate.dim() == 1 else tuple(range(1, X.dim() - 1))
        total = (lambda t: t.sum(over)) if over else (lambda t: t)
        out["d_gate"] = (total(v), total(e) + depth * total(v.abs()))
    dz, edz = dzs * g, edzs * g.abs() + 4 * E32 * (dzs * g).abs()
    if post is not None:
        out["d_post_w"] = ((dz * yh).sum(rows), (edz * yh.abs() + dz.abs() * eyh).sum(rows) + depth * (dz * yh).abs().sum(rows))
        if post.bias is not None:
            out["d_post_b"] = (dz.sum(rows), edz.sum(rows) + depth * dz.abs().sum(rows))
        w = post.weight.detach().double()
        gw, egw = dz * w, edz * w.abs() + 4 * E32 * (dz * w).abs()
        m0 = gw.mean(-1, keepdim=True) if post.kind == "layer" else torch.zeros_like(gw[..., :1])
        m1 = (gw * yh).mean(-1, keepdim=True)
        em0 = egw.mean(-1, keepdim=True) + 48 * E32 * gw.abs().mean(-1, keepdim=True)
        em1 = (egw * yh.abs() + gw.abs() * eyh).mean(-1, keepdim=True) + 48 * E32 * (gw * yh).abs().mean(-1, keepdim=True)
        dz = yr * (gw - m0 - yh * m1)
        edz = yr * (egw + em0 + yh.abs() * em1 + eyh * m1.abs()) + 64 * E32 * yr * (gw.abs() + m0.abs() + (yh * m1).abs())
        # the deviation is computed in 32 bits from 32-bit values
        edz = edz + dz.abs() * 96 * E32 * (1 + (ym.abs() * yr).square())
    out["d_y"] = (dz, u * dz.abs() + 1.01 * (edz + 4 * E32 * dz.abs()))
    return out


# ------------------------------------------------------------------------------------------ rotary
def rotary(qkv, pos, freqs, axis, H, interleaved, sign=1.0):
    """-> (value, bound).  Sine and cosine are within 8 * 2^-24: the fraction of a turn is rounded to 32 bits (at most
    2^-25 of a turn, pi 2^-24 radians) and evaluated to 2 units."""
    B, S, W = qkv.shape
    D, P = W // (3 * H), freqs.numel()
    v = qkv.detach().double().reshape(B, S, 3, H, D).clone()
    bound = U[qkv.dtype] * 0.0 * v.abs()
    angle = sign * pos.double()[..., axis.long()] * freqs.double()
    cos, sin = (t.reshape(B, S, 1, 1, P) if t.dim() == 3 else t.reshape(1, S, 1, 1, P) for t in (angle.cos(), angle.sin()))
    i, j = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    a, b = v[:, :, :2, :, i].clone(), v[:, :, :2, :, j].clone()
    first, second = a * cos - b * sin, a * sin + b * cos
    v[:, :, :2, :, i], v[:, :, :2, :, j] = first, second
    slack = 10 * E32 * (a.abs() + b.abs())
    bound[:, :, :2, :, i] = U[qkv.dtype] * first.abs() + slack
    bound[:, :, :2, :, j] = U[qkv.dtype] * second.abs() + slack
    return v.reshape(qkv.shape), bound.reshape(qkv.shape)


# ------------------------------------------------------------------------------------------ log probabilities
def token_logprobs(z, t, k, d_lp=None, d_ent=None, d_top=None):
    """-> {name: (value, bound)}; index as (value, None).  e^d is off by (|d| + 4) 2^-24 relative (the argument's rounding
    and the function's), a lane adds at most V / 256 + 8 of them in a row and 14 more join lanes, waves and parts."""
    Z = z.detach().double().cpu()
    t = t.cpu().long()
    N, V = Z.shape
    empty = (Z == -math.inf).all(1)
    Zs = torch.where(empty[:, None], torch.zeros_like(Z), Z)
    shift = Zs - Zs.amax(1, keepdim=True)          # (the largest is taken out first: 64 bits do not hold 10^38 + log V)
    logp = shift - shift.exp().sum(1, keepdim=True).log()
    p = logp.exp()
    fin = torch.where(logp == -math.inf, 0.0, logp)
    ent = -(p * fin).sum(1)
    valid = (t >= 0) & (t < V)
    lp = logp.gather(1, t.clamp(0, V - 1)[:, None])[:, 0]
    d = fin - fin.max(1, keepdim=True).values
    terms = (V / 256 + 24) * E32
    e_s = terms + (p * (d.abs() + 4) * E32).sum(1)                              # relative error of S
    e_lse = 1.1 * e_s + 4 * E32 * (1 + math.log(V + 1))
    mean_d = (p * d.abs()).sum(1)
    e_ent = 1.1 * (2 * e_s * (mean_d + 1) + (p * d.abs() * (d.abs() + 6) * E32).sum(1) + terms * mean_d) + 8 * E32 * (ent + mean_d + 1)
    idx = torch.sort(Z, dim=1, descending=True, stable=True).indices[:, :k]
    top = logp.gather(1, idx)
    out = {"logprob": (torch.where(valid, torch.where(empty, -math.inf, lp), 0.0), e_lse + 4 * E32 * torch.where(lp == -math.inf, 0.0, lp).abs()),
           "entropy": (torch.where(empty, 0.0, ent), e_ent),
           "top": (torch.where(empty[:, None], -math.inf, top), e_lse[:, None] + 4 * E32 * torch.where(top == -math.inf, 0.0, top).abs()),
           "index": (idx, None)}
    if d_lp is None and d_ent is None and d_top is None:
        return out
    glp = torch.where(valid, 0.0 if d_lp is None else d_lp.double().cpu(), 0.0)
    ge = torch.zeros(N, dtype=torch.float64) if d_ent is None else d_ent.double().cpu()
    gt = torch.zeros(N, k, dtype=torch.float64) if d_top is None else d_top.double().cpu()
    gsum = glp + gt.sum(1)
    a = -p * gsum[:, None]
    b = -ge[:, None] * p * (fin + ent[:, None])
    dz = a + b
    dz.scatter_add_(1, t.clamp(0, V - 1)[:, None], glp[:, None])
    dz.scatter_add_(1, idx, gt)
    rel = e_lse[:, None] + (fin.abs() + 6) * E32
    bound = p * rel * (gsum.abs()[:, None] + ge.abs()[:, None] * (fin.abs() + ent[:, None]))
    bound = bound + p * ge.abs()[:, None] * (e_lse[:, None] + e_ent[:, None] + 8 * E32 * (fin.abs() + ent[:, None]))
    extra = torch.zeros_like(p)
    extra.scatter_add_(1, t.clamp(0, V - 1)[:, None], glp.abs()[:, None])
    extra.scatter_add_(1, idx, gt.abs())
    bound = bound + (k + 8) * E32 * (p * (glp.abs() + gt.abs().sum(1))[:, None] + extra + dz.abs())
    dz = torch.where(empty[:, None], 0.0, dz)
    out["d_logits"] = (dz, U[z.dtype] * dz.abs() + bound)
    return out


# ------------------------------------------------------------------------------------------ Newton-Schulz
COEF = (3.4445, -4.7750, 2.0315)


def newton_schulz(g, steps=5, coef=COEF, eps=1e-7):
    """-> (value, relative bound on the 2-norm of the error of one matrix).  A step's products carry 22 to 24 significant
    bits: together at most 8 * 2^-23 of the result's norm, and a step enlarges what it is given by at most 4 (the
    largest slope of a x + b x^3 + c x^5 on the singular values that occur): 8 * 2^-23 * (4^steps - 1) / 3, then the
    rounding to the result's type."""
    a, b, c = coef
    x = g.detach().double().cpu()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + eps)
    for _ in range(steps):
        gram = x.mT @ x if x.shape[-2] > x.shape[-1] else x @ x.mT
        poly = b * gram + c * (gram @ gram)
        x = a * x + (x @ poly if x.shape[-2] > x.shape[-1] else poly @ x)
    return x, 8 * 2.0 ** -23 * (4.0 ** steps - 1) / 3 + U[g.dtype]
