"""FusedMuon on the GPU, and the transformer operators together as a training step uses them."""
import copy
import json

import pytest
import torch

import _transformer_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _named(request):
    print(request.node.name, flush=True)
    yield
    torch.cuda.synchronize()


SHAPES = [(64, 96), (96, 64), (64, 96), (40, 40), (130, 70), (24, 16, 3, 3), (24, 16, 3, 3)]


def _params(seed):
    g = torch.Generator().manual_seed(seed)
    ps = []
    for s in SHAPES:
        w = torch.randn(s, generator=g)
        if len(s) == 4:
            w = w.contiguous(memory_format=torch.channels_last)
        ps.append(torch.nn.Parameter(w.cuda()))
    ps.append(torch.nn.Parameter(torch.randn(50, generator=g).cuda()))
    return ps


def _opt(ps, **kw):
    from distributed_pytorch_amd.optim import FusedMuon

    return FusedMuon([dict(params=ps[:-1], orthogonal=True), dict(params=ps[-1:])], lr=0.1, momentum=0.9, weight_decay=0.01, **kw)


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(nesterov):
    """Three steps against 64 bits.  A matrix is off by at most the step's size times the bound of its orthogonalised
    update (tests/_transformer_ref.py), times 1 + 0.9 + 0.81 for what earlier steps left in it, and a rounding of the
    parameter itself per step."""
    ps = _params(0)
    opt = _opt(ps, nesterov=nesterov)
    w = [p.detach().double().cpu() for p in ps]
    buf = [torch.zeros_like(t) for t in w]
    slack = [0.0] * len(ps)
    g = torch.Generator().manual_seed(1)
    for step in range(3):
        opt.zero_grad()
        grads = [torch.randn(p.shape, generator=g) for p in ps]
        for p, t in zip(ps, grads):
            p.grad = torch.empty_like(p).copy_(t)
        opt.step()
        for i, t in enumerate(grads):
            t = t.double()
            if i == len(ps) - 1:
                t = t + 0.01 * w[i]
                buf[i] = t if step == 0 else 0.9 * buf[i] + t
                w[i] = w[i] - 0.1 * buf[i]
                slack[i] += 4 * 2.0 ** -23 * float(w[i].norm() + buf[i].norm())
                continue
            buf[i] = 0.9 * buf[i] + t
            u = (t + 0.9 * buf[i] if nesterov else buf[i]).reshape(t.shape[0], -1)
            o, rel = ref.newton_schulz(u.float())
            f = 0.1 * 0.2 * max(1.0, u.shape[0] / u.shape[1]) ** 0.5
            w[i] = w[i] * (1 - 0.1 * 0.01) - f * o.reshape(t.shape)
            # (the momentum in 32 bits: 2^-22 of it, which the update enlarges by at most 4^5 / 3 relative to itself)
            slack[i] += f * (rel + 2.0 ** -22 * 342) * float(o.norm()) + 2.0 ** -23 * float(w[i].norm())
        for i, p in enumerate(ps):
            off = float((p.detach().double().cpu() - w[i]).norm())
            assert off <= slack[i], (step, i, off, slack[i])


def test_muon_overflow_skips_everything():
    from distributed_pytorch_amd.amp import LossScaler

    ps = _params(2)
    opt = _opt(ps)
    scaler = LossScaler(torch.device("cuda"), init_scale=4.0)
    for rnd in range(2):
        opt.zero_grad()
        for p in ps:
            p.grad = torch.ones_like(p) * 4.0
        if rnd == 1:
            ps[3].grad[0, 0] = float("nan")
        scaler.check_overflow([p.grad for p in ps])
        before = [p.detach().clone() for p in ps]
        bufs = [opt.state[p]["momentum_buffer"].clone() if rnd else None for p in ps]
        opt.arm_scaler(scaler)
        opt.step()
        for p, w, b in zip(ps, before, bufs):
            assert torch.equal(p, w) == (rnd == 1)
            if rnd == 1:
                assert torch.equal(opt.state[p]["momentum_buffer"], b)
    assert scaler.loss_scale() == 2.0


def _tiny(rotary=True, seed=0):
    from distributed_pytorch_amd import models

    torch.manual_seed(seed)
    m = models.vit.VisionTransformer(64, 16, 2, 4, 128, 256, num_classes=40, rotary=rotary)
    torch.nn.init.normal_(m.heads.head.weight, std=0.05)
    return m


def _loss(F, logits, target):
    lp, ent, top, _ = F.token_logprobs(logits, target, 3)
    return -lp.mean() - 0.1 * ent.mean() + 0.01 * top.sum(1).mean()


def test_training_step_of_all_operators(monkeypatch):
    """Rotary positions -> attention -> residual sums with their norms -> log probabilities -> Muon, against the CPU
    backend.  The attention core rounds its operands to 11 bits (2^-11 each, two products, two layers deep), so the
    logits are held to 6e-3 like the other whole-model comparisons, gradients to 2e-2 of their norm."""
    from distributed_pytorch_amd import amp
    from distributed_pytorch_amd.ops import functional as F
    from distributed_pytorch_amd.optim import FusedMuon, muon_groups

    monkeypatch.setattr(F, "_FUSE_RESIDUAL_NORM", True)
    amp.state().reset()
    cpu = _tiny()
    gpu = copy.deepcopy(cpu).cuda()
    x, t = torch.randn(6, 3, 64, 64), torch.randint(0, 40, (6,))
    opts = [FusedMuon(muon_groups(m), lr=0.05, momentum=0.9) for m in (cpu, gpu)]
    res = []
    for m, o, a, b in ((cpu, opts[0], x, t), (gpu, opts[1], x.cuda(), t.cuda())):
        logits = m(a)
        loss = _loss(F, logits, b)
        o.zero_grad()
        loss.backward()
        grads = {n: p.grad.detach().float().cpu().clone() for n, p in m.named_parameters()}
        o.step()
        res.append((logits.detach().float().cpu(), float(loss.detach()), grads))
    (l0, s0, g0), (l1, s1, g1) = res
    assert float((l0 - l1).abs().max()) <= 6e-3 * max(1.0, float(l0.abs().max())) and abs(s0 - s1) <= 6e-3 * max(1.0, abs(s0))
    floor = 1e-4 * max(float(g.norm()) / g.numel() ** 0.5 for g in g0.values())
    for n in g0:
        # (the key projection's bias has no gradient: a constant added to all scores of a row)
        off = float((g0[n] - g1[n]).norm()) / (float(g0[n].norm()) + floor * g0[n].numel() ** 0.5)
        assert off <= 2e-2, (n, off)
    for (n, p), q in zip(cpu.named_parameters(), gpu.parameters()):
        assert torch.isfinite(q).all() and float((p.detach() - q.detach().cpu()).abs().max()) < 0.2, n


@pytest.mark.parametrize("level", ["O0", "O2"])
def test_graphed_muon_training_matches_eager(level, monkeypatch):
    """The captured step replays what the eager one does, bit for bit: every kernel sums in a fixed order."""
    from distributed_pytorch_amd import amp
    from distributed_pytorch_amd.ops import functional as F
    from distributed_pytorch_amd.optim import FusedMuon, muon_groups
    from distributed_pytorch_amd.utils.graph import GraphedTrainStep

    monkeypatch.setattr(F, "_FUSE_RESIDUAL_NORM", True)
    runs = []
    for graphed in (False, True):
        amp.state().reset()
        m = _tiny(seed=3).cuda().train()
        opt = FusedMuon(muon_groups(m), lr=0.05, momentum=0.9)
        m, opt = amp.initialize(m, opt, opt_level=level, dtype="bf16")
        step = GraphedTrainStep(m, opt, warmup=2, enabled=graphed)
        g = torch.Generator().manual_seed(9)
        losses = []
        for i in range(7):
            x = torch.randn(4, 3, 64, 64, generator=g).cuda()
            t = torch.randint(0, 40, (4,), generator=g).cuda()
            opt.param_groups[0]["lr"] = 0.05 / (1 + i)
            loss, rec = step(x, t)
            losses.append(float(loss.detach()))
        assert (step.replays > 0) == graphed
        runs.append((losses, [p.detach().clone() for p in m.parameters()]))
    amp.state().reset()
    assert runs[0][0] == runs[1][0]
    for a, b in zip(runs[0][1], runs[1][1]):
        assert torch.equal(a, b)


def test_trainer_with_muon_and_predictions(tmp_path):
    from distributed_pytorch_amd import cli, engine

    out = tmp_path / "pred.jsonl"
    args = cli.parse("nd", ["-a", "vit_b_32", "--gpu", "0", "--synthetic", "--num-classes", "12", "-b", "4", "--epochs", "1",
                            "--steps", "4", "--optimizer", "muon", "--lr", "0.01", "--predictions", str(out),
                            "--out-dir", str(tmp_path), "--seed", "1"])
    engine.main(args)
    lines = [json.loads(l) for l in out.read_text().splitlines()]
    assert len(lines) == 4
    for l in lines:
        assert len(set(l["top"])) == 5 and l["top_logprob"] == sorted(l["top_logprob"], reverse=True)
        if l["target"] in l["top"]:
            assert l["logprob"] == l["top_logprob"][l["top"].index(l["target"])]


@pytest.mark.parametrize("arch,size", [("swin_t", 64), ("swin_v2_t", 64), ("convnext_tiny", 64)])
def test_fused_residual_models(arch, size, monkeypatch):
    """One forward and backward of the fused paths against the separate ones on the GPU, float32: the order of additions
    differs, and the attention core's 11-bit operands round where they land."""
    from distributed_pytorch_amd import amp, models
    from distributed_pytorch_amd.ops import functional as F

    amp.state().reset()
    torch.manual_seed(0)
    base = models.create_model(arch, num_classes=7)
    for n, p in base.named_parameters():
        if n.endswith("layer_scale"):
            p.data.fill_(0.5)
    x, t = torch.randn(2, 3, size, size).cuda(), torch.tensor([1, 5]).cuda()
    res = []
    for fused in (False, True):
        monkeypatch.setattr(F, "_FUSE_RESIDUAL_NORM", fused)
        m = copy.deepcopy(base).cuda().train()
        torch.manual_seed(5)
        torch.cuda.manual_seed_all(5)
        out = m(x)
        F.cross_entropy(out, t).backward()
        res.append((out.detach(), {n: p.grad.clone() for n, p in m.named_parameters()}))
    assert float((res[0][0] - res[1][0]).abs().max()) <= 6e-3 * max(1.0, float(res[0][0].abs().max()))
    floor = 1e-4 * max(float(g.norm()) / g.numel() ** 0.5 for g in res[0][1].values())
    for n, a in res[0][1].items():
        off = float((a - res[1][1][n]).norm()) / (float(a.norm()) + floor * a.numel() ** 0.5)
        assert off <= 2e-2, (n, off)
