"""FusedMuon, the axial rotary module, the models' options and the trainer flags on the CPU backend."""
import copy
import json
import math

import pytest
import torch

from distributed_pytorch_amd import models
from distributed_pytorch_amd.nn.modules import AxialRotary, LayerNorm, RMSNorm
from distributed_pytorch_amd.ops import functional as F
from distributed_pytorch_amd.optim import FusedMuon, FusedSGD, muon_groups


def _params(seed=0):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g)) for s in ((6, 10), (10, 6), (7,), (4, 3, 3, 3))]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g)
    return ps


def test_muon_step_formula():
    ps = _params()
    before = [p.detach().clone() for p in ps]
    opt = FusedMuon([dict(params=[ps[0], ps[1], ps[3]], orthogonal=True), dict(params=[ps[2]])], lr=0.1, momentum=0.9,
                    weight_decay=0.01, matrix_scale=0.5)
    bufs = [torch.zeros_like(p) for p in ps]
    for _ in range(3):
        opt.step()
        for i, (p, w) in enumerate(zip(ps, before)):
            g = p.grad
            if i == 2:
                g = g + 0.01 * w
                bufs[i] = g.clone() if not bufs[i].any() else 0.9 * bufs[i] + g
                w.sub_(0.1 * bufs[i])
                continue
            bufs[i] = 0.9 * bufs[i] + g
            u = (g + 0.9 * bufs[i]).reshape(p.shape[0], -1)
            o = F.newton_schulz(u).reshape(p.shape)
            w.mul_(1 - 0.1 * 0.01).sub_(0.1 * 0.5 * max(1.0, u.shape[0] / u.shape[1]) ** 0.5 * o)
    for p, w in zip(ps, before):
        assert torch.allclose(p, w, rtol=1e-5, atol=1e-6)


def test_muon_without_matrices_is_sgd():
    a, b = _params(1), _params(1)
    x = FusedMuon([dict(params=a)], lr=0.1, momentum=0.9, weight_decay=0.01)
    y = FusedSGD(b, lr=0.1, momentum=0.9, weight_decay=0.01)
    for _ in range(3):
        x.step()
        y.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_muon_state_roundtrip_and_groups():
    a, b = _params(2), _params(2)
    x, y = FusedMuon(a, lr=0.1), FusedMuon(b, lr=0.1)
    assert [g["orthogonal"] for g in x.param_groups] == [True, False]
    x.step()
    y.load_state_dict(copy.deepcopy(x.state_dict()))       # (loading shares the buffers otherwise)
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    x.step()
    y.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    extra = torch.nn.Parameter(torch.ones(3))
    x.add_param_group(dict(params=[extra]))
    assert x.param_groups[-1]["orthogonal"] is False


def test_muon_skips_a_step_that_overflowed():
    from distributed_pytorch_amd.amp import LossScaler

    ps = _params(3)
    opt = FusedMuon(ps, lr=0.1)
    scaler = LossScaler(torch.device("cpu"), init_scale=8.0)
    ps[0].grad[0, 0] = math.inf
    scaler.check_overflow([p.grad for p in ps])
    before = [p.detach().clone() for p in ps]
    opt.arm_scaler(scaler)
    opt.step()
    assert all(torch.equal(p, w) for p, w in zip(ps, before)) and scaler.loss_scale() == 4.0


def test_muon_refusals():
    ps = _params()
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-1.0), dict(matrix_scale=0.0), dict(ns_steps=0),
               dict(ns_eps=0.0), dict(ns_coefficients=(5.0, 1.0, 1.0))):
        with pytest.raises(ValueError):
            FusedMuon(ps, **kw)
    for group in (dict(params=[ps[2]], orthogonal=True), dict(params=[ps[0]], orthogonal=True, ns_coefficients=(5.0, 1.0, 1.0)),
                  dict(params=[ps[0]], orthogonal=True, ns_steps=0), dict(params=[ps[0]], orthogonal=True, dampening=0.5)):
        with pytest.raises(ValueError):
            FusedMuon([group])


def test_muon_groups_of_models():
    vit = models.create_model("vit_b_32", num_classes=10)
    mats, rest = muon_groups(vit)
    names = {id(p): n for n, p in vit.named_parameters()}
    inside, outside = {names[id(p)] for p in mats["params"]}, {names[id(p)] for p in rest["params"]}
    assert "encoder.layers.encoder_layer_0.self_attention.in_proj_weight" in inside
    assert "encoder.layers.encoder_layer_3.mlp.3.weight" in inside
    assert {"conv_proj.weight", "heads.head.weight", "class_token", "encoder.pos_embedding"} <= outside
    assert len(inside) == 12 * 4 and len(inside) + len(outside) == len(names)
    res = models.create_model("resnet18", num_classes=10)
    mats, rest = muon_groups(res)
    assert all(p.dim() == 4 for p in mats["params"]) and not any(p is res.conv1.weight for p in mats["params"])


def test_axial_rotary_module():
    rot = AxialRotary(16, (6, 8), base=50.0)
    assert rot.freqs.dtype == torch.float64 and rot.axis.tolist() == [0] * 3 + [1] * 4
    assert rot.to(torch.bfloat16).freqs.dtype == torch.float64 and float(rot.freqs[1]) == pytest.approx(50.0 ** (-2 / 6), rel=1e-15)
    assert rot.half().double().freqs.dtype == torch.float64 and not rot.state_dict()
    grid = AxialRotary.grid(2, 3, class_token=True)
    assert grid.tolist() == [[0, 0], [1, 1], [1, 2], [1, 3], [2, 1], [2, 2], [2, 3]]
    x = torch.randn(2, 7, 3 * 2 * 16)
    assert torch.equal(rot(x, grid, 2)[:, 0], x[:, 0])             # the class token does not turn
    for bad in ((3, 4), (10, 8), ()):
        with pytest.raises(ValueError):
            AxialRotary(16, bad)


def test_vit_with_rotary_positions():
    torch.manual_seed(0)
    plain = models.vit.VisionTransformer(32, 8, 2, 2, 32, 64, num_classes=5)
    turned = models.vit.VisionTransformer(32, 8, 2, 2, 32, 64, num_classes=5, rotary=True)
    turned.load_state_dict(plain.state_dict())                     # the same keys
    torch.nn.init.normal_(plain.heads.head.weight)
    turned.heads.head.weight.data.copy_(plain.heads.head.weight)
    x = torch.randn(2, 3, 32, 32)
    a, b = plain(x), turned(x)
    assert a.shape == b.shape and not torch.allclose(a, b)
    b.sum().backward()
    assert all(p.grad is not None for p in turned.parameters())


@pytest.mark.parametrize("arch,size", [("vit_b_32", 224), ("swin_t", 64), ("swin_v2_t", 64), ("convnext_tiny", 64)])
def test_fused_residual_paths_agree(arch, size, monkeypatch):
    """The fused paths compute the same function, with the same random numbers: in float32 they differ by the order of
    additions alone (2^-24 each, some hundreds deep, through two blocks per layer: 1e-4 of the largest logit)."""
    torch.manual_seed(0)
    m = models.create_model(arch, num_classes=7).train()
    for n, p in m.named_parameters():
        if n.endswith("layer_scale"):
            p.data.fill_(0.5)
        if n == "heads.head.weight":
            torch.nn.init.normal_(p.data, std=0.02)
    x = torch.randn(2, 3, size, size)
    got = []
    for fused in (False, True):
        monkeypatch.setattr(F, "_FUSE_RESIDUAL_NORM", fused)
        torch.manual_seed(5)
        got.append(m(x))
    assert float((got[0] - got[1]).abs().max()) <= 1e-4 * float(got[0].abs().max())


def test_norm_specs():
    ln, rms = LayerNorm(8, eps=1e-3), RMSNorm(8, eps=1e-4)
    assert ln.spec().kind == "layer" and ln.spec().weight is ln.weight and ln.spec().eps == 1e-3
    assert rms.spec() == (rms.weight, None, 1e-4, "rms")
    x = torch.randn(3, 8)
    assert torch.equal(rms(x), F.rms_norm(x, rms.weight, 1e-4))


def test_trainer_with_muon_and_predictions(tmp_path):
    from distributed_pytorch_amd import cli, engine

    out = tmp_path / "pred.jsonl"
    args = cli.parse("nd", ["-a", "squeezenet1_1", "--cpu", "--synthetic", "--num-classes", "9", "-b", "4", "--epochs", "1",
                            "--steps", "4", "--optimizer", "muon", "--lr", "0.01", "--predictions", str(out),
                            "--out-dir", str(tmp_path), "--seed", "1"])
    engine.main(args)
    lines = [json.loads(l) for l in out.read_text().splitlines()]
    assert [l["sample"] for l in lines] == list(range(len(lines))) and len(lines) == 4
    for l in lines:
        assert len(l["top"]) == 5 and len(set(l["top"])) == 5 and 0.0 <= l["entropy"] <= math.log(9) + 1e-5
        assert l["logprob"] <= 0.0 and l["top_logprob"] == sorted(l["top_logprob"], reverse=True)
        if l["target"] in l["top"]:
            assert l["logprob"] == pytest.approx(l["top_logprob"][l["top"].index(l["target"])], abs=1e-6)


@pytest.mark.parametrize("arch", ["swin_t", "swin_v2_t", "vit_b_32"])
def test_groups_hold_products_only(arch):
    """Every orthogonalised parameter is the weight of a product: no position table, embedding, token or norm is one."""
    model = models.create_model(arch)
    names = {id(p): n for n, p in model.named_parameters()}
    groups = muon_groups(model)
    assert sum(len(g["params"]) for g in groups) == len(names)
    for p in groups[0]["params"]:
        assert names[id(p)].endswith("weight") and p.dim() in (2, 4)
    rest = {names[id(p)] for p in groups[1]["params"]}
    assert not any(n.endswith("bias_table") for n in names.values()) or any(n.endswith("bias_table") for n in rest)
    assert not any("bias_table" in names[id(p)] or "pos_embedding" in names[id(p)] for p in groups[0]["params"])
