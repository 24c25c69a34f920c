"""Worker of the data-parallel tests of FusedMuon and the fused residual sums; must be importable by spawned children."""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

PER = 4          # samples of a rank


def model_and_optimizer(wrap=lambda m: m, device="cpu"):
    """A small vision transformer with rotary positions (every parameter of the residual sums is a norm's) beside a ConvNeXt
    block (whose gate is a parameter)."""
    from distributed_pytorch_amd import models
    from distributed_pytorch_amd.models.convnext import CNBlock
    from distributed_pytorch_amd.optim import FusedMuon, muon_groups

    torch.manual_seed(11)
    vit = models.vit.VisionTransformer(32, 8, 2, 2, 64, 96, num_classes=10, rotary=True)
    torch.nn.init.normal_(vit.heads.head.weight, std=0.1)
    net = Pair(vit, CNBlock(16, 0.5, 0.0)).to(device)
    net = wrap(net)
    return net, FusedMuon(muon_groups(getattr(net, "module", net)), lr=0.05, momentum=0.9, weight_decay=0.01)


class Pair(torch.nn.Module):
    def __init__(self, vit, block):
        super().__init__()
        self.vit, self.block = vit, block

    def forward(self, x, y):
        return self.vit(x), self.block(y)


def batch(world):
    g = torch.Generator().manual_seed(5)
    n = PER * world
    return (torch.randn(2, n, 3, 32, 32, generator=g), torch.randn(2, n, 8, 8, 16, generator=g),
            torch.randint(0, 10, (2, n), generator=g))


def loss_of(net, x, y, t):
    from distributed_pytorch_amd.ops import functional as F

    logits, h = net(x, y)
    lp, ent, _, _ = F.token_logprobs(logits, t)
    return -lp.mean() - 0.1 * ent.mean() + h.float().square().mean()


def one_step(net, opt, x, y, t):
    loss = loss_of(net, x, y, t)
    opt.zero_grad()
    loss.backward()


def train(local_rank, world, port, out_dir, backend, device="cpu"):
    from distributed_pytorch_amd import amp, launch
    from distributed_pytorch_amd.ops import functional as F
    from distributed_pytorch_amd.parallel import DistributedDataParallel
    from distributed_pytorch_amd.parallel import process_group as pg

    if device == "cuda":
        import _gpu_dist_workers as G

        G._init(local_rank, world, port, window_mb=8)
        amp.state().reset()
    else:
        launch.init_process_group(backend, "tcp://127.0.0.1:%d" % port, world, local_rank, timeout_s=60, use_gpu=False)
    F._FUSE_RESIDUAL_NORM = True
    kw = dict(device_ids=[0]) if device == "cuda" else {}
    net, opt = model_and_optimizer(lambda m: DistributedDataParallel(m, bucket_cap_mb=0.05, first_bucket_mb=0.01,
                                                                     min_bucket_mb=0.0, **kw), device)
    x, y, t = batch(world)
    mine = slice(local_rank * PER, (local_rank + 1) * PER)
    grads, params = [], []
    for it in range(2):
        one_step(net, opt, *(v[it, mine].to(device) for v in (x, y, t)))
        if device == "cuda":
            torch.cuda.synchronize()
        grads.append({n: p.grad.detach().cpu().clone() for n, p in net.module.named_parameters()})
        opt.step()
        params.append({n: p.detach().cpu().clone() for n, p in net.module.named_parameters()})
    torch.save({"grads": grads, "params": params, "buckets": len(net.arena.buckets)}, os.path.join(out_dir, "rank%d.pt" % local_rank))
    pg.barrier()
    pg.destroy_process_group()


def check(out_dir, world, device="cpu", rel=1e-5):
    """All ranks hold the same bits; against one process on the whole batch the first step's gradients are off by `rel` of their
    norm at most, and a parameter by what its update makes of that: an orthogonalised one enlarges a relative error by at
    most 4 a step (the largest slope of the iteration), 4^5 in all, the others are linear in it."""
    from distributed_pytorch_amd.ops import functional as F

    rs = [torch.load(os.path.join(out_dir, "rank%d.pt" % r), weights_only=True) for r in range(world)]
    assert rs[0]["buckets"] > 1
    for r in rs[1:]:
        for kind in ("grads", "params"):
            for a, b in zip(rs[0][kind], r[kind]):
                for n in a:
                    assert torch.equal(a[n], b[n]), (kind, n)
    was, F._FUSE_RESIDUAL_NORM = F._FUSE_RESIDUAL_NORM, True
    try:
        net, opt = model_and_optimizer(device=device)
        before = {n: p.detach().cpu().clone() for n, p in net.named_parameters()}
        x, y, t = batch(world)
        one_step(net, opt, *(v[0].to(device) for v in (x, y, t)))
        grads = {n: p.grad.detach().cpu().clone() for n, p in net.named_parameters()}
        opt.step()
    finally:
        F._FUSE_RESIDUAL_NORM = was
    matrices = {id(p) for p in opt.param_groups[0]["params"]}
    # (gradients that cancel: those of a key projection's bias are rounding errors of the whole projection's)
    floor = 1e-3 * max(float(g.norm()) / g.numel() ** 0.5 for g in grads.values())
    for n, p in net.named_parameters():
        g, got = grads[n], rs[0]["grads"][0][n]
        size = float(g.norm()) + floor * g.numel() ** 0.5
        off = float((got - g).norm())
        assert off <= rel * size, ("gradient", n, off / size)
        w = before[n]
        if id(p) in matrices:
            rows, cols = w.shape[0], w.numel() // w.shape[0]
            f = 0.05 * 0.2 * max(1.0, rows / cols) ** 0.5
            slack = f * (4.0 ** 5 * off / float(g.norm()) + 1e-3) * 1.3 * min(rows, cols) ** 0.5
            assert float((p.detach().cpu() - w).norm()) > 0.1 * f * min(rows, cols) ** 0.5, n      # (it was orthogonalised)
        else:
            slack = 0.05 * off
        assert float((rs[0]["params"][0][n] - p.detach().cpu()).norm()) <= slack + 2.0 ** -22 * float(w.norm()) + 1e-7, n
