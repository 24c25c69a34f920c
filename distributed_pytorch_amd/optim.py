"""FusedSGD — SGD with momentum / weight decay as ONE multi-tensor HIP launch.

Semantics are those of ``torch.optim.SGD`` as used by the reference
(``nd_imagenet.py:174-176``; dampening 0, no nesterov by default):
``g += wd*p``; first step ``buf = g`` else ``buf = mu*buf + g``; ``p -= lr*buf``.
``state_dict()`` has torch's exact structure (``state[i]['momentum_buffer']``,
``param_groups[...]['params'] = [0..P-1]``) so optimizer state is interchangeable
with reference checkpoints.

GPU path (kernel ``sgd_momentum_multi_tensor``, N-K13/N-K14): one launch walks a
device-resident chunk table over all parameters; it reads the gradient (fp32 or
bf16/fp16) times ``1/loss_scale``, skips the whole update when the loss
scaler's ``found_inf`` flag is set, updates the fp32 master + momentum and writes
the low-precision compute copy used by the next forward.  ``lr`` / ``wd`` /
``momentum`` are read from a device buffer, so a per-iteration LR schedule
(``imagenet_ddp_apex.py:369``) costs no re-capture under hipGraph replay.
"""
from __future__ import annotations

from typing import List, Optional

import torch
from torch.optim import Optimizer

from . import amp as _amp
from .parallel import process_group as _pg


class FusedSGD(Optimizer):
    fused_unscale = True

    def __init__(self, params, lr: float = 0.1, momentum: float = 0.0, dampening: float = 0.0,
                 weight_decay: float = 0.0, nesterov: bool = False):
        if lr < 0.0:
            raise ValueError("Invalid learning rate: {}".format(lr))
        if nesterov and (momentum <= 0 or dampening != 0):
            raise ValueError("Nesterov momentum requires a momentum and zero dampening")
        defaults = dict(lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay,
                        nesterov=nesterov, maximize=False, foreach=None, differentiable=False,
                        fused=None)
        super().__init__(params, defaults)
        self._scaler = None          # armed by amp.scale_loss for the next step
        self._amp_state = None
        self._plan = None            # device chunk table (GPU path)
        self._own_arena = None       # single-GPU gradient arena (a DDP wrapper brings its own)
        self._steps = 0

    # ------------------------------------------------------------------ amp hooks
    def set_amp(self, amp_state) -> None:
        self._amp_state = amp_state
        self._plan = None

    def arm_scaler(self, scaler) -> None:
        self._scaler = scaler

    def rebind(self) -> None:
        """Parameters were re-typed (amp O3): drop cached plans / state."""
        self._plan = None
        self.state.clear()

    # ------------------------------------------------------------------ gradient arenas
    def register_arena(self, arena) -> None:
        """Kept for API symmetry: arenas are discovered through the parameters' sinks."""
        self._plan = None

    def _arenas(self):
        """Gradient arenas behind this optimizer's parameters.  On the GPU every fp32 parameter
        gets one (DDP's buckets, or a private flat arena on a single GPU) so backward kernels write
        gradients in place and the device tensor table never changes."""
        params = [p for g in self.param_groups for p in g["params"] if p.requires_grad]
        if not params:
            return []
        missing = [p for p in params if getattr(p, "_dpa_sink", None) is None]
        if missing and all(p.is_cuda and p.dtype == torch.float32 for p in missing):
            from .parallel.distributed import GradArena

            self._own_arena = GradArena(missing)
            self._plan = None
        seen, out = set(), []
        for p in params:
            s = getattr(p, "_dpa_sink", None)
            if s is not None and s.arena is not None and id(s.arena) not in seen:
                seen.add(id(s.arena))
                out.append(s.arena)
        return out

    # ------------------------------------------------------------------ zero_grad
    def zero_grad(self, set_to_none: Optional[bool] = None) -> None:
        """With a gradient arena nothing is zeroed on the GPU: the first kernel that delivers a
        gradient overwrites its slot (N-K18); CPU arenas (gloo plumbing) get one memset per bucket."""
        arenas = self._arenas()
        if not arenas:
            super().zero_grad(set_to_none=True if set_to_none is None else set_to_none)
            return
        for arena in arenas:
            if arena.params[0].is_cuda and set_to_none is not False:
                arena.begin_step()
                for p in arena.params:
                    p.grad = None
            else:
                arena.zero()
                arena.attach()

    # ------------------------------------------------------------------ step
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        scaler, self._scaler = self._scaler, None
        from .ops import hip_ops as _hip_ops

        _hip_ops.join_side_stream()
        if _pg.is_initialized():
            _pg.check_health()          # a timed-out SyncBN / metric all-reduce must not reach the weights
        for arena in self._arenas():
            arena.finish_step()
        any_cuda = any(p.is_cuda for g in self.param_groups for p in g["params"])
        if any_cuda:
            self._step_hip(scaler)
        else:
            self._step_reference(scaler)
        for arena in self._arenas():
            arena.end_step()
        if scaler is not None:
            scaler.update()
        self._steps += 1
        return loss

    def _momentum_buffer(self, p: torch.Tensor) -> torch.Tensor:
        st = self.state[p]
        buf = st.get("momentum_buffer")
        if buf is None:
            buf = torch.zeros_like(p, dtype=torch.float32 if p.dtype == torch.float32 else p.dtype,
                                   memory_format=torch.preserve_format)
            st["momentum_buffer"] = buf
        return buf

    def sgd_groups(self) -> list:
        """The groups that SGD updates."""
        return self.param_groups

    def _step_reference(self, scaler) -> None:
        skip = scaler is not None and float(scaler.found_inf.item()) > 0
        if skip:
            return
        inv = None if scaler is None else scaler.inv_scale
        for group in self.sgd_groups():
            lr, mu, wd = group["lr"], group["momentum"], group["weight_decay"]
            damp, nesterov = group["dampening"], group["nesterov"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                g = p.grad.to(p.dtype)
                if inv is not None:
                    g = g * inv.to(g.dtype).squeeze(0)
                if wd != 0:
                    g = g.add(p, alpha=wd)
                if mu != 0:
                    first = "momentum_buffer" not in self.state[p] or \
                        self.state[p]["momentum_buffer"] is None
                    buf = self._momentum_buffer(p)
                    if first:
                        buf.copy_(g)
                    else:
                        buf.mul_(mu).add_(g, alpha=1 - damp)
                    g = g.add(buf, alpha=mu) if nesterov else buf
                p.add_(g.to(p.dtype), alpha=-lr)

    def _step_hip(self, scaler) -> None:
        self._prepare_hip()                          # (what it refuses, it refuses before anything is updated)
        self._launch_hip(scaler)

    def _prepare_hip(self) -> None:
        from .ops import hip_ops

        if self._plan is None or not self._plan.matches(self):
            self._plan = hip_ops.SgdPlan(self)

    def _launch_hip(self, scaler) -> None:
        self._plan.launch(self, scaler)
        _amp.mark_copies_written(self._plan.params_with_copies)

    # ------------------------------------------------------------------ hipGraph support (utils/graph.py)
    def sync_hyper(self) -> None:
        if self._plan is not None:
            self._plan.sync_hyper(self)

    def after_graph_replay(self) -> None:
        """A replayed step ran the captured kernels only: advance the host-side bookkeeping."""
        from .ops import hip_ops

        self._steps += 1
        hip_ops.bump_generation()

    # ------------------------------------------------------------------ torch-compatible state
    def state_dict(self):
        sd = super().state_dict()
        if self._steps == 0:
            # torch.optim.SGD has empty state before its first step
            sd["state"] = {k: v for k, v in sd["state"].items()
                           if v.get("momentum_buffer") is not None and self._steps > 0}
        return sd

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        self._plan = None
        self._steps = max(self._steps, 1 if len(self.state) else 0)
        for p, st in self.state.items():
            buf = st.get("momentum_buffer")
            if buf is not None and p.dim() == 4 and not buf.is_contiguous(
                    memory_format=torch.channels_last):
                st["momentum_buffer"] = buf.contiguous(memory_format=torch.channels_last)


def muon_groups(model) -> list:
    """Parameter groups for ``FusedMuon``: the matrices inside the network are orthogonalised (Linear weights,
    attention projections, dense convolution filters as ``[K, C * R * S]``); the first convolution, the classifier,
    embeddings, position bias tables, depthwise filters, biases and norms take plain SGD."""
    from .nn.modules import Conv2d, Linear

    convs = [m for m in model.modules() if isinstance(m, Conv2d)]
    linears = [m for m in model.modules() if isinstance(m, Linear)]
    first = convs[0].weight if convs else None
    last = linears[-1].weight if linears else (convs[-1].weight if convs else None)
    grouped = {id(m.weight) for m in convs if m.groups > 1}
    matrices, rest = [], []
    tables = {id(m.weight) for m in model.modules() if isinstance(m, torch.nn.Embedding)}
    for name, p in model.named_parameters():
        if not p.requires_grad:
            continue
        inside = name.endswith("weight") and p.dim() in (2, 4) and p is not first and p is not last \
            and id(p) not in grouped and id(p) not in tables and min(p.shape[0], p.numel() // p.shape[0]) > 1
        (matrices if inside else rest).append(p)
    return [g for g in (dict(params=matrices, orthogonal=True), dict(params=rest, orthogonal=False)) if g["params"]]


class FusedMuon(FusedSGD):
    """Muon beside ``FusedSGD``: the matrices of groups with ``orthogonal=True`` are updated with the orthogonalised
    momentum, all other parameters by SGD with momentum in the same step.

        ``buf = momentum * buf + g``,  ``u = g + momentum * buf`` (nesterov) or ``buf``
        ``p = p * (1 - lr * weight_decay) - lr * matrix_scale * sqrt(max(1, rows / columns)) * newton_schulz(u)``

    ``g`` is the unscaled gradient; the decay is decoupled (it does not enter the momentum).  A group without
    ``orthogonal`` behaves exactly like one of ``FusedSGD`` (coupled decay, no nesterov).  ``params``: groups as
    ``muon_groups(model)`` makes them, or parameters, of which those of two dimensions are orthogonalised.

    On the GPU a step is two launches over a device-resident table per group plus ``newton_schulz`` once per matrix shape
    (matrices of one shape are a batch); loss scaling, the overflow skip, low-precision copies, gradient arenas and
    hipGraph capture work as in ``FusedSGD``.  ``state_dict`` holds ``momentum_buffer`` per parameter."""

    def __init__(self, params, lr: float = 0.1, momentum: float = 0.95, weight_decay: float = 0.0, nesterov: bool = True,
                 matrix_scale: float = 0.2, ns_steps: int = 5, ns_coefficients=(3.4445, -4.7750, 2.0315),
                 ns_eps: float = 1e-7):
        groups = list(params)
        if groups and not isinstance(groups[0], dict):
            groups = [g for g in (dict(params=[p for p in groups if p.dim() == 2], orthogonal=True),
                                  dict(params=[p for p in groups if p.dim() != 2], orthogonal=False)) if g["params"]]
        self._nesterov = bool(nesterov)              # (add_param_group, which the base constructor calls, reads it)
        super().__init__(groups, lr=lr, momentum=momentum, weight_decay=weight_decay)
        self._matrix_defaults = dict(orthogonal=False, matrix_scale=float(matrix_scale), ns_steps=int(ns_steps),
                                     ns_coefficients=tuple(float(v) for v in ns_coefficients), ns_eps=float(ns_eps))
        self._muon = None
        self._fill_groups()

    def _fill_groups(self) -> None:
        from .ops.functional import _check_schulz

        for group in self.param_groups:
            for k, v in self._matrix_defaults.items():
                group.setdefault(k, v)
            if not 0.0 <= group["momentum"] < 1.0:
                raise ValueError("Invalid momentum: {}".format(group["momentum"]))
            if group["weight_decay"] < 0.0 or group["matrix_scale"] <= 0.0:
                raise ValueError("weight_decay must not be negative and matrix_scale positive")
            if group["ns_steps"] < 1 or not group["ns_eps"] > 0.0:
                raise ValueError("ns_steps must be at least 1 and ns_eps positive")
            _check_schulz(tuple(float(v) for v in group["ns_coefficients"]), int(group["ns_steps"]))
            if group["orthogonal"]:
                if group["dampening"] != 0:
                    raise ValueError("FusedMuon: no dampening in an orthogonal group")
                if any(p.dim() < 2 for p in group["params"]):
                    raise ValueError("FusedMuon: an orthogonal group holds matrices (2 or more dimensions)")

    def add_param_group(self, group) -> None:
        if isinstance(group, dict) and group.get("orthogonal"):
            group.setdefault("nesterov", self._nesterov)
        super().add_param_group(group)
        if hasattr(self, "_matrix_defaults"):        # (the base constructor adds its groups through here)
            self._fill_groups()
            self._plan = self._muon = None

    def sgd_groups(self) -> list:
        return [g for g in self.param_groups if not g["orthogonal"]]

    def _step_reference(self, scaler) -> None:
        from .ops import functional as F

        if scaler is not None and float(scaler.found_inf.item()) > 0:
            return
        super()._step_reference(scaler)
        inv = None if scaler is None else scaler.inv_scale
        for group in self.param_groups:
            if not group["orthogonal"]:
                continue
            lr, mu = group["lr"], group["momentum"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                g = p.grad.to(p.dtype)
                if inv is not None:
                    g = g * inv.to(g.dtype).squeeze(0)
                buf = self._momentum_buffer(p)
                buf.mul_(mu).add_(g)
                u = g.add(buf, alpha=mu) if group["nesterov"] else buf
                rows, cols = p.shape[0], p.numel() // p.shape[0]
                o = F.newton_schulz(u.reshape(rows, cols), group["ns_steps"], group["ns_coefficients"], group["ns_eps"])
                p.mul_(1.0 - lr * group["weight_decay"])
                p.add_(o.reshape(p.shape), alpha=-lr * group["matrix_scale"] * max(1.0, rows / cols) ** 0.5)

    def _prepare_hip(self) -> None:
        from .ops.transformer_ops import MuonPlan

        if self._muon is None or not self._muon.matches(self):
            self._muon = MuonPlan(self)
        super()._prepare_hip()

    def _launch_hip(self, scaler) -> None:
        self._muon.launch(self, scaler)
        super()._launch_hip(scaler)                  # the other groups; then every derived copy is stale ...
        self._muon.stamp_copies()                    # ... but those that this step wrote
        _amp.mark_copies_written([p for gt in self._muon.groups for p, lp in gt["plist"] if lp is not None])

    def set_amp(self, amp_state) -> None:
        super().set_amp(amp_state)
        self._muon = None

    def rebind(self) -> None:
        super().rebind()
        self._muon = None

    def sync_hyper(self) -> None:
        super().sync_hyper()
        if self._muon is not None:
            self._muon.sync_hyper(self)

    def load_state_dict(self, state_dict) -> None:
        own = [{k: g[k] for k in ("nesterov", *self._matrix_defaults)} for g in self.param_groups]
        super().load_state_dict(state_dict)
        for group, saved, mine in zip(self.param_groups, state_dict["param_groups"], own):
            if "orthogonal" not in saved:            # SGD's: it has the momentum, which matrices take as it is, and no say in the rest
                group.update(mine)
        self._muon = None
        self._fill_groups()
