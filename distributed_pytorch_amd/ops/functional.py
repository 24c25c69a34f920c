"""Functional op layer.  Activations are **NHWC** tensors ``[N, H, W, C]``.

Dispatch rule (see ``backend.py``): CPU tensors -> pure PyTorch reference math
(the oracle for every test and the BASELINE "config #1" plumbing backend);
GPU tensors -> hand-written HIP kernels in ``csrc/kernels`` through
``ops/hip_ops.py``.  The op set is the implicit native surface of the reference
scripts: what cuDNN / cuBLAS / ATen / Apex ran for
``model(images)``, ``criterion``, ``loss.backward()`` and ``optimizer.step()``
(reference ``nd_imagenet.py:291-303``, ``imagenet_ddp_apex.py:339-383``).
"""
from __future__ import annotations

import functools
import math
import os
from typing import NamedTuple, Optional, Sequence, Tuple

import torch
import torch.nn.functional as TF
from torch.autograd import forward_ad


def _on_gpu(t: torch.Tensor) -> bool:
    """GPU tensors ALWAYS run the HIP kernels; the PyTorch ops below are the CPU reference backend.  (The stock
    PyTorch-ROCm comparison point lives outside the framework: ``bench/torch_baseline.py``.)"""
    return t.is_cuda


def _hip():
    from . import hip_ops

    return hip_ops


def _tops():
    from . import transformer_ops

    return transformer_ops


def _pair(v) -> Tuple[int, int]:
    return (v, v) if isinstance(v, int) else (int(v[0]), int(v[1]))


# ----------------------------------------------------------------------------- conv
def conv2d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           stride=1, padding=0, *, relu: bool = False, w_lp: Optional[torch.Tensor] = None,
           want_stats: bool = False, needs_input_grad: bool = True, skip: bool = False, groups: int = 1):
    """NHWC convolution.  ``weight`` is logical ``[K, C/groups, R, S]`` (memory KRSC).

    ``w_lp``: optional low-precision compute copy of ``weight`` (AMP O1/O2);
    gradients still flow to ``weight``.  ``want_stats`` additionally returns the
    per-channel ``(sum, sumsq)`` of the output computed in the conv epilogue
    (feeds the fused BatchNorm).  ``needs_input_grad=False`` skips dgrad (stem).
    ``skip=True`` returns ``(result, x_alias)``: feed ``x_alias`` to the residual branch and its
    gradient is added inside this convolution's dgrad epilogue instead of a separate accumulate pass.
    Contract: use ``x_alias`` ONCE -- as the ``residual`` of the block's last BatchNorm, or as the input of the
    block's downsample branch.  (A residual BN + ReLU returns the alias's gradient unmasked together with its ReLU
    bit mask, which only this convolution's epilogue knows how to apply.)
    ``groups > 1``: grouped / depthwise convolution, every pass one launch with the group on ``grid.y``.
    """
    stride, padding = _pair(stride), _pair(padding)
    if getattr(x, "_dpa_s2d", False):       # space-to-depth image (to_s2d): the 7x7 stride-2 stem as a 4x4 convolution
        if groups != 1 or skip or not _on_gpu(x):
            raise ValueError("space-to-depth input is only valid for a dense GPU stem convolution")
        return _hip().stem_s2d_conv(x, weight, bias, stride, padding, relu, want_stats)
    if groups > 1:
        if _on_gpu(x):
            out = _hip().group_conv2d(x, weight, bias, stride, padding, groups, relu, want_stats, needs_input_grad)
        else:
            w = weight if w_lp is None else _StraightThroughCast.apply(weight, x.dtype)
            if w.dtype != x.dtype:
                w = w.to(x.dtype)
            b = None if bias is None else bias.to(x.dtype)
            y = TF.conv2d(x.permute(0, 3, 1, 2), w, b, stride, padding, 1, groups).permute(0, 2, 3, 1)
            y = (TF.relu(y) if relu else y).contiguous()
            out = (y, None) if want_stats else y
        return (out, x) if skip else out
    if _on_gpu(x):
        return _hip().conv2d(x, weight, bias, stride, padding, relu, w_lp, want_stats,
                             needs_input_grad, skip)
    w = weight if w_lp is None else _StraightThroughCast.apply(weight, x.dtype)
    if w.dtype != x.dtype:
        w = w.to(x.dtype)
    b = None if bias is None else bias.to(x.dtype)
    y = TF.conv2d(x.permute(0, 3, 1, 2), w, b, stride, padding).permute(0, 2, 3, 1)
    if relu:
        y = TF.relu(y)
    y = y.contiguous()
    out = (y, None) if want_stats else y
    return (out, x) if skip else out


class _StraightThroughCast(torch.autograd.Function):
    """fp32 master -> low precision for compute; gradient returns in fp32."""

    @staticmethod
    def forward(ctx, w, dtype):
        return w.to(dtype)

    @staticmethod
    def backward(ctx, g):
        return g.float(), None


# ----------------------------------------------------------------------------- batch norm
def batch_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor,
               running_mean: Optional[torch.Tensor], running_var: Optional[torch.Tensor],
               num_batches_tracked: Optional[torch.Tensor], training: bool,
               momentum: float = 0.1, eps: float = 1e-5, *, relu: bool = False,
               residual: Optional[torch.Tensor] = None, stats=None, group=None, defer: bool = False) -> torch.Tensor:
    """Fused ``BN [+ residual] [+ ReLU]`` over NHWC (N-K4/K5/K7; SyncBN when
    ``group`` is a process group: N-K6).  Statistics are always fp32.
    ``running_var`` receives the unbiased variance, as in torch / cuDNN.
    ``relu=6`` applies ReLU6 (MobileNet) inside the same pass; ``relu="silu"`` / ``"hardswish"`` / ... a smooth
    activation (EfficientNet, MobileNetV3): the GPU training path applies it inside the normalise pass and folds its
    slope into the BN backward kernels, so no separate activation pass runs in either direction.
    ``defer=True`` (activation-free BN of a downsample branch): on the GPU in training mode nothing is written --
    the result aliases ``x`` and MUST only be used as the ``residual`` of another ``batch_norm``, which applies this
    BN's scale / shift on the fly (one activation-sized write and read less).  Ignored elsewhere.
    """
    if _on_gpu(x):
        return _hip().batch_norm(x, weight, bias, running_mean, running_var, num_batches_tracked,
                                 training, momentum, eps, relu, residual, stats, group, defer)
    if group is not None and training:
        from ..parallel.sync_batchnorm import sync_batch_norm_reference

        y = sync_batch_norm_reference(x, weight, bias, running_mean, running_var,
                                      num_batches_tracked, momentum, eps, group)
    else:
        xc = x.permute(0, 3, 1, 2)
        if training and num_batches_tracked is not None:
            num_batches_tracked.add_(1)
        y = TF.batch_norm(xc.float(), running_mean, running_var, weight.float(), bias.float(),
                          training, momentum, eps).to(x.dtype).permute(0, 2, 3, 1)
    if residual is not None:
        y = y + residual
    if isinstance(relu, str):
        y = _CPU_ACTS[relu](y)
    elif relu:
        y = TF.relu6(y) if (relu is not True and relu == 6) else TF.relu(y)
    return y.contiguous()


def bn_relu_max_pool2d(x, weight, bias, running_mean, running_var, num_batches_tracked, training, momentum, eps,
                       kernel_size, stride=None, padding=0, ceil_mode: bool = False, *, stats=None, group=None):
    """``max_pool2d(relu(batch_norm(x)))`` -- the stem of ResNet / DenseNet / GoogLeNet.  On the GPU in training mode
    (no SyncBN) this is the fused stem path: the normalised full-resolution tensor is never materialised."""
    k, s, p = _pair(kernel_size), _pair(stride if stride is not None else kernel_size), _pair(padding)
    if _on_gpu(x) and training and group is None and _hip().can_fuse_bn_relu_maxpool(x):
        return _hip().bn_relu_maxpool(x, weight, bias, running_mean, running_var, num_batches_tracked, momentum, eps,
                                      stats, k, s, p, ceil_mode)
    y = batch_norm(x, weight, bias, running_mean, running_var, num_batches_tracked, training, momentum, eps,
                   relu=True, stats=stats, group=group)
    return max_pool2d(y, k, s, p, ceil_mode)


# ----------------------------------------------------------------------------- pooling
def max_pool2d(x: torch.Tensor, kernel_size, stride=None, padding=0, ceil_mode: bool = False) -> torch.Tensor:
    k, s, p = _pair(kernel_size), _pair(stride if stride is not None else kernel_size), _pair(padding)
    if _on_gpu(x):
        return _hip().max_pool2d(x, k, s, p, ceil_mode)
    return TF.max_pool2d(x.permute(0, 3, 1, 2), k, s, p, ceil_mode=ceil_mode).permute(0, 2, 3, 1).contiguous()


def avg_pool2d(x: torch.Tensor, kernel_size, stride=None, padding=0) -> torch.Tensor:
    """Average pooling (floor mode, padding counted in the divisor like torch's default).  Non-overlapping windows
    that tile the input (DenseNet transitions: 2x2 stride 2) run on the adaptive average-pool kernel; everything
    else (Inception's 3x3 stride-1 pad-1 branch pool, its 5x5 stride-3 auxiliary pool) on the fixed-window kernel."""
    k, s, p = _pair(kernel_size), _pair(stride if stride is not None else kernel_size), _pair(padding)
    if k == s and p == (0, 0) and x.shape[1] % k[0] == 0 and x.shape[2] % k[1] == 0:
        return adaptive_avg_pool2d(x, (x.shape[1] // k[0], x.shape[2] // k[1]))
    if _on_gpu(x):
        return _hip().avg_pool2d_window(x, k, s, p)
    return TF.avg_pool2d(x.permute(0, 3, 1, 2), k, s, p).permute(0, 2, 3, 1).contiguous()


def cat_channels(xs) -> torch.Tensor:
    """Concatenate NHWC tensors along the channel axis."""
    xs = list(xs)
    if len(xs) == 1:
        return xs[0]
    if _on_gpu(xs[0]):
        return _hip().cat_channels(xs)
    return torch.cat(xs, dim=-1)


def attention(qkv: torch.Tensor, num_heads: int, scale, rel_bias: Optional[torch.Tensor] = None,
              mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Multi-head self-attention on the packed projection: ``qkv`` is ``[B, S, 3 * H * D]`` laid out ``[3][H][D]`` per
    token (what ``nn.MultiheadAttention``'s in-projection, Swin's and MaxViT's ``qkv`` Linear produce), the result
    ``[B, S, H * D]`` feeds the output projection.

        softmax(scale * q k^T + rel_bias[h] + mask[b % nW]) v

    ``scale``: a float or a per-head tensor ``[H]`` (not differentiated here).  ``rel_bias``: optional learnable
    ``[H, S, S]`` (Swin / MaxViT relative position bias; gets a gradient).  ``mask``: optional constant ``[nW, S, S]``
    (Swin's shifted-window mask), batch entry ``b`` uses window ``b % nW``.  On the GPU this is one fused MFMA kernel
    per direction (``csrc/kernels/attention.hip``): the scores never reach memory."""
    if _on_gpu(qkv):
        return _hip().attention(qkv, num_heads, scale, rel_bias, mask)
    B, S, W3 = qkv.shape
    H = num_heads
    D = W3 // (3 * H)
    q, k, v = qkv.reshape(B, S, 3, H, D).permute(2, 0, 3, 1, 4).float().unbind(0)      # [B, H, S, D]
    sc = scale.float().reshape(1, H, 1, 1) if isinstance(scale, torch.Tensor) else float(scale)
    att = (q @ k.transpose(-1, -2)) * sc
    if rel_bias is not None:
        att = att + rel_bias.float().reshape(1, H, S, S)
    if mask is not None:
        nW = mask.shape[0]
        att = (att.reshape(B // nW, nW, H, S, S) + mask.float().reshape(1, nW, 1, S, S)).reshape(B, H, S, S)
    out = att.softmax(-1) @ v
    return out.transpose(1, 2).reshape(B, S, H * D).to(qkv.dtype)


def window_geometry(B: int, H: int, W: int, wh: int, ww: int, sh: int = 0, sw: int = 0, grid: bool = False):
    """Geometry tuple of ``window_partition``: ``(B, H, W, wh, ww, nh, nw, sh, sw, grid)``.  Window mode: windows of
    ``wh x ww`` tokens over the image zero-padded to a multiple of the window, after a cyclic shift by ``(sh, sw)``
    (Swin).  Grid mode (MaxViT): ``wh x ww`` is the GRID size, token ``(i, j)`` of window ``(gh, gw)`` is pixel
    ``(i * nh + gh, j * nw + gw)``; the image must divide evenly."""
    if grid:
        if H % wh or W % ww:
            raise ValueError("grid partition needs H, W divisible by the grid size")
        return (B, H, W, wh, ww, H // wh, W // ww, 0, 0, True)
    return (B, H, W, wh, ww, -(-H // wh), -(-W // ww), sh, sw, False)


def window_partition(x: torch.Tensor, geom) -> torch.Tensor:
    """``[B, H, W, C] -> [B * nh * nw, wh * ww, C]`` (shift + pad + partition in one gather on the GPU)."""
    if _on_gpu(x):
        return _hip().window_partition(x, geom, False)
    B, H, W, wh, ww, nh, nw, sh, sw, grid = geom
    C = x.shape[-1]
    if grid:
        return x.reshape(B, wh, nh, ww, nw, C).permute(0, 2, 4, 1, 3, 5).reshape(B * nh * nw, wh * ww, C)
    x = TF.pad(x, (0, 0, 0, nw * ww - W, 0, nh * wh - H))
    if sh or sw:
        x = torch.roll(x, shifts=(-sh, -sw), dims=(1, 2))
    return x.reshape(B, nh, wh, nw, ww, C).permute(0, 1, 3, 2, 4, 5).reshape(B * nh * nw, wh * ww, C)


def window_reverse(win: torch.Tensor, geom) -> torch.Tensor:
    """Inverse of ``window_partition`` (the zero padding is dropped)."""
    if _on_gpu(win):
        return _hip().window_partition(win, geom, True)
    B, H, W, wh, ww, nh, nw, sh, sw, grid = geom
    C = win.shape[-1]
    if grid:
        return win.reshape(B, nh, nw, wh, ww, C).permute(0, 3, 1, 4, 2, 5).reshape(B, H, W, C)
    x = win.reshape(B, nh, nw, wh, ww, C).permute(0, 1, 3, 2, 4, 5).reshape(B, nh * wh, nw * ww, C)
    if sh or sw:
        x = torch.roll(x, shifts=(sh, sw), dims=(1, 2))
    return x[:, :H, :W, :].contiguous()


def qk_normalize(qkv: torch.Tensor, mult: torch.Tensor, num_heads: int) -> torch.Tensor:
    """Swin V2 cosine attention pre-pass on the packed ``[.., 3 * H * D]`` projection: ``q <- mult[h] * q / |q|``,
    ``k <- k / |k|`` (``F.normalize`` semantics, eps 1e-12), ``v`` unchanged.  Differentiable in ``qkv`` and ``mult``."""
    if _on_gpu(qkv):
        return _hip().qk_normalize(qkv, mult, num_heads)
    shp = qkv.shape
    H = num_heads
    D = shp[-1] // (3 * H)
    x = qkv.reshape(-1, 3, H, D).float()
    q = TF.normalize(x[:, 0], dim=-1) * mult.float().reshape(1, H, 1)
    k = TF.normalize(x[:, 1], dim=-1)
    return torch.stack([q, k, x[:, 2]], dim=1).reshape(shp).to(qkv.dtype)


def shuffle_pair(a: torch.Tensor, b: torch.Tensor, bf: int):
    """ShuffleNetV2's ``channel_shuffle(cat(a, b), groups=2)`` followed by the ``chunk(2)`` of the next block, as one op:
    returns the two halves.  ``a`` / ``b`` hold ``bf`` real channels (+ zero padding up to their width on the GPU)."""
    if _on_gpu(a):
        return _hip().shuffle_pair(a, b, bf)
    out = torch.stack([a[..., :bf], b[..., :bf]], dim=-1).flatten(-2)        # out[2i] = a[i], out[2i+1] = b[i]
    lo, ro = out[..., :bf], out[..., bf:]
    pad = a.shape[-1] - bf
    if pad:
        lo, ro = TF.pad(lo, (0, pad)), TF.pad(ro, (0, pad))
    return lo.contiguous(), ro.contiguous()


def adaptive_avg_pool2d(x: torch.Tensor, output_size) -> torch.Tensor:
    o = _pair(output_size)
    if _on_gpu(x):
        return _hip().adaptive_avg_pool2d(x, o)
    return TF.adaptive_avg_pool2d(x.permute(0, 3, 1, 2), o).permute(0, 2, 3, 1).contiguous()


def relu(x: torch.Tensor) -> torch.Tensor:
    if _on_gpu(x):
        return _hip().relu(x)
    return TF.relu(x)


def add_relu(x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """Residual ``relu(x + y)`` (N-K17) when it is not fused into BatchNorm."""
    if _on_gpu(x):
        return _hip().add_relu(x, y)
    return TF.relu(x + y)


def add(x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """Residual ``x + y`` without activation (EfficientNet / MobileNetV3 under stochastic depth)."""
    if _on_gpu(x):
        return _hip().add(x, y)
    return x + y


_CPU_ACTS = {"sigmoid": torch.sigmoid, "silu": TF.silu, "hardsigmoid": TF.hardsigmoid, "hardswish": TF.hardswish,
             "gelu": TF.gelu}


def activation(x: torch.Tensor, kind: str) -> torch.Tensor:
    """``sigmoid`` / ``silu`` / ``hardsigmoid`` / ``hardswish`` / ``gelu`` (erf form): EfficientNet, MobileNetV3,
    squeeze-excitation, ConvNeXt."""
    if kind not in _CPU_ACTS:
        raise ValueError("unknown activation %r" % (kind,))
    if _on_gpu(x):
        return _hip().activation(x, kind)
    return _CPU_ACTS[kind](x)


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """LayerNorm over the last (channel) axis -- in NHWC torchvision's ``LayerNorm2d`` and ``nn.LayerNorm`` coincide."""
    if _on_gpu(x):
        return _hip().layer_norm(x, weight, bias, eps)
    return TF.layer_norm(x.float(), (x.shape[-1],), weight.float(), bias.float(), eps).to(x.dtype)


class Norm(NamedTuple):
    """A norm over the last axis as ``residual_norm`` takes it: ``kind`` "layer" (``weight``, ``bias`` or None) or "rms"
    (``weight``).  ``nn.LayerNorm`` and ``nn.RMSNorm`` modules give theirs with ``.spec()``."""
    weight: torch.Tensor
    bias: Optional[torch.Tensor] = None
    eps: float = 1e-5
    kind: str = "layer"


def _check_norm(name: str, norm: Norm, x: torch.Tensor) -> None:
    C = x.shape[-1]
    if norm.kind not in ("layer", "rms"):
        raise ValueError("%s: unknown kind %r" % (name, norm.kind))
    if norm.weight.shape != (C,) or (norm.bias is not None and norm.bias.shape != (C,)):
        raise ValueError("%s: weight / bias must be [C]" % name)
    if norm.kind == "rms" and norm.bias is not None:
        raise ValueError("%s: an RMSNorm has no bias" % name)
    if not norm.eps >= 0.0:
        raise ValueError("%s: eps must not be negative" % name)
    if any(t is not None and t.device != x.device for t in norm[:2]):
        raise ValueError("%s: weight / bias must be on the input's device" % name)


_NORM_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check_rows(name: str, x: torch.Tensor) -> None:
    if x.dtype not in _NORM_DTYPES:
        raise TypeError("%s: float32, bfloat16 or float16 expected, got %s" % (name, x.dtype))
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("%s: rows of at least one channel expected" % name)
    most = 2048 * 16 // x.element_size()
    if x.shape[-1] > most:
        raise ValueError("%s: at most %d channels in %s" % (name, most, x.dtype))


def _never_on_gpu(name: str, x: torch.Tensor) -> None:
    if _on_gpu(x):
        raise RuntimeError("%s: arguments that the kernels do not take" % name)


def _norm_reference(v: torch.Tensor, norm: Norm) -> torch.Tensor:
    if norm.kind == "layer":
        return TF.layer_norm(v, (v.shape[-1],), norm.weight.float(), None if norm.bias is None else norm.bias.float(), norm.eps)
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + norm.eps) * norm.weight.float()


def residual_norm(x: torch.Tensor, y: torch.Tensor, *, post: Optional[Norm] = None, gate: Optional[torch.Tensor] = None,
                  scale: Optional[torch.Tensor] = None, pre: Optional[Norm] = None):
    """The residual sum of a transformer block with the norms around it:

        ``s = x + scale[n] * gate * post(y)``,   ``h = pre(s)``

    ``x`` (the residual stream) and ``y`` (the block's output) are ``[N, ..., C]`` of one shape and type.  ``post``: the
    norm behind the block (Swin V2), ``pre``: the norm in front of the next one (ViT, Swin); each a ``Norm`` or None.
    ``gate``: learnable, ``[C]`` (layer scale) or ``[N, C]`` (a conditioned block).  ``scale``: ``[N]``, a constant for
    each sample (stochastic depth: 0 or 1 / keep; a dropped sample's branch still has to be finite).  Returns ``s``, or
    ``(s, h)`` with ``pre``.  Everything between the inputs and the results is 32-bit arithmetic, rounded once: ``h`` is
    the norm of the unrounded sum.  On the GPU one pass per direction (``csrc/transformer/residual_norm*.hip``), any ``C`` up
    to 16384 (16-bit types; 8192 in float32)."""
    if _on_gpu(x):
        out = _tops().residual_norm(x, y, post, gate, scale, pre)
        if out is not None:
            return out                              # (what it does not take is named here)
    _check_rows("residual_norm", x)
    if x.dim() < 2 or y.shape != x.shape or y.dtype != x.dtype or y.device != x.device:
        raise ValueError("residual_norm: x and y must be [N, ..., C] of the same shape, dtype and device")
    if post is not None:
        _check_norm("residual_norm: post", post, x)
    if pre is not None:
        _check_norm("residual_norm: pre", pre, x)
    N, C = x.shape[0], x.shape[-1]
    if gate is not None and (tuple(gate.shape) not in ((C,), (N, C)) or gate.device != x.device):
        raise ValueError("residual_norm: gate must be [C] or [N, C] on the input's device")
    if scale is not None:
        if tuple(scale.shape) != (N,) or scale.device != x.device:
            raise ValueError("residual_norm: scale must be [N] on the input's device")
        if scale.requires_grad:
            raise ValueError("residual_norm: scale is a constant (use a gate for a learnable factor)")
    _never_on_gpu("residual_norm", x)
    z = y.float()
    if post is not None:
        z = _norm_reference(z, post)
    if gate is not None:
        z = z * (gate.float() if gate.dim() == 1 else gate.float().reshape((N,) + (1,) * (x.dim() - 2) + (C,)))
    if scale is not None:
        z = z * scale.float().reshape((N,) + (1,) * (x.dim() - 1))
    s = x.float() + z
    if pre is None:
        return s.to(x.dtype)
    return s.to(x.dtype), _norm_reference(s, pre).to(x.dtype)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """RMSNorm over the last axis: ``x / sqrt(mean(x^2) + eps) * weight``."""
    if _on_gpu(x):
        out = _tops().rms_norm(x, weight, eps)
        if out is not None:
            return out
    _check_rows("rms_norm", x)
    norm = Norm(weight, None, eps, "rms")
    _check_norm("rms_norm", norm, x)
    _never_on_gpu("rms_norm", x)
    return _norm_reference(x.float(), norm).to(x.dtype)


def rotary(qkv: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, axis: torch.Tensor, num_heads: int, *,
           interleaved: bool = False, inplace: bool = False) -> torch.Tensor:
    """Rotary positions of several axes (row and column of an image patch; time, row and column of a video's) on the
    packed projection that ``attention`` takes: ``qkv`` is ``[B, S, 3 * H * D]``, laid out ``[3][H][D]`` per token.  Pair
    ``j`` of every query and key head is turned by the angle ``positions[..., axis[j]] * freqs[j]``; the values are
    unchanged.  Pairs are ``(j, j + P)``, or ``(2j, 2j + 1)`` with ``interleaved``; what lies behind the ``P`` pairs of a
    head stays as it is.  ``positions``: ``[S, A]`` or ``[B, S, A]``, whole numbers or floats; ``freqs``: ``[P]`` float32
    or float64; ``axis``: ``[P]`` whole numbers in ``[0, A)`` (an entry outside turns its pair into NaN).  Angles are
    formed in 64 bits.  ``inplace`` (without gradients) overwrites ``qkv``.  ``nn.AxialRotary`` holds ``freqs`` and
    ``axis`` for the usual splits of a head."""
    if not inplace and _on_gpu(qkv):
        out = _tops().rotary(qkv, positions, freqs, axis, num_heads, interleaved, False)
        if out is not None:
            return out
    if qkv.dtype not in _NORM_DTYPES:
        raise TypeError("rotary: float32, bfloat16 or float16 expected, got %s" % (qkv.dtype,))
    if qkv.dim() != 3 or num_heads < 1 or qkv.shape[-1] % (3 * num_heads) or qkv.shape[-1] == 0:
        raise ValueError("rotary: qkv must be [B, S, 3 * heads * D]")
    B, S, D = qkv.shape[0], qkv.shape[1], qkv.shape[-1] // (3 * num_heads)
    if positions.dim() not in (2, 3) or tuple(positions.shape[:-1]) != ((S,) if positions.dim() == 2 else (B, S)) \
            or positions.shape[-1] < 1:
        raise ValueError("rotary: positions must be [S, A] or [B, S, A]")
    if positions.dtype not in (torch.int64, torch.int32, torch.float32, torch.float64):
        raise TypeError("rotary: positions must be int64, int32, float32 or float64, got %s" % (positions.dtype,))
    if freqs.dtype not in (torch.float32, torch.float64):
        raise TypeError("rotary: freqs must be float32 or float64, got %s" % (freqs.dtype,))
    if axis.dtype not in (torch.int32, torch.int64):
        raise TypeError("rotary: axis must be int32 or int64, got %s" % (axis.dtype,))
    if freqs.dim() != 1 or axis.shape != freqs.shape or 2 * freqs.numel() > D or freqs.numel() > 4096:
        raise ValueError("rotary: freqs and axis must be [P] with 2 P <= D (and P <= 4096)")
    if any(t.device != qkv.device for t in (positions, freqs, axis)):
        raise ValueError("rotary: positions, freqs and axis must be on the input's device")
    if positions.requires_grad or freqs.requires_grad:
        raise ValueError("rotary: positions and freqs are constants")
    if inplace:
        if torch.is_grad_enabled() and qkv.requires_grad:
            raise ValueError("rotary: inplace is for calls without gradients")
        # tokens of one after the other of the two axes, the outer one clear of all that the inner one covers
        reach, ok = qkv.shape[-1], qkv.stride(-1) == 1 or qkv.shape[-1] == 1
        for stride, size in sorted((qkv.stride(d), qkv.shape[d]) for d in (0, 1) if qkv.shape[d] > 1):
            ok, reach = ok and stride >= reach, stride * size
        if not ok:
            raise ValueError("rotary: inplace needs tokens that are dense and do not overlap")
    if inplace and _on_gpu(qkv):
        return _tops().rotary(qkv, positions, freqs, axis, num_heads, interleaved, True)
    _never_on_gpu("rotary", qkv)
    P = freqs.numel()
    ok = (axis >= 0) & (axis < positions.shape[-1])
    angle = positions.double()[..., axis.long().clamp(0, positions.shape[-1] - 1)] * freqs.double()
    angle = torch.where(ok, angle, math.nan)
    angle = angle.reshape((B if positions.dim() == 3 else 1, S, 1, 1, P))
    cos, sin = angle.cos().float(), angle.sin().float()
    v = qkv.reshape(B, S, 3, num_heads, D)
    qk = v[:, :, :2].float()
    a, b = (qk[..., 0:2 * P:2], qk[..., 1:2 * P:2]) if interleaved else (qk[..., :P], qk[..., P:2 * P])
    first, second = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([first, second], -1).flatten(-2) if interleaved else torch.cat([first, second], -1)
    out = torch.cat([torch.cat([turned, qk[..., 2 * P:]], -1).to(qkv.dtype), v[:, :, 2:]], 2).reshape(qkv.shape)
    return qkv.copy_(out) if inplace else out


def se_scale(x: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """``x[n, h, w, c] * s[n, c]``: the squeeze-excitation gate.  ``s`` is fp32 ``[N, C]``."""
    if _on_gpu(x):
        return _hip().se_scale(x, s)
    return x * s.to(x.dtype).view(s.shape[0], 1, 1, s.shape[1])


def se_fused() -> bool:
    return _hip()._SE_FUSED


def se_block(x, w1, b1, w2, b2, act: str, gate: str) -> torch.Tensor:
    """GPU only: the whole squeeze-excitation block as one autograd node (see ``hip_ops._SEBlockFn``); ``w1`` / ``w2``
    are the 1x1-conv shaped parameters of ``nn.SqueezeExcitation``."""
    return _hip().se_block(x, w1, b1, w2, b2, act, gate)


def stochastic_depth(x: torch.Tensor, p: float, training: bool) -> torch.Tensor:
    """torchvision ``StochasticDepth(p, "row")``: drops the whole residual branch of a sample with probability
    ``p`` and rescales the survivors by ``1 / (1 - p)``."""
    noise = stochastic_depth_scale(x, p, training)
    if noise is None:
        return x
    if _on_gpu(x):
        return _hip().se_scale(x, noise.view(-1, 1).expand(x.shape[0], x.shape[-1]))
    return x * noise.to(x.dtype).view(-1, 1, 1, 1)


def stochastic_depth_scale(x: torch.Tensor, p: float, training: bool) -> Optional[torch.Tensor]:
    """The factor of every sample under stochastic depth, ``[N]`` of 0 or ``1 / (1 - p)`` -- ``residual_norm``'s ``scale``;
    None where nothing is dropped.  The same random numbers as ``stochastic_depth`` draws."""
    if not training or p == 0.0:
        return None
    keep = 1.0 - p
    noise = torch.empty((x.shape[0], 1), dtype=torch.float32, device=x.device).bernoulli_(keep)
    if keep > 0.0:
        noise.div_(keep)
    return noise.view(-1)


# DPA_FUSE_RESIDUAL_NORM=1: ViT, Swin, Swin V2 and ConvNeXt blocks run their residual sums with the norms, layer scales and
# stochastic depth around them as residual_norm calls.  Off by default: a norm then sees the unrounded sum, so results
# differ from the separate passes by the rounding of the residual stream.
_FUSE_RESIDUAL_NORM = os.environ.get("DPA_FUSE_RESIDUAL_NORM", "0") == "1"


def fuse_residual_norm() -> bool:
    return _FUSE_RESIDUAL_NORM


def dropout(x: torch.Tensor, p: float, training: bool) -> torch.Tensor:
    if not training or p == 0.0:
        return x
    if _on_gpu(x):
        return _hip().dropout(x, p)
    return TF.dropout(x, p, True)


# ----------------------------------------------------------------------------- linear
def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
           relu: bool = False, w_lp: Optional[torch.Tensor] = None,
           out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``y = x @ weight.T + bias`` (N-K10), optional fused ReLU epilogue."""
    if _on_gpu(x):
        return _hip().linear(x, weight, bias, relu, w_lp, out_dtype)
    w = weight if w_lp is None else _StraightThroughCast.apply(weight, x.dtype)
    if w.dtype != x.dtype:
        w = w.to(x.dtype)
    y = TF.linear(x, w, None if bias is None else bias.to(x.dtype))
    if relu:
        y = TF.relu(y)
    if out_dtype is not None:
        y = y.to(out_dtype)
    return y


# ----------------------------------------------------------------------------- loss / metrics
def cross_entropy(logits: torch.Tensor, target: torch.Tensor, loss_scale=None) -> torch.Tensor:
    """Mean softmax cross-entropy (N-K11).  fp32 math regardless of input dtype."""
    if _on_gpu(logits):
        return _hip().cross_entropy(logits, target)
    return TF.cross_entropy(logits.float(), target)


def topk_correct(output: torch.Tensor, target: torch.Tensor, topk: Sequence[int] = (1, 5)) -> torch.Tensor:
    """Number of rows whose target is within the top-k, float32 ``[len(topk)]`` (N-K12)."""
    if _on_gpu(output):
        return _hip().topk_correct(output, target, tuple(topk))
    z = output.float()
    zt = z.gather(1, target.view(-1, 1))
    rank = (z > zt).sum(dim=1)
    return torch.stack([(rank < k).sum().float() for k in topk])


def loss_and_metrics(logits: torch.Tensor, target: torch.Tensor):
    """-> (mean loss with grad, float32[4] record = loss*n, correct@1, correct@5, n)."""
    if _on_gpu(logits):
        return _hip().loss_and_metrics(logits, target)
    loss = cross_entropy(logits, target)
    with torch.no_grad():
        n = float(target.numel())
        k5 = min(5, logits.shape[1])
        c = topk_correct(logits, target, (1, k5))
        rec = torch.stack([loss.detach().float() * n, c[0], c[1],
                           torch.tensor(n, device=logits.device)])
    return loss, rec


def token_logprobs(logits: torch.Tensor, target: torch.Tensor, k: int = 0):
    """-> ``(logprob, entropy, top_logprob, top_index)`` of every row of ``logits`` ``[..., V]``: the log probability of
    ``target`` ``[...]`` under the row's softmax, the entropy of that softmax, and its ``k`` most probable classes
    ``[..., k]`` in descending order (``k <= 64``; ties go to the lowest index).  float32 (indices int64) whatever the
    logits' type; the first three carry gradients.

    A logit of -inf (a masked class) has probability zero and adds nothing.  A row that is masked altogether has entropy
    0, log probabilities -inf and no gradient.  A ``target`` outside ``[0, V)`` is ignored: its log probability is 0 and
    carries no gradient, the row's other results are as usual.  A row with a NaN or a +inf gives NaN."""
    if _on_gpu(logits):
        out = _tops().token_logprobs(logits, target, k)
        if out is not None:
            return out                              # [N, V]
    if logits.dtype not in _NORM_DTYPES:
        raise TypeError("token_logprobs: float32, bfloat16 or float16 expected, got %s" % (logits.dtype,))
    if logits.dim() < 1 or logits.shape[-1] < 1 or logits.shape[:-1] != target.shape:
        raise ValueError("token_logprobs: logits [..., V] and target [...] expected")
    if target.dtype not in (torch.int64, torch.int32, torch.int16, torch.uint8):
        raise TypeError("token_logprobs: target must hold whole numbers, got %s" % (target.dtype,))
    if target.device != logits.device:
        raise ValueError("token_logprobs: target must be on the logits' device")
    V = logits.shape[-1]
    if V > 1 << 30:
        raise ValueError("token_logprobs: at most 2^30 classes")
    if not 0 <= k <= min(64, V):
        raise ValueError("token_logprobs: k must be 0 .. min(64, V), got %r" % (k,))
    lead = target.shape
    z, t = logits.reshape(-1, V) if logits.dim() != 2 else logits, target.reshape(-1)
    if _on_gpu(z):
        lp, ent, top, idx = _tops().token_logprobs(z, t, int(k))
    else:
        zf, t = z.float(), t.long()
        empty = (zf == -math.inf).all(1)
        zs = torch.where(empty[:, None], 0.0, zf)                 # such a row is answered apart, without a gradient
        m = zs.detach().amax(1, keepdim=True)
        logp = (zs - m) - (zs - m).exp().sum(1, keepdim=True).log()
        valid = (t >= 0) & (t < V)
        lp = torch.where(valid, logp.gather(1, t.clamp(0, V - 1)[:, None])[:, 0], 0.0)
        lp = torch.where(empty & valid, -math.inf, lp)
        ent = -(logp.exp() * torch.where(logp == -math.inf, 0.0, logp)).sum(1)
        ent = torch.where(empty, 0.0, ent)
        idx = torch.sort(zf.detach(), dim=1, descending=True, stable=True).indices[:, :k]
        top = torch.where(empty[:, None], -math.inf, logp.gather(1, idx))
    return lp.reshape(lead), ent.reshape(lead), top.reshape(lead + (k,)), idx.reshape(lead + (k,))


def newton_schulz(g: torch.Tensor, steps: int = 5, coefficients=(3.4445, -4.7750, 2.0315), eps: float = 1e-7, *,
                  fast: bool = False) -> torch.Tensor:
    """Orthogonalises the last two axes of ``g`` (``[..., m, n]``) approximately, as ``optim.FusedMuon`` does with its
    updates: ``X = g / (|g|_F + eps)``, then ``steps`` times ``X <- a X + (b A + c A A) X`` with ``A = X X^T`` (on the
    transposed matrix where ``m > n``).  With the default ``coefficients`` ``(a, b, c)`` five steps move the singular
    values into about [0.7, 1.2].  Products have about 22 significant bits and are summed in 32, whatever ``g``'s type; the
    result is rounded to that type once.  No gradient.  A matrix with an infinity or a NaN gives NaN.  The GPU takes up to
    65535 matrices a call.

    ``fast``, for bfloat16 alone: the GPU's products take operands of 11 significant bits, at a third of the matrix work.  The
    result is then off by 2e-4 to 7e-4 of its norm before it is rounded to bfloat16 (1.7e-3), 2e-3 where a few directions
    are 100 times the rest.

    The GPU holds matrices as fp16 pairs, so the singular values may not grow: coefficients that move any value of
    [0, 1] beyond 4 within ``steps`` steps are refused."""
    if g.dtype not in _NORM_DTYPES:
        raise TypeError("newton_schulz: float32, bfloat16 or float16 expected, got %s" % (g.dtype,))
    if g.dim() < 2 or g.numel() == 0:
        raise ValueError("newton_schulz: matrices [..., m, n] expected")
    if steps < 1 or not eps > 0.0:
        raise ValueError("newton_schulz: steps must be at least 1 and eps positive")
    if fast and g.dtype != torch.bfloat16:
        raise ValueError("newton_schulz: fast products are for bfloat16, got %s" % (g.dtype,))
    _check_schulz(tuple(float(v) for v in coefficients), int(steps))
    if torch.is_grad_enabled() and g.requires_grad:
        raise ValueError("newton_schulz: has no gradient (detach the update)")
    if forward_ad.unpack_dual(g).tangent is not None:
        raise ValueError("newton_schulz: has no gradient, forward-mode either (detach the update)")
    if _on_gpu(g):
        return _tops().newton_schulz(g, steps, coefficients, eps, bool(fast))
    a, b, c = coefficients
    x = g.float()
    turned = x.shape[-2] > x.shape[-1]
    x = x / (torch.linalg.vector_norm(x.double(), dim=(-2, -1), keepdim=True) + eps).float()
    x = x.mT if turned else x
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.mT if turned else x).to(g.dtype).contiguous()


@functools.lru_cache(maxsize=64)
def _check_schulz(coefficients, steps: int) -> None:
    if len(coefficients) != 3 or not all(math.isfinite(v) for v in coefficients):
        raise ValueError("newton_schulz: three finite coefficients expected")
    a, b, c = coefficients
    v = [i / 4096.0 for i in range(4097)]
    for _ in range(steps):          # what every singular value of [0, 1] becomes; fp16 pairs hold entries up to 63
        if max(abs(b * x * x + c * x ** 4) for x in v) > 32.0:
            raise ValueError("newton_schulz: coefficients %r let singular values grow" % (coefficients,))
        v = [x * (a + b * x * x + c * x ** 4) for x in v]
        if max(abs(x) for x in v) > 4.0:
            raise ValueError("newton_schulz: coefficients %r let singular values grow" % (coefficients,))


# ----------------------------------------------------------------------------- input pipeline
IMAGENET_MEAN = (0.485, 0.456, 0.406)
IMAGENET_STD = (0.229, 0.224, 0.225)


def normalize_u8(x: torch.Tensor, dtype: torch.dtype = torch.float32, pad_c: int = 0,
                 mean=IMAGENET_MEAN, std=IMAGENET_STD, input_layout: str = "nhwc") -> torch.Tensor:
    """uint8 image batch -> normalised NHWC ``dtype`` (N-K16).

    ``(x - 255*mean_c) / (255*std_c)``, identical to the reference prefetcher
    (``imagenet_ddp_apex.py:311-340``).  ``pad_c`` zero-pads channels 3 -> pad_c
    so the stem convolution sees a vector-width-aligned C.
    """
    if _on_gpu(x):
        return _hip().normalize_u8(x, dtype, pad_c, mean, std, input_layout)
    if input_layout == "nchw":
        x = x.permute(0, 2, 3, 1)
    m = torch.tensor(mean, dtype=torch.float32, device=x.device) * 255.0
    s = torch.tensor(std, dtype=torch.float32, device=x.device) * 255.0
    y = ((x.float() - m) / s).to(dtype)
    if pad_c and pad_c > y.shape[-1]:
        y = TF.pad(y, (0, pad_c - y.shape[-1]))
    return y.contiguous()


def s2d_ok(x: torch.Tensor) -> bool:
    """True when ``to_s2d`` applies: a 3-channel image batch with even extents on the GPU."""
    return _on_gpu(x) and _hip().s2d_ok(x)


def to_s2d(x: torch.Tensor, dtype: torch.dtype, mean=IMAGENET_MEAN, std=IMAGENET_STD) -> torch.Tensor:
    """Image batch (uint8 NHWC / NCHW: normalised like ``normalize_u8``; float NCHW: converted) -> the space-to-depth
    layout ``[N, H/2, W/2, 16]`` consumed by 7x7 stride-2 stems (ResNet, DenseNet, GoogLeNet).  GPU only."""
    return _hip().to_s2d(x, dtype, mean, std)


def to_nhwc(x: torch.Tensor, dtype: Optional[torch.dtype] = None, pad_c: int = 0) -> torch.Tensor:
    """Float NCHW (torchvision convention) -> NHWC compute layout."""
    if _on_gpu(x):
        return _hip().nchw_to_nhwc(x, dtype or x.dtype, pad_c)
    y = x.permute(0, 2, 3, 1)
    if dtype is not None:
        y = y.to(dtype)
    if pad_c and pad_c > y.shape[-1]:
        y = TF.pad(y, (0, pad_c - y.shape[-1]))
    return y.contiguous()
