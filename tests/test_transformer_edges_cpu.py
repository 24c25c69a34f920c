"""The transformer operators' refusals, modules and optimizer at their edges, on the CPU backend."""
import pytest
import torch

from distributed_pytorch_amd.ops import functional as F


def test_newton_schulz_fast_is_for_bf16():
    g = torch.randn(6, 9)
    for dtype in (torch.float32, torch.float16):
        with pytest.raises(ValueError, match="bfloat16"):
            F.newton_schulz(g.to(dtype), fast=True)
    assert torch.equal(F.newton_schulz(g.bfloat16(), fast=True), F.newton_schulz(g.bfloat16()))     # (32 bits here either way)
