"""Calls at the edge of what the transformer operators take: who watches a call (tangents, traces, tensor subclasses), every
size of workgroup, vectors, sinks of gates, extreme gradients.  Bounds are those of tests/_transformer_ref.py."""
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
