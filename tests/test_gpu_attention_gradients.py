"""Attention's results and gradients against their formulas in float64 where a looser bound would hide what goes wrong.

u = 2^-24 is a float32 operation's rounding, U[dtype] that of P, dS and results.
"""
import pytest
import torch

from trident_amd import encoder
from test_gpu_encoder import F64, TINY, TYPES, U, gen, randn, u, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_next_to_zero(dev, dtype):
    """A scale that float32 barely holds: all keys of a row count the same."""
    g = gen(2)
    q, k, v, grad = (randn(g, 40, 2, 32, dtype=dtype) for _ in range(4))
    for scale in (2.0 ** -149, 1e-44, 1e-40, 1e-37):
        out, lse = encoder.attention_forward(q, k, v, causal=True, scale=scale)
        mean = v.to(F64).cumsum(0) / torch.arange(1, 41, device=dev)[:, None, None]
        size = v.to(F64).abs().cumsum(0) / torch.arange(1, 41, device=dev)[:, None, None]
        held = 2.0 ** -32 * v.to(F64).abs().sum(0) if dtype is torch.float16 else 0.0
        within(out, mean, (U[dtype] + 60 * u) * size + held + U[dtype] * mean.abs() + TINY[dtype])
        for t in encoder.attention_grad(grad, q, k, v, out, lse, causal=True, scale=scale)[:2]:
            assert (t.abs() <= 1e-30).all()
