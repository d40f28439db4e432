"""The gated product's gradients where gates, gradients or pitches are very large or very small."""
import math

import pytest
import torch

from trident_amd import encoder
from test_gpu_encoder import TYPES, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", TYPES)
def test_slopes_of_very_large_gates(dev, dtype, act):
    """From 100 on every activation is its gate or zero, and its slope 1 or 0, in any precision: up to the largest float32."""
    far = [100.0, 250.0, 1e4, 6e4] + ([] if dtype is torch.float16 else [1e9, 1.1e13, 2e13, 1e18, 2e19, 1e30, 3e38])
    gate = torch.tensor([[s * g for g in far for s in (1, -1)]], device=dev)
    up, n = torch.ones_like(gate), gate.shape[1]
    x = torch.zeros((1, 8), dtype=dtype, device=dev)
    x[0, 0] = 1.0
    w = torch.zeros((n, 8), dtype=dtype, device=dev)
    dx, dwg, dwu = encoder.gated_linear_grad(torch.ones((1, n), dtype=dtype, device=dev), x, w, w, gate, up, act)
    assert torch.equal(dwg[:, 0].float(), (gate[0] > 0).float())
    assert torch.equal(dwu[:, 0], gate[0].clamp(min=0).to(dtype))
    assert (dx == 0).all() and (dwg[:, 1:] == 0).all()


@pytest.mark.parametrize("M", [8, 40])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_far_apart(dev, dtype, M):
    """The first token of every passage, and weights as far apart: the same bits as contiguous rows."""
    g, K, N, T = gen(M), 520, 24, 4096  # 2,129,920 elements from row to row
    x, wg, wu = randn(g, M, K, dtype=dtype), *((randn(g, N, K) / K ** 0.5).to(dtype) for _ in range(2))
    grad = (1e-2 * randn(g, M, N)).to(dtype)
    far = []
    for t in (x, wg, wu):
        big = torch.full((len(t), T, K), math.nan, dtype=dtype, device=dev)
        big[:, 0] = t
        far.append(big[:, 0])
    want = encoder.gated_linear_forward(x, wg, wu)
    grads = encoder.gated_linear_grad(grad, x, wg, wu, *want[1:])
    for operands in ((far[0], wg, wu), (x, far[1], wu), (x, wg, far[2]), far):
        got = encoder.gated_linear_forward(*operands)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(encoder.gated_linear(*operands), want[0])
        assert all(torch.equal(a, b) for a, b in zip(encoder.gated_linear_grad(grad, *operands, *got[1:]), grads))
