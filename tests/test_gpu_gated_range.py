"""The gated product's gradients where gates, gradients or pitches are very large or very small."""
import math

import pytest
import torch

from trident_amd import encoder
from test_gpu_encoder import F64, TYPES, U, gen, randn, u, within

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


def act_slope(name, g):
    """(act(g), act'(g)) in float64"""
    if name == "gelu":
        p = 0.5 * torch.erfc(-g * math.sqrt(0.5))
        return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    z, dz = (g, 1.0) if name == "silu" else (math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3),
                                              math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * g * g))
    p = torch.sigmoid(z)
    return g * p, p + g * p * torch.sigmoid(-z) * dz


# dg and du are multiplied in the operands' type.  In float16 that is times a power of two by which the largest of them comes to
# 2^14 or more: a rounding of 2^-11 relative down to 2^-28 of the largest, and 2^-39 of the largest below.
@pytest.mark.parametrize("M,N,K", [(1, 300, 64), (200, 300, 64), (130, 130, 1000), (2500, 64, 40), (1500, 1100, 1030),
                                   (2100, 2080, 264)])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_small_and_large_gradients_in_float16(dev, act, M, N, K):
    g, Un = gen(M + N), 2.0 ** -11
    x, wg, wu = (randn(g, *s, dtype=torch.float16) for s in ((M, K), (N, K), (N, K)))
    gate, up = randn(g, M, N), randn(g, M, N)
    # gradients of 1e-4 by products of 1e-2; of 50 by products of 1e4, past float16's largest; rows of unlike sizes
    rows = torch.exp2(-12 * torch.rand((M, 1), generator=g, device=dev))
    for name, dh, by, w in (("small", 1e-4, 1e-2, 10.0), ("tiny", 2e-7, 1.0, 30.0), ("large", 50.0, 1e4, 2.0 ** -13),
                            ("rows", rows, 1e-2, 10.0)):
        grad, u2 = (dh * randn(g, M, N)).half(), by * up
        ops = [(w * t).half() for t in (x, wg, wu)]
        got = encoder.gated_linear_grad(grad, *ops, gate, u2, act)
        xd, wgd, wud, d = (t.to(F64) for t in (*ops, grad))
        a, s = act_slope(act, gate.to(F64))
        dg, du = d * u2.to(F64) * s, d * a
        held = 2.0 ** -39 * max(dg.abs().max(), du.abs().max())
        # the activations' float32 evaluation is off by at most 16 u (1 + |g|)
        off = 16 * u * (1 + gate.to(F64).abs())
        eg = (Un + 3 * u) * dg.abs() + d.abs() * u2.to(F64).abs() * off + held
        eu = (Un + 3 * u) * du.abs() + d.abs() * off + held

        def product(p, ep, q, n):
            return p @ q, ep @ q.abs() + (n + 2) * u * ((p.abs() + ep) @ q.abs())

        (x1, b1), (x2, b2) = product(dg, eg, wgd, 2 * N), product(du, eu, wud, 2 * N)
        ref = ((x1 + x2, b1 + b2), product(dg.t(), eg.t(), xd, M), product(du.t(), eu.t(), xd, M))
        for n, t, (v, b) in zip(("dx", "dwg", "dwu"), got, ref):
            within(t, v, b + Un * v.abs() + 2.0 ** -25, what=f"{name} {n}")
            assert t.isfinite().all() or v.abs().max() > 65504


def test_gradients_that_are_zero_or_not_finite_in_float16(dev):
    """A factor made from the largest finite value: zeros stay zeros, and an infinity is alone in its row and weight."""
    g = gen(5)
    x, wg, wu = (randn(g, *s, dtype=torch.float16) for s in ((70, 40), (50, 40), (50, 40)))
    gate, up, grad = randn(g, 70, 50), randn(g, 70, 50), (1e-3 * randn(g, 70, 50)).half()
    assert all((t == 0).all() for t in encoder.gated_linear_grad(0 * grad, x, wg, wu, gate, up))
    clean = encoder.gated_linear_grad(grad, x, wg, wu, gate, up)
    grad[3, 7] = 0
    want = encoder.gated_linear_grad(grad, x, wg, wu, gate, up)
    assert not torch.equal(want[0], clean[0])
    for bad in (math.inf, math.nan):
        grad[3, 7] = bad
        dx, dwg, dwu = encoder.gated_linear_grad(grad, x, wg, wu, gate, up)
        assert not dx[3].isfinite().any() and not dwg[7].isfinite().any() and not dwu[7].isfinite().any()
        for t, like, at in ((dx, want[0], 3), (dwg, want[1], 7), (dwu, want[2], 7)):
            keep = [i for i in range(len(t)) if i != at]
            assert torch.equal(t[keep], like[keep])
