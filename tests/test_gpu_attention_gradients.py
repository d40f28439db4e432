"""Attention's gradients against their formulas in float64 where a looser bound would hide what goes wrong: values that share
a part (dP - delta cancels), keys whose infinities keep them from every row.

u = 2^-24 is a float32 operation's rounding, U[dtype] that of P, dS and results.  The bounds have no term for the rounding of
out: delta is the float32 sum of P dP, made of the rounded out and what the sum of dS shows it to lack.
"""
import math

import pytest
import torch

from trident_amd import encoder
from test_gpu_encoder import F64, TINY, TYPES, U, gen, randn, u, within

pytestmark = pytest.mark.gpu


def gradients(q, k, v, grad, hidden, scale):
    """dict of name -> (value, bound) for one sequence: q and grad [m, Hq, D], k and v [m, Hkv, D], `hidden` [m, m]."""
    dtype, (m, Hq, D), Hkv = q.dtype, q.shape, k.shape[1]
    Un, tiny, G = U[dtype], TINY[dtype], Hq // Hkv
    half = dtype is torch.float16
    q, k, v, grad = (t.to(F64) for t in (q, k, v, grad))
    res = {n: [torch.zeros_like(t), torch.zeros_like(t)] for n, t in (("dq", q), ("dk", k), ("dv", v))}
    for h in range(Hq):
        Q, K, V, dO, g = q[:, h], k[:, h // G], v[:, h // G], grad[:, h], h // G
        s = (scale * Q @ K.t()).masked_fill(hidden, -math.inf)
        size = (scale * Q.abs() @ K.abs().t()).masked_fill(hidden, 0.0)
        p = torch.softmax(s, 1)
        top = s.masked_fill(s.isinf(), 0.0).abs().amax(1, keepdim=True)
        E = ((D + 8) * u * size + 8 * u * top).amax(1, keepdim=True)  # of a score, and so of its exp
        rel, n = 3 * E + (m + 12) * u, m * G
        out = p @ V
        dP = dO @ V.t()
        delta = (dO * out).sum(1, keepdim=True)
        lacks = dO.abs() @ (Un * out.abs() + (Un + rel) * (p @ V.abs())).t()  # of the first delta, from the rounded out
        lacks = lacks.diagonal()[:, None]
        dS, spread = p * (dP - delta), p * (dP - delta).abs()
        e_dP = (D + 2) * u * (dO.abs() @ V.abs().t())
        # the sum of dS: each P and dP off by their own, m additions
        e_delta = ((rel + (m + 4) * u) * (spread + p * lacks) + p * e_dP).sum(1, keepdim=True) + 2 * u * delta.abs()
        held = 2.0 ** -38 * spread.max() if half else 0.0  # dS lies within 2^28 of its column's largest, or loses digits
        e_dS = p * (rel * (dP - delta).abs() + e_dP + e_delta) + (Un + (n + 4) * u) * dS.abs() + held
        # dq: dS made with the first delta is rounded, and so is P, whose sum with the keys makes up for it
        e_dq = e_dS + 2 * Un * p * lacks + (2.0 ** -24 * lacks if half else 0.0)
        res["dq"][0][:, h] = scale * dS @ K
        res["dq"][1][:, h] = scale * e_dq @ K.abs()
        res["dk"][0][:, g] += scale * dS.t() @ Q
        res["dk"][1][:, g] += scale * e_dS.t() @ Q.abs()
        res["dv"][0][:, g] += p.t() @ dO
        res["dv"][1][:, g] += (Un + n * u) * (p.t() @ dO.abs()) + (p * rel).t() @ dO.abs() + \
            2.0 ** -40 * dO.abs().sum(0) * half
    return {n: (value, bound + Un * value.abs() + tiny) for n, (value, bound) in res.items()}


def run(q, k, v, grad, causal, padded=0):
    """(dq, dk, dv) of one sequence, packed, or the first of two with `padded` slots"""
    if not padded:
        out, lse = encoder.attention_forward(q, k, v, causal=causal)
        return encoder.attention_grad(grad, q, k, v, out, lse, causal=causal)
    m = q.shape[0]

    def pad(t):
        p = torch.full((2, padded, *t.shape[1:]), math.nan, dtype=t.dtype, device=t.device)
        p[0, :m] = t
        return p

    q, k, v, grad = (pad(t) for t in (q, k, v, grad))
    how = dict(lengths=torch.tensor([m, 0], device=q.device), causal=causal)
    out, lse = encoder.attention_forward(q, k, v, **how)
    got = encoder.attention_grad(grad, q, k, v, out, lse, **how)
    assert all((t[0, m:] == 0).all() and (t[1] == 0).all() for t in got)
    return [t[0, :m] for t in got]


def hidden_keys(m, causal, device):
    t = torch.ones((m, m), dtype=torch.bool, device=device)
    return t.triu(1) if causal else t & False


@pytest.mark.parametrize("m,D", [(1, 64), (3, 64), (33, 32), (150, 64), (150, 128), (257, 80), (700, 16)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_share_a_part(dev, dtype, causal, m, D):
    """Values of 4 + r / 16 and keys of 2 + r: out's rounding is as large as what the gradients are made of."""
    g = gen(m + D)
    q, grad = randn(g, m, 4, D, dtype=dtype), (1e-2 * randn(g, m, 4, D)).to(dtype)
    k, v = (2 + randn(g, m, 2, D)).to(dtype), (4 + randn(g, m, 2, D) / 16).to(dtype)
    ref = gradients(q, k, v, grad, hidden_keys(m, causal, dev), D ** -0.5)
    for n, t in zip(("dq", "dk", "dv"), run(q, k, v, grad, causal, 0 if m % 2 else m + 40)):
        within(t, *ref[n], what=n)


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_that_pick_few_keys(dev, dtype):
    """Scores of some tens: a row's few heavy keys, each with a large dS."""
    g = gen(1)
    q, k, v = (randn(g, 200, H, 64, dtype=dtype) * s for H, s in ((4, 5), (2, 1), (2, 1)))
    grad = (1e-2 * randn(g, 200, 4, 64)).to(dtype)
    ref = gradients(q, k, v, grad, hidden_keys(200, False, dev), 0.125)
    for n, t in zip(("dq", "dk", "dv"), run(q, k, v, grad, False)):
        within(t, *ref[n], what=n)


@pytest.mark.parametrize("m", [31, 64, 70, 100, 129])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_key_that_its_infinity_hides(dev, dtype, causal, m):
    """A key of -inf in a column where every query is positive has scores of -inf: no row sees it, its gradients are zero and
    the others those without it, however far the sequence's end is from a tile's.  Only dq's own column has zero times
    infinity."""
    g = gen(m)
    q, k, v, grad = (randn(g, m, H, 64, dtype=dtype) for H in (4, 2, 2, 4))
    q[..., 0] = q[..., 0].abs() + 0.5
    hidden = hidden_keys(m, causal, dev)
    hidden[:, 5] = True
    ref = gradients(q, k, v, grad, hidden, 0.125)
    k[5, :, 0] = -math.inf
    for padded in (0, m + 33):
        dq, dk, dv = run(q, k, v, grad, causal, padded)
        assert (dk[5] == 0).all() and (dv[5] == 0).all()
        within(dk, *ref["dk"], what="dk")
        within(dv, *ref["dv"], what="dv")
        within(dq[..., 1:], *(t[..., 1:] for t in ref["dq"]), what="dq")
        assert dq[5:, :, 0].isnan().all()
        if causal:
            within(dq[:5], *(t[:5] for t in ref["dq"]), what="dq")


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
