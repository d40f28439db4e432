"""Rotary positions against a float64 implementation of the formula.

Bounds: an angle is off by at most 2^-51 of its size (two roundings in float64) plus 2^-23 of half a turn (one float32 rounding
of what is left of whole turns, and the sine's own), so a turned pair by about 8 u of its length; then the
result's rounding.
"""
import math

import pytest
import torch

from trident_amd import encoder
from test_gpu_encoder import F64, TINY, TYPES, U, gen, randn, u, within

pytestmark = pytest.mark.gpu


def reference(x, f, positions, interleaved, amplitude=1.0, inverse=False):
    """(value, bound) in float64"""
    n, y = f.numel(), x.to(F64).clone()
    t = (positions.to(F64)[..., None] * f)[..., None, :]
    c, s = amplitude * torch.cos(t), amplitude * torch.sin(t) * (-1.0 if inverse else 1.0)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    x0, x1 = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = x0 * c - x1 * s, x0 * s + x1 * c
    bound = U.get(x.dtype, 0.0) * y.abs() + TINY.get(x.dtype, 0.0)
    size = abs(amplitude) * (x0.abs() + x1.abs()) * (12 * u + 2.0 ** -51 * t.abs())
    bound[..., a] += size
    bound[..., b] += size
    return y, bound


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,R", [(1, 1, 2, 2), (3, 5, 64, 64), (16, 24, 64, 64), (100, 3, 128, 64), (7, 2, 33, 32),
                                     (50, 3, 100, 100), (50, 3, 100, 50), (33, 4, 80, 40), (2100, 2, 96, 96),
                                     (40000, 1, 8, 6), (5, 2, 2048, 2048), (9, 3, 20, 0), (4100, 3, 24, 10)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rotary(dev, dtype, T, H, D, R, interleaved):
    g = gen(T + D)
    x = randn(g, T, H, D, dtype=dtype)
    positions = torch.randint(0, 100_000, (T,), generator=g, device=dev)
    f = encoder.rotary_frequencies(R, device=dev) if R else torch.zeros(0, dtype=F64, device=dev)
    for inverse in (False, True):
        y = encoder.rotary(x, f, positions.int() if inverse else positions, interleaved, amplitude=1.25, inverse=inverse)
        assert y.dtype == dtype and y.shape == x.shape
        within(y, *reference(x, f, positions, interleaved, 1.25, inverse))
        assert torch.equal(y[..., R:], x[..., R:])


def test_far_and_negative_positions(dev):
    x = randn(gen(1), 6, 2, 32)
    f = encoder.rotary_frequencies(32, device=dev)
    positions = torch.tensor([0, -1, 1_000_003, 2 ** 31 - 1, -(2 ** 31), 2 ** 40 + 12345], device=dev)
    within(encoder.rotary(x, f, positions), *reference(x, f, positions, False))


def test_positions_shared_or_left_out(dev):
    x = randn(gen(2), 3, 50, 4, 64, dtype=torch.bfloat16)
    f = encoder.rotary_frequencies(64, device=dev)
    p = torch.arange(50, device=dev)
    want, bound = reference(x, f, p.expand(3, 50), False)
    for got in (encoder.rotary(x, f), encoder.rotary(x, f, p), encoder.rotary(x, f, p.expand(3, 50)),
                torch.stack([encoder.rotary(y, f) for y in x])):
        within(got, want, bound)
    one = randn(gen(3), 4, 64)  # a single token, no dimension of tokens
    assert torch.equal(encoder.rotary(one, f), one)
    within(encoder.rotary(one, f, torch.tensor(7, device=dev)),
           *reference(one, f, torch.tensor(7, device=dev), False))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_in_place(dev, dtype):
    g = gen(4)
    qkv = randn(g, 70, 9, 40, dtype=dtype)
    f = encoder.rotary_frequencies(24, device=dev)
    p = torch.randint(0, 1000, (70,), generator=g, device=dev)
    whole = qkv.clone()
    for interleaved in (False, True):
        want, bound = reference(whole[:, :6], f, p, interleaved)
        within(encoder.rotary(qkv[:, :6], f, p, interleaved), want, bound)
        within(encoder.rotary(qkv.transpose(0, 1).contiguous().transpose(0, 1)[:, :6], f, p, interleaved), want, bound)
        odd = torch.empty((70, 6, 41), dtype=dtype, device=dev)
        odd[..., 1:] = qkv[:, :6]
        within(encoder.rotary(odd[..., 1:], f, p, interleaved), want, bound)  # any element's address
        other = torch.full_like(whole, 7.0)
        assert encoder.rotary(qkv[:, :6], f, p, interleaved, out=other[:, 2:8]) is not None
        within(other[:, 2:8], want, bound)
        assert (other[:, :2] == 7).all() and (other[:, 8:] == 7).all()
        version = qkv._version
        encoder.rotary(qkv[:, :6], f, p, interleaved, out=qkv[:, :6])
        assert qkv._version > version
        within(qkv[:, :6], want, bound)
        assert torch.equal(qkv[:, 6:], whole[:, 6:])
        qkv.copy_(whole)


def test_frequencies():
    f = encoder.rotary_frequencies(8, base=100.0)
    assert f.dtype == F64 and torch.allclose(f, 100.0 ** (-torch.arange(4, dtype=F64) / 4), rtol=1e-14)
    assert torch.equal(encoder.rotary_frequencies(8, 100.0, "linear", 4.0), f / 4)
    b = encoder.rotary_frequencies(8, 100.0, "base", 4.0)
    assert b[0] == f[0] and abs(b[-1] * 4 / f[-1] - 1) < 1e-12
    t = encoder.rotary_frequencies(64, 10000.0, "turns", 8.0, trained=2048)
    plain = encoder.rotary_frequencies(64)
    turns = 2048 * plain / (2 * math.pi)
    assert torch.equal(t[turns >= 32], plain[turns >= 32]) and torch.equal(t[turns <= 1], plain[turns <= 1] / 8)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((t < plain) & (t > plain / 8))[between].all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(dev, interleaved):
    """The gradient against the formula's transpose (differences of a linear map are itself)."""
    g = gen(6)
    x, grad = randn(g, 30, 3, 24).requires_grad_(), randn(g, 30, 3, 24)
    f = encoder.rotary_frequencies(16, device=dev)
    p = torch.randint(0, 500, (30,), generator=g, device=dev)
    y = encoder.rotary(x, f, p, interleaved, amplitude=0.7)
    y.backward(grad)
    within(x.grad, *reference(grad, f, p, interleaved, 0.7, inverse=True))
    d = randn(g, 30, 3, 24).to(F64)
    moved = reference(x.detach().to(F64) + d, f, p, interleaved, 0.7)[0] - \
        reference(x.detach().to(F64) - d, f, p, interleaved, 0.7)[0]
    want = (moved / 2 * grad.to(F64)).sum()
    assert abs((x.grad.to(F64) * d).sum() - want) <= 20 * u * (grad.abs().to(F64) * 4).sum()


def test_captured_and_replayed(dev):
    x = randn(gen(7), 500, 4, 64, dtype=torch.bfloat16)
    f = encoder.rotary_frequencies(64, device=dev)
    p = torch.arange(500, device=dev)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        encoder.rotary(x, f, p)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        y = encoder.rotary(x, f, p)
    for i in range(3):
        p += 1000 * i
        want = encoder.rotary(x, f, p)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
