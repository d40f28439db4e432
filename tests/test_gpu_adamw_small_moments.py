"""AdamW's 8-bit moments beside larger ones of their block of 256: they have to fall as those of 32 bits do.

A step multiplies a second moment by 0.999 and a first one by 0.9, which is less than half a code for every
second moment and for first ones below code 10.  So codes are stored in the mean after the first 20 steps.
"""
import math

import pytest
import torch

from trident_amd import encoder

pytestmark = pytest.mark.gpu

LR = 1e-3


def run(bits, grad, n, steps, from_step=0):
    p = torch.zeros(n, device="cuda:0")
    opt = encoder.AdamW([p], lr=LR, weight_decay=0.0, state_bits=bits)
    opt.step_count = from_step
    for t in range(1, steps + 1):
        opt.step([grad(t)])
        if t == steps // 3:
            then = p.clone()
    m, v = (x.clone() for x in opt.state_values())
    return p, m, v, then


def stale_half(n, at, dev):
    """Every block's first half has a gradient in each step, its second half one in step `at` alone."""
    still = torch.arange(n, device=dev) % 256 >= 128
    busy = torch.where(still, 0.0, 1e-2)
    once = torch.where(still, 3e-4, 1e-2)
    return still, lambda t: once if t == at else busy


def test_moments_without_a_gradient_fall(dev):
    """From a count past the first 20 steps.  4,096 such elements, so the means are near: v's code (44 falling
    to 5) goes down by one with a probability of a quarter thousandth of it a step, which after 2,000 steps
    leaves each v off by its own size (the sum of 0.004 / code over the steps is about 1), and their mean by
    0.1 at six deviations; a first moment's way to zero varies by twice its mean, the mean of all by 0.19."""
    n = 8192
    still, grad = stale_half(n, 1, dev)
    p32, m32, v32, _ = run(32, grad, n, 2000, from_step=100)
    p8, m8, v8, then = run(8, grad, n, 2000, from_step=100)
    assert (m8[still] == 0).all()
    assert torch.equal(p8[still], then[still]), "still moves"
    assert abs(float(v8[still].mean() / v32[still].mean()) - 1) <= 0.15
    assert abs(float(p8[still].mean() / p32[still].mean()) - 1) <= 0.25
    # the busy half is at its blocks' top: its codes are the largest, its moments off by their rounding alone
    assert ((v8[~still] / v32[~still] - 1).abs() <= 1e-3).all()
    assert ((p8[~still] / p32[~still] - 1).abs() <= 1e-3).all()


def test_from_the_first_step(dev):
    """One gradient at step 10: until step 20 its moment stands still (at most ten more steps of the first
    one's length, which is a tenth of all that 32 bits move, so twice as far), and v's code stays while the
    block's top grows by the root of two, so v at most doubles."""
    n = 8192
    still, grad = stale_half(n, 10, dev)
    p32, m32, v32, _ = run(32, grad, n, 3000)
    p8, m8, v8, then = run(8, grad, n, 3000)
    print("moved, in lr:", float(p32[still].mean()) / LR, float(p8[still].mean()) / LR)
    assert (m8[still] == 0).all() and torch.equal(p8[still], then[still])
    assert 0.5 <= float(v8[still].mean() / v32[still].mean()) <= 2.2
    assert 0.5 <= float(p8[still].mean() / p32[still].mean()) <= 2.5


def test_gradients_that_shrink(dev):
    """Half of each block's gradients fall tenfold at step 500: the second moment follows as in 32 bits.  Its
    code walks by a few codes around its mean (below 0.35 of v at codes of 60 and more), 4,096 of them."""
    n = 8192
    half = torch.arange(n, device=dev) % 256 >= 128

    def grad(t):
        g = torch.Generator(device=dev).manual_seed(t)
        x = torch.randn(n, generator=g, device=dev) * 1e-2
        return torch.where(half, x * 0.1, x) if t > 500 else x

    _, _, v32, _ = run(32, grad, n, 4000)
    _, _, v8, _ = run(8, grad, n, 4000)
    for part in (half, ~half):
        assert abs(float(v8[part].mean() / v32[part].mean()) - 1) <= 0.05


def one_step(dev, n, step_count, m, v, grad):
    p = torch.zeros(n, device=dev)
    opt = encoder.AdamW([p], lr=LR, weight_decay=0.0, state_bits=8)
    opt.load_state(step_count, *coded(m, v))
    opt.step([grad])
    return opt


def coded(m, v):
    """Codes and scales of moments, in the nearest codes."""
    bm, bv = m.view(-1, 256), v.sqrt().view(-1, 256)
    sm, sv = bm.abs().amax(1) / 127 ** 2, bv.amax(1) / 255 ** 2
    cm = (torch.sign(bm) * torch.sqrt(bm.abs() / sm[:, None]).round()).to(torch.int8)
    cv = torch.sqrt(bv / sv[:, None]).round().clamp(min=1, max=255).to(torch.uint8)
    return cm, cv, sm, sv


def test_codes_are_neighbours_and_right_in_the_mean(dev):
    """Each code is the integer below or above the root of its value over the scale, and over 2^20 values the
    differences from the exact ones, in units of the step between the two codes, have the mean zero: six
    deviations of at most half a step each are 0.003, and 16 bits of dither are off by 1e-5."""
    n = 1 << 20
    g = torch.Generator(device=dev).manual_seed(5)
    r = lambda: torch.randn(n, generator=g, device=dev)  # noqa: E731
    m, v = 1e-3 * r() * torch.exp(r()), (1e-3 * r() * torch.exp(r())) ** 2
    grad = 1e-3 * r()
    cm, cv, sm, sv = coded(m, v)
    opt = one_step(dev, n, 200, m, v, grad)
    wide = lambda s: s.double().repeat_interleave(256)  # noqa: E731
    g64 = grad.double()
    m64 = 0.9 * (cm.double() * cm.double().abs()).view(-1) * wide(sm) + 0.1 * g64
    v64 = 0.999 * ((cv.double() ** 2).view(-1) * wide(sv)) ** 2 + 0.001 * g64 ** 2
    for code, scale, value, most, power in ((opt.exp_avg.double().abs(), opt.exp_avg_scale, m64.abs(), 127, 1),
                                            (opt.exp_avg_sq.double(), opt.exp_avg_sq_scale, v64.sqrt(), 255, 2)):
        root = torch.sqrt(value / wide(scale))
        assert ((code - root).abs() <= 1 + 1e-4 * root).all() and (code <= most).all()
        # the block's largest value has the largest code
        assert (code.view(-1, 256).amax(1) == most).all()
        lo = torch.floor(root + 1e-6)
        free = (root - lo > 1e-3) & (lo + 1 <= most) & (lo >= (1 if power == 2 else 0))
        a, b = lo ** (2 * power), (lo + 1) ** (2 * power)
        off = ((code ** (2 * power) - (value / wide(scale)) ** power) / (b - a))[free]
        assert int(free.sum()) > n // 2
        assert abs(float(off.mean())) <= 6 * 0.5 / math.sqrt(off.numel()) + 1e-4, float(off.mean())
        # the same among small codes, which a bias would hold up or pull down
        few = off[lo[free] <= 20]
        assert abs(float(few.mean())) <= 6 * 0.5 / math.sqrt(few.numel()) + 1e-4, float(few.mean())
    assert torch.equal(torch.sign(opt.exp_avg.double())[opt.exp_avg != 0], torch.sign(m64)[opt.exp_avg != 0])


def test_equal_calls_give_equal_bits_and_other_steps_other_ones(dev):
    n = 70_000 // 256 * 256
    g = torch.Generator(device=dev).manual_seed(6)
    m, v = 1e-3 * torch.randn(n, generator=g, device=dev), torch.rand(n, generator=g, device=dev) ** 4 * 1e-6
    grad = 1e-3 * torch.randn(n, generator=g, device=dev)
    codes = lambda t: torch.cat([x.float() for x in (lambda o: (o.exp_avg, o.exp_avg_sq))(  # noqa: E731
        one_step(dev, n, t, m, v, grad))])
    for t in (0, 5, 19):  # steps 1, 6 and 20: the nearest codes, whatever the step
        assert torch.equal(codes(t), codes(0))
    a = codes(20)
    assert torch.equal(codes(20), a) and torch.equal(codes(1 << 33), codes(1 << 33))
    for t in (21, 22, 400, (1 << 32) + 20, (1 << 33) + 20):
        share = float((codes(t) != a).float().mean())
        assert 0.02 <= share <= 0.5, (t, share)


def test_zeros_stay_zero(dev):
    """Elements without a gradient ever, and those past a tensor's end, keep moments of zero."""
    p = torch.ones(1000, device=dev)
    grad = torch.randn(1000, generator=torch.Generator(device=dev).manual_seed(7), device=dev)
    grad[100:300] = 0
    opt = encoder.AdamW([p], lr=LR, weight_decay=0.0, state_bits=8)
    for _ in range(60):
        opt.step([grad])
    m, v = opt.state_values()
    assert (m[100:300] == 0).all() and (v[100:300] == 0).all() and (m[1000:] == 0).all() and (v[1000:] == 0).all()
    assert (p[100:300] == 1).all() and (v[:100] > 0).all()


def test_not_finite_past_the_first_steps(dev):
    p = torch.ones(1000, device=dev)
    grad = torch.full((1000,), 0.5, device=dev)
    opt = encoder.AdamW([p], lr=LR, state_bits=8)
    for _ in range(25):
        opt.step([grad])
    grad[300], grad[700] = float("nan"), float("inf")
    opt.step([grad])
    m, v = opt.state_values()
    assert p[300].isnan() and m[300].isnan() and v[300].isnan()
    assert not m[700].isfinite() and not v[700].isfinite()
    others = torch.ones(1000, dtype=torch.bool, device=dev)
    others[256:768] = False
    assert p[others].isfinite().all() and m[:1000][others].isfinite().all() and v[:1000][others].isfinite().all()


def test_replays_of_a_captured_step(dev):
    """A graph replays one step number; the moments beside larger ones, whose gradients change from replay to
    replay, fall all the same.  After 600 replays a first moment is left with a probability of 0.9^600 of its
    code's square."""
    n = 8192
    still = torch.arange(n, device=dev) % 256 >= 128
    g = torch.Generator(device=dev).manual_seed(9)
    p, grad = torch.zeros(n, device=dev), torch.full((n,), 3e-4, device=dev)
    opt = encoder.AdamW([p], lr=LR, weight_decay=0.0, state_bits=8)
    opt.step_count = 100
    opt.step([grad])
    fresh = lambda: torch.where(still, 0.0, 1e-2 * torch.randn(n, generator=g, device=dev))  # noqa: E731
    grad.copy_(fresh())
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        opt.step([grad])
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        opt.step([grad])
    torch.cuda.synchronize()
    v0 = opt.state_values()[1][still].clone()
    for i in range(600):
        grad.copy_(fresh())
        graph.replay()
    torch.cuda.synchronize()
    m, v = opt.state_values()
    assert (m[still] == 0).all()
    # 0.999^600, 4,096 elements each off by no more than its own size
    assert abs(float(v[still].mean() / v0.mean()) / 0.999 ** 600 - 1) <= 0.15
