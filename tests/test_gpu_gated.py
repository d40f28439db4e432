"""The gated feed-forward product and its backward pass against float64 implementations of the formulas.

Bounds: a sum of n float32 products is off by (n + 2) u times the sum of their magnitudes.  The activations' slopes are at
most 1.13 in size and change by at most 0.8 a unit; their float32 evaluation is off by at most 16 u (1 + |g|).  g and u are
kept in float32; dg, du are multiplied in the elements' type: U[dtype] relative.
"""
import pytest
import torch

from trident_amd import encoder
from test_gpu_encoder import F64, TINY, TYPES, U, gen, randn, u, within

pytestmark = pytest.mark.gpu

ACTIVATIONS = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
               "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}


def act_and_slope(name, g):
    with torch.enable_grad():
        t = g.detach().clone().requires_grad_()
        a = ACTIVATIONS[name](t)
        (slope,) = torch.autograd.grad(a.sum(), t)
    return a.detach(), slope


def reference(x, wg, wu, act, grad=None):
    dtype, K = x.dtype, x.shape[-1]
    Un, tiny = U[dtype], TINY[dtype]
    x, wg, wu = (t.to(F64) for t in (x.reshape(-1, K), wg, wu))
    g, up = x @ wg.t(), x @ wu.t()
    eg, eu = ((K + 2) * u * (x.abs() @ w.abs().t()) for w in (wg, wu))
    a, slope = act_and_slope(act, g)
    ea = 1.13 * eg + 16 * u * (1 + g.abs()) * (a.abs() / (1 + g.abs()) + u + slope.abs())
    h = a * up
    res = dict(h=(h, Un * h.abs() + 2 * u * h.abs() + ea * up.abs() + (a.abs() + ea) * eu + tiny))
    if grad is None:
        return res
    dh = grad.to(F64).reshape(g.shape)
    M, N = dh.shape
    rg, ru = eg + u * g.abs(), eu + u * up.abs()  # of what is kept
    ea, es = 1.13 * rg + 16 * u * (1 + g.abs()), 0.8 * rg + 16 * u * (1 + g.abs())
    dg, du = dh * up * slope, dh * a
    edg = dh.abs() * (ru * (slope.abs() + es) + up.abs() * es) + (Un + 3 * u) * dg.abs() + tiny
    edu = dh.abs() * ea + (Un + 3 * u) * du.abs() + tiny

    def product(p, ep, q, n):  # p q with p off by ep
        v, size = p @ q, p.abs() @ q.abs()
        return v, ep @ q.abs() + (n + 2) * u * (size + ep @ q.abs())

    x1, b1 = product(dg, edg, wg, 2 * N)
    x2, b2 = product(du, edu, wu, 2 * N)
    for n, (v, b) in dict(dx=(x1 + x2, b1 + b2), dwg=product(dg.t(), edg.t(), x, M),
                          dwu=product(du.t(), edu.t(), x, M)).items():
        res[n] = v, b + Un * v.abs() + tiny
    return res


def operands(seed, dtype, M, N, K):
    g = gen(seed)
    return (randn(g, M, K, dtype=dtype), (randn(g, N, K) / K ** 0.5).to(dtype), (randn(g, N, K) / K ** 0.5).to(dtype),
            (1e-2 * randn(g, M, N)).to(dtype))


def check(x, wg, wu, act, grad):
    ref = reference(x, wg, wu, act, grad)
    h = encoder.gated_linear(x, wg, wu, act)
    kept = encoder.gated_linear_forward(x, wg, wu, act)
    assert torch.equal(kept[0], h) and h.dtype == x.dtype and h.shape == (*x.shape[:-1], wg.shape[0])
    dx, dwg, dwu = encoder.gated_linear_grad(grad, x, wg, wu, *kept[1:], act)
    assert dx.shape == x.shape and dwg.shape == wg.shape and dwu.shape == wu.shape
    for n, t in dict(h=h, dx=dx, dwg=dwg, dwu=dwu).items():
        within(t.reshape(-1, t.shape[-1]), *ref[n], what=n)


SIZES = [(1, 1, 1), (1, 16, 64), (2, 17, 7), (16, 100, 960), (17, 33, 8), (16, 64, 1000), (33, 65, 72), (64, 64, 64),
         (100, 130, 200), (129, 257, 136), (200, 96, 333), (300, 40, 1024), (777, 333, 100), (1030, 70, 48), (3, 2000, 515),
         (100, 333, 2500), (33, 65, 2101), (64, 64, 4500), (5000, 40, 56), (2100, 70, 33), (1, 1, 3000), (17, 2600, 24)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_sizes(dev, dtype, M, N, K):
    x, wg, wu, grad = operands(M + N, dtype, M, N, K)
    check(x, wg, wu, ("silu", "gelu", "gelu_tanh")[(M + N + K) % 3], grad)


@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("dtype", TYPES)
def test_activations_over_their_range(dev, dtype, act):
    g = torch.cat([torch.linspace(-12, 12, 997), torch.tensor([0.0, -0.0, 1e-8, 30.0, -30.0, 80.0, -80.0])])
    x = torch.ones((1, 8), device=dev)
    x[:, 1:] = 0
    wg = torch.zeros((g.numel(), 8), device=dev)
    wg[:, 0] = g.to(dev)
    wu = torch.ones_like(wg)
    grad = torch.ones((1, g.numel()), device=dev)
    for rows in (1, 20):  # either kernel
        check(x.expand(rows, 8).to(dtype), wg.to(dtype), wu.to(dtype), act, grad.expand(rows, -1).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(dev, dtype):
    g = gen(3)
    for K in (40, 37):
        both = (randn(g, 2 * 60, K) / K ** 0.5).to(dtype)  # the halves of one matrix
        wide = randn(g, 4, 30, K + 11, dtype=dtype)
        grad = (1e-2 * randn(g, 4, 30, 60)).to(dtype)
        check(wide[..., 3:3 + K], both[:60], both[60:], "silu", grad)
        x = wide[0, :, :K]
        check(x, both[::2], both[1::2], "gelu", grad[0])
        check(x, both[:60].t().contiguous().t(), both[60:], "gelu", grad[0].t().contiguous().t())
        check(wide[0, 0, :K], both[:60], both[60:], "silu", grad[0, 0])  # one row, no dimension of rows
        big = torch.zeros((30, 64), dtype=dtype, device=dev)
        big[:, 2:62] = grad[0]
        check(x, both[:60], both[60:], "silu", big[:, 2:62])


def test_no_rows_or_columns(dev):
    for M, N in ((0, 5), (4, 0)):
        x, wg, wu, grad = operands(4, torch.bfloat16, M, N, 24)
        h, gate, up = encoder.gated_linear_forward(x, wg, wu)
        assert h.shape == (M, N)
        for t, like in zip(encoder.gated_linear_grad(grad, x, wg, wu, gate, up), (x, wg, wu)):
            assert t.shape == like.shape and (t == 0).all()


def test_a_value_that_is_not_finite_stays_in_its_row(dev):
    for dtype in TYPES:
        for M in (5, 200):
            x, wg, wu, grad = operands(5, dtype, M, 70, 100)
            clean = encoder.gated_linear(x, wg, wu)
            x[3, 99] = float("nan")
            got = encoder.gated_linear(x, wg, wu)
            assert got[3].isnan().all()
            keep = [i for i in range(M) if i != 3]
            assert torch.equal(got[keep], clean[keep])


def test_what_lies_behind_the_rows_is_not_used(dev):
    for dtype in TYPES:
        for K in (72, 68):
            wide = torch.full((90, 128), float("nan"), dtype=dtype, device=dev)
            x, wg, wu, grad = operands(6, dtype, 90, 90, K)
            want = encoder.gated_linear_forward(x, wg, wu)
            wide[:, :K] = x
            wides = [torch.full_like(wide, float("inf")) for _ in range(2)]
            for t, w in zip(wides, (wg, wu)):
                t[:, :K] = w
            views = [wide[:, :K], wides[0][:, :K], wides[1][:, :K]]
            got = encoder.gated_linear_forward(*views)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            for a, b in zip(encoder.gated_linear_grad(grad, *views, *got[1:]),
                            encoder.gated_linear_grad(grad, x, wg, wu, *want[1:])):
                assert torch.equal(a, b)


@pytest.mark.parametrize("act", list(ACTIVATIONS))
def test_autograd_against_differences(dev, act):
    """Derivatives along random directions against differences of the float64 formula; what is left is the float32
    roundings of some hundred terms."""
    x, wg, wu, grad = operands(7, torch.float32, 40, 50, 60)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    encoder.gated_linear(*leaves, act).backward(grad)

    def value(x, wg, wu):
        return (ACTIVATIONS[act](x @ wg.t()) * (x @ wu.t()) * grad.to(F64)).sum()

    g = gen(8)
    for i, t in enumerate(leaves):
        d, e = randn(g, *t.shape).to(F64), 1e-5
        at = [v.detach().to(F64) for v in leaves]
        far = [[v + (e * s * d if i == j else 0) for j, v in enumerate(at)] for s in (1, -1)]
        want = (value(*far[0]) - value(*far[1])) / (2 * e)
        size = t.grad.to(F64).square().sum().sqrt() * d.square().mean().sqrt()
        assert abs((t.grad.to(F64) * d).sum() - want) <= 1e-5 * size


def test_autograd_needs(dev):
    x, wg, wu, grad = operands(9, torch.bfloat16, 40, 48, 56)
    h, gate, up = encoder.gated_linear_forward(x, wg, wu)
    want = encoder.gated_linear_grad(grad, x, wg, wu, gate, up)
    for which in ((0,), (1,), (2,), (0, 2)):
        t = [v.clone().requires_grad_(i in which) for i, v in enumerate((x, wg, wu))]
        out = encoder.gated_linear(*t)
        assert torch.equal(out, h)
        got = torch.autograd.grad(out, [t[i] for i in which], grad)
        assert all(torch.equal(a, want[i]) for a, i in zip(got, which))


def test_same_bits_each_time_and_captured(dev):
    x, wg, wu, grad = operands(10, torch.bfloat16, 500, 333, 200)
    xq = x[:3].clone()

    def run():
        h, gate, up = encoder.gated_linear_forward(x, wg, wu)
        return (h, *encoder.gated_linear_grad(grad, x, wg, wu, gate, up), encoder.gated_linear(xq, wg, wu))

    run()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        got = run()
    for i in range(3):
        x.mul_(0.9)
        want = run()
        assert all(torch.equal(a, b) for a, b in zip(want, run()))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_far_rows(dev):
    """Rows past 2^31 bytes of x and of the result."""
    M, N, K = 300_000, 4096, 4096
    x = torch.zeros((M, K), dtype=torch.bfloat16, device=dev)
    _, wg, wu, _ = operands(11, torch.bfloat16, 1, N, K)
    tail = randn(gen(12), 200, K, dtype=torch.bfloat16)
    x[-200:] = tail
    h = encoder.gated_linear(x, wg, wu)
    assert torch.equal(h[-200:], encoder.gated_linear(tail, wg, wu)) and (h[:100_000] == 0).all()
