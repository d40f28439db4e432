"""Attention and its backward pass against float64 implementations of the formulas.

Tolerances are bounds, derived here from the arithmetic: u = 2^-24 is a float32 operation's rounding, U[dtype] a
result's (and that of P and dS, which are rounded to the elements' type for the second products), and a sum of n
float32 terms is off by at most n u times the sum of their magnitudes.  A score is off by
E = (D + 8) u scale |q|.|k| + 8 u |scores|, which is the relative error of its exp.
"""
import math

import pytest
import torch

from trident_amd import _lib, encoder
from test_gpu_encoder import F64, TINY, TYPES, U, gen, randn, u, within

pytestmark = pytest.mark.gpu


def sequences(layout, lens, slots=None):
    """(leading dimensions, first row of each sequence)"""
    if layout == "padded":
        slots = slots or max(lens)
        return (len(lens), slots), [i * slots for i in range(len(lens))]
    return (sum(lens),), [sum(lens[:i]) for i in range(len(lens))]


def reference(q, k, v, lens, starts, causal, scale, grad=None):
    """dict of name -> (value, bound), flat over the leading dimensions."""
    dtype, D = q.dtype, q.shape[-1]
    Un, tiny = U.get(dtype, 0.0), TINY.get(dtype, 0.0)
    held = {torch.float16: 2.0 ** -32}.get(dtype, 0.0)  # of the largest: what float16's small exponents lose of P
    q, k, v = (t.to(F64).flatten(0, -3) for t in (q, k, v))
    Hq, Hkv = q.shape[1], k.shape[1]
    G = Hq // Hkv
    res = {n: (torch.zeros_like(t), torch.zeros_like(t)) for n, t in
           (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    if grad is not None:
        grad = grad.to(F64).flatten(0, -3)
    for m, a in zip(lens, starts):
        if m == 0:
            continue
        at = slice(a, a + m)
        hidden = torch.ones((m, m), dtype=torch.bool, device=q.device).triu(1) if causal else None
        for h in range(Hq):
            Q, K, V = q[at, h], k[at, h // G], v[at, h // G]
            s = scale * Q @ K.t()
            size = scale * Q.abs() @ K.abs().t()
            if causal:
                s = s.masked_fill(hidden, -math.inf)
                size = size.masked_fill(hidden, 0.0)
            p = torch.softmax(s, 1)
            top = s.masked_fill(s.isinf(), 0.0).abs().amax(1, keepdim=True)
            E = ((D + 8) * u * size + 8 * u * top).amax(1, keepdim=True)
            out = p @ V
            b_out = (Un + 2 * E + (m + 12) * u) * (p @ V.abs()) + held * V.abs().sum(0) + Un * out.abs() + tiny
            res["out"][0][at, h], res["out"][1][at, h] = out, b_out
            if grad is None:
                continue
            dO = grad[at, h]
            n = m * G
            rel = 3 * E + (m + 12) * u  # of P made again from lse
            dv = p.t() @ dO
            res["dv"][0][at, h // G] += dv
            res["dv"][1][at, h // G] += (Un + n * u) * (p.t() @ dO.abs()) + (p * rel).t() @ dO.abs() + \
                2.0 ** -40 * dO.abs().sum(0) * (dtype is torch.float16)
            dP = dO @ V.t()
            delta = (dO * out).sum(1, keepdim=True)
            e_delta = (dO.abs() * (b_out + D * u * out.abs())).sum(1, keepdim=True)
            dS = p * (dP - delta)
            e_dS = p * (rel * (dP - delta).abs() + (D + 2) * u * (dO.abs() @ V.abs().t()) + e_delta) + \
                (Un + (n + 4) * u) * dS.abs()
            # in float16 dS is held times a power of two that brings its column's largest so far to 2^14 or more
            # (2^15 at most): what lies 2^28 below the largest is lost in part
            if dtype is torch.float16:
                e_dS = e_dS + 2.0 ** -38 * dS.abs().max()
            res["dq"][0][at, h] = scale * dS @ K
            res["dq"][1][at, h] = scale * e_dS @ K.abs()
            res["dk"][0][at, h // G] += scale * dS.t() @ Q
            res["dk"][1][at, h // G] += scale * e_dS.t() @ Q.abs()
    for n in ("dq", "dk", "dv"):
        value, bound = res[n]
        bound += Un * value.abs() + tiny
        res[n] = value, bound
    return res


def check(q, k, v, lens, layout, causal, grad=None, scale=None, wide=False, slots=None):
    _, starts = sequences(layout, lens, slots)
    where = torch.tensor(lens if layout == "padded" else starts + [sum(lens)], device=q.device,
                         dtype=torch.int64 if wide else torch.int32)
    how = dict(causal=causal, scale=scale, **{"lengths" if layout == "padded" else "offsets": where})
    ref = reference(q, k, v, lens, starts, causal, 1 / math.sqrt(q.shape[-1]) if scale is None else scale, grad)
    got = dict(out=encoder.attention(q, k, v, **how))
    if grad is not None:
        out, lse = encoder.attention_forward(q, k, v, **how)
        assert torch.equal(out, got["out"])
        got["dq"], got["dk"], got["dv"] = encoder.attention_grad(grad, q, k, v, out, lse, **how)
    for n, t in got.items():
        assert t.shape == (k.shape if n in ("dk", "dv") else q.shape) and t.dtype == q.dtype
        within(t.flatten(0, -3), *ref[n], what=n)
    return got


def operands(seed, dtype, lead, Hq, Hkv, D, by=1.0):
    g = gen(seed)
    q, k, v, grad = (randn(g, *lead, H, D) for H in (Hq, Hkv, Hkv, Hq))
    return (by * q).to(dtype), k.to(dtype), v.to(dtype), (1e-2 * grad).to(dtype)


LENGTHS = [[1], [2, 1], [31, 32, 33], [63, 64, 65], [127, 128, 129, 0, 1], [300, 0, 0, 17], [1] * 70, [515]]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_packed(dev, dtype, lens, causal):
    lead, _ = sequences("packed", lens)
    q, k, v, grad = operands(sum(lens), dtype, lead, 4, 2, 64)
    check(q, k, v, lens, "packed", causal, grad)


@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_head_sizes(dev, dtype, D):
    lens = [70, 1, 130]
    q, k, v, grad = operands(D, dtype, (201,), 2, 1, D)
    check(q, k, v, lens, "packed", D % 16 == 0, grad)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 5), (6, 3), (8, 1), (12, 4)])
def test_groups(dev, Hq, Hkv):
    for dtype in TYPES:
        q, k, v, grad = operands(Hq, dtype, (150,), Hq, Hkv, 32)
        check(q, k, v, [100, 50], "packed", True, grad)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,slots", [([5, 0, 16], 16), ([40, 1, 33, 40], 40), ([100, 200, 0, 130], 200), ([7], 300)],
                         ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_padded(dev, dtype, lens, slots, causal):
    q, k, v, grad = operands(slots, dtype, (len(lens), slots), 4, 4, 48)
    for b, m in enumerate(lens):  # what empty slots hold is never used
        for t in (q, k, v, grad):
            t[b, m:] = math.nan
    got = check(q, k, v, lens, "padded", causal, grad, wide=True, slots=slots)
    for t in got.values():
        for b, m in enumerate(lens):
            assert (t[b, m:] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_outside_the_sequences(dev, dtype):
    """Rows before the first offset and after the last: NaN there reaches nothing, and they get zeros."""
    lens, before, after = [33, 70, 1], 5, 140
    T = before + sum(lens) + after
    q, k, v, grad = operands(3, dtype, (T,), 4, 2, 64)
    live = slice(before, before + sum(lens))
    for t in (q, k, v, grad):
        t[:before] = math.nan
        t[live.stop:] = math.inf
    offsets = torch.tensor([5, 38, 108, 109], dtype=torch.int32, device=dev)
    out, lse = encoder.attention_forward(q, k, v, offsets)
    grads = encoder.attention_grad(grad, q, k, v, out, lse, offsets)
    ref = reference(q[live], k[live], v[live], lens, [0, 33, 103], False, 0.125, grad[live])
    for t, n in zip((out, *grads), ("out", "dq", "dk", "dv")):
        within(t[live], *ref[n], what=n)
        assert (t[:before] == 0).all() and (t[live.stop:] == 0).all()


def test_offsets_outside_the_rows_are_brought_inside(dev):
    q, k, v, grad = operands(4, torch.bfloat16, (100,), 2, 2, 32)
    for bad, good in (([-5, 60, 1 << 40], [0, 60, 100]), ([0, 100, 100, 200], [0, 100, 100, 100])):
        a = torch.tensor(bad, dtype=torch.int64, device=dev)
        b = torch.tensor(good, dtype=torch.int32, device=dev)
        assert torch.equal(encoder.attention(q, k, v, a), encoder.attention(q, k, v, b))
    # descending ones are not sequences: whatever comes out, nothing outside the tensors is touched
    encoder.attention(q, k, v, torch.tensor([90, 10, 50, -7, 300, 2], device=dev))
    lengths = torch.tensor([-3, 1 << 40], device=dev)
    p = [t.view(2, 50, 2, 32) for t in (q, k, v)]
    got = encoder.attention(*p, lengths=lengths)
    assert (got[0] == 0).all() and torch.equal(got[1], encoder.attention(*(t[1] for t in p)))
    torch.cuda.synchronize()


@pytest.mark.parametrize("n", [63, 64, 200, 5000])
def test_many_short_sequences(dev, n):
    """More sequences than one search step looks at."""
    g = gen(n)
    lens = torch.randint(0, 9, (n,), generator=g, device=dev)
    lens[0], lens[n // 2] = 100, 40
    lens = lens.tolist()
    q, k, v, grad = operands(n, torch.float16, (sum(lens),), 2, 1, 16)
    check(q, k, v, lens, "packed", n % 2 == 0, grad)


@pytest.mark.parametrize("dtype", TYPES)
def test_parts_of_one_projection_and_other_strides(dev, dtype):
    g = gen(5)
    qkv = randn(g, 130, 8, 64, dtype=dtype)
    grad = (1e-2 * randn(g, 130, 4, 64)).to(dtype)
    check(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], [100, 30], "packed", True, grad)
    heads_first = [randn(g, H, 130, 64, dtype=dtype).transpose(0, 1) for H in (4, 2, 2)]
    check(*heads_first, [100, 30], "packed", False, grad.transpose(0, 1).contiguous().transpose(0, 1))
    odd = [randn(g, 130, H, 67, dtype=dtype)[..., 1:65] for H in (4, 2, 2)]  # copied
    check(*odd, [100, 30], "packed", False, grad)
    shared = randn(g, 130, 1, 64, dtype=dtype).expand(130, 2, 64)  # one head for both
    check(qkv[:, :4], shared, shared, [100, 30], "packed", False, grad)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_falling_scores(dev, dtype):
    """Scores up to hundreds, the largest key last or first: the reference value moves."""
    for by, order in ((20.0, 1), (20.0, -1), (1e-3, 1)):
        q, k, v, grad = operands(6, dtype, (400,), 2, 2, 64, by=by)
        k = (k * torch.linspace(0.1, 1.0, 400, device=dev)[::order][:, None, None] if order == 1 else
             k * torch.linspace(1.0, 0.1, 400, device=dev)[:, None, None]).to(dtype)
        check(q, k, v, [400], "packed", True, grad)


def test_scores_far_below_zero(dev):
    """All scores near -2000: no row is empty, whatever its exp would be."""
    g = gen(7)
    q = torch.ones((200, 1, 32), device=dev)
    k = -60.0 - randn(g, 200, 1, 32).abs()
    v = randn(g, 200, 1, 32)
    check(q, k, v, [200], "packed", True, scale=1.0)


def test_small_gradients_in_float16(dev):
    """dS of a long row with small gradients is far below float16's least normal number."""
    q, k, v, grad = operands(8, torch.float16, (3000,), 1, 1, 64)
    check(q, k, v, [3000], "packed", False, grad=(grad.float() * 0.1).half())


@pytest.mark.parametrize("dtype", TYPES)
def test_one_token_is_its_value(dev, dtype):
    q, k, v, _ = operands(9, dtype, (1,), 3, 3, 64)
    assert torch.equal(encoder.attention(q, k, v), v)


# Rows that share a block of 32 with such a token are summed row by row, so their bits are not those of the same call
# without it: a sum's order is free within the bound of n u times the magnitudes, which `reference` has.


def test_values_that_are_not_finite(dev):
    """They show in every row that sees them and, causal, in none before their own."""
    for dtype in TYPES:
        for causal in (False, True):
            for bad in (math.nan, math.inf):
                q, k, v, _ = operands(10, dtype, (300,), 2, 2, 64)
                clean = encoder.attention(q, k, v, causal=causal)
                ref, bound = reference(q, k, v, [300], [0], causal, 0.125)["out"]
                v[210, 0, 5] = bad
                got = encoder.attention(q, k, v, causal=causal)
                first = 210 if causal else 0
                assert torch.equal(got[:, 1], clean[:, 1]) and torch.equal(got[:first // 32 * 32], clean[:first // 32 * 32])
                within(got[:first], ref[:first], bound[:first])
                assert not got[first:, 0, 5].isfinite().any()
                within(got[:, 0, 6:], ref[:, 0, 6:], bound[:, 0, 6:])
                k[100, 1, 3] = math.nan
                got = encoder.attention(q, k, v, causal=causal)
                first = 100 if causal else 0
                within(got[:first, 1], ref[:first, 1], bound[:first, 1])
                assert got[first:, 1].isnan().all()


def test_gradients_of_values_that_are_not_finite(dev):
    """Causal: a token's key or gradient reaches no gradient that the formula keeps it from."""
    for dtype in TYPES:
        q, k, v, grad = operands(11, dtype, (300,), 1, 1, 64)

        def run(*t):
            q, k, v, grad = t
            out, lse = encoder.attention_forward(q, k, v, causal=True)
            return encoder.attention_grad(grad, q, k, v, out, lse, causal=True)

        ref = reference(q, k, v, [300], [0], True, 0.125, grad)
        bad = grad.clone()
        bad[100] = math.nan  # keys past 100 are hidden from it
        dq, dk, dv = run(q, k, v, bad)
        for t, n, keep in ((dk, "dk", slice(101, 300)), (dv, "dv", slice(101, 300)), (dq, "dq", slice(0, 100)),
                           (dq, "dq", slice(101, 300))):
            within(t[keep], ref[n][0][keep], ref[n][1][keep], what=n)
        assert dq[100].isnan().all() and dv[:101].isnan().all()
        bad = k.clone()
        bad[100] = math.inf
        dq, dk, dv = run(q, bad, v, grad)
        within(dq[:100], ref["dq"][0][:100], ref["dq"][1][:100])
        bad = q.clone()
        bad[100] = math.nan
        dq, dk, dv = run(bad, k, v, grad)
        for t, n in ((dk, "dk"), (dv, "dv")):
            within(t[101:], ref[n][0][101:], ref[n][1][101:], what=n)


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 1e-4), (torch.float16, 2e-2), (torch.bfloat16, 1e-1)])
def test_autograd_against_differences(dev, dtype, bound):
    """The derivative along random directions against differences of the float64 formula: the directions' part of the
    relative error is the roundings of a few hundred elements, far inside the bound."""
    q, k, v, grad = operands(12, dtype, (70,), 4, 2, 32)
    offsets = torch.tensor([0, 50, 70], dtype=torch.int32, device=dev)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = encoder.attention(*leaves, offsets, causal=True)
    out.backward(grad)

    def value(*t):
        return (reference(*t, [50, 20], [0, 50], True, 32 ** -0.5)["out"][0] * grad.to(F64)).sum()

    g = gen(13)
    for i, t in enumerate(leaves):
        d, h = randn(g, *t.shape).to(F64), 1e-5
        at = [x.detach().to(F64) for x in leaves]
        far = [[x + (h * sign * d if i == j else 0) for j, x in enumerate(at)] for sign in (1, -1)]
        want = (value(*far[0]) - value(*far[1])) / (2 * h)
        got = (t.grad.to(F64) * d).sum()
        size = (t.grad.to(F64).square().sum().sqrt() * d.square().mean().sqrt())
        assert abs(got - want) <= bound * size + 1e-9, (i, float(got), float(want))


def test_autograd_needs(dev):
    q, k, v, grad = operands(14, torch.bfloat16, (40,), 2, 2, 32)
    v.requires_grad_()
    out = encoder.attention(q, k, v)
    (dv,) = torch.autograd.grad(out, v, grad)
    o, lse = encoder.attention_forward(q, k, v)
    assert torch.equal(dv, encoder.attention_grad(grad, q, k, v, o, lse)[2])
    with torch.no_grad():
        assert not encoder.attention(q, k, v).requires_grad


def test_same_bits_each_time_and_on_another_stream(dev):
    q, k, v, grad = operands(15, torch.bfloat16, (1000,), 8, 2, 64)
    offsets = torch.tensor([0, 10, 600, 1000], device=dev)

    def run():
        out, lse = encoder.attention_forward(q, k, v, offsets, causal=True)
        return (out, *encoder.attention_grad(grad, q, k, v, out, lse, offsets, causal=True))

    want = run()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
        with torch.cuda.stream(st):
            got = run()
        st.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_and_replayed(dev):
    """A graph whose offsets change between replays; another program's work between them."""
    q, k, v, grad = operands(16, torch.float16, (700,), 4, 2, 64)
    offsets = torch.tensor([0, 300, 700], dtype=torch.int32, device=dev)

    def run():
        out, lse = encoder.attention_forward(q, k, v, offsets)
        return (out, *encoder.attention_grad(grad, q, k, v, out, lse, offsets))

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        got = run()
    for mid in (300, 0, 699, 128, 700):
        offsets[1] = mid
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), mid


def test_far_rows(dev):
    """Rows past 2^31 bytes of a tensor."""
    D, T = 128, 600_000
    q = torch.zeros((T, 16, D), dtype=torch.bfloat16, device=dev)  # 2.4 GB
    k = torch.zeros((T, 16, D), dtype=torch.bfloat16, device=dev)
    v = torch.zeros((T, 16, D), dtype=torch.bfloat16, device=dev)
    tail = operands(17, torch.bfloat16, (300,), 16, 16, D)
    for t, x in zip((q, k, v), tail):
        t[-300:] = x
    offsets = torch.tensor([T - 300, T - 300, T], device=dev)  # the rows before are no sequence's
    got = encoder.attention(q, k, v, offsets)
    assert torch.equal(got[-300:], encoder.attention(*tail[:3]))
    assert (got[:-300] == 0).all()
