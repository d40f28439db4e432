"""The transformer layer's operators together, as the example's encoder runs them: lookup, layer norm, rotation, attention
over a padded batch, gated feed-forward, mean, and back; against the same formulas in float64 by torch's autograd."""
import importlib.util
import math
import os

import pytest
import torch

from trident_amd import encoder
from test_gpu_encoder import F64, gen, randn

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_encoder.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("train_encoder", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def padded_ids(g, B, L, V):
    ids = torch.randint(0, V, (B, L), generator=g, device="cuda:0")
    lengths = torch.randint(L // 2, L + 1, (B, 1), generator=g, device="cuda:0")
    ids[torch.arange(L, device="cuda:0")[None, :] >= lengths] = -1
    return ids


def plain_pooled(model, ids, table, gamma, beta, params):
    """The model's formula in float64; ``params``: each layer's in the order of Layer.parameters()."""
    live = ids >= 0
    x = torch.where(live[..., None], table[ids.clamp(min=0)] * model.scale, 0.0)

    def norm(x, w, b=0.0):
        c = x - x.mean(-1, keepdim=True)
        return c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5) * w + b

    B, L = ids.shape
    for layer, (n0, n1, wqkv, wmix, wg, wu, wd) in zip(model.layers, params):
        H, D = layer.heads, layer.head_dim
        qkv = (norm(x, n0) @ wqkv.t()).view(B, L, 3, H, D)
        t = torch.arange(L, device=ids.device)[:, None, None] * layer.frequencies
        c, s = torch.cos(t), torch.sin(t)

        def turn(y):
            a, b = y[..., :D // 2], y[..., D // 2:]
            return torch.cat((a * c - b * s, a * s + b * c), -1)

        q, k, v = (y.transpose(1, 2) for y in (turn(qkv[:, :, 0]), turn(qkv[:, :, 1]), qkv[:, :, 2]))
        scores = (q @ k.transpose(-1, -2) / math.sqrt(D)).masked_fill(~live[:, None, None, :], -math.inf)
        o = (torch.softmax(scores, -1) @ v).transpose(1, 2).reshape(B, L, H * D)
        x = x + torch.where(live[..., None], o, 0.0) @ wmix.t()
        h = norm(x, n1)
        x = x + (torch.nn.functional.silu(h @ wg.t()) * (h @ wu.t())) @ wd.t()
    x = norm(x, gamma, beta)
    return (x * live[..., None]).sum(1) / live.sum(1, keepdim=True)


@pytest.mark.parametrize("dim,heads,L,B", [(64, 2, 17, 5), (128, 4, 40, 8), (96, 4, 130, 3)])
def test_values_and_gradients(dev, example, dim, heads, L, B):
    g = gen(dim)
    model = example.TextEncoder(300, dim, 32, g, dev, layers=2, heads=heads)
    ids = padded_ids(g, B, L, 300)
    out = model.pooled(ids)
    grad = randn(g, *out.shape)
    out.backward(grad)
    leaves = [model.table, model.gamma, model.beta] + [p for layer in model.layers for p in layer.parameters()]
    exact = [p.detach().to(F64).requires_grad_() for p in leaves]
    ref = plain_pooled(model, ids, *exact[:3], [exact[3 + 7 * i:10 + 7 * i] for i in range(2)])
    ref.backward(grad.to(F64))
    # float32 throughout: a few hundred roundings of 2^-24 of the values' own size on each path, far below 1e-4
    def close(got, want):
        assert (got.to(F64) - want).square().mean().sqrt() <= 1e-4 * want.square().mean().sqrt()
        return True

    assert close(out, ref)
    for p, e in zip(leaves, exact):
        assert close(p.grad, e.grad)


def test_empty_slots_do_not_matter(dev, example):
    """More empty slots give the same vectors, and slots a gradient that is zero."""
    g = gen(1)
    model = example.TextEncoder(300, 64, 32, g, dev, layers=1, heads=2)
    ids = padded_ids(g, 6, 30, 300)
    more = torch.cat((ids, torch.full((6, 45), -1, device=dev)), 1)
    with torch.no_grad():
        a, b = model.pooled(ids), model.pooled(more)
    assert (a - b).abs().max() <= 1e-5 * a.abs().max()


def test_example_runs_with_layers(dev, example):
    args = ["--vocab", "2000", "--dim", "64", "--out", "96", "--passages", "1500", "--length", "24", "--steps", "6",
            "--batch", "64", "--nlist", "8", "--nprobe", "8", "--layers", "2"]
    got = example.main(args)
    assert math.isfinite(got["first"]) and math.isfinite(got["last"])
    assert got["recall"] > 0.999, got  # every list is probed


def test_forward_captured_and_replayed(dev, example):
    """A query batch through the encoder in a graph: replays follow the ids."""
    g = gen(2)
    model = example.TextEncoder(500, 128, 64, g, dev, layers=2, heads=2)
    model.freeze()
    ids = padded_ids(g, 4, 16, 500)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        model.encode(ids)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        z = model.encode(ids)
    for i in range(4):
        ids.copy_(padded_ids(gen(10 + i), 4, 16, 500))
        want = model.encode(ids)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, want), i


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_packed_layer_in_16_bits(dev, dtype):
    """Packed sequences, causal, grouped heads: rotated in place, attention and a gated block, against the padded call on the
    same sequences one by one (the same kernels, so the same bits)."""
    g = gen(3)
    lens, Hq, Hkv, D = [1, 70, 33, 128, 5], 4, 2, 64
    offsets = torch.tensor([0, 1, 71, 104, 232, 237], device=dev)
    qkv = randn(g, 237, Hq + 2 * Hkv, D, dtype=dtype)
    wg, wu = (randn(g, 300, Hq * D, dtype=dtype) / 16 for _ in range(2))
    positions = torch.cat([torch.arange(m, device=dev) for m in lens])
    f = encoder.rotary_frequencies(D, device=dev)

    def run(x, p, offsets):
        x = x.clone()
        encoder.rotary(x[:, :Hq + Hkv], f, p, out=x[:, :Hq + Hkv])
        o = encoder.attention(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], offsets, causal=True)
        return o, encoder.gated_linear(o.flatten(1), wg, wu)

    o, h = run(qkv, positions, offsets)
    for m, a in zip(lens, offsets.tolist()):
        one, _ = run(qkv[a:a + m], positions[a:a + m], None)
        assert torch.equal(o[a:a + m], one)
    assert h.isfinite().all()
