"""Scratch memory of a call that is being captured into a graph is the graph's own: a later call that needs
more replaces the stream's workspace, and the graph's replays must not write to what that was."""
import contextlib
import types

import pytest
import torch

from trident_amd import encoder, ext

CPU = torch.device("cpu")


@pytest.fixture
def fake_stream(monkeypatch):
    """A stream without a GPU: its workspace is host memory; ``capturing`` is set by the test."""
    st = types.SimpleNamespace(cuda_stream=7, device_index=0, capturing=False)
    for at in (ext, encoder):
        monkeypatch.setattr(at, "_raw_stream", lambda index: 7, raising=False)
        monkeypatch.setattr(at, "_current_device", lambda: 0, raising=False)
    monkeypatch.setattr(ext, "_current_capturing", lambda: st.capturing, raising=False)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: st)
    monkeypatch.setattr(ext, "_ws_cache", {})
    return st


def test_the_encoders_calls(fake_stream, monkeypatch):
    used = []
    monkeypatch.setattr(encoder, "_call", lambda index, name, *args: used.append(args[-2:]))
    encoder._call_ws(CPU, 0, "f", 5000)
    slot = ext._ws_cache[(CPU, 7)]
    kept = slot.buf
    assert used[-1] == (kept.data_ptr(), kept.numel())
    fake_stream.capturing = True
    for nbytes in (5000, 3 << 20):  # less and more than the workspace has
        encoder._call_ws(CPU, 0, "f", nbytes)
        at, size = used[-1]
        assert size >= nbytes and at != kept.data_ptr() and slot.buf is kept
    fake_stream.capturing = False
    encoder._call_ws(CPU, 0, "f", 5000)
    assert used[-1] == (kept.data_ptr(), kept.numel())


def test_a_first_call_under_capture_leaves_no_workspace(fake_stream, monkeypatch):
    """What a capture allocates goes with its graph, so it never becomes the stream's workspace."""
    monkeypatch.setattr(encoder, "_call", lambda index, name, *args: None)
    fake_stream.capturing = True
    encoder._call_ws(CPU, 0, "f", 5000)
    assert ext._ws_cache[(CPU, 7)].buf is None


def test_the_searches(fake_stream):
    slot = ext._Workspace()
    kept = ext._scratch(slot, CPU, 100, fake_stream)
    assert slot.buf is kept
    fake_stream.capturing = True
    own = ext._scratch(slot, CPU, 100, fake_stream)
    assert own.numel() >= 100 and own.data_ptr() != kept.data_ptr() and slot.buf is kept


# ---------------------------------------------------------------------------------------------
# on a GPU


def capture(st, f):
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        f()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        out = f()
    return graph, out


def operands(seed, n=20_000, V=3000, D=64):
    g = torch.Generator(device="cuda:0").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda:0")  # noqa: E731
    ids = torch.randint(-1, V, (n,), generator=g, device="cuda:0")
    x, gamma = r(500, 4100), r(4100)
    wq = encoder.quantize_fp8(r(300, 4100))

    def f():
        y, mean, rstd = encoder.layer_norm_forward(x, gamma)
        return (encoder.embedding_grad(grad, ids, V), *encoder.layer_norm_grad(y, x, gamma, mean, rstd),
                encoder.fp8_linear(x, wq))

    grad = r(n, D)
    return f


@pytest.mark.gpu
def test_replays_after_the_workspace_was_outgrown(dev):
    st = torch.cuda.Stream()
    f = operands(1)
    graph, out = capture(st, f)
    want = [t.clone() for t in f()]
    for i in range(3):
        with torch.cuda.stream(st):  # needs far more than the capture did: the workspace is replaced
            big = operands(2 + i, n=300_000 << i, V=100_000, D=32)
            big()
        torch.cuda.synchronize()
        fresh = [torch.full((1 << 20,), 7.0, device=dev) for _ in range(64)]  # takes what was given back
        torch.cuda.synchronize()
        for t in out:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        assert all(bool((t == 7.0).all()) for t in fresh), i
        del fresh, big


@pytest.mark.gpu
def test_two_graphs_of_one_stream_at_once(dev):
    st, other = torch.cuda.Stream(), torch.cuda.Stream()
    f, h = operands(11), operands(12)
    (g1, out1), (g2, out2) = capture(st, f), capture(st, h)
    want1, want2 = [t.clone() for t in f()], [t.clone() for t in h()]
    torch.cuda.synchronize()
    for i in range(5):
        with torch.cuda.stream(st):
            g1.replay()
        with torch.cuda.stream(other):
            g2.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out1, want1)), i
        assert all(torch.equal(a, b) for a, b in zip(out2, want2)), i


@pytest.mark.gpu
def test_a_captured_search_after_the_workspace_was_outgrown(dev):
    from trident_amd import datagen
    from trident_amd.clustering import train_clustering
    from trident_amd.index import SharedClusterStorage, TridentV4Index

    xb, xq = datagen.cfg2(N=20_000, D=128, B=64, n_centers=64, seed=7)
    cen, lid, r, mean64, R64, _ = train_clustering(xb, 64, seed=0, niter=5)
    storage = SharedClusterStorage(xb.numpy(), lid, r, 64, device=dev)
    ix = TridentV4Index(storage, cen, mean64, R64, tile_size=64, device=dev, max_batch=2048, max_nprobe=16, k=10)
    few, many = xq[:8].to(dev).contiguous(), xq.to(dev).repeat(32, 1).contiguous()
    want = [t.clone() for t in ix.search(few, 8, mode=10)[:2]]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    graph, out = capture(st, lambda: ix.search(few, 8, mode=10)[:2])
    for i in range(3):
        with torch.cuda.stream(st):
            ix.search(many, 16, mode=10)
        torch.cuda.synchronize()
        fresh = [torch.full((1 << 20,), 7.0, device=dev) for _ in range(64)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        assert all(bool((t == 7.0).all()) for t in fresh), i
        del fresh
