"""The transformer layer's entry points on the CPU (no kernel launches): struct layouts, argument checks that come before any
launch, workspace sizes, and the Python boundary's refusals."""
import ctypes
import os
import subprocess

import pytest
import torch

from trident_amd import _lib, encoder

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "trident_hip.h")
STRUCTS = {"TridentAttention": _lib.TridentAttention, "TridentGated": _lib.TridentGated}
P = 256  # stands for a device address: never followed here


def test_struct_layout_matches_header(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text(
        '#include <stdio.h>\n#include <stddef.h>\n#include "trident_hip.h"\nint main(void){\n'
        + "".join(f'printf("{s} {f} %zu\\n", offsetof({s}, {f}));\n' for s, c in STRUCTS.items() for f, _ in c._fields_)
        + "".join(f'printf("size {s} %zu\\n", sizeof({s}));\n' for s in STRUCTS) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        a, b, c = line.split()
        got = ctypes.sizeof(STRUCTS[b]) if a == "size" else getattr(STRUCTS[a], b).offset
        assert got == int(c), line


def refused(rc, code, text):
    assert rc == code, (rc, _lib.lib().trident_last_error())
    assert text in _lib.lib().trident_last_error().decode(), _lib.lib().trident_last_error()


def test_rotary_arguments():
    L = _lib.lib()

    def call(x=P, dtype=0, tokens=4, heads=2, D=8, pairs=4, f=P, period=4, amplitude=1.0, out=P):
        return L.trident_rotary(x, dtype, tokens, heads, D, 16, 8, f, pairs, P, 0, period, 0, amplitude, 0, out, 16, 8, None)

    refused(call(dtype=5), 1, "dtype=5")
    refused(call(pairs=5), 1, "bad sizes")
    refused(call(tokens=-1), 1, "bad sizes")
    refused(call(tokens=1 << 31), 1, "bad sizes")
    refused(call(period=0), 1, "bad sizes")
    refused(call(D=1 << 13, pairs=2000), 2, "2000 pairs")
    refused(call(amplitude=float("nan")), 1, "amplitude")
    refused(call(x=None), 1, "NULL")
    refused(call(f=None), 1, "NULL")
    assert call(tokens=0, x=None, out=None) == 0


def attention(**kw):
    a = dict(q=P, k=P, v=P, out=P, lse=None, grad=None, dq=None, dk=None, dv=None, offsets=P, lengths=None, q_row=128, q_head=64,
             k_row=128, k_head=64, v_row=128, v_head=64, rows=1000, sequences=3, slots=0, q_heads=2, kv_heads=2, head_dim=64,
             scale=0.125, dtype=2, ids64=0, causal=0)
    a.update(kw)
    return _lib.TridentAttention(**a)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=3), 1, "dtype=3"), (dict(rows=-1), 1, "bad sizes"), (dict(rows=1 << 31), 1, "bad sizes"),
    (dict(sequences=-1), 1, "bad sizes"), (dict(kv_heads=0), 1, "bad sizes"), (dict(q_heads=3), 1, "bad sizes"),
    (dict(head_dim=0), 1, "bad sizes"), (dict(head_dim=60), 2, "head_dim=60"), (dict(head_dim=136), 2, "head_dim=136"),
    (dict(scale=0.0), 1, "scale"), (dict(scale=float("nan")), 1, "scale"), (dict(q_row=63), 1, "stride"),
    (dict(k_head=4), 1, "stride"), (dict(v_row=1 << 24), 1, "stride"), (dict(q=None), 1, "NULL"),
    (dict(offsets=None), 1, "NULL"), (dict(lengths=P), 1, "do not go"), (dict(slots=7), 1, "do not go"),
    (dict(offsets=None, slots=300, lengths=P), 1, "do not go"), (dict(k=P + 8), 1, "aligned")])
def test_attention_arguments(change, code, text):
    L = _lib.lib()
    a = attention(**change)
    refused(L.trident_attention(ctypes.byref(a), None), code, text)
    a = attention(lse=P, grad=P, dq=P, dk=P, dv=P, **change)
    assert L.trident_attention_grad_workspace_bytes(ctypes.byref(a)) == 0
    refused(L.trident_attention_grad(ctypes.byref(a), P, 1 << 40, None), code, text)


def test_attention_grad_arguments():
    L = _lib.lib()
    whole = dict(lse=P, grad=P, dq=P, dk=P, dv=P)
    for name in whole:
        a = attention(**{**whole, name: None})
        refused(L.trident_attention_grad(ctypes.byref(a), P, 1 << 40, None), 1, "NULL")
    a = attention(**whole)
    need = L.trident_attention_grad_workspace_bytes(ctypes.byref(a))
    assert need >= 1000 * 2 * 4
    refused(L.trident_attention_grad(ctypes.byref(a), P, need - 1, None), 3, str(need))
    refused(L.trident_attention_grad(ctypes.byref(a), P + 8, need, None), 3, "aligned")
    refused(L.trident_attention_grad(ctypes.byref(a), None, need, None), 3, str(need))
    # few key tiles: their queries are shared, and the sums of every share have a place
    a = attention(rows=2048, sequences=1, q_heads=8, kv_heads=1, q_row=512, **whole)
    many = L.trident_attention_grad_workspace_bytes(ctypes.byref(a))
    assert many >= 2048 * 8 * 4 + 2 * 2 * 2048 * 64 * 4
    for nothing in (attention(rows=0, q=None), attention(rows=0, sequences=0)):
        assert L.trident_attention(ctypes.byref(nothing), None) == 0
        assert L.trident_attention_grad(ctypes.byref(nothing), None, 0, None) == 0
    refused(L.trident_attention(None, None), 1, "NULL")
    refused(L.trident_attention_grad(None, None, 0, None), 1, "NULL")


def gated(**kw):
    a = dict(x=P, gate_weight=P, up_weight=P, h=P, gate=P, up=P, grad=P, dx=P, dgate_weight=P, dup_weight=P, M=100, N=64, K=32,
             ld_x=32, ld_gate=32, ld_up=32, ld_grad=64, dtype=2, activation=0)
    a.update(kw)
    return _lib.TridentGated(**a)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=9), 1, "dtype=9"), (dict(activation=3), 1, "activation=3"), (dict(M=-1), 1, "bad sizes"),
    (dict(K=0), 1, "bad sizes"), (dict(ld_x=31), 1, "bad sizes"), (dict(ld_up=31), 1, "bad sizes"),
    (dict(N=1 << 22), 1, "bad sizes"), (dict(x=None), 1, "NULL"), (dict(up=None), 1, "NULL")])
def test_gated_arguments(change, code, text):
    L = _lib.lib()
    a = gated(**change)
    refused(L.trident_gated_linear(ctypes.byref(a), P, 1 << 40, None), code, text)
    refused(L.trident_gated_linear_grad(ctypes.byref(a), P, 1 << 40, None), code, text)


def test_gated_workspaces():
    L = _lib.lib()
    assert L.trident_gated_linear_workspace_bytes(ctypes.byref(gated())) == 0  # taken as they are
    odd = gated(K=33, ld_x=33, ld_gate=40, ld_up=40)
    need = L.trident_gated_linear_workspace_bytes(ctypes.byref(odd))
    assert need >= (100 + 2 * 64) * 33 * 2
    refused(L.trident_gated_linear(ctypes.byref(odd), P, need - 1, None), 3, str(need))
    assert L.trident_gated_linear_workspace_bytes(ctypes.byref(gated(M=16, K=33, ld_x=33, ld_gate=33, ld_up=33))) == 0
    long = gated(K=8192, ld_x=8192, ld_gate=8192, ld_up=8192)  # shared sums
    assert L.trident_gated_linear_workspace_bytes(ctypes.byref(long)) >= 2 * 2 * 100 * 64 * 4
    need = L.trident_gated_linear_grad_workspace_bytes(ctypes.byref(gated()))
    assert need >= 2 * 100 * 64 * 2
    refused(L.trident_gated_linear_grad(ctypes.byref(gated()), P, need - 1, None), 3, str(need))
    refused(L.trident_gated_linear_grad(ctypes.byref(gated(ld_grad=63)), P, need, None), 1, "ld_grad")
    refused(L.trident_gated_linear_grad(ctypes.byref(gated(dup_weight=None)), P, need, None), 1, "without the other")
    refused(L.trident_gated_linear_grad(ctypes.byref(gated(M=0)), P, need, None), 1, "no rows")
    assert L.trident_gated_linear(ctypes.byref(gated(M=0)), None, 0, None) == 0
    refused(L.trident_gated_linear(None, None, 0, None), 1, "NULL")


def test_python_boundary_refuses_host_tensors():
    x, f = torch.zeros((4, 2, 8)), torch.zeros(4, dtype=torch.float64)
    w = torch.zeros((16, 8))
    for call in (lambda: encoder.rotary(x, f), lambda: encoder.attention(x, x, x), lambda: encoder.attention_forward(x, x, x),
                 lambda: encoder.attention_grad(x, x, x, x, x, x), lambda: encoder.gated_linear(x, w, w),
                 lambda: encoder.gated_linear_forward(x, w, w), lambda: encoder.gated_linear_grad(x, x, w, w, x, x)):
        with pytest.raises(_lib.TridentError, match="device tensor"):
            call()


@pytest.mark.parametrize("call,text", [
    (lambda: encoder.rotary_frequencies(7), "even"), (lambda: encoder.rotary_frequencies(0), "even"),
    (lambda: encoder.rotary_frequencies(8, base=0.0), "positive"), (lambda: encoder.rotary_frequencies(8, scaling="x"), "scaling"),
    (lambda: encoder.rotary_frequencies(8, scaling="turns", factor=2.0), "trained"),
    (lambda: encoder.rotary_frequencies(2, scaling="base", factor=2.0), "more than one pair")])
def test_frequencies_refused(call, text):
    with pytest.raises(_lib.TridentError, match=text):
        call()


@pytest.fixture
def on_gpu(monkeypatch):
    """Host tensors that say they are on the first GPU: what is refused here is refused before any launch."""
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(encoder, "_call", lambda *a: pytest.fail("launched"))
    monkeypatch.setattr(encoder, "_call_ws", lambda *a: pytest.fail("launched"))


def test_tensors_refused(on_gpu):
    t = lambda *s, d=torch.float32: torch.zeros(s, dtype=d)  # noqa: E731
    f = t(4, d=torch.float64)
    q, k = t(10, 4, 16), t(10, 2, 16)
    ids = torch.zeros(3, dtype=torch.int32)
    w, x, g32 = t(6, 8), t(5, 8), t(5, 6)
    cases = [
        (lambda: encoder.rotary(t(8), f), "heads, head_dim"), (lambda: encoder.rotary(q, f.float()), "float64"),
        (lambda: encoder.rotary(q, t(9, d=torch.float64)), "at most 8 pairs"),
        (lambda: encoder.rotary(q, f, ids), "positions"), (lambda: encoder.rotary(q, f, t(10)), "positions"),
        (lambda: encoder.rotary(q, f, out=k), "out must"), (lambda: encoder.rotary(q, f, out=q[:1].expand(10, 4, 16)), "one place"),
        (lambda: encoder.rotary(q.clone().requires_grad_(), f, out=q), "no gradient"),
        (lambda: encoder.rotary(q.double(), f), "float32, float16"),
        (lambda: encoder.attention(q, k, k[:, :1]), "alike"), (lambda: encoder.attention(q[0], k, k), "head_dim"),
        (lambda: encoder.attention(q, t(10, 3, 16), t(10, 3, 16)), "do not go"),
        (lambda: encoder.attention(t(10, 4, 12), t(10, 2, 12), t(10, 2, 12)), "multiple of 8"),
        (lambda: encoder.attention(t(10, 4, 136), t(10, 4, 136), t(10, 4, 136)), "up to 128"),
        (lambda: encoder.attention(q, k.half(), k), "k must be"), (lambda: encoder.attention(q, k, k, ids.float()), "offsets"),
        (lambda: encoder.attention(q, k, k, ids[:0]), "offsets"), (lambda: encoder.attention(q, k, k, lengths=ids), "packed"),
        (lambda: encoder.attention(t(2, 5, 4, 16), t(2, 5, 4, 16), t(2, 5, 4, 16), ids), "padded"),
        (lambda: encoder.attention(t(2, 5, 4, 16), t(2, 5, 4, 16), t(2, 5, 4, 16), lengths=ids), "lengths must"),
        (lambda: encoder.attention(q, k, k, scale=-1.0), "scale"),
        (lambda: encoder.attention_grad(k, q, k, k, q, t(4, 10)), "grad must"),
        (lambda: encoder.attention_grad(q, q, k, k, q, t(10, 4)), "lse must"),
        (lambda: encoder.gated_linear(x, w, w, "tanh"), "activation"), (lambda: encoder.gated_linear(x, w, w[:5]), "weights"),
        (lambda: encoder.gated_linear(x, w.half(), w.half()), "w_gate must"), (lambda: encoder.gated_linear(t(5, 7), w, w), "weights"),
        (lambda: encoder.gated_linear_grad(t(5, 5), x, w, w, g32, g32), "grad must"),
        (lambda: encoder.gated_linear_grad(g32, x, w, w, g32.half(), g32), "gate must"),
    ]
    for i, (call, text) in enumerate(cases):
        with pytest.raises(_lib.TridentError, match=text):
            call()
            pytest.fail(f"case {i} ({text}) was not refused")


def test_no_forward_mode_derivative(on_gpu):
    import torch.autograd.forward_ad as fwAD
    x, w = torch.zeros((5, 2, 8)), torch.zeros((6, 8))
    f = torch.zeros(4, dtype=torch.float64)
    with fwAD.dual_level():
        d = fwAD.make_dual(x, torch.ones_like(x))
        for call in (lambda: encoder.rotary(d, f), lambda: encoder.attention(d, x, x), lambda: encoder.attention_forward(x, d, x),
                     lambda: encoder.gated_linear(d, w, w), lambda: encoder.gated_linear_forward(d, w, w)):
            with pytest.raises(_lib.TridentError, match="forward-mode"):
                call()


def test_outputs_whose_elements_share_places():
    """_apart against the set of the places themselves."""
    for D in (1, 3):
        for heads in (1, 2, 4):
            for tokens in (2, 5):
                for head in range(1, 20):
                    for row in range(1, 20):
                        places = {t * row + h * head + d for t in range(tokens) for h in range(heads) for d in range(D)}
                        if encoder._apart(row, head if heads > 1 else D, tokens, heads, D):
                            assert len(places) == tokens * heads * D, (D, heads, tokens, head, row)
    for heads_within in (True, False):  # the usual orders are taken
        row, head = (12, 3) if heads_within else (3, 15)
        assert encoder._apart(row, head, 5, 4, 3)


def test_rotary_refuses_what_it_has_no_gradient_for(on_gpu):
    x, f = torch.zeros((5, 3, 8)), torch.zeros(4, dtype=torch.float64)
    with pytest.raises(_lib.TridentError, match="no gradient"):
        encoder.rotary(x, f.requires_grad_())
    out = torch.zeros(64).as_strided((5, 3, 8), (8, 8, 1))  # token t + 1 of one head is token t of the next
    with pytest.raises(_lib.TridentError, match="one place"):
        encoder.rotary(x, f.detach(), out=out)
