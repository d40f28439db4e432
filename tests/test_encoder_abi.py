"""The encoder's entry points on the CPU (no kernel launches): struct layouts, argument checks that come
before any launch, workspace sizes, and the Python boundary's refusals."""
import ctypes
import os
import subprocess

import pytest
import torch

from trident_amd import _lib, encoder

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "trident_hip.h")
STRUCTS = {"TridentAdamTensor": _lib.TridentAdamTensor, "TridentAdamState": _lib.TridentAdamState,
           "TridentAdamParams": _lib.TridentAdamParams}


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
    assert encoder._TABLE.itemsize == ctypes.sizeof(_lib.TridentAdamTensor)
    for name, field in zip(encoder._TABLE.names, _lib.TridentAdamTensor._fields_):
        assert encoder._TABLE.fields[name][1] == getattr(_lib.TridentAdamTensor, field[0]).offset


def refused(rc, code, text):
    assert rc == code, rc
    assert text in _lib.lib().trident_last_error().decode(), _lib.lib().trident_last_error()


P = 256  # stands for a device address: never followed here


def test_embedding_arguments():
    L = _lib.lib()
    refused(L.trident_embedding(P, 7, 10, 8, 8, P, 1, 4, 1.0, P, 8, None), 1, "dtype=7")
    refused(L.trident_embedding(P, 0, 10, 8, 7, P, 1, 4, 1.0, P, 8, None), 1, "bad sizes")
    refused(L.trident_embedding(P, 0, 0, 8, 8, P, 1, 4, 1.0, P, 8, None), 1, "bad sizes")
    refused(L.trident_embedding(P, 0, 10, 8, 8, P, 1, 1 << 31, 1.0, P, 8, None), 1, "bad sizes")
    refused(L.trident_embedding(None, 0, 10, 8, 8, P, 1, 4, 1.0, P, 8, None), 1, "NULL")
    assert L.trident_embedding(None, 0, 10, 8, 8, None, 1, 0, 1.0, None, 8, None) == 0
    assert L.trident_embedding_grad_workspace_bytes(1000, 50, 64) == 0
    need = L.trident_embedding_grad_workspace_bytes(10_000, 50, 64)
    assert need >= 51 * 8 + 10_000 * 8 + 2 * 313 * 64 * 4
    assert L.trident_embedding_grad_workspace_bytes(-1, 50, 64) == 0
    refused(L.trident_embedding_grad(P, 0, 64, P, 1, 10_000, 50, 64, 1.0, -1, P, 64, P, need - 1, None), 3, str(need))
    refused(L.trident_embedding_grad(P, 0, 64, P, 1, 10_000, 50, 64, 1.0, -1, None, 64, P, need, None), 1, "NULL")
    refused(L.trident_embedding_grad(P, 0, 63, P, 1, 10_000, 50, 64, 1.0, -1, P, 64, P, need, None), 1, "bad sizes")


def test_layer_norm_arguments():
    L = _lib.lib()
    refused(L.trident_layer_norm(P, 1, 4, 8, 8, P, P, 2, 1e-5, P, 8, None, None, None), 1, "weight_dtype=2")
    refused(L.trident_layer_norm(P, 0, 4, 0, 8, P, P, 0, 1e-5, P, 8, None, None, None), 1, "bad sizes")
    refused(L.trident_layer_norm(P, 0, 4, 8, 8, P, P, 0, float("nan"), P, 8, None, None, None), 1, "eps")
    refused(L.trident_layer_norm(P, 0, 4, 8, 8, P, P, 0, 1e-5, P, 8, P, None, None), 1, "NULL")
    assert L.trident_layer_norm(None, 0, 0, 8, 8, None, None, 0, 1e-5, None, 8, None, None, None) == 0
    need = L.trident_layer_norm_grad_workspace_bytes(100, 64)
    assert need > 0 and L.trident_layer_norm_grad_workspace_bytes(-1, 64) == 0
    refused(L.trident_layer_norm_grad(P, 64, P, 64, 0, 100, 64, P, 0, P, P, P, 64, P, P, P, need - 1, None), 3,
            str(need))
    refused(L.trident_layer_norm_grad(P, 64, P, 64, 0, 100, 64, P, 0, None, P, P, 64, P, P, P, need, None), 1, "NULL")


def test_adamw_arguments():
    L = _lib.lib()
    t = _lib.TridentAdamTensor(P, P, 300, 0, 0, 0)
    s = _lib.TridentAdamState(P, P, None, None, 512, 32)
    h = _lib.TridentAdamParams(1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 1)

    def call(t=t, s=s, h=h, n=1):
        return L.trident_adamw(ctypes.byref(t), n, ctypes.byref(s), ctypes.byref(h), None)

    refused(call(n=-1), 1, "count=-1")
    refused(call(h=_lib.TridentAdamParams(1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 0)), 1, "step=0")
    refused(call(h=_lib.TridentAdamParams(1e-3, 1.0, 0.999, 1e-8, 0.0, 1.0, 1)), 1, "betas")
    refused(call(s=_lib.TridentAdamState(P, P, None, None, 512, 16)), 2, "16 bits")
    refused(call(s=_lib.TridentAdamState(P, P, None, None, 512, 8)), 1, "NULL state")
    refused(call(s=_lib.TridentAdamState(P, P + 1, None, None, 512, 32)), 1, "aligned")
    refused(call(t=_lib.TridentAdamTensor(P, P, 300, 100, 0, 0)), 1, "multiple of 256")
    refused(call(t=_lib.TridentAdamTensor(P, P, 300, 256, 0, 0)), 1, "ends past")
    refused(call(t=_lib.TridentAdamTensor(P, P, 1 << 62, 0, 0, 0)), 1, "ends past")
    refused(call(t=_lib.TridentAdamTensor(P, P, 300, 0, 3, 0)), 1, "dtype=3")
    refused(call(t=_lib.TridentAdamTensor(P, None, 300, 0, 0, 0)), 1, "tensor 0")
    assert call(n=0) == 0
    refused(L.trident_adamw_state_values(ctypes.byref(s), P, P, None), 1, "NULL")


def test_fp8_arguments():
    L = _lib.lib()
    refused(L.trident_fp8_quantize(P, 0, 4, 100, 99, P, P, None), 1, "bad sizes")
    refused(L.trident_fp8_quantize(P, 0, 4, 100, 100, P + 8, P, None), 1, "16-byte aligned")
    refused(L.trident_fp8_matmul(P, P, 4, P, P, 4, 100, P, 1, P, 2, 4, 0, None), 1, "bias_dtype=1")
    refused(L.trident_fp8_matmul(P, P, 4, P, P, 4, 100, None, 0, P, 2, 3, 0, None), 1, "bad sizes")
    refused(L.trident_fp8_matmul(P, None, 4, P, P, 4, 100, None, 0, P, 2, 4, 0, None), 1, "NULL")
    refused(L.trident_fp8_matmul(P, P, 4, P + 8, P, 4, 100, None, 0, P, 2, 4, 0, None), 1, "16-byte")
    refused(L.trident_fp8_matmul(P, P, 4, P, P + 2, 4, 100, None, 0, P, 2, 4, 0, None), 1, "4-byte")
    refused(L.trident_fp8_matmul(P, P + 1, 4, P, P, 4, 100, None, 0, P, 2, 4, 0, None), 1, "4-byte")
    refused(L.trident_fp8_matmul(P, P, 4, P, P, 4, 1 << 23, None, 0, P, 2, 4, 0, None), 2, "too large")
    assert L.trident_fp8_matmul(P, P, 0, P, P, 4, 100, None, 0, P, 2, 4, 0, None) == 0
    need = L.trident_fp8_linear_workspace_bytes(100, 4, 1000)
    assert need >= 100 * 1024 + 100 * 8
    refused(L.trident_fp8_linear(P, 0, 100, 1000, 1000, P, P, 4, None, 0, P, 4, 0, P, need - 1, None), 3, str(need))


def test_python_boundary_refuses_host_tensors():
    f, ids = torch.zeros((4, 8)), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: encoder.embedding(ids, f), lambda: encoder.embedding_grad(f, ids, 10),
                 lambda: encoder.layer_norm(f), lambda: encoder.AdamW([f]), lambda: encoder.quantize_fp8(f),
                 lambda: encoder.fp8_linear(f, encoder.Fp8Blocks(f, f, 8))):
        with pytest.raises(_lib.TridentError, match="device tensor"):
            call()


@pytest.mark.parametrize("M,N,K", [(100, 0, 4096), (0, 100, 4096), (1 << 20, 0, 1 << 20), (0, 0, 1)])
def test_a_projection_without_rows_or_columns(M, N, K):
    """No workspace and nothing to do, whatever the length of K."""
    L = _lib.lib()
    assert L.trident_fp8_linear_workspace_bytes(M, N, K) == 0
    assert L.trident_fp8_linear(P, 0, M, K, K, P, P, N, None, 0, P, max(N, 1), 0, None, 0, None) == 0
