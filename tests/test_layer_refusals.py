"""Calls of the transformer layer's entry points that have no right answer are refused, and those that have one are not; a
kernel's registers (CPU only: nothing is launched)."""
import ctypes

import pytest
import torch

from trident_amd import _lib, encoder
from test_build_guards import code_objects, kernel_resources, pytestmark  # noqa: F401
from test_layer_abi import attention, gated, on_gpu, refused  # noqa: F401


@pytest.mark.parametrize("scale", [1e-46, 5e-324, 0.0, -1.0, float("inf")])
def test_scales_that_float32_does_not_hold(on_gpu, scale):  # noqa: F811
    L = _lib.lib()
    a = attention(scale=scale)
    refused(L.trident_attention(ctypes.byref(a), None), 1, "scale")
    a = attention(scale=scale, lse=256, grad=256, dq=256, dk=256, dv=256)
    assert L.trident_attention_grad_workspace_bytes(ctypes.byref(a)) == 0
    refused(L.trident_attention_grad(ctypes.byref(a), 256, 1 << 40, None), 1, "scale")
    q = torch.zeros((10, 4, 16))
    for call in (encoder.attention, encoder.attention_forward):
        with pytest.raises(_lib.TridentError, match="scale"):
            call(q, q, q, scale=scale)
    with pytest.raises(_lib.TridentError, match="scale"):
        encoder.attention_grad(q, q, q, q, q, torch.zeros((4, 10)), scale=scale)


def test_rows_far_apart_are_packed():
    """A pitch past what a tile's offsets reach: such rows go through the workspace, and those of few rows need none."""
    L, far = _lib.lib(), 1 << 22
    for name, rows in (("ld_x", 100), ("ld_gate", 64), ("ld_up", 64)):
        a = gated(**{name: far})
        need = L.trident_gated_linear_workspace_bytes(ctypes.byref(a))
        assert need >= rows * 32 * 2
        refused(L.trident_gated_linear(ctypes.byref(a), 256, need - 1, None), 3, str(need))
        near = L.trident_gated_linear_grad_workspace_bytes(ctypes.byref(gated()))
        assert L.trident_gated_linear_grad_workspace_bytes(ctypes.byref(a)) >= near + rows * 32 * 2
        assert L.trident_gated_linear_workspace_bytes(ctypes.byref(gated(M=16, **{name: far}))) == 0
        refused(L.trident_gated_linear(ctypes.byref(gated(**{name: 1 << 41})), 256, 1 << 40, None), 1, "bad sizes")


def test_no_scratch_in_the_kernel_of_the_largest_slope(code_objects):  # noqa: F811
    found = {k: r for k, r in kernel_resources(code_objects).items() if "20largest_slope_kernel" in k}
    assert found
    for k, r in found.items():
        assert r["private_segment_fixed_size"] == 0 and r["vgpr_spill_count"] == 0, (k, r)
