"""What the encoder's operators do with operands whose derivative is wanted: they give it or refuse."""
import pytest
import torch

from trident_amd import _lib, encoder

pytestmark = pytest.mark.gpu


def test_8_bit_products_refuse_operands_that_require_a_gradient(dev):
    x, w = torch.randn((5, 40), device=dev), torch.randn((7, 40), device=dev)
    bias = torch.randn(7, device=dev)
    wq, xq = encoder.quantize_fp8(w), encoder.quantize_fp8(x)
    want = encoder.fp8_linear(x, wq, bias)
    xg, bg = x.clone().requires_grad_(), bias.clone().requires_grad_()
    later = xg * 1.0  # with a history
    calls = [lambda: encoder.quantize_fp8(xg), lambda: encoder.fp8_linear(xg, wq, bias),
             lambda: encoder.fp8_linear(later, wq), lambda: encoder.fp8_linear(x, wq, bg),
             lambda: encoder.fp8_matmul(xq, wq, bg, out_dtype=torch.float32)]
    for call in calls:
        with pytest.raises(_lib.TridentError, match="has no gradient"):
            call()
    with torch.no_grad():
        for call in calls:
            call()
        assert torch.equal(encoder.fp8_linear(xg, wq, bg), want)
    assert torch.equal(encoder.fp8_linear(xg.detach(), wq, bg.detach()), want)
    with torch.inference_mode():
        assert torch.equal(encoder.fp8_linear(xg, wq, bg), want)
