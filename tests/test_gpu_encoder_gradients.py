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


def test_forward_mode_tangents_are_refused(dev):
    import torch.autograd.forward_ad as forward

    x, w, b = torch.randn((5, 40), device=dev), torch.randn(40, device=dev), torch.randn(40, device=dev)
    ids, table = torch.arange(5, device=dev), torch.randn((9, 40), device=dev)
    wq, bias = encoder.quantize_fp8(torch.randn((7, 40), device=dev)), torch.randn(7, device=dev)
    y, mean, rstd = encoder.layer_norm_forward(x, w, b)
    with forward.dual_level():
        dual = lambda t: forward.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: encoder.embedding(ids, dual(table)),
                     lambda: encoder.embedding(ids, dual(table.clone().requires_grad_())),
                     lambda: encoder.embedding_grad(dual(x), ids, 9),
                     lambda: encoder.layer_norm(dual(x), w, b), lambda: encoder.layer_norm(x, dual(w), b),
                     lambda: encoder.layer_norm(x.clone().requires_grad_(), w, dual(b)),
                     lambda: encoder.layer_norm_forward(dual(x)),
                     lambda: encoder.layer_norm_grad(dual(x), x, w, mean, rstd),
                     lambda: encoder.layer_norm_grad(x, x, w, dual(mean), rstd),
                     lambda: encoder.quantize_fp8(dual(x)), lambda: encoder.fp8_linear(dual(x), wq),
                     lambda: encoder.fp8_linear(x, wq, dual(bias))):
            with pytest.raises(_lib.TridentError, match="no forward-mode derivative"):
                call()
        # tensors without a tangent are taken as ever
        assert torch.equal(encoder.layer_norm(x, w, b), y) and torch.equal(encoder.embedding(ids, table), table[:5])
    assert torch.equal(encoder.layer_norm(x, w, b), y)


def test_function_transforms_raise(dev):
    """Wrapped tensors have no memory of their own to read: an error, and no result without a derivative."""
    x, t = torch.randn((5, 40), device=dev), torch.randn((5, 40), device=dev)
    wq = encoder.quantize_fp8(torch.randn((7, 40), device=dev))
    for f in (encoder.layer_norm, lambda x: encoder.fp8_linear(x, wq)):
        with pytest.raises(Exception):
            torch.func.jvp(f, (x,), (t,))
        with pytest.raises(Exception):
            torch.func.grad(lambda x: f(x).sum())(x)  # noqa: B023
        with pytest.raises(Exception):
            torch.func.vmap(f)(x)
