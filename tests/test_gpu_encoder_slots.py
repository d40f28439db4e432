"""Empty slots of a padded batch through a transformer layer and back: they get a gradient of zero and change none."""
import pytest
import torch

from trident_amd import encoder
from test_gpu_encoder import F64, gen, randn
from test_gpu_encoder_layer import example, padded_ids  # noqa: F401

pytestmark = pytest.mark.gpu


def test_slots_have_no_gradient_and_change_none(dev, example):  # noqa: F811
    g = gen(1)
    model = example.TextEncoder(300, 64, 32, g, dev, layers=2, heads=2)
    ids = padded_ids(g, 6, 30, 300)
    more = torch.cat((ids, torch.full((6, 45), -1, device=dev)), 1)
    grad = randn(g, 6, 64)
    leaves = [model.table, model.gamma, model.beta] + [p for layer in model.layers for p in layer.parameters()]
    few, many = (torch.autograd.grad(model.pooled(t), leaves, grad) for t in (ids, more))
    # float32 sums of a few hundred terms, in another order: far below 1e-4 of a gradient's size
    for a, b in zip(few, many):
        assert (a.to(F64) - b).square().mean().sqrt() <= 1e-4 * a.to(F64).square().mean().sqrt()
    for t in (ids, more):
        x = encoder.embedding(t, model.table, scale=model.scale).detach().requires_grad_()
        live = t >= 0
        y = model.layers[0](x, live.sum(1))
        (y * live[..., None] * randn(gen(2), *y.shape)).sum().backward()
        assert (x.grad[~live] == 0).all() and x.grad[live].isfinite().all() and (x.grad[live] != 0).any()
