"""What AdamW refuses after it was made: parameters that moved onto one another, states of other tensors."""
import pytest
import torch

from trident_amd import _lib, encoder

pytestmark = pytest.mark.gpu


def test_parameters_that_come_to_share_memory(dev):
    """A step takes the parameters where they are now, so that is where they must lie apart."""
    base = torch.zeros(4096, device=dev)
    a, b, c = base[:1000], torch.zeros(500, device=dev), torch.zeros(500, device=dev)
    grads = [torch.ones_like(p) for p in (a, b, c)]
    opt = encoder.AdamW([a, b, c])
    opt.step(grads)
    kept = b.data
    for other, which in ((base[999:1499], grads), (c.data, grads), (base[500:1000], [grads[0], grads[1], None])):
        b.data = other
        before = base.clone()
        for _ in range(2):  # a refusal is not forgotten
            with pytest.raises(_lib.TridentError, match="share memory"):
                opt.step(which)
        assert torch.equal(base, before) and opt.step_count == 1
    b.data = base[1000:1500]  # next to one another
    opt.step(grads)
    # of two that share memory, one may be stepped by itself
    b.data = base[500:1000]
    opt.step([None, grads[1], grads[2]])
    b.data = kept
    opt.step(grads)
    assert opt.step_count == 4


def test_parameters_that_grow_into_one_another(dev):
    """The same address with a wider type is more memory."""
    base = torch.zeros(2048, device=dev)
    half = base.view(torch.float16)
    a, b = half[:1000], half[1000:2000]
    grads = [torch.ones(1000, device=dev, dtype=torch.float16) for _ in range(2)]
    opt = encoder.AdamW([a, b])
    opt.step(grads)
    a.data = base[:1000]
    for _ in range(2):
        with pytest.raises(_lib.TridentError, match="share memory"):
            opt.step(grads)
    assert opt.step_count == 1
