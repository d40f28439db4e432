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


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_of_other_tensors(dev, bits):
    """The same length in all, in other pieces: 257 and 256 elements are three blocks of 256, as 256 and 257
    are, and as 700 are."""
    make = lambda *sizes: encoder.AdamW([torch.ones(n, device=dev) for n in sizes], state_bits=bits)  # noqa: E731
    opt = make(257, 256)
    opt.step([torch.ones(257, device=dev), torch.ones(256, device=dev)])
    state = opt.state_dict()
    for other in (make(256, 257), make(700), make(258, 256), make(257, 256, 0)):
        with pytest.raises(_lib.TridentError, match="the state is of tensors"):
            other.load_state_dict(state)
        assert other.step_count == 0 and (other.exp_avg == 0).all()
    same = make(257, 256)
    same.load_state_dict(state)
    assert same.step_count == 1 and torch.equal(same.exp_avg, opt.exp_avg)
    del state["numels"]  # as an earlier version saved it
    old = make(257, 256)
    old.load_state_dict(state)
    assert old.step_count == 1 and torch.equal(old.exp_avg, opt.exp_avg)
