"""The weights of an `Int8Expert` and the addresses that its calls hand on belong
together, without a GPU (the launch is recorded)."""

import pytest
import torch


@pytest.fixture
def expert(monkeypatch):
    from qmesh_b200 import int8
    sent = []
    monkeypatch.setattr(int8, "same_device", lambda dev, **t: None)
    monkeypatch.setattr(int8, "launch_on", lambda dev, fn, what, args: sent.append(args._obj))
    w = [torch.zeros(64, 32, dtype=torch.int8), torch.ones(64), torch.zeros(32, 32, dtype=torch.int8), torch.ones(32)]
    return int8.Int8Expert(*w), w, sent


def addresses(ex, sent):
    ex(torch.zeros(2, 32))
    a = sent[-1]
    return a.w13, a.w13_scale, a.w2, a.w2_scale


def test_weights_cannot_be_exchanged(expert):
    """An assignment that the calls would not see is refused."""
    ex, w, sent = expert
    for name in ("w13", "w13_scale", "w2", "w2_scale"):
        with pytest.raises(AttributeError):
            setattr(ex, name, torch.ones_like(getattr(ex, name)))


def test_addresses_are_the_weights(expert):
    """The call reads the memory that the expert shows as its weights, also after the
    caller's own tensors were pointed elsewhere or dropped."""
    ex, w, sent = expert
    want = tuple(t.data_ptr() for t in w)
    assert addresses(ex, sent) == want
    w[0].fill_(3)                                          # written in place: seen
    assert (ex.w13 == 3).all()
    for t in w:
        t.data = torch.zeros_like(t)
    ex.w2.data = torch.zeros(1, dtype=torch.int8)
    del t
    w.clear()
    assert addresses(ex, sent) == want
    assert tuple(t.data_ptr() for t in (ex.w13, ex.w13_scale, ex.w2, ex.w2_scale)) == want
    assert (ex.w13 == 3).all() and ex.w2.shape == (32, 32)
