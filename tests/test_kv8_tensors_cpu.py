"""KvCache8 holds the memory that its calls write, whatever becomes of the tensors
it was made of (nothing here runs on a GPU: a call that finds its tensors in order
is refused for their device)."""
import gc

import pytest
import torch

from lutmac_amd import torch_module
from lutmac_amd.kv8 import KvCache8

NAMES = ("k", "v", "k_scale", "v_scale")


def tensors():
    z = lambda *s, t: torch.zeros(2, 1, *s, dtype=t)
    return z(64, 64, t=torch.int8), z(64, 64, t=torch.int8), z(4, t=torch.float32), z(4, t=torch.float32)


def calls(c):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    x, where = torch.zeros(3, 1, 64), (i(2), i(1), i(1, 2))
    return [lambda: c.append(x, x, *where), lambda: c.attend(x, *where)]


@pytest.mark.parametrize("name", NAMES)
def test_tensors_are_not_replaced(name):
    c = KvCache8(*tensors())
    before = getattr(c, name)
    with pytest.raises(AttributeError):
        setattr(c, name, torch.empty_like(before))
    assert getattr(c, name) is before


def test_calls_keep_their_memory():
    """What the calls are given holds the tensors by itself."""
    t = list(tensors())
    handle = torch_module().kv8_cache(*t)
    assert [x._use_count() for x in t] == [2] * 4
    del handle
    gc.collect()
    assert [x._use_count() for x in t] == [1] * 4


@pytest.mark.parametrize("i,name", enumerate(NAMES))
def test_tensors_that_changed_are_refused(i, name):
    """Memory that a tensor gave up since is not written."""
    for change in (lambda t: t.resize_(0), lambda t: t.resize_(1, *t.shape[1:]), lambda t: t.transpose_(0, 1),
                   lambda t: t.set_(torch.zeros(8, dtype=t.dtype))):
        t = tensors()
        c = KvCache8(*t)
        change(t[i])
        for call in calls(c):
            with pytest.raises(ValueError, match="^(k|v|k_scale|v_scale): "):
                call()


def test_tensors_in_order_are_not_refused():
    t = tensors()
    c = KvCache8(*t)
    for x in t:
        x.set_(torch.zeros_like(x))   # (other memory of the same form is what the calls then use)
    for call in calls(c):
        with pytest.raises(ValueError, match="current device"):
            call()
