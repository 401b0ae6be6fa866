"""wavo_amd.Tree and wavo_amd.Rules keep what they point to: device memory whose only other holder is the expression that
made it must not be given back before the call that reads it.  Needs no GPU."""

import gc
import weakref

import pytest

import wavo_amd as wa


class Device:
    h = None  # (nothing to free)


def buffer(address):
    b = wa.Buffer.__new__(wa.Buffer)
    b.gpu, b.nbytes, b.ptr = Device(), 4, address
    return b


TREE = ["n", "count", "tokens", "mask"]
RULES = ["penalty", "history", "bias_start", "bias_id", "bias", "allow"]


@pytest.mark.parametrize("make,names", [(lambda **kw: wa.Tree(2, 3, **kw), TREE), (wa.Rules, RULES)], ids=["Tree", "Rules"])
def test_buffers_live_as_long_as_what_points_to_them(make, names):
    buffers = {x: buffer(4096 * (i + 1)) for i, x in enumerate(names)}
    alive = {x: weakref.ref(b) for x, b in buffers.items()}
    made = make(**buffers)
    del buffers
    gc.collect()
    assert [x for x in names if alive[x]() is None] == []
    assert [getattr(made, x) for x in names] == [4096 * (i + 1) for i in range(len(names))]
    del made
    gc.collect()
    assert [x for x in names if alive[x]() is not None] == []


def test_addresses_and_nothing_are_taken_as_they_are():
    t, r = wa.Tree(1, 1, 4096, mask=8192, mask_stride=7), wa.Rules(bias=64, bias_len=3, from_=5)
    assert (t.n, t.count, t.tokens, t.mask, t.mask_stride) == (4096, None, None, 8192, 7)
    assert (r.penalty, r.bias, r.bias_len, r.from_, r.allow) == (None, 64, 3, 5, None)
