"""How many rows a plane of queries has: its shape says so, or the call does; what could be read in two ways is refused."""
import numpy as np
import pytest

import overfit_amd as ov
from test_kv_refusals import BATCH, F, I, loose_cache


class Rows(Exception):
    pass


def rows_of(cache, name, place):
    """The call's rows and heads, as the library would get them."""
    def fn(*args):
        raise Rows(args[place], args[place + 1] if name != "ovfq_kv_append" else args[9])

    fn.__name__ = name
    setattr(cache.context.lib, name, fn)


ONE = dict(row_offsets=np.array([0, 1], I), lengths=np.array([5], I), tables=np.zeros((1, 2), I))
MANY = BATCH  # two requests of three rows


def calls(q, batch, rows=None):
    """(rows, heads) that each operator takes q to have."""
    got = []
    for name, place, call in (("ovfq_attend", 4, lambda c: ov.attend(c, q, **batch, rows=rows)),
                              ("ovfq_attend_selected", 4, lambda c: ov.attend_selected(c, q, **batch, top_pages=2, rows=rows)),
                              ("ovfq_kv_append", 5, lambda c: ov.kv_append(c, None, None, **batch, q=q, rope=ov.Rope(np.ones(4, F)), rows=rows))):
        cache = loose_cache()
        rows_of(cache, name, place)
        with pytest.raises(Rows) as e:
            call(cache)
        got.append(e.value.args)
    assert got[0] == got[1] == got[2]
    return got[0]


def test_shapes_that_say_their_rows():
    assert calls(np.zeros((3, 32), F), MANY) == (3, 4)
    assert calls(np.zeros((3, 4, 8), F), MANY) == (3, 4)
    assert calls(np.zeros((1, 32), F), ONE) == (1, 4)
    assert calls(np.zeros((1, 4, 8), F), ONE) == (1, 4)
    assert calls(np.zeros(32, F), ONE) == (1, 4)


def test_rows_that_are_given():
    for shape in ((96,), (3, 32), (1, 3, 32), (3, 4, 8), (1, 3, 4, 8), (1, 96)):
        assert calls(np.zeros(shape, F), MANY, 3) == (3, 4)


@pytest.mark.parametrize("shape,batch,rows", [
    ((96,), MANY, None),        # would be one row of twelve heads
    ((1, 3, 32), MANY, None),   # likewise
    ((1, 3, 4, 8), MANY, None),
    ((3, 32), MANY, 5),         # not whole heads
    ((3, 32), MANY, 0),
    ((3, 32), MANY, -3),
])
def test_shapes_that_do_not(shape, batch, rows):
    q = np.zeros(shape, F)
    for call in (lambda c: ov.attend(c, q, **batch, rows=rows), lambda c: ov.attend_selected(c, q, **batch, top_pages=2, rows=rows),
                 lambda c: ov.kv_append(c, None, None, **batch, q=q, rope=ov.Rope(np.ones(4, F)), rows=rows)):
        cache = loose_cache()
        with pytest.raises(ov.OverfitArgumentError):
            call(cache)
        assert not cache.context.lib.calls


def test_rows_beside_keys():
    """Keys say how many rows there are, whatever the queries' shape."""
    k, rope = np.zeros(48, F), ov.Rope(np.ones(4, F))
    for q in (np.zeros(96, F), np.zeros((1, 3, 32), F)):
        cache = loose_cache()
        rows_of(cache, "ovfq_kv_append", 5)
        with pytest.raises(Rows) as e:
            ov.kv_append(cache, k, k, **BATCH, q=q, rope=rope)
        assert e.value.args == (3, 4)
    with pytest.raises(ov.OverfitArgumentError):
        ov.kv_append(loose_cache(), k, k, **BATCH, rows=2)
