"""Refusals of the join of attention outputs (no GPU)."""

import pytest

from torch_spyre_b200 import _lib

A = 1 << 20  # an aligned address that is never touched


def combine(**over):
    a = dict(o=A, dt=1, lse=A, parts=2, rows=3, dim=8, out=A, lo=None, stream=None)
    a.update(over)
    return _lib.lib().b200kv_lse_combine(*a.values())


@pytest.mark.parametrize("over,msg", [(dict(dt=3), "dtype"), (dict(dt=-1), "dtype"), (dict(parts=0), "num_parts"),
                                      (dict(rows=-1), "rows"), (dict(dim=0), "head_dim"), (dict(o=None), "null"),
                                      (dict(lse=None), "null"), (dict(out=None), "null")])
def test_refusals(over, msg):
    assert combine(**over) == 1 and msg in _lib.last_error()


def test_no_rows_is_nothing_to_do():
    assert combine(rows=0, o=None) == 0
