"""Positions, slots and lengths as any sequence or iterator of integers."""
from __future__ import annotations

import array

import numpy as np
import pytest
import torch


@pytest.mark.parametrize("make", [list, tuple, iter, lambda v: (x for x in v), np.array, lambda v: np.array(v, dtype=np.uint8), bytes, bytearray,
                                  torch.tensor, lambda v: array.array("q", v), lambda v: [float(x) for x in v], lambda v: dict.fromkeys(v)],
                         ids=["list", "tuple", "iterator", "generator", "numpy", "numpy uint8", "bytes", "bytearray", "tensor", "array", "floats", "dict"])
@pytest.mark.parametrize("values", [[3, 1, 2, 7], [], [5]])
def test_values_become_int32(qkvlib, make, values):
    got = qkvlib._i32_array(make(values))
    assert list(got)[:len(values)] == values and len(got) == max(1, len(values))
    if make is not iter:
        assert qkvlib._i32s(make(values)).tolist() == values


def test_calls_take_iterators(qkvlib):
    eng = qkvlib.Engine(n_layer=1, n_head=16, n_head_kv=2, n_ctx=512, n_slots=3, n_pages=6, device=-1)
    for s in range(3):
        eng.seq_alloc(s)
    with pytest.raises(qkvlib.QkvError) as e:       # host-only: reserved, no maps
        eng.batch_map([0], [0], [300], 300, torch.zeros(2, dtype=torch.int32))
    assert e.value.status == qkvlib.ERR_UNSUPPORTED
    snap = eng.snapshot_save(0)
    eng.snapshot_load_many(snap, [1, 2], n_keep=iter([300, 300]))
    assert eng.n_past(1) == eng.n_past(2) == 300
    for slots, want in ((bytes([2, 1]), [310, 310]), (np.array([1, 2]), [320, 320])):
        with pytest.raises(qkvlib.QkvError) as e:
            eng.batch_map(slots, [300 if want[0] == 310 else 310] * 2, [10, 10], 20, torch.zeros(3, dtype=torch.int32))
        assert e.value.status == qkvlib.ERR_UNSUPPORTED
        assert [eng.n_past(1), eng.n_past(2)] == want
