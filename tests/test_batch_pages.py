"""Pages that a ragged batch needs where its slots share some, on a host-only engine (no kernels)."""
from __future__ import annotations

import pytest
import torch


def sharing(qkvlib, n_share, n_pages, keep=False):
    """`n_share` slots with one page of 100 positions between them (and, if keep, a snapshot that holds it too)."""
    eng = qkvlib.Engine(n_layer=1, n_head=16, n_head_kv=2, n_ctx=512, n_slots=n_share, n_pages=n_pages, device=-1)
    for s in range(n_share):
        eng.seq_alloc(s)
    batch(eng, [0], [0], [100])
    snap = eng.snapshot_save(0)
    for s in range(1, n_share):
        eng.snapshot_load(snap, s)
    if not keep:
        snap.release()
        snap = None
    page = eng.pages(0)[0]
    assert eng.refcount(page) == n_share + keep and all(eng.pages(s) == [page] for s in range(n_share))
    return eng, page, snap


def batch(eng, slots, pos0, new):
    try:
        eng.batch_map(slots, pos0, new, sum(new), torch.zeros(len(slots) + 1, dtype=torch.int32))
    except Exception as e:
        import qwfn_hybrid_b200 as Q
        assert isinstance(e, Q.QkvError)
        return e.status                    # host-only: UNSUPPORTED once the pages are reserved
    raise AssertionError("a host-only engine wrote maps")


@pytest.mark.parametrize("n_share,keep,writers,copies", [(2, False, 2, 1), (3, False, 3, 2), (3, False, 2, 2), (2, True, 2, 2), (2, True, 1, 1)])
def test_a_shared_page_is_kept_by_its_last_holder(qkvlib, n_share, keep, writers, copies):
    """With just the pages that reserving slot by slot takes, the batch goes through; with one fewer nothing changes."""
    eng, page, snap = sharing(qkvlib, n_share, 1 + copies, keep)
    assert eng.pages_free() == copies
    assert batch(eng, list(range(writers)), [100] * writers, [5] * writers) == qkvlib.ERR_UNSUPPORTED
    assert eng.pages_free() == 0 and [eng.n_past(s) for s in range(writers)] == [105] * writers
    held = [eng.pages(s)[0] for s in range(writers)]
    assert len(set(held)) == writers
    assert eng.refcount(page) == n_share + keep - copies
    eng, page, snap = sharing(qkvlib, n_share, copies, keep)
    assert batch(eng, list(range(writers)), [100] * writers, [5] * writers) == qkvlib.ERR_NO_MEMORY
    assert eng.pages_free() == copies - 1 and all(eng.pages(s) == [page] and eng.n_past(s) == 100 for s in range(n_share))


def test_shared_and_new_pages_together(qkvlib):
    """Rows that start in a shared page and go on into new ones: one copy between two slots, a new page each."""
    eng, page, _ = sharing(qkvlib, 2, 4)
    assert batch(eng, [1, 0], [90, 100], [170, 200]) == qkvlib.ERR_UNSUPPORTED
    assert eng.pages_free() == 0 and len(eng.pages(0)) == len(eng.pages(1)) == 2 and eng.refcount(page) == 1
