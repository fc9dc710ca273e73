"""The block tables of a ragged batch's maps as the cache view that the allocation-free decode attends over."""
from __future__ import annotations

import ctypes

import pytest
import torch

from helpers import assert_close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("contexts,T", [([700, 1, 255, 256, 900], 1), ([3, 513, 64], 3)])
def test_static_decode_over_the_table_of_the_maps(cuda, qkvlib, contexts, T):
    """A batch's slots in any order: row i of the table is sequence i; the same attention as over the slots themselves."""
    n = len(contexts)
    eng = qkvlib.Engine(n_layer=2, n_head=16, n_head_kv=2, n_ctx=1024, n_slots=n + 2, device=0)
    gen = torch.Generator(device="cuda").manual_seed(111)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)   # noqa: E731
    slots = [(3 * i + 1) % (n + 2) for i in range(n)] if (n + 2) % 3 else list(range(n + 1, 1, -1))
    assert len(set(slots)) == n
    i32 = lambda *s: torch.full(s, -9, dtype=torch.int32, device="cuda")   # noqa: E731
    for s in slots:
        eng.seq_alloc(s)
    for pos0, new in (([0] * n, contexts), (contexts, [T] * n)):     # the contexts, then the step's rows
        rows = sum(new)
        cu, cell, table = i32(n + 1), torch.empty(rows, dtype=torch.int64, device="cuda"), i32(n, 4)
        eng.batch_map(slots, pos0, new, rows, cu, cell=cell, table=table)
        for layer in range(2):
            eng.append_mapped(layer, cell, rnd(rows, 512), rnd(rows, 512))
    Q = rnd(n, T, 16, 256)
    for layer in range(2):
        want, got = torch.empty_like(Q), torch.full_like(Q, float("nan"))
        eng.attn_decode(layer, slots, contexts, Q, T, 1 / 16, want)
        view = eng.cache_view(layer)
        view.block_table = table.data_ptr()
        ints = ctypes.c_int32 * n
        st = qkvlib.lib().qkv_attn_decode_static(ctypes.byref(view), n, ints(*range(n)), ints(*contexts), n, 16, Q.data_ptr(), T, 1 / 16,
                                                 got.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert st == qkvlib.OK
        code = ctypes.c_int32(-1)
        assert qkvlib.lib().qkv_static_status(torch.cuda.current_stream().cuda_stream, ctypes.byref(code)) == qkvlib.OK and code.value == 0
        assert eng.device_status() == 0
        assert_close(got.cpu().numpy(), want.cpu().numpy(), f"layer {layer}")
