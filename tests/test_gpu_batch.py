"""Ragged batches: maps built on the device, the append through the slot map, and a run of the ragged
operators together as a serving step uses them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import assert_close, normal, read_rows, to_dev
from rec_reference import HD, convolution, recurrence

pytestmark = pytest.mark.gpu


def i32(*shape):
    return torch.full(shape, -9, dtype=torch.int32, device="cuda")


def maps(eng, slots, pos0, n_new, n_rows):
    n = len(slots)
    cu, seq, pos = i32(n + 1), i32(n_rows), i32(n_rows)
    cell = torch.full((n_rows,), -9, dtype=torch.int64, device="cuda")
    table = i32(n, (eng.cfg.n_ctx + 255) // 256)
    eng.batch_map(slots, pos0, n_new, n_rows, cu, seq, pos, cell, table)
    torch.cuda.synchronize()
    assert eng.device_status() == 0
    return cu, seq, pos, cell, table


def expected(eng, slots, pos0, n_new, n_rows):
    width = (eng.cfg.n_ctx + 255) // 256
    cu, seq, pos, cell, table = [0], [], [], [], []
    for i, (s, p, m) in enumerate(zip(slots, pos0, n_new)):
        pages = eng.pages(s)
        cu.append(cu[-1] + m)
        for t in range(p, p + m):
            seq.append(i)
            pos.append(t)
            cell.append(pages[t // 256] * 256 + t % 256)
        need = (p + m + 255) // 256
        table.append(pages[:need] + [-1] * (width - need))
    pad = [-1] * (n_rows - len(seq))
    return cu, seq + pad, pos + pad, cell + pad, table


@pytest.mark.parametrize("n_seq,seed,most,spare", [(1, 1, 1, 0), (1, 2, 700, 5), (7, 3, 3, 0), (40, 4, 300, 1000), (300, 5, 9, 1)])
def test_maps(cuda, qkvlib, n_seq, seed, most, spare):
    r = np.random.default_rng(seed)
    eng = qkvlib.Engine(n_layer=1, n_head=16, n_head_kv=2, n_ctx=1500, n_slots=n_seq + 1, device=0)
    slots = [int(s) for s in r.permutation(n_seq + 1)[:n_seq]]
    for s in slots:
        eng.seq_alloc(s)
    first = [int(x) for x in r.integers(0, 600, n_seq)]
    maps(eng, slots, [0] * n_seq, first, sum(first))
    pos0 = [int(r.integers(0, p + 1)) for p in first]       # anywhere up to the end
    new = [int(x) for x in r.integers(0, most + 1, n_seq)]
    new[0] = most
    n_rows = sum(new) + spare
    got = maps(eng, slots, pos0, new, n_rows)
    for g, w in zip(got, expected(eng, slots, pos0, new, n_rows)):
        assert g.tolist() == w
    assert [eng.n_past(s) for s in slots] == [max(a, b + c) for a, b, c in zip(first, pos0, new)]


def test_maps_of_nothing_and_alone(cuda, qkvlib):
    eng = qkvlib.Engine(n_layer=1, n_head=16, n_head_kv=2, n_ctx=300, n_slots=2, device=0)
    eng.seq_alloc(0)
    eng.seq_alloc(1)
    cu, seq, pos, cell, table = maps(eng, [1, 0], [0, 0], [0, 0], 4)
    assert cu.tolist() == [0, 0, 0] and seq.tolist() == [-1] * 4 and cell.tolist() == [-1] * 4 and table.tolist() == [[-1, -1]] * 2
    cu = i32(2)
    eng.batch_map([1], [0], [5], 5, cu)                       # offsets alone
    assert cu.tolist() == [0, 5]
    cu = i32(3)
    eng.batch_map([1, 0], [5, 0], [0, 0], 0, cu)              # no rows at all
    assert cu.tolist() == [0, 0, 0]


def test_maps_copy_shared_pages(cuda, qkvlib, oracle):
    """A batch that appends into a page a snapshot shares gets a page of its own; the snapshot keeps its rows."""
    eng = qkvlib.Engine(n_layer=2, n_head=16, n_head_kv=2, n_ctx=512, n_slots=1, n_pages=4, device=0)
    eng.seq_alloc(0)
    Kf, Vf = normal(1, (100, 512)), normal(2, (100, 512))
    for layer in range(2):
        eng.append(layer, 0, 0, to_dev(Kf), to_dev(Vf))
    snap = eng.snapshot_save(0)
    old = eng.pages(0)
    _, _, _, cell, _ = maps(eng, [0], [90], [20], 20)
    assert eng.pages(0) != old and eng.refcount(old[0]) == 1
    K2, V2 = normal(3, (20, 512)), normal(4, (20, 512))
    for layer in range(2):
        eng.append_mapped(layer, cell, to_dev(K2), to_dev(V2))
    for layer in range(2):
        k, v = read_rows(eng, layer, 0, 0, 110)
        assert np.array_equal(k, oracle.quantize_rows(np.concatenate([Kf[:90], K2])))
        assert np.array_equal(v, oracle.quantize_rows(np.concatenate([Vf[:90], V2])))
    eng.snapshot_load(snap, 0)
    k, _ = read_rows(eng, 1, 0, 0, 100)
    assert np.array_equal(k, oracle.quantize_rows(Kf))


@pytest.mark.parametrize("n_head_kv", [1, 2])
@pytest.mark.parametrize("first,new", [([0], [1]), ([3], [40]), ([0, 16, 250], [16, 16, 16]), ([5, 17, 254, 63, 0], [3, 30, 5, 130, 0]),
                                       ([1] * 20, [1] * 20), ([2] * 9, [3] * 9)])
def test_append_mapped_is_the_append(cuda, qkvlib, first, new, n_head_kv):
    """Bit for bit the rows that qkv_append writes, and no byte beside them."""
    n, width = len(first), 256 * n_head_kv
    gen = torch.Generator().manual_seed(9)
    rows = sum(new)
    K = torch.randn(rows + 2, width, generator=gen).cuda()
    V = torch.randn(rows + 2, width, generator=gen).cuda()
    pools = []
    for mapped in (True, False):
        eng = qkvlib.Engine(n_layer=2, n_head=16, n_head_kv=n_head_kv, n_ctx=512, n_slots=n, device=0)
        view = eng.cache_view(1)
        raw = type("Pool", (), {"__cuda_array_interface__": {"shape": (view.n_pages * view.page_bytes,), "typestr": "|u1",
                                                             "data": (view.pool, False), "version": 3}})()
        pool = torch.as_tensor(raw, device="cuda")
        pool.fill_(0x5A)
        for s in range(n):
            eng.seq_alloc(s)
            if first[s]:
                eng.append(0, s, 0, torch.zeros(first[s], width, device="cuda"), torch.zeros(first[s], width, device="cuda"))
        for s in range(n):
            eng.reserve(s, first[s] + new[s])
        if mapped:
            _, _, _, cell, _ = maps(eng, list(range(n)), first, new, rows + 2)
            eng.append_mapped(1, cell, K, V)
        else:
            at = 0
            for s in range(n):
                if new[s]:
                    eng.append(1, s, first[s], K[at:at + new[s]].contiguous(), V[at:at + new[s]].contiguous())
                at += new[s]
        torch.cuda.synchronize()
        assert eng.device_status() == 0
        pools.append((eng, pool))
    assert torch.equal(pools[0][1], pools[1][1])


def test_append_mapped_reports_cells_outside(cuda, qkvlib):
    eng = qkvlib.Engine(n_layer=1, n_head=16, n_head_kv=2, n_ctx=256, n_slots=1, device=0)
    eng.seq_alloc(0)
    maps(eng, [0], [0], [4], 4)
    K = torch.randn(4, 512, device="cuda")
    cell = torch.tensor([0, 256, -2, 1 << 40], dtype=torch.int64, device="cuda")
    eng.append_mapped(0, cell, K, K)
    assert eng.device_status() == 2
    a, _ = read_rows(eng, 0, 0, 0, 1)
    eng.append(0, 0, 0, K[:1].contiguous(), K[:1].contiguous())
    b, _ = read_rows(eng, 0, 0, 0, 1)
    assert np.array_equal(a, b)


def test_a_ragged_step_of_a_hybrid_model(cuda, qkvlib, oracle):
    """Two prompts and a continued sequence through one attention and one recurrent layer, as a server runs
    them: maps, mapped append, convolution, chunked recurrence; the appends and the recurrence captured
    once and replayed over the next batch's maps; then one decode step with a rollback."""
    H, Hk, cap, n = 4, 2, 160, 3
    ch = (2 * Hk + H) * HD
    eng = qkvlib.Engine(n_layer=1, n_head=16, n_head_kv=2, n_ctx=512, n_slots=n, rec_n_layer=1, rec_n_head=H,
                        conv_channels=ch, n_rollback=1, device=0)
    for s in range(n):
        eng.seq_alloc(s)
        eng.reset(s)
    gen = torch.Generator().manual_seed(77)
    rnd = lambda *s: torch.randn(*s, generator=gen).cuda()  # noqa: E731
    w = rnd(ch, 4) * 0.5
    cu, seq, pos, cell = i32(n + 1), i32(cap), i32(cap), torch.empty(cap, dtype=torch.int64, device="cuda")
    table = i32(n, 2)
    K, V, x = torch.zeros(cap, 512, device="cuda"), torch.zeros(cap, 512, device="cuda"), torch.zeros(cap, ch, dtype=torch.bfloat16, device="cuda")
    g, beta = torch.zeros(cap, H, device="cuda"), torch.zeros(cap, H, device="cuda")
    y, out = torch.zeros_like(x), torch.zeros(cap, H, HD, dtype=torch.bfloat16, device="cuda")
    slots = [2, 0, 1]

    def layers():
        eng.append_mapped(0, cell, K, V)
        eng.rec_conv(0, slots, cu, x, w, y, n_norm=2 * Hk * HD)
        eng.rec_chunk(0, slots, cu, y[:, :Hk * HD], y[:, Hk * HD:2 * Hk * HD], y[:, 2 * Hk * HD:], g, beta, HD ** -0.5, out)

    graph = torch.cuda.CUDAGraph()
    kept = {s: [np.zeros((0, 512), np.float32)] * 2 for s in slots}
    hist = {s: torch.zeros(ch, 3).cuda() for s in slots}
    state = {s: torch.zeros(H, HD, HD).cuda() for s in slots}
    for batch, new in enumerate(([70, 1, 33], [3, 100, 0])):
        rows = sum(new)
        for t in (K, V):
            t[:rows] = rnd(rows, 512)
        x[:rows] = rnd(rows, ch).to(torch.bfloat16)
        g[:rows], beta[:rows] = -torch.rand(rows, H, generator=gen).cuda() * 0.2, torch.rand(rows, H, generator=gen).cuda()
        pos0 = [eng.n_past(s) for s in slots]
        eng.batch_map(slots, pos0, new, cap, cu, seq, pos, cell, table)
        if batch == 0:
            layers()
        else:
            before = [eng.rec_state(0).clone(), eng.rec_state(0, 1).clone()]
            with torch.cuda.graph(graph):
                layers()
            assert torch.equal(before[0], eng.rec_state(0)) and torch.equal(before[1], eng.rec_state(0, 1))   # capture runs nothing
            graph.replay()
        torch.cuda.synchronize()
        assert eng.device_status() == 0
        at = 0
        for s, m in zip(slots, new):
            r = slice(at, at + m)
            at += m
            kept[s] = [np.concatenate([a, b[r].cpu().numpy()]) for a, b in zip(kept[s], (K, V))]
            yr, hs = convolution(hist[s], x[r], w, 2 * Hk * HD, 1e-6)
            assert float((y[r].double() - yr).norm()) <= 2.0 ** -8 * float(yr.norm())
            hist[s] = hs[-1].float()
            yy = y[r].unflatten(-1, (-1, HD))
            o, states, W, A = recurrence(state[s], yy[:, :Hk], yy[:, Hk:2 * Hk], yy[:, 2 * Hk:], g[r], beta[r], HD ** -0.5)
            assert bool(((out[r].double() - o).abs() <= 2.0 ** -8 * o.abs() + 3 * 2.0 ** -11 * W).all())
            assert float((eng.rec_state(0)[s].double() - states[-1]).norm()) <= 4 * 64 * 2.0 ** -24 * float(A[-1].norm())
            state[s] = eng.rec_state(0)[s].clone()
            assert torch.equal(eng.rec_state(0, 1)[s], hist[s])
    for s in slots:
        k, v = read_rows(eng, 0, s, 0, len(kept[s][0]))
        assert np.array_equal(k, oracle.quantize_rows(kept[s][0])) and np.array_equal(v, oracle.quantize_rows(kept[s][1]))
    # a decode step: the maps' table serves the attention of a view, the recurrence keeps the state before it
    eng.batch_map(slots, [eng.n_past(s) for s in slots], [1] * n, cap, cu, seq, pos, cell, table)
    K[:n], V[:n] = rnd(n, 512), rnd(n, 512)
    eng.append_mapped(0, cell[:n], K[:n], V[:n])
    Q, o = rnd(n, 1, 16, 256), torch.empty(n, 1, 16, 256, device="cuda")
    at = [eng.n_past(s) - 1 for s in slots]
    eng.attn_decode(0, slots, at, Q, 1, 1 / 16, o)
    for i, s in enumerate(slots):
        k, v = read_rows(eng, 0, s, 0, at[i] + 1)
        ref = oracle.attn(Q[i].cpu().numpy(), k, v, np.array([at[i]]), 2, 1 / 16)
        assert_close(o[i].cpu().numpy(), ref, f"slot {s}")
    xs, ys, os_ = rnd(n, ch), torch.empty(n, ch, device="cuda"), torch.empty(n, H, HD, device="cuda")
    eng.rec_conv(0, slots, cu, xs, w, ys, n_norm=2 * Hk * HD, save=True)
    eng.rec_step(0, slots, ys[:, :Hk * HD], ys[:, Hk * HD:2 * Hk * HD], ys[:, 2 * Hk * HD:], g[:n], beta[:n], 1, HD ** -0.5, os_, save=True)
    assert not torch.equal(eng.rec_state(0)[0], state[0])
    for s in slots:
        eng.rollback_arm(s, 1)
        eng.rollback_n(s, 1)
    torch.cuda.synchronize()
    for s in slots:
        assert torch.equal(eng.rec_state(0)[s], state[s]) and torch.equal(eng.rec_state(0, 1)[s], hist[s])
