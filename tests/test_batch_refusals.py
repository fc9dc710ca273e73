"""Refusals and host bookkeeping of the ragged-batch and recurrent-layer calls, on a host-only engine (no kernels)."""
from __future__ import annotations

import pytest
import torch


def host_engine(qkvlib, **kw):
    args = dict(n_layer=1, n_head=16, n_head_kv=2, n_ctx=1024, n_slots=4, n_pages=6, rec_n_layer=2, rec_n_head=4,
                conv_channels=1024, n_rollback=2, device=-1)
    args.update(kw)
    eng = qkvlib.Engine(**args)
    for s in range(args["n_slots"] - 1):
        eng.seq_alloc(s)
    return eng


CU = torch.zeros(9, dtype=torch.int32)


def batch(eng, slots, pos0, new, rows=5000):
    eng.batch_map(slots, pos0, new, rows, torch.zeros(len(slots) + 1, dtype=torch.int32))


@pytest.mark.parametrize("slots,pos0,new,rows,status", [
    ([], [], [], 5, "INVALID"), ([0, 0], [0, 0], [1, 1], 5, "INVALID"), ([9], [0], [1], 5, "INVALID"), ([3], [0], [1], 5, "STATE"),
    ([0], [1], [1], 5, "INVALID"), ([0], [-1], [1], 5, "INVALID"), ([0], [0], [-1], 5, "INVALID"), ([0], [0], [6], 5, "INVALID"),
    ([0], [0], [1025], 5000, "STATE"), ([0, 1], [0, 0], [1024, 1024], 5000, "NO_MEMORY"), ([0], [0], [1], -1, "INVALID"),
    ([0], [0], [2147483647], 2147483647, "STATE")])
def test_batch_map_refusals_change_nothing(qkvlib, slots, pos0, new, rows, status):
    eng = host_engine(qkvlib)
    with pytest.raises(qkvlib.QkvError) as e:
        batch(eng, slots, pos0, new, rows)
    assert e.value.status == getattr(qkvlib, "ERR_" + status)
    assert eng.pages_free() == 6 and eng.n_past(0) == 0 and eng.n_past(1) == 0


def test_batch_map_reserves_like_append(qkvlib):
    eng = host_engine(qkvlib)
    with pytest.raises(qkvlib.QkvError) as e:      # host-only: pages reserved, no maps written
        batch(eng, [1, 0, 2], [0, 0, 0], [300, 0, 256])
    assert e.value.status == qkvlib.ERR_UNSUPPORTED
    assert [eng.n_past(s) for s in (0, 1, 2)] == [0, 300, 256] and [len(eng.pages(s)) for s in (0, 1, 2)] == [0, 2, 1]
    snap = eng.snapshot_save(1)
    with pytest.raises(qkvlib.QkvError):
        batch(eng, [1], [299], [2])
    assert eng.n_past(1) == 301 and eng.refcount(eng.pages(1)[0]) == 2 and eng.refcount(eng.pages(1)[1]) == 1
    snap.release()


def test_batch_map_checks_tensors(qkvlib):
    eng = host_engine(qkvlib)
    with pytest.raises(ValueError):
        eng.batch_map([0, 1], [0], [1, 1], 2, CU)
    with pytest.raises(ValueError):
        eng.batch_map([0, 1], [0, 0], [1, 1], 2, CU[:2])
    with pytest.raises(ValueError):
        eng.batch_map([0], [0], [1], 1, CU, cell=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        eng.batch_map([0], [0], [1], 4, CU, seq=torch.zeros(3, dtype=torch.int32))


def test_append_mapped_refusals(qkvlib):
    eng = host_engine(qkvlib)
    K = torch.zeros(2, 512)
    cell = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(qkvlib.QkvError) as e:
        eng.append_mapped(1, cell, K, K)
    assert e.value.status == qkvlib.ERR_INVALID
    with pytest.raises(ValueError):
        eng.append_mapped(0, cell[:1], K, K)
    with pytest.raises(ValueError):
        eng.append_mapped(0, cell, K, K[:, :256])
    with pytest.raises(qkvlib.QkvError) as e:
        eng.append_mapped(0, cell, K, K)
    assert e.value.status == qkvlib.ERR_UNSUPPORTED


def rows(n=2, H=4, Hk=2, dtype=torch.float32):
    x = torch.zeros(n, (2 * Hk + H) * 128, dtype=dtype)
    return dict(q=x[:, :Hk * 128], k=x[:, Hk * 128:2 * Hk * 128], v=x[:, 2 * Hk * 128:], g=torch.zeros(n, H), beta=torch.zeros(n, H))


def step(eng, layer=0, slots=(0, 1), T=1, save=False, out=None, **kw):
    r = rows()
    r.update(kw)
    eng.rec_step(layer, list(slots), r["q"], r["k"], r["v"], r["g"], r["beta"], T, 1.0, torch.zeros(2, 4, 128) if out is None else out, save=save)


@pytest.mark.parametrize("kw,status", [
    (dict(layer=2), "INVALID"), (dict(layer=-1), "INVALID"), (dict(slots=(0, 0)), "INVALID"), (dict(slots=(0, 7)), "INVALID"),
    (dict(slots=(0, 3)), "STATE"), (dict(), "UNSUPPORTED"), (dict(beta=None), "UNSUPPORTED"), (dict(save=True), "UNSUPPORTED"),
    (dict(slots=(0,), T=2), "UNSUPPORTED")])
def test_rec_step_refusals(qkvlib, kw, status):
    with pytest.raises(qkvlib.QkvError) as e:
        step(host_engine(qkvlib), **kw)
    assert e.value.status == getattr(qkvlib, "ERR_" + status)


def test_rec_step_refuses_shapes(qkvlib):
    eng = host_engine(qkvlib)
    z = rows(dtype=torch.bfloat16)
    for kw in (dict(q=z["q"]), dict(q=rows()["q"][:1]), dict(v=rows()["v"][:, :384]), dict(g=torch.zeros(2, 3)), dict(k=rows()["k"][:, ::2]),
               dict(out=torch.zeros(2, 4, 64)), dict(out=torch.zeros(2, 4, 128, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            step(eng, **kw)
    for T in (0, 5):
        n = 2 * T
        x = rows(max(n, 1))
        with pytest.raises((qkvlib.QkvError, ValueError)):
            eng.rec_step(0, [0, 1], x["q"][:n], x["k"][:n], x["v"][:n], x["g"], x["beta"], T, 1.0, torch.zeros(10, 4, 128))
    with pytest.raises(qkvlib.QkvError) as e:                     # three heads of q for four of v
        step(eng, q=torch.zeros(2, 384), k=torch.zeros(2, 384))
    assert e.value.status == qkvlib.ERR_INVALID
    wide = torch.zeros(2, 1026)                                    # rows that start off 16 bytes
    with pytest.raises(qkvlib.QkvError) as e:
        step(eng, q=wide[:, 1:257])
    assert e.value.status == qkvlib.ERR_INVALID
    with pytest.raises(qkvlib.QkvError) as e:
        step(host_engine(qkvlib, n_rollback=0), save=True)
    assert e.value.status == qkvlib.ERR_INVALID
    with pytest.raises(qkvlib.QkvError) as e:
        step(host_engine(qkvlib, rec_head_dim=64), q=torch.zeros(2, 128), k=torch.zeros(2, 128), v=torch.zeros(2, 256))
    assert e.value.status == qkvlib.ERR_UNSUPPORTED


def test_rec_chunk_refusals(qkvlib):
    eng = host_engine(qkvlib)
    r = rows(6, dtype=torch.bfloat16)
    out = torch.zeros(6, 4, 128, dtype=torch.bfloat16)
    call = lambda cu=CU, slots=(0, 1), q=r["q"], out=out: eng.rec_chunk(0, list(slots), cu, q, r["k"], r["v"], r["g"], r["beta"], 1.0, out)  # noqa: E731
    for kw in (dict(cu=CU[:2]), dict(cu=CU.long()), dict(q=rows(6)["q"]), dict(out=out[:5])):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(qkvlib.QkvError) as e:
        call(slots=(1, 1))
    assert e.value.status == qkvlib.ERR_INVALID
    with pytest.raises(qkvlib.QkvError) as e:
        call()
    assert e.value.status == qkvlib.ERR_UNSUPPORTED


def test_rec_conv_refusals(qkvlib):
    eng = host_engine(qkvlib)
    x, w = torch.zeros(4, 1024), torch.zeros(1024, 4)

    def call(eng=eng, x=x, w=w, y=None, n_norm=0, eps=1e-6, cu=CU, **kw):
        eng.rec_conv(0, [0, 1], cu, x, w, torch.zeros(x.shape, dtype=x.dtype) if y is None else y, n_norm=n_norm, eps=eps, **kw)

    for kw in (dict(x=x.half()), dict(x=x[:, :512]), dict(w=w[:512]), dict(y=torch.zeros(3, 1024)), dict(y=x.bfloat16()), dict(cu=CU[:2])):
        with pytest.raises(ValueError):
            call(**kw)
    wide = torch.zeros(4, 1026)
    for kw in (dict(n_norm=64), dict(n_norm=1152), dict(n_norm=-128), dict(eps=-1.0), dict(eps=float("nan")), dict(y=x), dict(x=wide[:, :1024])):
        with pytest.raises(qkvlib.QkvError) as e:
            call(**kw)
        assert e.value.status == qkvlib.ERR_INVALID, kw
    for bad in (dict(conv_hist=4), dict(conv_channels=1000)):
        c = bad.get("conv_channels", 1024)
        with pytest.raises(qkvlib.QkvError) as e:
            call(host_engine(qkvlib, **bad), x=torch.zeros(4, c), w=torch.zeros(c, 4))
        assert e.value.status == qkvlib.ERR_UNSUPPORTED
    with pytest.raises(qkvlib.QkvError) as e:
        call(host_engine(qkvlib, n_rollback=0), save=True)
    assert e.value.status == qkvlib.ERR_INVALID
    with pytest.raises(qkvlib.QkvError) as e:
        call()
    assert e.value.status == qkvlib.ERR_UNSUPPORTED


def test_rec_output_over_an_input_is_refused(qkvlib):
    eng = host_engine(qkvlib)
    for name in ("q", "k", "v", "g", "beta"):
        buf = torch.zeros(6 * 1024)
        out = buf[:2 * 512].view(2, 4, 128)                    # the last values of out and the first of the input
        width = {"q": 256, "k": 256, "v": 512, "g": 4, "beta": 4}[name]
        at = 2 * 512
        for start, status in ((at - 4, "INVALID"), (at, "UNSUPPORTED")):
            with pytest.raises(qkvlib.QkvError) as e:
                step(eng, out=out, **{name: buf[start:start + 2 * width].view(2, width)})
            assert e.value.status == getattr(qkvlib, "ERR_" + status), (name, start)
    r = rows(6, dtype=torch.bfloat16)
    with pytest.raises(qkvlib.QkvError) as e:                     # out in the place of v
        v = torch.zeros(6, 512, dtype=torch.bfloat16)
        eng.rec_chunk(0, [0, 1], CU, r["q"], r["k"], v, r["g"], r["beta"], 1.0, v.view(6, 4, 128))
    assert e.value.status == qkvlib.ERR_INVALID


def test_tensors_of_another_device_are_refused(qkvlib):
    eng = host_engine(qkvlib)
    eng.device = 0                                                 # host tensors for a device's engine: nothing is called
    i32 = torch.zeros(3, dtype=torch.int32)
    r, b = rows(), rows(6, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device"):
        eng.batch_map([0], [0], [1], 1, i32)
    with pytest.raises(ValueError, match="device"):
        eng.append_mapped(0, torch.zeros(2, dtype=torch.int64), torch.zeros(2, 512), torch.zeros(2, 512))
    with pytest.raises(ValueError, match="device"):
        step(eng, **r)
    with pytest.raises(ValueError, match="device"):
        eng.rec_chunk(0, [0, 1], CU, b["q"], b["k"], b["v"], b["g"], None, 1.0, torch.zeros(6, 4, 128, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="device"):
        eng.rec_conv(0, [0, 1], CU, torch.zeros(6, 1024), torch.zeros(1024, 4), torch.zeros(6, 1024))
