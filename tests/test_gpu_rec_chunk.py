"""The chunked recurrence where its hand-overs and its arithmetic are strained: grids that fill the GPU, chunks that are worked
token by token among others, scores that change from chunk to chunk, repeated and long keys; against bounds made chunk by
chunk from the 64-bit recurrence (rec_bounds)."""
from __future__ import annotations

import pytest
import torch

import rec_bounds
from rec_reference import HD, inputs

pytestmark = pytest.mark.gpu
SCALE = HD ** -0.5
FULL = dict(H=37, Hk=37)                       # 4 sequences of 37 heads: 148 thread blocks
LENGTHS = [1900, 2048, 1985, 2111]


def engine(qkvlib, H, n_slots, Hk):
    eng = qkvlib.Engine(n_layer=1, n_head=16, n_head_kv=2, n_ctx=256, n_slots=n_slots, n_pages=1, rec_n_layer=1, rec_n_head=H,
                        conv_channels=(2 * Hk + H) * HD, device=0)
    for s in range(n_slots):
        eng.seq_alloc(s)
    return eng


def offsets(lengths):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


def run(qkvlib, lengths, q, k, v, g, beta, H, Hk, times=1, S0=None):
    """`times` runs from the same states, the same bits each time: the first states, the last ones, the output."""
    n, rows = len(lengths), sum(lengths)
    eng = engine(qkvlib, H, n, Hk)
    if S0 is None:
        S0 = torch.randn(n, H, HD, HD, generator=torch.Generator().manual_seed(91)).cuda() * 0.3
    S, first = eng.rec_state(0), None
    for i in range(times):
        S.copy_(S0)
        out = torch.full((rows, H, HD), 7.0, dtype=torch.bfloat16, device="cuda")
        eng.rec_chunk(0, list(range(n)), offsets(lengths), q, k, v, g, beta, SCALE, out)
        torch.cuda.synchronize()
        assert eng.device_status() == 0
        if first is None:
            first = out, S.clone()
        # (as integers: a NaN is the same NaN)
        assert torch.equal(out.view(torch.int16), first[0].view(torch.int16)), f"run {i}: {int((out != first[0]).sum())} outputs differ"
        assert torch.equal(S.view(torch.int32), first[1].view(torch.int32)), f"run {i}: the state differs"
    return S0, first[1], first[0]


@pytest.mark.parametrize("delta", [True, False])
def test_full_grid_is_the_same_every_time(cuda, qkvlib, delta):
    """Every SM at work, some 30 chunks each: the outputs' second part of a chunk is made while the next chunk's state is
    handed over, and the issuing warp is slowest then."""
    q, k, v, g, beta = inputs(92, sum(LENGTHS), FULL["H"], FULL["Hk"], torch.bfloat16, decay=0.02)
    beta = beta if delta else None
    S0, S1, out = run(qkvlib, LENGTHS, q, k, v, g, beta, **FULL, times=8)
    rec_bounds.check(S0, S1, LENGTHS, q, k, v, g, beta, out, SCALE)


@pytest.mark.parametrize("delta", [True, False])
def test_chunks_worked_token_by_token_among_others(cuda, qkvlib, delta):
    """A growing state (g > 0) sends a chunk down the path token by token: none, every, every second, third and fourth chunk
    of a head, three in a row, the first and the last."""
    lengths = [700, 577, 640, 833]
    q, k, v, g, beta = inputs(94, sum(lengths), FULL["H"], FULL["Hk"], torch.bfloat16, decay=0.02)
    at = 0
    for i, n in enumerate(lengths):
        chunks = (n + 63) // 64
        for h in range(FULL["H"]):
            kind = (h + i) % 8
            for c in range(chunks):
                if (kind in (1, 2, 3, 4) and c % kind == (h // 8) % kind) or (kind == 5 and c in (3, 4, 5)) or (kind == 6 and c in (0, chunks - 1)):
                    g[at + min(c * 64 + (5 * h + 11 * c) % 64, n - 1), h] = 0.01
        at += n
    beta = beta if delta else None
    S0, S1, out = run(qkvlib, lengths, q, k, v, g, beta, **FULL, times=4)
    rec_bounds.check(S0, S1, lengths, q, k, v, g, beta, out, SCALE)


@pytest.mark.parametrize("delta", [True, False])
def test_scores_of_another_size_in_each_chunk(cuda, qkvlib, delta):
    """Two producer groups take turns with the columns of the scores: q (and without the delta rule k) a hundred times as
    large in every second chunk, so that a score of another chunk shows."""
    lengths = [1344, 1217, 1281, 1400]
    q, k, v, g, beta = inputs(95, sum(lengths), FULL["H"], FULL["Hk"], torch.bfloat16, decay=0.02)
    at = 0
    for i, n in enumerate(lengths):
        odd = (torch.arange(n, device="cuda") // 64 + i) % 2 == 1
        size = torch.where(odd, 128.0, 1.0).bfloat16()[:, None]
        q[at:at + n] *= size
        if not delta:
            k[at:at + n] *= size
        at += n
    beta = beta if delta else None
    S0, S1, out = run(qkvlib, lengths, q, k, v, g, beta, **FULL, times=4)
    rec_bounds.check(S0, S1, lengths, q, k, v, g, beta, out, SCALE)


@pytest.mark.parametrize("at", [0, 3, 31, 33, 62, 64, 100, 190])
def test_finite_inputs_that_leave_the_range_late_in_a_chunk(cuda, qkvlib, at):
    """One key of length 10^6, repeated from row `at` on: the delta rule multiplies the state by 10^12 a token and F32 is left a
    few tokens on.  Rows before that keep their outputs, other heads are not touched, rows behind it are not finite."""
    lengths, H = [64, 200, 130], 3
    rows = sum(lengths)
    q, k, v, g, beta = inputs(96, rows, H, H, torch.bfloat16, decay=0.02)
    first = 64 + at                                     # in the second sequence, head 1
    k[first:264, HD:2 * HD] = k[first, HD:2 * HD] * 2 ** 20
    beta[first:264, 1] = 1.0
    S0, S1, out = run(qkvlib, lengths, q, k, v, g, beta, H, H, times=2)
    head = lambda x, h: x[:, h * HD:(h + 1) * HD]       # noqa: E731
    for h in (0, 2):
        rec_bounds.check(S0[:, h:h + 1], S1[:, h:h + 1], lengths, head(q, h), head(k, h), head(v, h), g[:, h:h + 1], beta[:, h:h + 1], out[:, h:h + 1], SCALE)
    for i, r in ((0, slice(0, 64)), (2, slice(264, 394))):
        rec_bounds.check(S0[i:i + 1, 1:2], S1[i:i + 1, 1:2], [lengths[i]], head(q[r], 1), head(k[r], 1), head(v[r], 1), g[r, 1:2], beta[r, 1:2], out[r, 1:2], SCALE)
    # token by token in 64 bits: the largest value of the state and of what makes it, per value row
    S, high = S0[1, 1].double(), torch.zeros(HD, dtype=torch.float64, device="cuda")
    for t in range(64, 264):
        kt, before = head(k, 1)[t].double(), high.clone()
        S = S * torch.exp(g[t, 1].double())
        u = beta[t, 1].double() * (head(v, 1)[t].double() - S @ kt)
        S = S + u[:, None] * kt
        high = torch.maximum(before, torch.maximum(S.abs().amax(1), u.abs() * kt.abs().amax()))
        finite = torch.isfinite(out[t, 1].float())
        assert bool(finite[high < 1e36].all()), f"row {t - 64}"
        assert not bool(finite[before > 1e42].any()), f"row {t - 64}"
        if bool((high < 1e36).all()):
            last = t + 1
    n = last - 64
    assert at <= n < at + 12
    if n:
        o, _, bound, _ = rec_bounds.sequence(S0[1, 1:2], *(head(x, 1)[64:last] for x in (q, k, v)), g[64:last, 1:2], beta[64:last, 1:2], SCALE)
        assert bool(((out[64:last, 1:2].double() - o).abs() <= bound).all())
    assert not torch.isfinite(S1[1, 1]).any()


def test_a_state_that_is_not_finite_stays_in_its_value_rows(cuda, qkvlib):
    lengths, H = [300, 200], 2
    q, k, v, g, beta = inputs(97, sum(lengths), H, 1, torch.bfloat16, decay=0.02)
    S0 = torch.randn(2, H, HD, HD, generator=torch.Generator().manual_seed(98)).cuda() * 0.3
    bad = S0.clone()
    bad[0, 1, 5, 7], bad[0, 1, 77, 100], bad[1, 0, 3, 3] = float("nan"), float("inf"), -float("inf")
    for d in (beta, None):
        _, S1, out = run(qkvlib, lengths, q, k, v, g, d, H, 1, S0=bad, times=2)
        rest = torch.ones(2, H, HD, dtype=torch.bool, device="cuda")
        rest[0, 1, 5] = rest[0, 1, 77] = rest[1, 0, 3] = False
        mask = torch.repeat_interleave(rest, torch.tensor(lengths, device="cuda"), 0)
        assert torch.isfinite(S1[rest]).all() and torch.isfinite(out[mask].float()).all() and not torch.isfinite(out[~mask].float()).any()
        _, S2, clean = run(qkvlib, lengths, q, k, v, g, d, H, 1, S0=S0)
        assert torch.equal(S1[rest], S2[rest]) and torch.equal(out[mask], clean[mask])


@pytest.mark.parametrize("lengths,n_keys,low", [([64], 1, 1.0), ([200, 64, 7], 1, 1.0), ([1000], 4, 1.0), ([333, 128], 2, 0.5), ([150], 1, 2.0), ([257], 3, 0.0)])
def test_repeated_keys(cuda, qkvlib, lengths, n_keys, low):
    """Few keys over and over (padding, repeated tokens), write strengths of `low` to low + 1 (2: two always, where each write
    mirrors the state): the inverse T is far from the identity, no token lengthens an error."""
    H, rows = 3, sum(lengths)
    q, k, v, g, beta = inputs(101, rows, H, H, torch.bfloat16, decay=0.002)
    pick = torch.randint(n_keys, (rows,), generator=torch.Generator().manual_seed(102)).cuda()
    k.copy_(k[pick])
    beta = torch.full_like(beta, 2.0) if low == 2.0 else beta + low
    S0, S1, out = run(qkvlib, lengths, q, k, v, g, beta, H, H, times=2)
    rec_bounds.check(S0, S1, lengths, q, k, v, g, beta, out, SCALE)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("size,at,n", [(1.75, 0, 700), (1.75, 100, 200), (1.25, 0, 2400), (3.0, 30, 40)])
def test_long_keys(cuda, qkvlib, size, at, n, delta):
    """Keys longer than one: with the delta rule a token may lengthen what it meets."""
    rows, H = 2400 if n > 700 else 700, 2
    q, k, v, g, beta = inputs(103, rows, H, 1, torch.bfloat16, decay=1e-2)
    k[at:at + n] *= size
    beta = beta if delta else None
    S0, S1, out = run(qkvlib, [rows], q, k, v, g, beta, H, 1)
    rec_bounds.check(S0, S1, [rows], q, k, v, g, beta, out, SCALE)


@pytest.mark.parametrize("piece", [2400, 333])
@pytest.mark.parametrize("what", ["nan in v", "inf in k", "nan in q", "nan in beta"])
@pytest.mark.parametrize("at", [0, 1023, 2000])
def test_values_that_are_not_finite_against_the_definition(cuda, qkvlib, what, at, piece):
    """The rows and value rows that the 64-bit recurrence leaves finite are finite and within bounds, and no others; in calls whose
    chunks begin at other rows too."""
    rows, H = 2400, 2
    q, k, v, g, beta = inputs(104, rows, H, 2, torch.bfloat16, decay=1e-2)
    where, value = what.split(" in ")[1], float(what.split(" ")[0])
    if where == "beta":
        beta[at, 1] = value
    else:
        dict(q=q, k=k, v=v)[where][at, HD + 5] = value
    eng = engine(qkvlib, H, 1, 2)
    S0 = torch.randn(1, H, HD, HD, generator=torch.Generator().manual_seed(105)).cuda() * 0.3
    eng.rec_state(0).copy_(S0)
    out = torch.full((rows, H, HD), 7.0, dtype=torch.bfloat16, device="cuda")
    for a in range(0, rows, piece):
        r = slice(a, min(a + piece, rows))
        eng.rec_chunk(0, [0], offsets([r.stop - r.start]), q[r], k[r], v[r], g[r], beta[r], SCALE, out[r])
    torch.cuda.synchronize()
    S1 = eng.rec_state(0)
    head = lambda x, h: x[:, h * HD:(h + 1) * HD]       # noqa: E731
    # the other head as if nothing were there, and this one up to the row
    o, S, bound, E = rec_bounds.sequence(S0[0, :1], *(head(x, 0) for x in (q, k, v)), g[:, :1], beta[:, :1], SCALE, piece)
    assert bool(((out[:, :1].double() - o).abs() <= bound).all())
    assert bool(((S1[0, :1].double() - S).flatten(1).norm(dim=1) <= E).all())
    if at:
        o, _, bound, _ = rec_bounds.sequence(S0[0, 1:], *(head(x, 1)[:at] for x in (q, k, v)), g[:at, 1:], beta[:at, 1:], SCALE, piece)
        assert bool(((out[:at, 1:].double() - o).abs() <= bound).all())
    # from the row on: finite where the definition is
    S, finite = S0[0, 1].double(), torch.empty(rows, HD, dtype=torch.bool, device="cuda")
    for t in range(rows):
        kt = head(k, 1)[t].double()
        S = S * torch.exp(g[t, 1].double())
        u = beta[t, 1].double() * (head(v, 1)[t].double() - S @ kt)
        S = S + u[:, None] * kt
        finite[t] = torch.isfinite(S @ head(q, 1)[t].double())
    assert torch.equal(torch.isfinite(out[:, 1].float()), finite)
    assert torch.equal(torch.isfinite(S1[0, 1]), torch.isfinite(S))


def test_a_first_token_near_the_end_of_the_range(cuda, qkvlib):
    """u of a chunk's first token between 3.0e38 and the largest F32 value is a number like any other."""
    q, k, v, g, beta = inputs(106, 64, 1, 1, torch.bfloat16, decay=1e-3)
    v[0, 5], v[0, 6] = 3.3e38, -3.2e38
    v[1:] = 0
    k.zero_()
    k[0, 9] = 1.0
    beta[0] = 1.0
    S0 = torch.zeros(1, 1, HD, HD, device="cuda")
    _, S1, out = run(qkvlib, [64], q, k, v, g, beta, 1, 1, S0=S0)
    assert torch.isfinite(S1).all() and float(S1[0, 0, 5, 9]) > 2e38 and torch.isfinite(out.float()).all()
    rec_bounds.check(S0, S1, [64], q, k, v, g, beta, out, SCALE)
