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
