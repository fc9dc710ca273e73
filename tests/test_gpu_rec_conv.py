"""The ragged convolution's walks through their ring of copies, every row against the definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

from rec_reference import HD

pytestmark = pytest.mark.gpu


def definition(hist, x, w, n_norm, eps, lengths):
    """Rows of all sequences at once.  Returns y, its error bound without the last rounding, the histories after."""
    y, bound, after, at = [], [], [], 0
    w = w.double()
    for i, m in enumerate(lengths):
        z = torch.cat([hist[i].double().T, x[at:at + m].double()])
        at += m
        a = sum(z[j:j + m] * w[:, j] for j in range(4))
        # four products and sums, an exponential, a division; the norm a root and a sum of 128 squares: under 32 half steps of
        # 2^-24 of the sum over absolute values (silu's slope is at most 1.1)
        d = sum(z[j:j + m].abs() * w[:, j].abs() for j in range(4)) * 32 * 2.0 ** -24
        a = a / (1 + torch.exp(-a))
        if n_norm:
            head = a[:, :n_norm].reshape(m, n_norm // HD, HD)
            size = torch.clamp(head.norm(dim=-1, keepdim=True), min=eps)
            a[:, :n_norm] = (head / size).reshape(m, n_norm)
            d[:, :n_norm] = (d[:, :n_norm].reshape(m, n_norm // HD, HD) / size).reshape(m, n_norm) + 32 * 2.0 ** -24
        y.append(a)
        bound.append(d)
        after.append(z[m:].T)
    return torch.cat(y), torch.cat(bound), torch.stack(after)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths,spare", [([100 + (89 * i) % 201 for i in range(80)], 70), ([203] * 50, 5), ([1, 2, 3, 4, 5, 6, 7] * 150, 0)])
def test_every_row_of_long_walks(cuda, qkvlib, lengths, spare, dtype):
    """Walks of tens of rows, starts of sequences at every offset of a walk; more sequences than a launch takes (each
    launch passes over the rows of the others), rows of no sequence behind the last."""
    channels, n_norm = 8192, 4096
    n, rows = len(lengths), sum(lengths)
    eng = qkvlib.Engine(n_layer=1, n_head=16, n_head_kv=2, n_ctx=256, n_slots=n, n_pages=1, rec_n_layer=1, rec_n_head=1,
                        rec_head_dim=128, conv_channels=channels, device=0)
    for s in range(n):
        eng.seq_alloc(s)
    gen = torch.Generator(device="cuda").manual_seed(93)
    hist = eng.rec_state(0, 1)
    first = torch.randn(n, channels, 3, device="cuda", generator=gen)
    hist.copy_(first)
    x = torch.randn(rows + spare, channels, device="cuda", generator=gen).to(dtype)
    w = torch.randn(channels, 4, device="cuda", generator=gen)
    y = torch.full((rows + spare, channels), 7.0, dtype=dtype, device="cuda")
    cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    eng.rec_conv(0, list(range(n)), cu, x, w, y, n_norm=n_norm)
    torch.cuda.synchronize()
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    at = 0
    for a in range(0, n, 16):
        part = lengths[a:a + 16]
        r = slice(at, at + sum(part))
        at = r.stop
        ref, bound, after = definition(first[a:a + 16], x[r], w, n_norm, 1e-6, part)
        bad = ~((y[r].double() - ref).abs() <= bound + half * (ref.abs() + bound))
        assert not bad.any(), f"sequences {a} ..: {int(bad.sum())} values in rows {bad.any(1).nonzero().flatten()[:20].tolist()}"
        assert torch.equal(hist[a:a + 16].double(), after)
    assert bool((y[rows:] == 7.0).all())
