"""The recurrent layers' kernels (convolution, linear attention with a decay per head, gated delta rule) over
the engine's state slabs, against their definitions in 64 bits."""
from __future__ import annotations

import pytest
import torch

from rec_reference import HD, convolution, inputs, recurrence

pytestmark = pytest.mark.gpu
SCALE = HD ** -0.5


def rec_engine(qkvlib, H=4, Hk=2, n_slots=8, n_rollback=0, channels=None, layers=2):
    eng = qkvlib.Engine(n_layer=1, n_head=16, n_head_kv=2, n_ctx=256, n_slots=n_slots, n_pages=1, rec_n_layer=layers,
                        rec_n_head=H, conv_channels=channels or (2 * Hk + H) * HD, n_rollback=n_rollback, device=0)
    for s in range(n_slots):
        eng.seq_alloc(s)
    return eng


def fill(eng, seed, kind=0, layer=0, scale=0.3):
    S = eng.rec_state(layer, kind)
    S.copy_(torch.randn(S.shape, generator=torch.Generator().manual_seed(seed)) * scale)
    return S.clone()


def heads(x):
    return x.unflatten(-1, (-1, HD))


def offsets(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def within(got, ref, bound, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / bound.clamp(min=1e-300)).max()):.2f} of the bound"


# A token costs a state value: one rounding of e^g (2 steps of expf), of e^g S and of the sum; u the
# roundings of a dot product in 16 + 3 steps, a difference and a product; the output 19 more: under 32 half
# steps of 2^-24 of the same sums over absolute values per token.
STEP = 32 * 2.0 ** -24


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("n_seq,T,H,Hk", [(1, 1, 4, 2), (3, 2, 4, 4), (2, 4, 6, 2), (5, 3, 3, 1), (70, 1, 2, 1)])
def test_step(cuda, qkvlib, n_seq, T, H, Hk, delta):
    eng = rec_engine(qkvlib, H, Hk, n_slots=n_seq + 2)
    S0 = fill(eng, 1, layer=1)
    slots = [(5 * i + 1) % (n_seq + 2) for i in range(n_seq)] if (n_seq + 2) % 5 else list(range(n_seq))
    q, k, v, g, beta = inputs(2, n_seq * T, H, Hk, torch.float32)
    out = torch.full((n_seq * T, H, HD), float("nan"), device="cuda")
    other = eng.rec_state(0).clone()
    eng.rec_step(1, slots, q, k, v, g, beta if delta else None, T, SCALE, out)
    torch.cuda.synchronize()
    S1 = eng.rec_state(1)
    for i, s in enumerate(slots):
        r = slice(i * T, i * T + T)
        o, states, W, A = recurrence(S0[s], heads(q[r]), heads(k[r]), heads(v[r]), g[r], beta[r] if delta else None, SCALE)
        within(out[r], o, T * STEP * W, f"out of sequence {i}")
        within(S1[s], states[-1], T * STEP * A[-1], f"state of slot {s}")
    for s in set(range(n_seq + 2)) - set(slots):
        assert torch.equal(S1[s], S0[s])
    assert torch.equal(eng.rec_state(0), other) and eng.device_status() == 0


@pytest.mark.parametrize("T,n_rollback", [(1, 1), (3, 3), (4, 2), (2, 4)])
def test_step_and_conv_save_rollback_states(cuda, qkvlib, T, n_rollback):
    H, Hk = 4, 2
    eng = rec_engine(qkvlib, H, Hk, n_slots=2, n_rollback=n_rollback)
    S0, h0 = fill(eng, 3), fill(eng, 4, kind=1)
    q, k, v, g, beta = inputs(5, 2 * T, H, Hk, torch.float32)
    out = torch.empty(2 * T, H, HD, device="cuda")
    x = torch.randn(2 * T, 8 * HD, device="cuda")
    w = torch.randn(8 * HD, 4, device="cuda")
    y = torch.empty_like(x)
    slots = [1, 0]
    eng.rec_conv(0, slots, offsets([T, T]), x, w, y, save=True)
    eng.rec_step(0, slots, q, k, v, g, beta, T, SCALE, out, save=True)
    torch.cuda.synchronize()
    depth = min(T, n_rollback)
    want = {}
    for i, s in enumerate(slots):
        r = slice(i * T, i * T + T)
        _, states, _, A = recurrence(S0[s], heads(q[r]), heads(k[r]), heads(v[r]), g[r], beta[r], SCALE)
        _, hists = convolution(h0[s], x[r], w, 0, 1e-6)
        assert torch.equal(eng.rec_state(0, 1)[s].double(), hists[T])
        for back in range(1, depth + 1):
            # (the sums of that moment: a later decay makes the ones of the end smaller)
            within(eng.rec_state(0, 0, back)[s], states[T - back], T * STEP * A[T - back], f"{back} back")
            assert torch.equal(eng.rec_state(0, 1, back)[s].double(), hists[T - back])
            want[s, back] = eng.rec_state(0, 0, back)[s].clone(), eng.rec_state(0, 1, back)[s].clone()
    if depth == T:
        assert torch.equal(eng.rec_state(0, 0, T), S0)
    # the engine's own rollback takes them: K/V rows for the positions, then one token back
    eng.append(0, 0, 0, torch.randn(T, 512, device="cuda"), torch.randn(T, 512, device="cuda"))
    eng.rollback_arm(0, depth)
    eng.rollback_n(0, depth)
    torch.cuda.synchronize()
    assert eng.n_past(0) == T - depth
    assert torch.equal(eng.rec_state(0, 0)[0], want[0, depth][0]) and torch.equal(eng.rec_state(0, 1)[0], want[0, depth][1])


def test_step_forgets_at_minus_infinity(cuda, qkvlib):
    eng = rec_engine(qkvlib, 2, 1, n_slots=1)
    fill(eng, 6, scale=1e3)
    q, k, v, g, beta = inputs(7, 1, 2, 1, torch.float32)
    g.fill_(-float("inf"))
    out = torch.empty(1, 2, HD, device="cuda")
    eng.rec_step(0, [0], q, k, v, g, None, 1, SCALE, out)
    assert torch.equal(eng.rec_state(0)[0], heads(v)[0][:, :, None] * heads(k)[0][:, None, :])


# A chunk of 64 tokens: state and sums in 32 bits, products of operands split so that a factor is off by at most
# 2^-22 of its row's largest value; under 64 half steps of 2^-24 of the sums over absolute values for
# each 64 tokens and the ones that the first state carries.  The output meets three operands cut to 16
# bits (the state, the scores, u), under 2^-15 each of those sums (2^-11 is allowed), and its own rounding, 2^-8 of the
# value.
CHUNK = 64 * 2.0 ** -24


def check_chunk(eng, S0, slots, lengths, q, k, v, g, beta, out, layer=0, scale=SCALE):
    at, S1 = 0, eng.rec_state(layer)
    for i, (s, n) in enumerate(zip(slots, lengths)):
        r = slice(at, at + n)
        at += n
        o, states, W, A = recurrence(S0[s], heads(q[r]), heads(k[r]), heads(v[r]), g[r], None if beta is None else beta[r], scale)
        steps = (n + 63) // 64 + 1
        within(out[r], o, 2.0 ** -8 * o.abs() + 3 * 2.0 ** -11 * W + 1e-30, f"out of sequence {i} ({n} rows)")
        if n:
            rel = float((S1[s].double() - states[-1]).norm() / A[-1].norm())
            assert rel <= steps * CHUNK, f"state of sequence {i}: {rel:.2e}"
        within(S1[s], states[-1], steps * CHUNK * A[-1].amax((-1,), keepdim=True) + 1e-30, f"state of slot {s} ({n} rows)")
        if n == 0:
            assert torch.equal(S1[s], S0[s])


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("lengths,H,Hk", [([1], 2, 1), ([64], 4, 2), ([65, 0, 1], 4, 4), ([63, 130, 7, 64], 6, 2),
                                          ([0, 0, 200], 3, 1), ([15, 16, 17, 31, 33, 49], 2, 2), ([517], 4, 2)])
def test_chunk(cuda, qkvlib, lengths, H, Hk, delta):
    n = len(lengths)
    eng = rec_engine(qkvlib, H, Hk, n_slots=n + 1)
    S0 = fill(eng, 11)
    slots = list(range(n, 0, -1))
    rows = sum(lengths)
    q, k, v, g, beta = inputs(12, rows + 3, H, Hk, torch.bfloat16, decay=0.05)
    out = torch.full((rows + 3, H, HD), 7.0, dtype=torch.bfloat16, device="cuda")
    eng.rec_chunk(0, slots, offsets(lengths), q, k, v, g, beta if delta else None, SCALE, out)
    torch.cuda.synchronize()
    assert eng.device_status() == 0
    check_chunk(eng, S0, slots, lengths, q, k, v, g, beta if delta else None, out)
    assert bool((out[rows:] == 7.0).all()) and torch.equal(eng.rec_state(0)[0], S0[0])   # rows and slots of nobody


def test_chunk_many_sequences(cuda, qkvlib):
    """More sequences than a launch takes, more heads and sequences than the GPU holds at once."""
    lengths = [(37 * i) % 131 for i in range(70)]
    eng = rec_engine(qkvlib, 4, 1, n_slots=70)
    S0 = fill(eng, 25)
    q, k, v, g, beta = inputs(26, sum(lengths), 4, 1, torch.bfloat16, decay=0.05)
    out = torch.empty(sum(lengths), 4, HD, dtype=torch.bfloat16, device="cuda")
    slots = [(i * 11) % 70 for i in range(70)]
    eng.rec_chunk(0, slots, offsets(lengths), q, k, v, g, beta, SCALE, out)
    check_chunk(eng, S0, slots, lengths, q, k, v, g, beta, out)
    assert eng.device_status() == 0


def test_chunk_growing_state(cuda, qkvlib):
    """g > 0 in one chunk: a growing state, token by token."""
    eng = rec_engine(qkvlib, 2, 1, n_slots=1)
    S0 = fill(eng, 27)
    q, k, v, g, beta = inputs(28, 300, 2, 1, torch.bfloat16, decay=0.05)
    g[130:135] = 0.5
    out = torch.empty(300, 2, HD, dtype=torch.bfloat16, device="cuda")
    eng.rec_chunk(0, [0], offsets([300]), q, k, v, g, beta, SCALE, out)
    check_chunk(eng, S0, [0], [300], q, k, v, g, beta, out)


@pytest.mark.parametrize("decay", [0.0, 1e-4, 3.0, 60.0])
def test_chunk_decays(cuda, qkvlib, decay):
    """No decay at all, and decays whose sums over a chunk are far below the smallest exponent."""
    eng = rec_engine(qkvlib, 2, 1, n_slots=1)
    S0 = fill(eng, 13)
    q, k, v, g, beta = inputs(14, 200, 2, 1, torch.bfloat16, decay=decay)
    out = torch.empty(200, 2, HD, dtype=torch.bfloat16, device="cuda")
    eng.rec_chunk(0, [0], offsets([200]), q, k, v, g, beta, SCALE, out)
    check_chunk(eng, S0, [0], [200], q, k, v, g, beta, out)


def test_chunk_forgets_at_minus_infinity(cuda, qkvlib):
    """A state forgotten in the middle of a chunk, twice: nothing before it is left, nothing is NaN."""
    eng = rec_engine(qkvlib, 2, 1, n_slots=1)
    S0 = fill(eng, 15)
    q, k, v, g, beta = inputs(16, 150, 2, 1, torch.bfloat16, decay=0.05)
    g[20] = g[90, 0] = g[91] = -float("inf")
    out = torch.empty(150, 2, HD, dtype=torch.bfloat16, device="cuda")
    eng.rec_chunk(0, [0], offsets([150]), q, k, v, g, beta, SCALE, out)
    check_chunk(eng, S0, [0], [150], q, k, v, g, beta, out)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("qs,ks,vs,ss", [(1e3, 0.05, 1e-6, 1e-3), (1e-4, 1.0, 1e5, 1e5), (1e-20, 1e-3, 1e20, 1e-20), (1.0, 1.0, 0.0, 1.0)])
def test_chunk_magnitudes(cuda, qkvlib, qs, ks, vs, ss, delta):
    """Values far from one: no operand's rounding may depend on a fixed range."""
    eng = rec_engine(qkvlib, 2, 1, n_slots=1)
    S0 = fill(eng, 17, scale=ss)
    q, k, v, g, beta = inputs(18, 130, 2, 1, torch.bfloat16, decay=0.05)
    q, k, v = q * qs, k * ks, v * vs
    out = torch.empty(130, 2, HD, dtype=torch.bfloat16, device="cuda")
    eng.rec_chunk(0, [0], offsets([130]), q, k, v, g, beta if delta else None, SCALE, out)
    check_chunk(eng, S0, [0], [130], q, k, v, g, beta if delta else None, out)


def test_chunk_not_a_number_stays_in_its_head_and_rows(cuda, qkvlib):
    eng = rec_engine(qkvlib, 2, 2, n_slots=2)
    S0 = fill(eng, 19)
    q, k, v, g, beta = inputs(20, 140, 2, 2, torch.bfloat16, decay=0.05)
    v[70, :HD] = float("nan")          # head 0 of the second sequence
    q[139, HD:] = float("inf")
    out = torch.empty(140, 2, HD, dtype=torch.bfloat16, device="cuda")
    lengths = [66, 74]
    eng.rec_chunk(0, [0, 1], offsets(lengths), q, k, v, g, beta, SCALE, out)
    S1 = eng.rec_state(0)
    assert torch.isfinite(out[:70]).all() and torch.isfinite(S1[0]).all() and torch.isfinite(S1[1, 1]).all()
    assert torch.isfinite(out[70:139, 1]).all() and not torch.isfinite(out[139, 1]).any()
    assert torch.isnan(out[70:, 0]).all() and torch.isnan(S1[1, 0]).all()
    check_chunk(eng, S0, [0], [66], q[:66], k[:66], v[:66], g[:66], beta[:66], out[:66])


def test_chunk_is_the_same_twice_and_continues(cuda, qkvlib):
    """The same bits on every run; a prompt in two calls, then single tokens, is the prompt in one."""
    H, Hk, n = 4, 2, 200
    q, k, v, g, beta = inputs(21, n, H, Hk, torch.bfloat16, decay=0.05)
    outs, states = [], []
    for cut in (n, n, 96):
        eng = rec_engine(qkvlib, H, Hk, n_slots=1)
        S0 = fill(eng, 22)
        out = torch.empty(n, H, HD, dtype=torch.bfloat16, device="cuda")
        for a, b in ((0, cut), (cut, n)):
            if b > a:
                eng.rec_chunk(0, [0], offsets([b - a]), q[a:b], k[a:b], v[a:b], g[a:b], beta[a:b], SCALE, out[a:b])
        outs.append(out)
        states.append(eng.rec_state(0).clone())
        check_chunk(eng, S0, [0], [n], q, k, v, g, beta, out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(states[0], states[1])


def long_reference(S, q, k, v, g, beta, scale):
    """One long sequence in 64 bits: out, the last state, and the largest norm of a head's state on the way."""
    S, q, k, v, e, beta = S.double(), heads(q).double(), heads(k).double(), heads(v).double(), torch.exp(g.double()), beta.double()
    n = S.shape[0] // q.shape[1]
    q, k = q.repeat_interleave(n, 1), k.repeat_interleave(n, 1)
    out, most = torch.empty_like(v), S.flatten(1).norm(dim=1)
    for t in range(v.shape[0]):
        S = S * e[t, :, None, None]
        u = beta[t, :, None] * (v[t] - (S * k[t, :, None, :]).sum(-1))
        S = S + u[:, :, None] * k[t, :, None, :]
        out[t] = scale * (S * q[t, :, None, :]).sum(-1)
        most = torch.maximum(most, S.flatten(1).norm(dim=1))
    return out, S, most


def in_pieces(eng, slots, lengths, q, k, v, g, beta, out, piece=1024):
    """The same sequences, `piece` rows to a call."""
    at = 0
    for s, n in zip(slots, lengths):
        for a in range(at, at + n, piece):
            r = slice(a, min(a + piece, at + n))
            eng.rec_chunk(0, [s], offsets([r.stop - r.start]), q[r], k[r], v[r], g[r], beta[r], SCALE, out[r])
        at += n


@pytest.mark.parametrize("lengths,H,Hk,decay", [([2048], 4, 2, 1e-3), ([2049, 4161, 2500], 3, 3, 1e-3), ([3000, 0, 4000], 2, 1, 0.3),
                                                ([5000, 1500, 77], 2, 2, 1e-5)])
def test_chunk_long_sequences(cuda, qkvlib, lengths, H, Hk, decay):
    """Many chunks, in one call and in calls of 1024 rows."""
    n, rows = len(lengths), sum(lengths)
    engs = [rec_engine(qkvlib, H, Hk, n_slots=n, layers=1) for _ in range(2)]
    S0 = fill(engs[0], 61, scale=1.0)
    fill(engs[1], 61, scale=1.0)
    q, k, v, g, beta = inputs(62, rows, H, Hk, torch.bfloat16, decay=decay)
    out, other = (torch.full((rows + 1, H, HD), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    engs[0].rec_chunk(0, list(range(n)), offsets(lengths), q, k, v, g, beta, SCALE, out)
    in_pieces(engs[1], range(n), lengths, q, k, v, g, beta, other)
    assert bool((out[rows] == 7.0).all())
    S1, S2, at = engs[0].rec_state(0), engs[1].rec_state(0), 0
    for i, m in enumerate(lengths):
        r = slice(at, at + m)
        at += m
        ref, S, most = long_reference(S0[i], q[r], k[r], v[r], g[r], beta[r], SCALE)
        # keys of length one, beta below one and no growth: no token lengthens an error, so each chunk adds its own, under
        # 64 half steps of 2^-24 of the state's norm; the output is rounded once, 2^-8, its operands by less than a
        # tenth of that
        for what, got in (("whole", S1[i]), ("pieces", S2[i])):
            err = (got.double() - S).flatten(1).norm(dim=1)
            assert bool((err <= ((m + 63) // 64 + 1) * CHUNK * most).all()), f"{what}, state of sequence {i}: {float((err / most).max()):.2e}"
        if m:
            for what, got in (("whole", out[r]), ("pieces", other[r])):
                rel = ((got.double() - ref).flatten().norm() / ref.flatten().norm()).item()
                assert rel <= 1.1 * 2.0 ** -8, f"{what}, out of sequence {i}: {rel:.2e}"


@pytest.mark.parametrize("what", ["nan", "inf in k", "nan in q", "grows", "long keys"])
@pytest.mark.parametrize("at", [100, 1000, 2000])
def test_chunk_long_sequences_out_of_range(cuda, qkvlib, what, at):
    """A value early, in the middle and late that is not finite, or a state that grows: as in calls of 1024 rows."""
    m, H = 2400, 2
    engs = [rec_engine(qkvlib, H, 1, n_slots=1, layers=1) for _ in range(2)]
    for e in engs:
        fill(e, 63)
    q, k, v, g, beta = inputs(64, m, H, 1, torch.bfloat16, decay=1e-2)
    if what == "nan":
        v[at, 5] = float("nan")
    elif what == "inf in k":
        k[at, 3] = float("inf")
    elif what == "nan in q":
        q[at, 3] = float("nan")
    elif what == "grows":
        g[at, 1] = 0.25
    else:
        k[at:at + 200] *= 1.75
    outs = [torch.zeros(m, H, HD, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    engs[0].rec_chunk(0, [0], offsets([m]), q, k, v, g, beta, SCALE, outs[0])
    in_pieces(engs[1], [0], [m], q, k, v, g, beta, outs[1])
    for a, b, tol in ((engs[0].rec_state(0), engs[1].rec_state(0), 2 * 39 * CHUNK), (*outs, 2.2 * 2.0 ** -8)):
        assert torch.equal(a.isfinite(), b.isfinite())
        a, b = (x.double().nan_to_num(0.0, 0.0, 0.0) for x in (a, b))
        assert float((a - b).norm()) <= tol * float(b.norm())


def test_chunk_bad_offsets_are_reported(cuda, qkvlib):
    eng = rec_engine(qkvlib, 2, 1, n_slots=3)
    S0 = fill(eng, 23)
    q, k, v, g, beta = inputs(24, 40, 2, 1, torch.bfloat16)
    out = torch.zeros(40, 2, HD, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 10, 5, 41], dtype=torch.int32, device="cuda")   # falls, then passes the rows
    eng.rec_chunk(0, [0, 1, 2], cu, q, k, v, g, beta, SCALE, out)
    assert eng.device_status() == 2
    check_chunk(eng, S0, [0], [10], q, k, v, g, beta, out)
    assert torch.equal(eng.rec_state(0)[1:], S0[1:]) and not out[10:].any()


# ------------------------------------------------------------------------------------ convolution
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths,channels,n_norm", [([1], 128, 0), ([2, 1, 3, 4], 1024, 512), ([0, 5, 0, 300], 384, 384),
                                                     ([1] * 70, 640, 256), ([97, 3], 8192, 4096)])
def test_conv(cuda, qkvlib, lengths, channels, n_norm, dtype):
    n, rows = len(lengths), sum(lengths)
    eng = rec_engine(qkvlib, 2, 1, n_slots=n + 1, channels=channels)
    h0 = fill(eng, 31, kind=1, layer=1, scale=1.0)
    gen = torch.Generator().manual_seed(32)
    wide = torch.randn(rows + 2, channels + 64, generator=gen).to(dtype).cuda()
    x = wide[:, 64:]
    w = torch.randn(channels, 4, generator=gen).cuda()
    y = torch.full((rows + 2, channels), 7.0, dtype=dtype, device="cuda")
    slots = list(range(n, 0, -1))
    eng.rec_conv(1, slots, offsets(lengths), x, w, y, n_norm=n_norm)
    torch.cuda.synchronize()
    at, h1 = 0, eng.rec_state(1, 1)
    # four products and sums, an exponential, a division; the norm a root and a sum of 128 squares: under
    # 32 half steps of 2^-24 of the sum over absolute values (silu's slope is at most 1.1), then y's rounding
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    for i, (s, m) in enumerate(zip(slots, lengths)):
        r = slice(at, at + m)
        at += m
        ref, hists = convolution(h0[s], x[r], w, n_norm, 1e-6)
        z = torch.cat([h0[s].double().T, x[r].double()]).abs()
        bound = sum(z[j:j + m] * w[:, j].double().abs() for j in range(4)) * 32 * 2.0 ** -24
        if n_norm:
            raw, _ = convolution(h0[s], x[r], w, 0, 1e-6)
            size = raw[:, :n_norm].reshape(m, n_norm // HD, HD).norm(dim=-1, keepdim=True)
            bound[:, :n_norm] = (bound[:, :n_norm].reshape(m, n_norm // HD, HD) / size).reshape(m, n_norm) + 32 * 2.0 ** -24
        within(y[r], ref, bound + half * ref.abs(), f"y of sequence {i}")
        assert torch.equal(h1[s].double(), hists[m])
    assert bool((y[rows:] == 7.0).all()) and torch.equal(h1[0], h0[0])


@pytest.mark.parametrize("ahead,dtype", [(1, torch.bfloat16), (2, torch.bfloat16), (2, torch.float32)])
def test_conv_history_is_read_before_it_is_replaced(cuda, qkvlib, ahead, dtype):
    """Sequences that start one or two rows before a multiple of four, those among them where a wave of thread blocks
    ends: a thread whose rows begin just behind a sequence's start needs what the start replaces."""
    channels, n = 8192, 24
    step = 4 * (2 * torch.cuda.get_device_properties(0).multi_processor_count * 256 * 8 // channels)
    lengths = [step - ahead] + [step] * (n - 1)
    rows, gen = sum(lengths), torch.Generator().manual_seed(35)
    engs = [rec_engine(qkvlib, 2, 1, n_slots=n, channels=channels, layers=1) for _ in range(2)]
    for e in engs:
        fill(e, 36, kind=1, scale=1.0)
    x = torch.randn(rows, channels, generator=gen).to(dtype).cuda()
    w = torch.randn(channels, 4, generator=gen).cuda()
    y, alone = torch.empty_like(x), torch.empty_like(x)
    engs[0].rec_conv(0, list(range(n)), offsets(lengths), x, w, y, n_norm=4096)
    at = 0
    for i, m in enumerate(lengths):   # a sequence's first three rows as a call of their own
        engs[1].rec_conv(0, [i], offsets([3]), x[at:at + 3], w, alone[at:at + 3], n_norm=4096)
        assert torch.equal(y[at:at + 3], alone[at:at + 3]), f"sequence {i}"
        at += m


def test_conv_zero_head(cuda, qkvlib):
    eng = rec_engine(qkvlib, 2, 1, n_slots=1, channels=256)
    eng.reset(0)
    x = torch.zeros(3, 256, device="cuda")
    y = torch.full_like(x, float("nan"))
    eng.rec_conv(0, [0], offsets([3]), x, torch.ones(256, 4, device="cuda"), y, n_norm=128)
    assert torch.equal(y, torch.zeros_like(y))


# ------------------------------------------------------------------------------ streams and graphs
def test_captured_and_replayed(cuda, qkvlib):
    """One captured decode step (convolution, recurrence) replayed on another stream: the state moves on."""
    H, Hk, n, T = 4, 2, 3, 2
    engs = [rec_engine(qkvlib, H, Hk, n_slots=n) for _ in range(2)]
    ch = 8 * HD
    gen = torch.Generator().manual_seed(41)
    x = torch.randn(3, n * T, ch, generator=gen).cuda()
    g = -torch.rand(n * T, H, generator=gen).cuda()
    beta = torch.rand(n * T, H, generator=gen).cuda()
    w = torch.randn(ch, 4, generator=gen).cuda()
    cu = offsets([T] * n)

    def step(eng, xin, y, out):
        eng.rec_conv(0, list(range(n)), cu, xin, w, y, n_norm=4 * HD)
        eng.rec_step(0, list(range(n)), y[:, :2 * HD], y[:, 2 * HD:4 * HD], y[:, 4 * HD:], g, beta, T, SCALE, out)

    want = []
    for e in engs:
        fill(e, 42)
        fill(e, 43, kind=1)
    y, out = torch.empty(n * T, ch, device="cuda"), torch.empty(n * T, H, HD, device="cuda")
    for i in range(3):
        step(engs[0], x[i], y, out)
        want.append(out.clone())
    side = torch.cuda.Stream()
    xin = x[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(engs[1], xin, y, out)
    for i in range(3):
        xin.copy_(x[i])
        graph.replay()
        assert torch.equal(out, want[i])
    assert torch.equal(engs[0].rec_state(0), engs[1].rec_state(0))


def test_layers_on_two_streams_at_once(cuda, qkvlib):
    """Calls share nothing but the engine: two layers' prompts and steps on two streams, eager beside a replayed graph."""
    H, Hk, lengths = 4, 2, [700, 65, 1300]
    n, rows = len(lengths), sum(lengths)
    eng, other = (rec_engine(qkvlib, H, Hk, n_slots=n) for _ in range(2))
    cu, ch = offsets(lengths), (2 * Hk + H) * HD
    gen = torch.Generator().manual_seed(71)
    x = [torch.randn(rows, ch, generator=gen).bfloat16().cuda() for _ in range(2)]
    w = torch.randn(ch, 4, generator=gen).cuda()
    g, beta = -torch.rand(rows, H, generator=gen).cuda(), torch.rand(rows, H, generator=gen).cuda()
    y, out = [torch.empty_like(x[0]) for _ in range(2)], [torch.empty(rows, H, HD, dtype=torch.bfloat16, device="cuda") for _ in range(2)]

    def prompt(e, layer, y, out):
        e.rec_conv(layer, list(range(n)), cu, x[layer], w, y, n_norm=2 * Hk * HD)
        e.rec_chunk(layer, list(range(n)), cu, y[:, :Hk * HD], y[:, Hk * HD:2 * Hk * HD], y[:, 2 * Hk * HD:], g, beta, SCALE, out)

    want = []
    for layer in range(2):
        for e in (eng, other):
            fill(e, 72 + layer, layer=layer)
            fill(e, 74 + layer, kind=1, layer=layer)
        prompt(other, layer, y[0], out[0])
        prompt(other, layer, y[0], out[0])
        want.append(out[0].clone())
    streams = [torch.cuda.Stream() for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        prompt(eng, 0, y[0], out[0])
    torch.cuda.synchronize()
    for _ in range(2):
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            prompt(eng, 1, y[1], out[1])
    torch.cuda.synchronize()
    for layer in range(2):
        assert torch.equal(out[layer], want[layer])
        for kind in range(2):
            assert torch.equal(eng.rec_state(layer, kind), other.rec_state(layer, kind))
