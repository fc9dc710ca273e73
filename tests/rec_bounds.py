"""How far the chunked recurrence may be off, chunk by chunk, from quantities of the 64-bit recurrence itself.

Sums over absolute values along a whole sequence grow by a factor per token and bound nothing after a few
chunks.  Here each chunk of 64 tokens adds what its own roundings can add, and the error of the state it starts from goes
through the chunk's true transition.  H = half a step of 2^-24 of F32, per chunk with G = sums of g, A, T = (1 + A)^-1,
R_j = beta_j (v_j - e^(G_j) S k_j), U = T R, P_ij = (q_i . k_j) e^(G_i - G_j):

* R: a dot product of 128, two products and a difference, or token by token the sum in order: 160 H of
  beta (|v| + e^G |S| |k|).  Split into two f16 terms of a scaled row: 2^-22 of the row's largest of 32 tokens.
* T: the entries of A (a dot product, decays from two exponentials) within 64 H, tiles multiplied as pairs of TF32 terms
  (each cut by under 2^-20, the product of the two rests dropped: 48 H): |dT| <= 64 H |T| |A| |T|.
* U: what R's and T's errors make of it, and 64 H of |T| |R| for its sums.
* the state: 160 H of the largest state on the way (three bf16 terms are the value; F32 sums; a product and a sum), and
  U's error times the keys; then on through the transition of the chunks after it.
* the output: the state and the scores enter as two truncated bf16 terms (each cut by under 2^-15 of the value), u too, and
  the product of two second terms (each under 2^-7) is left out: 2^-15 of |S| |q|, 2^-13 of |P| |u|, together
  under 3 * 2^-14 of their sum; U's and the state's errors; one rounding to bf16, 2^-8 of the value.
"""
from __future__ import annotations

import torch

HD, C = 128, 64
H = 2.0 ** -24


def _rows(x):
    return x.double().unflatten(-1, (-1, HD)) if x.dim() == 2 else x.double()


def spectral(Phi):
    """No less than each matrix's spectral norm, and under 1.002 times it: |(Phi^T Phi)^p|_F^(1 / 2p), p = 1024."""
    M = Phi.transpose(-1, -2) @ Phi
    log = torch.zeros(M.shape[:-2], dtype=M.dtype, device=M.device)
    for i in range(11):
        f = torch.linalg.matrix_norm(M).clamp(min=1e-300)
        log = log + torch.log(f) / 2 ** i
        M = M / f[..., None, None]
        M = M @ M
    return torch.exp(log / 2)


def sequence(S, q, k, v, g, beta, scale, piece=1 << 30):
    """One sequence from state S [heads, value, key].  Returns the 64-bit outputs [n, heads, 128] and last state, the
    outputs' bound (same shape) and the state's, a norm per head.  piece: rows of a call, where chunks begin anew."""
    S, g = S.double(), g.double()
    q, k, v = _rows(q), _rows(k), _rows(v)
    n, heads = v.shape[0], v.shape[1]
    q, k = (x.repeat_interleave(heads // x.shape[1], 1) for x in (q, k))
    b = torch.ones_like(g) if beta is None else beta.double()
    e = torch.exp(g)
    out, bound = torch.empty_like(v), torch.empty_like(v)
    E = torch.zeros(heads, dtype=torch.float64, device=v.device)
    for t0 in (t for a in range(0, n, piece) for t in range(a, min(a + piece, n), C)):
        r = slice(t0, min(t0 + C, t0 - t0 % piece + piece, n))
        m = r.stop - t0
        S0, us = S, []
        Phi = torch.eye(HD, dtype=torch.float64, device=v.device).expand(heads, HD, HD)
        size, grow, most = S.flatten(1).norm(dim=1), torch.ones_like(E), torch.ones_like(E)
        grown = []
        for t in range(t0, r.stop):
            S = S * e[t, :, None, None]
            u = v[t]
            if beta is not None:
                u = b[t, :, None] * (u - (S * k[t, :, None, :]).sum(-1))
            S = S + u[:, :, None] * k[t, :, None, :]
            out[t] = scale * (S * q[t, :, None, :]).sum(-1)
            us.append(u)
            size = torch.maximum(size, S.flatten(1).norm(dim=1))
            Phi = Phi * e[t, :, None, None]
            f = e[t]
            if beta is not None:
                Phi = Phi - (Phi * k[t, :, None, :]).sum(-1, keepdim=True) * (b[t, :, None] * k[t])[:, None, :]
                f = f * torch.clamp((1 - b[t] * k[t].square().sum(-1)).abs(), min=1.0)
            grow = grow * f
            most = torch.maximum(most, torch.clamp(f, min=1.0) * most)
            grown.append(grow)
        hd = lambda x: x[r].transpose(0, 1)                                  # noqa: E731  [heads, m, ...]
        G = g[r].cumsum(0).T                                                 # [heads, m]
        low = torch.ones(m, m, dtype=torch.bool, device=v.device).tril()
        D = torch.where(low, G[:, :, None] - G[:, None, :], torch.full_like(G[:, :, None], -float("inf"))).nan_to_num(nan=-float("inf")).exp()
        gam, end = torch.exp(G), torch.exp(torch.where(G.isinf(), torch.zeros_like(G), G[:, -1:] - G)) * (~(G[:, -1:].isinf() & ~G.isinf()))
        ks, qs, vs, U = hd(k), hd(q), hd(v), torch.stack(us, 1)              # U [heads, m, value]
        Sk = torch.einsum("hvk,hmk->hmv", S0.abs(), ks.abs()) * gam[..., None]
        if beta is not None:
            bb = b[r].T
            A = (bb[..., None] * (ks @ ks.transpose(1, 2)) * D).tril(-1)
            Aabs = (bb.abs()[..., None] * (ks.abs() @ ks.abs().transpose(1, 2)) * D).tril(-1)
            T = torch.linalg.solve_triangular(A + torch.eye(m, dtype=A.dtype, device=A.device), torch.eye(m, dtype=A.dtype, device=A.device).expand_as(A), upper=False, unitriangular=True).abs()
            R = bb[..., None] * (vs - gam[..., None] * torch.einsum("hvk,hmk->hmv", S0, ks))
            dR = 160 * H * bb.abs()[..., None] * (vs.abs() + Sk)
            for a in range(0, m, 32):
                dR[:, a:a + 32] += 2.0 ** -22 * R[:, a:a + 32].abs().amax(1, keepdim=True)
            dU = T @ dR + 64 * H * (T @ (Aabs @ (T @ R.abs()))) + 64 * H * (T @ R.abs())
        else:
            dU = torch.zeros_like(U)
        P = (qs @ ks.transpose(1, 2)).abs() * D
        W = abs(scale) * (gam[..., None] * torch.einsum("hvk,hmk->hmv", S0.abs(), qs.abs()) + P @ U.abs())
        d = abs(scale) * (P @ dU + (torch.stack(grown, 1) * E[:, None] * qs.norm(dim=-1))[..., None])
        # (a chunk worked token by token rounds the state on the way: as the state's own error below, met by q)
        d = d + abs(scale) * (160 * H * size * most)[:, None, None] * qs.norm(dim=-1)[..., None]
        d = d + 3 * 2.0 ** -14 * W
        o = out[r].abs()
        bound[r] = (d.transpose(0, 1) * (1 + 2.0 ** -8) + 2.0 ** -8 * o) + 1e-30
        E = spectral(Phi) * E + 160 * H * size * most + (end[..., None] * dU).norm(dim=-1).mul(ks.norm(dim=-1)).sum(-1)
    return out, S, bound, E + 1e-30


def check(S0, S1, lengths, q, k, v, g, beta, out, scale, what=""):
    """Sequences one after another in the rows; S0 and S1 [sequence, head, value, key].  Returns the worst ratio of the
    outputs' error to the bound and the state's error relative to its norm."""
    at, worst, rel = 0, 0.0, 0.0
    for i, n in enumerate(lengths):
        r = slice(at, at + n)
        at += n
        if n == 0:
            assert torch.equal(S1[i], S0[i]), f"{what}: state of sequence {i}"
            continue
        o, S, bound, E = sequence(S0[i], q[r], k[r], v[r], g[r], None if beta is None else beta[r], scale)
        err = (out[r].double() - o).abs()
        bad = ~(err <= bound)
        assert not bad.any(), (f"{what}: out of sequence {i}, {int(bad.sum())} of {bad.numel()} outside, first row "
                               f"{int(bad.flatten(1).any(1).nonzero()[0])} of {n}, worst {float((err / bound).max()):.2f} of the bound")
        es = (S1[i].double() - S).flatten(1).norm(dim=1)
        assert bool((es <= E).all()), f"{what}: state of sequence {i}: {float((es / E).max()):.2f} of the bound"
        worst = max(worst, float((err / bound).max()))
        rel = max(rel, float((es / S.flatten(1).norm(dim=1)).max()))
    return worst, rel
