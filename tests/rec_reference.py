"""64-bit definitions of the recurrent-layer operators for the tests, token by token."""
from __future__ import annotations

import math

import torch

HD = 128


def recurrence(S, q, k, v, g, beta, scale):
    """One sequence: S [H, value, key], q and k [n, Hk, 128], v [n, H, 128], g and beta [n, H] (beta None: no
    delta rule).  Returns out [n, H, 128], the states after 0 .. n tokens, and W and A: the same sums over absolute
    values per output and (after 0 .. n tokens) per state value, which bound what roundings of the terms can add."""
    S, q, k, v, g = (t.double() for t in (S, q, k, v, g))
    H, Hk = v.shape[1], q.shape[1]
    q, k = q.repeat_interleave(H // Hk, 1), k.repeat_interleave(H // Hk, 1)
    A = S.abs()
    out, absolute, states, sums = [], [], [S], [A]
    for t in range(v.shape[0]):
        e = torch.exp(g[t])[:, None, None]
        S, A = S * e, A * e
        u, a = v[t], v[t].abs()
        if beta is not None:
            b = beta[t].double()[:, None]
            u, a = b * (u - (S * k[t, :, None, :]).sum(-1)), b.abs() * (a + (A * k[t, :, None, :].abs()).sum(-1))
        S = S + u[:, :, None] * k[t, :, None, :]
        A = A + torch.maximum(a, u.abs())[:, :, None] * k[t, :, None, :].abs()
        out.append(scale * (S * q[t, :, None, :]).sum(-1))
        absolute.append(abs(scale) * (A * q[t, :, None, :].abs()).sum(-1))
        states.append(S)
        sums.append(A)
    empty = v.new_zeros((0, *v.shape[1:]))
    return (torch.stack(out) if out else empty), states, (torch.stack(absolute) if out else empty), sums


def convolution(hist, x, w, n_norm, eps):
    """One sequence: hist [C, 3], x [n, C], w [C, 4] -> y [n, C], the histories after 0 .. n rows."""
    x, w = x.double(), w.double()
    z = torch.cat([hist.double().T, x])
    n = x.shape[0]
    y = sum(z[j:j + n] * w[:, j] for j in range(4))
    y = y / (1 + torch.exp(-y))
    if n_norm:
        head = y[:, :n_norm].reshape(n, n_norm // HD, HD)
        y[:, :n_norm] = (head / torch.clamp(head.norm(dim=-1, keepdim=True), min=eps)).reshape(n, n_norm)
    return y, [z[t:t + 3].T for t in range(n + 1)]


def inputs(seed, rows, H, Hk, dtype, unit=True, decay=1.0, device="cuda"):
    """q and k (of length one when `unit`), v, g <= 0 of about -decay, beta in (0, 1), as slices of one fused row."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, (2 * Hk + H) * HD, generator=gen)
    if unit:
        qk = x[:, :2 * Hk * HD].view(rows, 2 * Hk, HD)
        qk /= qk.norm(dim=-1, keepdim=True)
    g = -decay * torch.exp(torch.randn(rows, H, generator=gen) * math.log(4.0))
    beta = torch.sigmoid(torch.randn(rows, H, generator=gen))
    x, g, beta = x.to(dtype).to(device), g.to(device), beta.to(device)
    return x[:, :Hk * HD], x[:, Hk * HD:2 * Hk * HD], x[:, 2 * Hk * HD:], g, beta
