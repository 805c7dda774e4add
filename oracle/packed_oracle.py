"""CPU restatement in float64 of the packed-sequence operators: attention over
sequences of different lengths, rotary positions, and the root-mean-square
norm with the residual's addition, forward and backward.

TEST INFRASTRUCTURE ONLY: the parity checker for the CUDA kernels in
``vision_rs_b200``; only ``tests/`` and ``__graft_entry__.smoke()`` may import
it.  The reference (spinorml/vision-rs) has none of these operators, so parity
is unpinned by the reference; the formulas are the definitions themselves.

Attention, for query i and key j of one sequence of lq queries and lk keys
(causal: i sees j ≤ i + lk − lq), query head h reading key head h // (H/Hkv):

    S = scale · q kᵀ,  lse_i = log Σ_j exp S_ij,  P = exp(S − lse),  O = P v

and a row that sees no key has O = 0, lse = −∞ and no gradient.
"""
from __future__ import annotations

import math

import torch


def _mask(lq, lk, causal):
    if not causal:
        return torch.zeros(lq, lk, dtype=torch.bool)
    return torch.arange(lk)[None, :] > torch.arange(lq)[:, None] + (lk - lq)


def attention_one(q, k, v, scale, causal):
    """One sequence and head: q [lq, D], k and v [lk, D] → (P, O, lse) in f64.
    A key that a row does not see never enters that row's sums, so NaN or
    infinity there stays out."""
    lq, lk = q.shape[0], k.shape[0]
    hide = _mask(lq, lk, causal)
    s = (scale * (q @ k.T)).masked_fill(hide, -math.inf)
    if lk == 0:
        return s, torch.zeros(lq, v.shape[1], dtype=torch.float64), torch.full((lq,), -math.inf, dtype=torch.float64)
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[:, None])
    o = p @ v if torch.isfinite(v).all() else \
        torch.where((p == 0)[:, :, None], 0.0, p[:, :, None] * v[None]).sum(1)
    return p, o, lse


def _sequences(lengths_q, lengths_k):
    q0 = k0 = 0
    for lq, lk in zip(lengths_q, lengths_k):
        yield slice(q0, q0 + lq), slice(k0, k0 + lk)
        q0, k0 = q0 + lq, k0 + lk


def attention_forward(q, k, v, lengths_q, lengths_k, scale, causal):
    """q [Tq, H, D], k and v [Tk, Hkv, D] (any float type) → O f64 [Tq, H, D], lse f64 [H, Tq]."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    group = q.shape[1] // k.shape[1]
    o, lse = torch.zeros_like(q), torch.full((q.shape[1], q.shape[0]), -math.inf, dtype=torch.float64)
    for sq, sk in _sequences(lengths_q, lengths_k):
        for h in range(q.shape[1]):
            _, o[sq, h], lse[h, sq] = attention_one(q[sq, h], k[sk, h // group], v[sk, h // group], scale, causal)
    return o, lse


def attention_backward(do, q, k, v, lengths_q, lengths_k, scale, causal):
    """Gradients (dq, dk, dv) in f64 by the formula: dV = Pᵀ dO,
    dS = P ⊙ (dO Vᵀ − rowsum(dO ⊙ O)), dQ = scale · dS K, dK = scale · dSᵀ Q."""
    do, q, k, v = (t.detach().cpu().double() for t in (do, q, k, v))
    group = q.shape[1] // k.shape[1]
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for sq, sk in _sequences(lengths_q, lengths_k):
        for h in range(q.shape[1]):
            g = h // group
            p, o, _ = attention_one(q[sq, h], k[sk, g], v[sk, g], scale, causal)
            d = do[sq, h]
            dv[sk, g] += p.T @ d
            ds = scale * p * (d @ v[sk, g].T - (d * o).sum(1, keepdim=True))
            dq[sq, h] = ds @ k[sk, g]
            dk[sk, g] += ds.T @ q[sq, h]
    return dq, dk, dv


def rotary(x, positions, inv_freq, interleaved, factor=1.0, backward=False):
    """x [tokens, heads, D] turned in f64; the first 2·len(inv_freq) dimensions."""
    x, inv = x.detach().cpu().double(), inv_freq.detach().cpu().double()
    th = positions.cpu().double()[:, None, None] * inv
    c, s = factor * torch.cos(th), factor * torch.sin(th) * (-1 if backward else 1)
    n, y = inv.shape[0], x.clone()
    ia, ib = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    return y


def rms_norm(x, w, residual, eps):
    """(h, y) in f64."""
    h = x.detach().cpu().double()
    if residual is not None:
        h = h + residual.detach().cpu().double()
    return h, h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * w.detach().cpu().double()


def rms_norm_backward(dy, h, w, eps, grad_h=None):
    """(dh, dw) in f64 by the formula."""
    dy, h, w = (t.detach().cpu().double() for t in (dy, h, w))
    r = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    g = dy * w
    dh = r * (g - h * r * r * (g * h).mean(-1, keepdim=True))
    if grad_h is not None:
        dh = dh + grad_h.detach().cpu().double()
    return dh, (dy * h * r).reshape(-1, h.shape[-1]).sum(0)
