"""Plain 64-bit forms of the speculative-decoding operators (test infrastructure, CPU, one row at a time)."""

from __future__ import annotations

import math

import numpy as np
import torch


def norm_rope(x, positions, inv_freq, weight=None, eps=1e-6, interleaved=False):
    """x [B, H, T, D] -> fp64, from the definition."""
    y = x.double()
    if eps is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt()
        if weight is not None:
            y = y * weight.double()
    half = inv_freq.numel()
    pos = positions.double()
    pos = pos.expand(x.shape[0], x.shape[2]) if pos.dim() == 1 else pos
    angle = pos[:, None, :, None] * inv_freq.double()
    out = y.clone()
    for j in range(half):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        c, s = angle[..., j].cos(), angle[..., j].sin()
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
    return out


def entmax_weights(z: np.ndarray, alpha: float):
    """(weights, tau) of one row of fp64 scores z (already times alpha - 1), by bisection."""
    if z.size == 0 or np.all(np.isneginf(z)):
        return np.zeros_like(z), math.inf
    beta = 1.0 / (alpha - 1.0)
    hi = z.max()
    lo = hi - 1.0
    for _ in range(200):
        mid = 0.5 * (lo + hi)
        if (np.clip(z - mid, 0, None) ** beta).sum() > 1:
            lo = mid
        else:
            hi = mid
    tau = 0.5 * (lo + hi)
    d = np.clip(z - tau, 0, None)
    return np.where(d > 0, d, 0.0) ** beta * (d > 0), tau


def tree_attention(q, k, v, lens, k_draft, v_draft, mask, draft_lens, alpha, out0, tau0):
    """k, v [B, Hkv, S, D] dense; out0, tau0: what rows behind a short tree keep.

    Returns fp64 (out, tau, out_tol, tau_tol); the tolerances bound what fp32 scores, sums and thresholds may change
    (the rounding of the output to its type is not in them):
      a score is a sum of D products in any order with each addition off by at most 2^-23 of the partial sum (tensor
      cores truncate): delta = D 2^-23 Z, Z = largest zscale sum |q_d k_d|;
      tau moves by at most the largest score error, plus the solver's last step, 2^-23 (|top| + 1) with the scores' own
      rounding;
      with e = their sum, a weight d^beta moves by at most beta (d + e)^(beta-1) e (beta >= 1), or e^beta (beta < 1), and
      keys up to e under the threshold may enter; the output moves by that times the values, plus the fp32 sum
      itself and the power function: (n + 64) 2^-23 of sum w |v|.
    """
    B, Hq, T, D = q.shape
    G, beta = Hq // k.shape[1], 1.0 / (alpha - 1.0)
    out, tau = out0.double().numpy().copy(), tau0.double().numpy().copy()
    out_tol, tau_tol = np.zeros_like(out), np.zeros_like(tau)
    zs = (alpha - 1) / math.sqrt(D)
    for b in range(B):
        m = T if draft_lens is None else int(draft_lens[b])
        seen = (mask if mask.dim() == 2 else mask[b]).numpy()
        for h in range(Hq):
            kk = k[b, h // G, :lens[b]].double().numpy()
            vv = v[b, h // G, :lens[b]].double().numpy()
            kd, vd = k_draft[b, h // G].double().numpy(), v_draft[b, h // G].double().numpy()
            for t in range(m):
                qv = q[b, h, t].double().numpy() * zs
                js = [j for j in range(m) if seen[t, j]]
                keys, values = np.concatenate([kk, kd[js]]), np.concatenate([vv, vd[js]])
                z = keys @ qv
                w, tau[b, h, t] = entmax_weights(z, alpha)
                out[b, h, t] = w @ values
                if z.size == 0:
                    continue
                delta = D * 2.0 ** -23 * (np.abs(keys) @ np.abs(qv)).max()
                e = 2 * delta + 2.0 ** -22 * (abs(z.max()) + 1)
                near = z > tau[b, h, t] - e
                d = np.clip(z[near] - tau[b, h, t], 0, None) + e
                dw = beta * d ** (beta - 1) * e if beta >= 1 else np.full(d.shape, e ** beta)
                av = np.abs(values[near])
                out_tol[b, h, t] = dw @ av + (near.sum() + 64) * 2.0 ** -23 * (w[near] @ av)
                tau_tol[b, h, t] = e
    return tuple(torch.from_numpy(x) for x in (out, tau, out_tol, tau_tol))


def plan(seq, new, table, free, page, n_slots):
    """Python loops over sequences, pages and tokens.  Returns (table, slots, positions, row_starts)."""
    B = len(seq)
    new = [new] * B if isinstance(new, int) else new
    held = [-(-max(s, 0) // page) for s in seq]
    head = sum(held)
    table = [list(r) for r in table]
    slots, positions, starts = [], [], [0]
    for b in range(B):
        for p in range(held[b], -(-(max(seq[b], 0) + max(new[b], 0)) // page)):
            if p < len(table[b]):
                table[b][p] = free[head] if head < len(free) else -1
            head += 1
        for i in range(max(new[b], 0)):
            pos = max(seq[b], 0) + i
            block = table[b][pos // page] if pos // page < len(table[b]) else -1
            slots.append(block * page + pos % page if block >= 0 else -1)
            positions.append(pos)
        starts.append(len(positions))
    pad = max(n_slots - len(slots), 0)
    return table, (slots + [-1] * pad)[:n_slots], (positions + [-1] * pad)[:n_slots], starts


def release(seq, keep, table, free, page):
    table, free = [list(r) for r in table], list(free)
    keep = [keep] * len(seq) if isinstance(keep, int) else keep
    kept = [min(max(k, 0), s) for k, s in zip(keep, seq)]
    at = sum(-(-k // page) for k in kept)
    for b, (s, k) in enumerate(zip(seq, kept)):
        for p in range(-(-k // page), -(-s // page)):
            free[at] = table[b][p]
            table[b][p] = -1
            at += 1
    return table, free, kept
