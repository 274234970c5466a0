"""The serving operators around the paged cache from their definitions, in 64
bits on the CPU: per-head norm and rotation, attention with a sliding window
and visible first tokens, eviction by attention weight.

These have no counterpart in the reference. Each function also returns what a
test's error bound is made of (the magnitudes that an error is relative to).
"""
from __future__ import annotations

import math

import torch


def norm_rotate(x, weight, positions, inv_freq, eps=1e-6, norm=True, interleaved=False):
    """x [B, H, T, D], positions [B, T] -> (y, magnitude of each element's pair)."""
    y = x.detach().cpu().double()
    if norm:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.cpu().double()
    f = inv_freq.cpu().double()
    half = f.numel()
    t = positions.cpu().double()[:, None, :, None] * f
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out, mag = y.clone(), y.abs()
    out[..., a] = y[..., a] * t.cos() - y[..., b] * t.sin()
    out[..., b] = y[..., b] * t.cos() + y[..., a] * t.sin()
    mag[..., a] = mag[..., b] = y[..., a].abs() + y[..., b].abs()
    return out, mag


def visible(first, rows, T, L, window, sinks):
    """[B, T, L] of which key each query sees; first[b] is the position of
    query 0 and rows[b] the queries that are no padding."""
    j = torch.arange(L)[None, None]
    t = torch.arange(T)[None, :, None]
    pos = torch.as_tensor(first)[:, None, None] + t
    ok = (j <= pos) & (t < torch.as_tensor(rows)[:, None, None])
    if window is not None:
        ok = ok & ((j > pos - window) | (j < sinks))
    return ok


def attention(q, k, v, see, scale=None):
    """q [B, H, T, D], k / v [B, Hk, L, D], see [B, T, L] ->
    out            sum_j p_j v_j, zero for a row that sees no key
    spread         sum_j p_j |v_j|
    weights        [B, Hk, L]: p summed over the rows of a key head
    score          [B, H, T]: the largest sum_d |q_d k_jd| * scale of a visible key
    A hidden key contributes nothing, whatever its row holds."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    B, H, T, D = q.shape
    Hk, L = k.shape[1:3]
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    out = torch.zeros(B, H, T, D, dtype=torch.float64)
    spread, score = torch.zeros_like(out), torch.zeros(B, H, T, dtype=torch.float64)
    weights = torch.zeros(B, Hk, L, dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            g = h // (H // Hk)
            some = see[b].any(0)  # keys that a row sees at all
            kk, vv, ok = k[b, g, some], v[b, g, some], see[b][:, some]
            if not bool(some.any()):
                continue
            s = (q[b, h] @ kk.t() * scale).masked_fill(~ok, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(neginf=0.0))
            p = p / p.sum(-1, keepdim=True).masked_fill(~ok.any(-1, keepdim=True), 1.0)
            p = p.masked_fill(~ok, 0.0)
            if bool(torch.isfinite(vv).all()):
                out[b, h], spread[b, h] = p @ vv, p @ vv.abs()
            else:  # 0 * inf of a hidden key must not count
                for t in range(T):
                    out[b, h, t] = p[t, ok[t]] @ vv[ok[t]]
                    spread[b, h, t] = p[t, ok[t]] @ vv[ok[t]].abs()
            weights[b, g, some] += p.sum(0)
            score[b, h] = (q[b, h].abs() @ kk.abs().t() * scale).masked_fill(~ok, 0.0).amax(-1)
    return out, spread, weights, score


def rows_of(pages, table, page_size):
    """[B, H, L, D] rows that a table names (page 0 where it names none) and
    [B, L] of whether it names one."""
    pages, table = pages.cpu(), table.cpu().long()
    ok = (table >= 0) & (table < pages.shape[0])
    b = torch.arange(table.shape[0])[:, None]
    slot = torch.arange(table.shape[1]) % page_size
    return pages[table.masked_fill(~ok, 0), b, :, slot[None]].transpose(1, 2), ok


def evict(weights, lengths, k_pages, v_pages, page_table, out_table, sinks, recent):
    """(kept, weights, lengths, k_pages, v_pages) by sorting each head's entries."""
    w, table, out_table = weights.cpu(), page_table.cpu(), out_table.cpu()
    kp, vp = k_pages.cpu().clone(), v_pages.cpu().clone()
    P, ps = kp.shape[0], kp.shape[3]
    B, Hk, L = w.shape
    keep = out_table.shape[1]
    kept = torch.full((B, Hk, keep), -1, dtype=torch.int32)
    ow = torch.zeros(B, Hk, keep)
    n_out = torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), L)
        live = [j for j in range(n) if 0 <= int(table[b, j]) < P]
        for h in range(Hk):
            def rank(j):
                if j < sinks or j >= n - recent:
                    return (0, 0.0, j)
                x = float(w[b, h, j])
                return (1, 0.0, j) if x != x else (2, -x, j)
            idx = sorted(sorted(live, key=rank)[:keep])
            n_out[b] = len(idx)
            for i, j in enumerate(idx):
                kept[b, h, i], ow[b, h, i] = j, w[b, h, j]
                to = int(out_table[b, i])
                if 0 <= to < P:
                    src = (int(table[b, j]), b, h, j % ps)
                    kp[to, b, h, i % ps], vp[to, b, h, i % ps] = k_pages[src], v_pages[src]
    return kept, ow, n_out, kp, vp
