"""Plain restatements, in Python integers and float64 on the CPU, of the serving step's operators."""
from __future__ import annotations

import math

import numpy as np
import torch


def step_metadata(query_lens, context_lens, tables, free, block_size, num_tokens, free_start=0):
    """(tables, query_start_loc, seq_lens, positions, slots, free_end), one token after another."""
    tables = [list(r) for r in tables]
    columns = len(tables[0]) if tables else 0
    start, seq, pos, slots, taken = [0], [], [], [], free_start
    for r, (q, c) in enumerate(zip(query_lens, context_lens)):
        c = min(max(c, 0), columns * block_size)
        q = min(max(q, 0), num_tokens - start[-1])
        held, live, room = -(-c // block_size), 0, True
        for t in range(q):
            p = c + t
            col, inside = divmod(p, block_size)
            slot = -1
            if col < columns:
                if col >= held and inside == 0 or (t == 0 and col >= held):
                    room = room and taken < len(free)
                    if taken < len(free):
                        tables[r][col] = free[taken]
                    taken += 1
                if room:
                    slot = tables[r][col] * block_size + inside
                    live += 1
            pos.append(p)
            slots.append(slot)
        start.append(start[-1] + q)
        seq.append(c + live)
    pad = num_tokens - len(pos)
    return tables, start, seq, pos + [0] * pad, slots + [-1] * pad, taken


def rotate(x, positions, inv_freq, interleaved, scale):
    """float64 [N, H, D] and what bounds its fp32 rounding, |x1| + |x2| of each dim's pair."""
    f = x.double()
    half = inv_freq.numel()
    a = positions.double()[:, None, None] * inv_freq.double()
    c, s = a.cos() * scale, a.sin() * scale
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y, bound = f.clone(), torch.zeros_like(f)
    y[..., one] = f[..., one] * c - f[..., two] * s
    y[..., two] = f[..., two] * c + f[..., one] * s
    bound[..., one] = bound[..., two] = f[..., one].abs() + f[..., two].abs()
    return y, bound


def prompt_attention(q, k, v, q_start, k_start, causal, scale):
    """float64 [N, H, D] (NaN where no sequence has the row) and the bounds of its roundings: the mean of |v| under
    the weights, and the largest sum of |q||k| of a row's scores."""
    N, H, D = q.shape
    G = H // k.shape[1]
    out = torch.full((N, H, D), math.nan, dtype=torch.float64)
    mean, span = torch.zeros_like(out), torch.zeros((N, H, 1), dtype=torch.float64)
    for r in range(len(q_start) - 1):
        a, b, c, d = q_start[r], q_start[r + 1], k_start[r], k_start[r + 1]
        n, m = b - a, d - c
        if n <= 0:
            continue
        see = torch.arange(m)[None] <= torch.arange(n)[:, None] + (m - n) if causal else torch.ones((n, m), dtype=torch.bool)
        for h in range(H):
            qq, kk, vv = q[a:b, h].double(), k[c:d, h // G].double(), v[c:d, h // G].double()
            z = (qq @ kk.T * scale).masked_fill(~see, -math.inf)
            w = torch.softmax(z, -1)
            # what a row does not see is no part of its sum, whatever it holds
            rows = []
            for i in range(n) if not bool(torch.isfinite(vv).all()) else ():
                rows.append(w[i, see[i]] @ vv[see[i]])
            o = torch.stack(rows) if rows else torch.where(see, w, 0.0) @ vv
            none = ~see.any(-1)
            o[none] = 0.0
            out[a:b, h] = o
            mean[a:b, h] = torch.where(see, w, 0.0) @ vv.abs().nan_to_num(0.0, posinf=0.0)
            if m:
                span[a:b, h, 0] = (qq.abs() @ kk.abs().nan_to_num(0.0, posinf=0.0).T).amax(-1) * scale
    return out, mean, span


def sample(row, u, temperature, top_k, top_p, min_p):
    """(token, probability) of one row of logits (float64)."""
    l = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    top = l.max()
    if top == -np.inf:
        return 0, 0.0
    if not temperature > 0:
        return int(np.argmax(l)), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        d = np.where(l == top, 0.0, (top - l) / float(temperature))
    w = np.exp(-d)
    order = np.lexsort((np.arange(l.size), -l))
    if 0 < top_k < l.size:
        order = order[:top_k]
    s = w[order]
    n = order.size
    if top_p < 1.0:
        before = np.concatenate([[0.0], np.cumsum(s)[:-1]])
        n = max(1, int((before < top_p * s.sum()).sum()))
    keep = order[:n]
    keep = keep[(w[keep] >= min(min_p, 1.0)) | (keep == order[0])]
    keep.sort()
    c = np.cumsum(w[keep])
    at = min(int(np.searchsorted(c, max(float(u), 0.0) * c[-1], side="right")), keep.size - 1)
    while w[keep[at]] == 0.0:
        at -= 1
    return int(keep[at]), float(w[keep[at]] / c[-1])
