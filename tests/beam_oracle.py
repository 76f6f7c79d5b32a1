"""Plain restatements, in float64 and Python integers on the CPU, of beam search and shared-prompt attention."""
from __future__ import annotations

import math

import numpy as np
import torch

from oracle import quant as oq


def rows(cache, table, n, block_size):
    """float64 k, v [n, KV, D], and the rulers [n, KV, 4], of the first n tokens of a row of block tables."""
    d = cache.shape[-1] - 8
    t = np.arange(n)
    x = cache[np.asarray(table)[t // block_size], t % block_size]                 # [n, KV, D + 8]
    ruler = np.ascontiguousarray(x[..., d:]).view(np.float16).astype(np.float64)
    code = np.stack([x[..., :d] & 15, x[..., :d] >> 4], -1).reshape(*x.shape[:-1], 2 * d).astype(np.float64)
    return (code[..., :d] * ruler[..., 1:2] + ruler[..., 0:1], code[..., d:] * ruler[..., 3:4] + ruler[..., 2:3], ruler)


def attend(q, cache, table, n, block_size):
    """float64 [H, D] of one sequence, and the bound of the fp32 kernel's error.

    A score (base 2) is c (kstep sum q (n - 8) + (kmin + 8 kstep) sum q), c = log2(e) / sqrt(D), |n - 8| <= 8: its fp32 terms
    are at most A = c sum |q| (8 kstep + |kmin + 8 kstep|), and D + 8 roundings of 2^-24 lie in it.  A weight is off by ln 2
    times that, by the exponential's and its own 2^-21; every weight counts above and below the line (the factor 2).  The sums
    of values grow to M = sum p (8 vstep + |vmin + 8 vstep|) / sum p in a rounding for each 16 keys and 64 of the joins."""
    H, D = q.shape
    if n <= 0:
        return np.zeros((H, D)), np.zeros((H, 1))
    k, v, ruler = rows(cache, table, n, block_size)
    out, bound = np.empty((H, D)), np.empty((H, 1))
    G = H // k.shape[1]
    c = math.log2(math.e) / math.sqrt(D)
    for h in range(H):
        j = h // G
        qq = q[h].astype(np.float64)
        z = k[:, j] @ qq / math.sqrt(D)
        p = np.exp(z - z.max())
        p /= p.sum()
        out[h] = p @ v[:, j]
        r = np.abs(ruler[:, j])
        span = c * np.abs(qq).sum() * (8 * r[:, 1] + np.abs(ruler[:, j, 0] + 8 * ruler[:, j, 1])).max()
        mean = p @ (8 * r[:, 3] + np.abs(ruler[:, j, 2] + 8 * ruler[:, j, 3]))
        bound[h] = mean * (2 * math.log(2) * (D + 8) * 2.0 ** -24 * span + 2.0 ** -20 + (n / 16 + 64) * 2.0 ** -24)
    return out, bound


def select(logits, scores, keep, finished=None, lengths=None, penalty=0.0, eos=-1, pad=0, keep_rows=False):
    """[(token, parent, score, finished, length)] * keep of every request; logits float64 [R * W, V] (lists of tensors)."""
    R, W = len(scores), len(scores[0])
    answers = []
    for r in range(R):
        found = []
        for w in range(W):
            score = scores[r][w]
            if not score > -math.inf:
                continue
            done = bool(finished is not None and finished[r][w])
            n = (lengths[r][w] if lengths is not None else 0) + (0 if done else 1)
            weigh = float(max(n, 1)) ** penalty if penalty else 1.0
            if done:
                found.append((score / weigh, w, pad, score))
                continue
            x = logits[r * W + w].double().clone()
            x[torch.isnan(x)] = -math.inf
            x = x.clamp(max=torch.finfo(torch.float32).max)
            top = x.max()
            if not float(top) > -math.inf:
                continue
            total = (x - top) + (score - math.log(float((x - top).exp().sum())))
            order = torch.sort(x, descending=True, stable=True).indices[:keep]     # (a beam's order is that of its logits)
            found += [(float(total[i]) / weigh, w, int(i), float(total[i])) for i in order if float(total[i]) > -math.inf]
        found = sorted(found, key=lambda c: (-c[0], c[1]))[:keep]                  # (stable)
        found = [(t, w, s) for _, w, t, s in found] + [(0, 0, -math.inf)] * (keep - len(found))
        if keep_rows:
            place, spare = [None] * W, []
            for c in found:
                if place[c[1]] is None:
                    place[c[1]] = c
                else:
                    spare.append(c)
            found = [c if c is not None else spare.pop(0) for c in place]
        answer = []
        for t, w, s in found:
            done = bool(finished is not None and finished[r][w])
            n = lengths[r][w] + (0 if done else 1) if lengths is not None else None
            answer.append((t, w, s, done or t == eos, n))
        answers.append(answer)
    return answers


def reorder(caches, tables, lens, parents, block_size):
    """The caches (numpy, one a layer) and tables after the move, from copies of both."""
    new_caches, new = [c.copy() for c in caches], [list(t) for t in tables]
    W, blocks = len(parents[0]), caches[0].shape[0] if caches else 0
    for r, row in enumerate(parents):
        n = max(lens[r], 0)
        full, rest = divmod(n, block_size)
        for j, p in enumerate(row):
            if not 0 <= p < W:
                continue
            a, b = tables[r * W + j], tables[r * W + p]
            new[r * W + j][:full] = list(b[:full])
            if full < len(a) and rest and 0 <= a[full] < blocks and 0 <= b[full] < blocks:
                for c, old in zip(new_caches, caches):
                    c[a[full], :rest] = old[b[full], :rest]
    return new_caches, new


def store(cache, k, v, slots, block_size):
    """Quantize fp16 k, v [N, KV, D] into the slots of a numpy cache."""
    oq.quantize_store(k, v, cache, slots, block_size)
