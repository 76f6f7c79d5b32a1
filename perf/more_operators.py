"""The operators of beam search and of shared prompts over the packed 4-bit cache, with their inputs, plain forms, exact
results and minimal work.

* ``shared``   decode attention of sequences that share a prompt, whose keys and values are read once for all of them;
* ``select``   the best continuations of every request, over its beams and the vocabulary, from logits and scores;
* ``reorder``  the beams' cache rows after the selection: block tables, and the tokens of the block that is still filling.

With ``own`` false ``run`` computes them from elementary torch operations, with ``own`` true by the framework's calls.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "slm-turbo_amd")


def _kernels():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from kernels import kv_dequant, serving

    return kv_dequant, serving


def listed():
    return [
        # The least: two beams behind one short prompt, 14 query / 2 KV heads of 64 dims.
        dict(name="shared-pair", kind="shared", heads=14, kv=2, dim=64, groups=1, fewest=2, most=2, prompt_lo=150, prompt_hi=150,
             own_lo=9, own_hi=9, block=16, bits=32, out="float16"),
        # Beam search in the 1.1B Llama-style model: 8 prompts of different lengths, 4 beams of 60 tokens each.
        dict(name="shared-beams", kind="shared", heads=32, kv=4, dim=64, groups=8, fewest=4, most=4, prompt_lo=1001, prompt_hi=4096,
             own_lo=60, own_hi=60, block=16, bits=32, out="float16"),
        # A long document and 8 answers to it, 32 query / 8 KV heads of 128 dims.
        dict(name="shared-document", kind="shared", heads=32, kv=8, dim=128, groups=1, fewest=8, most=8, prompt_lo=32768,
             prompt_hi=32768, own_lo=100, own_hi=700, block=16, bits=32, out="float16"),
        # A server's system prompt before 64 conversations.
        dict(name="shared-system", kind="shared", heads=32, kv=8, dim=128, groups=1, fewest=64, most=64, prompt_lo=8192, prompt_hi=8192,
             own_lo=200, own_hi=2000, block=16, bits=32, out="float16"),
        # Groups of one to nine sequences, 80 dims, larger pages, int64 tables, fp32 results.
        dict(name="shared-groups", kind="shared", heads=32, kv=8, dim=80, groups=9, fewest=1, most=9, prompt_lo=33, prompt_hi=3001,
             own_lo=1, own_hi=400, block=32, bits=64, out="float32"),
        # One user's request, 4 beams, a vocabulary of 32000.
        dict(name="select-single", kind="select", requests=1, beams=4, keep=4, vocab=32000, dtype="float16", first=False,
             ended=0.0, penalty=0.0, rows=True),
        # The first step of 8 requests, of which one beam each is alive, as many spare candidates as beams.
        dict(name="select-first", kind="select", requests=8, beams=5, keep=10, vocab=50001, dtype="float32", first=True,
             ended=0.0, penalty=0.0, rows=False),
        # A batch over a large vocabulary, some beams ended, scores weighed by length.
        dict(name="select-batch", kind="select", requests=16, beams=8, keep=8, vocab=151936, dtype="bfloat16", first=False,
             ended=0.2, penalty=0.8, rows=True),
        # One request's 4 beams in the 1.1B model's 22 layers.
        dict(name="reorder-single", kind="reorder", requests=1, beams=4, stay=2, layers=22, kv=4, dim=64, block=16, shortest=1033,
             longest=1033),
        # A batch of 16 requests with 8 beams, 32 layers of 8 KV heads of 128 dims.
        dict(name="reorder-batch", kind="reorder", requests=16, beams=8, stay=4, layers=32, kv=8, dim=128, block=16, shortest=700,
             longest=1300),
        # Few layers, large pages, five beams.
        dict(name="reorder-pages", kind="reorder", requests=6, beams=5, stay=2, layers=3, kv=2, dim=80, block=64, shortest=60,
             longest=3000),
    ]


# (query heads, KV heads, dims) of the tests' and the benchmark's layers
_LAYERS = [(14, 2, 64), (12, 2, 128), (32, 4, 64), (32, 8, 128), (64, 8, 128), (16, 2, 64), (4, 4, 64), (32, 8, 64),
           (24, 6, 128), (16, 8, 64), (32, 4, 128), (8, 8, 80), (12, 2, 80), (32, 8, 80)]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "shared", "select", "select", "reorder"])
    h, kv, d = rng.choice(_LAYERS)
    if kind == "shared":
        groups = _spread(rng, 1, 16)
        most = _spread(rng, 1, 64 if groups == 1 else 64 // groups + 1)
        room = 75_000 // (groups * (most + 1))        # tokens in all, as many as the system prompt's conversations
        long = _spread(rng, 20, max(20, min(32768 // max(1, h * most // 256), 4 * room)))
        mine = _spread(rng, 1, max(1, min(2000, room)))
        return dict(kind=kind, heads=h, kv=kv, dim=d, groups=groups, fewest=rng.randint(1, most), most=most,
                    prompt_lo=rng.randint(1, long), prompt_hi=long, own_lo=rng.randint(1, mine), own_hi=mine,
                    block=rng.choice([16, 16, 32, 64]), bits=rng.choice([32, 64]), out=rng.choice(["float16", "float32"]))
    if kind == "select":
        beams, dtype = _spread(rng, 1, 16), rng.choice(["float16", "bfloat16", "float32"])
        return dict(kind=kind, requests=_spread(rng, 1, (64 if dtype == "float32" else 128) // beams), beams=beams, keep=beams,
                    vocab=_spread(rng, 1000, 151936), dtype=dtype, first=rng.random() < 0.2, ended=rng.choice([0.0, 0.3]),
                    penalty=rng.choice([0.0, 0.0, 0.6, 1.0]), rows=rng.choice([False, True]))
    beams = _spread(rng, 2, 16)
    block = rng.choice([16, 16, 32])
    requests = _spread(rng, 1, 1024 // (beams * block))
    long = _spread(rng, 20, 2500)
    return dict(kind=kind, requests=requests, beams=beams, stay=rng.randint(1, beams - 1), layers=_spread(rng, 1, 32), kv=kv, dim=d,
                block=block, shortest=rng.randint(1, long), longest=long)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 29)


def _normal(g, shape):
    return torch.randn(shape, generator=g, device=DEV)


def _between(lo, hi, n):
    """n whole numbers spread evenly over [lo, hi]."""
    return [(lo + hi) // 2] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _shuffled(values, seed):
    order = torch.randperm(len(values), generator=torch.Generator().manual_seed(int(seed) * 31 + 7))
    return torch.tensor(values)[order]


def _pack(x):
    """fp32 [..., D] -> codes uint8 [..., D/2] and their ruler (min, step) fp16 [..., 2]."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = (hi - lo) / 15
    code = ((x - lo) / step + 0.5).floor_().clamp_(0, 15).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat([lo, step], -1).half()


def _pages(g, n, block, kv, d):
    """n pages of a packed cache, full of a model's keys and values: some channels of the keys are larger than the others,
    the values have a mean."""
    k, v = _normal(g, (n, block, kv, d)), _normal(g, (n, block, kv, d))
    k[..., ::9] *= 3.0
    v += 0.3 * _normal(g, (kv, d))
    (kc, kr), (vc, vr) = _pack(k), _pack(v)
    return torch.cat([kc, vc, torch.cat([kr, vr], -1).view(torch.uint8)], -1)


def _sizes(case):
    """Sequences of every group, prompts' lengths and the sequences' own tokens, in some order."""
    rows = _between(case["fewest"], case["most"], case["groups"])
    return rows, _between(case["prompt_lo"], case["prompt_hi"], case["groups"]), _between(case["own_lo"], case["own_hi"], sum(rows))


def _make_shared(case, seed):
    h, kv, d, bs = case["heads"], case["kv"], case["dim"], case["block"]
    g = _gen(seed)
    # (the groups' sizes in the order of the list, so that the work is the same for every seed)
    rows, prompt, mine = torch.tensor(_sizes(case)[0]), torch.tensor(_sizes(case)[1]), _shuffled(_sizes(case)[2], seed)
    of = torch.repeat_interleave(torch.arange(len(rows)), rows)          # a sequence's group
    lens = prompt[of] + mine
    whole, rest = prompt // bs, prompt % bs
    # pages: the prompts' whole ones, one with each prompt's last tokens, and every sequence's own
    mine_pages = (lens + bs - 1) // bs - whole[of]
    first_whole = whole.cumsum(0) - whole
    first_mine = int(whole.sum()) + len(rows) + mine_pages.cumsum(0) - mine_pages
    n = int(whole.sum()) + len(rows) + int(mine_pages.sum())
    cache = _pages(g, n, bs, kv, d)
    tails = (int(whole.sum()) + of).to(DEV)
    copied = (torch.arange(bs) < rest[of][:, None]).to(DEV)[..., None, None]
    at = first_mine.to(DEV)
    cache[at] = torch.where(copied, cache[tails], cache[at])             # every sequence has them in its first page
    col = torch.arange(int((lens + bs - 1).max()) // bs)
    table = torch.where(col < whole[of][:, None], first_whole[of][:, None] + col, first_mine[:, None] + col - whole[of][:, None])
    table = torch.where(col < ((lens + bs - 1) // bs)[:, None], table, 0)
    place = torch.randperm(n, generator=torch.Generator().manual_seed(int(seed) * 13 + 1))
    cache[place.to(DEV)] = cache.clone()
    start = torch.cat([torch.zeros(1, dtype=torch.int64), rows.cumsum(0)])
    q = _normal(g, (len(of), (h + 2 * kv) * d)).half()                   # as the fused projection hands them over
    return dict(q=q[:, :h * d].view(-1, h, d), cache=cache, tables=place[table].to(torch.int64 if case["bits"] == 64 else torch.int32).to(DEV),
                lens=lens.int().to(DEV), start=start.int().to(DEV), prompt=prompt.int().to(DEV), most=int(rows.max()),
                longest=int(prompt.max()), longest_own=int(mine.max()))


def _make_select(case, seed):
    r, w, v = case["requests"], case["beams"], case["vocab"]
    g = _gen(seed)
    # a request's beams see much the same continuations: a background and some tokens that a trained model favours
    x = 2.0 * _normal(g, (r, 1, v)) + 0.7 * _normal(g, (r, w, v))
    at = torch.randint(0, v, (r, 60), generator=g, device=DEV)[:, None].expand(r, w, 60)
    x.scatter_add_(2, at, 5.0 + 5.0 * torch.rand((r, w, 60), generator=g, device=DEV))
    scores = -20.0 * torch.rand((r, 1), generator=g, device=DEV) - 4.0 * torch.rand((r, w), generator=g, device=DEV)
    lengths = torch.randint(1, 40, (r, 1), generator=g, device=DEV, dtype=torch.int32).expand(r, w).contiguous()
    ended = torch.rand((r, w), generator=g, device=DEV) < case["ended"]
    if case["first"]:
        scores[:] = -math.inf
        scores[:, 0] = 0.0
        lengths.fill_(0)
        ended.fill_(False)
    lengths = torch.where(ended, torch.clamp(lengths - 1, min=1), lengths)
    return dict(logits=x.view(r * w, v).to(getattr(torch, case["dtype"])), scores=scores, lengths=lengths, ended=ended, eos=2, pad=0)


def _make_reorder(case, seed):
    r, w, bs = case["requests"], case["beams"], case["block"]
    g = _gen(seed)
    lens = torch.tensor(_between(case["shortest"], case["longest"], r))
    cols = int(lens.max()) // bs + 1
    # whole pages that any beams may share, and one to fill for each beam
    cache = torch.randint(0, 256, (case["layers"], 4 * cols + r * w, bs, case["kv"], case["dim"] + 8), dtype=torch.uint8, generator=g, device=DEV)
    place = torch.randperm(cache.shape[1], generator=g, device=DEV).int()
    table = place[torch.randint(0, 4 * cols, (r, w, cols), generator=g, device=DEV)]
    col = (lens // bs).to(DEV)[:, None, None].expand(r, w, 1)
    table.scatter_(2, col, place[4 * cols:].view(r, w, 1))
    # the best of each surviving beam's continuations stays in its row, the others take the rows of the beams that end
    order = torch.rand((r, w), generator=g, device=DEV).argsort(1)
    parent = torch.arange(w, device=DEV).expand(r, w).clone()
    pick = torch.randint(0, case["stay"], (r, w - case["stay"]), generator=g, device=DEV)
    parent.scatter_(1, order[:, case["stay"]:], order.gather(1, pick))
    return dict(cache=cache, tables=table.view(r * w, cols), lens=lens.int().to(DEV), parents=parent.int())


def prepare(case, seed):
    make = {"shared": _make_shared, "select": _make_select, "reorder": _make_reorder}[case["kind"]]
    return dict(make(case, seed), case=case)


# ------------------------------------------------------------------ plain forms
def _rows(cache, tables, at, d):
    """Keys and values, fp32 [N, T, KV, D], of the tokens at [N, T] of rows of block tables [N, columns]."""
    bs = cache.shape[1]
    block = tables.long().gather(1, torch.clamp(at // bs, max=tables.shape[1] - 1))
    x = cache[block, at % bs]
    ruler = x[..., d:].contiguous().view(torch.float16).float()
    code = torch.stack([x[..., :d] & 15, x[..., :d] >> 4], -1).flatten(-2).float()
    return code[..., :d] * ruler[..., 1:2] + ruler[..., 0:1], code[..., d:] * ruler[..., 3:4] + ruler[..., 2:3]


def _plain_shared(s):
    """The prompts' scores for all sequences of a group at once, padded to the largest; then each sequence's own."""
    case, d = s["case"], s["case"]["dim"]
    h, kv = case["heads"], case["kv"]
    g, n, r, b = h // kv, s["most"], s["start"].numel() - 1, s["lens"].numel()
    start, prompt, lens = s["start"].long(), s["prompt"].long(), s["lens"].long()
    q = s["q"].float() * d ** -0.5
    seq = torch.clamp(start[:-1, None] + torch.arange(n, device=DEV), max=b - 1)                 # [R, n]
    of = torch.searchsorted(start[1:].contiguous(), torch.arange(b, device=DEV), right=True)     # a sequence's group
    at = torch.arange(s["longest"], device=DEV)
    k, v = _rows(s["cache"], s["tables"][start[:-1]], torch.minimum(at, prompt[:, None] - 1), d)
    qg = q[seq].view(r, n, kv, g, d).permute(0, 2, 1, 3, 4).reshape(r * kv, n * g, d)
    w = torch.bmm(qg, k.permute(0, 2, 3, 1).reshape(r * kv, d, -1).contiguous()).view(r, kv, n, g, -1)
    w.masked_fill_(at >= prompt[:, None, None, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w.sub_(top).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.bmm(w.view(r * kv, n * g, -1), v.permute(0, 2, 1, 3).reshape(r * kv, -1, d).contiguous()).view(r, kv, n, g, d)
    place = (of, slice(None), torch.arange(b, device=DEV) - start[of])
    top, total, o = top[place], total[place], o[place]                                           # [B, KV, G, ...]
    at = prompt[of][:, None] + torch.arange(s["longest_own"], device=DEV)
    k, v = _rows(s["cache"], s["tables"], torch.minimum(at, lens[:, None] - 1), d)
    w = torch.bmm(q.reshape(b * kv, g, d), k.permute(0, 2, 3, 1).reshape(b * kv, d, -1).contiguous()).view(b, kv, g, -1)
    w.masked_fill_((at >= lens[:, None])[:, None, None], -math.inf)
    both = torch.maximum(top, w.amax(-1, keepdim=True))
    w.sub_(both).exp_()
    part = torch.exp(top - both)
    o = o * part + torch.bmm(w.view(b * kv, g, -1), v.permute(0, 2, 1, 3).reshape(b * kv, -1, d).contiguous()).view(b, kv, g, d)
    o = o / (total * part + w.sum(-1, keepdim=True))
    return {"out": o.reshape(b, h, d).to(getattr(torch, case["out"]))}


def _plain_select(s):
    case = s["case"]
    r, w, v, k = case["requests"], case["beams"], case["vocab"], case["keep"]
    x = s["logits"].double()
    x = x - x.amax(1, keepdim=True)
    x = x - x.exp().sum(1, keepdim=True).log()
    total = s["scores"].double()[..., None] + x.view(r, w, v)
    done = torch.full_like(total[:1, :1], -math.inf).expand(r, w, v).clone()
    done[..., s["pad"]] = s["scores"].double()
    total = torch.where(s["ended"][..., None], done, total)
    lengths = s["lengths"] + ~s["ended"]
    rank = total / lengths.double()[..., None] ** case["penalty"]
    at = torch.sort(rank.view(r, w * v), dim=1, descending=True, stable=True)[1][:, :k]
    parents, tokens, scores = at // v, at % v, total.view(r, w * v).gather(1, at)
    if case["rows"]:       # the best child of each beam takes its row, the others the rows that are left, in order
        again = (parents[:, :, None] == parents[:, None, :]).tril(-1).any(2)
        taken = torch.zeros((r, w), dtype=torch.int64, device=DEV).scatter_(1, parents, 1)
        left = torch.argsort(taken, dim=1, stable=True)
        row = torch.where(again, left.gather(1, torch.clamp(again.cumsum(1) - 1, min=0)), parents)
        order = torch.argsort(row, dim=1)
        parents, tokens, scores = parents.gather(1, order), tokens.gather(1, order), scores.gather(1, order)
    return {"tokens": tokens, "parents": parents.int(), "scores": scores.float(),
            "finished": s["ended"].gather(1, parents) | (tokens == s["eos"]), "lengths": lengths.gather(1, parents).int()}


def _plain_reorder(s):
    case, bs = s["case"], s["case"]["block"]
    r, w, tables = case["requests"], case["beams"], s["tables"]
    lens = s["lens"].long().repeat_interleave(w)
    src = (s["parents"].long() + torch.arange(r, device=DEV)[:, None] * w).view(-1)
    last = (lens // bs)[:, None]
    block = tables.gather(1, last).long()[:, 0]
    filled = (torch.arange(bs, device=DEV) < (lens % bs)[:, None])[None, ..., None, None]
    s["cache"][:, block] = torch.where(filled, s["cache"][:, block[src]], s["cache"][:, block])
    tables.copy_(torch.where(torch.arange(tables.shape[1], device=DEV) < last, tables[src], tables))
    return {"tables": tables, "cache": s["cache"]}


def run(state):
    s, case = state, state["case"]
    if own:
        kd, sv = _kernels()
        if case["kind"] == "shared":
            return {"out": kd.kv_dequant_decode_paged_shared(s["q"], s["cache"], s["tables"], s["lens"], s["start"], s["prompt"],
                                                             case["block"], case["kv"], out_dtype=getattr(torch, case["out"]))}
        if case["kind"] == "select":
            b = sv.beam_select(s["logits"], s["scores"], case["keep"], finished=s["ended"], lengths=s["lengths"],
                               length_penalty=case["penalty"], eos_token=s["eos"], pad_token=s["pad"], keep_rows=case["rows"])
            return {"tokens": b.tokens, "parents": b.parents, "scores": b.scores, "finished": b.finished, "lengths": b.lengths}
        sv.kv_reorder_beams(s["cache"], s["tables"], s["lens"], s["parents"], case["block"])
        return {"tables": s["tables"], "cache": s["cache"]}
    return {"shared": _plain_shared, "select": _plain_select, "reorder": _plain_reorder}[case["kind"]](s)


def work(case):
    """Every input read once, every output written once; two flops per multiply-add."""
    if case["kind"] == "shared":
        h, kv, d = case["heads"], case["kv"], case["dim"]
        rows, prompt, mine = _sizes(case)
        seen = sum(n * p for n, p in zip(rows, prompt)) + sum(mine)
        size = 4 if case["out"] == "float32" else 2
        return {"bytes": sum(rows) * h * d * (2 + size) + (sum(prompt) + sum(mine)) * (kv * (d + 8) + 4 / case["block"]),
                "flops": 4 * h * d * seen}
    if case["kind"] == "select":
        rows = case["requests"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * (4 if case["dtype"] == "float32" else 2) + 9) + case["requests"] * case["keep"] * 21,
                "flops": rows * case["vocab"] * 4}
    w, lens = case["beams"], _between(case["shortest"], case["longest"], case["requests"])
    moved = w - case["stay"]
    tokens = sum(n % case["block"] for n in lens) * case["layers"]
    return {"bytes": moved * (2 * tokens * case["kv"] * (case["dim"] + 8) + 8 * sum(n // case["block"] for n in lens)) + 4 * w * len(lens),
            "flops": 0}


# ------------------------------------------------------------------ exact results
def exact(case, seed):
    if case["kind"] == "reorder":        # (bytes and table entries)
        return None
    s = prepare(case, seed)
    if case["kind"] == "select":
        r, w = case["requests"], case["beams"]
        ends = s["ended"].tolist()
        scores = torch.empty((r, case["keep"]), dtype=torch.float64)
        for i in range(r):
            best = []
            for j in range(w):
                score, n = float(s["scores"][i, j]), int(s["lengths"][i, j])
                if ends[i][j]:
                    best.append((score / n ** case["penalty"], j, s["pad"], score))
                elif score > -math.inf:
                    p, token = torch.log_softmax(s["logits"][i * w + j].double(), 0).cpu().sort(descending=True, stable=True)
                    best += [(float(x + score) / (n + 1) ** case["penalty"], j, int(t), float(x + score))
                             for x, t in zip(p[:case["keep"]], token[:case["keep"]])]
            best = sorted(best, key=lambda c: (-c[0], c[1], c[2]))[:case["keep"]]
            if case["rows"]:
                row, spare = {}, []
                for c in best:
                    (spare if c[1] in row else row.setdefault(c[1], [])).append(c)
                for j in range(w):
                    row.setdefault(j, None)
                best = [row[j][0] if row[j] else spare.pop(0) for j in range(w)]
            scores[i] = torch.tensor([c[3] for c in best], dtype=torch.float64)
        return {"tokens": None, "parents": None, "scores": scores, "finished": None, "lengths": None}
    h, d, bs = case["heads"], case["dim"], case["block"]
    g, out = h // case["kv"], []
    for b, n in enumerate(s["lens"].tolist()):
        x = s["cache"][s["tables"][b, :-(-n // bs)].long()].flatten(0, 1)[:n]
        lo, step, vlo, vstep = x[..., d:].contiguous().view(torch.float16).double().unbind(-1)
        code = torch.empty((n, case["kv"], 2 * d), dtype=torch.float64, device=DEV)
        code[..., 0::2], code[..., 1::2] = x[..., :d].bitwise_and(15).double(), x[..., :d].div(16, rounding_mode="floor").double()
        k = (code[..., :d] * step[..., None] + lo[..., None]).transpose(0, 1).contiguous()      # [KV, n, D]
        v = (code[..., d:] * vstep[..., None] + vlo[..., None]).transpose(0, 1).contiguous()
        z = torch.matmul(k, s["q"][b].double().view(-1, g, d).transpose(1, 2).contiguous()) / math.sqrt(d)
        p = torch.softmax(z, 1).transpose(1, 2).contiguous()                                      # [KV, G, n]
        out.append(torch.matmul(p, v).reshape(h, d))
    return {"out": torch.stack(out)}
