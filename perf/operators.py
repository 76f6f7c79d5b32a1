"""The operators of a serving step around the packed 4-bit cache, with their inputs, plain forms, exact results
and minimal work.

* ``metadata``  positions, slots and block tables of a step, from the requests' lengths and a list of free blocks;
* ``store``     a step's queries and keys rotated, keys and values quantized into the packed paged cache;
* ``rotary``    queries and keys rotated, as a prompt's attention takes them;
* ``prompt``    causal attention of packed prompts of different lengths over their own K/V;
* ``sample``    the next token of every row of logits, from given uniforms.

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
    from kernels import serving

    return serving


def listed():
    return [
        # The host's work of every decode step: 32 requests behind 4096-token prompts, one token each.
        dict(name="metadata-decode", kind="metadata", requests=32, shortest=1, longest=1, cached=4224, idle=0, block=16),
        # A mixed step: 200 requests, some idle, some that decode, some that bring a chunk.
        dict(name="metadata-mixed", kind="metadata", requests=200, shortest=1, longest=300, cached=3000, idle=20, block=16),
        # A large batch of prompts at once.
        dict(name="metadata-prompts", kind="metadata", requests=96, shortest=200, longest=2500, cached=0, idle=0, block=32),
        # A decode step's store: 64 requests, 32 query / 8 KV heads of 128 dims, far positions.
        dict(name="store-step", kind="store", heads=32, kv=8, dim=128, rotary=128, tokens=64, interleaved=False,
             stretch=8.0, block=16),
        # A batch of prompts written into the cache.
        dict(name="store-prompts", kind="store", heads=32, kv=8, dim=128, rotary=128, tokens=7001, interleaved=False,
             stretch=1.0, block=16),
        # The other pair layout, on part of the head, in bfloat16: 12 query / 2 KV heads.
        dict(name="rotary-part", kind="rotary", heads=12, kv=2, dim=128, rotary=64, tokens=3001, interleaved=True,
             stretch=4.0, dtype="bfloat16"),
        # One short prompt: 14 query / 2 KV heads of 64 dims.
        dict(name="prompt-short", kind="prompt", heads=14, kv=2, dim=64, prompts=1, shortest=150, longest=150, dtype="float16"),
        # A batch of prompts of different lengths through one layer of the 1.1B Llama-style model.
        dict(name="prompt-batch", kind="prompt", heads=32, kv=4, dim=64, prompts=8, shortest=17, longest=2000, dtype="float16"),
        # A long prompt, 32 query / 8 KV heads of 128 dims.
        dict(name="prompt-long", kind="prompt", heads=32, kv=8, dim=128, prompts=1, shortest=8192, longest=8192, dtype="bfloat16"),
        # One user chatting, a vocabulary of 32000.
        dict(name="sample-single", kind="sample", rows=1, vocab=32000, temperature=0.7, top_k=50, top_p=0.9, min_p=0.0,
             dtype="float16"),
        # A batch with nucleus sampling over a large vocabulary.
        dict(name="sample-batch", kind="sample", rows=64, vocab=151936, temperature=1.0, top_k=0, top_p=0.95, min_p=0.0,
             dtype="float16"),
        # Rows of float32 logits, min-p, and no other cut.
        dict(name="sample-minp", kind="sample", rows=16, vocab=128001, temperature=1.5, top_k=0, top_p=1.0, min_p=0.02,
             dtype="float32"),
    ]


# (query heads, KV heads, dims) of the tests' and the benchmark's layers
_LAYERS = [(14, 2, 64), (12, 2, 128), (32, 4, 64), (32, 8, 128), (64, 8, 128), (16, 2, 64), (4, 4, 64), (32, 8, 64),
           (24, 6, 128), (16, 8, 64), (32, 4, 128), (8, 8, 80), (12, 2, 80), (32, 8, 80)]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["metadata", "store", "rotary", "prompt", "prompt", "prompt", "sample", "sample"])
    h, kv, d = rng.choice(_LAYERS)
    if kind == "metadata":
        n = _spread(rng, 1, 256)
        lo = _spread(rng, 1, 400)
        return dict(kind=kind, requests=n, shortest=lo, longest=_spread(rng, lo, max(lo, 200_000 // n)),
                    cached=rng.choice([0, _spread(rng, 1, 8000)]), idle=rng.choice([0, n // 10]),
                    block=rng.choice([16, 32, 64]))
    if kind in ("store", "rotary"):
        case = dict(kind=kind, heads=h, kv=kv, dim=d, rotary=rng.choice([d, d, d // 2]),
                    tokens=_spread(rng, 1, 7001 * 32 * 128 // (h * d) if h * d > 4096 else 7001),
                    interleaved=rng.choice([False, True]), stretch=rng.choice([1.0, 4.0, 8.0]))
        if kind == "store":
            case["block"] = rng.choice([16, 32])
        else:
            case["dtype"] = rng.choice(["float16", "bfloat16", "float32"])
        return case
    if kind == "prompt":
        prompts = rng.choice([1, 1, rng.randint(2, 24)])
        most = int(8192 * math.sqrt(32 * 128 / (h * d * prompts)))
        longest = _spread(rng, 20, min(8192, most))
        return dict(kind=kind, heads=h, kv=kv, dim=d, prompts=prompts, longest=longest,
                    shortest=longest if prompts == 1 else rng.randint(1, longest),
                    dtype=rng.choice(["float16", "bfloat16"]))
    rows = _spread(rng, 1, 64)
    return dict(kind=kind, rows=rows, vocab=_spread(rng, 1000, 151936), temperature=rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]),
                top_k=rng.choice([0, 0, 1, 40, 1000]), top_p=rng.choice([1.0, 0.5, 0.9, 0.99]),
                min_p=rng.choice([0.0, 0.0, 0.05]), dtype=rng.choice(["float16", "bfloat16", "float32"]))


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)


def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def _lengths(case, seed, n):
    """n lengths of the case's range with the same total for every seed."""
    g = torch.Generator().manual_seed(int(seed) * 31 + 3)
    lo, hi = case["shortest"], case["longest"]
    lens = torch.randint(lo, hi + 1, (n,), generator=g)
    more = n * (lo + hi) // 2 - int(lens.sum())
    room = hi - lens if more > 0 else lens - lo
    part = (abs(more) - (room.cumsum(0) - room)).clamp(min=0).minimum(room)
    return lens + (part if more > 0 else -part)


def _qkv(g, n, h, kv, d, dtype):
    """The projections of n tokens as a model hands them over: views of one fused buffer.  Some channels of the keys
    are larger than the others, as trained models have them, and the values have a mean."""
    x = _normal(g, (n, (h + 2 * kv) * d))
    k = x[:, h * d:(h + kv) * d].view(n, kv, d)
    k[:, :, ::9] *= 3.0
    x[:, (h + kv) * d:] += 0.3 * _normal(g, (kv * d,))
    x = x.to(dtype)
    return x[:, :h * d].view(n, h, d), x[:, h * d:(h + kv) * d].view(n, kv, d), x[:, (h + kv) * d:].view(n, kv, d)


def _make_metadata(case, seed):
    n, bs = case["requests"], case["block"]
    g = torch.Generator().manual_seed(int(seed) * 104729 + 5)
    q = torch.zeros(n, dtype=torch.int64)
    q[torch.randperm(n, generator=g)[case["idle"]:]] = _lengths(case, seed, n - case["idle"])
    ctx = torch.randint(0, case["cached"] + 1, (n,), generator=g)
    most = -(-(case["cached"] + case["longest"]) // bs)
    have, need = -(-ctx // bs), -(-(ctx + q) // bs)
    pool = torch.randperm(int(need.sum()) + 64, generator=g, dtype=torch.int32)
    used = int(have.sum())
    tables = torch.zeros((n, most), dtype=torch.int32)
    tables[torch.arange(most)[None] < have[:, None]] = pool[:used]
    return dict(query_lens=q.to(torch.int32).to(DEV), context_lens=ctx.to(torch.int32).to(DEV), tables=tables.to(DEV),
                free=pool[used:].clone().to(DEV), tokens=-(-int(q.sum()) // 8) * 8)     # (padded to a multiple of 8)


def _make_rotary(case, seed):
    n, r, d = case["tokens"], case["rotary"], case["dim"]
    g = _gen(seed + 1000)
    s = {}
    s["q"], s["k"], s["v"] = _qkv(g, n, case["heads"], case["kv"], d, getattr(torch, case.get("dtype", "float16")))
    far = int(16384 * case["stretch"])
    if n <= 256:        # a decode step: every token of a request of its own
        s["positions"] = torch.randint(0, far, (n,), generator=g, device=DEV)
    else:               # prompts behind one another
        first = torch.arange(n, device=DEV) % 2500
        s["positions"] = first + far // 2
    # an interpolated base with the attention factor that goes with it
    s["inv_freq"] = (10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r) / case["stretch"]).float().to(DEV)
    s["scale"] = 1.0 + 0.1 * math.log(case["stretch"])
    if case["kind"] == "store":
        bs = case["block"]
        s["cache"] = torch.zeros((-(-n // bs) + 3, bs, case["kv"], d + 8), dtype=torch.uint8, device=DEV)
        slots = torch.randperm(s["cache"].shape[0], generator=g, device=DEV)[:, None] * bs + torch.arange(bs, device=DEV)
        s["slots"] = slots.reshape(-1)[:n].clone()
        s["slots"][n - n // 20:] = -1     # padding tokens
    return s


def _make_prompt(case, seed):
    lens = _lengths(case, seed, case["prompts"])
    q, k, v = _qkv(_gen(seed + 1000), int(lens.sum()), case["heads"], case["kv"], case["dim"], getattr(torch, case["dtype"]))
    start = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    return dict(q=q, k=k, v=v, lens=lens.tolist(), start=start.to(torch.int32).to(DEV), longest=int(lens.max()))


def _make_sample(case, seed):
    b, v = case["rows"], case["vocab"]
    g = _gen(seed + 1000)
    # a broad background and some tokens that a trained model favours
    x = _normal(g, (b, v)) * 2.0
    at = torch.randint(0, v, (b, 60), generator=g, device=DEV)
    x.scatter_add_(1, at, 5.0 + 5.0 * torch.rand((b, 60), generator=g, device=DEV))
    return dict(logits=x.to(getattr(torch, case["dtype"])), uniforms=torch.rand(b, generator=g, device=DEV))


def prepare(case, seed):
    make = {"metadata": _make_metadata, "store": _make_rotary, "rotary": _make_rotary, "prompt": _make_prompt,
            "sample": _make_sample}[case["kind"]]
    return dict(make(case, seed), case=case)


# ------------------------------------------------------------------ plain forms
def _plain_metadata(s):
    bs, n = s["case"]["block"], s["tokens"]
    q, ctx = s["query_lens"].long(), s["context_lens"].long()
    ends = q.cumsum(0)
    t = torch.arange(n, device=DEV)
    live = t < ends[-1]
    t = torch.minimum(t, ends[-1] - 1)       # (padding repeats the last token)
    r = torch.searchsorted(ends, t, right=True)
    pos = ctx[r] + t - (ends - q)[r]
    held = (ctx + bs - 1) // bs
    need = (ctx + q + bs - 1) // bs - held
    col = pos // bs
    new = col >= held[r]
    nth = (need.cumsum(0) - need)[r] + col - held[r]
    block = torch.where(new, s["free"][torch.where(new, nth, 0)], s["tables"][r, col])
    s["tables"].index_put_((r, col), block)      # (tokens that bring no block write the entry that they read)
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    return {"tables": s["tables"], "start": torch.cat([zero, ends]).int(), "lens": (ctx + q).int(),
            "positions": torch.where(live, pos, 0), "slots": torch.where(live, block.long() * bs + pos % bs, -1),
            "free": need.sum().int().view(1)}


def _plain_rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    f = x.float()
    a, b = (f[..., 0:2 * half:2], f[..., 1:2 * half:2]) if interleaved else (f[..., :half], f[..., half:2 * half])
    c, s = cos[:, None], sin[:, None]
    y1, y2 = a * c - b * s, b * c + a * s
    y = torch.stack([y1, y2], -1).flatten(-2) if interleaved else torch.cat([y1, y2], -1)
    return torch.cat([y, f[..., 2 * half:]], -1).to(x.dtype)


def _angles(s):
    a = s["positions"].double()[:, None] * s["inv_freq"].double()
    return (a.cos() * s["scale"]).float(), (a.sin() * s["scale"]).float()


def _plain_quantize(x):
    """fp16 [..., D] -> packed uint8 [..., D/2], fp16 min and step [...]."""
    f = x.float()
    mn, mx = f.amin(-1), f.amax(-1)
    step = (mx - mn) / torch.full_like(mn, 15.0)     # a tensor: torch multiplies by 1/15 for a number
    step = torch.where(step > 0, step, torch.ones_like(step))
    codes = ((f - mn[..., None]) / step[..., None] + 0.5).to(torch.int32).clamp_(0, 15).to(torch.uint8)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), mn.half(), step.half()


def _plain_store(s):
    cos, sin = _angles(s)
    q = _plain_rotate(s["q"], cos, sin, s["case"]["interleaved"])
    kp, kmin, kstep = _plain_quantize(_plain_rotate(s["k"], cos, sin, s["case"]["interleaved"]))
    vp, vmin, vstep = _plain_quantize(s["v"])
    rulers = torch.stack([kmin, kstep, vmin, vstep], -1).contiguous().view(torch.uint8)
    rows = torch.cat([kp, vp, rulers], -1)
    cache, slots = s["cache"].flatten(0, 1), s["slots"]
    live = slots >= 0
    cache[slots[live]] = rows[live]
    return {"q": q, "cache": s["cache"]}


def _plain_rotary(s):
    cos, sin = _angles(s)
    return {"q": _plain_rotate(s["q"], cos, sin, s["case"]["interleaved"]),
            "k": _plain_rotate(s["k"], cos, sin, s["case"]["interleaved"])}


def _plain_prompt(s):
    """All prompts at once, each padded to the longest."""
    q, k, v, start = s["q"], s["k"], s["v"], s["start"].long()
    h, kv, d, n = q.shape[1], k.shape[1], q.shape[2], s["longest"]
    at = torch.arange(n, device=DEV)
    live = at[None] < (start[1:] - start[:-1])[:, None]                          # [R, n]
    rows = torch.where(live, start[:-1, None] + at, 0)
    qp = q[rows].float().permute(0, 2, 1, 3).reshape(-1, h // kv * n, d)         # (query heads are grouped by KV head)
    kt = k[rows].float().permute(0, 2, 3, 1).reshape(-1, d, n).contiguous()
    vp = v[rows].float().permute(0, 2, 1, 3).reshape(-1, n, d).contiguous()
    w = torch.bmm(qp, kt).mul_(d ** -0.5).view(-1, n, n)
    w.masked_fill_(at[None] > at[:, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.bmm(w.view(qp.shape[0], -1, n), vp).view(-1, n, d).div_(total)
    o = o.view(-1, h, n, d).transpose(1, 2)                                      # [R, n, H, D]
    return {"out": o[live].to(q.dtype)}


def _plain_sample(s):
    case, v = s["case"], s["logits"].shape[1]
    x, order = torch.sort(s["logits"].double(), dim=1, descending=True, stable=True)
    if case["temperature"] == 0.0:
        return {"tokens": order[:, 0], "probs": torch.ones_like(x[:, 0]).float()}
    w = ((x - x[:, :1]) / case["temperature"]).exp()
    w[:, case["top_k"] or v:] = 0.0
    before = w.cumsum(1) - w
    top_p, min_p = (torch.tensor(case[key], dtype=torch.float32).item() for key in ("top_p", "min_p"))
    keep = w >= min_p
    if top_p < 1.0:
        keep &= before < top_p * w.sum(1, keepdim=True)
    keep[:, 0] = True
    w = torch.where(keep, w, 0.0)
    c = torch.zeros_like(w).scatter_(1, order, w).cumsum(1)
    u = s["uniforms"].double()[:, None] * c[:, -1:]
    token = torch.searchsorted(c, u, right=True)
    return {"tokens": token[:, 0], "probs": ((c.gather(1, token) - (c - torch.zeros_like(w).scatter_(1, order, w))
            .gather(1, token)) / c[:, -1:])[:, 0].float()}


def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if own:
        kd = _kernels()
        if kind == "metadata":
            m = kd.kv_step_metadata(s["query_lens"], s["context_lens"], s["tables"], s["free"], case["block"], s["tokens"])
            return {"tables": s["tables"], "start": m.query_start_loc, "lens": m.seq_lens, "positions": m.positions,
                    "slots": m.slot_mapping, "free": m.free_end}
        if kind == "store":
            q = kd.kv_rotary_quantize_store(s["q"], s["k"], s["v"], s["cache"], s["slots"], case["block"], s["positions"],
                                            s["inv_freq"], interleaved=case["interleaved"], scale=s["scale"])
            return {"q": q, "cache": s["cache"]}
        if kind == "rotary":
            q, k = kd.kv_rotary(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=case["interleaved"],
                                scale=s["scale"])
            return {"q": q, "k": k}
        if kind == "prompt":
            return {"out": kd.kv_prompt_attention(s["q"], s["k"], s["v"], s["start"])}
        tokens, probs = kd.sample_tokens(s["logits"], s["uniforms"], temperature=case["temperature"], top_k=case["top_k"],
                                         top_p=case["top_p"], min_p=case["min_p"], return_probs=True)
        return {"tokens": tokens, "probs": probs}
    return {"metadata": _plain_metadata, "store": _plain_store, "rotary": _plain_rotary, "prompt": _plain_prompt,
            "sample": _plain_sample}[kind](s)


def work(case):
    """Every input read once, every output written once; two flops per multiply-add."""
    kind = case["kind"]
    if kind == "metadata":
        n, each = case["requests"], (case["shortest"] + case["longest"]) / 2
        tokens = (n - case["idle"]) * each
        return {"bytes": n * 20 + tokens * (16 + 8 / case["block"]), "flops": tokens * 8}
    if kind in ("store", "rotary"):
        n, h, kv, d = case["tokens"], case["heads"], case["kv"], case["dim"]
        size = 4 if case.get("dtype") == "float32" else 2
        rows = 2 * (h + kv) if kind == "rotary" else 2 * h + 2 * kv
        packed = kv * (d + 8) + 8 if kind == "store" else 0
        return {"bytes": n * (rows * d * size + packed + 8), "flops": n * ((h + kv) * case["rotary"] * 3 + kv * d * 8)}
    if kind == "prompt":
        lo, hi, n = case["shortest"], case["longest"], case["prompts"]
        mean = (lo + hi) / 2
        square = mean ** 2 + ((hi - lo + 1) ** 2 - 1) / 12
        h, kv, d = case["heads"], case["kv"], case["dim"]
        return {"bytes": n * mean * (2 * h + 2 * kv) * d * 2, "flops": 4 * h * d * n * (square + mean) / 2}
    size = 4 if case["dtype"] == "float32" else 2
    return {"bytes": case["rows"] * (case["vocab"] * size + 16), "flops": case["rows"] * case["vocab"] * 8}


# ------------------------------------------------------------------ exact results
def _exact_rotate(x, s, interleaved):
    a = s["positions"].double()[:, None, None] * s["inv_freq"].double()
    pairs = torch.polar(torch.full_like(a, s["scale"]), a)
    f, r = x.double(), 2 * a.shape[-1]
    turned = f[..., :r].reshape(*f.shape[:-1], -1, 2) if interleaved else f[..., :r].reshape(*f.shape[:-1], 2, -1).mT
    y = torch.view_as_real(torch.view_as_complex(turned.contiguous()) * pairs)
    return torch.cat([(y if interleaved else y.mT).flatten(-2), f[..., r:]], -1)


def exact(case, seed):
    kind = case["kind"]
    if kind == "metadata":
        return None
    s = prepare(case, seed)
    if kind == "store":     # (the packed bytes are whole numbers)
        return {"q": _exact_rotate(s["q"], s, case["interleaved"]), "cache": None}
    if kind == "rotary":
        return {"q": _exact_rotate(s["q"], s, case["interleaved"]), "k": _exact_rotate(s["k"], s, case["interleaved"])}
    if kind == "prompt":
        h, g, at, rows = case["heads"], case["heads"] // case["kv"], 0, []
        for n in s["lens"]:
            q, k, v = (s[x][at:at + n].double() for x in "qkv")
            see = torch.ones((n, n), dtype=torch.bool, device=DEV).tril()
            o = torch.empty_like(q)
            for i in range(h):
                z = torch.matmul(q[:, i].contiguous(), k[:, i // g].t().contiguous()) / math.sqrt(case["dim"])
                o[:, i] = torch.matmul(torch.softmax(z.masked_fill_(~see, -math.inf), -1), v[:, i // g].contiguous())
            rows.append(o)
            at += n
        return {"out": torch.cat(rows)}
    tokens, probs = [], []
    top_p, min_p = (torch.tensor(case[key], dtype=torch.float32).item() for key in ("top_p", "min_p"))
    for x, u in zip(s["logits"].double().cpu(), s["uniforms"].double().cpu().tolist()):
        if case["temperature"] == 0.0:
            tokens.append(int(x.argmax()))
            probs.append(1.0)
            continue
        p = torch.softmax(x / case["temperature"], 0)
        order = torch.argsort(x, descending=True, stable=True)[:case["top_k"] or None]
        ps = p[order] / p[order].sum()
        n = 1 + int((ps.cumsum(0)[:-1] < top_p).sum()) if top_p < 1.0 else ps.numel()
        n = max(1, min(n, int((ps >= min_p * ps[0] * (1 - 1e-15)).sum())))
        kept = order[:n].sort().values
        c = (p[kept] / p[kept].sum()).cumsum(0)
        at = min(int((c <= u).sum()), n - 1)
        tokens.append(int(kept[at]))
        probs.append(float(p[kept[at]] / p[kept].sum()))
    return {"tokens": torch.tensor(tokens), "probs": torch.tensor(probs, dtype=torch.float64)}
