"""GPU: beam search and shared-prompt attention (kernels.kv_dequant, kernels.serving) against plain restatements in
64 bits, at the sizes, lengths, strides and masks where they can go wrong, alone and together."""
import math

import numpy as np
import pytest
import torch

import beam_oracle as bo

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _kd():
    from kernels import kv_dequant

    return kv_dequant


def _sv():
    from kernels import serving

    return serving


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


# =============================================================================
#  attention over a shared prompt
# =============================================================================
def _shared_case(seed, H, KV, D, groups, block=16, loose=(), spare=2):
    """groups: [(shared tokens, [tokens in all of each sequence])]; loose: lengths of sequences of no group (behind them).
    Whole shared blocks are one, the block in which the prompt ends is every sequence's own."""
    g = _gen(seed)
    lens = [n for _, own in groups for n in own] + list(loose)
    cols = max([-(-max(n, p, 1) // block) for p, own in groups for n in own + [p]] + [-(-max(n, 1) // block) for n in loose] + [1]) + spare
    pool = torch.randperm(len(lens) * cols + 1, generator=g).tolist()
    cache = torch.randint(0, 256, (len(pool), block, KV, D + 8), dtype=torch.uint8, generator=g).numpy()
    ruler = torch.stack([-1.5 + 0.3 * torch.randn(cache.shape[:3], generator=g), 0.2 + 0.05 * torch.rand(cache.shape[:3], generator=g)], -1)
    cache[..., D:] = torch.cat([ruler, ruler + 0.05], -1).half().contiguous().view(torch.uint8).numpy()
    tables, starts, at = [], [0], 0
    for p, own in groups:
        first = None
        for n in own:
            row = [pool[at + i] for i in range(cols)]
            at += cols
            if first is None:
                first = row
            else:
                row[:p // block] = first[:p // block]
                if p % block:
                    cache[row[p // block], :p % block] = cache[first[p // block], :p % block]
            tables.append(row)
        starts.append(len(tables))
    for _ in loose:
        tables.append([pool[at + i] for i in range(cols)])
        at += cols
    q = torch.randn((len(lens), H, D), generator=g).half()
    return dict(q=q, cache=cache, tables=tables, lens=lens, starts=starts, prefix=[p for p, _ in groups], block=block, KV=KV)


def _run_shared(c, dtype=torch.float32, bits=32, q=None, out=None, cache=None):
    return _kd().kv_dequant_decode_paged_shared(
        c["q"].to(DEV) if q is None else q, torch.from_numpy(c["cache"]).to(DEV) if cache is None else cache,
        _int(c["tables"], torch.int64 if bits == 64 else torch.int32).view(len(c["lens"]), len(c["tables"][0]) if c["tables"] else 0), _int(c["lens"]), _int(c["starts"]),
        _int(c["prefix"]), c["block"], c["KV"], out=out, out_dtype=dtype)


def _check_shared(c, got, seqs=None):
    got = got.double().cpu().numpy()
    half = 2.0 ** -11 if c.get("dtype") is torch.float16 else 2.0 ** -24
    cols = len(c["tables"][0]) * c["block"] if c["tables"] else 0
    for b in range(len(c["lens"])) if seqs is None else seqs:
        n = min(max(c["lens"][b], 0), cols)
        want, bound = bo.attend(c["q"][b].numpy(), c["cache"], c["tables"][b], n, c["block"])
        worst = np.abs(got[b] - want) - (bound + half * (np.abs(want) + bound) + 2.0 ** -25)
        assert np.isfinite(got[b]).all() and worst.max() <= 0, f"sequence {b} of {n}: off by {np.abs(got[b] - want).max()}, bound {bound.max()}"


LAYERS = [(14, 2, 64), (4, 4, 64), (32, 4, 64), (12, 2, 128), (32, 8, 128), (3, 1, 128), (20, 1, 64), (8, 8, 80), (12, 2, 80), (34, 2, 80)]


@pytest.mark.parametrize("H,KV,D", LAYERS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_shared_layers(H, KV, D, dtype):
    c = _shared_case(H + D, H, KV, D, [(100, [101, 164, 300]), (17, [18]), (64, [65, 128, 129, 200, 90])])
    _check_shared(dict(c, dtype=dtype), _run_shared(c, dtype))


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 255, 700])
@pytest.mark.parametrize("more", [0, 1, 2, 16, 63, 64, 65])
def test_shared_lengths(prefix, more):
    """Prompts and own tokens that end before, at and behind blocks and tiles."""
    c = _shared_case(7 * prefix + more, 8, 2, 64, [(prefix, [prefix + more, prefix, prefix + 2 * more])])
    _check_shared(c, _run_shared(c))


@pytest.mark.parametrize("block,bits", [(16, 64), (32, 32), (48, 32), (64, 64), (80, 64), (256, 32)])
def test_shared_blocks(block, bits):
    c = _shared_case(block, 8, 2, 128, [(200, [201, 333, 290]), (block, [block + 1, 2 * block]), (0, [1, 70])], block=block)
    _check_shared(c, _run_shared(c, bits=bits))


def test_shared_sequences_without_tokens_groups_or_prompts():
    # a group of nobody, sequences shorter than what their group shares, empty ones, ones behind the last group
    c = _shared_case(3, 8, 2, 64, [(40, [50, 30, 0, 40, 1]), (90, []), (0, [0, 33]), (5, [5])], loose=[70, 0, 1])
    got = _run_shared(c)
    _check_shared(c, got)
    assert (got[[2, 5, 9]] == 0).all()
    # the first sequences in no group either, and no groups at all
    d = dict(c, starts=[2, 5, 5, 7, 8])
    d["prefix"] = [0] * 4
    _check_shared(d, _run_shared(d))
    e = dict(c, starts=[0], prefix=[])
    _check_shared(e, _run_shared(e))
    # lengths below 0 and past a row's columns
    cols = len(c["tables"][0]) * 16
    f = dict(c, lens=[cols + 100, 45, -3, 40, 2 ** 31 - 1] + c["lens"][5:])
    _check_shared(f, _run_shared(f))
    # a prompt said to be longer than the rows
    h = _shared_case(4, 4, 4, 64, [(64, [64, 64, 50])], spare=0)
    _check_shared(h, _run_shared(dict(h, prefix=[1 << 30])))


def test_shared_no_sequences():
    c = _shared_case(0, 4, 4, 64, [])
    c["q"] = torch.zeros((0, 4, 64), dtype=torch.float16)
    assert _run_shared(c).shape == (0, 4, 64)


def test_shared_starts_that_fall_or_leave_the_batch():
    """They name no groups; the call still ends, and every sequence with one group of its own is right."""
    c = _shared_case(5, 8, 2, 64, [(32, [60, 70]), (16, [40])])
    for starts in ([5, -1, 2], [-4, 2, 100], [0, 2, 1]):
        assert _run_shared(dict(c, starts=starts)).shape == (3, 8, 64)
    _check_shared(c, _run_shared(dict(c, starts=[-4, 2, 100])))


@pytest.mark.parametrize("sizes", [[1], [2], [16], [17], [63], [64], [65], [130], [5, 1, 33, 2]])
def test_shared_group_sizes(sizes):
    """Columns that end before, at and behind a set of 16."""
    c = _shared_case(sum(sizes), 6, 2, 64, [(150 + 10 * i, [150 + 10 * i + 1 + (7 * j) % 80 for j in range(n)]) for i, n in enumerate(sizes)])
    _check_shared(c, _run_shared(c))


def test_shared_many_sequences_and_parts():
    """More items than workgroups, and a prompt in more parts than a merging team has threads."""
    c = _shared_case(11, 2, 1, 64, [(65, [66 + i % 5 for i in range(3)]) for _ in range(150)], loose=[10] * 60)
    _check_shared(c, _run_shared(c), seqs=range(0, 510, 7))
    c = _shared_case(12, 8, 1, 128, [(40000, [40001, 40020])], block=64)
    _check_shared(c, _run_shared(c))


def test_shared_unseen_slots_hold_anything():
    """What no sequence sees: slots behind the last token, the blocks that a row names past its length, other rows' own."""
    c = _shared_case(21, 8, 2, 80, [(37, [41, 90, 37]), (0, [20])])
    want = _run_shared(c)
    cache = c["cache"].copy()
    seen = np.zeros(cache.shape[:2], dtype=bool)
    for row, n in zip(c["tables"], c["lens"]):
        for t in range(n):
            seen[row[t // 16], t % 16] = True
    nan = np.array([math.nan, math.inf, -math.inf, math.nan], dtype=np.float16).view(np.uint8)
    cache[~seen, :, 80:] = nan
    assert torch.equal(want, _run_shared(dict(c, cache=cache)))


@pytest.mark.parametrize("H,KV,D", [(1, 1, 64), (4, 4, 128), (2, 1, 80), (6, 2, 128), (12, 2, 80), (16, 2, 64)])
def test_shared_tokens_that_some_do_not_see_hold_anything(H, KV, D):
    """Shared tokens past a sequence's own last one, infinite or NaN for those that see them; and a prompt said to be longer
    than any sequence, over slots that nobody wrote."""
    c = _shared_case(22, H, KV, D, [(150, [170, 60, 150, 0, 100])])
    want = _run_shared(c)
    _check_shared(c, want)
    cache, row = c["cache"].copy(), c["tables"][0]
    for t, ruler in ((101, (0.5, 0.1, math.inf, 0.1)), (127, (0.5, 0.1, -1.0, math.nan)), (128, (0.5, 0.1, -math.inf, math.inf)),
                     (143, (math.nan, math.inf, math.nan, 0.2))):
        cache[row[t // 16], t % 16, :, D:] = np.array(ruler, dtype=np.float16).view(np.uint8)
    got = _run_shared(dict(c, cache=cache))
    assert torch.equal(got[[1, 3, 4]], want[[1, 3, 4]]) and not bool(torch.isfinite(got[[0, 2]]).any())
    d = _shared_case(23, H, KV, D, [(70, [70, 60, 33])])
    cache = d["cache"].copy()
    for t in range(70, 96):
        cache[d["tables"][0][t // 16], t % 16, :, D:] = np.array([math.nan, math.inf, -math.inf, math.nan], dtype=np.float16).view(np.uint8)
    far = _run_shared(dict(d, prefix=[96]))
    assert torch.equal(_run_shared(dict(d, cache=cache, prefix=[96])), far)
    _check_shared(dict(d, prefix=[96]), far)


def test_shared_strides_and_given_outputs():
    c = _shared_case(31, 12, 2, 64, [(50, [60, 55, 51])], loose=[9])
    want = _run_shared(c)
    fused = torch.randn((4, 16 * 64 + 24), device=DEV).half()
    view = fused[:, 8:8 + 12 * 64].view(4, 12, 64)
    view.copy_(c["q"])
    assert torch.equal(want, _run_shared(c, q=view))
    odd = torch.zeros((4, 12, 65), device=DEV, dtype=torch.float16)[:, :, 1:]          # rows that are not 16-byte aligned
    odd.copy_(c["q"])
    assert torch.equal(want, _run_shared(c, q=odd))
    wide = torch.full((6, 14, 72), -5.0, device=DEV)
    out = wide[1:5, 1:13, 4:68]
    assert _run_shared(c, out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out, want)
    wide[1:5, 1:13, 4:68] = -5.0
    assert (wide == -5.0).all()
    # tables: a view of wider ones, and one whose columns are not side by side
    t = _int(c["tables"])
    args = lambda x: (c["q"].to(DEV), torch.from_numpy(c["cache"]).to(DEV), x, _int(c["lens"]), _int(c["starts"]), _int(c["prefix"]), 16, 2)  # noqa: E731
    for x in (torch.cat([t, t - 100000], 1)[:, :t.shape[1]], t.T.contiguous().T):
        assert torch.equal(want, _kd().kv_dequant_decode_paged_shared(*args(x)))


def test_shared_agrees_with_the_batched_decode():
    c = _shared_case(41, 32, 8, 128, [(1000, [1001, 1100, 1333]), (300, [900])])
    want = _kd().kv_dequant_decode_paged_batched(c["q"].to(DEV), torch.from_numpy(c["cache"]).to(DEV), _int(c["tables"]), _int(c["lens"]), 16, 8)
    got = _run_shared(c)
    # (both within their bounds of the same 64-bit results: the batched one's tests have 2e-3 + 1e-2 |x|)
    assert float(((got - want).abs() - 2e-3 - 1e-2 * want.abs()).max()) <= 0
    _check_shared(c, got)


def test_shared_a_tail_far_below_a_sink():
    """One key takes nearly all weight, thousands lie 2^-20 below it: their sum still counts."""
    c = _shared_case(51, 4, 4, 64, [(9000, [9001, 9100])], block=64)
    d, q = 64, c["q"]
    q[:] = 1.0
    ruler = np.ascontiguousarray(c["cache"][..., d:]).view(np.float16)
    ruler[..., 0], ruler[..., 1] = 0.0, 0.0                   # scores of 0
    ruler[c["tables"][0][0], 0, :, 0] = 14.0 / 8.0             # one of 14 (64 dims of 14 / 8, over 8)
    ruler[..., 2], ruler[..., 3] = 1.0, 0.25
    c["cache"][..., d:] = ruler.view(np.uint8)
    c["cache"][c["tables"][0][0], 0, :, d // 2:d] = 0
    _check_shared(c, _run_shared(c))


@pytest.mark.parametrize("H,KV,D", [(8, 2, 64), (40, 2, 64), (8, 2, 80), (24, 2, 80), (16, 4, 128), (64, 4, 128)])
def test_shared_error_of_the_whole_answer(H, KV, D):
    """The norm of the error, which the bounds of single values leave far more room.  A weight is off by its exponential's and its
    two fp16 parts' roundings, 2^-21 of it, and its score's, each key's by itself: what they do to a mean of values is no
    larger a part of it.  As much again for the sums' own roundings: 2^-20 of the norm, where nothing is lost in one direction."""
    c = _shared_case(31 + D + H, H, KV, D, [(4099, [4099 + 70 * i for i in range(1, 5)]), (515, [530, 1500])])
    got = _run_shared(c).double().cpu().numpy()
    want = np.stack([bo.attend(c["q"][b].numpy(), c["cache"], c["tables"][b], n, c["block"])[0] for b, n in enumerate(c["lens"])])
    assert np.linalg.norm(got - want) <= 2.0 ** -20 * np.linalg.norm(want)


def test_shared_offsets_past_32_bits():
    """Blocks on both ends of a cache of 5 GiB."""
    H, KV, D, block = 32, 32, 128, 64
    n = (5 << 30) // (block * KV * (D + 8)) + 1
    cache = torch.empty((n, block, KV, D + 8), dtype=torch.uint8, device=DEV)
    c = _shared_case(61, H, KV, D, [(70, [80, 140]), (64, [65])], block=block)
    m = c["cache"].shape[0]
    place = [i if i % 2 else n - 1 - i for i in range(m)]
    cache[place] = torch.from_numpy(c["cache"]).to(DEV)
    far = dict(c, tables=[[place[x] for x in row] for row in c["tables"]])
    _check_shared(c, _run_shared(far, bits=64, cache=cache))
    assert torch.equal(_run_shared(far, cache=cache), _run_shared(c))


def test_shared_in_graphs_and_on_other_streams():
    c = _shared_case(71, 16, 2, 64, [(200, [210, 230, 205]), (90, [99, 100])], spare=8)
    cache, q, tables = torch.from_numpy(c["cache"]).to(DEV), c["q"].to(DEV), _int(c["tables"])
    lens, starts, prefix = _int(c["lens"]), _int(c["starts"]), _int(c["prefix"])
    call = lambda out=None: _kd().kv_dequant_decode_paged_shared(q, cache, tables, lens, starts, prefix, 16, 2, out=out)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, want)
    graphs = []
    for _ in range(2):                       # two graphs in one pool
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
            got = call()
        graphs.append((g, got))
    for step in range(4):                    # lengths that grow between the replays, eager work among them
        now = dict(c, lens=[n + 3 * step for n in c["lens"]])
        lens.copy_(_int(now["lens"]))
        graphs[step % 2][0].replay()
        got = graphs[step % 2][1].clone()
        torch.cuda.synchronize()
        assert torch.equal(got, call())
        _check_shared(now, got)


# =============================================================================
#  selection
# =============================================================================
def _select(logits, scores, keep=None, out=None, **kw):
    t = lambda x, d: None if x is None else torch.tensor(x, dtype=d, device=DEV).view(scores.shape)  # noqa: E731
    return _sv().beam_select(logits, scores, keep, finished=t(kw.pop("finished", None), torch.bool), lengths=t(kw.pop("lengths", None), torch.int32), **kw)


def _check_select(logits, scores, keep=None, **kw):
    scores = torch.as_tensor(scores, dtype=torch.float32)
    R, W = scores.shape
    keep = W if keep is None else keep
    got = _select(logits if logits.is_cuda else logits.to(DEV), scores.to(DEV), keep, **kw)
    want = bo.select(logits.cpu(), scores.double().tolist(), keep, kw.get("finished"), kw.get("lengths"), kw.get("length_penalty", 0.0),
                     -1 if kw.get("eos_token") is None else kw["eos_token"], kw.get("pad_token", 0), kw.get("keep_rows", False))
    assert got.tokens.tolist() == [[c[0] for c in a] for a in want]
    assert got.parents.tolist() == [[c[1] for c in a] for a in want]
    ref = torch.tensor([[c[2] for c in a] for a in want], dtype=torch.float64)
    s = got.scores.double().cpu()
    fine = torch.isfinite(ref)
    assert torch.equal(s[~fine], ref[~fine])
    # one rounding to fp32 of a sum in 64 bits (whose terms are below 2^11: 2^-30 is far above their roundings)
    assert float(((s - ref).abs() - 2.0 ** -24 * ref.abs() - 2.0 ** -30)[fine].max() if fine.any() else 0.0) <= 0
    if kw.get("finished") is None and kw.get("eos_token") is None:
        assert got.finished is None
    else:
        assert got.finished.tolist() == [[c[3] for c in a] for a in want]
    assert got.lengths is None if kw.get("lengths") is None else got.lengths.tolist() == [[c[4] for c in a] for a in want]
    return got


def _logits(seed, rows, vocab, dtype=torch.float32, scale=3.0):
    return (scale * torch.randn((rows, vocab), generator=_gen(seed))).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,W,V,K", [(1, 1, 1, 1), (1, 4, 32000, 4), (2, 3, 7, 3), (3, 2, 1000, 4), (1, 1, 50001, 64), (5, 7, 4097, 7), (2, 64, 333, 64),
                                     (1, 16, 20000, 32), (40, 8, 9001, 8), (1, 2, 300000, 5)])
def test_select_sizes(R, W, V, K, dtype):
    s = -10.0 * torch.rand((R, W), generator=_gen(V + W))
    _check_select(_logits(R + V, R * W, V, dtype), s, K)


@pytest.mark.parametrize("R,W,V,K", [(1, 64, 5000, 64), (1, 1, 151936, 64), (2, 20, 9000, 40), (1, 32, 40000, 17), (3, 5, 2000, 33), (1, 64, 32000, 16)])
@pytest.mark.parametrize("scores", ["near", "far", "one"])
def test_select_many_candidates(R, W, V, K, scores):
    """Many of many: beams that share the places, beams far behind one another, and one beam that has them all."""
    s = -torch.rand((R, W), generator=_gen(V + K)) * {"near": 1.0, "far": 300.0, "one": 1e-3}[scores]
    if scores == "one":
        s[:, 1:] -= 1000.0
    _check_select(_logits(R + V + K, R * W, V, torch.float16), s, K)


@pytest.mark.parametrize("W,V,K", [(1, 151936, 64), (8, 40000, 64), (64, 3000, 64), (8, 40000, 16), (3, 100000, 20)])
def test_select_many_that_tie(W, V, K):
    """More equal ranks than a workgroup lists, in all beams and in some."""
    x = torch.zeros((W, V), dtype=torch.float16)
    _check_select(x, torch.full((1, W), -3.0), K)
    x[:, V // 2:] = -1.0
    x[W // 2, 5::7] = 1.0
    _check_select(x, -3.0 * torch.ones((1, W)), K)


@pytest.mark.parametrize("keep_rows", [False, True])
def test_select_finished_lengths_and_penalties(keep_rows):
    g = _gen(4)
    R, W, V = 12, 6, 700
    x = _logits(9, R * W, V, torch.float16)
    s = (-6.0 * torch.rand((R, W), generator=g)).float()
    done = (torch.rand((R, W), generator=g) < 0.4).tolist()
    done[3], done[4] = [True] * W, [False] * W
    n = torch.randint(0, 30, (R, W), generator=g).tolist()
    for penalty in (0.0, 1.0, 0.6, -0.5):
        got = _check_select(x, s, finished=done, lengths=n, length_penalty=penalty, eos_token=5, pad_token=699, keep_rows=keep_rows)
    assert got.finished[3].all()
    _check_select(x, s, finished=done, keep_rows=keep_rows)
    _check_select(x, s, lengths=n, eos_token=int(x[0].argmax()), keep_rows=keep_rows)
    if keep_rows:                            # every parent that goes on has its own row
        p = _check_select(x, s, keep_rows=True).parents.cpu()
        for row in p.tolist():
            assert all(row[q] == q for q in set(row))


def test_select_beams_without_continuations():
    x = _logits(3, 8, 50)
    inf = math.inf
    _check_select(x, [[0.0, -inf, -inf, -inf], [-inf, -2.0, math.nan, -1.0]])
    got = _check_select(x, [[-inf] * 4, [-1.0] * 4], keep_rows=True)
    assert (got.scores[0] == -inf).all() and (got.parents[0] == 0).all()
    y = x.clone()
    y[0], y[1, 3:], y[2, ::2], y[5] = -inf, -inf, math.nan, math.nan
    _check_select(y, [[-1.0, -2.0, -3.0, -4.0], [-1.0, -0.5, -3.0, -4.0]], 16)
    # fewer continuations than wanted
    z = torch.full((2, 10), -inf)
    z[0, 7], z[1, 2] = 1.0, -5.0
    _check_select(z, [[-1.0, -2.0]], 9)
    _check_select(z[:1], [[-1.0]], 64, eos_token=0)


def test_select_infinite_and_huge_logits():
    x = _logits(3, 4, 40)
    x[0, 5] = x[0, 30] = math.inf            # they share the row's probability
    x[1, 7] = 3.0e38
    x[2] = -3.0e38
    x[3, 9] = -math.inf
    _check_select(x, [[-1.0, -1.5], [-2.0, -0.25]], 6)


def test_select_ties_go_to_the_lowest():
    for dtype in (torch.float16, torch.float32):
        for R, W, V, K in ((1, 4, 20000, 8), (2, 2, 9000, 64), (1, 1, 70000, 64), (1, 64, 5000, 64)):
            x = torch.zeros((R * W, V), dtype=dtype)
            _check_select(x, [[-1.0] * W] * R, K)                       # all alike
            x[:, 1::2] = -0.0
            _check_select(x, [[-1.0] * W] * R, K)                       # (two zeros are one number)
            x[:, V // 2:] = 1.0
            _check_select(x, [[-1.0] * W] * R, K)
    x = torch.randint(-3, 4, (8, 3000), generator=_gen(1)).half()       # many equal ones, and beams that are copies
    x[4:] = x[:4]
    s = torch.tensor([[-1.0, -2.0, -1.0, -2.0]]).repeat(2, 1)
    x[2:4] = x[:2]
    _check_select(x, s, 30)


def test_select_near_values_keep_their_order():
    """fp32 logits a last bit apart far from 0, and beams whose scores differ by as little."""
    x = 80.0 + 2.0 ** -17 * torch.randperm(6000, generator=_gen(2)).float()
    x = torch.stack([x, x.flip(0), x])
    s = torch.tensor([[-30.0, -30.0 + 2.0 ** -19, -30.0 - 2.0 ** -19]])
    _check_select(x, s, 40)


def test_select_strides_and_alignment():
    for dtype in (torch.float16, torch.float32):
        base = _logits(5, 12, 1300, dtype).to(DEV)
        for off in (0, 1, 3, 5, 8):
            for V in (1, 2, 9, 1291):
                _check_select(base[::2, off:off + V], -torch.rand((2, 3), generator=_gen(off)), 4)
        _check_select(base.T[:12, :900].T.contiguous().T, -torch.rand((3, 4), generator=_gen(3)))
        _check_select(base[:1].expand(6, 1300), -torch.rand((2, 3), generator=_gen(4)), 5)
    s = -torch.rand((4, 6), generator=_gen(6)).to(DEV)
    x = _logits(7, 12, 500).to(DEV)
    assert torch.equal(_sv().beam_select(x, s[:, ::2]).tokens, _sv().beam_select(x, s[:, ::2].contiguous()).tokens)


def test_select_repeats_and_graphs():
    x = _logits(8, 32, 30000, torch.float16).to(DEV)
    s = -torch.rand((4, 8), generator=_gen(8)).to(DEV)
    call = lambda: _sv().beam_select(x, s, keep_rows=True)  # noqa: E731
    want = call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call()
    for i in range(4):
        if i:
            x.copy_(_logits(80 + i, 32, 30000, torch.float16))
            want = call()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert a is b is None or torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other.tokens, want.tokens) and torch.equal(other.scores, want.scores)


# =============================================================================
#  reordering
# =============================================================================
def _reorder_case(seed, R, W, layers, KV, D, block, lens, columns=None):
    g = _gen(seed)
    columns = columns or max(lens) // block + 2
    blocks = R * W * columns + 3
    caches = [torch.randint(0, 256, (blocks, block, KV, D + 8), dtype=torch.uint8, generator=g).numpy() for _ in range(layers)]
    tables = torch.randperm(blocks, generator=g)[:R * W * columns].view(R * W, columns)
    return caches, tables


def _check_reorder(caches, tables, lens, parents, block, dtype=torch.int32, stacked=False):
    want_c, want_t = bo.reorder(caches, tables.tolist(), lens, parents, block)
    on = [torch.from_numpy(c).to(DEV) for c in caches]
    wide = torch.full((tables.shape[0], tables.shape[1] + 3), -9, dtype=dtype, device=DEV)
    t = wide[:, 1:1 + tables.shape[1]]
    t.copy_(tables)
    arg = torch.stack(on) if stacked else on
    assert _sv().kv_reorder_beams(arg, t, _int(lens), _int(parents).view(len(lens), -1), block) is None
    for a, b in zip(arg, want_c):
        assert np.array_equal(a.cpu().numpy(), b)
    assert t.tolist() == want_t
    assert (wide[:, 0] == -9).all() and (wide[:, -2:] == -9).all()


def _parents(seed, R, W, kind):
    g = _gen(seed)
    if kind == "any":
        return torch.randint(0, W, (R, W), generator=g).tolist()
    if kind == "turn":
        return [[(j + 1) % W for j in range(W)] for _ in range(R)]
    if kind == "one":
        return [[int(torch.randint(0, W, (1,), generator=g))] * W for _ in range(R)]
    return [list(range(W)) for _ in range(R)]


@pytest.mark.parametrize("kind", ["any", "turn", "one", "stay"])
@pytest.mark.parametrize("W", [1, 2, 4, 5, 8, 13, 16, 17, 40, 64])
def test_reorder_beams(W, kind):
    lens = [0, 1, 15, 16, 17, 31, 40]
    caches, tables = _reorder_case(W, 7, W, 2, 2, 64, 16, lens)
    _check_reorder(caches, tables, lens, _parents(W, 7, W, kind), 16)


@pytest.mark.parametrize("KV,D,block,layers", [(1, 64, 16, 1), (3, 80, 5, 3), (8, 128, 16, 33), (2, 128, 64, 2), (1, 80, 1, 2), (5, 128, 3, 130), (4, 64, 300, 1)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_reorder_caches(KV, D, block, layers, dtype):
    """Bytes of a block that are and are not a multiple of 16, many layers, blocks of one token."""
    lens = [2 * block + block // 2, block - 1, 3 * block]
    caches, tables = _reorder_case(D + block, 3, 4, layers, KV, D, block, lens)
    _check_reorder(caches, tables, lens, _parents(3, 3, 4, "any"), block, dtype, stacked=layers % 2 == 0)


def test_reorder_rows_without_room_and_odd_entries():
    lens = [64, 70, 1000, -5, 37]                      # rows of 4 blocks of 16: full, past it, far past it, below 0
    caches, tables = _reorder_case(1, 5, 3, 2, 2, 64, 16, lens, columns=4)
    _check_reorder(caches, tables, lens, _parents(2, 5, 3, "turn"), 16)
    # parents outside the request leave their row; blocks outside the cache are not copied
    lens = [20, 37, 5]
    caches, tables = _reorder_case(2, 3, 4, 2, 2, 64, 16, lens)
    tables[5, 2], tables[8, 0] = -1, caches[0].shape[0]
    _check_reorder(caches, tables, lens, [[1, -1, 4, 0], [1, 0, 3, 1 << 30], [3, 2, 1, 0]], 16)
    _check_reorder(caches, tables, lens, [[1, -1, 4, 0], [1, 0, 3, 1 << 30], [3, 2, 1, 0]], 16, torch.int64)


def test_reorder_forms_of_caches():
    lens = [21, 9]
    caches, tables = _reorder_case(5, 2, 3, 1, 2, 64, 16, lens)
    parents = _parents(5, 2, 3, "turn")
    want_c, want_t = bo.reorder(caches, tables.tolist(), lens, parents, 16)
    for form in (lambda c: c, lambda c: [c], lambda c: (c,), lambda c: c.unsqueeze(0)):
        c, t = torch.from_numpy(caches[0]).to(DEV), tables.int().to(DEV)
        _sv().kv_reorder_beams(form(c), t, _int(lens), _int(parents), 16)
        assert np.array_equal(c.cpu().numpy(), want_c[0]) and t.tolist() == want_t
    t = tables.int().to(DEV)                           # no caches: the tables alone
    _sv().kv_reorder_beams([], t, _int(lens), _int(parents), 16)
    assert t.tolist() == want_t
    e = torch.zeros((0, 4), dtype=torch.int32, device=DEV)
    _sv().kv_reorder_beams(torch.from_numpy(caches[0]).to(DEV), e, _int([]), _int([]).view(0, 3), 16)


def test_reorder_in_a_graph():
    lens = [21, 39]
    caches, tables = _reorder_case(6, 2, 5, 3, 2, 64, 16, lens)
    on, t, n = [torch.from_numpy(c).to(DEV) for c in caches], tables.int().to(DEV), _int(lens)
    p = _int(_parents(0, 2, 5, "stay"))
    _sv().kv_reorder_beams(on, t, n, p, 16)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _sv().kv_reorder_beams(on, t, n, p, 16)
    now, rows = caches, tables.tolist()
    for i in range(4):
        parents = _parents(60 + i, 2, 5, "any")
        p.copy_(_int(parents))
        g.replay()
        torch.cuda.synchronize()
        now, rows = bo.reorder(now, rows, lens, parents, 16)
        assert t.tolist() == rows and all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(on, now))


# =============================================================================
#  a search's steps
# =============================================================================
def test_steps_of_a_search():
    """metadata, store, attention over the shared prompts, selection, reordering, for more steps than a block holds; the other
    side keeps every beam's tokens by itself and copies them."""
    kd, sv = _kd(), _sv()
    g = _gen(77)
    R, W, H, KV, D, V, bs, steps = 3, 4, 8, 2, 64, 120, 16, 40
    lens = [37, 16, 5]
    B, room = R * W, -(-(max(lens) + steps) // bs)
    blocks = B * room
    cache = torch.zeros((blocks, bs, KV, D + 8), dtype=torch.uint8, device=DEV)
    free = torch.randperm(blocks, generator=g).int().to(DEV)
    tables = torch.zeros((B, room), dtype=torch.int32, device=DEV)
    prompt = [torch.randn((n, 2, KV, D), generator=g).half() for n in lens]
    head = torch.randn((H * D, V), generator=g).double().to(DEV) * 0.2
    # the prompts, for the first beam of each request; the others take over its row
    k = torch.cat(prompt)
    n = torch.zeros(B, dtype=torch.int32)
    n[::W] = torch.tensor(lens, dtype=torch.int32)
    m = sv.kv_step_metadata(n.to(DEV), _int([0] * B), tables, free, bs, sum(lens))
    kd.kv_quantize_store(k[:, 0].contiguous().to(DEV), k[:, 1].contiguous().to(DEV), cache, m.slot_mapping, bs)
    taken = m.free_end
    mine = torch.zeros((R, W, 1), dtype=torch.int64)   # a block of its own for every other beam's part of the prompt's last block
    at = int(taken)
    rows = tables.cpu()
    for r in range(R):
        for w in range(1, W):
            rows[r * W + w] = rows[r * W]
            if lens[r] % bs:
                rows[r * W + w, lens[r] // bs] = int(free[at])
                at += 1
    tables.copy_(rows)
    taken = _int([at])
    start = _int([W * r for r in range(R + 1)])
    ctx, own = _int(lens), _int([x for x in lens for _ in range(W)])
    sv.kv_reorder_beams(cache, tables, ctx, _int([[0] * W] * R), bs)
    scores = torch.full((R, W), -math.inf, device=DEV)
    scores[:, 0] = 0.0
    told = [[[(t[0], t[1]) for t in p] for _ in range(W)] for p in prompt]      # every beam's keys and values
    ref_scores = scores.double().tolist()
    for step in range(steps):
        q, k, v = (torch.randn((B, x, D), generator=g).half() for x in (H, KV, KV))
        m = sv.kv_step_metadata(_int([1] * B), own, tables, free, bs, B, free_start=taken)
        own, taken = m.seq_lens, m.free_end
        kd.kv_quantize_store(k.to(DEV), v.to(DEV), cache, m.slot_mapping, bs)
        out = kd.kv_dequant_decode_paged_shared(q.to(DEV), cache, tables, own, start, _int(lens), bs, KV)
        for b in range(B):
            told[b // W][b % W].append((k[b], v[b]))
        if step % 9 == 0:                              # against caches of each beam's tokens alone
            for b in range(B):
                kk, vv = (torch.stack([x[i] for x in told[b // W][b % W]]).numpy() for i in (0, 1))
                c = np.zeros((-(-len(kk) // bs), bs, KV, D + 8), dtype=np.uint8)
                bo.store(c, kk, vv, np.arange(len(kk)), bs)
                want, bound = bo.attend(q[b].numpy(), c, np.arange(len(c)), len(kk), bs)
                assert (np.abs(out[b].double().cpu().numpy() - want) <= bound + 2.0 ** -24 * np.abs(want)).all(), (step, b)
        logits = (out.double().view(B, -1) @ head).float()
        got = sv.beam_select(logits, scores)
        want = bo.select(logits.cpu(), ref_scores, W)
        assert got.tokens.tolist() == [[c[0] for c in a] for a in want] and got.parents.tolist() == [[c[1] for c in a] for a in want]
        scores = got.scores
        ref_scores = scores.double().tolist()
        ctx = own.view(R, W)[:, 0].contiguous()
        sv.kv_reorder_beams([cache], tables, ctx, got.parents, bs)
        parents = got.parents.tolist()
        told = [[list(told[r][p]) for p in parents[r]] for r in range(R)]
    assert int(taken) <= blocks
