"""GPU: shared-prompt attention and beam selection where single roundings, ties and NaN decide: value steps of all sizes, tails far
below a sink, keys that are no numbers, rows that lie differently in memory; against plain restatements in 64 bits."""
import math

import numpy as np
import pytest
import torch

import beam_oracle as bo
from test_gpu_beams import DEV, _check_select, _gen, _run_shared, _shared_case, _sv

pytestmark = pytest.mark.gpu


# =============================================================================
#  weights of values, whatever their steps
# =============================================================================
def _rulers(c):
    """The case's rulers (kmin, kstep, vmin, vstep), float64 [blocks, tokens, KV, 4], to be changed and put back by _put."""
    d = c["q"].shape[2]
    return np.ascontiguousarray(c["cache"][..., d:]).view(np.float16).astype(np.float64)


def _put(c, ruler):
    d = c["q"].shape[2]
    c["cache"][..., d:] = ruler.astype(np.float16).view(np.uint8)
    return c


def _peaked(c, step):
    """Keys and values about 0: scores of a deviation of 2.5 (q has one of 1, codes of 4.6), values with steps of `step`, give or
    take 30 %.  (Each ruler from the one that was there, so that copies of a token stay alike.)"""
    r = _rulers(c)
    r[..., 1] = (2.4 * r[..., 1]).astype(np.float16)
    r[..., 3] = (4.0 * step * r[..., 3]).astype(np.float16)
    r[..., 0], r[..., 2] = -7.5 * r[..., 1], -7.5 * r[..., 3]
    return _put(c, r)


def _norms(c, got, seqs=None):
    """Errors of the sequences' answers, and their own size, as norms."""
    pairs = []
    for b in range(len(c["lens"])) if seqs is None else seqs:
        want = bo.attend(c["q"][b].numpy(), c["cache"], c["tables"][b], c["lens"][b], c["block"])[0]
        pairs.append((np.linalg.norm(got[b].double().cpu().numpy() - want), np.linalg.norm(want)))
    return pairs


# 4, 8, 16, 32, 32 + 16, 64 and 80 columns; own tokens of 1, 2, 4, 8, 12, 16 and 16 + 4
WIDTHS = [(2, 2, 64), (4, 2, 128), (8, 2, 80), (16, 2, 64), (24, 2, 80), (64, 4, 128), (40, 2, 64)]


@pytest.mark.parametrize("H,KV,D", WIDTHS)
@pytest.mark.parametrize("step", [0.2, 0.02, 2e-3, 2e-4])
def test_shared_error_at_any_step(H, KV, D, step):
    """Every key's weight is off by its own roundings.  Its score, a number below 16 (four deviations of 2.5, base 2), is rounded
    some five times by up to 2^-21, which is 2^-21 / sqrt(3) sqrt(5) ln 2 of the weight in the mean, 2^-21.2; the exponential and the
    weight's two fp16 parts give 2^-23 and 2^-22.  With values about 0 their sum is off by as much of its norm, 2^-20.8
    together; the sums' own roundings, 2^-24 of what they hold, are below that: 2^-20 in all, whatever the steps are."""
    c = _peaked(_shared_case(int(131 + D + H), H, KV, D, [(4099, [4099 + 70 * i for i in range(1, 5)]), (515, [530, 1500])]), step)
    pairs = _norms(c, _run_shared(c))
    assert math.hypot(*[e for e, _ in pairs]) <= 2.0 ** -20 * math.hypot(*[n for _, n in pairs])


def _sink(H, KV, D, tokens, step, below, groups=1):
    """One key of value codes 0 that takes nearly all weight, the others, of codes from 12 to 15, `below` (base e) it; values
    without a minimum.  The same for many groups, so that each wave has many tiles."""
    c = _shared_case(151, H, KV, D, [(tokens, [tokens + 1, tokens + 100])], block=64)
    c["q"][:] = 1.0
    r = np.zeros_like(_rulers(c))
    r[c["tables"][0][0], 0, :, 0] = below / math.sqrt(D)      # (D dims of below / sqrt(D), over sqrt(D))
    r[..., 3] = step
    _put(c, r)
    c["cache"][..., D // 2:D] |= 0xCC
    c["cache"][c["tables"][0][0], 0, :, D // 2:D] = 0
    c.update(q=c["q"].repeat(groups, 1, 1), tables=c["tables"] * groups, lens=c["lens"] * groups, starts=[2 * i for i in range(groups + 1)],
             prefix=c["prefix"] * groups)
    return c


def _check_all(c, got, seqs=None):
    """Within the oracle's bound and half a step of the output: nothing for small values."""
    for b in range(len(c["lens"])) if seqs is None else seqs:
        n = c["lens"][b]
        want, bound = bo.attend(c["q"][b].numpy(), c["cache"], c["tables"][b], n, c["block"])
        x = got[b].double().cpu().numpy()
        assert (np.abs(x - want) <= bound + 2.0 ** -24 * (np.abs(want) + bound)).all(), (b, np.abs(x - want).max(), bound.max(), np.abs(want).max())


@pytest.mark.parametrize("H,KV,D", [(2, 1, 64), (4, 1, 80), (8, 1, 128), (16, 1, 64), (16, 1, 128), (20, 1, 80)])
@pytest.mark.parametrize("step", [2.0 ** -2, 2.0 ** -5, 2.0 ** -7, 2.0 ** -10, 2.0 ** -20])
def test_shared_tails_of_small_values(H, KV, D, step):
    c = _sink(H, KV, D, 9000, step, 14.0, groups=512)
    _check_all(c, _run_shared(c), [0, 1, 510, 1023])


@pytest.mark.parametrize("H,KV,D", [(2, 1, 64), (16, 1, 64)])
@pytest.mark.parametrize("step", [2.0 ** -2, 2.0 ** -5])
def test_shared_a_long_tail(H, KV, D, step):
    c = _sink(H, KV, D, 131072, step, 16.5, groups=512)
    _check_all(c, _run_shared(c), [0, 1, 1023])


@pytest.mark.parametrize("H,KV,D", WIDTHS)
def test_shared_steps_of_keys_without_weight(H, KV, D):
    """Keys of no weight, a millionth of it and less, whose steps are 2^18 times the others', take nothing from these.

    The queries' sum is D / 2 here, so a score is the difference of two terms of up to 7.5 kstep D / 2 log2(e) / sqrt(D) each, kstep up
    to 0.6: 26 with 64 dims and 37 with 128, whose roundings are up to 2^-20 and 2^-19.  Four are of that size (the integer sum's, the
    two rulers' and the first product's): 2^-19 / sqrt(3) sqrt(4) ln 2 = 2^-19.3 of a weight in the mean at most, with 2^-20.8
    for all that test_shared_error_at_any_step counts 2^-19.2.  So 2^-19 of the norm."""
    c = _peaked(_shared_case(7 + H, H, KV, D, [(1003, [1003 + 90 * i for i in range(1, 5)])]), 2.0 ** -8)
    c["q"] = (0.5 + 0.5 * c["q"].float()).half()
    r = _rulers(c)
    for i in range(0, 1003, 97):               # (also in the block that every sequence has for itself)
        for row in c["tables"]:
            r[row[i // 16], i % 16, :, 0] = -12.0 - 7.5 * r[row[i // 16], i % 16, :, 1]
            r[row[i // 16], i % 16, :, 3] = 2.0 ** 10
            r[row[i // 16], i % 16, :, 2] = -7.5 * 2.0 ** 10
    _put(c, r)
    for e, n in _norms(c, _run_shared(c)):
        assert e <= 2.0 ** -19 * n


@pytest.mark.parametrize("H,KV,D", WIDTHS)
def test_shared_steps_that_some_do_not_see(H, KV, D):
    """Shared tokens of the largest steps there are, behind the last one of shorter sequences."""
    c = _peaked(_shared_case(8 + H, H, KV, D, [(700, [720, 300, 700, 20, 417])]), 2.0 ** -8)
    r, row = _rulers(c), c["tables"][0]
    for i in (301, 420, 511, 640):
        r[row[i // 16], i % 16, :, 2:] = (-40000.0, 6000.0 if i < 500 else 60000.0)
    _put(c, r)
    for e, n in _norms(c, _run_shared(c), [1, 3, 4]):
        assert e <= 2.0 ** -20 * n
    _check_all(c, _run_shared(c))


@pytest.mark.parametrize("H,KV,D", WIDTHS)
def test_shared_values_without_steps(H, KV, D):
    """Values that are all alike in a key (steps of 0), for all keys and for those with nearly all the weight."""
    c = _peaked(_shared_case(9 + H, H, KV, D, [(600, [601, 650, 777])]), 0.2)
    r = _rulers(c)
    r[..., 2], r[..., 3] = 0.75, 0.0
    _put(c, r)
    _check_all(c, _run_shared(c))
    c = _sink(H, KV, D, 2000, 2.0 ** -9, 14.0)
    r = _rulers(c)
    r[c["tables"][0][0], 0, :, 3] = 0.0
    _put(c, r)
    _check_all(c, _run_shared(c))


# =============================================================================
#  keys that are no numbers
# =============================================================================
@pytest.mark.parametrize("H,KV,D", WIDTHS)
@pytest.mark.parametrize("tokens", [1, 64, 65, 66, 129, 300])
def test_shared_keys_that_are_no_numbers(H, KV, D, tokens):
    """A NaN score reaches every sequence that sees it, also where it is all that a tile holds, and no other."""
    c = _shared_case(tokens, H, KV, D, [(tokens, [tokens + 5, tokens - 1, tokens, tokens + 70]), (40, [41, 90])])
    want = _run_shared(c)
    row, at = c["tables"][0], tokens - 1
    for ruler in ((math.nan, 0.1), (0.5, math.nan)):
        cache = c["cache"].copy()
        cache[row[at // 16], at % 16, :, D:D + 4] = np.array(ruler, dtype=np.float16).view(np.uint8)
        got = _run_shared(dict(c, cache=cache))
        assert torch.equal(got[[1, 4, 5]], want[[1, 4, 5]])
        assert bool(torch.isnan(got[[0, 2, 3]]).all())
    cache = c["cache"].copy()                  # a prompt of nothing else
    for t in range(tokens):
        cache[row[t // 16], t % 16, :, D:D + 2] = np.array(math.nan, dtype=np.float16).view((np.uint8, 2))
    got = _run_shared(dict(c, cache=cache))
    assert torch.equal(got[[4, 5]], want[[4, 5]]) and bool(torch.isnan(got[[0, 2, 3]]).all())
    assert bool(torch.isnan(got[1]).all()) if tokens > 1 else bool((got[1] == 0).all())


@pytest.mark.parametrize("H,KV,D", WIDTHS)
def test_own_keys_that_are_no_numbers(H, KV, D):
    """The same of a sequence's own tokens: one, the last of several, and all of them."""
    c = _shared_case(3, H, KV, D, [(100, [101, 300, 229]), (0, [1, 70])])
    want = _run_shared(c)
    for b, at in ((0, 100), (1, 150), (1, 299), (3, 0), (4, 64)):
        cache = c["cache"].copy()
        cache[c["tables"][b][at // 16], at % 16, :, D:D + 2] = np.array(math.nan, dtype=np.float16).view((np.uint8, 2))
        got = _run_shared(dict(c, cache=cache))
        others = [i for i in range(5) if i != b]
        assert torch.equal(got[others], want[others]) and bool(torch.isnan(got[b]).all())


# =============================================================================
#  equal beams
# =============================================================================
@pytest.mark.parametrize("V", [1001, 4099, 32001, 50257, 151935])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_select_equal_beams_go_by_their_places(V, dtype):
    """Rows of the same logits that lie differently in memory, as those of an odd vocabulary do, have the same ranks."""
    for seed in range(4):
        x = (3.0 * torch.randn((3, V), generator=_gen(10 * V + seed))).to(dtype)
        x = x[[0, 0, 1, 0, 2, 1, 0, 2, 2, 0, 0, 1, 2, 1, 1, 0]]          # two requests of eight beams
        s = torch.tensor([[-1.0] * 8, [-2.5] * 8])
        _check_select(x, s, 24)
        _check_select(x, s, keep_rows=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_select_results_do_not_hang_on_the_place_in_memory(dtype):
    """The same logits at every place of 16 bytes: the same scores to the last bit; and every row of a batch like the first."""
    V = 20011
    x = (3.0 * torch.randn((4, V), generator=_gen(5))).to(dtype).to(DEV)
    s = torch.tensor([[-0.5, -0.75, -1.0, -0.25]], device=DEV)
    want = _sv().beam_select(x, s, 16)
    for off in range(1, 9):
        wide = torch.zeros((4, V + 11), dtype=dtype, device=DEV)
        wide[:, off:off + V] = x
        got = _sv().beam_select(wide[:, off:off + V], s, 16)
        assert torch.equal(got.tokens, want.tokens) and torch.equal(got.parents, want.parents) and torch.equal(got.scores, want.scores)
    got = _sv().beam_select(x[:1].expand(7, V).contiguous(), torch.zeros((7, 1), device=DEV), 20)
    for i in range(1, 7):
        assert torch.equal(got.tokens[i], got.tokens[0]) and torch.equal(got.scores[i], got.scores[0])
