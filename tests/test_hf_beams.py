"""Beam search in a model (adapters.hf_llama.beam_search): metadata, shared decode, selection and reordering together, every
step's choice against the plain selection, every beam's logits against generation from the beam's own tokens."""
import pytest
import torch

import beam_oracle as bo
from adapters import hf_llama as hl

DEV = "cuda:0"
VOCAB = 997


def _model(dtype=torch.float16, device=DEV, heads=(8, 2, 64), seed=11):
    cfg = hl.llama_1b_config(vocab_size=VOCAB, hidden_size=heads[0] * 64, intermediate_size=704, num_hidden_layers=3, num_attention_heads=heads[0],
                             num_key_value_heads=heads[1], head_dim=heads[2], max_position_embeddings=512)
    return hl.build_model(cfg, device, dtype=dtype, seed=seed)


def _prompts(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, VOCAB, (n,), generator=g) for n in lens]


def test_beam_search_refuses_what_it_cannot_serve():
    with pytest.raises(ValueError, match="fp16"):
        hl.beam_search(_model(torch.float32, "cpu"), _prompts([3]), 2, 2)
    model = _model(device="cpu")
    for prompts, n in (([], 2), (_prompts([3, 0]), 2), (_prompts([3]), 0), ([torch.zeros(1, 3, dtype=torch.int64)], 1)):
        with pytest.raises(ValueError, match="prompts must be"):
            hl.beam_search(model, prompts, n, 2)
    for W, bs in ((0, 16), (65, 16), (2, 8), (2, 24)):
        with pytest.raises(ValueError, match="1 to 64 beams"):
            hl.beam_search(model, _prompts([3]), 2, W, block_size=bs)
    with pytest.raises(ValueError, match="4096 beams"):
        hl.beam_search(model, _prompts([1] * 65), 2, 64)
    for kw in (dict(pad_token=-1), dict(pad_token=VOCAB), dict(eos_token=VOCAB), dict(eos_token=-1)):
        with pytest.raises(ValueError, match="must be tokens"):
            hl.beam_search(model, _prompts([3]), 2, 2, **kw)


def _check_choices(steps, W, **kw):
    """Every step's results are the plain selection's."""
    for i, (logits, scores, finished, lengths, best) in enumerate(steps):
        want = bo.select(logits.cpu(), scores.double().tolist(), W, finished.tolist(), lengths.tolist(), kw.get("length_penalty", 0.0),
                         -1 if kw.get("eos_token") is None else kw["eos_token"], kw.get("pad_token", 0), i > 0)
        assert best.tokens.tolist() == [[c[0] for c in a] for a in want], i
        assert best.parents.tolist() == [[c[1] for c in a] for a in want], i
        assert best.finished.tolist() == [[c[3] for c in a] for a in want] and best.lengths.tolist() == [[c[4] for c in a] for a in want]
        if i + 1 < len(steps):
            assert all(a is b for a, b in zip(steps[i + 1][1:4], best[2:]))


def _paths(steps, tokens, scores, lengths, penalty=0.0):
    """The beams' rows of every step's logits, from the choices; the results are those of the last step, in order."""
    last, (R, W, n) = steps[-1][4], tokens.shape
    assert n == len(steps)
    rows = []
    for r in range(R):
        rank = [float(last.scores[r, w].double()) / max(int(last.lengths[r, w]), 1) ** penalty for w in range(W)]
        order = sorted(range(W), key=lambda w: -rank[w])
        assert scores[r].tolist() == [float(last.scores[r, w]) for w in order]
        assert lengths[r].tolist() == [int(last.lengths[r, w]) for w in order]
        for place, w in enumerate(order):
            row, told = [], []
            for s in reversed(steps):
                told.append(int(s[4].tokens[r, w]))
                w = int(s[4].parents[r, w])
                row.append(w)
            assert tokens[r, place].tolist() == told[::-1]
            rows.append(row[::-1])
    return rows


@pytest.mark.gpu
@pytest.mark.parametrize("heads,W,lens,N", [((8, 2, 64), 4, [5, 1, 70, 32], 22), ((4, 4, 128), 3, [16, 31], 20),
                                            ((6, 1, 80), 5, [33, 47, 15], 18), ((8, 2, 64), 1, [40, 3], 4), ((8, 2, 64), 64, [17], 3), ((8, 2, 64), 2, [32, 16], 17)])
def test_beams_match_generation_from_their_own_tokens(heads, W, lens, N):
    """More steps than a block holds.  The logits of a beam along its path against those of its tokens alone, without beams,
    sharing or moves: 4-bit codes are the same but where a K/V value that differs in its last bit rounds to another."""
    model = _model(heads=heads)
    prompts = _prompts(lens)
    tokens, scores, lengths, steps = hl.beam_search(model, prompts, N, W, return_logits=True)
    assert tokens.shape == (len(lens), W, N) and bool((lengths == N).all())
    _check_choices(steps, W)
    rows = _paths(steps, tokens, scores, lengths)
    for r, p in enumerate(prompts):
        _, alone = hl.generate(model, [p] * W, N, forced=tokens[r].cpu(), return_logits=True)
        for w in range(W):
            total = 0.0
            for i in range(N):
                now = steps[i][0].view(len(lens), -1, VOCAB)[r, rows[r * W + w][i]].double()
                cos = torch.nn.functional.cosine_similarity(now, alone[i, w].double(), dim=0)
                assert float(cos) > 0.999, f"prompt {r}, beam {w}, step {i}: cosine {float(cos)}"
                total += float(torch.log_softmax(now, 0)[tokens[r, w, i]])
            # every step rounds the sum once to fp32
            assert abs(float(scores[r, w]) - total) <= N * 2.0 ** -24 * abs(total) + 1e-9
    assert all(len({tuple(t) for t in beams}) == W for beams in tokens.tolist())      # (no beam twice)
    again = hl.beam_search(model, prompts, N, W)
    assert len(again) == 3 and torch.equal(again[0], tokens) and torch.equal(again[1], scores)


@pytest.mark.gpu
@pytest.mark.parametrize("penalty", [0.0, 1.0, -0.5])
def test_beams_that_end(penalty):
    """An end that some beams draw: padding behind it, scores and lengths that stand, and an early end where all have ended."""
    model = _model()
    prompts, W, N = _prompts([20, 7], seed=4), 3, 12
    free = hl.beam_search(model, prompts, N, W)[0]
    eos = int(free[0, 0, 1])
    kw = dict(length_penalty=penalty, eos_token=eos, pad_token=5)
    tokens, scores, lengths, steps = hl.beam_search(model, prompts, N, W, return_logits=True, **kw)
    _check_choices(steps, W, **kw)
    _paths(steps, tokens, scores, lengths, penalty)
    for told, n in zip(tokens.flatten(0, 1).tolist(), lengths.flatten().tolist()):
        assert told[n:] == [5] * (len(told) - n) and eos not in told[:n - 1]
        assert n == len(told) or told[n - 1] == eos


@pytest.mark.gpu
def test_a_search_ends_when_all_beams_have():
    model = _model()
    with torch.no_grad():                              # every token is drawn often: a vocabulary of few likely ones
        model.lm_head.weight[4:].zero_()
        model.lm_head.weight[:4].mul_(40.0)
    tokens, scores, lengths, steps = hl.beam_search(model, _prompts([9, 30]), 200, 2, eos_token=0, return_logits=True)
    _check_choices(steps, 2, eos_token=0)
    _paths(steps, tokens, scores, lengths)
    ended = [bool(s[4].finished.all()) for s in steps]
    assert not any(ended[:-1]) and (ended[-1] or len(steps) == 200)
