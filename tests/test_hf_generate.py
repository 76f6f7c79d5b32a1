"""Generation from prompts of different lengths (adapters.hf_llama.generate): metadata, prompt attention, packed
decode and sampling together in a model, against each prompt by itself and the plain sampler."""
import numpy as np
import pytest
import torch

import serving_oracle as so
from adapters import hf_llama as hl

DEV = "cuda:0"


def _model(dtype=torch.float16, device=DEV):
    cfg = hl.llama_1b_config(vocab_size=997, hidden_size=512, intermediate_size=704, num_hidden_layers=3, num_attention_heads=8,
                             num_key_value_heads=2, head_dim=64, max_position_embeddings=512)
    return hl.build_model(cfg, device, dtype=dtype, seed=11)


def _prompts(lens, vocab=997, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g) for n in lens]


def test_generate_refuses_what_it_cannot_serve():
    model = _model(torch.float32, "cpu")
    with pytest.raises(ValueError, match="fp16"):
        hl.generate(model, _prompts([3]), 2)
    for prompts, n in (([], 2), (_prompts([3, 0]), 2), (_prompts([3]), 0), ([torch.zeros(1, 3, dtype=torch.int64)], 1)):
        with pytest.raises(ValueError, match="prompts must be"):
            hl.generate(model, prompts, n)


@pytest.mark.gpu
def test_prompts_together_match_each_by_itself():
    """The logits of every step against the packed mode's for that prompt alone, fed the same tokens.  Prefill differs by the
    rounding of two fp16 attentions; the decode steps read the same 4-bit codes but where a K/V value that differs in its last
    bit rounds to another code.  A prompt of one token is a decode step for that mode, which reads its value from the 4-bit
    cache: it is compared with the fp16 mode, and its later steps with this function's for that prompt alone."""
    model = _model()
    lens, N = [5, 1, 70, 33, 16], 5
    prompts = _prompts(lens)
    forced = torch.randint(0, 997, (len(lens), N), generator=torch.Generator().manual_seed(3))
    _, logits = hl.generate(model, prompts, N, forced=forced, return_logits=True)
    for b, p in enumerate(prompts):
        if lens[b] > 1:
            run = hl.DecodeRunner(model, "packed", 1, lens[b] + N)
            want = [run(p.unsqueeze(0).to(DEV))] + [run(forced[b:b + 1, i:i + 1].to(DEV)) for i in range(N - 1)]
        else:
            first = hl.DecodeRunner(model, "fp16", 1, 1)(p.unsqueeze(0).to(DEV))
            want = [first] + list(hl.generate(model, [p], N, forced=forced[b:b + 1], return_logits=True)[1][1:])
        for i in range(N):
            cos = torch.nn.functional.cosine_similarity(logits[i, b].double(), want[i][0].double(), dim=0)
            assert float(cos) > 0.999, f"prompt {b}, step {i}: cosine {float(cos)}"


@pytest.mark.gpu
def test_sampled_tokens_are_those_of_the_plain_sampler():
    model = _model()
    lens, N = [9, 20, 1], 6
    u = torch.rand((N, len(lens)), generator=torch.Generator().manual_seed(5))
    u = u.to(DEV)
    kw = dict(temperature=0.8, top_k=50, top_p=0.9)
    tokens, logits = hl.generate(model, _prompts(lens), N, uniforms=u, return_logits=True, **kw)
    f32 = lambda x: float(np.float32(x))  # noqa: E731
    for i in range(N):
        for b in range(len(lens)):
            want, _ = so.sample(logits[i, b].double().cpu().numpy(), float(u[i, b]), f32(0.8), 50, f32(0.9), 0.0)
            assert int(tokens[b, i]) == want
    again = hl.generate(model, _prompts(lens), N, uniforms=u, **kw)
    assert torch.equal(tokens, again)
    greedy, logits = hl.generate(model, _prompts(lens), 2, return_logits=True)
    assert torch.equal(greedy, logits.argmax(-1).T)
