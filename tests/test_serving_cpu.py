"""The serving step's operators without a GPU: what the entry points refuse (before any HIP call), through
the Python functions, the C ABI and the METH_FASTCALL binding, and the plain restatements that the GPU
tests compare with, against values worked out by hand."""
import math

import numpy as np
import pytest
import torch

import serving_oracle as so
from kernels import _native, serving


@pytest.fixture(scope="module")
def lib():
    if not _native.library_path().exists():
        pytest.fail(f"{_native.library_path()} is not built: run `python slm-turbo_amd/build_lib.py`")
    return _native.load()


def _args(defaults, kw):
    assert set(kw) <= set(defaults), set(kw) - set(defaults)
    return list({**defaults, **kw}.values())


def _metadata(**kw):
    return _args(dict(q=16, c=16, R=2, bt=16, bits=32, row=8, columns=8, free=16, F=4, fs=None, bs=16, N=5, qsl=16, sl=16,
                      pos=16, slots=16, fe=16, stream=None), kw)


def _rotary(**kw):
    return _args(dict(q=16, qt=512, qh=64, k=16, kt=128, kh=64, qo=16, qot=512, qoh=64, ko=16, kot=128, koh=64, N=3, H=8, KV=2,
                      D=64, dtype=1, pos=16, bits=64, inv=16, rot=64, inter=0, scale=1.0, stream=None), kw)


def _rotary_store(**kw):
    return _args(dict(q=16, qt=512, qh=64, k=16, kt=128, kh=64, v=16, vt=128, vh=64, qo=16, qot=512, qoh=64, ko=None, kot=0,
                      koh=0, cache=16, nb=4, bs=16, slots=16, N=3, H=8, KV=2, D=64, pos=16, bits=64, inv=16, rot=64, inter=0,
                      scale=1.0, stream=None), kw)


def _prompt(**kw):
    return _args(dict(q=16, qt=512, qh=64, k=16, kt=128, kh=64, v=16, vt=128, vh=64, qs=16, ks=None, R=1, N=3, M=3, H=8, KV=2,
                      D=64, dtype=1, causal=1, scale=0.125, out=16, ot=512, oh=64, clear=0, ws=None, wsb=0, stream=None), kw)


def _sample(**kw):
    return _args(dict(x=16, dtype=0, row=100, B=2, V=100, u=16, ts=None, t=1.0, ks=None, k=0, ps=None, p=1.0, ms=None, m=0.0,
                      tokens=16, probs=None, ws=None, wsb=0, stream=None), kw)


REFUSED = [
    ("step_metadata", _metadata, [
        (dict(R=-1), "invalid sizes"), (dict(columns=-1), "invalid sizes"), (dict(F=-1), "invalid sizes"),
        (dict(N=-1), "invalid sizes"), (dict(N=2**31 - 1), "invalid sizes"), (dict(bs=0), "block_size must be positive"),
        (dict(bits=16), "block table must be int32 or int64"), (dict(row=7), "rows overlap"), (dict(q=None), "null pointer"),
        (dict(bt=None), "null pointer"), (dict(free=None), "null pointer"), (dict(slots=None), "null pointer"),
        (dict(fe=None), "null pointer"),
        (dict(sl=1024, c=1024), "overlaps an input"), (dict(fe=2048, fs=2048), "overlaps an input"),
        (dict(pos=4096, q=4100), "overlaps an input"), (dict(qsl=8192, free=8192 + 8), "overlaps an input")]),
    ("rotary", _rotary, [
        (dict(D=96), "head_dim must be 64/80/128"), (dict(N=-1), "invalid sizes"), (dict(H=-1), "invalid sizes"),
        (dict(rot=0), "rotary_dim must be even"), (dict(rot=33), "rotary_dim must be even"), (dict(rot=66), "rotary_dim must be even"),
        (dict(bits=16), "positions must be int32 or int64"), (dict(dtype=3), "dtype must be"), (dict(q=None), "null pointer"),
        (dict(k=None), "null pointer"), (dict(ko=None), "null pointer"), (dict(inv=None), "null pointer")]),
    ("rotary_quantize_store", _rotary_store, [
        (dict(D=96), "head_dim must be 64/80/128"), (dict(KV=0), "invalid sizes"), (dict(bs=0), "invalid sizes"),
        (dict(nb=-1), "invalid sizes"), (dict(rot=80), "rotary_dim must be even"), (dict(v=None), "null pointer"),
        (dict(slots=None), "null pointer"), (dict(cache=4), "8-byte aligned")]),
    ("prompt_attention", _prompt, [
        (dict(D=96), "head_dim must be 64/80/128"), (dict(KV=3), "H not divisible"), (dict(KV=0), "H not divisible"),
        (dict(dtype=0), "dtype must be fp16 or bf16"), (dict(N=-1), "invalid sizes"), (dict(R=-1), "invalid sizes"),
        (dict(scale=0.0), "scale must be positive"), (dict(scale=-1.0), "scale must be positive"),
        (dict(scale=math.nan), "scale must be positive"), (dict(scale=math.inf), "scale must be positive"),
        (dict(q=None), "null pointer"), (dict(v=None), "null pointer"), (dict(q=8), "16-byte aligned"),
        (dict(kt=130), "16-byte aligned"), (dict(vh=4), "16-byte aligned"), (dict(out=4), "8-byte aligned"), (dict(oh=66), "8-byte aligned"),
        (dict(q=32, out=64, ws=2), "workspace must be 4-byte aligned"), (dict(q=32, v=48), "out must not be k or v"), (dict(q=32, k=48), "out must not be k or v")]),
    ("sample_tokens", _sample, [
        (dict(B=-1), "invalid sizes"), (dict(V=0), "invalid sizes"), (dict(dtype=5), "dtype must be"),
        (dict(t=-1.0), "temperature must be"), (dict(t=math.nan), "temperature must be"), (dict(k=-1), "top_k must be"),
        (dict(p=1.5), "top_p must lie"), (dict(p=math.nan), "top_p must lie"), (dict(m=-0.1), "min_p must lie"),
        (dict(m=2.0), "min_p must lie"), (dict(x=None), "null pointer"), (dict(u=None), "null pointer"),
        (dict(tokens=None), "null pointer"), (dict(V=50_000), "workspace of"), (dict(V=50_000, ws=8, wsb=1 << 30), "workspace of")]),
]


@pytest.mark.parametrize("name,make,kw,message", [(n, m, kw, msg) for n, m, cases in REFUSED for kw, msg in cases])
def test_refused_by_both_bindings(lib, name, make, kw, message):
    args = make(**kw)
    assert getattr(lib, "slmt_" + name)(*args) == _native.ERR_INVALID
    assert message in _native.last_error(lib)
    fast = _native.fast()
    if fast is None:
        pytest.fail("kernels/_slmt_fast is not built: run `python slm-turbo_amd/build_lib.py`")
    assert lib.slmt_quantize_store(None, 1024, None, 1024, None, 4, 16, None, 0, 8, 128, None) == _native.OK   # clears the message
    assert getattr(fast, name)(*[0 if a is None else a for a in args]) == _native.ERR_INVALID
    assert message in _native.last_error(lib)


@pytest.mark.parametrize("name,args", [
    ("rotary", _rotary(N=0, q=None, k=None)), ("rotary_quantize_store", _rotary_store(N=0, q=None)),
    ("prompt_attention", _prompt(N=0, q=None)), ("prompt_attention", _prompt(R=0, out=None)), ("sample_tokens", _sample(B=0, x=None))])
def test_nothing_to_do(lib, name, args):
    assert getattr(lib, "slmt_" + name)(*args) == _native.OK


def test_vocabularies_past_the_limit(lib):
    assert lib.slmt_sample_workspace_bytes(3, 1 << 22) > 0
    assert lib.slmt_sample_workspace_bytes(3, (1 << 22) + 1) == -1
    assert "vocabularies of up to" in _native.last_error(lib)
    assert lib.slmt_sample_tokens(*_sample(V=(1 << 22) + 1)) == _native.ERR_UNSUPPORTED


def test_workspaces_of_prompts(lib):
    for args, message in (((1, 5000, 1, 8, 96), "head_dim must be"), ((1, 5000, 1, 0, 64), "invalid sizes"), ((-1, 5000, 1, 8, 64), "invalid sizes"),
                          ((1, -1, 1, 8, 64), "invalid sizes"), ((1, 5000, -1, 8, 64), "invalid sizes")):
        assert lib.slmt_prompt_workspace_bytes(*args) == -1
        assert message in _native.last_error(lib)
    assert lib.slmt_prompt_workspace_bytes(0, 5000, 1, 8, 64) == 0 and lib.slmt_prompt_workspace_bytes(1, 5000, 0, 8, 64) == 0


def test_floats_reach_the_binding_as_numbers():
    fast = _native.fast()
    with pytest.raises(TypeError):
        fast.prompt_attention(*[0 if a is None else a for a in _prompt(scale="x")])
    with pytest.raises(TypeError):
        fast.rotary(1.5, *[0 if a is None else a for a in _rotary()][1:])
    with pytest.raises(TypeError):
        fast.sample_tokens(1, 2)


def _half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def test_python_calls_want_tensors_of_the_gpu():
    pos, inv = torch.zeros(3, dtype=torch.int64), torch.ones(32)
    start = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="rotary: q must be a CUDA tensor"):
        serving.kv_rotary(_half(3, 4, 64), None, pos, inv)
    with pytest.raises(RuntimeError, match="rotary store: q must be a CUDA tensor"):
        serving.kv_rotary_quantize_store(_half(3, 4, 64), _half(3, 2, 64), _half(3, 2, 64),
                                         torch.zeros((2, 16, 2, 72), dtype=torch.uint8), pos, 16, pos, inv)
    with pytest.raises(RuntimeError, match="prompt attention: q must be a CUDA tensor"):
        serving.kv_prompt_attention(_half(3, 4, 64), _half(3, 2, 64), _half(3, 2, 64), start)
    with pytest.raises(RuntimeError, match="sample: logits must be a CUDA tensor"):
        serving.sample_tokens(torch.zeros(2, 5), torch.zeros(2))
    with pytest.raises(RuntimeError, match="step metadata: query_lens must be a CUDA tensor"):
        serving.kv_step_metadata(start, start, torch.zeros((2, 3), dtype=torch.int32), start, 16, 4)


def test_python_calls_refuse_shapes_and_gradients():
    with pytest.raises(AssertionError, match="q must be"):
        serving.kv_rotary(_half(3, 64), None, None, None)
    with pytest.raises(AssertionError, match="head_dim"):
        serving.kv_rotary(_half(3, 1, 96), None, None, None)
    with pytest.raises(AssertionError, match="not divisible"):
        serving.kv_prompt_attention(_half(3, 4, 64), _half(3, 3, 64), _half(3, 3, 64), None)
    with pytest.raises(AssertionError, match="logits must be"):
        serving.sample_tokens(torch.zeros(5), None)
    for call in (lambda t: serving.kv_rotary(t, None, None, None), lambda t: serving.kv_prompt_attention(t, t, t, None),
                 lambda t: serving.sample_tokens(t[:, 0], None)):
        with pytest.raises(RuntimeError, match="no gradients"):
            call(torch.zeros((2, 2, 64), requires_grad=True))


def test_rotary_frequencies_refuse_what_they_do_not_know():
    with pytest.raises(ValueError, match="rotary_dim"):
        serving.rotary_frequencies(7)
    with pytest.raises(ValueError, match="rope_type"):
        serving.rotary_frequencies(8, scaling=dict(rope_type="longest"))
    with pytest.raises(ValueError, match="rope_type"):
        serving.rotary_frequencies(8, scaling=dict(type="longest"))
    yarn = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64)
    for name, value in (("mscale", 1.0), ("mscale_all_dim", 1.0), ("truncate", False)):
        with pytest.raises(ValueError, match=name):
            serving.rotary_frequencies(8, scaling={**yarn, name: value})
    want = serving.rotary_frequencies(8, scaling=yarn)
    old = dict(yarn, type=yarn["rope_type"], truncate=True, mscale=None)
    del old["rope_type"]
    got = serving.rotary_frequencies(8, scaling=old)
    assert torch.equal(got[0], want[0]) and got[1] == want[1]


def test_the_metadata_walk_by_hand():
    tables, start, seq, pos, slots, taken = so.step_metadata([3, 0, 2], [15, 4, 0], [[8, -7], [9, -7], [-7, -7]], [1, 2, 3], 16, 6)
    assert tables == [[8, 1], [9, -7], [2, -7]]
    assert start == [0, 3, 3, 5] and seq == [18, 4, 2] and taken == 2
    assert pos == [15, 16, 17, 0, 1, 0] and slots == [143, 16, 17, 32, 33, -1]
    # one block short: the second request's token keeps its place and has no slot
    assert so.step_metadata([17, 1], [0, 16], [[-7, -7], [5, -7]], [1, 2], 16, 18)[2:] == (
        [17, 16], list(range(17)) + [16], list(range(16, 32)) + [32, -1], 3)


def test_the_sampler_by_hand():
    row = np.log(np.array([0.1, 0.4, 0.1, 0.3, 0.1]))
    draw = lambda u, **kw: so.sample(row, u, **{**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **kw})  # noqa: E731
    assert [draw(u)[0] for u in (0.0, 0.05, 0.15, 0.55, 0.75, 0.95)] == [0, 0, 1, 2, 3, 4]
    assert draw(0.55, top_k=2) == (1, pytest.approx(4 / 7)) and draw(0.6, top_k=2)[0] == 3
    assert draw(0.0, top_k=3)[0] == 0 and draw(0.99, top_k=3)[0] == 3        # of equal ones the lowest index
    assert draw(0.99, top_p=0.41)[0] == 3 and draw(0.99, top_p=0.39)[0] == 1
    assert draw(0.99, min_p=0.5)[0] == 3 and draw(0.99, min_p=0.8)[0] == 1
    assert draw(0.9, temperature=0.0) == (1, 1.0)


def test_the_attention_by_hand():
    q = torch.ones((2, 1, 1))
    k, v = torch.tensor([[[0.0]], [[math.log(3.0)]]]), torch.tensor([[[4.0]], [[math.inf]]])
    out = so.prompt_attention(q, k, v, [0, 2], [0, 2], True, 1.0)[0]
    assert out[0].item() == 4.0 and out[1].item() == math.inf
    v[1] = 8.0
    assert so.prompt_attention(q, k, v, [0, 2], [0, 2], True, 1.0)[0][1].item() == pytest.approx(7.0)
    assert so.prompt_attention(q, k[:1], v[:1], [0, 2], [0, 1], True, 1.0)[0].flatten().tolist() == [0.0, 4.0]
