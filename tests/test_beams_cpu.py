"""Beam search and shared-prompt attention without a GPU: what the entry points refuse (before any HIP call), through the
Python functions, the C ABI and the METH_FASTCALL binding, and the plain restatements that the GPU tests compare with,
against values worked out by hand."""
import ctypes
import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import beam_oracle as bo
from kernels import _native, kv_dequant, serving


@pytest.fixture(scope="module")
def lib():
    if not _native.library_path().exists():
        pytest.fail(f"{_native.library_path()} is not built: run `python slm-turbo_amd/build_lib.py`")
    return _native.load()


def _args(defaults, kw):
    assert set(kw) <= set(defaults), set(kw) - set(defaults)
    return list({**defaults, **kw}.values())


def _shared(**kw):
    return _args(dict(q=16, qs=512, qh=64, cache=16, nb=40, bs=16, bt=16, bits=32, row=8, columns=8, lens=16, start=16, prefix=16,
                      R=2, B=5, H=8, KV=2, D=64, out=16, dtype=0, os=512, oh=64, ws=None, wsb=0, stream=None), kw)


def _select(**kw):
    at = {n: 4096 * (i + 1) for i, n in enumerate("x s fin n t p os of on".split())}
    return _args(dict(x=at["x"], dtype=1, row=100, R=2, W=3, V=100, s=at["s"], fin=at["fin"], n=at["n"], penalty=0.5, eos=-1, pad=0, K=3,
                      keep=0, t=at["t"], p=at["p"], os=at["os"], of=at["of"], on=at["on"], ws=None, wsb=0, stream=None), kw)


_POINTERS = {n: (ctypes.c_void_p * len(v))(*v) for n, v in {
    "two": [1 << 20, 1 << 24], "same": [1 << 20, 1 << 20], "close": [1 << 24, 1 << 20, (1 << 20) + 8], "odd": [1 << 20, (1 << 24) + 4],
    "null": [1 << 20, None]}.items()}


def _reorder(caches="two", **kw):
    at = ctypes.addressof(_POINTERS[caches]) if caches else None
    return _args(dict(caches=at, L=len(_POINTERS[caches]) if caches else 2, step=0, nb=40, bs=16, KV=2, D=64, bt=16, bits=32, row=8, columns=8,
                      lens=16, parents=16, R=2, W=4, stream=None), kw)


REFUSED = [
    ("decode_paged_shared", _shared, [
        (dict(D=96), "head_dim must be 64/80/128"), (dict(KV=3), "H not divisible"), (dict(KV=0), "H not divisible"), (dict(B=-1), "invalid sizes"),
        (dict(R=-1), "invalid sizes"), (dict(bs=8), "multiple of 16"), (dict(bs=0), "multiple of 16"), (dict(bs=-16), "multiple of 16"),
        (dict(bits=16), "block table must be int32 or int64"), (dict(dtype=2), "out must be fp32 or fp16"), (dict(nb=-1), "invalid sizes"),
        (dict(nb=1 << 31), "invalid sizes"), (dict(columns=-1), "invalid sizes"), (dict(q=None), "null pointer"), (dict(out=None), "null pointer"),
        (dict(lens=None), "null pointer"), (dict(start=None), "null pointer"), (dict(prefix=None), "null pointer"), (dict(cache=20), "8-byte aligned"),
        (dict(q=8), "16-byte aligned"), (dict(qh=68), "16-byte aligned"), (dict(out=8), "aligned to four elements"), (dict(oh=66), "aligned to four elements"),
        (dict(out=4, dtype=1), "aligned to four elements"), (dict(), "workspace of"), (dict(ws=16, wsb=1000), "workspace of"),
        (dict(ws=8, wsb=1 << 40), "16-byte aligned")]),
    ("beam_select", _select, [
        (dict(R=-1), "invalid sizes"), (dict(V=0), "invalid sizes"), (dict(dtype=3), "dtype must be"), (dict(penalty=math.nan), "length_penalty must be finite"),
        (dict(penalty=math.inf), "length_penalty must be finite"), (dict(n=None, on=None), "length_penalty needs lengths"),
        (dict(n=None, penalty=0.0), "lengths out need lengths"), (dict(pad=-1), "pad_token must be a token"), (dict(pad=100), "pad_token must be a token"),
        (dict(keep=1, K=4), "keep_rows needs as many"), (dict(x=None), "null pointer"), (dict(s=None), "null pointer"), (dict(t=None), "null pointer"),
        (dict(p=None), "null pointer"), (dict(os=None), "null pointer"), (dict(x=4097), "aligned to their type"), (dict(dtype=0, x=4098), "aligned to their type"),
        (dict(row=-1), "aligned to their type"), (dict(os=4096 * 2), "overlaps an input"), (dict(of=4096 * 3 + 5), "overlaps an input"),
        (dict(on=4096 * 4 - 23), "overlaps an input"), (dict(t=4096 + 1198), "overlaps an input"), (dict(of=4096 * 5 + 47), "outputs overlap"),
        (dict(p=4096 * 7 - 23), "outputs overlap"), (dict(), "workspace of"), (dict(ws=16, wsb=8), "workspace of"), (dict(ws=8, wsb=1 << 40), "workspace of")]),
    ("reorder_beams", _reorder, [
        (dict(D=96), "head_dim must be 64/80/128"), (dict(L=-1), "invalid sizes"), (dict(nb=-1), "invalid sizes"), (dict(bs=0), "invalid sizes"),
        (dict(KV=0), "invalid sizes"), (dict(columns=-1), "invalid sizes"), (dict(R=-1), "invalid sizes"), (dict(bits=8), "block table must be int32 or int64"),
        (dict(row=7), "rows overlap"), (dict(bt=None), "null pointer"), (dict(lens=None), "null pointer"), (dict(parents=None), "null pointer"),
        (dict(caches=None), "null pointer"), (dict(caches="null"), "null pointer"), (dict(caches="same"), "two caches overlap"),
        (dict(caches="close"), "two caches overlap"), (dict(step=40 * 16 * 2 * 72 - 8), "two caches overlap"), (dict(step=-8, L=3), "two caches overlap"),
        (dict(step=(1 << 24) + 4), "8-byte aligned"), (dict(caches="odd"), "8-byte aligned")]),
]
PAST = [
    ("decode_paged_shared", _shared, [
        (dict(B=4097), "at most 4096 sequences"), (dict(R=4097), "at most 4096 sequences"), (dict(KV=70000, H=70000), "too many heads"),
        (dict(columns=1 << 25, B=1), "too wide"), (dict(columns=1 << 27, bs=1 << 20, B=4096), "too wide"), (dict(columns=1 << 20, B=4096), "too wide"), (dict(bs=1 << 24, columns=1, KV=2), "2 GiB or more")]),
    ("beam_select", _select, [
        (dict(W=0), "must lie in 1 .. 64"), (dict(W=65), "must lie in 1 .. 64"), (dict(K=0), "must lie in 1 .. 64"), (dict(K=65), "must lie in 1 .. 64"),
        (dict(V=(1 << 22) + 1), "go up to 4194304"), (dict(R=1 << 30), "too many rows")]),
    ("reorder_beams", _reorder, [
        (dict(W=0), "must lie in 1 .. 64"), (dict(W=65), "must lie in 1 .. 64"), (dict(R=65536), "too many requests"), (dict(bs=1 << 24), "2 GiB or more")]),
]
CASES = [(n, m, kw, msg, s) for table, s in ((REFUSED, _native.ERR_INVALID), (PAST, _native.ERR_UNSUPPORTED)) for n, m, cases in table for kw, msg in cases]


@pytest.mark.parametrize("name,make,kw,message,status", CASES)
def test_refused_by_both_bindings(lib, name, make, kw, message, status):
    args = make(**kw)
    if name == "decode_paged_shared" and args[-3] is None and status == _native.ERR_UNSUPPORTED:
        args[-3:-1] = [16, 1 << 60]
    fast = _native.fast()
    if fast is None:
        pytest.fail("kernels/_slmt_fast is not built: run `python slm-turbo_amd/build_lib.py`")
    for call in (getattr(lib, "slmt_" + name), getattr(fast, name)):
        assert lib.slmt_quantize_store(None, 1024, None, 1024, None, 4, 16, None, 0, 8, 128, None) == _native.OK   # clears the message
        assert call(*[0 if a is None else a for a in args]) == status
        assert message in _native.last_error(lib)


def test_workspaces(lib):
    for args, message in (((5, 2, 8, 2, 96), "head_dim"), ((5, 2, 8, 3, 64), "H not divisible"), ((-1, 2, 8, 2, 64), "invalid sizes"),
                          ((5, -2, 8, 2, 64), "invalid sizes"), ((4097, 2, 8, 2, 64), "at most 4096")):
        assert lib.slmt_shared_workspace_bytes(*args) == -1
        assert message in _native.last_error(lib)
    for args, message in (((1, 0, 9, 1), "must lie"), ((1, 4, 0, 4), "invalid sizes"), ((1, 4, 9, 65), "must lie"), ((-1, 4, 9, 4), "invalid sizes")):
        assert lib.slmt_beam_workspace_bytes(*args) == -1
        assert message in _native.last_error(lib)
    assert lib.slmt_beam_workspace_bytes(0, 4, 9, 4) == 0
    # beams' partial results stay below the cache that they read: 64 sequences of 32 / 8 heads, 128 dims
    assert 0 < lib.slmt_shared_workspace_bytes(64, 1, 32, 8, 128) < 32 << 20
    assert lib.slmt_shared_workspace_bytes(0, 0, 32, 8, 128) > 0


@pytest.mark.parametrize("name,args", [
    ("decode_paged_shared", _shared(B=0, q=None)), ("beam_select", _select(R=0, x=None)), ("reorder_beams", _reorder(R=0, bt=None)),
    ("reorder_beams", _reorder(columns=0, lens=None))])
def test_nothing_to_do(lib, name, args):
    assert getattr(lib, "slmt_" + name)(*args) == _native.OK


def test_more_requests_than_a_launch_holds(lib):
    """One beam and few tokens: the rows would fit, but not a request's larger workgroups; refused before anything is launched."""
    far = {n: (i + 1) << 36 for i, n in enumerate("x s fin n t p os of on".split())}
    for R in (1 << 22, 15 << 20):
        args = _select(**far, R=R, W=1, K=1, ws=1 << 46, wsb=1 << 60)
        for call in (lib.slmt_beam_select, _native.fast().beam_select):
            assert call(*[0 if a is None else a for a in args]) == _native.ERR_UNSUPPORTED
            assert "too many rows for a launch" in _native.last_error(lib)


def test_python_calls_refuse_what_they_cannot_take():
    half = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    start = torch.zeros(2, dtype=torch.int32)
    cache = torch.zeros((2, 16, 2, 72), dtype=torch.uint8)
    shared = lambda q: kv_dequant.kv_dequant_decode_paged_shared(q, cache, start.view(1, 2), start[:1], start, start[:1], 16, 2)  # noqa: E731
    with pytest.raises(RuntimeError, match="shared decode: q must be a CUDA tensor"):
        shared(half(1, 4, 64))
    with pytest.raises(AssertionError, match="q must be"):
        shared(half(4, 64))
    with pytest.raises(AssertionError, match="head_dim"):
        shared(half(1, 4, 96))
    with pytest.raises(AssertionError, match="not divisible"):
        shared(half(1, 3, 64))
    select = lambda x, s, **kw: serving.beam_select(x, s, **kw)  # noqa: E731
    with pytest.raises(RuntimeError, match="beam select: logits must be a CUDA tensor"):
        select(torch.zeros(4, 9), torch.zeros(2, 2))
    with pytest.raises(AssertionError, match="logits must be"):
        select(torch.zeros(9), torch.zeros(2, 2))
    with pytest.raises(AssertionError, match="scores must be"):
        select(torch.zeros(4, 9), torch.zeros(4))
    with pytest.raises(AssertionError, match="parents must be"):
        serving.kv_reorder_beams(cache, start.view(2, 1), start, start, 16)
    with pytest.raises(RuntimeError, match="kv_caches must be"):
        serving.kv_reorder_beams(cache, start.view(2, 1), start[:1], start.view(1, 2), 32)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        serving.kv_reorder_beams(cache, start.view(2, 1), start[:1], start.view(1, 2), 16)
    for call in (lambda t: shared(t.half()), lambda t: select(t[0], torch.zeros(1, 2)), lambda t: select(t[0].detach(), t[0, :1, :2].view(1, 2))):
        with pytest.raises(RuntimeError, match="no gradients"):
            call(torch.zeros((1, 2, 64), requires_grad=True))
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no gradients"):
            call(forward_ad.make_dual(torch.zeros((1, 2, 64)), torch.ones((1, 2, 64))))


# =============================================================================
#  the plain restatements, by hand
# =============================================================================
def test_the_selection_by_hand():
    # softmax of (0, ln 3): 1/4, 3/4; of (ln 1, ln 1): 1/2, 1/2
    x = torch.tensor([[0.0, math.log(3.0)], [0.0, 0.0]], dtype=torch.float64)
    got = bo.select(x, [[math.log(0.5), math.log(0.4)]], 3)[0]
    # 3/8 (beam 0, token 1), then 1/5 twice (beam 1)
    assert [(t, w) for t, w, *_ in got] == [(1, 0), (0, 1), (1, 1)]
    assert np.allclose([math.exp(c[2]) for c in got], [0.375, 0.2, 0.2])
    # beam 0 has ended: its one continuation keeps its score; by length 1 / 3 it goes behind ln 0.2 / 4
    got = bo.select(x, [[math.log(0.5), math.log(0.4)]], 3, finished=[[True, False]], lengths=[[1, 3]], penalty=1.0, eos=1, pad=0)[0]
    assert got == [(0, 1, pytest.approx(math.log(0.2)), False, 4), (1, 1, pytest.approx(math.log(0.2)), True, 4), (0, 0, pytest.approx(math.log(0.5)), True, 1)]
    # two of beam 1 and none of beam 0: the first stays in row 1, the second takes row 0
    got = bo.select(x, [[-9.0, 0.0]], 2, keep_rows=True)[0]
    assert [(t, w) for t, w, *_ in got] == [(1, 1), (0, 1)]
    assert bo.select(x[:1], [[-math.inf]], 2)[0] == [(0, 0, -math.inf, False, None)] * 2


def test_the_reordering_by_hand():
    cache = np.arange(5 * 2 * 1 * 72, dtype=np.uint64).astype(np.uint8).reshape(5, 2, 1, 72)
    new, tables = bo.reorder([cache], [[0, 1], [2, 3]], [3], [[1, 1]], 2)
    assert tables == [[2, 1], [2, 3]]                    # the full block is shared, the filling one stays
    assert np.array_equal(new[0][1, 0], cache[3, 0]) and np.array_equal(new[0][1, 1], cache[1, 1])
    assert np.array_equal(new[0][[0, 2, 3, 4]], cache[[0, 2, 3, 4]])


def test_the_attention_by_hand():
    D = 64
    cache = np.zeros((2, 2, 1, D + 8), dtype=np.uint8)
    ruler = np.ascontiguousarray(cache[..., D:]).view(np.float16)
    ruler[1, 0, 0], ruler[1, 1, 0] = [0.0, 0.0, 1.0, 0.5], [math.log(3.0) / 8, 0.0, 5.0, 0.0]      # keys 0 and ln 3 / 8
    cache[..., D:] = ruler.view(np.uint8)
    cache[1, 0, 0, D // 2:D] = 0x31                      # values 1 + 0.5 and 1 + 1.5
    out, bound = bo.attend(np.ones((1, D), dtype=np.float16), cache, [1], 2, 2)
    # scores 0 and 64 ln(3) / 8 / 8 = ln 3 (fp16's): weights 1/4 and 3/4
    assert np.allclose(out[0, 0::2], 0.25 * 1.5 + 0.75 * 5.0, atol=2e-3) and np.allclose(out[0, 1::2], 0.25 * 2.5 + 0.75 * 5.0, atol=2e-3)
    assert 0 < bound[0, 0] < 1e-3
    assert np.array_equal(bo.attend(np.ones((1, D), dtype=np.float16), cache, [1], 0, 2)[0], np.zeros((1, D)))
