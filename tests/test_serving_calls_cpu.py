"""Without a GPU: what the serving step's calls (kernels.serving) make of arguments off the usual ones, and what they refuse,
through the Python functions, the C ABI and the METH_FASTCALL binding."""
import re
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

from kernels import _native, serving


@pytest.fixture(scope="module")
def lib():
    if not _native.library_path().exists():
        pytest.fail(f"{_native.library_path()} is not built: run `python slm-turbo_amd/build_lib.py`")
    return _native.load()


def _both(lib, name, args):
    """(status, message) of a call that is refused, the same from ctypes and from the METH_FASTCALL binding."""
    status = getattr(lib, "slmt_" + name)(*args)
    message = _native.last_error(lib)
    assert getattr(_native.fast(), name)(*[0 if a is None else a for a in args]) == status
    assert _native.last_error(lib) == message
    return status, message


# =============================================================================
#  step metadata
# =============================================================================
def _metadata(**kw):
    """Arguments that do not overlap: two requests, tables of 8 columns in rows of 10, at 4096 bytes' distance each."""
    names = "q c R bt bits row columns free F fs bs N qsl sl pos slots fe stream".split()
    at = {n: 4096 * (i + 1) for i, n in enumerate("q c bt free fs qsl sl pos slots fe".split())}
    args = {**at, "R": 2, "bits": 32, "row": 10, "columns": 8, "F": 4, "bs": 16, "N": 5, "stream": None, **kw}
    return [args[n] for n in names]


@pytest.mark.parametrize("bits", [32, 64])
def test_metadata_refuses_what_overlaps(lib, bits):
    """(A call that passes the checks would launch; a refused one never does.  What does not overlap is shown by the refusal
    that it gets further on.)"""
    size, bt, row = bits // 8, 3 * 4096, 10 * bits // 8
    tables = [(name, at) for name in ("q", "c", "free", "fs", "sl", "qsl", "pos", "slots", "fe")
              for at in (bt, bt + 8 * size - 4, bt + row, bt + row + 8 * size - 4)]
    for name, at in tables:
        status, message = _both(lib, "step_metadata", _metadata(bits=bits, **{name: at}))
        assert status == _native.ERR_INVALID and message.endswith("overlaps the block tables"), (name, at, message)
    for name, ahead in (("q", 8), ("free", 4 * size), ("fs", 4), ("qsl", 12), ("sl", 8), ("pos", 40), ("slots", 40), ("fe", 4)):
        status, message = _both(lib, "step_metadata", _metadata(bits=bits, **{name: bt - ahead + 1}))
        assert message.endswith("overlaps the block tables"), (name, message)
    # ahead of them, in the gap between the rows, and behind the last row: the outputs that overlap are what is refused
    for name, at in (("sl", bt - 8), ("fe", bt + 8 * size), ("fe", bt + 9 * size), ("q", bt + 8 * size), ("sl", bt + row + 8 * size)):
        status, message = _both(lib, "step_metadata", _metadata(bits=bits, **{name: at, "slots": 8 * 4096}))
        assert status == _native.ERR_INVALID and message == "step metadata: outputs overlap", (name, message)
    for a, b, distance in (("qsl", "sl", 11), ("sl", "qsl", 7), ("pos", "slots", 39), ("slots", "pos", 39), ("fe", "pos", 3), ("qsl", "fe", 0)):
        at = 50 * 4096
        status, message = _both(lib, "step_metadata", _metadata(bits=bits, **{a: at, b: at + distance}))
        assert message == "step metadata: outputs overlap", (a, b)
    status, message = _both(lib, "step_metadata", _metadata(bits=bits, sl=4096))
    assert message == "step metadata: an output overlaps an input"


# =============================================================================
#  prompt attention
# =============================================================================
def test_rows_that_the_attention_cannot_read_are_copied():
    """Also those that torch calls contiguous: an odd address, an odd stride of a dim of one element."""
    flat = torch.arange(9000, dtype=torch.float32).half()
    for t in (flat[1:1 + 20 * 3 * 64].view(20, 3, 64), flat.as_strided((1, 3, 64), (195, 64, 1)), flat.as_strided((20, 1, 64), (64, 67, 1)),
              flat.as_strided((1, 1, 80), (3, 5, 1)), flat.as_strided((5, 2, 64), (128, 64, 1), 4), flat.as_strided((1, 2, 64), (1 << 29, 64, 1)),
              flat.as_strided((5, 2, 64), (130, 65, 1)), flat.as_strided((5, 2, 64), (128, 1, 2))):
        got = serving._rows16(t)
        assert torch.equal(got, t) and got.data_ptr() % 16 == 0
        assert got.stride() == (t.shape[1] * t.shape[2], t.shape[2], 1)
    for t in (flat[8:8 + 20 * 2 * 64].view(20, 2, 64), flat.as_strided((5, 2, 64), (256, 64, 1)), flat.as_strided((2, 5, 64), (64, 128, 1))):
        assert serving._rows16(t) is t


def test_attention_refuses_scales_that_fp32_has_not(lib):
    """(The others' refusal is that of v's stride.)"""
    for scale, refused in ((1e-300, True), (5e-46, True), (1e-39, True), (1e-38, False), (0.125, False), (1e38, False), (3e38, True)):
        args = [1 << 24, 512, 64, 1 << 25, 128, 64, 1 << 40, 1 << 28, 64, 16, None, 1, 3, 3, 8, 2, 64, 1, 1, scale, 1 << 26, 512, 64, 0, None, 0, None]
        status, message = _both(lib, "prompt_attention", args)
        assert status == (_native.ERR_INVALID if refused else _native.ERR_UNSUPPORTED)
        assert ("scale must be positive" if refused else "below 2^28") in message


def _layout(rng, rows, heads, D):
    """(token stride, head stride) of rows that do not overlap: tokens outside or heads outside, with gaps or without."""
    gap = lambda: 8 * rng.choice([0, 0, 1, 5, 40])  # noqa: E731
    if rng.random() < 0.7:
        head = D + rng.choice([0, gap()])
        return heads * head + gap(), head
    token = D + gap()
    return token, rows * token + gap()


def _elements(base, rows, heads, D, token, head):
    at = base // 2 + torch.arange(rows)[:, None, None] * token + torch.arange(heads)[:, None] * head + torch.arange(D)
    return set(at.flatten().tolist())


def test_attention_refuses_outputs_that_overlap(lib):
    """out against k and against q, over many layouts, with the sets of their elements.  (v lies far off, with a stride that is
    refused in turn: no call of these launches.)"""
    import random

    rng, D, seen = random.Random(5), 64, {}
    for _ in range(1500):
        which = rng.choice("kkq")
        N, M, KV = rng.randint(1, 5), rng.randint(1, 6), rng.choice([1, 2, 3])
        H = KV * rng.choice([1, 2])
        rows, heads = (M, KV) if which == "k" else (N, H)
        ot, oh = _layout(rng, N, H, D)
        xt, xh = (ot, oh) if which == "q" and rng.random() < 0.4 else _layout(rng, rows, heads, D)
        if rng.random() < 0.4:                                       # parts of one buffer
            ot = xt = max(ot, xt)
        base = 1 << 20
        out = base + 16 * rng.choice([0, rng.randint(-300, 300), rng.randint(-10, 10), D // 8 * rng.randint(-8, 8)])
        far = dict(q=1 << 24, k=1 << 25)
        q, k = (far["q"], base) if which == "k" else (base, far["k"])
        qt, qh, kt, kh = (H * D, D, xt, xh) if which == "k" else (xt, xh, KV * D, D)
        args = [q, qt, qh, k, kt, kh, 1 << 40, 1 << 28, D, 16, None, 1, N, M, H, KV, D, 1, 1, 0.125, out, ot, oh, 0, None, 0, None]
        status, message = _both(lib, "prompt_attention", args)
        x, o = _elements(base, rows, heads, D, xt, xh), _elements(out, N, H, D, ot, oh)
        itself = which == "q" and out == base and (N == 1 or ot == xt) and (H == 1 or oh == xh)
        shares = bool(x & o) and not itself
        exact = len(x) == max(x) - min(x) + 1 or len(o) == max(o) - min(o) + 1 or N == 1 or rows == 1 or ot == xt
        refused = status == _native.ERR_INVALID
        if refused:
            assert ("must not be k or v" in message or "overlaps k or v" in message) if which == "k" else "must be q itself" in message
        else:
            assert status == _native.ERR_UNSUPPORTED and "below 2^28" in message
        assert refused <= shares and (not exact or refused == shares), (which, N, M, H, KV, (ot, oh), (xt, xh), out - base, message)
        seen[which, shares, refused] = seen.get((which, shares, refused), 0) + 1
    assert all(seen.get((w, s, s), 0) > 50 for w in "kq" for s in (False, True)), seen


# =============================================================================
#  launches
# =============================================================================
def test_more_rows_than_a_launch_holds_are_refused(lib):
    """2^32 threads, before any HIP call."""
    ws = lib.slmt_sample_workspace_bytes(1 << 23, 40_000)
    assert ws > 0
    rotary = [16, 512, 64, None, 0, 0, 16, 512, 64, None, 0, 0, 1 << 24, 32, 0, 64, 1, 16, 64, 16, 64, 0, 1.0, None]
    few = [16, 64, 64, None, 0, 0, 16, 64, 64, None, 0, 0, (1 << 27) + 1, 1, 0, 64, 1, 16, 64, 16, 64, 0, 1.0, None]
    sample = lambda B, V, w, n: [16, 0, V, B, V, 16, None, 1.0, None, 0, None, 1.0, None, 0.0, 16, None, w, n, None]  # noqa: E731
    prompt = [1 << 24, 512, 64, 1 << 25, 128, 64, 1 << 26, 128, 64, 16, None, 1 << 22, 3, 3, 8, 2, 64, 1, 1, 0.125, 1 << 28, 512, 64, 0, None, 0, None]
    for name, args in (("rotary", rotary), ("rotary", few), ("sample_tokens", sample(1 << 22, 100, None, 0)),
                       ("sample_tokens", sample(1 << 23, 40_000, 16, ws)), ("prompt_attention", prompt)):
        status, message = _both(lib, name, args)
        assert status == _native.ERR_UNSUPPORTED and "too many rows for a launch" in message, (name, message)


# =============================================================================
#  gradients
# =============================================================================
def _asks(call, *args):
    """The call with one argument after another that wants a gradient, or that has a tangent."""
    for i, a in enumerate(args):
        if not a.is_floating_point():
            continue
        with pytest.raises(RuntimeError, match="no gradients"):
            call(*args[:i], a.clone().requires_grad_(), *args[i + 1:])
        with torch.no_grad(), forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="no gradients"):
                call(*args[:i], forward_ad.make_dual(a, torch.ones_like(a)), *args[i + 1:])


def test_python_calls_refuse_tensors_that_want_gradients():
    half = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    q, k, pos, inv = half(3, 4, 64), half(3, 2, 64), torch.zeros(3, dtype=torch.int64), torch.ones(32)
    cache, start = torch.zeros((2, 16, 2, 72), dtype=torch.uint8), torch.zeros(2, dtype=torch.int32)
    _asks(serving.kv_rotary, q, k, pos, inv)
    _asks(lambda a, f: serving.kv_rotary(a, None, pos, f), q, inv)
    _asks(lambda a, b, c, f: serving.kv_rotary_quantize_store(a, b, c, cache, pos, 16, pos, f), q, k, k, inv)
    _asks(lambda a, b, c: serving.kv_prompt_attention(a, b, c, start), q, k, k)
    _asks(lambda x: serving.sample_tokens(x, torch.zeros(2)), torch.zeros(2, 5))
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="must be a CUDA tensor"):      # (none of them has a tangent)
        serving.kv_rotary(q, k, pos, inv)


# =============================================================================
#  the sources
# =============================================================================
def test_inline_assembly_names_what_it_changes():
    """Every asm statement that writes m0 lists it (and memory, where it loads to LDS): the compiler may hold a value there."""
    csrc, seen = Path(serving.__file__).resolve().parents[1] / "csrc", 0
    for path in sorted([*csrc.glob("*.hip"), *csrc.glob("*.h")]):
        for statement in re.findall(r"\basm\b[^;]*?;", path.read_text()):
            if re.search(r"\bs_mov_b32 m0\b", statement):
                seen += 1
                outputs = statement.rsplit(":", 1)[1]
                assert '"m0"' in outputs and '"memory"' in outputs, f"{path.name}: {statement}"
    assert seen >= 4
