"""The serving step around the packed 4-bit cache, on the GPU (HIP, gfx950).

What a step needs next to the store and the attention of ``kernels.kv_dequant``:

    kv_step_metadata(...)            positions, slots and block tables from the requests' lengths
    kv_rotary(...)                   queries and keys turned by their positions
    kv_rotary_quantize_store(...)    the same, with the keys and values quantized into the packed cache
    kv_prompt_attention(...)         causal attention of packed prompts over their own K/V
    sample_tokens(...)               the next token of every row of logits

    rotary_frequencies(...)          a model's rotary settings as the frequencies that the rotary calls take

As in ``kernels.kv_dequant`` the device code is libslmturbo_hip.so, launches go to the current torch
stream, nothing waits for the device and there is no CPU path.  All of it can be captured in a HIP graph.
The calls compute results alone: they have no gradients, and refuse tensors that want them.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _native
from .kv_dequant import _current_device, _entry, _load_native_extension, _no_switch, _raw_stream, _require

__all__ = [
    "StepMetadata",
    "kv_step_metadata",
    "rotary_frequencies",
    "kv_rotary",
    "kv_rotary_quantize_store",
    "kv_prompt_attention",
    "sample_tokens",
]

_stream = _raw_stream or (lambda di: torch.cuda.current_stream(di).cuda_stream)


def _on(di):
    """Make GPU di current for the call (no switch when it already is)."""
    return _no_switch if di == _current_device() else torch.cuda.device(di)


_I32 = (1 << 31) - 1


def _refuse_sizes(phase, *sizes):
    """The library takes sizes as 32-bit numbers; called before any copy of what has them."""
    raise RuntimeError(f"{phase}: tensors must have fewer than 2^31 rows and columns, got {list(sizes)}")


_DTYPES = {torch.float32: _native.F32, torch.float16: _native.F16, torch.bfloat16: _native.BF16}
_ALL = tuple(_DTYPES)


def _no_grad(phase, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError(f"{phase}: no gradients; call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{phase}: no gradients; call it on tensors without tangents")


def _check(phase, name, t, di, dtypes, shape):
    """t is a tensor of GPU di with one of dtypes and the given shape.  (Calls of a few microseconds: each attribute is
    read once, and messages are made only when a check fails.)"""
    if t.get_device() != di or di < 0:
        raise RuntimeError(f"{phase}: {name} must be a CUDA tensor" + (f" on cuda:{di}" if di >= 0 else ""))
    if t.dtype not in dtypes:
        raise RuntimeError(f"{phase}: {name} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {str(t.dtype)[6:]}")
    if t.shape != shape:
        raise RuntimeError(f"{phase}: {name} must be {list(shape)}, got {list(t.shape)}")


def _check_out(phase, name, t, like):
    _no_grad(phase, t)
    _check(phase, name, t, like.get_device(), (like.dtype,), like.shape)
    if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())) or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise RuntimeError(f"{phase}: {name} must have unit stride over the last dim and no repeated elements")


# =============================================================================
#  step metadata
# =============================================================================
class StepMetadata(NamedTuple):
    """Where a step's tokens are (``kv_step_metadata``)."""

    query_start_loc: torch.Tensor   # [R + 1] int32
    seq_lens: torch.Tensor          # [R] int32, context and the step's tokens
    positions: torch.Tensor         # [N] int64
    slot_mapping: torch.Tensor      # [N] int64, -1 for padding
    free_end: torch.Tensor          # [1] int32, the next step's free_start


_INT = (torch.int32,)


def kv_step_metadata(query_lens, context_lens, block_tables, free_blocks, block_size, num_tokens, free_start=None,
                     out=None):
    """A step's positions, slots and block tables from its requests' lengths, in one launch.

        query_lens, context_lens  [R] int32 (device): the step's new tokens of each request (0 for none)
                                  and those that the cache holds
        block_tables  [R, max_blocks] int32 or int64, updated in place: the columns that the step opens
                      get the next free blocks, requests and columns in order
        free_blocks   [F], of the tables' type: the blocks to take
        num_tokens    N, the rows of the step's tensors; those behind the last request's token are padding
        free_start    optional [1] int32 (device): where in free_blocks to begin
        out           optional StepMetadata of the right shapes, written in place; its tensors must not
                      overlap the inputs (copy free_end and seq_lens to the next step's) or one another,
                      and nothing may overlap block_tables
    Returns a StepMetadata, in the form that kv_quantize_store, kv_dequant_chunk_paged,
    kv_dequant_decode_paged_batched and the rotary calls take.  A token for which its table row or the
    free list has no room gets the slot -1, which the store skips, and seq_lens counts the tokens before
    it; free_end > F says that the list was too short.  Tokens past num_tokens are no part of the step, and
    a context that is longer than its table row counts as a full row.
    """
    phase = "step metadata"
    R = query_lens.numel()
    dev, di = query_lens.device, query_lens.get_device()
    _check(phase, "query_lens", query_lens, di, _INT, (R,))
    _check(phase, "context_lens", context_lens, di, _INT, (R,))
    if block_tables.dim() != 2:
        raise RuntimeError(f"{phase}: block_tables must be [R, max_blocks], got {list(block_tables.shape)}")
    columns, F = block_tables.shape[1], free_blocks.numel()
    if R > _I32 or columns > _I32 or F > _I32:
        _refuse_sizes(phase, R, columns, F)
    _check(phase, "block_tables", block_tables, di, (torch.int32, torch.int64), (R, columns))
    row = block_tables.stride(0)
    if (columns > 1 and block_tables.stride(1) != 1) or (R > 1 and row < columns):
        raise RuntimeError(f"{phase}: block_tables must have unit stride over the columns and rows of their own")
    _check(phase, "free_blocks", free_blocks, di, (block_tables.dtype,), (F,))
    if free_start is not None:
        _check(phase, "free_start", free_start, di, _INT, (1,))
    block_size, N = int(block_size), int(num_tokens)
    if not (0 <= N <= _I32 and 0 < block_size <= _I32):
        raise RuntimeError(f"{phase}: num_tokens must be >= 0 and block_size positive, both below 2^31, got {N} and {block_size}")
    lib = _load_native_extension()
    with _on(di):
        if out is None:
            # (parts of one allocation: 1.1 us less of 10.5 for the call)
            starts, seq_lens, end = query_lens.new_empty(2 * R + 2).split_with_sizes((R + 1, R, 1))
            positions = torch.empty(N, dtype=torch.int64, device=dev)
            out = StepMetadata(starts, seq_lens, positions, torch.empty_like(positions), end)
        else:
            for name, t, dtype, n in zip(out._fields, out, (torch.int32, torch.int32, torch.int64, torch.int64, torch.int32),
                                         (R + 1, R, N, N, 1)):
                _check(phase, "out." + name, t, di, (dtype,), (n,))
                _require(t.is_contiguous(), f"{phase}: out.{name} must be contiguous")
        query_lens, context_lens, free_blocks = query_lens.contiguous(), context_lens.contiguous(), free_blocks.contiguous()
        rc = _entry(lib, "step_metadata")(
            query_lens.data_ptr(), context_lens.data_ptr(), R, block_tables.data_ptr(),
            64 if block_tables.dtype is torch.int64 else 32, row, columns, free_blocks.data_ptr(), F,
            0 if free_start is None else free_start.data_ptr(), block_size, N, out.query_start_loc.data_ptr(),
            out.seq_lens.data_ptr(), out.positions.data_ptr(), out.slot_mapping.data_ptr(), out.free_end.data_ptr(),
            _stream(di))
        if rc:
            _native.check(lib, rc)
    return out


# =============================================================================
#  rotary positions
# =============================================================================
def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, device=None):
    """(inv_freq [rotary_dim / 2] fp32, scale) of a model's rotary settings, for kv_rotary.

    scaling: None, or a dict as model configurations carry it, by its "rope_type" (older ones: "type"):
        "linear"  factor: positions divided by it
        "llama3"  factor, low_freq_factor, high_freq_factor, original_max_position_embeddings: wavelengths
                  past original / low are divided by factor, those below original / high kept, linear in
                  between
        "yarn"    factor, original_max_position_embeddings, beta_fast (32), beta_slow (1): dims that turn
                  more than beta_fast times over the original length are kept, those below beta_slow
                  divided by factor, a ramp over the dims in between; scale is attention_factor, or
                  0.1 ln(factor) + 1
    The sums are in fp64, and the frequencies are rounded to fp32 once.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    freq, scale = float(base) ** (-i / rotary_dim), 1.0
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "linear":
        freq = freq / float(scaling["factor"])
    elif kind == "llama3":
        factor, lo, hi = (float(scaling[k]) for k in ("factor", "low_freq_factor", "high_freq_factor"))
        turns = float(scaling["original_max_position_embeddings"]) * freq / (2 * math.pi)
        keep = ((turns - lo) / (hi - lo)).clamp(0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
    elif kind == "yarn":
        for name, usual in (("mscale", None), ("mscale_all_dim", None), ("truncate", True)):
            if scaling.get(name, usual) not in (None, usual):
                raise ValueError(f"yarn settings with {name} are not supported, got {scaling[name]!r}")
        factor, length = float(scaling["factor"]), float(scaling["original_max_position_embeddings"])
        dim_of = lambda turns: rotary_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo = max(math.floor(dim_of(float(scaling.get("beta_fast") or 32.0))), 0)
        hi = min(math.ceil(dim_of(float(scaling.get("beta_slow") or 1.0))), rotary_dim - 1)
        keep = 1.0 - ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
        given = scaling.get("attention_factor")
        scale = float(given) if given is not None else (0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0)
    elif kind != "default":
        raise ValueError(f"rope_type must be 'default', 'linear', 'llama3' or 'yarn', got {kind!r}")
    return freq.to(torch.float32).to(device), scale


def _like(t):
    """A new contiguous tensor of t's shape and type (a third faster than one of a shape)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _unit(t):
    """t with unit stride over its last dim."""
    return t if t.stride(-1) == 1 else t.contiguous()


def _check_positions(phase, positions, inv_freq, di, N):
    _check(phase, "positions", positions, di, (torch.int64, torch.int32), (N,))
    _check(phase, "inv_freq", inv_freq, di, (torch.float32,), (inv_freq.numel(),))
    return positions.contiguous(), inv_freq.contiguous(), 64 if positions.dtype is torch.int64 else 32


def kv_rotary(q, k, positions, inv_freq, interleaved=False, scale=1.0, out=None):
    """Queries and keys turned by their tokens' positions.  Returns (q, k) turned.

        q           [N, H, D], k [N, KV, D] or None: fp16, bf16 or fp32, D 64, 80 or 128
        positions   [N] int64 or int32 (device)
        inv_freq    [R / 2] fp32 (device), R <= D: the first R dims of a head turn, the others stay
        interleaved pairs are dims (2i, 2i + 1), otherwise (i, i + R / 2)
        scale       factor of cosine and sine (models scaled for long contexts have one)
        out         optional (q, k) to write into; they may be the inputs themselves, but must not
                    overlap them otherwise
    Angles are the exact products position * inv_freq, of up to 2^52, their cosines and sines are rounded
    to fp32 and the result once to the tensors' type.
    """
    phase = "rotary"
    assert q.dim() == 3, f"q must be [N, H, D], got {tuple(q.shape)}"
    N, H, D = q.shape
    assert D in (64, 80, 128), f"head_dim must be 64/80/128, got {D}"
    _no_grad(phase, q, inv_freq) if k is None else _no_grad(phase, q, k, inv_freq)
    dev, di = q.device, q.get_device()
    _check(phase, "q", q, di, _ALL, q.shape)
    KV = 0
    if k is not None:
        KV = k.shape[1] if k.dim() == 3 else 0
        _check(phase, "k", k, di, (q.dtype,), (N, KV, D))
    rot = 2 * inv_freq.numel()
    if N > _I32 or H > _I32 or KV > _I32 or rot > _I32:
        _refuse_sizes(phase, N, H, KV, rot)
    positions, inv_freq, bits = _check_positions(phase, positions, inv_freq, di, N)
    lib = _load_native_extension()
    with _on(di):
        if out is None:
            out = (_like(q), None if k is None else _like(k))
        else:
            qo, ko = out
            _check_out(phase, "out q", qo, q)
            _require((ko is None) == (k is None), f"{phase}: out must hold q and k like the inputs")
            if k is not None:
                _check_out(phase, "out k", ko, k)
        qo, ko = out
        q = _unit(q)
        qs, os = q.stride(), qo.stride()
        if k is None:
            keys, keys_out = (0, 0, 0), (0, 0, 0)
        else:
            k = _unit(k)
            keys, keys_out = (k.data_ptr(), *k.stride()[:2]), (ko.data_ptr(), *ko.stride()[:2])
        rc = _entry(lib, "rotary")(
            q.data_ptr(), qs[0], qs[1], *keys, qo.data_ptr(), os[0], os[1], *keys_out, N, H, KV, D, _DTYPES[q.dtype],
            positions.data_ptr(), bits, inv_freq.data_ptr(), rot, 1 if interleaved else 0, float(scale),
            _stream(di))
        if rc:
            _native.check(lib, rc)
    return out


def kv_rotary_quantize_store(q, key, value, kv_cache, slot_mapping, block_size, positions, inv_freq, interleaved=False,
                             scale=1.0, q_out=None, key_out=None):
    """kv_rotary of q and key, and kv_quantize_store of the turned key and the value, in one launch.  Returns q turned.

        q                 [N, H, D], key and value [N, KV, D]: fp16 (strides: any over tokens and heads)
        kv_cache          [num_blocks, block_size, KV, D+8] uint8, contiguous
        slot_mapping      [N] int64, no slot twice; those that are negative or past the cache are skipped
        positions ... scale   as in kv_rotary
        q_out             optional [N, H, D] to write into (it may be q)
        key_out           optional [N, KV, D] for the turned keys (it may be key); without it they go to
                          the cache alone
    The cache's bytes are those of the two calls.
    """
    phase = "rotary store"
    assert q.dim() == 3, f"q must be [N, H, D], got {tuple(q.shape)}"
    assert key.dim() == 3, f"key must be [N, KV, D], got {tuple(key.shape)}"
    assert kv_cache.is_contiguous(), "kv_cache must be contiguous"
    N, H, D = q.shape
    assert D in (64, 80, 128), f"head_dim must be 64/80/128, got {D}"
    KV = key.shape[1]
    dev, di = q.device, q.get_device()
    _no_grad(phase, q, key, value, inv_freq)
    half = (torch.float16,)
    _check(phase, "q", q, di, half, q.shape)
    _check(phase, "key", key, di, half, (N, KV, D))
    _check(phase, "value", value, di, half, (N, KV, D))
    if kv_cache.dim() != 4:
        raise RuntimeError(f"{phase}: kv_cache must be [num_blocks, {block_size}, {KV}, {D + 8}], got {list(kv_cache.shape)}")
    _check(phase, "kv_cache", kv_cache, di, (torch.uint8,), (kv_cache.shape[0], block_size, KV, D + 8))
    _check(phase, "slot_mapping", slot_mapping, di, (torch.int64,), (N,))
    rot = 2 * inv_freq.numel()
    if N > _I32 or H > _I32 or KV > _I32 or rot > _I32:
        _refuse_sizes(phase, N, H, KV, rot)
    positions, inv_freq, bits = _check_positions(phase, positions, inv_freq, di, N)
    lib = _load_native_extension()
    with _on(di):
        if q_out is None:
            q_out = _like(q)
        else:
            _check_out(phase, "q_out", q_out, q)
        if key_out is not None:
            _check_out(phase, "key_out", key_out, key)
        q, key, value, slot_mapping = _unit(q), _unit(key), _unit(value), slot_mapping.contiguous()
        qs, ks, vs, os = q.stride(), key.stride(), value.stride(), q_out.stride()
        keys_out = (0, 0, 0) if key_out is None else (key_out.data_ptr(), *key_out.stride()[:2])
        rc = _entry(lib, "rotary_quantize_store")(
            q.data_ptr(), qs[0], qs[1], key.data_ptr(), ks[0], ks[1], value.data_ptr(), vs[0], vs[1], q_out.data_ptr(),
            os[0], os[1], *keys_out, kv_cache.data_ptr(), kv_cache.shape[0], int(block_size), slot_mapping.data_ptr(),
            N, H, KV, D, positions.data_ptr(), bits, inv_freq.data_ptr(), rot, 1 if interleaved else 0,
            float(scale), _stream(di))
        if rc:
            _native.check(lib, rc)
    return q_out


# =============================================================================
#  attention of packed prompts
# =============================================================================
def _rows16(t):
    """t as the attention reads it: unit stride over D, rows 16-byte aligned and less than 2^28 elements apart."""
    s = t.stride()
    ok = s[2] == 1 and s[1] % 8 == 0 and s[0] % 8 == 0 and s[0] < 1 << 28 and t.data_ptr() % 16 == 0
    # (contiguous() would return t itself where only its address, or the stride of a dim of one element, is odd)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def kv_prompt_attention(q, k, v, query_start_loc, key_start_loc=None, causal=True, scale=None, out=None):
    """Attention of packed prompts over their own K/V.  Returns [N, H, D] of q's type.

        q                [N, H, D], k and v [M, KV, D]: fp16 or bf16, D 64, 80 or 128 (strides: any, with
                         unit stride over D); query head h reads KV head h // (H // KV)
        query_start_loc  [R + 1] int32 (device): sequence r has the rows from its entry r to the next
        key_start_loc    optional [R + 1] int32: the sequences' rows of k and v, where they are not those of q
        causal           the last row of a sequence sees all its keys, each one before it one key less
        scale            of the scores, positive (1 / sqrt(D))
        out              optional tensor like q, written in place; it may be q itself, and must not overlap q otherwise,
                         k or v
    Rows that see no key are zeros; those of no sequence keep what ``out`` held there (a new one holds zeros).
    """
    phase = "prompt attention"
    assert q.dim() == 3, f"q must be [N, H, D], got {tuple(q.shape)}"
    assert k.dim() == 3, f"k must be [M, KV, D], got {tuple(k.shape)}"
    N, H, D = q.shape
    M, KV, _ = k.shape
    assert D in (64, 80, 128), f"head_dim must be 64/80/128, got {D}"
    assert KV > 0 and H % KV == 0, f"H {H} not divisible by the KV heads {KV}"
    dev, di, dtype = q.device, q.get_device(), q.dtype
    _no_grad(phase, q, k, v)
    _check(phase, "q", q, di, (torch.float16, torch.bfloat16), q.shape)
    _check(phase, "k", k, di, (dtype,), (M, KV, D))
    _check(phase, "v", v, di, (dtype,), (M, KV, D))
    R = query_start_loc.numel() - 1
    _require(R >= 0, f"{phase}: query_start_loc must hold at least one entry")
    if N > _I32 or M > _I32 or R > _I32 or H > _I32:
        _refuse_sizes(phase, N, M, R, H)
    _check(phase, "query_start_loc", query_start_loc, di, _INT, (R + 1,))
    if key_start_loc is None:
        _require(M == N, f"{phase}: k and v must have q's {N} rows without a key_start_loc, got {M}")
    else:
        _check(phase, "key_start_loc", key_start_loc, di, _INT, (R + 1,))
        key_start_loc = key_start_loc.contiguous()
    lib = _load_native_extension()
    with _on(di):
        clear = out is None
        if clear:
            out = _like(q) if R else torch.zeros((N, H, D), dtype=dtype, device=dev)
        else:
            _check_out(phase, "out", out, q)
        os = out.stride()
        if not clear:                        # (the strides of a dim of one element are of no account)
            os = (os[0] if N > 1 else 0, os[1] if H > 1 else 0)
            _require(os[0] % 4 == 0 and os[1] % 4 == 0 and out.data_ptr() % 8 == 0, f"{phase}: out's rows must be 8-byte aligned")
        q, k, v, query_start_loc = _rows16(q), _rows16(k), _rows16(v), query_start_loc.contiguous()
        qs, ks, vs = q.stride(), k.stride(), v.stride()
        # (only few rows with many keys need one; of this call alone, in stream order like any tensor)
        need = _entry(lib, "prompt_workspace_bytes")(N, M, R, H, D) if M >= 1024 * R else 0
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
        rc = _entry(lib, "prompt_attention")(
            q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], query_start_loc.data_ptr(),
            0 if key_start_loc is None else key_start_loc.data_ptr(), R, N, M, H, KV, D, _DTYPES[dtype],
            1 if causal else 0, D ** -0.5 if scale is None else float(scale), out.data_ptr(), os[0], os[1], 1 if clear else 0,
            0 if ws is None else ws.data_ptr(), need, _stream(di))
        if rc:
            _native.check(lib, rc)
    return out


# =============================================================================
#  sampling
# =============================================================================
def _per_row(name, value, di, dtype, B):
    """(pointer, single value) of a sampling argument: a number for all rows or a tensor of one a row."""
    if isinstance(value, torch.Tensor):
        _no_grad("sample", value)
        _check("sample", name, value, di, (dtype,), (B,))
        return value.contiguous()
    return None


def sample_tokens(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_probs=False, out=None):
    """The next token of every row of logits, from given random numbers.  Returns [B] int64.

        logits       [B, V] fp16, bf16 or fp32 (rows may be strided); NaN counts as -infinity
        uniforms     [B] fp32 (device), each from [0, 1)
        temperature, top_k, top_p, min_p   a number for all rows, or a tensor [B] (fp32; top_k int32)
        out          optional [B] int64, written in place
    In the order largest logit first, equal ones by index, the tokens kept are those among the first top_k
    (0: all) before which less than top_p of these k's probability lies and whose probability is at least
    min_p times the largest; the first is kept in any case.  The answer is the first token, by index, at
    which the running probability of the kept ones passes the row's uniform.  temperature 0 takes the
    largest logit, the lowest index among equals.  The same inputs give the same tokens.
    With return_probs also the tokens' probabilities among the kept ones, [B] fp32.  A row that leaves
    nothing (every logit -infinity) gives token 0 with probability 0.
    """
    phase = "sample"
    assert logits.dim() == 2, f"logits must be [B, V], got {tuple(logits.shape)}"
    B, V = logits.shape
    dev, di = logits.device, logits.get_device()
    _no_grad(phase, logits)
    _check(phase, "logits", logits, di, _ALL, logits.shape)
    _check(phase, "uniforms", uniforms, di, (torch.float32,), (B,))
    if B > _I32 or V > _I32:
        _refuse_sizes(phase, B, V)
    t, k, p, m = (_per_row(name, value, di, dtype, B) for name, value, dtype in (
        ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
        ("min_p", min_p, torch.float32)))
    lib = _load_native_extension()
    with _on(di):
        if out is None:
            out = torch.empty(B, dtype=torch.int64, device=dev)
        else:
            _check(phase, "out", out, di, (torch.int64,), (B,))
            _require(out.is_contiguous(), f"{phase}: out must be contiguous")
        probs = torch.empty_like(uniforms, memory_format=torch.contiguous_format) if return_probs else None
        need = _entry(lib, "sample_workspace_bytes")(B, V)
        if need < 0:
            raise RuntimeError(_native.last_error(lib))
        if logits.stride(1) != 1:
            logits = logits.contiguous()
        uniforms = uniforms.contiguous()
        # (of this call alone, in stream order like any tensor, so that graphs share none)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        at = lambda x: 0 if x is None else x.data_ptr()  # noqa: E731
        rc = _entry(lib, "sample_tokens")(
            logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), B, V, uniforms.data_ptr(),
            at(t), 1.0 if t is not None else float(temperature), at(k), 0 if k is not None else max(min(int(top_k), V), -1),
            at(p), 1.0 if p is not None else float(top_p), at(m), 0.0 if m is not None else float(min_p),
            out.data_ptr(), at(probs), at(ws), need, _stream(di))
        if rc:
            _native.check(lib, rc)
    return (out, probs) if return_probs else out
