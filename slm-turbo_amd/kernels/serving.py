"""The serving step around the packed 4-bit cache, on the GPU (HIP, gfx950).

What a step needs next to the store and the attention of ``kernels.kv_dequant``:

    kv_step_metadata(...)            positions, slots and block tables from the requests' lengths
    kv_rotary(...)                   queries and keys turned by their positions
    kv_rotary_quantize_store(...)    the same, with the keys and values quantized into the packed cache
    kv_prompt_attention(...)         causal attention of packed prompts over their own K/V
    sample_tokens(...)               the next token of every row of logits
    beam_select(...)                 the best continuations of every request's beams
    kv_reorder_beams(...)            the beams' block tables and filling blocks after the selection

    rotary_frequencies(...)          a model's rotary settings as the frequencies that the rotary calls take

As in ``kernels.kv_dequant`` the device code is libslmturbo_hip.so, launches go to the current torch
stream, nothing waits for the device and there is no CPU path.  All of it can be captured in a HIP graph.
The calls compute results alone: they have no gradients, and refuse tensors that want them.
"""
from __future__ import annotations

import array
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _native
from .kv_dequant import (_I32, _check, _current_device, _entry, _load_native_extension, _no_grad, _no_switch, _raw_stream,
                         _refuse_sizes, _require)

__all__ = [
    "StepMetadata",
    "kv_step_metadata",
    "rotary_frequencies",
    "kv_rotary",
    "kv_rotary_quantize_store",
    "kv_prompt_attention",
    "sample_tokens",
    "BeamCandidates",
    "beam_select",
    "kv_reorder_beams",
]

_stream = _raw_stream or (lambda di: torch.cuda.current_stream(di).cuda_stream)


def _on(di):
    """Make GPU di current for the call (no switch when it already is)."""
    return _no_switch if di == _current_device() else torch.cuda.device(di)


_DTYPES = {torch.float32: _native.F32, torch.float16: _native.F16, torch.bfloat16: _native.BF16}
_ALL = tuple(_DTYPES)


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


# =============================================================================
#  beam search
# =============================================================================
class BeamCandidates(NamedTuple):
    """Continuations of beams (``beam_select``), [R, K] each."""

    tokens: torch.Tensor                 # int64
    parents: torch.Tensor                # int32, the beam that each continues
    scores: torch.Tensor                 # fp32, the sum of its tokens' log probabilities
    finished: Optional[torch.Tensor]     # bool
    lengths: Optional[torch.Tensor]      # int32


def beam_select(logits, scores, num_candidates=None, finished=None, lengths=None, length_penalty=0.0, eos_token=None,
                pad_token=0, keep_rows=False):
    """The best continuations of every request, over its beams and the vocabulary.  Returns BeamCandidates.

        logits          [R * W, V] fp16, bf16 or fp32 (rows may be strided), the beams of a request behind one another;
                        NaN counts as -infinity
        scores          [R, W] fp32: the beams' sums of log probabilities; a beam of -infinity has no continuations
        num_candidates  K, results a request (W); up to 64, as W
        finished        optional [R, W] bool: beams that have ended; such a beam has one continuation, pad_token, with
                        its score and length as they are
        lengths         optional [R, W] int32, the beams' tokens
        length_penalty  results are ranked by score / length^length_penalty, the length with the new token (at least 1)
        eos_token       the token that ends a beam
        keep_rows       False: results in the order of their ranks.  True (K = W): the first continuation of a beam
                        has that beam's place among the results, the others have those left, in order, so that
                        kv_reorder_beams moves as little as it can
    Largest rank first, equal ones by beam, logit and token; the ranks are in 64 bits, a row's sum of exponentials right to
    5e-11 of it and the same for equal rows, the scores rounded once.  Results that no continuation is left for have token 0,
    parent 0 and the score -infinity; their ``finished`` and ``lengths`` are those of token 0 behind beam 0.  ``finished`` of
    the results (a finished parent, or eos_token) is None without ``finished`` and eos_token, ``lengths`` without ``lengths``.
    """
    phase = "beam select"
    assert logits.dim() == 2, f"logits must be [R * W, V], got {tuple(logits.shape)}"
    assert scores.dim() == 2, f"scores must be [R, W], got {tuple(scores.shape)}"
    shape = scores.shape
    R, W = shape
    N, V = logits.shape
    K = W if num_candidates is None else int(num_candidates)
    # (Once a step: what fails here is looked at again for its message.)
    di, dtype = logits.get_device(), _DTYPES.get(logits.dtype)
    if logits.requires_grad or scores.requires_grad or forward_ad._current_level >= 0:
        _no_grad(phase, logits, scores)
    if dtype is None or N != R * W or di < 0:
        _check(phase, "logits", logits, di, _ALL, (R * W, V))
    if scores.dtype is not torch.float32 or scores.get_device() != di:
        _check(phase, "scores", scores, di, (torch.float32,), shape)
    if N > _I32 or V > _I32 or not 0 < K <= _I32:
        _refuse_sizes(phase, N, V, K)
    if finished is not None:
        if finished.dtype is not torch.bool or finished.shape != shape or finished.get_device() != di:
            _check(phase, "finished", finished, di, (torch.bool,), shape)
        finished = finished.contiguous()
    if lengths is not None:
        if lengths.dtype is not torch.int32 or lengths.shape != shape or lengths.get_device() != di:
            _check(phase, "lengths", lengths, di, _INT, shape)
        lengths = lengths.contiguous()
    eos, pad = -1 if eos_token is None else int(eos_token), int(pad_token)
    if not (-1 <= eos < V and 0 <= pad < V):
        raise RuntimeError(f"{phase}: eos_token and pad_token must be tokens, got {eos_token} and {pad_token}")
    lib = _load_native_extension()
    with _on(di):
        need = _entry(lib, "beam_workspace_bytes")(R, W, V, K)
        if need < 0:
            raise RuntimeError(_native.last_error(lib))
        ls = logits.stride()
        if ls[1] != 1:
            logits = logits.contiguous()
            ls = logits.stride()
        scores = scores.contiguous()
        like = scores if K == W else scores.new_empty((R, K))
        tokens, parents, best = torch.empty_like(like, dtype=torch.int64), torch.empty_like(like, dtype=torch.int32), torch.empty_like(like)
        ended = None if finished is None and eos_token is None else torch.empty_like(like, dtype=torch.bool)
        grown = None if lengths is None else torch.empty_like(parents)
        # (of this call alone, in stream order like any tensor, so that graphs share none)
        ws = scores.new_empty(need + 3 >> 2)
        rc = _entry(lib, "beam_select")(
            logits.data_ptr(), dtype, ls[0], R, W, V, scores.data_ptr(), 0 if finished is None else finished.data_ptr(),
            0 if lengths is None else lengths.data_ptr(), float(length_penalty), eos, pad, K, 1 if keep_rows else 0,
            tokens.data_ptr(), parents.data_ptr(), best.data_ptr(), 0 if ended is None else ended.data_ptr(),
            0 if grown is None else grown.data_ptr(), ws.data_ptr(), need, _stream(di))
        if rc:
            _native.check(lib, rc)
    return BeamCandidates(tokens, parents, best, ended, grown)


def kv_reorder_beams(kv_caches, block_tables, seq_lens, parents, block_size):
    """The beams' rows after a selection, in place: row r * W + j becomes what row r * W + parents[r, j] was.

        kv_caches     the layers' caches, uint8, contiguous: [num_blocks, block_size, KV, D+8] each, in a list or tuple, or
                      one tensor of them, with a leading dim of layers or (one layer) without; no cache twice
        block_tables  [R * W, max_blocks] int32 or int64 (device), updated in place
        seq_lens      [R] int32 (device): the cached tokens of each of a request's beams
        parents       [R, W] int32 (device), any of 0 .. W - 1, up to 64; others leave their row as it is
    Entries of full blocks are copied, so that beams share them.  In the block that is still filling (column seq_len //
    block_size) every row keeps its own, which must not be another's of the request, and its tokens are copied in all
    layers.  Blocks outside the cache are not copied.
    """
    phase = "reorder beams"
    assert parents.dim() == 2, f"parents must be [R, W], got {tuple(parents.shape)}"
    R, W = parents.shape
    di = block_tables.get_device()
    step = 0
    if isinstance(kv_caches, torch.Tensor):
        caches = (kv_caches,)
        one = shape = kv_caches.shape
        if len(one) == 5:
            shape = one[1:]
            step = kv_caches.stride(0)
    else:
        caches = tuple(kv_caches)
        one = shape = caches[0].shape if caches else (0, block_size, 1, 72)    # (none: the tables alone)
    if len(shape) != 4 or shape[1] != block_size:
        raise RuntimeError(f"{phase}: kv_caches must be [num_blocks, {block_size}, KV, D + 8], got {list(shape)}")
    blocks, _, KV, slot = shape
    for t in caches:
        if t.get_device() != di or t.dtype is not torch.uint8 or t.shape != one or not t.is_contiguous():
            _check(phase, "kv_caches", t, di, (torch.uint8,), one)
            raise RuntimeError(f"{phase}: kv_caches must be contiguous")
    if block_tables.dim() != 2:
        raise RuntimeError(f"{phase}: block_tables must be [R * W, max_blocks], got {list(block_tables.shape)}")
    rows, columns = block_tables.shape
    row, unit = block_tables.stride()
    wide = block_tables.dtype is torch.int64
    if not (wide or block_tables.dtype is torch.int32) or rows != R * W or di < 0:
        _check(phase, "block_tables", block_tables, di, (torch.int32, torch.int64), (R * W, columns))
    if (columns > 1 and unit != 1) or (rows > 1 and row < columns):
        raise RuntimeError(f"{phase}: block_tables must have unit stride over the columns and rows of their own")
    if seq_lens.dtype is not torch.int32 or seq_lens.shape != (R,) or seq_lens.get_device() != di:
        _check(phase, "seq_lens", seq_lens, di, _INT, (R,))
    if parents.dtype is not torch.int32 or parents.get_device() != di:
        _check(phase, "parents", parents, di, _INT, (R, W))
    if rows > _I32 or columns > _I32 or KV > _I32 or slot > _I32:
        _refuse_sizes(phase, rows, columns, *shape)
    lib = _load_native_extension()
    with _on(di):
        pointers = array.array("Q", [t.data_ptr() for t in caches])
        seq_lens, parents = seq_lens.contiguous(), parents.contiguous()
        rc = _entry(lib, "reorder_beams")(
            pointers.buffer_info()[0], one[0] if len(one) == 5 else len(caches), step, blocks, int(block_size), KV, slot - 8,
            block_tables.data_ptr(), 64 if wide else 32, max(row, columns), columns, seq_lens.data_ptr(), parents.data_ptr(),
            R, W, _stream(di))
        if rc:
            _native.check(lib, rc)
