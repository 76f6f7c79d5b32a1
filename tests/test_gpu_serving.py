"""GPU: the serving step's operators (kernels.serving) against plain restatements in 64 bits, at the sizes,
strides and masks where they can go wrong, alone and together."""
import math

import numpy as np
import pytest
import torch

import serving_oracle as so

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _sv():
    from kernels import serving

    return serving


def _kd():
    from kernels import kv_dequant

    return kv_dequant


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


# =============================================================================
#  step metadata
# =============================================================================
def _metadata_case(R, most, cached, block, seed, idle=0.2):
    g = _gen(seed)
    q = [0 if float(torch.rand(1, generator=g)) < idle else int(torch.randint(1, most + 1, (1,), generator=g)) for _ in range(R)]
    c = torch.randint(0, cached + 1, (R,), generator=g).tolist()
    columns = max([-(-(a + b) // block) for a, b in zip(q, c)] + [1])
    held = [-(-b // block) for b in c]
    need = sum(-(-(a + b) // block) - h for a, b, h in zip(q, c, held))
    blocks = torch.randperm(sum(held) + need + 5, generator=g).tolist()
    tables, at = [], 0
    for h in held:
        tables.append(blocks[at:at + h] + [-7] * (columns - h))
        at += h
    return q, c, tables, blocks[at:]


def _check_metadata(q, c, tables, free, block, N, dtype=torch.int32, free_start=None, columns=None):
    want = so.step_metadata(q, c, tables, free, block, N, free_start or 0)
    columns = len(tables[0]) if tables else columns or 0
    wide = torch.full((len(q), columns + 3), -9, dtype=dtype)          # (rows longer than what they hold)
    for r, row in enumerate(tables):
        wide[r, :columns] = torch.tensor(row, dtype=dtype)
    wide = wide.to(DEV)
    start = None if free_start is None else _int([free_start])
    m = _sv().kv_step_metadata(_int(q), _int(c), wide[:, :columns], _int(free, dtype), block, N, free_start=start)
    got = (wide[:, :columns].tolist(), *(t.tolist() for t in m[:4]), int(m.free_end))
    for name, a, b in zip(("tables", "query_start_loc", "seq_lens", "positions", "slots", "free_end"), got, want):
        assert a == b, name
    assert wide[:, columns:].eq(-9).all()
    assert [t.dtype for t in m] == [torch.int32, torch.int32, torch.int64, torch.int64, torch.int32]
    return m


@pytest.mark.parametrize("R,most,cached,block,pad,dtype", [
    (1, 1, 0, 16, 0, torch.int32), (1, 1, 40, 16, 3, torch.int64), (3, 70, 100, 16, 1, torch.int32),
    (64, 1, 5000, 16, 0, torch.int32), (255, 9, 50, 1, 7, torch.int64), (256, 20, 300, 24, 0, torch.int32),
    (257, 30, 0, 32, 11, torch.int32), (700, 12, 64, 16, 0, torch.int64), (5, 3000, 100, 64, 100, torch.int32)])
def test_metadata_matches_the_token_by_token_walk(R, most, cached, block, pad, dtype):
    q, c, tables, free = _metadata_case(R, most, cached, block, seed=R + most)
    _check_metadata(q, c, tables, free, block, sum(q) + pad, dtype)


def test_metadata_without_requests_or_tokens():
    m = _check_metadata([], [], [], [3, 4], 16, 5)
    assert m.slot_mapping.tolist() == [-1] * 5 and m.query_start_loc.tolist() == [0]
    _check_metadata([0, 0], [5, 0], [[8], [9]], [1], 16, 0)
    _check_metadata([4, 2], [5, 0], [[8], [9]], [1], 16, 0)           # no token fits the step


@pytest.mark.parametrize("drop", [1, 2, 40, 10_000])
def test_metadata_with_too_few_free_blocks(drop):
    """Tokens without a block have no slot, seq_lens counts those before them, free_end tells."""
    q, c, tables, free = _metadata_case(40, 60, 100, 16, seed=9)
    free = free[:-5]                                   # exactly what the step needs
    m = _check_metadata(q, c, tables, free[:max(len(free) - drop, 0)], 16, sum(q))
    assert int(m.free_end) == len(free)
    assert (m.slot_mapping < 0).any()


def test_metadata_cuts():
    """Full rows, contexts past the row, a step with fewer rows than tokens, negative lengths, an offset."""
    free = list(range(100, 140))
    _check_metadata([40, 5], [0, 3], [[-7, -7], [1, -7]], free, 16, 45)
    _check_metadata([4, 5], [1000, 3], [[5, 6], [1, -7]], free, 16, 9)
    _check_metadata([30, 30, 30], [0, 5, 0], [[-7] * 4, [1, -7, -7, -7], [-7] * 4], free, 16, 47)
    _check_metadata([-3, 5, -1], [4, -2, 7], [[1], [-7], [2]], free, 16, 8)
    _check_metadata([20, 3], [0, 16], [[-7, -7], [1, -7]], free, 16, 23, free_start=7)
    _check_metadata([20, 3], [0, 16], [[-7, -7], [1, -7]], free, 16, 23, free_start=1000)


def test_metadata_steps_in_a_graph():
    """Steps chained by free_end, replayed with the lengths rewritten in place."""
    sv = _sv()
    R, block = 9, 16
    ctx, q = torch.zeros(R, dtype=torch.int32, device=DEV), torch.ones(R, dtype=torch.int32, device=DEV)
    tables = torch.full((R, 8), -7, dtype=torch.int32, device=DEV)
    free, at = _int(list(range(500, 600))), _int([0])
    ref_tables, ref_at = tables.tolist(), 0
    out = sv.kv_step_metadata(q, ctx, tables.clone(), free, block, 40, free_start=at)

    def step():
        sv.kv_step_metadata(q, ctx, tables, free, block, 40, free_start=at, out=out)
        at.copy_(out.free_end)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = _gen(4)
    for i in range(6):
        lens = torch.randint(0, 5, (R,), generator=g).tolist()
        q.copy_(_int(lens))
        before = ctx.tolist()
        graph.replay()
        torch.cuda.synchronize()
        want = so.step_metadata(lens, before, ref_tables, free.tolist(), block, 40, ref_at)
        assert (tables.tolist(), *(t.tolist() for t in out[:4]), int(at)) == want
        ref_tables, ref_at = want[0], want[5]
        ctx.copy_(out.seq_lens)


# =============================================================================
#  rotary
# =============================================================================
def _step(dtype):
    return torch.finfo(dtype).eps / 2


def _check_rotated(got, x, positions, inv_freq, interleaved, scale, what):
    """cos and sin within half a step of fp32 (2^-24), two products and their sum as much again, then one rounding."""
    want, pair = so.rotate(x.cpu(), positions.cpu(), inv_freq.cpu(), interleaved, scale)
    err = (got.cpu().double() - want).abs()
    tiny = 2.0 ** -25 if got.dtype is torch.float16 else 0.0           # half a step of the subnormals
    tol = _step(got.dtype) * want.abs() + 4 * 2.0 ** -24 * scale * pair + tiny
    assert bool((err <= tol).all()), f"{what}: off by {float((err - tol).max()):.3e} more than allowed"


@pytest.mark.parametrize("D,rot,interleaved", [
    (64, 64, False), (64, 32, True), (64, 24, False), (80, 80, False), (80, 40, False), (80, 20, True), (80, 2, False),
    (128, 128, False), (128, 128, True), (128, 64, False), (128, 6, True), (128, 36, False)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_rotary_matches_64_bits(D, rot, interleaved, dtype):
    g = _gen(D + rot)
    for N, H, KV in ((1, 1, 1), (3, 14, 2), (37, 5, 5), (700, 2, 1)):
        x = torch.randn((N, (H + KV) * D + 8), generator=g).to(dtype).to(DEV)
        q, k = x[:, :H * D].view(N, H, D), x[:, H * D:(H + KV) * D].view(N, KV, D)
        positions = torch.randint(-5, 1 << 20, (N,), generator=g).to(DEV)
        inv_freq, _ = _sv().rotary_frequencies(rot, 10000.0, device=DEV)
        scale = 1.25
        keep = x.clone()
        qr, kr = _sv().kv_rotary(q, k, positions, inv_freq, interleaved=interleaved, scale=scale)
        assert torch.equal(x, keep)
        _check_rotated(qr, q, positions, inv_freq, interleaved, scale, f"q {N, H, KV}")
        _check_rotated(kr, k, positions, inv_freq, interleaved, scale, f"k {N, H, KV}")
        assert torch.equal(qr[..., rot:], q[..., rot:])
        # the same in place, with 32-bit positions, and q alone
        alone, none = _sv().kv_rotary(q, None, positions.int(), inv_freq, interleaved=interleaved, scale=scale)
        assert none is None and torch.equal(alone, qr)
        _sv().kv_rotary(q, k, positions, inv_freq, interleaved=interleaved, scale=scale, out=(q, k))
        assert torch.equal(q, qr) and torch.equal(k, kr)
        assert torch.equal(x[:, (H + KV) * D:], keep[:, (H + KV) * D:])


def test_rotary_far_positions_and_other_strides():
    """Positions up to 2^31, where fp32 angles would be noise; heads before tokens; a row without unit stride."""
    g = _gen(3)
    N, H, D = 50, 3, 128
    q = torch.randn((H, N, D), generator=g).to(DEV).transpose(0, 1)
    k = torch.randn((N, D, 2), generator=g).to(DEV).transpose(1, 2)
    positions = torch.randint(0, 2**31 - 1, (N,), generator=g).to(DEV)
    inv_freq, _ = _sv().rotary_frequencies(D, device=DEV)
    qr, kr = _sv().kv_rotary(q, k, positions, inv_freq)
    _check_rotated(qr, q, positions, inv_freq, False, 1.0, "q")
    _check_rotated(kr, k, positions, inv_freq, False, 1.0, "k")
    empty = _sv().kv_rotary(q[:0], k[:0], positions[:0], inv_freq)
    assert empty[0].shape == (0, H, D) and empty[1].shape == (0, 2, D)


@pytest.mark.parametrize("H,KV,D,rot,interleaved", [
    (32, 8, 128, 128, False), (14, 2, 64, 64, False), (4, 4, 64, 32, True), (12, 2, 80, 80, False), (8, 8, 80, 40, False),
    (3, 1, 128, 64, True), (64, 8, 128, 128, True)])
@pytest.mark.parametrize("N", [1, 7, 130, 1500])
def test_rotary_store_is_the_rotation_and_the_store(H, KV, D, rot, interleaved, N):
    sv, kd = _sv(), _kd()
    g = _gen(N + H)
    x = torch.randn((N, (H + 2 * KV) * D), generator=g).half().to(DEV)
    x[N // 2, H * D + 3] = math.inf                                 # what the store makes of it, this one has to make too
    q, k, v = x[:, :H * D].view(N, H, D), x[:, H * D:(H + KV) * D].view(N, KV, D), x[:, (H + KV) * D:].view(N, KV, D)
    positions = torch.randint(0, 100_000, (N,), generator=g).to(DEV)
    inv_freq, scale = sv.rotary_frequencies(rot, scaling=dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=4096),
                                            device=DEV)
    bs, nb = 16, N // 16 + 3
    slots = torch.randperm(nb * bs, generator=g)[:N].to(DEV)
    slots[::5] = -1
    slots[N // 3] = nb * bs                                         # past the cache
    kw = dict(interleaved=interleaved, scale=scale)
    want = torch.full((nb, bs, KV, D + 8), 77, dtype=torch.uint8, device=DEV)
    got = want.clone()
    qr, kr = sv.kv_rotary(q, k, positions, inv_freq, **kw)
    kd.kv_quantize_store(kr, v, want, slots, bs)
    assert torch.equal(sv.kv_rotary_quantize_store(q, k, v, got, slots, bs, positions, inv_freq, **kw).view(torch.int16), qr.view(torch.int16))
    assert torch.equal(got, want)
    # in place, with the keys written too
    got.fill_(77)
    sv.kv_rotary_quantize_store(q, k, v, got, slots, bs, positions, inv_freq, q_out=q, key_out=k, **kw)
    assert torch.equal(q.contiguous().view(torch.int16), qr.view(torch.int16))
    assert torch.equal(k.contiguous().view(torch.int16), kr.view(torch.int16))
    assert torch.equal(got, want)


def test_rotary_frequencies_follow_their_formulas():
    sv = _sv()
    i = np.arange(0, 64, 2) / 64
    plain = 500000.0 ** -i
    f, s = sv.rotary_frequencies(64, 500000.0)
    assert s == 1.0 and np.array_equal(f.numpy(), plain.astype(np.float32))
    f, s = sv.rotary_frequencies(64, 500000.0, dict(rope_type="linear", factor=4.0))
    assert s == 1.0 and np.array_equal(f.numpy(), (plain / 4).astype(np.float32))
    f, s = sv.rotary_frequencies(64, 500000.0, dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                                    original_max_position_embeddings=8192))
    for got, freq in zip(f.tolist(), plain):
        wave = 2 * math.pi / freq
        if wave < 8192 / 4:
            want = freq
        elif wave > 8192:
            want = freq / 8
        else:
            smooth = (8192 / wave - 1.0) / 3.0
            want = (1 - smooth) * freq / 8 + smooth * freq
        assert got == pytest.approx(want, rel=2 ** -23)
    f, s = sv.rotary_frequencies(64, 10000.0, dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096))
    assert s == pytest.approx(0.1 * math.log(16.0) + 1.0)
    plain = 10000.0 ** -i
    assert f[0] == 1.0 and f[-1].item() == pytest.approx(plain[-1] / 16, rel=2 ** -23)
    assert bool((f.double() <= torch.tensor(plain) * (1 + 2 ** -23)).all())
    assert bool((f.double() >= torch.tensor(plain) / 16 * (1 - 2 ** -23)).all())


# =============================================================================
#  prompt attention
# =============================================================================
def _prompt_tolerance(dtype, want, mean, span, D, keys, vmax):
    """Weights rounded by half a step each, in the numerator and the sum alike: half a step of (mean |v| + |o|); the output's
    rounding, half a step of |o|; the scores' fp32 sums, (D + 8) 2^-24 of their products' absolute sum in either direction,
    and e^x of that; half a step of fp16's subnormals for every weight, and for the result."""
    u = _step(dtype)
    e = (D + 8) * 2.0 ** -24 * span + 4 * 2.0 ** -23
    tiny = 2.0 ** -25 * (keys * vmax + 1.0) if dtype is torch.float16 else 0.0
    return u * (2 * want.abs() + mean) * (1 + u) + 2.5 * e * mean + tiny


def _check_prompts(q, k, v, q_start, k_start=None, causal=True, scale=None, out=None):
    D = q.shape[2]
    fill = 7.0
    kw = {} if out is None else {"out": out.fill_(fill)}
    got = _sv().kv_prompt_attention(q, k, v, _int(q_start), None if k_start is None else _int(k_start), causal=causal,
                                    scale=scale, **kw)
    torch.cuda.synchronize()
    want, mean, span = so.prompt_attention(q.cpu(), k.cpu(), v.cpu(), q_start, k_start or q_start, causal, scale or D ** -0.5)
    rows = torch.zeros(q.shape[0], dtype=torch.bool)
    rows[q_start[0]:q_start[-1]] = True
    g = got.cpu().double()
    assert bool((g[~rows] == (0.0 if out is None else fill)).all()), "rows of no sequence"
    finite = torch.isfinite(want[rows])
    assert torch.equal(torch.isnan(g[rows]), torch.isnan(want[rows])), "NaN where the formula has a number, or the other way"
    vmax = float(v.float().nan_to_num(0.0, posinf=0.0, neginf=0.0).abs().max()) if v.numel() else 0.0
    tol = _prompt_tolerance(q.dtype, want.nan_to_num(0.0, posinf=0.0, neginf=0.0), mean, span, D, k.shape[0], vmax)[rows]
    err = (g[rows] - want[rows]).abs()
    over = torch.where(finite, err - tol, torch.zeros_like(err)).nan_to_num(0.0)
    assert float(over.max() if over.numel() else 0.0) <= 0.0, f"off by {float(over.max()):.3e} more than allowed"
    assert torch.equal(g[rows][~finite & ~torch.isnan(want[rows])], want[rows][~finite & ~torch.isnan(want[rows])])
    return got


def _prompt_inputs(N, M, H, KV, D, dtype, seed):
    g = _gen(seed)
    r = lambda n, h: torch.randn((n, h, D), generator=g)  # noqa: E731
    return r(N, H).to(dtype).to(DEV), r(M, KV).to(dtype).to(DEV), (r(M, KV) + 0.3).to(dtype).to(DEV)


def _starts(lens, first=0):
    s = [first]
    for n in lens:
        s.append(s[-1] + n)
    return s


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,KV,D", [(4, 2, 64), (3, 1, 80), (4, 4, 80), (8, 2, 128), (5, 5, 128)])
@pytest.mark.parametrize("lens", [[1], [2, 0, 1], [31, 32, 33], [64], [65, 127, 0, 0, 128], [129], [300, 1, 511], [257, 640]])
def test_prompts_match_64_bits(dtype, H, KV, D, lens):
    q, k, v = _prompt_inputs(sum(lens), sum(lens), H, KV, D, dtype, seed=sum(lens) + D)
    _check_prompts(q, k, v, _starts(lens))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_with_keys_of_their_own(dtype, D, causal):
    """More keys than queries (a chunk behind its context), fewer (rows that see none), none at all."""
    ql, kl = [5, 100, 64, 1, 130, 7], [300, 100, 20, 1, 0, 65]
    q, k, v = _prompt_inputs(sum(ql) + 5, sum(kl) + 6, 4, 2, D, dtype, seed=D)
    _check_prompts(q, k, v, _starts(ql, 2), _starts(kl, 3), causal=causal, out=torch.empty_like(q))
    _check_prompts(q, k, v, _starts(ql, 2), _starts(kl, 3), causal=causal, scale=0.3)


def test_prompts_of_many_short_sequences():
    lens = [(7 * i) % 5 for i in range(300)]
    q, k, v = _prompt_inputs(sum(lens), sum(lens), 2, 1, 64, torch.float16, seed=1)
    _check_prompts(q, k, v, _starts(lens))
    assert _sv().kv_prompt_attention(q[:0], k[:0], v[:0], _int([0])).shape == (0, 2, 64)
    assert _sv().kv_prompt_attention(q[:0], k[:0], v[:0], _int([0, 0])).shape == (0, 2, 64)
    assert float(_sv().kv_prompt_attention(q, k, v, _int([0])).abs().max()) == 0.0


@pytest.mark.parametrize("D", [64, 80, 128])
def test_prompts_in_other_layouts(D):
    """Views of a fused buffer, heads before tokens, rows that are not 16-byte aligned, a strided output."""
    H, KV, lens = 4, 2, [70, 130]
    N = sum(lens)
    g = _gen(D)
    x = torch.randn((N, (H + 2 * KV) * D), generator=g).half().to(DEV)
    q, k, v = x[:, :H * D].view(N, H, D), x[:, H * D:(H + KV) * D].view(N, KV, D), x[:, (H + KV) * D:].view(N, KV, D)
    wide = torch.empty((N, H, 2 * D), dtype=torch.float16, device=DEV)
    _check_prompts(q, k, v, _starts(lens), out=wide[:, :, :D])
    hq = torch.randn((H, N, D), generator=g).half().to(DEV).transpose(0, 1)
    hk = torch.randn((KV, N, D), generator=g).half().to(DEV).transpose(0, 1)
    hv = torch.randn((N, D, KV), generator=g).half().to(DEV).transpose(1, 2)
    _check_prompts(hq, hk, hv, _starts(lens), out=torch.empty((H, N, D), dtype=torch.float16, device=DEV).transpose(0, 1))
    odd = torch.randn((N, KV * D + 1), generator=g).half().to(DEV)[:, 1:].view(N, KV, D)
    _check_prompts(hq, odd, hv, _starts(lens))


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("n", [200, 1100])
def test_prompts_into_rows_of_8_bytes(D, n):
    """The least alignment that an output may have, and what lies between its rows kept."""
    H = 2
    q, k, v = _prompt_inputs(n, n, H, 1, D, torch.bfloat16, seed=D)
    flat = torch.full((n * H * (D + 4) + 4,), 5.0, dtype=torch.bfloat16, device=DEV)
    out = flat[4:].as_strided((n, H, D), (H * (D + 4), D + 4, 1))
    assert out.data_ptr() % 16 == 8
    got = _sv().kv_prompt_attention(q, k, v, _int([0, n]), out=out)
    assert torch.equal(got, _sv().kv_prompt_attention(q, k, v, _int([0, n])))
    assert bool((flat[4:].as_strided((n, H, 4), (H * (D + 4), D + 4, 1), 4 + D)[:-1] == 5.0).all()) and bool((flat[:4] == 5.0).all())
    with pytest.raises(RuntimeError, match="8-byte aligned"):
        _sv().kv_prompt_attention(q, k, v, _int([0, n]), out=flat[2:].as_strided((n, H, D), (H * (D + 4), D + 4, 1)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 80, 128])
def test_prompts_do_not_see_what_is_masked(dtype, D):
    """Keys and values that are no numbers reach the rows that see them and no other: later tokens of a sequence, the next
    sequence's, and those behind the last."""
    lens = [90, 200, 64]
    q, k, v = _prompt_inputs(sum(lens) + 3, sum(lens) + 3, 2, 1, D, dtype, seed=D + 1)
    v[60, 0, 3], v[70, 0, D - 1] = math.inf, -math.inf
    v[90 + 130, 0, 0] = math.nan
    k[90 + 150, 0, 5] = math.nan
    k[-3:], v[-3:] = math.nan, math.inf
    _check_prompts(q, k, v, _starts(lens))


def test_prompts_with_extreme_scores():
    """Scores of thousands in growing and falling order, all equal, all -infinity."""
    for dtype in (torch.float16, torch.bfloat16):
        D, n = 64, 400
        q, k, v = _prompt_inputs(n, n, 1, 1, D, dtype, seed=11)
        q[..., 1:], k[..., 1:] = 0.0, 0.0
        q[..., 0] = 8.0
        for ramp in (torch.linspace(-500, 500, n), torch.linspace(500, -500, n), torch.full((n,), 30.0)):
            k[:, 0, 0] = ramp.to(dtype).to(DEV)
            _check_prompts(q, k, v, [0, n])
        q[..., 0], k[:, 0, 0] = 1.0, -math.inf                   # every score -infinity: 0 / 0, as in a softmax
        assert bool(torch.isnan(_sv().kv_prompt_attention(q, k, v, _int([0, n]))).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,KV,D", [(4, 2, 64), (3, 1, 80), (6, 2, 128)])
@pytest.mark.parametrize("lens", [[513], [640], [1025], [700, 500], [1, 1300], [900, 0, 1000]])
def test_prompts_of_few_workgroups_and_many_keys(dtype, H, KV, D, lens):
    """Where two halves of a workgroup share the keys: an odd and an even number of tiles, one half without any."""
    q, k, v = _prompt_inputs(sum(lens), sum(lens), H, KV, D, dtype, seed=sum(lens) + D)
    _check_prompts(q, k, v, _starts(lens))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 80, 128])
def test_prompts_of_few_workgroups_with_keys_of_their_own(dtype, D):
    ql, kl = [1, 200, 64, 0, 130, 300], [1500, 1000, 700, 100, 0, 64]
    q, k, v = _prompt_inputs(sum(ql) + 5, sum(kl) + 6, 4, 2, D, dtype, seed=D)
    for causal in (True, False):
        _check_prompts(q, k, v, _starts(ql, 2), _starts(kl, 3), causal=causal, out=torch.empty_like(q))
    want = _sv().kv_prompt_attention(q, k, v, _int(_starts(ql)), _int(_starts(kl)))
    out = _sv().kv_prompt_attention(q, k, v, _int(_starts(ql)), _int(_starts(kl)), out=q)      # (rows of no sequence stay)
    assert out is q and torch.equal(q[:sum(ql)], want[:sum(ql)])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 80, 128])
def test_prompts_of_few_workgroups_do_not_see_what_is_masked(dtype, D):
    lens = [900, 700]
    q, k, v = _prompt_inputs(sum(lens) + 3, sum(lens) + 3, 2, 1, D, dtype, seed=D + 1)
    v[700, 0, 3], v[780, 0, D - 1] = math.inf, -math.inf             # (an even tile and an odd one)
    v[900 + 650, 0, 0] = math.nan
    k[900 + 600, 0, 5] = math.nan
    k[-3:], v[-3:] = math.nan, math.inf
    _check_prompts(q, k, v, _starts(lens))
    n = 1100                                                        # scores of thousands, in both orders
    q, k, v = _prompt_inputs(n, n, 1, 1, D, dtype, seed=11)
    q[..., 1:], k[..., 1:] = 0.0, 0.0
    q[..., 0] = 8.0
    for ramp in (torch.linspace(-500, 500, n), torch.linspace(500, -500, n), torch.full((n,), 30.0)):
        k[:, 0, 0] = ramp.to(dtype).to(DEV)
        _check_prompts(q, k, v, [0, n])
    q[..., 0], k[:, 0, 0] = 1.0, -math.inf
    assert bool(torch.isnan(_sv().kv_prompt_attention(q, k, v, _int([0, n]))).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,KV,D", [(2, 1, 64), (3, 3, 80), (4, 1, 128)])
@pytest.mark.parametrize("ql,kl", [([1], [2500]), ([130], [4097]), ([1, 7, 0, 40], [3000, 1, 900, 5000]), ([300, 3], [2, 4500])])
def test_prompts_of_few_rows_whose_keys_are_shared_out(dtype, H, KV, D, ql, kl):
    """Parts of the keys in several workgroups, joined: shares that a row sees nothing of, sequences shorter than the shares."""
    q, k, v = _prompt_inputs(sum(ql) + 5, sum(kl) + 6, H, KV, D, dtype, seed=D + sum(kl))
    need = int(_sv()._entry(_sv()._load_native_extension(), "prompt_workspace_bytes")(q.shape[0], k.shape[0], len(ql), H, D))
    assert need > 0
    for causal in (True, False):
        _check_prompts(q, k, v, _starts(ql, 2), _starts(kl, 3), causal=causal, out=torch.empty_like(q))
    got = _check_prompts(q, k, v, _starts(ql, 2), _starts(kl, 3))
    assert torch.equal(got, _sv().kv_prompt_attention(q, k, v, _int(_starts(ql, 2)), _int(_starts(kl, 3))))
    last = 3 + sum(kl) - 1                                          # the last key alone is none of the first rows'
    k[last, 0, 0], v[last, 0, 1] = math.inf, math.nan
    v[3 + kl[0] // 2, 0, 2] = -math.inf
    _check_prompts(q, k, v, _starts(ql, 2), _starts(kl, 3))
    out = _sv().kv_prompt_attention(q, k, v, _int(_starts(ql, 2)), _int(_starts(kl, 3)), out=q)
    assert out is q


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompts_of_few_rows_with_extreme_scores(dtype):
    n, D = 6000, 64
    q, k, v = _prompt_inputs(3, n, 1, 1, D, dtype, seed=11)
    q[..., 1:], k[..., 1:] = 0.0, 0.0
    q[..., 0] = 8.0
    for ramp in (torch.linspace(-500, 500, n), torch.linspace(500, -500, n), torch.full((n,), 30.0)):
        k[:, 0, 0] = ramp.to(dtype).to(DEV)
        _check_prompts(q, k, v, [0, 3], [0, n])
    q[..., 0], k[:, 0, 0] = 1.0, -math.inf
    assert bool(torch.isnan(_sv().kv_prompt_attention(q, k, v, _int([0, 3]), _int([0, n]))).all())
    k[4000, 0, 0] = 1.0                                             # the only key that has weight
    _check_prompts(q, k, v, [0, 3], [0, n])


def test_prompts_of_few_rows_in_graphs():
    """Two captured calls with a workspace each, replayed in turn, between eager ones."""
    sv = _sv()
    stream = torch.cuda.Stream()
    calls = []
    for seed, (N, M) in enumerate(((2, 5000), (100, 3000))):
        q, k, v = _prompt_inputs(N, M, 4, 2, 128, torch.float16, seed=seed)
        qs, ks = _int([0, N]), _int([0, M])
        sv.kv_prompt_attention(q, k, v, qs, ks)
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = sv.kv_prompt_attention(q, k, v, qs, ks)
        calls.append((q, k, v, qs, ks, graph, out))
    for turn in range(3):
        for i, (q, k, v, qs, ks, graph, out) in enumerate(calls):
            for a, b in zip((q, k, v), _prompt_inputs(q.shape[0], k.shape[0], 4, 2, 128, torch.float16, seed=9 + 2 * turn + i)):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, sv.kv_prompt_attention(q, k, v, qs, ks))


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("lens", [[1200], [500, 0, 640, 1], [300, 300, 300, 300]])
def test_prompts_of_one_to_two_workgroups_a_cu(D, lens):
    """Their order is another: falling, then rising."""
    q, k, v = _prompt_inputs(sum(lens), sum(lens), 32, 4, D, torch.float16, seed=sum(lens) + D)
    _check_prompts(q, k, v, _starts(lens))


def test_prompts_whose_offsets_pass_32_bits():
    n, D, stride = 300, 64, 1 << 24
    flat = torch.empty(n * stride + 3 * D, dtype=torch.float16, device=DEV)     # 10 GB
    q = flat.as_strided((n, 1, D), (stride, D, 1))
    k, v = flat.as_strided((n, 1, D), (stride, D, 1), D), flat.as_strided((n, 1, D), (stride, D, 1), 2 * D)
    a, b, c = _prompt_inputs(n, n, 1, 1, D, torch.float16, seed=5)
    q.copy_(a), k.copy_(b), v.copy_(c)
    want = _sv().kv_prompt_attention(a, b, c, _int([0, n]))
    assert torch.equal(_sv().kv_prompt_attention(q, k, v, _int([0, n])), want)
    _sv().kv_prompt_attention(q, k, v, _int([0, n]), out=q)
    assert torch.equal(q, want)


# =============================================================================
#  sampling
# =============================================================================
def _check_sample(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens equal, probabilities within fp32 rounding (half a step, and the weights' own 2^-40)."""
    tokens, probs = _sv().sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p, return_probs=True)
    x, u = logits.double().cpu().numpy(), uniforms.double().cpu().numpy()
    each = lambda a, i: float(torch.tensor(a, dtype=torch.float32)) if not isinstance(a, torch.Tensor) else a[i].item()  # noqa: E731
    for i in range(x.shape[0]):
        token, prob = so.sample(x[i], u[i], each(temperature, i), int(each(top_k, i)), each(top_p, i), each(min_p, i))
        assert int(tokens[i]) == token, f"row {i}"
        assert float(probs[i]) == pytest.approx(prob, rel=2.0 ** -22, abs=2.0 ** -40), f"row {i}"
    return tokens


def _logits(B, V, seed, dtype=torch.float32, spread=3.0):
    x = torch.randn((B, V), generator=_gen(seed)) * spread
    return x.to(dtype).to(DEV)


def _uniforms(B, seed):
    return torch.rand(B, generator=_gen(seed + 100)).to(DEV)


CUTS = [dict(), dict(top_k=1), dict(top_k=40), dict(top_k=3000), dict(top_p=0.9), dict(top_p=0.05), dict(top_p=0.0),
        dict(min_p=0.1), dict(min_p=1.0), dict(top_k=50, top_p=0.8), dict(top_k=200, top_p=0.999, min_p=0.01),
        dict(temperature=0.0), dict(temperature=0.3, top_p=0.95), dict(temperature=2.5, top_k=1000, top_p=0.7)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 63, 4095, 4097, 32000])
def test_samples_match_the_sorted_row(dtype, V):
    B = 5
    x = _logits(B, V + 3, V, dtype)[:, 1:V + 1]                     # (strided rows, two-byte alignment)
    for i, kw in enumerate(CUTS):
        _check_sample(x, _uniforms(B, 10 * V + i), **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [32_768, 32_769, 50_257, 151_936])
def test_samples_of_long_rows(dtype, V):
    B = 3
    x = _logits(B, V + 3, V, dtype)[:, 1:V + 1]
    for i, kw in enumerate(CUTS):
        _check_sample(x, _uniforms(B, 10 * V + i), **kw)


def test_samples_of_many_long_rows():
    """As many rows as leave each a single workgroup, and more."""
    V = 33_001
    x = _logits(530, V, 4, torch.float16)
    for i, kw in enumerate((dict(top_k=40, top_p=0.9), dict(top_p=0.9), dict())):
        _check_sample(x, _uniforms(530, i), **kw)


def test_samples_of_the_longest_rows():
    V = 1 << 22
    x = _logits(2, V, 4, torch.float32)
    x[1] = 0.0                                                       # (4 million equal ones)
    for i, kw in enumerate((dict(), dict(top_k=500), dict(top_p=0.5), dict(temperature=0.0))):
        _check_sample(x, _uniforms(2, i), **kw)


@pytest.mark.parametrize("V", [5000, 9000, 50_001])
@pytest.mark.parametrize("kind", ["equal", "two", "near", "steps"])
def test_samples_of_rows_that_crowd_one_bin(V, kind):
    """More elements about the cut than the list holds: equal logits, two values, values a millionth apart, whole numbers."""
    g = _gen(V)
    x = {"equal": torch.full((4, V), 2.5), "two": torch.randint(0, 2, (4, V), generator=g).float(),
         "near": 1.0 + torch.randint(0, 1000, (4, V), generator=g) * 2.0 ** -20,
         "steps": torch.randint(-3, 3, (4, V), generator=g).float()}[kind].to(DEV)
    for i, kw in enumerate((dict(top_k=V // 3), dict(top_p=0.5), dict(top_k=V // 2, top_p=0.25), dict(top_k=3, top_p=0.9),
                            dict(top_p=0.7, min_p=0.9), dict(top_k=V - 1), dict(top_p=0.0))):
        _check_sample(x, _uniforms(4, i), **kw)


@pytest.mark.parametrize("V", [300, 1500, 2048, 45_000])
@pytest.mark.parametrize("kind", ["equal", "two", "near", "steps", "far"])
def test_samples_of_a_few_hundred_kept(V, kind):
    """Lists long enough to be ordered by parts of their range: one value, two, close ones, whole numbers, and one far away."""
    g = _gen(V + 1)
    x = {"equal": torch.full((3, V), -2.5), "two": torch.randint(0, 2, (3, V), generator=g).float(),
         "near": 1.0 + torch.randint(0, 1000, (3, V), generator=g) * 2.0 ** -20,
         "steps": torch.randint(-20, 20, (3, V), generator=g).float() / 8, "far": torch.randn((3, V), generator=g) * 0.5}[kind]
    if kind == "far":
        x[:, V // 2] = 9.0
    if V > 2048:                                                    # all but 1800 of them far below
        x[:, torch.randperm(V, generator=g)[1800:]] = -100.0
    x = x.to(DEV)
    for i, kw in enumerate((dict(top_k=min(V - 1, 1024)), dict(top_k=V // 3 if V < 3000 else 700), dict(top_k=290, top_p=0.6),
                            dict(top_k=min(V - 1, 1000), top_p=0.97, min_p=0.2), dict(top_p=0.8), dict(top_p=0.3, min_p=0.5))):
        _check_sample(x, _uniforms(3, i), **kw)


@pytest.mark.parametrize("V", [6000, 40_000])
def test_samples_of_rows_with_other_values(V):
    """-infinity (masked tokens), NaN, +infinity, both zeros, logits of 10^30, a row that leaves nothing."""
    x = _logits(8, V, 3)
    x[0, 5:] = -math.inf
    x[1, ::2] = math.nan
    x[2, [17, 900, 5999]] = math.inf
    x[3] = -math.inf
    x[4] = math.nan
    x[5] = torch.where(torch.arange(V, device=DEV) % 2 == 0, 0.0, -0.0)
    x[6] *= 1e30
    x[7] = -math.inf
    x[7, V - 1] = -3e38
    for i, kw in enumerate(CUTS):
        tokens = _check_sample(x, _uniforms(8, i), **kw)
        assert int(tokens[3]) == 0 and int(tokens[4]) == 0 and int(tokens[7]) == V - 1


@pytest.mark.parametrize("V", [10_000, 40_000])
def test_samples_at_the_ends_of_the_uniforms(V):
    x = _logits(6, V, 8)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, -1.0, math.nan, 2.0 ** -60], device=DEV)
    for kw in (dict(), dict(top_k=20), dict(top_p=0.5), dict(min_p=0.2)):
        _check_sample(x, torch.where(torch.isnan(u), torch.zeros_like(u), u), **kw)
        _sv().sample_tokens(x, u, **kw)


@pytest.mark.parametrize("V", [7000, 40_000])
def test_samples_with_an_argument_for_every_row(V):
    B = 40
    g = _gen(2)
    pick = lambda values, dtype: torch.tensor([values[int(torch.randint(0, len(values), (1,), generator=g))] for _ in range(B)],  # noqa: E731
                                              dtype=dtype, device=DEV)
    t, k = pick([0.0, 0.5, 1.0, 1.7, -1.0], torch.float32), pick([0, 1, 7, 100, V, 2 * V, -3], torch.int32)
    p, m = pick([1.0, 0.9, 0.3, 0.0, 1.5], torch.float32), pick([0.0, 0.05, 1.0], torch.float32)
    x, u = _logits(B, V, 5, torch.float16), _uniforms(B, 5)
    tokens = _check_sample(x, u, t, k, p, m)
    out = torch.empty(B, dtype=torch.int64, device=DEV)
    assert _sv().sample_tokens(x, u, t, k, p, m, out=out) is out and torch.equal(out, tokens)
    assert _sv().sample_tokens(x[:0], u[:0]).shape == (0,)


def test_samples_repeat_bit_for_bit_and_from_a_graph():
    """The sums do not depend on the order of their atomics; a graph's replays give the eager tokens."""
    B, V = 16, 60_000
    x, u = _logits(B, V, 6, torch.bfloat16, spread=1.0), _uniforms(B, 6)
    kw = dict(temperature=0.8, top_k=5000, top_p=0.95, return_probs=True)
    first = [t.clone() for t in _sv().sample_tokens(x, u, **kw)]
    for _ in range(5):
        again = _sv().sample_tokens(x, u, **kw)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = _sv().sample_tokens(x, u, **kw)
    for seed in range(4):
        u.copy_(_uniforms(B, 50 + seed))
        x.copy_(_logits(B, V, 50 + seed, torch.bfloat16, spread=1.0))
        graph.replay()
        torch.cuda.synchronize()
        want = _sv().sample_tokens(x, u, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# =============================================================================
#  together
# =============================================================================
def _dequantized(cache, table, n, bs, D):
    pos = torch.arange(n)
    slot = cache.cpu()[table.cpu().long()[pos // bs], pos % bs]
    r = slot[..., D:].contiguous().view(torch.float16).double()
    code = lambda x: torch.stack([x & 15, x >> 4], -1).flatten(-2).double()  # noqa: E731
    return code(slot[..., :D // 2]) * r[..., 1:2] + r[..., 0:1], code(slot[..., D // 2:D]) * r[..., 3:4] + r[..., 2:3]


@pytest.mark.parametrize("H,KV,D", [(8, 2, 64), (8, 8, 80), (16, 2, 128)])
def test_serving_steps_together(H, KV, D):
    """Prompts of different lengths and the decode steps behind them through every operator: metadata, rotation with the store,
    attention of the prompts and of the packed cache, sampling.  Each step is checked in 64 bits on the bytes before it."""
    sv, kd = _sv(), _kd()
    g = _gen(H + D)
    bs, lens, steps, V = 16, [37, 1, 80, 16], 4, 500
    R = len(lens)
    inv_freq, scale = sv.rotary_frequencies(D, device=DEV)
    head = torch.randn((H * D, V), generator=g).to(DEV) * 0.2
    cache = torch.zeros((40, bs, KV, D + 8), dtype=torch.uint8, device=DEV)
    tables = torch.zeros((R, 8), dtype=torch.int32, device=DEV)
    free = torch.randperm(40, generator=g).to(torch.int32).to(DEV)
    ctx, at = torch.zeros(R, dtype=torch.int32, device=DEV), _int([0])
    total = lens
    for step in range(steps + 1):
        new = lens if step == 0 else [1] * R
        N = sum(new) + 3                                            # three padding rows
        x = torch.randn((N, (H + 2 * KV) * D), generator=g).half().to(DEV)
        q, k, v = x[:, :H * D].view(N, H, D), x[:, H * D:(H + KV) * D].view(N, KV, D), x[:, (H + KV) * D:].view(N, KV, D)
        m = sv.kv_step_metadata(_int(new), ctx, tables, free, bs, N, free_start=at)
        raw = k.clone()
        turned = torch.zeros_like(raw)
        qr = sv.kv_rotary_quantize_store(q, k, v, cache, m.slot_mapping, bs, m.positions, inv_freq, scale=scale, key_out=turned)
        if step == 0:
            out = sv.kv_prompt_attention(qr, turned, v, m.query_start_loc)
            want, mean, span = so.prompt_attention(qr.cpu(), turned.cpu(), v.cpu(), _starts(lens), _starts(lens), True, D ** -0.5)
            rows = torch.arange(sum(lens))
            tol = _prompt_tolerance(torch.float16, want[rows], mean[rows], span[rows], D, N, float(v.abs().max()))
            assert bool(((out.cpu().double() - want).abs()[rows] <= tol).all())
            last = (m.query_start_loc[1:] - 1).long()
        else:
            out = kd.kv_dequant_decode_paged_batched(qr[:R], cache, tables, m.seq_lens, bs, KV, out_dtype=torch.float16)
            total = [n + 1 for n in total]
            for r in range(R):
                kk, vv = _dequantized(cache, tables[r], total[r], bs, D)
                z = torch.einsum("hd,nhd->hn", qr[r].cpu().double(), kk.repeat_interleave(H // KV, 1)) * D ** -0.5
                o = torch.einsum("hn,nhd->hd", torch.softmax(z, -1), vv.repeat_interleave(H // KV, 1))
                # the decode's bar: 2e-3 and one per cent
                assert bool(((out[r].cpu().double() - o).abs() <= 2e-3 + 1e-2 * o.abs()).all())
            last = torch.arange(R, device=DEV)
        assert m.seq_lens.tolist() == total
        ctx, at = m.seq_lens, m.free_end
        logits = out[last].flatten(1).float() @ head
        _check_sample(logits, _uniforms(R, step), temperature=0.9, top_k=100, top_p=0.9)
    assert int(at) == sum(-(-n // bs) for n in total)


def test_operators_on_another_stream():
    sv = _sv()
    N, H, KV, D = 300, 4, 2, 64
    q, k, v = _prompt_inputs(N, N, H, KV, D, torch.float16, seed=2)
    pos = torch.arange(N, device=DEV)
    inv_freq, _ = sv.rotary_frequencies(D, device=DEV)
    x, u = _logits(4, 9000, 1), _uniforms(4, 1)

    def all_of_them():
        qr, kr = sv.kv_rotary(q, k, pos, inv_freq)
        return qr, kr, sv.kv_prompt_attention(qr, kr, v, _int([0, 100, N])), sv.sample_tokens(x, u, top_p=0.9)

    want = all_of_them()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = all_of_them()
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def _everything(q, k, v, cache, lens, ctx, tables, free, inv_freq, logits, u):
    """A step through every operator, on tensors that stay where they are."""
    sv = _sv()
    N, bs = q.shape[0], cache.shape[1]
    m = sv.kv_step_metadata(lens, ctx, tables, free, bs, N)
    qr, kr = sv.kv_rotary(q, k, m.positions, inv_freq)
    qs = sv.kv_rotary_quantize_store(q, k, v, cache, m.slot_mapping, bs, m.positions, inv_freq)
    out = sv.kv_prompt_attention(qr, kr, v, m.query_start_loc)
    return (*m, qr, kr, qs, out, *sv.sample_tokens(logits, u, top_p=0.9, return_probs=True))


def _everything_inputs(seed, N=700, R=3, H=4, KV=2, D=64, V=40_000):
    g = _gen(seed)
    r = lambda *s: torch.randn(s, generator=g).half().to(DEV)  # noqa: E731
    lens = torch.randint(0, N // R, (R,), generator=g).to(torch.int32).to(DEV)
    ctx = torch.randint(0, 40, (R,), generator=g).to(torch.int32).to(DEV)
    tables = torch.arange(R * 64, dtype=torch.int32).view(R, 64).to(DEV)
    free = (R * 64 + torch.randperm(200, generator=g)).to(torch.int32).to(DEV)
    cache = torch.zeros((R * 64 + 200, 16, KV, D + 8), dtype=torch.uint8, device=DEV)
    inv_freq, _ = _sv().rotary_frequencies(D, device=DEV)
    return [r(N, H, D), r(N, KV, D), r(N, KV, D), cache, lens, ctx, tables, free, inv_freq, r(3, V) * 3, _uniforms(3, seed)]


def _same(a, b):
    return a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_operators_from_two_graphs_between_eager_steps():
    """Two captured steps, replayed in turn with inputs rewritten in place and eager steps between them."""
    stream = torch.cuda.Stream()
    steps = []
    for seed in (1, 2):
        static = _everything_inputs(seed)
        _everything(*static)
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = _everything(*static)
        steps.append((static, graph, got))
    for turn in range(3):
        for i, (static, graph, got) in enumerate(steps):
            new = _everything_inputs(10 * turn + i + 3)
            for a, b in zip(static, new):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            want = _everything(*new)
            assert all(_same(a, b) for a, b in zip(got, want))
            assert _same(static[3], new[3]) and _same(static[6], new[6])     # the cache and the tables


def test_operators_on_two_streams_at_once():
    inputs = [_everything_inputs(seed, N=2000) for seed in (5, 6)]
    want = [_everything(*[t.clone() for t in x]) for x in inputs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    rounds = []
    for _ in range(3):
        copies = [[t.clone() for t in x] for x in inputs]
        torch.cuda.synchronize()
        got = [None, None]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _everything(*copies[i])
        torch.cuda.synchronize()
        rounds.append(got)
    for got in rounds:
        for a, b in zip(got, want):
            assert all(_same(x, y) for x, y in zip(a, b))


def test_numbers_that_do_not_fit_are_refused():
    """Nothing past 32 bits reaches the library cut to them."""
    sv = _sv()
    lens, tables, free = _int([1, 2]), torch.zeros((2, 4), dtype=torch.int32, device=DEV), _int([0, 1])
    for block, n in ((16, -1), (16, 1 << 32), (16, (1 << 32) + 3), (0, 3), (-16, 3), ((1 << 32) + 16, 3)):
        with pytest.raises(RuntimeError, match="below 2\\^31"):
            sv.kv_step_metadata(lens, lens, tables, free, block, n)
    x, u = _logits(2, 50, 1), _uniforms(2, 1)
    for k in (-1, -(1 << 32), -(1 << 32) + 5):
        with pytest.raises(RuntimeError, match="top_k must be"):
            sv.sample_tokens(x, u, top_k=k)
    assert torch.equal(sv.sample_tokens(x, u, top_k=1 << 40), sv.sample_tokens(x, u))
    with pytest.raises(RuntimeError, match="fewer than 2\\^31"):
        sv.sample_tokens(x[:, :1].expand(2, (1 << 32) + 5), u)
    with pytest.raises(RuntimeError, match="vocabularies of up to"):
        sv.sample_tokens(x[:, :1].expand(2, (1 << 22) + 1), u)


@pytest.mark.parametrize("H,KV,D", [(3, 1, 64), (2, 2, 128)])
@pytest.mark.parametrize("lens", [[128], [256, 128], [1, 129, 127, 128], [1] * 200, [128] * 9, [129] * 9, [0, 0, 1]])
def test_prompts_fill_their_blocks(H, KV, D, lens):
    """As many blocks as the rows can make, and no row without one."""
    q, k, v = _prompt_inputs(sum(lens), sum(lens), H, KV, D, torch.float16, seed=sum(lens))
    _check_prompts(q, k, v, _starts(lens))
