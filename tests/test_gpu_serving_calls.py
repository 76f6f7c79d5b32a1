"""GPU: calls of the serving step's operators (kernels.serving) that their documentation allows and that sizes, strides and
values off the usual ones make hard, against the definitions in 64 bits."""
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


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


# =============================================================================
#  prompt attention
# =============================================================================
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("n,m,H,causal", [
    (3, 20_000, 2, False),      # the keys shared out over workgroups
    (200, 1500, 2, False),      # two halves of a workgroup
    (130, 1000, 300, True),     # one workgroup for a block of rows
    (40, 60, 2, False)])        # a tile that no row sees whole
def test_prompts_count_keys_of_little_weight(dtype, D, n, m, H, causal):
    """One key that outweighs each of the others by 2^17 to 2^30, ahead of them or behind: together they count."""
    for bits in (17.3, 20.6, 22.4, 24.1, 25.4, 27.2, 30.1):
        for heavy in (0, m - 1):
            q, k, v = (torch.zeros((x, h, D), dtype=dtype) for x, h in ((n, H), (m, 1), (m, 1)))
            q[..., 0] = 1.0
            k[:, 0, 0] = -bits * math.log(2.0)
            k[heavy, 0, 0] = 0.0
            v[:, 0] = (1.0 + torch.arange(D) / 64.0).to(dtype)
            v[heavy] = 0.0
            got = _sv().kv_prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), _int([0, n]), _int([0, m]), causal=causal, scale=1.0)
            # row i sees the keys up to i + m - n: `light` ones of weight w beside the heavy one (if it sees that)
            w = math.exp(float(k[1 if heavy == 0 else 0, 0, 0]))
            seen = torch.arange(n) + (m - n) + 1 if causal else torch.full((n,), m)
            sees = seen > heavy
            light = (seen - sees.long()).double()
            share = torch.where(sees, light * w / (1.0 + light * w), 1.0)
            want = share[:, None] * v[1 if heavy == 0 else 0, 0].double()
            # Weights relative to the largest are rounded by half a step each, in fp16 at least by half a step of its subnormals,
            # 2^-25, of 2^-6: a light key's by 2^-31, `light` of them by light 2^-31 of a sum of 1 and more, times v; the sums add
            # the same weights (a second time the error, times the result).  The output's own half step; its subnormals' 2^-25.
            # The exponent: 2^-24 of its |bits| ln 2 twice, and 2^-22 for the exponential itself.
            u = torch.finfo(dtype).eps / 2
            vmax = v[1 if heavy == 0 else 0, 0].double()
            tiny = (light[:, None] * 2.0 ** -31 * (vmax + want) + 2.0 ** -25) if dtype is torch.float16 else 0.0
            tol = want * (3 * u + 2 * bits * 2.0 ** -24 + 2.0 ** -22) * (1 + u) + tiny
            err = (got.cpu().double() - want[:, None]).abs()
            over = (err - tol[:, None]).max()
            assert float(over) <= 0.0, f"{bits} bits, heavy key {heavy}: off by {float(over):.3e} more than allowed"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 80, 128])
def test_prompts_from_rows_of_any_alignment(dtype, D):
    """Rows that torch calls contiguous and that do not lie on 16 bytes: a whole tensor at an odd offset, one token, one head."""
    H, KV, n = 4, 2, 150
    g = _gen(D)
    odd = lambda rows, heads, at: torch.randn(rows * heads * D + at, generator=g).to(dtype).to(DEV)[at:].view(rows, heads, D)  # noqa: E731
    for at in (1, 2, 4, 7):
        q, k, v = odd(n, H, at), odd(n, KV, at), odd(n, KV, at)
        assert q.is_contiguous() and q.data_ptr() % 16
        want = _sv().kv_prompt_attention(*(torch.empty_like(t).copy_(t) for t in (q, k, v)), _int([0, 50, n]))
        assert torch.equal(_sv().kv_prompt_attention(q, k, v, _int([0, 50, n])), want)
    # one token of a buffer whose rows are odd apart; the strides of a dim of one element are of no account
    def one(heads, token, head):
        flat = torch.randn(4000, generator=g).to(dtype).to(DEV)
        return flat.as_strided((1, heads, D), (token, head, 1))
    q, k, v = one(H, H * D + 3, D), one(KV, 2 * D + 5, D), one(KV, 1, D)
    want = _sv().kv_prompt_attention(*(t.reshape(-1).clone().view(t.shape) for t in (q, k, v)), _int([0, 1]))
    assert torch.equal(_sv().kv_prompt_attention(q, k, v, _int([0, 1])), want)
    k, v = (torch.randn(n * D, generator=g).to(dtype).to(DEV).as_strided((n, 1, D), (D, 67, 1)) for _ in "kv")
    q = torch.randn(n * D, generator=g).to(dtype).to(DEV).as_strided((n, 1, D), (D, 3, 1))
    want = _sv().kv_prompt_attention(*(t.reshape(-1).clone().view(n, 1, D) for t in (q, k, v)), _int([0, n]))
    assert torch.equal(_sv().kv_prompt_attention(q, k, v, _int([0, n])), want)


@pytest.mark.parametrize("D", [64, 80, 128])
def test_prompts_into_one_token_or_one_head_of_any_stride(D):
    H, n = 3, 70
    g = _gen(D)
    r = lambda rows, heads: torch.randn((rows, heads, D), generator=g).half().to(DEV)  # noqa: E731
    q, k, v = r(1, H), r(1, H), r(1, H)
    out = torch.zeros(H * D, dtype=torch.float16, device=DEV).as_strided((1, H, D), (5, D, 1))
    assert torch.equal(_sv().kv_prompt_attention(q, k, v, _int([0, 1]), out=out), _sv().kv_prompt_attention(q, k, v, _int([0, 1])))
    q, k, v = r(n, 1), r(n, 1), r(n, 1)
    out = torch.zeros(n * D, dtype=torch.float16, device=DEV).as_strided((n, 1, D), (D, 7, 1))
    assert torch.equal(_sv().kv_prompt_attention(q, k, v, _int([0, n]), out=out), _sv().kv_prompt_attention(q, k, v, _int([0, n])))


# =============================================================================
#  rotary positions
# =============================================================================
def _exact_turns(positions, inv_freq):
    """cos and sin of positions * inv_freq: the position in parts of 26 bits, whose products with the 24 bits of a frequency
    are exact, and the sum of the parts' angles by the addition formulas."""
    c, s = (np.empty((len(positions), len(inv_freq))) for _ in "cs")
    for i, p in enumerate(positions):
        for j, f in enumerate(inv_freq):
            a, b = float(p >> 26 << 26) * f, float(p & (1 << 26) - 1) * f
            c[i, j] = math.cos(a) * math.cos(b) - math.sin(a) * math.sin(b)
            s[i, j] = math.sin(a) * math.cos(b) + math.cos(a) * math.sin(b)
    return torch.from_numpy(c), torch.from_numpy(s)


@pytest.mark.parametrize("bits", [17, 31, 38, 45, 52])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_angles_are_exact_at_any_position(bits, interleaved):
    D, N = 64, 40
    g = _gen(bits)
    positions = torch.randint(1 << bits - 1, 1 << bits, (N,), generator=g)
    positions[::3] *= -1
    inv_freq, _ = _sv().rotary_frequencies(D, device="cpu")
    c, s = _exact_turns(positions.tolist(), inv_freq.tolist())
    # pairs of (1, 0): the results are the cosines and sines themselves, rounded to fp32 once (values below 1: 2^-25 at most;
    # the sums in fp64 are within 2^-50)
    x = torch.zeros((N, 1, D))
    first, second = (slice(0, D, 2), slice(1, D, 2)) if interleaved else (slice(0, D // 2), slice(D // 2, D))
    x[..., first] = 1.0
    got, _ = _sv().kv_rotary(x.to(DEV), None, positions.to(DEV), inv_freq.to(DEV), interleaved=interleaved)
    got = got.cpu().double()[:, 0]
    for a, b in ((got[:, first], c), (got[:, second], s)):
        assert float((a - b).abs().max()) <= 2.0 ** -25 + 2.0 ** -50
    if bits <= 31:
        again, _ = _sv().kv_rotary(x.to(DEV), None, positions.int().to(DEV), inv_freq.to(DEV), interleaved=interleaved)
        assert torch.equal(again.cpu().double()[:, 0], got)


# =============================================================================
#  sampling
# =============================================================================
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("V,gaps", [(50, (33.0, 34.0, 35.0)), (2000, (33.0, 34.0, 35.0)), (2048, (33.5, 35.0)), (12_000, (33.0, 33.5)),
                                    (30_000, (32.0, 32.5)), (40_000, (31.0,))])
def test_samples_of_a_small_k_reach_far_elements(dtype, V, gaps):
    """Elements that far below the largest that their weight is a few units of the sums': whatever the cut by number is, one
    that is kept and first by index is what a uniform of 0 gives."""
    for gap in gaps:
        x = torch.full((1, V), -math.inf)
        x[0, V // 2], x[0, V // 3], x[0, 7] = 0.0, -1.0, -gap
        x[0, 3] = -gap - 30.0                                        # of no weight in any case
        for k in (0, 3, 40, V - 1, min(1025, V - 1)):
            token, prob = _sv().sample_tokens(x.to(dtype).to(DEV), torch.zeros(1, device=DEV), top_k=k, return_probs=True)
            want = so.sample(x[0].double().numpy()[4:], 0.0, 1.0, 0, 1.0, 0.0)
            assert int(token) == 7 == want[0] + 4, (gap, k)
            # (in units of 2^-(62 - ceil(log2 V)), 2^-51 at most: half a unit off, and fp32's rounding)
            unit = 2.0 ** -min(62 - math.ceil(math.log2(V)), 51)
            assert abs(float(prob) - want[1]) <= 0.51 * unit + 2.0 ** -23 * want[1], (gap, k)


# =============================================================================
#  gradients
# =============================================================================
def test_no_argument_wants_a_gradient():
    sv = _sv()
    x, u = torch.zeros((2, 50), device=DEV), torch.zeros(2, device=DEV)
    one = torch.ones(2, device=DEV)
    for name in ("temperature", "top_p", "min_p"):
        sv.sample_tokens(x, u, **{name: one})
        with pytest.raises(RuntimeError, match="sample: no gradients"):
            sv.sample_tokens(x, u, **{name: one.clone().requires_grad_()})
    q, start = torch.zeros((2, 1, 64), dtype=torch.float16, device=DEV), _int([0, 2])
    pos, inv = torch.zeros(2, dtype=torch.int64, device=DEV), torch.ones(32, device=DEV)
    leaf = q.clone().requires_grad_()
    for call in (lambda: sv.kv_prompt_attention(q, q, q, start, out=leaf), lambda: sv.kv_rotary(q, None, pos, inv, out=(leaf, None))):
        with pytest.raises(RuntimeError, match="no gradients"):
            call()
        with torch.no_grad():
            call()


# =============================================================================
#  sizes
# =============================================================================
def test_sizes_that_do_not_fit_are_refused():
    """Nothing past 32 bits reaches the library cut to them, and no copy of such a tensor is made first."""
    sv = _sv()
    wide = (1 << 32) + 2
    q = torch.zeros((1, 1, 64), dtype=torch.float16, device=DEV)
    far = q.expand(wide, 1, 64)
    pos = torch.zeros(1, dtype=torch.int64, device=DEV)
    inv = torch.ones(32, device=DEV)
    with pytest.raises(RuntimeError, match="fewer than 2\\^31"):
        sv.kv_prompt_attention(q, far, far, _int([0, 1]), _int([0, 1]))
    with pytest.raises(RuntimeError, match="fewer than 2\\^31"):
        sv.kv_prompt_attention(far, far, far, _int([0, 1]))
    with pytest.raises(RuntimeError, match="fewer than 2\\^31"):
        sv.kv_rotary(far, None, pos.expand(wide), inv)
    with pytest.raises(RuntimeError, match="fewer than 2\\^31"):
        sv.kv_rotary(q, None, pos, inv[:1].expand(wide))
    with pytest.raises(RuntimeError, match="fewer than 2\\^31"):
        cache = torch.zeros((1, 16, 1, 72), dtype=torch.uint8, device=DEV)
        sv.kv_rotary_quantize_store(far, far, far, cache, pos.expand(wide), 16, pos.expand(wide), inv)
    lens, tables, free = _int([1]), torch.zeros((1, 4), dtype=torch.int32, device=DEV), _int([0])
    with pytest.raises(RuntimeError, match="fewer than 2\\^31"):
        sv.kv_step_metadata(lens, lens, tables, free.expand(wide), 16, 1)
    with pytest.raises(RuntimeError, match="fewer than 2\\^31"):
        sv.kv_step_metadata(lens.expand(wide), lens.expand(wide), tables.expand(wide, 4), free, 16, 1)
