"""Serving operators at the limits of their types: scores and values that are
infinite or NaN, and scales near the ends of fp32."""

import pytest
import torch

from serving_util import make_batch, randn

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

BF, HF = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True)
def _no_reported_errors():
    yield
    from b200ar.ops.gemm import check_errors

    torch.cuda.synchronize()
    check_errors()


# Blocks of up to 32, 128 and 256 rows, single tokens, and blocks that several SMs share.
# new, total, decode
BLOCKS = [([1], [1], True), ([1, 1], [300, 40], True), ([1], [6000], True), ([4, 1], [300, 40], False),
          ([16], [300], False), ([32, 9], [300, 200], False), ([40], [6000], False)]
PAGE = 16


def _inputs(new, total, decode, dtype, d, hq=8, hkv=1):
    batch, pool = make_batch(new, total, PAGE, "cuda", decode=decode)
    q = randn((sum(new), hq, d), dtype, "cuda", 1)
    k, v = (randn((pool, PAGE, hkv, d), dtype, "cuda", i) for i in (2, 3))
    return q, k, v, batch


def _slot(batch, s, p):
    return int(batch.page_table[s, p // PAGE]), p % PAGE


@pytest.mark.parametrize("new,total,decode", BLOCKS)
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)])
def test_attention_rows_that_see_only_minus_infinity(new, total, decode, dtype, d):
    """exp(-inf - max) with a maximum of -inf is NaN; a row that sees nothing gives zeros."""
    from b200ar.ops.paged import paged_attention

    q, k, v, batch = _inputs(new, total, decode, dtype, d)
    q.abs_().clamp_(min=0.01)
    k.fill_(-INF)
    assert torch.isnan(paged_attention(q, k, v, batch)).all()
    # One finite score, seen by the last token of the first sequence alone: all the weight is its.
    p = total[0] - 1
    pg, slot = _slot(batch, 0, p)
    k[pg, slot] = 1.0
    out = paged_attention(q, k, v, batch).view(-1, 8, d)
    assert torch.equal(out[new[0] - 1], v[pg, slot].expand(8, d))
    rest = torch.arange(out.shape[0]) != new[0] - 1
    assert torch.isnan(out[rest]).all()
    if not decode:  # lengths below the number of new tokens: rows before position 0 see nothing
        batch.kv_len.fill_(2)
        k.fill_(-INF)
        out = paged_attention(q, k, v, batch).view(-1, 8, d)
        at = 0
        for n in new:
            nothing = max(n - 2, 0)
            assert (out[at:at + nothing] == 0).all() and torch.isnan(out[at + nothing:at + n]).all()
            at += n


@pytest.mark.parametrize("new,total,decode", BLOCKS)
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)])
def test_attention_rows_that_see_a_score_of_nan(new, total, decode, dtype, d):
    """Wherever it stands, the first position included: all outputs of the row are NaN, and of no other."""
    from b200ar.ops.paged import paged_attention

    q, k, v, batch = _inputs(new, total, decode, dtype, d)
    clean = paged_attention(q, k, v, batch)
    for p in (0, total[0] // 2, total[0] - 1):
        pg, slot = _slot(batch, 0, p)
        old = k[pg, slot].clone()
        k[pg, slot, 0, 3] = NAN
        out = paged_attention(q, k, v, batch)
        k[pg, slot] = old
        sees = torch.zeros(out.shape[0], dtype=torch.bool)
        sees[:new[0]] = torch.arange(total[0] - new[0], total[0]) >= p
        assert torch.isnan(out[sees]).all() and torch.equal(out[~sees], clean[~sees])


@pytest.mark.parametrize("new,total,decode", [([1], [300], True), ([1], [6000], True), ([4], [300], False),
                                              ([16], [300], False), ([40], [6000], False)])
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)])
def test_attention_infinite_value_under_a_vanishing_weight(new, total, decode, dtype, d):
    """An infinite value where a whole part of the positions weighs e^-181 of the rest (nothing in fp32): its column
    is not finite, the others are what they were."""
    from b200ar.ops.paged import paged_attention

    q, k, v, batch = _inputs(new, total, decode, dtype, d)
    q.fill_(4.0 * (128 / d) ** 0.25)
    k.zero_()
    low = range(128, 256) if total[0] == 300 else range(3000)
    for p in low:
        k[_slot(batch, 0, p)] = -4.0 * (128 / d) ** 0.25  # -16 d sqrt(128 / d) / sqrt(d) = -181 after the scale
    clean = paged_attention(q, k, v, batch).view(-1, 8, d)
    pg, slot = _slot(batch, 0, 130)
    v[pg, slot, 0, 7] = INF
    out = paged_attention(q, k, v, batch).view(-1, 8, d)
    assert not torch.isfinite(out[:, :, 7]).any()
    out[:, :, 7] = clean[:, :, 7]
    # Recomputed rows round elsewhere: both are within u A + u |o| of the formula, A the mean of |v|, at most 4.
    u = torch.finfo(dtype).eps / 2
    assert (out.float() - clean.float()).abs().max() <= 2 * u * (4 + clean.float().abs().max())


def _settled(out0, v, batch, hq, hkv, d, causal=True, window=0):
    """Outputs over values that are not finite, from those over the same values with zeros in their places: a column
    is inf, -inf or NaN as the sum of what the row sees in it that is not finite, whatever its (positive) weight."""
    want = out0.view(-1, hkv, hq // hkv, d).clone()
    starts = list(range(batch.sequences + 1)) if batch.q_start is None else batch.q_start.tolist()
    table = batch.page_table.cpu()
    for s, total in enumerate(batch.kv_len.tolist()):
        n = starts[s + 1] - starts[s]
        p = torch.arange(total)
        vals = v[table[s, p // PAGE].long(), p % PAGE]
        odd = torch.where(torch.isfinite(vals), torch.zeros_like(vals), vals).float()
        for i in range(n):
            pos = total - n + i
            hi, lo = (pos + 1 if causal else total), (max(0, pos - window + 1) if window else 0)
            add = odd[lo:hi].sum(0).to(want.dtype)[:, None]
            want[starts[s] + i] = torch.where(torch.isfinite(add), want[starts[s] + i], add)
    return want.view(out0.shape)


@pytest.mark.parametrize("new,total,decode", BLOCKS + [([260], [700], False), ([70, 1, 33], [70, 400, 3000], False)])
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("hkv", [1, 4, 8])
def test_attention_values_that_are_not_finite(new, total, decode, dtype, d, hkv):
    """Infinities and NaN among the values: seen by every row, by some, behind the lengths, in several columns."""
    from b200ar.ops.paged import paged_attention

    q, k, v, batch = _inputs(new, total, decode, dtype, d, 8, hkv)
    g = torch.Generator().manual_seed(5)
    for s, t in enumerate(total):
        for value in (INF, -INF, NAN, INF):
            for p in {0, t - 1, max(t - new[s] // 2 - 1, 0), *torch.randint(t, (3,), generator=g).tolist()}:
                pg, slot = _slot(batch, s, p)
                head, column = (int(torch.randint(top, (1,), generator=g)) for top in (hkv, d))
                v[pg, slot, head, column] = value
        end = torch.arange(t, -(-t // PAGE) * PAGE)
        v[batch.page_table.cpu()[s, end // PAGE].long(), end % PAGE] = NAN
    clean = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    for kw in ({}, {"window": 1}, {"window": 50}, {"window": 300}, {"causal": False}):
        want = _settled(paged_attention(q, k, clean, batch, **kw), v, batch, 8, hkv, d, **kw)
        out = paged_attention(q, k, v, batch, **kw)
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        assert torch.equal(out.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))


@pytest.mark.parametrize("decode", [True, False])
def test_attention_nan_before_a_long_context(decode):
    """What a NaN costs does not grow with rows times positions: every wait ends in time, and the sequences beside
    it are what they were."""
    from b200ar.ops.paged import paged_attention

    new, total = ([1, 1, 1], [90, 120000, 3000]) if decode else ([40, 600, 1, 9], [90, 120000, 3000, 9])
    q, k, v, batch = _inputs(new, total, decode, BF, 128)
    clean = paged_attention(q, k, v, batch).view(-1, 8, 128)
    pg, slot = _slot(batch, 1, 0)
    v[pg, slot, 0, 5] = NAN
    out = paged_attention(q, k, v, batch).view(-1, 8, 128)
    sees = slice(new[0], new[0] + new[1])
    assert torch.isnan(out[sees, :, 5]).all()
    out[sees, :, 5] = clean[sees, :, 5]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("new,total,decode", BLOCKS)
def test_attention_large_values_within_the_type(new, total, decode):
    """Values of 2^114 under weights that sum up to 6000, below 2^13: in range as long as none counts more than 1."""
    from b200ar.ops.paged import paged_attention

    q, k, v, batch = _inputs(new, total, decode, BF, 128)
    # Pages of different sizes, so that the bound on a row's maximum moves.
    k.mul_(torch.linspace(0.01, 3, k.shape[0], device="cuda").to(BF)[:, None, None, None])
    small = paged_attention(q, k, v.sign(), batch)
    assert torch.equal(paged_attention(q, k, v.sign() * 2.0 ** 114, batch), small * 2.0 ** 114)


# ------------------------------------------------------------------ 8-bit linear
# On 148 SMs a K block of 256 x 256 outputs is a unit, and from 888 units on a call of over 128 rows takes CTA pairs.
FEW = [(3, 264, 512), (17, 264, 512), (40, 264, 512), (100, 264, 512), (200, 264, 512)]
MANY = [(300, 4096, 8192)]


def _linear_inputs(m, n, k, x_scale, w_scale):
    from b200ar.ops.fp8 import quantize_fp8, quantize_fp8_weight

    x = (randn((m, k), torch.float32, "cuda", 1) * x_scale).to(BF)
    w = randn((n, k), torch.float32, "cuda", 2) * w_scale
    return (x, *quantize_fp8(x), *quantize_fp8_weight(w))


def _check_linear(out, x_q, x_s, w_q, w_s):
    """check_linear's bound, whose smallest rounding step also covers sums of subnormal fp32 numbers: 64 blocks are
    off by 64 2^-149, far below u 2^-126."""
    from serving_util import check_linear

    assert torch.isfinite(out).all()
    check_linear(out, x_q, x_s, w_q, w_s)


@pytest.mark.parametrize("m,n,k", FEW)
def test_linear_fp8_large_activations_few_rows(m, n, k):
    """Activations of 1e36 against weights of 0.02: sums of 1e36 are in the type, sums of codes times x's scales not."""
    from b200ar.ops.fp8 import linear_fp8

    size = torch.ones(m, 1, device="cuda")
    size[::2] = 1e36
    x, x_q, x_s, w_q, w_s = _linear_inputs(m, n, k, size, 0.02)
    _check_linear(linear_fp8(x, w_q, w_s), x_q, x_s, w_q, w_s)
    _check_linear(linear_fp8(x_q, w_q, w_s, x_scale=x_s), x_q, x_s, w_q, w_s)


def _tiny_and_zero(m, n, k):
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8_weight

    # Scales whose product is below fp32 (1e-45), sums of K products of 1e-40 that are not.
    x, x_q, x_s, w_q, w_s = _linear_inputs(m, n, k, 1e-20, 1e-20)
    x, x_q = x.abs(), x_q.float().abs().to(x_q.dtype)
    w_q = w_q.float().abs().to(w_q.dtype)
    _check_linear(linear_fp8(x, w_q, w_s), x_q, x_s, w_q, w_s)
    # Scales whose product is above fp32, and products of zero.
    x[:, ::2] = 0
    w = randn((n, k), torch.float32, "cuda", 2, 1e16)
    w[:, 1::2] = 0
    w_q, w_s = quantize_fp8_weight(w)
    assert (linear_fp8((x.float() * 1e36 * 1e20).to(BF), w_q, w_s) == 0).all()


@pytest.mark.parametrize("m,n,k", FEW)
def test_linear_fp8_scales_at_the_ends_of_fp32_few_rows(m, n, k):
    _tiny_and_zero(m, n, k)


@pytest.mark.parametrize("m,n,k", MANY)
def test_linear_fp8_large_activations_many_rows(m, n, k):
    test_linear_fp8_large_activations_few_rows(m, n, k)


@pytest.mark.parametrize("m,n,k", MANY)
def test_linear_fp8_scales_at_the_ends_of_fp32_many_rows(m, n, k):
    _tiny_and_zero(m, n, k)


@pytest.mark.parametrize("rows,k", [(3, 48), (5, 384)])
def test_quantize_fp8_blocks_whose_scale_is_below_fp32(rows, k):
    """amax / 448 rounds to 0 up to 224 2^-149, and to 2^-149 above: no code is NaN, those of zeros are zero."""
    from b200ar.ops.fp8 import quantize_fp8, quantize_fp8_weight

    step = 2.0 ** -149
    for top, scale in ((1, 1.0), (224, 1.0), (225, step), (448, step)):
        x = torch.zeros(rows, k, device="cuda")
        x[0, 1], x[0, 2], x[rows - 1, k - 1] = top * step, -step, -top * step
        codes, scales = quantize_fp8(x)
        codes_w, scales_w = quantize_fp8_weight(x)
        want = torch.where(x == 0, torch.zeros_like(x), (x.double() / scale).clamp(-448, 448).float())
        want = want.to(torch.float8_e4m3fn).float()
        assert torch.equal(codes.float(), want) and torch.equal(codes_w.float(), want)
        assert scales[0, 0] == scale and scales[rows - 1, -1] == scale and (scales[1:-1] == 1).all()
        assert scales_w[0, 0] == scale


def test_rope_refuses_pools_that_share_memory():
    """Shifted views of one buffer are refused, views that lie between each other taken."""
    from serving_pools import rope_on_pools

    rope_on_pools("cuda")


def test_linear_fp8_refuses_an_output_over_an_input():
    from serving_pools import linear_over_inputs

    linear_over_inputs("cuda")


def test_attention_refuses_heads_between_units_of_64_values():
    from serving_pools import attention_on_padded_heads

    attention_on_padded_heads("cuda")
