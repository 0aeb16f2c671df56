"""Serving operators on the instances that prompts run: the 8-bit product for
many rows, the rotary step with several heads a thread, attention of prompts in
each type and head width."""

import pytest
import torch

from serving_util import (check_attention, check_linear, check_rope, make_batch, plain_quantize, plain_rope, randn,
                          starts_of)

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _no_reported_errors():
    yield
    from b200ar.ops.gemm import check_errors

    torch.cuda.synchronize()
    check_errors()


# Parts of the line of K blocks with whole tiles, tiles cut in two (both orders of arrival) and in three, several tiles
# of rows and of columns, remainders in each direction; on 148 SMs 74 parts of 14 to 48 K blocks.
PAIR = [(2050, 4104, 2064), (700, 3592, 2832), (257, 16392, 1040), (1030, 2568, 4096), (4100, 1032, 4112)]


@pytest.mark.parametrize("m,n,k", PAIR)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_fp8_many_rows(m, n, k, dtype):
    from b200ar._native import _C
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight

    assert _C.linear_fp8_takes_pairs(m, n, k)
    x, w = randn((m, k), dtype, "cuda", 1), randn((n, k), dtype, "cuda", 2, 0.02)
    x[m // 2, :16] = 0
    w_q, w_s = quantize_fp8_weight(w)
    x_q, x_s = quantize_fp8(x)
    out = linear_fp8(x, w_q, w_s)
    check_linear(out, x_q, x_s, w_q, w_s)
    for _ in range(20):  # whichever pair finishes a tile, the sums have one order
        assert torch.equal(linear_fp8(x, w_q, w_s), out)
    wide = torch.full((m, n + 8), 7.0, dtype=dtype, device="cuda")
    assert torch.equal(linear_fp8(x_q, w_q, w_s, x_scale=x_s, dtype=dtype, out=wide[:, :n]), out)
    assert (wide[:, n:] == 7).all()


def test_linear_fp8_few_rows_stay_few():
    """The cases of the other tests that are meant for the kernel for few rows."""
    from b200ar._native import _C

    for m, n, k in ((128, 7168, 8192), (200, 264, 512), (300, 520, 1024), (333, 1288, 1040), (1025, 1280, 2048)):
        assert not _C.linear_fp8_takes_pairs(m, n, k)
    for m, n, k in ((129, 8192, 8192), (300, 4096, 8192), (257, 3592, 7184)):
        assert _C.linear_fp8_takes_pairs(m, n, k)


def test_linear_fp8_many_rows_in_graphs_and_on_streams():
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight

    m, n, k = 700, 3592, 2832
    x = [randn((m, k), BF, "cuda", i) for i in (1, 2)]
    w = [quantize_fp8_weight(randn((n, k), BF, "cuda", i)) for i in (3, 4)]
    codes = [quantize_fp8(t) for t in x]
    out = [linear_fp8(x[i], *w[i]) for i in range(2)]
    want = [o.clone() for o in out]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(3):
                linear_fp8(x[i], *w[i], out=out[i])
            given = linear_fp8(codes[i][0], *w[i], x_scale=codes[i][1])
        graphs.append((g, given))
    streams = [torch.cuda.Stream() for _ in range(2)]
    eager = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            out[i].zero_()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graphs[i][0].replay()
                eager[i].append(linear_fp8(x[i], *w[i]))
            torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(out[i], want[i]) and torch.equal(graphs[i][1], want[i])
        assert all(torch.equal(e, want[i]) for e in eager[i])


def test_linear_fp8_many_rows_on_two_streams_at_once():
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8_weight

    m, n, k = 700, 3592, 2832
    x = [randn((m, k), BF, "cuda", i) for i in (1, 2)]
    w = [quantize_fp8_weight(randn((n, k), BF, "cuda", i)) for i in (3, 4)]
    want = [linear_fp8(x[i], *w[i]) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(linear_fp8(x[i], *w[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_linear_fp8_many_rows_extremes():
    """Rows of NaN and infinities leave the others as they are; blocks whose scales span many orders."""
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight

    m, n, k = 700, 3592, 2832
    x = randn((m, k), BF, "cuda", 1)
    w_q, w_s = quantize_fp8_weight(randn((n, k), BF, "cuda", 2))
    clean = linear_fp8(x, w_q, w_s)
    odd = x.clone()
    odd[1, 300], odd[300, 7], odd[699, 511] = float("nan"), float("inf"), -float("inf")
    out = linear_fp8(odd, w_q, w_s)
    keep = [i for i in range(m) if i not in (1, 300, 699)]
    assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[[1, 300, 699]]).all()
    steps = (10.0 ** torch.linspace(-30, 3, -(-k // 128), device="cuda")).repeat_interleave(128)[:k]
    x = (x * steps).to(BF)
    x[0] = 0
    x_q, x_s = quantize_fp8(x)
    codes, scales = plain_quantize(x)
    assert torch.equal(x_q.double().cpu(), codes) and torch.equal(x_s.double().cpu(), scales)
    out = linear_fp8(x, w_q, w_s)
    check_linear(out, x_q, x_s, w_q, w_s)
    assert not out[0].any()


@pytest.mark.parametrize("m,k", [(1, 16), (5, 400), (600, 272)])
def test_quantize_fp8_of_fp32(m, k):
    from b200ar.ops.fp8 import quantize_fp8, quantize_fp8_weight

    x = torch.randn(m, k, generator=torch.Generator().manual_seed(1)) * torch.logspace(-20, 20, k)
    x[m // 2, :16] = 0
    x = x.cuda()
    for t in (x, torch.cat([x, x], 1)[:, 8:8 + k]):  # rows that start between 16-byte boundaries, too
        codes, scales = quantize_fp8(t)
        want = plain_quantize(t)
        assert torch.equal(codes.double().cpu(), want[0]) and torch.equal(scales.double().cpu(), want[1])
        codes, scales = quantize_fp8_weight(t)
        want = plain_quantize(t, 128)
        assert torch.equal(codes.double().cpu(), want[0]) and torch.equal(scales.double().cpu(), want[1])


# From 512 rows on a thread of the rotary step has up to three heads: two from 33 heads of 128 or 65 of 64, three from
# 65 or 129, and from 97 or 193 a row takes two blocks.
HEADS = [(30, 4, 128), (43, 1, 128), (56, 4, 128), (64, 8, 128), (80, 10, 128), (64, 8, 64), (101, 7, 64),
         (128, 16, 64), (160, 20, 64)]


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("dtype,norm", [(BF, True), (HF, False)])
def test_rope_paged_of_prompts(hq, hkv, d, dtype, norm):
    from b200ar.ops.layers import RotaryTable
    from b200ar.ops.paged import qk_norm_rope_paged

    new, total, page = [300, 0, 1, 211, 5], [300, 7, 40, 600, 5], 24
    batch, pool = make_batch(new, total, page, "cuda")
    rows = sum(new) + 2
    qkv = randn((rows, (hq + 2 * hkv) * d), dtype, "cuda", 1)
    k, v = (randn((pool, page, hkv, d), dtype, "cuda", i) for i in (2, 3))
    gq, gk = (randn((d,), dtype, "cuda", i) if norm else None for i in (4, 5))
    want = plain_rope(qkv, batch, 500000.0, d, (k, v), hq, hkv, gq, gk)
    rot = RotaryTable(d, 600, 500000.0, "cuda")
    q = torch.full((rows, hq, d), 9.0, dtype=dtype, device="cuda")
    before = q.clone()
    k2, v2, kept = k.clone(), v.clone(), qkv.clone()
    qk_norm_rope_paged(qkv, batch, rot, k, v, hq, hkv, gq, gk, q_out=q)
    check_rope(q, k, v, want, before)
    assert torch.equal(qkv, kept)
    own = qkv[:, :hq * d].unflatten(1, (hq, d))  # in place: the same values
    qk_norm_rope_paged(qkv, batch, rot, k2, v2, hq, hkv, gq, gk, q_out=own)
    used = sum(new)
    assert torch.equal(own[:used], q[:used]) and torch.equal(k2, k) and torch.equal(v2, v)
    assert torch.equal(qkv[used:], kept[used:]) and torch.equal(qkv[:, hq * d:], kept[:, hq * d:])


@pytest.mark.parametrize("new,total,page,hq,hkv", [
    ([128], [128], 16, 1, 1), ([16, 17], [16, 200], 64, 8, 1), ([1, 33, 0, 7, 260], [300, 33, 50, 8, 261], 16, 8, 2),
    ([5, 3], [3, 0], 16, 4, 2), ([257], [1300], 48, 4, 2), ([3, 2], [130, 500], 32, 96, 1), ([600], [600], 64, 2, 2),
    ([300], [5000], 128, 8, 1)])
@pytest.mark.parametrize("dtype,d", [(HF, 128), (BF, 64)])
def test_attention_of_prompts(new, total, page, hq, hkv, dtype, d):
    from b200ar.ops.paged import paged_attention

    batch, pool = make_batch(new, total, page, "cuda")
    rows = starts_of(new)[-1] + 3
    q = randn((rows, hq, d), dtype, "cuda", 1)
    k, v = (randn((pool, page, hkv, d), dtype, "cuda", i) for i in (2, 3))
    for kw in ({}, {"window": 1}, {"window": 70}, {"causal": False}, {"scale": 0.3}):
        out = torch.full((rows, hq * d), 7.0, dtype=dtype, device="cuda")
        paged_attention(q, k, v, batch, out=out, **kw)
        check_attention(out, q, k, v, batch, **kw)
        assert (out[-3:] == 7).all()
