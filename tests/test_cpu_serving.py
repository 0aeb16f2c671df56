"""Serving operators on CPU tensors: the fp32 reference math against plain
64-bit implementations, the refusals, and a serving step made of them."""

import pytest
import torch

from serving_util import (check_attention, check_linear, check_rope, make_batch, plain_quantize, plain_rope, randn,
                          refuse_attention, refuse_linear_fp8, refuse_rope, starts_of)

BATCHES = [
    ([1], [1], 16), ([1, 1, 1], [1, 37, 0], 8), ([5, 1, 0, 9], [5, 30, 12, 20], 24), ([3, 4], [2, 4], 16),
]


@pytest.mark.parametrize("new,total,page", BATCHES)
@pytest.mark.parametrize("window", [0, 1, 7])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_attention_reference(new, total, page, window, dtype, d):
    from b200ar.ops.paged import paged_attention

    batch, pool = make_batch(new, total, page, "cpu")
    rows = starts_of(new)[-1] + 2
    q = randn((rows, 4, d), dtype, "cpu", 1)
    k, v = (randn((pool, page, 2, d), dtype, "cpu", i) for i in (2, 3))
    out = torch.full((rows, 4 * d), 9.0, dtype=dtype)
    paged_attention(q, k, v, batch, window=window, out=out)
    check_attention(out, q, k, v, batch, window=window)
    assert (out[-2:] == 9).all()
    if not window:
        check_attention(paged_attention(q, k, v, batch, causal=False), q, k, v, batch, causal=False)


def test_attention_reference_hides_non_finite_values():
    from b200ar.ops.paged import paged_attention

    batch, pool = make_batch([4], [10], 8, "cpu")
    q = randn((4, 2, 64), torch.bfloat16, "cpu", 1)
    k, v = (randn((pool, 8, 1, 64), torch.bfloat16, "cpu", i) for i in (2, 3))
    clean = paged_attention(q, k, v, batch)
    page = int(batch.page_table[0, 1])
    k[page, 1, 0, 3], v[page, 1, 0, 5] = float("nan"), float("inf")  # position 9: row 3 alone sees it
    k[page, 2:], v[page, 2:] = float("nan"), float("inf")           # behind the sequence
    out = paged_attention(q, k, v, batch)
    assert torch.equal(out[:3], clean[:3])
    assert torch.isnan(out[3]).all()


@pytest.mark.parametrize("new,total,page", BATCHES)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_rope_reference(new, total, page, norm, dtype, d):
    from b200ar.ops.layers import RotaryTable
    from b200ar.ops.paged import qk_norm_rope_paged

    hq, hkv = 4, 2
    batch, pool = make_batch(new, total, page, "cpu")
    rows = starts_of(new)[-1] + 1
    qkv = randn((rows, (hq + 2 * hkv) * d), dtype, "cpu", 1)
    k, v = (randn((pool, page, hkv, d), dtype, "cpu", i) for i in (2, 3))
    gq, gk = (randn((d,), dtype, "cpu", i) if norm else None for i in (4, 5))
    q = torch.full((rows, hq, d), 9.0, dtype=dtype)
    before = q.clone()
    want = plain_rope(qkv, batch, 500000.0, d, (k, v), hq, hkv, gq, gk, max_pos=64)
    qk_norm_rope_paged(qkv, batch, RotaryTable(d, 64, 500000.0, "cpu"), k, v, hq, hkv, gq, gk, q_out=q)
    check_rope(q, k, v, want, before)


@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (3, 136, 144), (9, 128, 128), (130, 264, 400)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_fp8_reference(m, n, k, dtype):
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight

    x, w = randn((m, k), dtype, "cpu", 1), randn((n, k), torch.float32, "cpu", 2, 0.02)
    x[0, :16] = 0
    w_q, w_s = quantize_fp8_weight(w)
    want_q, want_s = plain_quantize(w, 128)
    assert torch.equal(w_q.double(), want_q) and torch.equal(w_s.double(), want_s)
    x_q, x_s = quantize_fp8(x)
    want_q, want_s = plain_quantize(x)
    assert torch.equal(x_q.double(), want_q) and torch.equal(x_s.double(), want_s)
    out = linear_fp8(x, w_q, w_s)
    assert out.dtype == dtype
    check_linear(out, x_q, x_s, w_q, w_s)
    assert torch.equal(linear_fp8(x_q, w_q, w_s, x_scale=x_s, dtype=dtype), out)
    out3 = torch.empty(m, 1, n, dtype=dtype)
    assert torch.equal(linear_fp8(x.view(m, 1, k), w_q, w_s, out=out3).view(m, n), out)


def test_linear_fp8_blocks_with_nothing_and_with_non_finite_values():
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight

    x = randn((4, 256), torch.bfloat16, "cpu", 1)
    x[0, :128] = 0
    x[1] = 0
    x[2, 5], x[3, 200] = float("nan"), float("inf")
    codes, scale = quantize_fp8(x)
    assert scale[0, 0] == 1 and (scale[1] == 1).all() and not codes[1].float().any()
    w_q, w_s = quantize_fp8_weight(randn((8, 256), torch.bfloat16, "cpu", 2))
    out = linear_fp8(x, w_q, w_s)
    assert torch.isfinite(out[:2]).all() and (out[1] == 0).all() and torch.isnan(out[2:]).all()


def test_batch_refusals():
    from b200ar.ops.paged import PagedBatch

    t, l, s = (torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
               torch.zeros(3, dtype=torch.int32))
    PagedBatch(t, l, s)
    for args in ((t.long(), l, s), (t[0], l, s), (t.t(), l, s), (t, l.long(), s), (t, l[:1], s), (t, l, s[:2]),
                 (t, l, s.float()), (t, l, torch.zeros(6, dtype=torch.int32)[::2]),
                 (t, l, torch.zeros(3, dtype=torch.int32, device="meta"))):
        with pytest.raises(ValueError):
            PagedBatch(*args)


def test_refusals():
    refuse_rope("cpu")
    refuse_attention("cpu")
    refuse_linear_fp8("cpu")


def test_error_texts():
    from b200ar.ops import gemm

    old = dict(gemm._ERR)
    try:
        for code, text in ((1, "bounded wait"), (3, "rotary table"), (4, "no page")):
            gemm._ERR.clear()
            gemm._ERR[0] = torch.tensor([code], dtype=torch.int32)
            with pytest.raises(RuntimeError, match=text):
                gemm.check_errors()
            gemm.check_errors()
    finally:
        gemm._ERR.clear()
        gemm._ERR.update(old)


def test_offsets_outside_the_rows_are_cut():
    from b200ar.ops.paged import PagedBatch, paged_attention

    batch, pool = make_batch([2, 3], [40, 70], 16, "cpu")
    q, k, v = (randn(s, torch.bfloat16, "cpu", i) for i, s in enumerate([(5, 4, 64)] + [(pool, 16, 1, 64)] * 2))
    want = paged_attention(q, k, v, batch)
    for starts in ([0, 2, 900], [-7, 2, 5]):
        cut = PagedBatch(batch.page_table, batch.kv_len, torch.tensor(starts, dtype=torch.int32))
        assert torch.equal(paged_attention(q, k, v, cut), want)
