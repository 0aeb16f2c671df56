"""Serving operators on CPU tensors at the limits of their types."""

import pytest
import torch

from serving_util import make_batch, randn

NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_scores_and_values_that_are_not_finite(dtype):
    """What the GPU tests of the same calls expect: NaN for rows whose scores are all -inf or hold a NaN, zeros for
    rows that see nothing, and infinities of v whatever their weight."""
    from b200ar.ops.paged import PagedBatch, paged_attention

    batch, pool = make_batch([3], [10], 8, "cpu")
    q = randn((3, 2, 64), dtype, "cpu", 1).abs() + 0.1
    k, v = (randn((pool, 8, 1, 64), dtype, "cpu", i) for i in (2, 3))
    slots = [(int(batch.page_table[0, p // 8]), p % 8) for p in range(10)]
    clean = paged_attention(q, k, v, batch).view(3, 2, 64)
    low = k.clone()
    low.fill_(-INF)
    assert torch.isnan(paged_attention(q, low, v, batch)).all()
    first = PagedBatch(batch.page_table, torch.ones(1, dtype=torch.int32), batch.q_start)  # rows 0, 1 before position 0
    out = paged_attention(q, low, v, first)
    assert (out[:2] == 0).all() and torch.isnan(out[2]).all()
    bad = k.clone()
    bad[slots[8]][0, 3] = NAN
    out = paged_attention(q, bad, v, batch).view(3, 2, 64)
    assert torch.equal(out[0], clean[0]) and torch.isnan(out[1:]).all()
    odd = v.clone()
    odd[slots[0]][0, 5], odd[slots[9]][0, 6], odd[slots[1]][0, 7], odd[slots[2]][0, 7] = INF, -INF, INF, -INF
    far = k.clone()
    far[slots[0]] = -60.0  # a weight of 0 in fp32
    out = paged_attention(q, far, odd, batch).view(3, 2, 64)
    assert (out[:, :, 5] == INF).all() and (out[2, :, 6] == -INF).all() and torch.isnan(out[:, :, 7]).all()
    assert torch.isfinite(out[:2, :, 6]).all() and torch.isfinite(out[:, :, :5]).all()


@pytest.mark.parametrize("rows,k", [(3, 48), (5, 384)])
def test_quantize_fp8_blocks_whose_scale_is_below_fp32(rows, k):
    """amax / 448 rounds to 0 up to 224 2^-149, and to 2^-149 above: no code is NaN, those of zeros are zero."""
    from b200ar.ops.fp8 import quantize_fp8, quantize_fp8_weight

    step = 2.0 ** -149
    for top, scale in ((1, 1.0), (224, 1.0), (225, step), (448, step)):
        x = torch.zeros(rows, k)
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

    rope_on_pools("cpu")


def test_linear_fp8_refuses_an_output_over_an_input():
    from serving_pools import linear_over_inputs

    linear_over_inputs("cpu")


def test_attention_refuses_heads_between_units_of_64_values():
    from serving_pools import attention_on_padded_heads

    attention_on_padded_heads("cpu")


def test_error_texts_name_the_operator():
    from b200ar.ops import gemm

    old = dict(gemm._ERR)
    try:
        for code, text in ((1, "GEMM"), (2, "paged_attention.*bounded wait"), (3, "rotary table"), (4, "no page"),
                           (5, "linear_fp8.*bounded wait"), (9, "error 9 on cuda:0")):
            gemm._ERR.clear()
            gemm._ERR[0] = torch.tensor([code], dtype=torch.int32)
            with pytest.raises(RuntimeError, match=text):
                gemm.check_errors()
    finally:
        gemm._ERR.clear()
        gemm._ERR.update(old)
