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
