"""Layouts of key and value pools in one buffer, for the tests on both devices."""

import pytest
import torch

from serving_util import make_batch, randn

PAGES, PAGE, HKV, D = 6, 16, 2, 64


def _views(device):
    """(name, k, v, whether they are apart) of one buffer each."""
    def buf(*shape):
        return torch.zeros(*shape, dtype=torch.bfloat16, device=device)

    pages = buf(PAGES, 2, PAGE, HKV, D)
    yield "in each page", pages[:, 0], pages[:, 1], True
    pages = buf(PAGES, 2, PAGE, HKV, D)
    yield "value first", pages[:, 1], pages[:, 0], True
    halves = buf(2 * PAGES, PAGE, HKV, D)
    yield "one behind the other", halves[:PAGES], halves[PAGES:], True
    halves = buf(2 * PAGES, PAGE, HKV, D)
    yield "every other page", halves[::2], halves[1::2], True
    tokens = buf(PAGES, PAGE, 2, HKV, D)
    yield "in each token", tokens[:, :, 0], tokens[:, :, 1], True
    heads = buf(PAGES, PAGE, HKV, 2, D)
    yield "in each head", heads[:, :, :, 0], heads[:, :, :, 1], True
    hnd = buf(PAGES, 2, HKV, PAGE, D)
    yield "heads first", hnd[:, 0].transpose(1, 2), hnd[:, 1].transpose(1, 2), True
    mixed = buf(PAGES, 2 * PAGE * HKV * D)
    half = PAGE * HKV * D
    yield ("two orders", mixed[:, :half].unflatten(1, (PAGE, HKV, D)),
           mixed[:, half:].unflatten(1, (HKV, PAGE, D)).transpose(1, 2), True)
    yield "the same", pages[:, 0], pages[:, 0], False
    yield "a page further", halves[:-1], halves[1:], False
    yield "a page back", halves[1:], halves[:-1], False
    yield "half a page further", *(halves.flatten()[o:o + PAGES * half].view(PAGES, PAGE, HKV, D)
                                   for o in (0, half // 2)), False
    wide = buf(PAGES, PAGE, HKV + 1, D)
    yield "a head further in one buffer", wide[:, :, :HKV], wide[:, :, 1:], False
    long = buf(PAGES, PAGE + 1, HKV, D)
    yield "a token further in one buffer", long[:, :PAGE], long[:, 1:], False


def rope_on_pools(device):
    from b200ar.ops.layers import RotaryTable
    from b200ar.ops.paged import qk_norm_rope_paged

    rot = RotaryTable(D, 64, 1e4, device)
    batch, _ = make_batch([20, 1], [30, 9], PAGE, device)
    qkv = randn((21, (2 + 2 * HKV) * D), torch.bfloat16, device, 1)
    want = None
    for name, k, v, apart in _views(device):
        if not apart:
            with pytest.raises(ValueError, match="share memory"):
                qk_norm_rope_paged(qkv, batch, rot, k, v, 2, HKV)
            continue
        q = qk_norm_rope_paged(qkv, batch, rot, k, v, 2, HKV)
        got = (q, k[:PAGES].clone(), v[:PAGES].clone())
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name


def linear_over_inputs(device):
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight

    x = randn((32, 256), torch.bfloat16, device, 1)
    w_q, w_s = quantize_fp8_weight(randn((16, 256), torch.bfloat16, device, 2))
    x_q, x_s = quantize_fp8(x)
    out = torch.zeros(32, 2 * 256, dtype=torch.bfloat16, device=device)
    scale = out.view(torch.float32)[:, 8:10]  # bytes 32 to 40 of a row of 1024
    scale.copy_(x_s)
    want = linear_fp8(x, w_q, w_s)
    assert torch.equal(linear_fp8(x_q, w_q, w_s, x_scale=scale), want)
    codes = out.view(torch.float8_e4m3fn)[:, :256]
    with pytest.raises(ValueError):
        linear_fp8(x_q, w_q, w_s, out=out[:, 16:32], x_scale=scale)
    with pytest.raises(ValueError):
        linear_fp8(codes, w_q, w_s, out=out[:, 256:272], x_scale=x_s)
    with pytest.raises(ValueError):
        linear_fp8(x, w_q, w_s, out=x[:, :16])
    assert torch.equal(scale, x_s)


def attention_on_padded_heads(device):
    """Heads d + 64 values apart are read, d + 8 apart refused before anything runs; a single head has no distance."""
    from b200ar.ops.paged import paged_attention

    batch, pool = make_batch([2, 1], [30, 9], PAGE, device)
    q = randn((3, 4, D), torch.bfloat16, device, 1)
    k, v = (randn((pool, PAGE, HKV, D), torch.bfloat16, device, i) for i in (2, 3))
    want = paged_attention(q, k, v, batch)

    def padded(t, by):
        wide = torch.zeros(*t.shape[:3], D + by, dtype=t.dtype, device=device)
        wide[..., :D] = t
        return wide[..., :D]

    assert torch.equal(paged_attention(q, padded(k, 64), padded(v, 64), batch), want)
    for a, b in ((padded(k, 8), v), (k, padded(v, 8))):
        with pytest.raises(ValueError, match="64 values apart"):
            paged_attention(q, a, b, batch)
    one = paged_attention(q, k[:, :, :1], v[:, :, :1], batch)
    assert torch.equal(paged_attention(q, padded(k, 8)[:, :, :1], padded(v, 8)[:, :, :1], batch), one)
