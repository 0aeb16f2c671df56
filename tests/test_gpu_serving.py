"""Serving operators on the GPU against plain 64-bit implementations."""

import pytest
import torch

from serving_util import (check_attention, check_linear, check_rope, make_batch, plain_quantize, plain_rope, randn,
                          refuse_attention, refuse_linear_fp8, refuse_rope, starts_of)

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


def _attention_inputs(new, total, page, hq, hkv, d, dtype, seed=0, pad=0, decode=False):
    batch, pool = make_batch(new, total, page, "cuda", decode=decode, seed=seed)
    rows = starts_of(new)[-1] + pad
    q = randn((rows, hq, d), dtype, "cuda", seed + 1)
    k, v = (randn((pool, page, hkv, d), dtype, "cuda", seed + i) for i in (2, 3))
    return q, k, v, batch


def test_refusals():
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8_weight
    from b200ar.ops.paged import PagedBatch, paged_attention

    refuse_rope("cuda")
    refuse_attention("cuda")
    refuse_linear_fp8("cuda")
    # Tensors of two devices.
    q, k, v, batch = _attention_inputs([2], [20], 16, 4, 1, 64, BF)
    there = PagedBatch(batch.page_table.cpu(), batch.kv_len.cpu(), batch.q_start.cpu())
    w_q, w_s = quantize_fp8_weight(torch.zeros(16, 32, dtype=BF))
    for f in (lambda: paged_attention(q, k, v, there), lambda: paged_attention(q, k.cpu(), v.cpu(), batch),
              lambda: paged_attention(q.cpu(), k, v, there), lambda: linear_fp8(q[0, :, :32], w_q, w_s)):
        with pytest.raises(ValueError):
            f()


# ------------------------------------------------------------------ attention
DECODE = [
    # lengths, page, hq, hkv
    ([1], 16, 8, 1), ([2], 8, 4, 4), ([0], 16, 8, 1), ([127, 128, 129], 64, 8, 1), ([2049], 64, 8, 1),
    ([5, 0, 700, 1, 64], 24, 16, 2), ([300, 41], 256, 7, 1), ([33] * 9, 32, 32, 2), ([1000, 3], 48, 17, 1),
    ([255, 256, 257, 512], 128, 64, 8), ([90] * 40, 16, 12, 4), ([4100], 16, 16, 1), ([77, 130], 8, 130, 2),
]


@pytest.mark.parametrize("lens,page,hq,hkv", DECODE)
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 128), (BF, 64), (HF, 64)])
def test_attention_single_tokens(lens, page, hq, hkv, dtype, d):
    from b200ar.ops.paged import paged_attention

    q, k, v, batch = _attention_inputs([1] * len(lens), lens, page, hq, hkv, d, dtype, decode=True)
    check_attention(paged_attention(q, k, v, batch), q, k, v, batch)
    check_attention(paged_attention(q, k, v, batch, window=100), q, k, v, batch, window=100)


CHUNKS = [
    # new, total, page, hq, hkv
    ([2], [2], 16, 8, 1), ([128], [128], 16, 1, 1), ([129], [129], 8, 1, 1), ([16, 17], [16, 200], 64, 8, 1),
    ([100], [400], 24, 16, 2), ([1, 33, 0, 7, 260], [300, 33, 50, 8, 261], 16, 8, 2), ([5, 3], [3, 0], 16, 4, 2),
    ([40, 1, 1, 1], [40, 513, 1, 128], 256, 7, 1), ([257], [1300], 48, 4, 2), ([64, 64], [1024, 64], 128, 6, 3),
    ([3, 2], [130, 500], 32, 96, 1), ([2, 1], [140, 20], 16, 129, 1), ([600], [600], 64, 2, 2),
]


@pytest.mark.parametrize("new,total,page,hq,hkv", CHUNKS)
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)])
def test_attention_chunks(new, total, page, hq, hkv, dtype, d):
    from b200ar.ops.paged import paged_attention

    q, k, v, batch = _attention_inputs(new, total, page, hq, hkv, d, dtype, pad=3)
    for kw in ({}, {"window": 1}, {"window": 70}, {"causal": False}, {"scale": 0.3}):
        out = torch.full((q.shape[0], hq * d), 7.0, dtype=dtype, device="cuda")
        paged_attention(q, k, v, batch, out=out, **kw)
        check_attention(out, q, k, v, batch, **kw)
        assert (out[-3:] == 7).all()  # rows behind the last sequence


@pytest.mark.parametrize("new,total,hq,hkv", [([300], [5000], 8, 1), ([1] * 30 + [200], [900] * 30 + [2000], 16, 2)])
def test_attention_long_caches(new, total, hq, hkv):
    from b200ar.ops.paged import paged_attention

    q, k, v, batch = _attention_inputs(new, total, 64, hq, hkv, 128, BF)
    first = paged_attention(q, k, v, batch)
    check_attention(first, q, k, v, batch)
    assert torch.equal(paged_attention(q, k, v, batch), first)  # the order of sums is fixed


@pytest.mark.parametrize("decode", [True, False])
def test_attention_strides(decode):
    """Pools as views: keys and values in one buffer, heads before tokens; q inside a qkv product."""
    from b200ar.ops.paged import paged_attention

    new, total = ([1, 1, 1], [40, 300, 7]) if decode else ([3, 20, 1], [40, 300, 7])
    hq, hkv, d, page = 8, 2, 128, 16
    batch, pool = make_batch(new, total, page, "cuda", decode=decode)
    rows = sum(new)
    q = randn((rows, (hq + 2 * hkv) * d), BF, "cuda", 1)[:, :hq * d].unflatten(1, (hq, d))
    both = randn((pool, 2, page, hkv, d), BF, "cuda", 2)
    check_attention(paged_attention(q, both[:, 0], both[:, 1], batch), q, both[:, 0], both[:, 1], batch)
    hnd = randn((2, pool, hkv, page, d), BF, "cuda", 3).transpose(2, 3)
    wide = torch.full((rows, hq * d + 64), 5.0, dtype=BF, device="cuda")
    out = paged_attention(q, hnd[0], hnd[1], batch, out=wide[:, :hq * d])
    check_attention(out.contiguous(), q, hnd[0], hnd[1], batch)
    assert (wide[:, hq * d:] == 5).all()


@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("decode", [True, False])
def test_attention_hides_what_it_must(decode, dtype, d):
    """NaN and infinities behind the lengths, in pages that nobody owns, before
    the window and at positions that only later rows see."""
    from b200ar.ops.paged import paged_attention

    new, total = ([1, 1, 1], [5, 130, 200]) if decode else ([4, 70, 1], [5, 130, 200])
    page, window = 16, 90
    q, k, v, batch = _attention_inputs(new, total, page, 8, 2, d, dtype, decode=decode)
    clean = {w: paged_attention(q, k, v, batch, window=w) for w in (0, window)}
    table = batch.page_table.cpu()
    owned = torch.zeros(k.shape[0], page, dtype=torch.bool)
    for s, t in enumerate(total):
        p = torch.arange(t)
        owned[table[s, p // page].long(), p % page] = True
    nan, inf = float("nan"), float("inf")
    hidden = (~owned).cuda()
    k[hidden], v[hidden] = nan, inf
    for w in (0, window):
        assert torch.equal(paged_attention(q, k, v, batch, window=w), clean[w])
    # Before the window of every row of sequence 2 nothing is read, not even the table.
    gone = total[2] - new[2] - window + 1
    k2, v2, t2 = k.clone(), v.clone(), batch.page_table.clone()
    p = torch.arange(gone)
    k2[table[2, p // page].long(), p % page] = nan
    v2[table[2, p // page].long(), p % page] = -inf
    t2[2, :gone // page] = -1
    from b200ar.ops.paged import PagedBatch
    assert torch.equal(paged_attention(q, k2, v2, PagedBatch(t2, batch.kv_len, batch.q_start), window=window),
                       clean[window])
    if decode:
        return
    # Position 100 of sequence 1 (rows 4 + 40 and later see it) holds an infinite value, 101 a NaN.
    k3, v3 = k.clone(), v.clone()
    v3[int(table[1, 100 // page]), 100 % page, 0, 3] = inf
    k3[int(table[1, 101 // page]), 101 % page, 1, 3] = nan
    out = paged_attention(q, k3, v3, batch).view(-1, 8, d)
    want = clean[0].view(-1, 8, d)
    assert torch.isinf(out[4 + 40:-1, :4, 3]).all() and torch.isnan(out[4 + 41:-1, 4:]).all()
    out[4 + 40:-1, :4, 3] = want[4 + 40:-1, :4, 3]
    out[4 + 41:-1, 4:] = want[4 + 41:-1, 4:]
    k[hidden], v[hidden] = 0, 0
    check_attention(out, q, k, v, batch)


@pytest.mark.parametrize("decode", [True, False])
def test_attention_scores_of_any_size(decode):
    """Scores far outside the range of exp, equal ones, and rows whose largest score comes last."""
    from b200ar.ops.paged import paged_attention

    new, total = ([1, 1], [300, 129]) if decode else ([20, 5], [300, 129])
    q, k, v, batch = _attention_inputs(new, total, 16, 4, 1, 128, BF, decode=decode)
    k.mul_(torch.linspace(0.1, 1, k.shape[0], device="cuda").to(BF)[:, None, None, None])
    check_attention(paged_attention(q, k, v, batch, scale=0.0), q, k, v, batch, scale=0.0)
    check_attention(paged_attention(q, k, v, batch, scale=-0.05), q, k, v, batch, scale=-0.05)
    # One position far above the rest: its value is the answer.
    table = batch.page_table.cpu()
    k.zero_()
    q.fill_(16.0)
    pg = int(table[0, 280 // 16])
    k[pg, 280 % 16] = 16.0  # score 128 * 256 / sqrt(128) = 2896
    out = paged_attention(q, k, v, batch).view(-1, 4, 128)
    want = v[pg, 280 % 16, 0].expand(4, 128)
    row = 0 if decode else 1  # position 281 (299 for the single token)
    assert torch.equal(out[row], want)


@pytest.mark.parametrize("decode", [True, False])
def test_attention_graph_with_other_lengths(decode):
    """A captured call replayed with other lengths, offsets, pages and values; two graphs side by side."""
    from b200ar.ops.paged import PagedBatch, paged_attention

    hq, hkv, d, page, rows = 8, 2, 128, 16, 12
    if decode:
        cases = [([1] * 12, [40 + 9 * i for i in range(12)]), ([1] * 12, [700 - 50 * i for i in range(12)])]
    else:
        cases = [([3, 1, 0, 8], [30, 600, 9, 8]), ([1, 1, 1, 1], [1, 2, 3, 900]), ([9, 0, 1, 1], [700, 5, 1, 64])]
    seqs = len(cases[0][0])
    table = torch.full((seqs, 60), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    starts = None if decode else torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
    batch = PagedBatch(table, lens, starts)
    pool = 480
    q = [randn((rows, hq, d), BF, "cuda", i) for i in (1, 2)]
    k, v = (randn((pool, page, hkv, d), BF, "cuda", i) for i in (3, 4))
    out = [torch.zeros(rows, hq * d, dtype=BF, device="cuda") for _ in range(2)]

    def fill(case, seed):
        b, _ = make_batch(*case, page, "cuda", decode=decode, seed=seed)
        table.fill_(-1)
        w = min(60, b.page_table.shape[1])
        table[:, :w] = b.page_table[:, :w]
        lens.copy_(b.kv_len)
        if starts is not None:
            starts.copy_(b.q_start)

    fill(cases[0], 0)
    graphs = []
    for i in range(2):
        paged_attention(q[i], k, v, batch, out=out[i])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            paged_attention(q[i], k, v, batch, out=out[i])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for seed, case in enumerate(cases):
        fill(case, seed)
        for o in out:
            o.fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            check_attention(out[i], q[i], k, v, batch)
            assert (out[i][sum(case[0]):] == 7).all()


def test_attention_on_two_streams():
    from b200ar.ops.paged import paged_attention

    jobs = [_attention_inputs([1, 30, 2], [900, 500, 2], 16, 8, 2, 128, BF, seed=10 * i) for i in range(2)]
    want = [paged_attention(*j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(*jobs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_attention_offsets_past_32_bits():
    """A pool of more than 2^32 elements, the cached pages at its end."""
    from b200ar.ops.paged import PagedBatch, paged_attention

    page, hkv, d = 128, 8, 128
    pool = (2**32 // (page * hkv * d)) + 64
    k = torch.zeros(pool, page, hkv, d, dtype=BF, device="cuda")
    small, ids = 6, torch.randperm(6).to(torch.int32)
    k[-small:] = randn((small, page, hkv, d), BF, "cuda", 1)
    ks = k[-small:].clone()
    for new, decode in (([1, 1], True), ([40, 1], False)):
        total = [300, 290]
        q = randn((sum(new), 16, d), BF, "cuda", 2)
        table = ids.view(2, 3).cuda()
        lens = torch.tensor(total, dtype=torch.int32, device="cuda")
        starts = None if decode else torch.tensor(starts_of(new), dtype=torch.int32, device="cuda")
        out = paged_attention(q, k, k, PagedBatch(table + (pool - small), lens, starts))
        check_attention(out, q, ks, ks, PagedBatch(table, lens, starts))
    del k
    torch.cuda.empty_cache()


@pytest.mark.parametrize("decode", [True, False])
def test_attention_reports_missing_pages(decode):
    from b200ar.ops.gemm import check_errors
    from b200ar.ops.paged import PagedBatch, paged_attention

    new = [1, 1] if decode else [2, 3]
    q, k, v, batch = _attention_inputs(new, [40, 70], 16, 4, 1, 64, BF, decode=decode)
    good = paged_attention(q, k, v, batch)
    torch.cuda.synchronize()
    check_errors()
    for bad in (-1, k.shape[0], 2**31 - 1, -2**31):
        table = batch.page_table.clone()
        table[1, 1] = bad
        out = paged_attention(q, k, v, PagedBatch(table, batch.kv_len, batch.q_start))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="no page"):
            check_errors()
        assert torch.equal(out[:new[0]], good[:new[0]])
    # A length behind the table's last column.
    lens = batch.kv_len.clone()
    lens[1] = 16 * batch.page_table.shape[1] + 5
    out = paged_attention(q, k, v, PagedBatch(batch.page_table, lens, batch.q_start))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="no page"):
        check_errors()
    assert torch.equal(out[:new[0]], good[:new[0]])


def test_offsets_outside_the_rows_are_cut():
    """Offsets behind the inputs (or before them) lead to no row that is not there."""
    from b200ar.ops.layers import RotaryTable
    from b200ar.ops.paged import PagedBatch, paged_attention, qk_norm_rope_paged

    q, k, v, batch = _attention_inputs([2, 3], [40, 70], 16, 4, 1, 64, BF)
    qkv, rot = randn((5, 6 * 64), BF, "cuda", 9), RotaryTable(64, 128, 1e4, "cuda")
    for starts, cut in (([0, 2, 900], [0, 2, 5]), ([0, 2, 2**31 - 1], [0, 2, 5]), ([-7, 2, 5], [0, 2, 5]),
                        ([0, 2**31 - 1, 2**31 - 1], [0, 5, 5]), ([9, 9, 9], [5, 5, 5])):
        outs = []
        for s in (starts, cut):
            b = PagedBatch(batch.page_table, batch.kv_len, torch.tensor(s, dtype=torch.int32, device="cuda"))
            kp, vp, out, q_out = k.clone(), v.clone(), torch.full_like(q, 3).flatten(1), torch.full_like(q, 3)
            qk_norm_rope_paged(qkv, b, rot, kp, vp, 4, 1, q_out=q_out)
            outs.append((paged_attention(q, k, v, b, out=out), kp, vp, q_out))
        assert all(torch.equal(x, y) for x, y in zip(*outs))


@pytest.mark.parametrize("decode", [True, False])
def test_many_sequences(decode):
    """More sequences than a block of the schedule has threads, and than two searches of 32 cover."""
    from b200ar.ops.layers import RotaryTable
    from b200ar.ops.paged import paged_attention, qk_norm_rope_paged

    new = [1 if decode else (5 * i) % 3 for i in range(1500)]
    total = [n + (7 * i) % 50 for i, n in enumerate(new)]
    q, k, v, batch = _attention_inputs(new, total, 8, 4, 1, 64, BF, decode=decode)
    check_attention(paged_attention(q, k, v, batch), q, k, v, batch)
    qkv, rot = randn((sum(new), 6 * 64), BF, "cuda", 7), RotaryTable(64, 64, 1e4, "cuda")
    out = torch.zeros_like(q)
    want = plain_rope(qkv, batch, 1e4, 64, (k, v), 4, 1, None, None)
    qk_norm_rope_paged(qkv, batch, rot, k, v, 4, 1, q_out=out)
    check_rope(out, k, v, want, torch.zeros_like(q))


def test_attention_of_nothing():
    from b200ar.ops.paged import PagedBatch, paged_attention

    q, k, v, batch = _attention_inputs([2], [2], 16, 4, 1, 64, BF)
    assert paged_attention(q[:0], k, v, PagedBatch(batch.page_table[:0], batch.kv_len[:0])).shape == (0, 256)
    empty = PagedBatch(batch.page_table[:0], batch.kv_len[:0], torch.zeros(1, dtype=torch.int32, device="cuda"))
    out = torch.full((2, 256), 3.0, dtype=BF, device="cuda")
    assert (paged_attention(q, k, v, empty, out=out) == 3).all()
    none = PagedBatch(batch.page_table, batch.kv_len, torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert (paged_attention(q, k, v, none, out=out) == 3).all()


# ------------------------------------------------------------------ rotary step
ROPE = [
    # new, total, page, hq, hkv, decode
    ([1], [2049], 64, 8, 1, True), ([1] * 5, [1, 9, 17, 8, 4000], 8, 64, 8, True), ([1, 1], [3, 4], 16, 7, 1, True),
    ([5], [5], 16, 8, 1, False), ([3, 0, 40, 1], [3, 11, 300, 77], 24, 12, 4, False), ([9, 2], [5, 0], 16, 4, 4, False),
    ([130, 1], [600, 1], 128, 5, 1, False), ([1] * 70, list(range(70, 0, -1)), 256, 2, 1, False),
]


@pytest.mark.parametrize("new,total,page,hq,hkv,decode", ROPE)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 128), (BF, 64), (HF, 64)])
def test_rope_paged(new, total, page, hq, hkv, decode, norm, dtype, d):
    from b200ar.ops.gemm import check_errors
    from b200ar.ops.layers import RotaryTable
    from b200ar.ops.paged import qk_norm_rope_paged

    batch, pool = make_batch(new, total, page, "cuda", decode=decode)
    rows = sum(new) + (0 if decode else 2)
    qkv = randn((rows, (hq + 2 * hkv) * d), dtype, "cuda", 1)
    k, v = (randn((pool, page, hkv, d), dtype, "cuda", i) for i in (2, 3))
    gq, gk = (randn((d,), dtype, "cuda", i) if norm else None for i in (4, 5))
    want = plain_rope(qkv, batch, 500000.0, d, (k, v), hq, hkv, gq, gk)
    rot = RotaryTable(d, max(total), 500000.0, "cuda")
    q = torch.full((rows, hq, d), 9.0, dtype=dtype, device="cuda")
    before = q.clone()
    kept = qkv.clone()
    qk_norm_rope_paged(qkv, batch, rot, k, v, hq, hkv, gq, gk, q_out=q)
    torch.cuda.synchronize()
    if any(n > t for n, t in zip(new, total)):  # tokens before their sequence: skipped and reported
        with pytest.raises(RuntimeError, match="rotary table"):
            check_errors()
    check_rope(q, k, v, want, before)
    assert torch.equal(qkv, kept)


def test_rope_paged_strides_and_in_place():
    from b200ar.ops.layers import RotaryTable
    from b200ar.ops.paged import qk_norm_rope_paged

    hq, hkv, d, page, new, total = 6, 2, 128, 16, [4, 9], [20, 9]
    batch, pool = make_batch(new, total, page, "cuda")
    wide = randn((13, (hq + 2 * hkv) * d + 64), BF, "cuda", 1)
    qkv = wide[:, :-64]
    both = randn((pool, 2, hkv, page, d), BF, "cuda", 2)
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    gq, gk = randn((d,), BF, "cuda", 4), randn((d,), BF, "cuda", 5)
    rot = RotaryTable(d, 32, 500000.0, "cuda")
    want = plain_rope(qkv, batch, 500000.0, d, (k, v), hq, hkv, gq, gk)
    tail, rest = wide[:, -64:].clone(), wide[:, hq * d:-64].clone()
    q = qkv[:, :hq * d].unflatten(1, (hq, d))
    before = q.clone()
    qk_norm_rope_paged(qkv, batch, rot, k, v, hq, hkv, gq, gk, q_out=q)
    check_rope(q, k, v, want, before)
    assert torch.equal(wide[:, -64:], tail) and torch.equal(wide[:, hq * d:-64], rest)


def test_rope_paged_skips_and_reports():
    from b200ar.ops.gemm import check_errors
    from b200ar.ops.layers import RotaryTable
    from b200ar.ops.paged import PagedBatch, qk_norm_rope_paged

    hq, hkv, d, page, new, total = 4, 1, 64, 16, [20, 3], [40, 40]
    batch, pool = make_batch(new, total, page, "cuda")
    rot = RotaryTable(d, 64, 500000.0, "cuda")
    qkv = randn((23, (hq + 2 * hkv) * d), BF, "cuda", 1)

    def run(b, r, match):
        k, v = (randn((pool, page, hkv, d), BF, "cuda", i) for i in (2, 3))
        want = plain_rope(qkv, b, 500000.0, d, (k, v), hq, hkv, max_pos=r.cos.shape[0])
        q = torch.full((23, hq, d), 9.0, dtype=BF, device="cuda")
        before = q.clone()
        qk_norm_rope_paged(qkv, b, r, k, v, hq, hkv, q_out=q)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match=match):
            check_errors()
        check_rope(q, k, v, want, before)

    for bad in (-1, pool, 2**31 - 1, -2**31):
        table = batch.page_table.clone()
        table[0, 2] = bad
        run(PagedBatch(table, batch.kv_len, batch.q_start), rot, "no page")
    run(PagedBatch(batch.page_table[:, :2], batch.kv_len, batch.q_start), rot, "no page")
    run(batch, RotaryTable(d, 39, 500000.0, "cuda"), "rotary table")


def test_rope_paged_far_positions_and_large_pools():
    from b200ar.ops.layers import RotaryTable
    from b200ar.ops.paged import PagedBatch, qk_norm_rope_paged

    hq, hkv, d, page = 8, 8, 128, 64
    pool = (2**32 // (page * hkv * d)) + 8
    k = torch.zeros(pool, page, hkv, d, dtype=BF, device="cuda")
    v = torch.zeros_like(k)
    pos = 131071
    table = torch.full((1, (pos + page) // page), -1, dtype=torch.int32)
    table[0, pos // page] = pool - 1
    batch = PagedBatch(table.cuda(), torch.tensor([pos + 1], dtype=torch.int32).cuda())
    qkv = randn((1, (hq + 2 * hkv) * d), BF, "cuda", 1)
    q = qk_norm_rope_paged(qkv, batch, RotaryTable(d, pos + 1, 500000.0, "cuda"), k, v, hq, hkv)
    table[0, pos // page] = 0
    small = PagedBatch(table, batch.kv_len.cpu())
    zero = torch.zeros(1, page, hkv, d, dtype=BF)
    want = plain_rope(qkv, small, 500000.0, d, (zero, zero), hq, hkv)
    check_rope(q, k[-1:], v[-1:], want, q)
    assert not k[0].any() and not v[pool // 2].any()
    del k, v
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ 8-bit linear
SHAPES = [(1, 8, 16), (1, 7168, 1024), (3, 136, 144), (16, 256, 128), (17, 264, 400), (48, 8192, 512), (64, 1280, 2048),
          (65, 512, 272), (128, 128, 128), (129, 392, 656), (333, 1288, 1040), (513, 1024, 384), (1000, 72, 48),
          (140, 7168, 4096), (257, 3592, 7184), (900, 2056, 2832), (1025, 1280, 2048)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_fp8(m, n, k, dtype):
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight

    x = randn((m, k), dtype, "cuda", 1)
    w = randn((n, k), dtype, "cuda", 2, 0.02)
    x[m // 2, :16] = 0
    w_q, w_s = quantize_fp8_weight(w)
    want_q, want_s = plain_quantize(w, 128)
    assert torch.equal(w_q.double().cpu(), want_q) and torch.equal(w_s.double().cpu(), want_s)
    x_q, x_s = quantize_fp8(x)
    want_q, want_s = plain_quantize(x)
    assert torch.equal(x_q.double().cpu(), want_q) and torch.equal(x_s.double().cpu(), want_s)
    out = linear_fp8(x, w_q, w_s)
    assert out.dtype == dtype
    check_linear(out, x_q, x_s, w_q, w_s)
    assert torch.equal(linear_fp8(x, w_q, w_s), out)
    assert torch.equal(linear_fp8(x_q, w_q, w_s, x_scale=x_s.contiguous(), dtype=dtype), out)


def test_linear_fp8_long_sums():
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight

    for m, n, k in ((2, 128, 28672), (300, 256, 28672), (300, 1024, 28672)):
        x, w = randn((m, k), BF, "cuda", 1).abs(), randn((n, k), BF, "cuda", 2).abs()
        w_q, w_s = quantize_fp8_weight(w)
        check_linear(linear_fp8(x, w_q, w_s), *quantize_fp8(x), w_q, w_s)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("order", ["sorted", "mixed", "exact"])
def test_quantize_fp8_every_value(dtype, order):
    """All finite 16-bit values: codes are those of the rounded quotient, ties between two codes included."""
    from b200ar.ops.fp8 import quantize_fp8, quantize_fp8_weight

    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[torch.isfinite(x)]
    if order == "mixed":
        x = x[torch.randperm(x.numel(), generator=torch.Generator().manual_seed(1))]
    elif order == "exact":  # a largest value of 448: the scale is 1, and the values themselves lie on the middles
        x = x[x.abs() <= 448]
        x = x[: x.numel() // 127 * 127].view(-1, 127)
        x = torch.cat([x, torch.full((x.shape[0], 1), 448.0, dtype=dtype)], 1).flatten()
    x = x[: x.numel() // 512 * 512].view(-1, 512)
    blocks = x.float().view(x.shape[0], 4, 128)
    top = blocks.abs().amax(-1)
    scale = torch.where(top > 0, top / 448.0, torch.ones_like(top))
    want = (blocks / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(x.shape)
    codes, got = quantize_fp8(x.cuda())
    assert torch.equal(got.cpu(), scale)
    assert torch.equal(codes.cpu().float(), want.float())
    n = x.shape[0] // 128 * 128
    tiles = x[:n].float().view(-1, 128, 4, 128)
    top = tiles.abs().amax((1, 3))
    scale = torch.where(top > 0, top / 448.0, torch.ones_like(top))
    want = (tiles / scale[:, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(n, 512)
    codes, got = quantize_fp8_weight(x[:n].cuda())
    assert torch.equal(got.cpu(), scale)
    assert torch.equal(codes.cpu().float(), want.float())


@pytest.mark.parametrize("m", [3, 40, 200])
def test_linear_fp8_scales_of_all_sizes(m):
    """Blocks whose scales span many orders, zero blocks, and the extremes of the types."""
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight

    k, n = 1024, 136
    x = randn((m, k), BF, "cuda", 1) * (10.0 ** torch.linspace(-30, 3, k // 128, device="cuda")).repeat_interleave(128)
    x = x.to(BF)
    x[0] = 0
    x[1, :128] = torch.finfo(BF).tiny * 2.0 ** -6
    w = randn((n, k), torch.float32, "cuda", 2)
    w[:128, 256:384] = 0
    w_q, w_s = quantize_fp8_weight(w)
    assert torch.equal(w_q.double().cpu(), plain_quantize(w, 128)[0])
    x_q, x_s = quantize_fp8(x)
    want_q, want_s = plain_quantize(x)
    assert torch.equal(x_q.double().cpu(), want_q) and torch.equal(x_s.double().cpu(), want_s)
    out = linear_fp8(x, w_q, w_s)
    check_linear(out, x_q, x_s, w_q, w_s)
    assert not out[0].any()


@pytest.mark.parametrize("m", [4, 200])
def test_linear_fp8_non_finite_rows(m):
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8_weight

    x = randn((m, 512), BF, "cuda", 1)
    w_q, w_s = quantize_fp8_weight(randn((264, 512), BF, "cuda", 2))
    clean = linear_fp8(x, w_q, w_s)
    x[1, 300], x[2, 7], x[3, 511] = float("nan"), float("inf"), -float("inf")
    out = linear_fp8(x, w_q, w_s)
    keep = [i for i in range(m) if i not in (1, 2, 3)]
    assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[1:4]).all()


def test_linear_fp8_strides_and_views():
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight

    w_q, w_s = quantize_fp8_weight(randn((264, 256), BF, "cuda", 2))
    base = randn((2, 50, 512), BF, "cuda", 1)
    for x in (base[..., :256], base[..., 8:264], base[..., 3:259], base[:, ::2, :256],
              base[0, :, :256].t().contiguous().t()):
        plain = x.contiguous().view(-1, 256)
        want = linear_fp8(plain, w_q, w_s)
        assert torch.equal(linear_fp8(x, w_q, w_s).view(-1, 264), want)
        codes, scale = quantize_fp8(x)
        assert codes.shape == x.shape and scale.shape == (*x.shape[:-1], 2)
        assert torch.equal(linear_fp8(codes, w_q, w_s, x_scale=scale).view(-1, 264), want)
    one = linear_fp8(base[0, 0, :256], w_q, w_s)
    assert one.shape == (264,) and torch.equal(one, linear_fp8(base[0, :1, :256], w_q, w_s)[0])
    assert linear_fp8(base[:, :0, :256], w_q, w_s).shape == (2, 0, 264)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_fp8_in_graphs_and_on_streams(m):
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8_weight

    k, n = 1024, 520
    x = [randn((m, k), BF, "cuda", i) for i in (1, 2)]
    w = [quantize_fp8_weight(randn((n, k), BF, "cuda", i)) for i in (3, 4)]
    out = [linear_fp8(x[i], *w[i]) for i in range(2)]
    want = [o.clone() for o in out]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(3):
                linear_fp8(x[i], *w[i], out=out[i])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    eager = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            out[i].zero_()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graphs[i].replay()
                eager[i].append(linear_fp8(x[i], *w[i]))
            torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(out[i], want[i]) and all(torch.equal(e, want[i]) for e in eager[i])


# ------------------------------------------------------------------ together
def test_serving_step_of_all_operators():
    """Two chunks of prompts, then single tokens: 8-bit projections, the rotary
    step and attention over the same pages, against 64-bit attention over
    everything that was written."""
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight
    from b200ar.ops.layers import RotaryTable, rmsnorm
    from b200ar.ops.paged import PagedBatch, paged_attention, qk_norm_rope_paged

    H, hq, hkv, d, page = 512, 8, 2, 64, 16
    wqkv, wo = (quantize_fp8_weight(randn(s, BF, "cuda", i, 0.05)) for i, s in
                enumerate((((hq + 2 * hkv) * d, H), (H, hq * d))))
    gq, gk, gn = (1 + randn((n,), BF, "cuda", 9 + i, 0.1) for i, n in enumerate((d, d, H)))
    rot = RotaryTable(d, 256, 500000.0, "cuda")
    pool = 20
    k, v = (torch.full((pool, page, hkv, d), float("nan"), dtype=BF, device="cuda") for _ in range(2))
    table = torch.randperm(pool)[:16].view(2, 8).to(torch.int32).cuda()
    lens = [0, 0]
    for step, new in enumerate(([20, 50], [33, 2], [1, 1], [1, 1])):
        lens = [a + b for a, b in zip(lens, new)]
        starts = torch.tensor(starts_of(new), dtype=torch.int32, device="cuda")
        batch = PagedBatch(table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                           None if max(new) == 1 else starts)
        x = randn((sum(new), H), BF, "cuda", 20 + step)
        h = rmsnorm(x, gn)
        codes, scale = quantize_fp8(h)
        qkv = linear_fp8(codes, *wqkv, x_scale=scale)
        check_linear(qkv, codes, scale, *wqkv)
        want = plain_rope(qkv, batch, 500000.0, d, (k.nan_to_num(), v.nan_to_num()), hq, hkv, gq, gk)
        q = qk_norm_rope_paged(qkv, batch, rot, k, v, hq, hkv, gq, gk)
        check_rope(q, k.nan_to_num(), v.nan_to_num(), want, q)
        a = paged_attention(q, k, v, batch)
        check_attention(a, q, k, v, batch)
        y = linear_fp8(a, *wo)
        check_linear(y, *quantize_fp8(a), *wo)
