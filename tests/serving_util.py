"""Plain 64-bit implementations of the serving operators, one row at a time,
and the batches that their tests use.

Error bounds. One rounding to nearest of y is off by u max(|y|, t): u = eps / 2
of the type, t its smallest normal number, below which the steps stay the same.

* rotary step: fp32 inside. Two products and a sum of values with at most four
  roundings each, and table entries rounded once: below 2^-20 of |a| + |b|.
  Then one rounding.
* attention: the weights p are rounded to the type before they meet v, at most
  u A with A = sum p |v| / sum p, and the output is rounded once. Scores
  are fp32 sums of d products, d 2^-24 scale sum |q k|, which is below 2^-13
  for the inputs used here, and enter numerator and denominator: 2^-12 A.
* 8-bit product: products are exact; a block of 128 is four sums of 32 in at
  least 23 bits below their largest term and each of the K / 128 blocks is
  scaled and added in fp32: below 2^-17 of sum |x w| for K up to 8192. Then one rounding.
"""

import math

import pytest
import torch

from b200ar.ops.paged import PagedBatch


def unit(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def rounding(y, dtype):
    """Bound on the error of one rounding of y to the type."""
    return unit(dtype) * y.abs().clamp(min=torch.finfo(dtype).smallest_normal)


def starts_of(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def make_batch(new, total, page, device, spare=2, decode=False, seed=0, extra_cols=1):
    """A batch with its pages in random order; unused entries hold -1. Returns
    (batch, number of pages)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(t, 0) // page) for t in total]
    pool = sum(need) + spare
    ids = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((len(new), max(need, default=0) + extra_cols), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(need):
        table[s, :c] = ids[at:at + c]
        at += c
    return PagedBatch(table.to(device), torch.tensor(total, dtype=torch.int32, device=device),
                      None if decode else torch.tensor(starts_of(new), dtype=torch.int32, device=device)), pool


def randn(shape, dtype, device, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype).to(device)


def _row_starts(batch):
    s = batch.sequences
    return list(range(s + 1)) if batch.q_start is None else batch.q_start.tolist()


def plain_attention(q, k_pages, v_pages, batch, scale=None, causal=True, window=0):
    """(o, A) in fp64 [rows, hq, d], NaN in rows behind the last sequence; A is
    the mean of |v| under the same weights."""
    rows, hq, d = q.shape
    hkv = k_pages.shape[2]
    page_size = k_pages.shape[1]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    q, kp, vp = q.double().cpu(), k_pages.double().cpu(), v_pages.double().cpu()
    table, lens, starts = batch.page_table.cpu(), batch.kv_len.tolist(), _row_starts(batch)
    o = torch.full((rows, hq, d), float("nan"), dtype=torch.float64)
    a = torch.zeros_like(o)
    for s, total in enumerate(lens):
        n = starts[s + 1] - starts[s]
        for i in range(n):
            pos = total - n + i
            hi = pos + 1 if causal else total
            lo = max(0, pos - window + 1) if window else 0
            row = starts[s] + i
            if hi <= lo:
                o[row] = 0
                continue
            p = torch.arange(lo, hi)
            pg = table[s, p // page_size].long()
            k = kp[pg, p % page_size].repeat_interleave(hq // hkv, 1)
            v = vp[pg, p % page_size].repeat_interleave(hq // hkv, 1)
            w = torch.softmax(torch.einsum("hd,phd->hp", q[row], k) * scale, -1)
            o[row] = torch.einsum("hp,phd->hd", w, v)
            a[row] = torch.einsum("hp,phd->hd", w, v.abs())
    return o, a


def check_attention(out, q, k_pages, v_pages, batch, **kw):
    want, avg = plain_attention(q, k_pages, v_pages, batch, **kw)
    got = out.view(q.shape).double().cpu()
    used = ~torch.isnan(want).flatten(1).all(1)
    bound = rounding(want, q.dtype) + (unit(q.dtype) + 2.0 ** -12) * avg
    err = (got - want).abs()[used]
    worst = (err / bound[used]).max().item() if err.numel() else 0.0
    assert torch.isfinite(got[used]).all()
    assert worst <= 1.0, f"error {worst:.3f} of the bound"


def plain_rope(qkv, batch, theta, d, pools, hq, hkv, q_gamma=None, k_gamma=None, eps=1e-5, max_pos=1 << 30):
    """fp64 (q, k pool, v pool, size of the inputs of each rotation like q and like the k pool)."""
    x = qkv.double().cpu().view(qkv.shape[0], -1, d)
    kp, vp = pools[0].double().cpu().clone(), pools[1].double().cpu().clone()
    page_size = kp.shape[1]
    q_out = torch.full((x.shape[0], hq, d), float("nan"), dtype=torch.float64)
    q_mag, k_mag = torch.zeros_like(q_out), torch.zeros_like(kp)
    table, lens, starts = batch.page_table.cpu(), batch.kv_len.tolist(), _row_starts(batch)
    for s, total in enumerate(lens):
        n = starts[s + 1] - starts[s]
        for i in range(n):
            pos, row = total - n + i, starts[s] + i
            if pos < 0 or pos >= max_pos or pos // page_size >= table.shape[1]:
                continue
            pg = int(table[s, pos // page_size])
            if pg < 0 or pg >= kp.shape[0]:
                continue
            ang = torch.tensor([pos * theta ** (-2.0 * j / d) for j in range(d // 2)], dtype=torch.float64)
            c, sn = ang.cos(), ang.sin()

            def turn(t, gamma):
                if gamma is not None:
                    t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * gamma.double().cpu()
                a, b = t[:, :d // 2], t[:, d // 2:]
                return torch.cat([a * c - b * sn, a * sn + b * c], -1), torch.cat([a.abs() + b.abs()] * 2, -1)

            q_out[row], q_mag[row] = turn(x[row, :hq], q_gamma)
            kp[pg, pos % page_size], k_mag[pg, pos % page_size] = turn(x[row, hq:hq + hkv], k_gamma)
            vp[pg, pos % page_size] = x[row, hq + hkv:]
    return q_out, kp, vp, q_mag, k_mag


def check_rope(q, k_pages, v_pages, plain, q_before):
    want_q, want_k, want_v, q_mag, k_mag = plain
    skipped = torch.isnan(want_q).flatten(1).all(1)
    got_q = q.double().cpu()
    assert torch.equal(got_q[skipped], q_before.double().cpu()[skipped])  # rows that are not the call's
    for got, want, mag in ((got_q[~skipped], want_q[~skipped], q_mag[~skipped]),
                           (k_pages.double().cpu(), want_k, k_mag)):
        err = (got - want).abs()
        bound = torch.where(mag > 0, rounding(want, q.dtype) + 2.0 ** -20 * mag, torch.zeros_like(mag))
        assert (err <= bound).all(), (err - bound).max().item()
    assert torch.equal(v_pages.double().cpu(), want_v)


def plain_quantize(x, rows_per_scale=1):
    """Codes (as fp64 values) and scales by the formula, in fp64 but for the scale's own rounding to fp32."""
    x = x.double().cpu()
    m, k = x.shape
    kb, mb = -(-k // 128), -(-m // rows_per_scale)
    scale = torch.ones(mb, kb, dtype=torch.float64)
    codes = torch.zeros_like(x)
    for b in range(kb):
        for r in range(mb):
            blk = x[r * rows_per_scale:(r + 1) * rows_per_scale, b * 128:(b + 1) * 128]
            top = blk.abs().max()
            if top > 0:
                scale[r, b] = (top / 448.0).float().double()
            c = (blk / scale[r, b]).clamp(-448, 448)
            codes[r * rows_per_scale:(r + 1) * rows_per_scale, b * 128:(b + 1) * 128] = \
                c.float().to(torch.float8_e4m3fn).double()
    return codes, scale


def plain_linear(x_codes, x_scale, w_codes, w_scale):
    """(y, sum |x w|) in fp64 from codes and scales."""
    k, n = x_codes.shape[1], w_codes.shape[0]
    a = x_codes.double().cpu() * x_scale.double().cpu().repeat_interleave(128, 1)[:, :k]
    b = w_codes.double().cpu() * w_scale.double().cpu().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return a @ b.t(), a.abs() @ b.abs().t()


def check_linear(out, x_codes, x_scale, w_codes, w_scale):
    want, mag = plain_linear(x_codes, x_scale, w_codes, w_scale)
    got = out.double().cpu().view(want.shape)
    err = (got - want).abs()
    bound = rounding(want, out.dtype) + 2.0 ** -17 * mag
    assert (err <= bound).all(), (err - bound).max().item()


# ------------------------------------------------------------------ refusals
def _paged_setup(device, dtype=torch.bfloat16, d=64, hq=4, hkv=2, page=16):
    from b200ar.ops.layers import RotaryTable

    batch, pool = make_batch([2, 1], [5, 3], page, device)
    k, v = (torch.zeros(pool, page, hkv, d, dtype=dtype, device=device) for _ in range(2))
    return {"batch": batch, "k_pages": k, "v_pages": v, "rot": RotaryTable(d, 32, 500000.0, device),
            "qkv": torch.zeros(3, (hq + 2 * hkv) * d, dtype=dtype, device=device),
            "q": torch.zeros(3, hq, d, dtype=dtype, device=device)}


def _lapping(pool):
    """A pool of the same shape whose pages share half their tokens."""
    n, page, h, d = pool.shape
    return torch.zeros(n * page * h * d, dtype=pool.dtype, device=pool.device).as_strided(
        pool.shape, (page * h * d // 2, h * d, d, 1))


def refuse_rope(device):
    """Every call that the rotary step must refuse; the first two it must take."""
    from b200ar.ops.layers import RotaryTable
    from b200ar.ops.paged import PagedBatch, qk_norm_rope_paged

    a = _paged_setup(device)

    def call(**kw):
        b = {**a, **kw}
        return qk_norm_rope_paged(b["qkv"], b["batch"], b["rot"], b["k_pages"], b["v_pages"], b.get("hq", 4),
                                  b.get("hkv", 2), q_gamma=b.get("q_gamma"), k_gamma=b.get("k_gamma"),
                                  q_out=b.get("q_out"))

    assert call().shape == (3, 4, 64)
    own = a["qkv"][:, :256].view(3, 4, 64)
    assert call(q_out=own).data_ptr() == own.data_ptr()  # in place
    g = torch.ones(64, dtype=torch.bfloat16, device=device)
    bad = [dict(hq=5), dict(hkv=0), dict(qkv=a["qkv"][0]), dict(v_pages=a["v_pages"][1:]), dict(q_gamma=g),
           dict(q_gamma=g, k_gamma=g.float()), dict(q_gamma=g, k_gamma=g[:32]),
           dict(rot=RotaryTable(128, 8, 1e4, device)), dict(q_out=own[:2]), dict(q_out=own.float()),
           dict(q_out=a["qkv"][:, 64:320].view(3, 4, 64)),
           dict(q_out=torch.zeros(1, 4, 64, device=device).bfloat16().expand(3, 4, 64)),
           dict(batch=PagedBatch(a["batch"].page_table, a["batch"].kv_len)),
           dict(k_pages=a["k_pages"][:1].expand(5, 16, 2, 64), v_pages=a["v_pages"][:1].expand(5, 16, 2, 64)),
           dict(v_pages=a["k_pages"]), dict(k_pages=_lapping(a["k_pages"])),
           dict(q_out=torch.zeros(600, device=device).bfloat16().as_strided((3, 4, 64), (128, 64, 1))),
           dict(q_out=a["v_pages"].flatten()[:768].view(3, 4, 64)),
           dict(qkv=a["k_pages"].flatten()[:1536].view(3, 512))]
    for kw in bad:
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(k_pages=a["k_pages"].float(), v_pages=a["v_pages"].float()), dict(qkv=a["qkv"].half()),
               dict(qkv=a["qkv"].float(), k_pages=a["k_pages"].float(), v_pages=a["v_pages"].float())):
        with pytest.raises(TypeError):
            call(**kw)


def refuse_attention(device):
    from b200ar.ops.paged import PagedBatch, paged_attention

    a = _paged_setup(device)

    def call(**kw):
        b = {**a, **kw}
        return paged_attention(b["q"], b["k_pages"], b["v_pages"], b["batch"], scale=b.get("scale"),
                               causal=b.get("causal", True), window=b.get("window", 0), out=b.get("out"))

    assert call().shape == (3, 256)
    for kw in (dict(q=a["q"][0]), dict(q=torch.zeros(3, 3, 64, device=device).bfloat16()),
               dict(q=torch.zeros(3, 4, 32, device=device).bfloat16()),
               dict(window=-1), dict(window=4, causal=False), dict(scale=float("nan")),
               dict(out=torch.zeros(3, 255, device=device).bfloat16()), dict(out=torch.zeros(3, 256, device=device)),
               dict(out=a["q"].view(3, 256)), dict(out=torch.zeros(1, 256, device=device).bfloat16().expand(3, 256)),
               dict(out=torch.zeros(800, device=device).bfloat16().as_strided((3, 256), (128, 1))),
               dict(batch=PagedBatch(a["batch"].page_table, a["batch"].kv_len)),
               dict(k_pages=a["k_pages"][:, :12], v_pages=a["v_pages"][:, :12])):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(TypeError):
        call(q=a["q"].half())


def refuse_linear_fp8(device):
    from b200ar.ops.fp8 import linear_fp8, quantize_fp8, quantize_fp8_weight

    x, w = torch.zeros(3, 32, device=device).bfloat16(), torch.zeros(16, 32, device=device).bfloat16()
    w_q, w_s = quantize_fp8_weight(w)
    x_q, x_s = quantize_fp8(x)
    for f in (lambda: quantize_fp8(x[:, :20]), lambda: quantize_fp8_weight(w[0]),
              lambda: linear_fp8(x[:, :16], w_q, w_s),
              lambda: linear_fp8(x, w_q[:12], w_s), lambda: linear_fp8(x, w_q, w_s[:, :0]),
              lambda: linear_fp8(x, w_q, w_s.double()),
              lambda: linear_fp8(x, w_q, w_s, out=torch.zeros(3, 16, device=device)),
              lambda: linear_fp8(x, w_q, w_s, out=torch.zeros(3, 8, device=device).bfloat16()),
              lambda: linear_fp8(x_q, w_q, w_s, x_scale=x_s[:2])):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: quantize_fp8(x.long()), lambda: linear_fp8(x.float(), w_q, w_s), lambda: linear_fp8(x, w, w_s),
              lambda: linear_fp8(x, w_q, w_s, x_scale=x_s), lambda: linear_fp8(x_q, w_q, w_s),
              lambda: linear_fp8(x_q, w_q, w_s, x_scale=x_s, dtype=torch.float32)):
        with pytest.raises(TypeError):
            f()
