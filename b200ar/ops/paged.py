"""Serving ops on a paged KV cache (``csrc/paged``), for prompts, chunks of
prompts and single tokens in one call.

* ``PagedBatch``          which tokens a call holds, and where their cache is
* ``qk_norm_rope_paged``  norms of q and k for each head (optional), rotary
                          embedding, q to a buffer, k and v into the pages
* ``paged_attention``     attention of the new tokens over the pages

The cache of a layer is two pools ``[pages, page_size, kv_heads, d]`` (bf16 or
fp16, d 64 or 128) with contiguous heads that start on 16-byte boundaries and,
for ``paged_attention``, are a multiple of 64 values apart. They may be views of
one buffer ``[pages, 2, page_size, kv_heads, d]`` or of a pool that keeps heads
before tokens. Position p of sequence s lives in slot
``p % page_size`` of page ``page_table[s, p // page_size]``.

Lengths, offsets and page tables stay on the device: nothing is read back, so
both calls can be captured into a CUDA graph and replayed with other lengths.
What only the device sees is checked there: a page that is missing or outside
the pool, or a position outside the rotary table, is not accessed and reported
by ``b200ar.ops.gemm.check_errors``. The rotary step skips such a token; the
rows of attention that need such a page have no defined result.

CPU tensors run the fp32 reference math; CUDA tensors always run the kernels.
These ops have no backward pass.
"""

from __future__ import annotations

import dataclasses
import math
from typing import Optional

import torch

from .._native import _C
from .gemm import error_word
from .layers import RotaryTable

HEAD_DIMS = (64, 128)


@dataclasses.dataclass(frozen=True)
class PagedBatch:
    """The tokens of one call and their cache.

    Args:
        page_table: int32 ``[S, max_pages]``; entries behind a sequence's last
            page (and before a sliding window) are not read.
        kv_len: int32 ``[S]``, tokens of each sequence in the cache, the new
            ones of this call included.
        q_start: int32 ``[S + 1]``, ascending: rows ``q_start[s]`` to
            ``q_start[s + 1]`` of the call's inputs are the last tokens of
            sequence s. Rows from ``q_start[S]`` on are padding and left
            alone; offsets outside the rows are cut to them. None: one new
            token for each sequence (row s).

    Sequences may share pages (a common prefix) that no call writes while
    they do: of two new tokens with one slot, either's k and v may stay.
    """

    page_table: torch.Tensor
    kv_len: torch.Tensor
    q_start: Optional[torch.Tensor] = None

    def __post_init__(self):
        pt, kl, qs = self.page_table, self.kv_len, self.q_start
        if pt.dim() != 2 or pt.dtype != torch.int32 or (pt.shape[1] > 1 and pt.stride(1) != 1):
            raise ValueError("page_table must be int32 [sequences, pages] with contiguous rows")
        s = pt.shape[0]
        if kl.dtype != torch.int32 or tuple(kl.shape) != (s,) or not kl.is_contiguous():
            raise ValueError("kv_len must be int32 [sequences]")
        if qs is not None and (qs.dtype != torch.int32 or tuple(qs.shape) != (s + 1,) or not qs.is_contiguous()):
            raise ValueError("q_start must be int32 [sequences + 1]")
        if any(t is not None and t.device != pt.device for t in (kl, qs)):
            raise ValueError("page_table, kv_len and q_start must be on one device")
        if pt.is_cuda:
            error_word(pt.device)  # exists before a graph that uses it is captured

    @property
    def sequences(self) -> int:
        return self.page_table.shape[0]


def _check_pools(k_pages, v_pages, like, d):
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.shape[3] != d:
        raise ValueError("k_pages and v_pages must be [pages, page_size, kv_heads, d]")
    if k_pages.dtype != like.dtype or v_pages.dtype != like.dtype:
        raise TypeError(f"the pools must have the type of the input, {like.dtype}")
    if like.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"paged ops take bfloat16 or float16, got {like.dtype}")
    if d not in HEAD_DIMS:
        raise ValueError(f"head dimension must be one of {HEAD_DIMS}, got {d}")
    if k_pages.device != like.device or v_pages.device != like.device:
        raise ValueError(f"the pools must be on {like.device}")


def _check_batch(batch: PagedBatch, rows: int, device) -> None:
    if batch.page_table.device != device:
        raise ValueError(f"the batch is on {batch.page_table.device}, the tensors on {device}")
    if batch.q_start is None and rows != batch.sequences:
        raise ValueError(f"without q_start every sequence has one new token: {batch.sequences} sequences, {rows} rows")


def _overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors meet."""
    def span(t):
        if t.numel() == 0:
            return 0, 0
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether an element of ``a`` may be one of ``b``, of the same sizes and
    type. Dimension by dimension from the largest stride down: where both have
    the same, not below what the rest spans, only the two slices can meet whose
    distance is less than it. Other strides count as meeting."""
    dims = sorted(((sa, sb, n) for n, sa, sb in zip(a.shape, a.stride(), b.stride()) if n > 1), reverse=True)

    def meet(dims, at):
        span_a, span_b = (1 + sum((d[2] - 1) * d[i] for d in dims) for i in (0, 1))
        if at >= span_a or -at >= span_b:
            return False
        if not dims:
            return True
        stride, other, n = dims[0]
        if stride != other or stride < max(span_a, span_b) - (n - 1) * stride:
            return True
        steps, rest = divmod(at, stride)
        return (abs(steps) < n and meet(dims[1:], rest)) or (abs(steps + 1) < n and meet(dims[1:], rest - stride))

    at, odd = divmod(b.data_ptr() - a.data_ptr(), a.element_size())
    return a.numel() > 0 and _overlaps(a, b) and (odd != 0 or meet(dims, at))


def _shares_memory(t: torch.Tensor) -> bool:
    """Whether two indices of ``t`` may be one element."""
    span = 1
    for stride, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if stride < span:
            return True
        span += (n - 1) * stride
    return False


def qk_norm_rope_paged(qkv: torch.Tensor, batch: PagedBatch, rot: RotaryTable, k_pages: torch.Tensor,
                       v_pages: torch.Tensor, hq: int, hkv: int, q_gamma: Optional[torch.Tensor] = None,
                       k_gamma: Optional[torch.Tensor] = None, eps: float = 1e-5,
                       q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The rotary step between the QKV projection and ``paged_attention``.

    ``qkv`` [rows, (hq + 2 hkv) * d], heads ordered [q | k | v]. With
    ``q_gamma`` and ``k_gamma`` [d] every head of q and k is normed first,
    ``x * rsqrt(mean(x^2) + eps) * gamma``. q and k are rotated (rotate-half)
    by their position; q goes to ``q_out`` [rows, hq, d] (returned), k and v
    into the pages. ``q_out`` may be the q part of ``qkv`` itself
    (``qkv[:, :hq * d].view(rows, hq, d)``). fp32 inside, rounded once.
    A row whose position has no page, or is outside ``rot``, is skipped.
    """
    if qkv.is_cuda:  # checked there
        return _C.qk_norm_rope_paged(qkv, batch.page_table, batch.kv_len, batch.q_start, rot.cos, rot.sin, k_pages,
                                     v_pages, hq, hkv, q_gamma, k_gamma, q_out, error_word(qkv.device), eps)
    d = rot.head_dim
    if hq < 1 or hkv < 1:
        raise ValueError("hq and hkv must be positive")
    if qkv.dim() != 2 or qkv.shape[1] != (hq + 2 * hkv) * d:
        raise ValueError(f"qkv must be [rows, (hq + 2 hkv) * {d}]")
    _check_pools(k_pages, v_pages, qkv, d)
    if k_pages.shape[2] != hkv:
        raise ValueError(f"the pools hold {k_pages.shape[2]} heads, not {hkv}")
    rows = qkv.shape[0]
    _check_batch(batch, rows, qkv.device)
    if (q_gamma is None) != (k_gamma is None):
        raise ValueError("give the norm weights of both q and k, or neither")
    for g in (q_gamma, k_gamma):
        if g is not None and (tuple(g.shape) != (d,) or g.dtype != qkv.dtype or g.device != qkv.device):
            raise ValueError(f"the norm weights must be [{d}], of the type and on the device of qkv")
    if q_out is None:
        q_out = torch.empty(rows, hq, d, dtype=qkv.dtype, device=qkv.device)
    elif tuple(q_out.shape) != (rows, hq, d) or q_out.dtype != qkv.dtype or q_out.device != qkv.device:
        raise ValueError("q_out must be [rows, hq, d], of the type and on the device of qkv")
    in_place = q_out.data_ptr() == qkv.data_ptr() and q_out.stride()[:2] == (qkv.stride(0), d)
    if not in_place and _overlaps(q_out, qkv):
        raise ValueError("q_out overlaps qkv but is not its q part")
    for t, name in ((q_out, "q_out"), (k_pages, "k_pages"), (v_pages, "v_pages")):
        if t.numel() and _shares_memory(t):
            raise ValueError(f"{name} is written and its rows must not share memory")
    if _share_memory(k_pages, v_pages):
        raise ValueError("k_pages and v_pages share memory")
    if any(_overlaps(a, b) for a in (qkv, q_out) for b in (k_pages, v_pages)):
        raise ValueError("the pools overlap qkv or q_out")
    ref_qk_norm_rope_paged(qkv, batch, rot, k_pages, v_pages, hq, hkv, q_gamma, k_gamma, eps, q_out)
    return q_out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, batch: PagedBatch,
                    scale: Optional[float] = None, causal: bool = True, window: int = 0,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of new tokens ``q`` [rows, hq, d] over the pages, grouped
    queries included; returns [rows, hq * d].

    Row i of the n new rows of a sequence stands at position
    ``kv_len - n + i`` and sees the positions up to its own, with ``window``
    only the last ``window`` of them; with ``causal=False`` all ``kv_len``.
    A row that sees nothing gets zeros, one whose scores are all -inf or hold
    a NaN gets NaN. Where a row sees infinities or NaN in v, its columns there
    are their sum, whatever their weights. ``scale`` defaults to 1 / sqrt(d).
    Nothing behind a sequence's length, and nothing that a row's mask hides,
    reaches its output, whatever the pages hold there.
    """
    if q.is_cuda:  # checked there
        return _C.paged_attention(q, k_pages, v_pages, batch.page_table, batch.kv_len, batch.q_start, out,
                                  error_word(q.device), scale, causal, window)
    if q.dim() != 3:
        raise ValueError("q must be [rows, heads, d]")
    rows, hq, d = q.shape
    _check_pools(k_pages, v_pages, q, d)
    hkv = k_pages.shape[2]
    if k_pages.shape[1] % 8:
        raise ValueError(f"the page size must be a multiple of 8, got {k_pages.shape[1]}")
    if hkv < 1 or hq < 1 or hq % hkv:
        raise ValueError("query heads must be a multiple of the KV heads")
    if hkv > 1 and (k_pages.stride(2) % 64 or v_pages.stride(2) % 64):
        raise ValueError("the pools' heads must be a multiple of 64 values apart")
    _check_batch(batch, rows, q.device)
    if window < 0 or (window and not causal):
        raise ValueError("window must be 0 (all) or a number of positions, with causal attention")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if out is None:
        out = torch.empty(rows, hq * d, dtype=q.dtype, device=q.device)
    elif tuple(out.shape) != (rows, hq * d) or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must be [rows, hq * d], of the type and on the device of q")
    if out.numel() and _shares_memory(out):
        raise ValueError("out is written and its rows must not share memory")
    out3 = out.unflatten(1, (hq, d))
    for t, name in ((q, "q"), (k_pages, "k_pages"), (v_pages, "v_pages")):
        if _overlaps(out3, t):
            raise ValueError(f"out overlaps {name}")
    ref_paged_attention(q, k_pages, v_pages, batch, scale, causal, window, out3)
    return out


# ------------------------------------------------------------------ references
def _rows_of(batch: PagedBatch, rows: int):
    """(sequence, first row, rows, cached tokens) of every sequence."""
    lens = batch.kv_len.tolist()
    starts = list(range(len(lens) + 1)) if batch.q_start is None else batch.q_start.clamp(0, rows).tolist()
    return [(s, starts[s], max(starts[s + 1] - starts[s], 0), lens[s]) for s in range(len(lens))]


def _pages_of(batch: PagedBatch, s: int, pos: torch.Tensor, page_size: int, pages: int):
    """Pages of positions of one sequence; -1 where there is none."""
    idx = torch.div(pos, page_size, rounding_mode="floor")
    ok = (idx >= 0) & (idx < batch.page_table.shape[1])
    page = batch.page_table[s].long()[idx.clamp(0, max(batch.page_table.shape[1] - 1, 0))]
    return torch.where(ok & (page >= 0) & (page < pages), page, torch.full_like(page, -1))


def ref_qk_norm_rope_paged(qkv, batch, rot, k_pages, v_pages, hq, hkv, q_gamma, k_gamma, eps, q_out) -> None:
    """fp32 reference of ``qk_norm_rope_paged`` (any device; reads lengths back)."""
    d = rot.head_dim
    for s, first, n, total in _rows_of(batch, qkv.shape[0]):
        pos = torch.arange(total - n, total, device=qkv.device)
        page = _pages_of(batch, s, pos, k_pages.shape[1], k_pages.shape[0])
        ok = (pos >= 0) & (pos < rot.cos.shape[0]) & (page >= 0)
        rows = torch.arange(first, first + n, device=qkv.device)[ok]
        pos, page = pos[ok], page[ok]
        x = qkv[rows].float().view(-1, hq + 2 * hkv, d)

        def turned(t, gamma):
            if gamma is not None:
                t = t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps) * gamma.float()
            c, sn = rot.cos[pos][:, None], rot.sin[pos][:, None]
            a, b = t[..., :d // 2], t[..., d // 2:]
            return torch.cat([a * c - b * sn, b * c + a * sn], dim=-1).to(qkv.dtype)

        slot = pos % k_pages.shape[1]
        k_pages[page, slot] = turned(x[:, hq:hq + hkv], k_gamma)
        v_pages[page, slot] = x[:, hq + hkv:].to(qkv.dtype)
        q_out[rows] = turned(x[:, :hq], q_gamma)


def ref_paged_attention(q, k_pages, v_pages, batch, scale, causal, window, out) -> None:
    """fp32 reference of ``paged_attention`` (any device; reads lengths back)."""
    group = q.shape[1] // k_pages.shape[2]
    for s, first, n, total in _rows_of(batch, q.shape[0]):
        if n <= 0:
            continue
        total = max(total, 0)
        col = torch.arange(total, device=q.device)
        page = _pages_of(batch, s, col, k_pages.shape[1], k_pages.shape[0])
        at = torch.arange(total - n, total, device=q.device)[:, None]
        see = (page >= 0)[None] & ((col[None] <= at) if causal else torch.ones_like(at, dtype=torch.bool))
        if window:
            see = see & (col[None] > at - window)
        # Rows and positions that see nothing of each other never meet: hidden values become zeros.
        used = see.any(0)
        k = torch.where(used[:, None, None], k_pages[page.clamp(min=0), col % k_pages.shape[1]].float(), 0.0)
        v = torch.where(used[:, None, None], v_pages[page.clamp(min=0), col % k_pages.shape[1]].float(), 0.0)
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        w = torch.einsum("nhd,chd->hnc", q[first:first + n].float(), k) * scale
        w = w.masked_fill(~see[None], float("-inf"))
        top = w.amax(-1, keepdim=True) if total else torch.zeros(*w.shape[:2], 1, device=q.device)
        w = torch.where(see[None], torch.exp(w - top), 0.0)
        norm = w.sum(-1, keepdim=True)
        w = w / torch.where(norm == 0, torch.ones_like(norm), norm)
        # A weight of zero times an infinity that only other rows see would be NaN: add it where it is seen, and as it
        # is, since no weight is zero in the formula.
        bad = ~torch.isfinite(v)
        o = torch.einsum("hnc,chd->nhd", w, torch.where(bad, 0.0, v))
        for c in bad.flatten(1).any(1).nonzero().flatten().tolist():
            o = o + torch.where(see[:, c][:, None, None] & bad[c][None], v[c][None], 0.0)
        out[first:first + n] = o.to(out.dtype)
