"""Linear layers with 8-bit weights and activations (``csrc/fp8``).

e4m3 values with an fp32 scale for each block of 128 along K: one scale for
each row and block of the activations, one for each 128 x 128 block of a
weight. A block's scale is ``amax / 448`` (1 where that is 0), a value's
code ``x / scale`` rounded to the nearest e4m3 number, both quotients in fp32.

* ``quantize_fp8_weight(w)``       once, when weights are loaded
* ``linear_fp8(x, w_q, w_scale)``  ``x @ w.T`` for bf16 or fp16 activations
* ``quantize_fp8(x)``              the activations' codes and scales, for inputs
                                   that several layers share

CPU tensors run the fp32 reference math; CUDA tensors always run the kernels.
A row that holds a NaN or an infinity gives NaN or infinite outputs. These ops
have no backward pass.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .._native import _C
from .gemm import error_word
from .paged import _overlaps

BLOCK = 128
E4M3_MAX = 448.0
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _check_input(t: torch.Tensor, name: str) -> None:
    if t.dim() < 1 or t.dtype not in _FLOATS:
        raise TypeError(f"{name} must be bfloat16, float16 or float32")
    if t.shape[-1] < 1 or t.shape[-1] % 16:
        raise ValueError(f"K must be a positive multiple of 16, got {t.shape[-1]}")


def quantize_fp8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x`` [..., K] -> (codes float8_e4m3fn [..., K], scales fp32 [..., ceil(K / 128)]).

    The scales are a view of storage that keeps the rows of a block together,
    which is what ``linear_fp8`` reads."""
    if x.is_cuda:
        return _C.quantize_fp8(x)
    _check_input(x, "x")
    codes, scale = ref_quantize_fp8(x.reshape(-1, x.shape[-1]))
    return codes.view(x.shape), scale.t().contiguous().t().view(*x.shape[:-1], -1)


def quantize_fp8_weight(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``w`` [N, K] -> (codes float8_e4m3fn [N, K], scales fp32 [ceil(N / 128), ceil(K / 128)])."""
    if w.is_cuda:
        error_word(w.device)  # exists before a graph that uses it is captured
        return _C.quantize_fp8_weight(w)
    if w.dim() != 2:
        raise ValueError("w must be [N, K]")
    _check_input(w, "w")
    return ref_quantize_fp8_weight(w)


def linear_fp8(x: torch.Tensor, w_q: torch.Tensor, w_scale: torch.Tensor, out: Optional[torch.Tensor] = None,
               x_scale: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x @ w.T`` with the weight as ``quantize_fp8_weight`` gives it.

    ``x`` [..., K] bf16 or fp16 is quantized here and gives an output of its
    type; with ``x_scale`` it is the codes of ``quantize_fp8`` and the output
    is of ``dtype`` (bf16 or fp16). K must be a multiple of 16 and N of 8.
    Products are exact, sums fp32, and each block of 128 along K is scaled
    before it is added."""
    if x.is_cuda:  # checked there
        like = None if x_scale is None else _like(dtype)
        return _C.linear_fp8(x, w_q, w_scale, out, x_scale, like, error_word(x.device))
    if w_q.dim() != 2 or w_q.dtype != torch.float8_e4m3fn or not w_q.is_contiguous():
        raise TypeError("w_q must be contiguous float8_e4m3fn [N, K]")
    n, k = w_q.shape
    if k < 1 or k % 16 or n < 1 or n % 8:
        raise ValueError(f"K must be a multiple of 16 and N of 8, got N {n}, K {k}")
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x must be [..., {k}]")
    if w_scale.dtype != torch.float32 or tuple(w_scale.shape) != (_blocks(n), _blocks(k)) or \
            not w_scale.is_contiguous():
        raise ValueError(f"w_scale must be contiguous fp32 [{_blocks(n)}, {_blocks(k)}]")
    if w_q.device != x.device or w_scale.device != x.device:
        raise ValueError(f"the weight must be on {x.device}")
    if x_scale is None:
        if x.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("x must be bfloat16 or float16, or codes with their x_scale")
        dtype = x.dtype
    else:
        if x.dtype != torch.float8_e4m3fn:
            raise TypeError("with x_scale, x must be float8_e4m3fn")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("dtype must be bfloat16 or float16")
        if tuple(x_scale.shape) != (*x.shape[:-1], _blocks(k)) or x_scale.dtype != torch.float32 or \
                x_scale.device != x.device:
            raise ValueError(f"x_scale must be fp32 [..., {_blocks(k)}] on {x.device}")
    shape = (*x.shape[:-1], n)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=x.device)
    elif tuple(out.shape) != shape or out.dtype != dtype or out.device != x.device:
        raise ValueError(f"out must be {dtype} {list(shape)} on {x.device}")
    if any(t is not None and _overlaps(out, t) for t in (x, w_q, w_scale, x_scale)):
        raise ValueError("out overlaps an input")
    x2 = x.reshape(-1, k)
    codes, scale = ref_quantize_fp8(x2) if x_scale is None else (x2, x_scale.reshape(-1, _blocks(k)))
    out.view(-1, n).copy_(ref_linear_fp8(codes, scale, w_q, w_scale).to(dtype))
    return out


_LIKE = {}


def _like(dtype: torch.dtype) -> torch.Tensor:
    """An empty tensor that carries a type into the native call."""
    if dtype not in _LIKE:
        _LIKE[dtype] = torch.empty(0, dtype=dtype)
    return _LIKE[dtype]


# ------------------------------------------------------------------ references
def _scale(amax: torch.Tensor) -> torch.Tensor:
    scale = amax / torch.full_like(amax, E4M3_MAX)
    return torch.where(scale == 0, torch.ones_like(scale), scale)


def ref_quantize_fp8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 reference of ``quantize_fp8`` for [rows, K]."""
    m, k = x.shape
    full = torch.zeros(m, _blocks(k) * BLOCK, device=x.device)
    full[:, :k] = x.float()
    full = full.view(m, -1, BLOCK)
    amax = full.abs().amax(-1)
    scale = _scale(amax)
    codes = (full / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes.view(m, -1)[:, :k].contiguous(), scale


def ref_quantize_fp8_weight(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 reference of ``quantize_fp8_weight``."""
    n, k = w.shape
    nb, kb = _blocks(n), _blocks(k)
    full = torch.zeros(nb * BLOCK, kb * BLOCK, device=w.device)
    full[:n, :k] = w.float()
    full = full.view(nb, BLOCK, kb, BLOCK)
    amax = full.abs().amax(dim=(1, 3))
    scale = _scale(amax)
    codes = (full / scale[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes.view(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous(), scale


def ref_linear_fp8(x_q, x_scale, w_q, w_scale) -> torch.Tensor:
    """fp32 reference of the product of codes and scales, [M, N]."""
    n, k = w_q.shape
    a = x_q.float() * x_scale.repeat_interleave(BLOCK, 1)[:, :k]
    b = w_q.float() * w_scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return a @ b.t()
