"""W8A8 int8 operators: the per-token quantiser, the product with scales per token and per output channel, and the linear layer
that runs both. CUDA tensors only; no fallback.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native as N

int8_max = 127


def rows_of(x: torch.Tensor, name: str) -> Tuple[torch.Tensor, int]:
    """``x`` as rows whose elements are contiguous, and the distance between rows: a 2-D tensor may be a slice of wider
    rows, any other has to be contiguous."""
    if x.dim() == 2 and (x.stride(1) == 1 or x.shape[1] <= 1):
        return x, x.stride(0) if x.shape[0] > 1 else x.shape[1]
    assert x.dim() >= 1 and x.is_contiguous(), f"`{name}` is not contiguous"
    return x, x.shape[-1]


def per_token_quant_int8(
    x: torch.Tensor,
    scale_dtype: torch.dtype = torch.float32,
    cal_sum: bool = False,
    fuse_silu_and_mul: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Symmetric 8-bit integers with one scale per row; returns ``(x_q [.., K] int8, x_s [.., 1] fp32)``.

    ``x_s = max(|x|, 1e-10) / 127`` over the row, ``x_q = x / x_s`` rounded to the nearest integer, ties to even (both IEEE
    divisions, in fp32). ``x`` (bf16, fp16 or fp32) is contiguous, or 2-D with contiguous rows at any distance.
    ``fuse_silu_and_mul``: ``x`` is ``[.., 2K]`` = gate | up and ``y = silu(gate) * up``, in fp32, is quantised: ``x_s = max(|y|, 1e-10) / 127``,
    ``x_q`` the integer nearest to the unrounded product of ``y`` and ``127 / max(|y|, 1e-10)``, a quotient rounded once. The bits are the same
    for every alignment and number of rows. A NaN or an
    infinity in a row leaves the row's scale NaN or infinite. ``scale_dtype`` other than fp32 and ``cal_sum`` (row sums for
    asymmetric weights) are not built.
    """
    if scale_dtype != torch.float32 or cal_sum:
        raise NotImplementedError("per_token_quant_int8: only fp32 scales without row sums are built")
    N.load()
    pair = N.host.quant_int8(x, bool(fuse_silu_and_mul))
    if pair is not None:
        return pair
    assert x.dtype in (torch.bfloat16, torch.float16, torch.float32), f"unsupported input dtype {x.dtype}"
    x, ld = rows_of(x, "x")
    width = x.shape[-1]
    assert not fuse_silu_and_mul or width % 2 == 0, "gate | up rows have an even number of elements"
    K = width // 2 if fuse_silu_and_mul else width
    assert K > 0, "rows without elements have no scale"
    N.require_cuda(x)
    x_q = torch.empty((*x.shape[:-1], K), dtype=torch.int8, device=x.device)
    x_s = torch.empty((*x.shape[:-1], 1), dtype=torch.float32, device=x.device)
    if x_s.numel() == 0:
        return x_q, x_s
    with N.on_device(x):
        st = N.load().b200_per_token_quant_int8(N.ptr(x), ld, N.DTYPE_CODE[x.dtype], N.ptr(x_q), N.ptr(x_s), x_s.numel(), K,
                                                int(fuse_silu_and_mul), N.current_stream())
    N.check(st, "per_token_quant_int8")
    return x_q, x_s


def int8_scaled_mm(
    mat_a: torch.Tensor,
    mat_b: torch.Tensor,
    scales_a: torch.Tensor,
    scales_b: torch.Tensor,
    out_dtype: torch.dtype,
    bias: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``(mat_a @ mat_b) * scales_a[:, None] * scales_b[None, :] (+ bias)`` on the tcgen05 tensor cores.

    ``mat_a [M, K]`` int8 with contiguous rows, ``mat_b [K, N]`` int8 column-major (a transposed ``[N, K]`` weight), ``scales_a``
    fp32 with ``M`` elements, ``scales_b`` fp32 with ``N``, ``bias [N]`` of ``out_dtype`` (bf16, fp16; fp32 is built, too). The
    integer sums are exact; scales and bias are applied in fp32 and the result is rounded once. Preconditions: rows of ``mat_a`` and columns of ``mat_b`` start at multiples of 16 bytes, ``K`` is a multiple of 16, ``N`` of 8;
    beyond ``K`` = 131071 a 32-bit sum could overflow and the call is refused.
    """
    N.load()
    out = N.host.int8_mm(mat_a, mat_b, scales_a, scales_b, N.DTYPE_CODE.get(out_dtype, -1), bias)
    if out is not None:
        return out
    assert mat_a.dim() == 2 and mat_b.dim() == 2, "mat_a and mat_b must be 2D tensors"
    M, K = mat_a.shape
    Nn = mat_b.shape[1]
    assert mat_b.shape[0] == K, "mat_a and mat_b shapes cannot be multiplied"
    assert mat_a.dtype == torch.int8 and mat_b.dtype == torch.int8, "mat_a and mat_b must be int8"
    assert mat_a.stride(1) == 1 or K <= 1, "mat_a must be a row major tensor"
    assert mat_b.stride(0) == 1 or K <= 1, "mat_b must be a column major tensor"
    assert scales_a.dtype == torch.float32 and scales_b.dtype == torch.float32, "scales must be Float32"
    assert scales_a.numel() == M and scales_a.is_contiguous(), "size of scales_a is not matched"
    assert scales_b.numel() == Nn and scales_b.is_contiguous(), "size of scales_b is not matched"
    assert out_dtype in (torch.bfloat16, torch.float16, torch.float32), "out_dtype must be Half, BFloat16 or Float"
    if bias is not None:
        assert bias.numel() == Nn and bias.is_contiguous(), "size of bias is not matched"
        assert bias.dtype == out_dtype, "bias dtype must match output dtype"
    assert K > 0, "K is zero"
    N.require_cuda(mat_a, mat_b, scales_a, scales_b, bias)
    same_device(mat_a, mat_b, scales_a, scales_b, bias)
    out = torch.empty((M, Nn), dtype=out_dtype, device=mat_a.device)
    if out.numel() == 0:
        return out
    with N.on_device(mat_a):
        st = N.load().b200_int8_scaled_mm(
            N.ptr(mat_a), mat_a.stride(0) if M > 1 else K, N.ptr(scales_a), N.ptr(mat_b), mat_b.stride(1) if Nn > 1 else K,
            N.ptr(scales_b), N.ptr(bias), N.ptr(out), N.DTYPE_CODE[out_dtype], M, Nn, K, N.current_stream())
    N.check(st, "int8_scaled_mm")
    return out


def same_device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    for t in others:
        assert t is None or t.device == first.device, f"tensors on {first.device} and {t.device}"


def w8a8_int8_linear(
    input: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Quantise the activation per token, multiply, apply the scales and the bias. ``input [.., K]`` bf16 or fp16, ``weight [N, K]`` int8, ``weight_scale`` fp32 with ``N``
    elements, ``bias [N]`` of the input's type; the result has the input's type."""
    N.load()
    out = N.host.int8_linear(input, weight, weight_scale, bias)
    if out is not None:
        return out
    assert input.dtype in (torch.bfloat16, torch.float16), f"unsupported input dtype {input.dtype}"
    assert weight.dim() == 2, "weight must be a 2D tensor"
    input_2d = input if input.dim() == 2 else input.reshape(-1, input.shape[-1])
    x_q, x_s = per_token_quant_int8(input_2d)
    out = int8_scaled_mm(x_q, weight.t(), x_s, weight_scale, input.dtype, bias)
    return out.view(*input.shape[:-1], weight.shape[0])
