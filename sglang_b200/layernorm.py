"""RMSNorm in front of a quantised linear, with the residual's addition and the linear's quantiser in the same pass over the
rows, without the 16-bit tensor in between. CUDA tensors only; no fallback.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native as N
from .fp8_kernel import create_per_token_group_quant_fp8_output_scale, fp8_dtype
from .int8_kernel import rows_of, same_device

ROW_INT8, ROW_FP8, ROW_FP8_UE8M0 = 0, 1, 2


def _check(x, weight, residual):
    assert x.dtype in (torch.bfloat16, torch.float16, torch.float32), f"unsupported input dtype {x.dtype}"
    assert weight.shape == (x.shape[-1],) and weight.is_contiguous(), "weight has one element per column"
    assert weight.dtype == x.dtype, "weight and x must have the same dtype"
    if residual is not None:
        assert residual.shape == x.shape and residual.dtype == x.dtype, "residual must match x"
    N.require_cuda(x, weight, residual)
    same_device(x, weight, residual)


def _run(x, weight, eps, residual, kind, x_q, x_s, sm, sg):
    x, ld = rows_of(x, "x")
    res_out, r_ld = None, 0
    if residual is not None:
        residual, r_ld = rows_of(residual, "residual")
        res_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    H = x.shape[-1]
    rows = x.numel() // H if H else 0
    if rows > 0:
        with N.on_device(x):
            st = N.load().b200_rmsnorm_quant(N.ptr(x), ld, N.ptr(residual), r_ld, N.ptr(weight), N.DTYPE_CODE[x.dtype], kind,
                                             N.ptr(x_q), N.ptr(x_s), sm, sg, N.ptr(res_out), rows, H, eps, N.current_stream())
        N.check(st, "rmsnorm_quant")
    return (x_q, x_s) if res_out is None else (x_q, x_s, res_out)


def rmsnorm_quant_int8(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    residual: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, ...]:
    """RMSNorm, then 8-bit integers with one scale per row (``per_token_quant_int8``): the input of ``int8_scaled_mm``.

    ``h = x + residual`` (or ``x``), ``y = h * weight / sqrt(mean(h^2) + eps)``, all in fp32; ``y`` is quantised unrounded. The root
    cancels in a code, the integer nearest to ``v / (max|v| / 127)``, ``v = h * weight`` (IEEE divisions), so codes do not depend on the alignment or the number of
    rows; the last bits of the scales may, with the order of the sum of squares.
    Returns ``(x_q [.., H] int8, x_s [.., 1] fp32)`` and, with ``residual``, ``h`` rounded to the input type as a new tensor.
    ``x`` and ``residual`` are contiguous, or 2-D with contiguous rows at any distance; ``weight [H]``; one dtype for all."""
    N.load()
    out = N.host.norm_quant(x, weight, eps, residual, 0)
    if out is not None:
        return out
    assert x.shape[-1] > 0, "rows without elements have no scale"
    _check(x, weight, residual)
    x_q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    x_s = torch.empty((*x.shape[:-1], 1), dtype=torch.float32, device=x.device)
    return _run(x, weight, eps, residual, ROW_INT8, x_q, x_s, 1, 0)


def rmsnorm_quant_fp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    group_size: int = 128,
    eps: float = 1e-6,
    residual: Optional[torch.Tensor] = None,
    column_major_scales: bool = False,
    scale_tma_aligned: bool = False,
    scale_ue8m0: bool = False,
) -> Tuple[torch.Tensor, ...]:
    """RMSNorm, then FP8 E4M3 with one scale per row and ``group_size`` columns: the input of ``w8a8_block_fp8_matmul``.

    Norm, residual and result as for ``rmsnorm_quant_int8`` (codes ``e4m3(v * f)``, ``f = 448 / max|v|`` of the group; a power-of-two scale does not
    cancel the root); scales and their layouts (row-major, column-major, padded, packed
    powers of two) as for ``per_token_group_quant_fp8``. Only ``group_size`` 128, the K block of the GEMM, is built."""
    if group_size != 128:
        raise NotImplementedError("rmsnorm_quant_fp8: only group_size 128 is built")
    assert not scale_ue8m0 or (column_major_scales and scale_tma_aligned), "packed scales are column-major and padded"
    N.load()
    out = N.host.norm_quant(x, weight, eps, residual, 4 if scale_ue8m0 else 1 if not column_major_scales else 3 if scale_tma_aligned else 2)
    if out is not None:
        return out
    assert x.shape[-1] % group_size == 0, "the last dimension of `x` cannot be divisible by `group_size`"
    assert x.dim() == 2 or not column_major_scales, "column-major scales need a 2-D input"
    _check(x, weight, residual)
    x_q = torch.empty(x.shape, dtype=fp8_dtype, device=x.device)
    x_s = create_per_token_group_quant_fp8_output_scale(x.shape, x.device, group_size, column_major_scales, scale_tma_aligned,
                                                        scale_ue8m0)
    if scale_ue8m0:
        sm, sg = 1, (x.shape[0] + 3) // 4 * 4
    elif column_major_scales:
        sm, sg = x_s.stride(0), x_s.stride(1)
    else:
        sm, sg = x.shape[-1] // group_size, 1
    return _run(x, weight, eps, residual, ROW_FP8_UE8M0 if scale_ue8m0 else ROW_FP8, x_q, x_s, sm, sg)
