"""Heads of q, k and v between the qkv linear and attention: norms of q and k per head, rotation by position and the append to a
paged cache, each head read and written once. CUDA tensors only; no fallback.
"""
from __future__ import annotations

import ctypes
from ctypes import c_float, c_int, c_int64, c_void_p
from typing import List, Optional, Tuple

import torch

from . import _native as N
from .int8_kernel import same_device

fp8_dtype = torch.float8_e4m3fn


class RopeArgs(ctypes.Structure):
    """``b200_rope_args`` of the C ABI."""

    _fields_ = (
        [(n, c_void_p) for n in ("q", "k", "v")]
        + [(n, c_int64) for n in ("q_token", "q_head", "k_token", "k_head", "v_token", "v_head")]
        + [(n, c_void_p) for n in ("q_weight", "k_weight", "q_out", "k_out", "positions")]
        + [("positions_ld", c_int64), ("cos_sin", c_void_p), ("cos_sin_ld", c_int64), ("table_rows", c_int64)]
        + [(n, c_void_p) for n in ("k_cache", "v_cache")]
        + [(f"{c}_cache_{n}", c_int64) for c in "kv" for n in ("page", "token", "head")]
        + [("pages", c_int64)]
        + [(n, c_void_p) for n in ("slots", "k_scale", "v_scale")]
        + [("rows", c_int64)]
        + [(n, c_int) for n in ("q_heads", "kv_heads", "dim", "dtype", "rotated", "neox", "axes")]
        + [("sections", c_int * 4)]
        + [(n, c_int) for n in ("sections_interleaved", "positions_dtype", "page_size", "cache_dtype", "slots_dtype", "k_scales", "v_scales")]
        + [("eps", c_float)]
    )


def check_sizes(*sizes: int) -> None:
    """Sizes that the C ABI holds in 32 bits: ctypes would take the low ones of a larger number."""
    if max(sizes) > 0x7FFFFFFF:
        raise NotImplementedError("heads, head sizes, page sizes and mask widths from 2^31 on are not built")


def check_index(t: torch.Tensor, what: str) -> None:
    assert t.dtype in (torch.int32, torch.int64), f"{what} are int32 or int64"


def _set_rotation(a: RopeArgs, dim, positions, cos_sin_cache, is_neox, mrope_section, mrope_interleaved):
    """Positions and their table; nothing rotates where both are None."""
    assert (positions is None) == (cos_sin_cache is None), "positions and cos_sin_cache go together"
    if positions is None:
        return
    assert cos_sin_cache.dim() == 2 and cos_sin_cache.dtype == torch.float32, "cos_sin_cache is [positions, rotated] float32"
    assert cos_sin_cache.stride(1) == 1 or cos_sin_cache.shape[1] <= 1, "rows of cos_sin_cache are contiguous"
    a.rotated = cos_sin_cache.shape[1]
    assert a.rotated % 2 == 0 and a.rotated <= dim, f"cos_sin_cache has {a.rotated} columns for heads of {dim}"
    check_index(positions, "positions")
    a.axes = 1 if mrope_section is None else len(mrope_section)
    if a.axes > 4:
        raise NotImplementedError("more than four axes are not built")
    if mrope_section is None:
        assert positions.shape == (a.rows,), f"positions have the shape {(a.rows,)}"
    else:
        assert a.axes >= 1, "mrope_section names no axis"
        assert positions.shape == (a.axes, a.rows), f"positions have the shape {(a.axes, a.rows)}"
        assert min(mrope_section) >= 0 and sum(mrope_section) == a.rotated // 2, "mrope_section sums to the number of pairs"
        if mrope_interleaved:
            assert all(n == 0 or (n - 1) * a.axes + k < a.rotated // 2 for k, n in enumerate(mrope_section) if k), \
                "an interleaved section reaches past the last pair"
        for k, n in enumerate(mrope_section):
            a.sections[k] = n
    assert a.rows <= 1 or positions.stride(-1) == 1, "positions of an axis are contiguous"
    a.positions, a.positions_dtype = N.ptr(positions), N.DTYPE_CODE[positions.dtype]
    a.positions_ld = positions.stride(0) if positions.dim() == 2 else 0
    a.cos_sin, a.cos_sin_ld, a.table_rows = N.ptr(cos_sin_cache), cos_sin_cache.stride(0), cos_sin_cache.shape[0]
    a.neox, a.sections_interleaved = int(bool(is_neox)), int(bool(mrope_interleaved))


def check_caches(k_cache, v_cache, kv_heads, dim):
    for t in (k_cache, v_cache):
        assert t.dim() == 4 and t.shape[2:] == (kv_heads, dim), f"a cache is [pages, page size, {kv_heads}, {dim}]"
        assert t.stride(3) == 1 or dim <= 1, "elements of a head are contiguous in the cache"
    assert k_cache.shape == v_cache.shape and k_cache.dtype == v_cache.dtype, "the caches differ"
    check_sizes(k_cache.shape[1])


def check_scale(scale, kv_heads, cache_dtype, what):
    if scale is None:
        return
    assert cache_dtype == fp8_dtype, f"{what} belongs to an FP8 cache"
    assert scale.dtype == torch.float32 and scale.is_contiguous() and scale.numel() in (1, kv_heads), \
        f"{what} is float32, one element or one per kv head"


def _set_cache(a: RopeArgs, dtype, k_cache, v_cache, slots, k_scale, v_scale):
    check_caches(k_cache, v_cache, a.kv_heads, a.dim)
    assert k_cache.dtype in (dtype, fp8_dtype), "the caches have the type of k and v, or float8_e4m3fn"
    assert k_cache.shape[1] > 0, "pages without tokens"
    check_index(slots, "slots")
    assert slots.shape == (a.rows,) and (a.rows <= 1 or slots.stride(0) == 1), f"slots are {a.rows} contiguous elements"
    check_scale(k_scale, a.kv_heads, k_cache.dtype, "k_scale")
    check_scale(v_scale, a.kv_heads, v_cache.dtype, "v_scale")
    a.pages, a.page_size = k_cache.shape[:2]
    a.k_cache, a.v_cache = N.ptr(k_cache), N.ptr(v_cache)
    a.k_cache_page, a.k_cache_token, a.k_cache_head = k_cache.stride()[:3]
    a.v_cache_page, a.v_cache_token, a.v_cache_head = v_cache.stride()[:3]
    a.cache_dtype = E4M3 if k_cache.dtype == fp8_dtype else N.DTYPE_CODE[dtype]
    a.slots, a.slots_dtype = N.ptr(slots), N.DTYPE_CODE[slots.dtype]
    a.k_scale, a.v_scale = N.ptr(k_scale), N.ptr(v_scale)
    a.k_scales, a.v_scales = (0 if t is None else t.numel() for t in (k_scale, v_scale))


E4M3 = 5


def _qkv_args(qkv, num_heads, num_kv_heads, q_weight, k_weight, eps) -> RopeArgs:
    """q and k as heads of the qkv linear's rows ``[tokens, (num_heads + 2 num_kv_heads) * dim]``."""
    assert qkv.dtype in (torch.bfloat16, torch.float16, torch.float32), f"unsupported input dtype {qkv.dtype}"
    assert num_heads > 0 and num_kv_heads > 0, "num_heads and num_kv_heads are positive"
    heads = num_heads + 2 * num_kv_heads
    assert qkv.dim() == 2 and qkv.shape[1] % heads == 0 and qkv.shape[1] > 0, f"qkv is [tokens, {heads} * dim]"
    assert qkv.stride(1) == 1, "rows of qkv are contiguous"
    check_sizes(num_heads, num_kv_heads, qkv.shape[1] // heads)
    a = RopeArgs(rows=qkv.shape[0], q_heads=num_heads, kv_heads=num_kv_heads, dim=qkv.shape[1] // heads, dtype=N.DTYPE_CODE[qkv.dtype], eps=eps)
    for w in (q_weight, k_weight):
        assert w is None or (w.shape == (a.dim,) and w.dtype == qkv.dtype and w.is_contiguous()), "norm weights are [dim], of qkv's type"
    size, ld = qkv.element_size(), qkv.stride(0) if a.rows > 1 else qkv.shape[1]
    a.q, a.q_token, a.q_head = N.ptr(qkv), ld, a.dim
    a.k, a.k_token, a.k_head = N.ptr(qkv) + num_heads * a.dim * size, ld, a.dim
    a.q_weight, a.k_weight = N.ptr(q_weight), N.ptr(k_weight)
    return a


def _run(a: RopeArgs, first: torch.Tensor, what: str) -> None:
    if a.rows > 0:
        with N.on_device(first):
            st = N.load().b200_qk_norm_rope(ctypes.addressof(a), N.current_stream())
        N.check(st, what)


def qk_norm_rope(
    qkv: torch.Tensor,
    num_heads: int,
    num_kv_heads: int,
    positions: Optional[torch.Tensor],
    cos_sin_cache: Optional[torch.Tensor],
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    is_neox: bool = True,
    mrope_section: Optional[List[int]] = None,
    mrope_interleaved: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm of every head of q and k (where its weight is given), then the rotation by position; returns new tensors
    ``(q [T, num_heads, dim], k [T, num_kv_heads, dim])`` of qkv's type.

    ``qkv`` (bf16, fp16 or fp32) ``[T, (num_heads + 2 num_kv_heads) * dim]`` = q | k | v of the qkv linear, rows at any distance; v is not
    read. ``cos_sin_cache`` fp32 ``[positions, rotated]`` holds ``cos | sin`` of a position's ``rotated / 2`` angles; the first ``rotated``
    elements of a head turn, pair ``j`` being elements ``j`` and ``j + rotated / 2`` (``is_neox``) or ``2j`` and ``2j + 1``, the others pass.
    ``positions`` int32 or int64 ``[T]``; with ``mrope_section`` ``[axes, T]`` (up to four axes): the pairs take the axes in runs of these
    lengths, or with ``mrope_interleaved`` in turn, pair ``j`` axis ``j % axes`` while that has pairs left (``j < axes * section``), else axis 0.
    All in fp32, rounded once. A position outside the table makes its pairs NaN. ``positions`` and ``cos_sin_cache`` None: no rotation."""
    N.load()
    out = N.host.qkv_rope(qkv, num_heads, num_kv_heads, positions, cos_sin_cache, is_neox, mrope_section, mrope_interleaved, q_weight, k_weight,
                          eps)
    if out is not None:
        return out
    a = _qkv_args(qkv, num_heads, num_kv_heads, q_weight, k_weight, eps)
    _set_rotation(a, a.dim, positions, cos_sin_cache, is_neox, mrope_section, mrope_interleaved)
    N.require_cuda(qkv, positions, cos_sin_cache, q_weight, k_weight)
    same_device(qkv, positions, cos_sin_cache, q_weight, k_weight)
    q = torch.empty((a.rows, num_heads, a.dim), dtype=qkv.dtype, device=qkv.device)
    k = torch.empty((a.rows, num_kv_heads, a.dim), dtype=qkv.dtype, device=qkv.device)
    a.q_out, a.k_out = N.ptr(q), N.ptr(k)
    _run(a, qkv, "qk_norm_rope")
    return q, k


def qk_norm_rope_append(
    qkv: torch.Tensor,
    num_heads: int,
    num_kv_heads: int,
    positions: Optional[torch.Tensor],
    cos_sin_cache: Optional[torch.Tensor],
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    is_neox: bool = True,
    mrope_section: Optional[List[int]] = None,
    mrope_interleaved: bool = False,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``qk_norm_rope`` whose keys, with the values, go straight into a paged cache (``append_paged_kv``): what a layer calls behind its
    qkv linear. Returns q ``[T, num_heads, dim]``; a token without a slot has a q all the same."""
    N.load()
    out = N.host.qkv_rope(qkv, num_heads, num_kv_heads, positions, cos_sin_cache, is_neox, mrope_section, mrope_interleaved, q_weight, k_weight,
                          eps, k_cache, v_cache, slots, k_scale, v_scale)
    if out is not None:
        return out
    a = _qkv_args(qkv, num_heads, num_kv_heads, q_weight, k_weight, eps)
    _set_rotation(a, a.dim, positions, cos_sin_cache, is_neox, mrope_section, mrope_interleaved)
    a.v, a.v_token, a.v_head = a.k + num_kv_heads * a.dim * qkv.element_size(), a.k_token, a.dim
    _set_cache(a, qkv.dtype, k_cache, v_cache, slots, k_scale, v_scale)
    tensors = (qkv, positions, cos_sin_cache, k_cache, v_cache, slots, q_weight, k_weight, k_scale, v_scale)
    N.require_cuda(*tensors)
    same_device(*tensors)
    q = torch.empty((a.rows, num_heads, a.dim), dtype=qkv.dtype, device=qkv.device)
    a.q_out = N.ptr(q)
    _run(a, qkv, "qk_norm_rope_append")
    return q


def append_paged_kv(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    positions: Optional[torch.Tensor] = None,
    cos_sin_cache: Optional[torch.Tensor] = None,
    is_neox: bool = True,
    mrope_section: Optional[List[int]] = None,
    mrope_interleaved: bool = False,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> None:
    """Keys, rotated on the way (as in ``qk_norm_rope``) where ``positions`` are given, and values into a paged cache, in place.

    ``k``, ``v`` ``[T, kv heads, dim]`` (bf16, fp16 or fp32), heads contiguous, at any distance. ``k_cache``, ``v_cache``
    ``[pages, page size, kv heads, dim]``, of k's type or ``float8_e4m3fn``, any strides but the last. ``slots`` int32 or int64 ``[T]``: token
    ``slot % page size`` of page ``slot // page size``; a slot that the cache does not have (-1 for padding) leaves its token out, the others are
    distinct. An FP8 cache holds ``e4m3(x / scale)``, the quotient and the rotation unrounded, saturated at 448; ``k_scale``, ``v_scale`` fp32 of one
    element or one per kv head (None: 1)."""
    N.load()
    if N.host.append_kv(k, v, k_cache, v_cache, slots, positions, cos_sin_cache, is_neox, mrope_section, mrope_interleaved, k_scale, v_scale):
        return
    assert k.dtype in (torch.bfloat16, torch.float16, torch.float32), f"unsupported input dtype {k.dtype}"
    assert k.dim() == 3 and v.shape == k.shape and v.dtype == k.dtype, "k and v are [tokens, kv heads, dim], alike"
    rows, heads, dim = k.shape
    assert dim > 0 and heads > 0, "heads without elements"
    check_sizes(heads, dim)
    assert dim <= 1 or (k.stride(2) == 1 and v.stride(2) == 1), "elements of a head are contiguous"
    a = RopeArgs(rows=rows, kv_heads=heads, dim=dim, dtype=N.DTYPE_CODE[k.dtype])
    _set_rotation(a, dim, positions, cos_sin_cache, is_neox, mrope_section, mrope_interleaved)
    a.k, a.k_token, a.k_head = N.ptr(k), k.stride(0), k.stride(1)
    a.v, a.v_token, a.v_head = N.ptr(v), v.stride(0), v.stride(1)
    _set_cache(a, k.dtype, k_cache, v_cache, slots, k_scale, v_scale)
    tensors = (k, v, k_cache, v_cache, slots, positions, cos_sin_cache, k_scale, v_scale)
    N.require_cuda(*tensors)
    same_device(*tensors)
    _run(a, k, "append_paged_kv")
