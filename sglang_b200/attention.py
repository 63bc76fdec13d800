"""Attention of the newest tokens of every sequence over the paged cache that ``append_paged_kv`` and ``qk_norm_rope_append`` fill.
CUDA tensors only; no fallback.
"""
from __future__ import annotations

import ctypes
from ctypes import c_float, c_int, c_int64, c_void_p
from typing import Optional, Tuple, Union

import torch

from . import _native as N
from .int8_kernel import same_device
from .rotary import E4M3, check_caches, check_scale, check_sizes, fp8_dtype


class TreeAttentionArgs(ctypes.Structure):
    """``b200_tree_attention_args`` of the C ABI."""

    _fields_ = (
        [("q", c_void_p), ("q_token", c_int64), ("q_head", c_int64), ("out", c_void_p), ("lse", c_void_p), ("k_cache", c_void_p), ("v_cache", c_void_p)]
        + [(f"{c}_{n}", c_int64) for c in "kv" for n in ("page", "token", "head")]
        + [("pages", c_int64), ("page_table", c_void_p), ("page_table_ld", c_int64), ("max_pages", c_int64), ("seq_lens", c_void_p),
           ("q_starts", c_void_p), ("mask", c_void_p), ("mask_ld", c_int64), ("k_scale", c_void_p), ("v_scale", c_void_p),
           ("tokens", c_int64), ("sequences", c_int64)]
        + [(n, c_int) for n in ("q_heads", "kv_heads", "dim", "dtype", "page_size", "cache_dtype", "mask_width", "k_scales", "v_scales")]
        + [("scale", c_float)]
    )


def tree_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    q_starts: Optional[torch.Tensor] = None,
    tree_mask: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of one new token per sequence, of a tree of drafted tokens, or of the end of a prompt, over a paged cache that already
    holds their keys and values. Returns ``out [T, heads, dim]`` of q's type, with ``return_lse`` also the logarithm of the sum of the exponentials
    ``[T, heads]`` fp32.

    ``q [T, heads, dim]`` bf16 or fp16, ``dim`` 64, 128 or 256, heads a multiple of the kv heads. ``k_cache``, ``v_cache`` ``[pages, page size, kv
    heads, dim]``, of q's type or ``float8_e4m3fn`` (``k_scale``, ``v_scale``: positive fp32, one element or one per kv head). ``page_table`` int32
    ``[B, columns]``: pages of a sequence in order. ``seq_lens`` int32 ``[B]``: keys of a sequence, its new tokens among them. ``q_starts`` int32
    ``[B + 1]``: the new tokens of sequence ``b`` are rows ``q_starts[b]`` to ``q_starts[b + 1] - 1`` (None: one each, ``T == B``).
    Every new token sees the keys before its sequence's new ones, and of those the ones up to itself, or with ``tree_mask`` (bool, ``[T, widest]``)
    those where its row is True. ``scale`` is ``dim ** -0.5`` unless given, positive.

    Softmax in fp32, results rounded once. Weights are rounded for the product with the values, to q's type over a 16-bit cache and to fp16 over an FP8 one
    (bf16 queries too become fp16 there, by a power of two per row); in fp16 a weight is off by up to 2^-32 of the row's largest, however small it is itself. A token that sees nothing gives 0 (lse -inf). Rows behind the
    last sequence are not written: they keep what ``out`` (a tensor of its own) held. A page that the cache does not have makes the rows that see it NaN; lengths
    past the page table are cut. Heads of q and of the caches start at multiples of 16 bytes."""
    N.load()
    if not return_lse:
        got = N.host.attention(q, k_cache, v_cache, page_table, seq_lens, q_starts, tree_mask, scale, k_scale, v_scale, out)
        if got is not None:
            return got
    assert q.dim() == 3 and q.dtype in (torch.bfloat16, torch.float16), "q is [tokens, heads, dim], bfloat16 or float16"
    T, heads, dim = q.shape
    assert heads > 0 and dim > 0 and q.stride(2) == 1, "elements of a head are contiguous"
    assert k_cache.dim() == 4 and k_cache.shape[2] > 0 and heads % k_cache.shape[2] == 0, "heads are a multiple of the cache's kv heads"
    kv_heads = k_cache.shape[2]
    check_sizes(heads, dim, 0 if tree_mask is None else tree_mask.shape[-1])
    check_caches(k_cache, v_cache, kv_heads, dim)
    assert k_cache.dtype in (q.dtype, fp8_dtype), "the caches have q's type, or float8_e4m3fn"
    assert k_cache.shape[1] > 0, "pages without tokens"
    assert page_table.dim() == 2 and page_table.dtype == torch.int32, "page_table is [sequences, columns] int32"
    B = page_table.shape[0]
    assert page_table.shape[1] <= 1 or page_table.stride(1) == 1, "rows of page_table are contiguous"
    assert seq_lens.shape == (B,) and seq_lens.dtype == torch.int32 and (B <= 1 or seq_lens.stride(0) == 1), f"seq_lens are {B} int32"
    if q_starts is None:
        assert T == B, f"without q_starts there is one token per sequence, not {T} for {B}"
    else:
        assert q_starts.shape == (B + 1,) and q_starts.dtype == torch.int32 and q_starts.stride(0) == 1, f"q_starts are {B + 1} int32"
    if tree_mask is not None:
        assert tree_mask.dim() == 2 and tree_mask.shape[0] == T and tree_mask.dtype == torch.bool, f"tree_mask is [{T}, widest] bool"
        assert tree_mask.shape[1] <= 1 or tree_mask.stride(1) == 1, "rows of tree_mask are contiguous"
    check_scale(k_scale, kv_heads, k_cache.dtype, "k_scale")
    check_scale(v_scale, kv_heads, v_cache.dtype, "v_scale")
    if out is not None:
        assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous(), "out is a contiguous tensor like q"
    tensors = (q, k_cache, v_cache, page_table, seq_lens, q_starts, tree_mask, k_scale, v_scale, out)
    N.require_cuda(*tensors)
    same_device(*tensors)
    if out is None:
        out = torch.empty((T, heads, dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((T, heads), dtype=torch.float32, device=q.device) if return_lse else None
    a = TreeAttentionArgs(
        q=N.ptr(q), q_token=q.stride(0), q_head=q.stride(1), out=N.ptr(out), lse=N.ptr(lse), k_cache=N.ptr(k_cache), v_cache=N.ptr(v_cache),
        k_page=k_cache.stride(0), k_token=k_cache.stride(1), k_head=k_cache.stride(2), v_page=v_cache.stride(0), v_token=v_cache.stride(1),
        v_head=v_cache.stride(2), pages=k_cache.shape[0], page_table=N.ptr(page_table), page_table_ld=page_table.stride(0),
        max_pages=page_table.shape[1], seq_lens=N.ptr(seq_lens), q_starts=N.ptr(q_starts),
        mask=None if tree_mask is None else N.ptr(tree_mask) or N.ptr(q),  # no pointer means no mask; one of width 0 is not read
        mask_ld=0 if tree_mask is None else tree_mask.stride(0), k_scale=N.ptr(k_scale), v_scale=N.ptr(v_scale), tokens=T, sequences=B,
        q_heads=heads, kv_heads=kv_heads, dim=dim, dtype=N.DTYPE_CODE[q.dtype], page_size=k_cache.shape[1],
        cache_dtype=E4M3 if k_cache.dtype == fp8_dtype else N.DTYPE_CODE[q.dtype], mask_width=0 if tree_mask is None else tree_mask.shape[1],
        k_scales=0 if k_scale is None else k_scale.numel(), v_scales=0 if v_scale is None else v_scale.numel(),
        scale=dim**-0.5 if scale is None else scale)
    lib = N.load()
    if T > 0 and B > 0:
        with N.on_device(q):
            # a block of the caching allocator: calls captured into two graphs may be replayed at the same time
            need = lib.b200_tree_attention_workspace_bytes(ctypes.addressof(a))
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            st = lib.b200_tree_attention(ctypes.addressof(a), N.ptr(ws), need, N.current_stream())
        N.check(st, "tree_attention")
    return (out, lse) if return_lse else out
