"""Calls that the attention over the paged cache refuses, and the size of its workspace (no GPU: a refusal comes before any launch)."""
import ctypes

import pytest
import torch

import sglang_b200 as S
from sglang_b200 import _native as N
from sglang_b200.attention import TreeAttentionArgs

BF, FP8 = torch.bfloat16, torch.float8_e4m3fn


def good():
    return dict(q=torch.zeros(5, 8, 128, dtype=BF), k_cache=torch.zeros(4, 16, 2, 128, dtype=BF), v_cache=torch.zeros(4, 16, 2, 128, dtype=BF),
                page_table=torch.zeros(2, 3, dtype=torch.int32), seq_lens=torch.ones(2, dtype=torch.int32), q_starts=torch.zeros(3, dtype=torch.int32),
                tree_mask=torch.ones(5, 4, dtype=torch.bool))


def test_a_good_call_lacks_only_the_gpu():
    with pytest.raises(RuntimeError, match="no CPU path"):
        S.tree_attention(**good())


FP8_CACHES = dict(k_cache=torch.zeros(4, 16, 2, 128).to(FP8), v_cache=torch.zeros(4, 16, 2, 128).to(FP8))
BAD = {
    "fp32 queries": dict(q=torch.zeros(5, 8, 128)),
    "flat queries": dict(q=torch.zeros(5, 8 * 128, dtype=BF)),
    "heads that do not divide": dict(q=torch.zeros(5, 7, 128, dtype=BF)),
    "another head size": dict(q=torch.zeros(5, 8, 64, dtype=BF)),
    "elements of a head apart": dict(q=torch.zeros(5, 8, 256, dtype=BF)[..., ::2]),
    "another type of cache": dict(k_cache=torch.zeros(4, 16, 2, 128, dtype=torch.float16), v_cache=torch.zeros(4, 16, 2, 128, dtype=torch.float16)),
    "caches of two types": dict(k_cache=FP8_CACHES["k_cache"]),
    "caches of two sizes": dict(v_cache=torch.zeros(5, 16, 2, 128, dtype=BF)),
    "elements of a cached head apart": dict(v_cache=torch.zeros(4, 16, 2, 256, dtype=BF)[..., ::2]),
    "64-bit pages": dict(page_table=torch.zeros(2, 3, dtype=torch.int64)),
    "pages apart": dict(page_table=torch.zeros(2, 6, dtype=torch.int32)[:, ::2]),
    "lengths of another batch": dict(seq_lens=torch.ones(3, dtype=torch.int32)),
    "64-bit lengths": dict(seq_lens=torch.ones(2, dtype=torch.int64)),
    "starts without the end": dict(q_starts=torch.zeros(2, dtype=torch.int32)),
    "starts of every second element": dict(q_starts=torch.zeros(6, dtype=torch.int32)[::2]),
    "five tokens, two sequences, no starts": dict(q_starts=None),
    "a mask of other tokens": dict(tree_mask=torch.ones(4, 4, dtype=torch.bool)),
    "a mask of bytes": dict(tree_mask=torch.ones(5, 4, dtype=torch.uint8)),
    "a mask read across": dict(tree_mask=torch.ones(4, 5, dtype=torch.bool).t()),
    "scale of a 16-bit cache": dict(k_scale=torch.ones(1)),
    "a scale per token": dict(v_scale=torch.ones(5), **FP8_CACHES),
    "a 16-bit scale": dict(v_scale=torch.ones(2, dtype=BF), **FP8_CACHES),
    "an output of another shape": dict(out=torch.zeros(5, 8, 64, dtype=BF)),
    "an output of another type": dict(out=torch.zeros(5, 8, 128)),
    "an output with gaps": dict(out=torch.zeros(5, 16, 128, dtype=BF)[:, ::2]),
}


@pytest.mark.parametrize("what", BAD)
def test_refused(what):
    with pytest.raises(AssertionError):
        S.tree_attention(**{**good(), **BAD[what]})


def args(**fields):
    base = dict(q=64, out=64, k_cache=64, v_cache=64, page_table=64, seq_lens=64, q_token=1024, q_head=128, k_page=4096, k_token=256, k_head=128,
                v_page=4096, v_token=256, v_head=128, pages=4, page_table_ld=3, max_pages=3, tokens=5, sequences=5, q_heads=8, kv_heads=2, dim=128,
                dtype=N.BF16, page_size=16, cache_dtype=N.BF16, scale=1.0)
    return TreeAttentionArgs(**{**base, **fields})


def call(**fields):
    return N.load().b200_tree_attention(ctypes.byref(args(**fields)), None, 0, None)


def test_abi_refuses_before_a_launch():
    bad = N.E_BAD_ARG
    assert N.load().b200_tree_attention(None, None, 0, None) == bad
    assert call() == N.E_WORKSPACE
    assert call(tokens=0) == 0 and call(sequences=0) == 0
    for f in (dict(q_heads=7), dict(kv_heads=0), dict(tokens=-1), dict(dtype=N.F32), dict(cache_dtype=N.F16), dict(page_size=0), dict(q=None),
              dict(out=None), dict(seq_lens=None), dict(page_table=None), dict(k_cache=None), dict(q=72), dict(v_cache=80 - 8), dict(q_head=130),
              dict(k_token=130), dict(v_page=4), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(k_scale=64, k_scales=1),
              dict(cache_dtype=5, k_scale=64, k_scales=3), dict(cache_dtype=5, k_token=8), dict(mask=64, mask_width=-1), dict(lse=66)):
        assert call(**f) == bad, f
    for f in (dict(dim=96), dict(tokens=1 << 30), dict(page_size=1 << 20, max_pages=1 << 20)):
        assert call(**f) == N.E_UNSUPPORTED, f


def test_distances_that_lead_nowhere_are_not_checked():
    assert call(tokens=1, sequences=1, q_token=1028) == call(q_heads=1, kv_heads=1, q_head=1, k_head=3, v_head=5) == N.E_WORKSPACE
    assert call(pages=1, k_page=1, v_page=3) == call(page_size=1, k_token=1, v_token=3) == N.E_WORKSPACE


def test_workspace():
    size = lambda **f: N.load().b200_tree_attention_workspace_bytes(ctypes.byref(args(**f)))  # noqa: E731
    assert size() > 0 and size(tokens=0) == 0 and size(dim=100) == 0
    # two pieces of a row tile for each of at most 148 CTAs: 16 rows where a sequence has 4, 128 where it may have more than 64
    for rows, f in ((16, {}), (128, dict(q_starts=64)), (32, dict(q_starts=64, mask=64, mask_width=7))):
        big = size(tokens=100000, sequences=1000, max_pages=10000, pages=10000, **f)
        assert big == size(tokens=200000, sequences=2000, max_pages=20000, pages=10000, **f)
        assert 2 * 148 * rows * (128 + 2) * 4 <= big < 2 * 148 * rows * (128 + 2) * 4 + 16384


def test_sizes_past_32_bits_are_not_taken_for_their_low_bits():
    far, meta = (1 << 32) + 64, dict(dtype=BF, device="meta")
    cache = torch.zeros(1, 1, 2, 128, dtype=BF).expand(4, far, 2, 128)
    for bad in (dict(k_cache=cache, v_cache=cache), dict(tree_mask=torch.empty(5, far, dtype=torch.bool, device="meta")),
                dict(q=torch.empty(5, 8, far, **meta), k_cache=torch.empty(4, 16, 2, far, **meta), v_cache=torch.empty(4, 16, 2, far, **meta)),
                dict(q=torch.empty(5, far, 128, **meta))):
        with pytest.raises(NotImplementedError):
            S.tree_attention(**{**good(), **bad})
