"""Calls that the operators between qkv and attention refuse (no GPU: a refusal comes before any launch)."""
import ctypes

import pytest
import torch

import sglang_b200 as S
from sglang_b200 import _native as N
from sglang_b200.rotary import RopeArgs

BF, FP8 = torch.bfloat16, torch.float8_e4m3fn


def good():
    """Arguments of qk_norm_rope_append that only lack a GPU."""
    return dict(qkv=torch.zeros(3, 12 * 64, dtype=BF), num_heads=8, num_kv_heads=2, positions=torch.arange(3), cos_sin_cache=torch.zeros(9, 64),
                k_cache=torch.zeros(4, 4, 2, 64, dtype=BF), v_cache=torch.zeros(4, 4, 2, 64, dtype=BF), slots=torch.arange(3),
                q_weight=torch.ones(64, dtype=BF), k_weight=torch.ones(64, dtype=BF))


def test_a_good_call_lacks_only_the_gpu():
    a = good()
    with pytest.raises(RuntimeError, match="no CPU path"):
        S.qk_norm_rope_append(**a)
    for n in ("k_cache", "v_cache", "slots"):
        del a[n]
    with pytest.raises(RuntimeError, match="no CPU path"):
        S.qk_norm_rope(**a)
    with pytest.raises(RuntimeError, match="no CPU path"):
        S.append_paged_kv(torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, 2, 64, dtype=BF), *(torch.zeros(4, 4, 2, 64, dtype=BF),) * 2, torch.arange(3))


BAD = {
    "double": dict(qkv=torch.zeros(3, 12 * 64, dtype=torch.float64)),
    "width": dict(qkv=torch.zeros(3, 12 * 64 + 1, dtype=BF)),
    "columns apart": dict(qkv=torch.zeros(3, 24 * 64, dtype=BF)[:, ::2]),
    "no heads": dict(num_kv_heads=0),
    "weight size": dict(q_weight=torch.ones(65, dtype=BF)),
    "weight type": dict(k_weight=torch.ones(64)),
    "float positions": dict(positions=torch.zeros(3)),
    "positions of another length": dict(positions=torch.arange(4)),
    "positions without a table": dict(cos_sin_cache=None),
    "16-bit table": dict(cos_sin_cache=torch.zeros(9, 64, dtype=BF)),
    "table wider than a head": dict(cos_sin_cache=torch.zeros(9, 66)),
    "odd table": dict(cos_sin_cache=torch.zeros(9, 63)),
    "one axis of positions for three": dict(mrope_section=[10, 11, 11]),
    "sections of another sum": dict(mrope_section=[10, 11, 10], positions=torch.zeros(3, 3, dtype=torch.int64)),
    "a negative section": dict(mrope_section=[40, -8], positions=torch.zeros(2, 3, dtype=torch.int64)),
    "an interleaved section that does not fit": dict(mrope_section=[6, 13, 13], mrope_interleaved=True,
                                                     positions=torch.zeros(3, 3, dtype=torch.int64)),
    "cache heads": dict(k_cache=torch.zeros(4, 4, 3, 64, dtype=BF)),
    "cache type": dict(k_cache=torch.zeros(4, 4, 2, 64, dtype=torch.float16), v_cache=torch.zeros(4, 4, 2, 64, dtype=torch.float16)),
    "caches of two types": dict(v_cache=torch.zeros(4, 4, 2, 64).to(FP8)),
    "caches of two sizes": dict(v_cache=torch.zeros(5, 4, 2, 64, dtype=BF)),
    "heads of a cache apart": dict(k_cache=torch.zeros(4, 4, 2, 128, dtype=BF)[..., ::2]),
    "float slots": dict(slots=torch.zeros(3)),
    "too few slots": dict(slots=torch.arange(2)),
    "scale of a 16-bit cache": dict(k_scale=torch.ones(1)),
    "16-bit scale": dict(k_cache=torch.zeros(4, 4, 2, 64).to(FP8), v_cache=torch.zeros(4, 4, 2, 64).to(FP8), k_scale=torch.ones(1, dtype=BF)),
    "scales per token": dict(k_cache=torch.zeros(4, 4, 2, 64).to(FP8), v_cache=torch.zeros(4, 4, 2, 64).to(FP8), v_scale=torch.ones(3)),
}


@pytest.mark.parametrize("what", BAD)
def test_refused(what):
    with pytest.raises(AssertionError):
        S.qk_norm_rope_append(**{**good(), **BAD[what]})


def test_five_axes_are_not_built():
    with pytest.raises(NotImplementedError):
        S.qk_norm_rope_append(**{**good(), "mrope_section": [8, 8, 8, 4, 4], "positions": torch.zeros(5, 3, dtype=torch.int64)})


def test_keys_and_values_have_to_match():
    c = torch.zeros(4, 4, 2, 64, dtype=BF)
    k = torch.zeros(3, 2, 64, dtype=BF)
    for a, b in ((k, k[:2]), (k, k.half()), (k[0], k[0]), (k.transpose(1, 2), k.transpose(1, 2))):
        with pytest.raises(AssertionError):
            S.append_paged_kv(a, b, c, c, torch.arange(3))


def test_abi_refuses_before_a_launch():
    lib = N.load()

    def call(**fields):
        sections = fields.pop("sections", [])
        a = RopeArgs(rows=3, q_heads=2, kv_heads=1, dim=64, **{**dict(dtype=N.BF16, q=64, k=64, q_out=64, k_out=64, axes=1), **fields})
        for i, n in enumerate(sections):
            a.sections[i] = n
        return lib.b200_qk_norm_rope(ctypes.addressof(a), None)

    bad = N.E_BAD_ARG
    assert lib.b200_qk_norm_rope(None, None) == bad
    assert call(rotated=7) == bad and call(rotated=66) == bad and call(rotated=64) == bad
    table = dict(rotated=64, positions=64, cos_sin=64, positions_dtype=N.I64, table_rows=4, cos_sin_ld=64)
    assert call(**{**table, "positions_dtype": N.F32}) == bad
    assert call(**{**table, "axes": 1, "cos_sin": 65}) == bad
    assert call(k_cache=64) == bad and call(slots=64) == bad
    cache = dict(k_cache=64, v_cache=64, slots=64, v=64, pages=4, page_size=4, slots_dtype=N.I64, cache_dtype=5)
    assert call(**{**cache, "cache_dtype": N.F16}) == bad and call(**{**cache, "page_size": 0}) == bad
    assert call(**{**cache, "k_scale": 64, "k_scales": 3}) == bad
    assert call(**{**cache, "cache_dtype": N.BF16, "k_scale": 64, "k_scales": 1}) == bad
    a = RopeArgs(rows=3, q_heads=2, kv_heads=1, dim=64, dtype=9, q=64, k=64, q_out=64, k_out=64)
    assert lib.b200_qk_norm_rope(ctypes.addressof(a), None) == bad
    a = RopeArgs(rows=0, q_heads=2, kv_heads=1, dim=64, dtype=N.BF16)
    assert lib.b200_qk_norm_rope(ctypes.addressof(a), None) == 0


def test_abi_has_nothing_to_do_without_heads():
    for heads in (dict(q_heads=0, kv_heads=3, q=64, q_out=64), dict(q_heads=3, kv_heads=0, k=64, k_out=64), dict(q=64, k=64, q_out=64, k_out=64)):
        a = RopeArgs(rows=3, dim=64, dtype=N.BF16, **heads)
        assert N.load().b200_qk_norm_rope(ctypes.addressof(a), None) == 0


def test_fake_implementations_describe_the_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import sglang_b200.custom_ops  # noqa: F401

    ops = torch.ops.sglang_b200
    with FakeTensorMode():
        x = torch.empty(5, 12 * 64, dtype=BF, device="cuda")
        cache = torch.empty(4, 16, 2, 64, dtype=BF, device="cuda")
        index = torch.empty(5, dtype=torch.int32, device="cuda")
        q, k = ops.qk_norm_rope(x, 8, 2, None, None)
        assert q.shape == (5, 8, 64) and k.shape == (5, 2, 64) and q.dtype == BF
        assert ops.qk_norm_rope_append(x, 8, 2, None, None, cache, cache.clone(), index).shape == (5, 8, 64)
        assert ops.append_paged_kv(k, k, cache, cache.clone(), index) is None
        assert ops.tree_attention(q, cache, cache, torch.empty(5, 3, dtype=torch.int32, device="cuda"), index).shape == q.shape


FAR = (1 << 32) + 16  # 16 in 32 bits


def test_sizes_past_32_bits_are_not_taken_for_their_low_bits():
    a = good()
    for n in ("k_cache", "v_cache"):
        a[n] = torch.zeros(1, 1, 2, 64, dtype=BF).expand(4, FAR, 2, 64)
    with pytest.raises(NotImplementedError):
        S.qk_norm_rope_append(**a)
    with pytest.raises(NotImplementedError):
        S.append_paged_kv(torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, 2, 64, dtype=BF), a["k_cache"], a["v_cache"], torch.arange(3))
    meta = dict(dtype=BF, device="meta")
    for heads, kv, dim in ((FAR, 2, 1), (8, FAR, 1), (8, 2, FAR)):
        with pytest.raises(NotImplementedError):
            S.qk_norm_rope(torch.empty(3, (heads + 2 * kv) * dim, **meta), heads, kv, None, None)
    k = torch.empty(3, FAR, 1, **meta)
    with pytest.raises(NotImplementedError):
        S.append_paged_kv(k, k, k, k, torch.arange(3))
