"""Refusals of the int8 and norm operators: none of them needs a GPU."""
import pytest
import torch

import sglang_b200 as S
from sglang_b200 import _native as N


def a_b(M=4, n=64, K=64):
    return (torch.zeros(M, K, dtype=torch.int8), torch.zeros(n, K, dtype=torch.int8).t(), torch.ones(M, 1), torch.ones(n, 1))


def test_cpu_tensors_are_refused():
    a, b, sa, sb = a_b()
    x, w = torch.zeros(2, 256).bfloat16(), torch.zeros(256).bfloat16()
    for call in (lambda: S.int8_scaled_mm(a, b, sa, sb, torch.bfloat16), lambda: S.per_token_quant_int8(x),
                 lambda: S.rmsnorm_quant_int8(x, w), lambda: S.rmsnorm_quant_fp8(x, w, residual=x),
                 lambda: S.w8a8_int8_linear(x, torch.zeros(8, 256, dtype=torch.int8), torch.ones(8))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("change", [
    dict(mat_a=torch.zeros(4, 64)), dict(mat_a=torch.zeros(64, 4, dtype=torch.int8).t()), dict(mat_a=torch.zeros(4, 32, dtype=torch.int8)),
    dict(mat_a=torch.zeros(4, 64, 1, dtype=torch.int8)), dict(mat_b=torch.zeros(64, 64, dtype=torch.int8)),
    dict(scales_a=torch.ones(3)), dict(scales_a=torch.ones(4).double()), dict(scales_b=torch.ones(1)), dict(scales_b=torch.ones(128)[::2]),
    dict(out_dtype=torch.int32), dict(bias=torch.zeros(64)), dict(bias=torch.zeros(32).bfloat16())])
def test_product_refuses(change):
    a, b, sa, sb = a_b()
    args = {**dict(mat_a=a, mat_b=b, scales_a=sa, scales_b=sb, out_dtype=torch.bfloat16), **change}
    with pytest.raises(AssertionError):
        S.int8_scaled_mm(**args)


def test_norm_and_quantiser_refuse():
    x, w = torch.zeros(2, 256).bfloat16(), torch.zeros(256).bfloat16()
    for call in (lambda: S.rmsnorm_quant_int8(x, w.half()), lambda: S.rmsnorm_quant_int8(x, w[:128]), lambda: S.rmsnorm_quant_int8(x, w, residual=x[:1]),
                 lambda: S.rmsnorm_quant_int8(x, w, residual=x.half()), lambda: S.rmsnorm_quant_int8(x.double(), w.double()),
                 lambda: S.rmsnorm_quant_int8(x[:, :0], w[:0]), lambda: S.rmsnorm_quant_fp8(x[:, :200], w[:200]),
                 lambda: S.rmsnorm_quant_fp8(x, w, scale_ue8m0=True), lambda: S.rmsnorm_quant_fp8(x.view(2, 1, 256), w, column_major_scales=True),
                 lambda: S.per_token_quant_int8(x.to(torch.int8)), lambda: S.per_token_quant_int8(x[:, :255], fuse_silu_and_mul=True),
                 lambda: S.per_token_quant_int8(x.t()), lambda: S.per_token_quant_int8(x.view(2, 2, 128)[:, :, ::2]), lambda: S.per_token_quant_int8(x[:, :0]),
                 lambda: S.w8a8_int8_linear(x.float(), torch.zeros(8, 256, dtype=torch.int8), torch.ones(8))):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(NotImplementedError):
        S.rmsnorm_quant_fp8(x, w, group_size=64)
    with pytest.raises(NotImplementedError):
        S.per_token_quant_int8(x, cal_sum=True)
    with pytest.raises(NotImplementedError):
        S.per_token_quant_int8(x, scale_dtype=torch.bfloat16)


def test_dispatcher_ops_describe_their_results():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.sglang_b200
    schema = ops.int8_scaled_mm.default._schema
    assert [(a.name, str(a.type)) for a in schema.arguments] == [
        ("mat_a", "Tensor"), ("mat_b", "Tensor"), ("scales_a", "Tensor"), ("scales_b", "Tensor"), ("out_dtype", "int"), ("bias", "Optional[Tensor]")]
    with FakeTensorMode():
        x, w = torch.empty(6, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(512, dtype=torch.bfloat16, device="cuda")
        q, s, r = ops.rmsnorm_quant_int8(x, w, 1e-6, x)
        assert (q.dtype, q.shape, s.shape, r.dtype) == (torch.int8, (6, 512), (6, 1), torch.bfloat16)
        q, s = ops.rmsnorm_quant_fp8(x, w, 128, 1e-6, None, True, True, True)
        assert (q.dtype, s.dtype, s.shape, s.stride()) == (torch.float8_e4m3fn, torch.int32, (6, 1), (1, 8))
        q, s = ops.per_token_quant_int8(x, True)
        assert q.shape == (6, 256) and s.shape == (6, 1)
        out = ops.int8_scaled_mm(q, torch.empty(64, 256, dtype=torch.int8, device="cuda").t(), s, torch.empty(64, 1, device="cuda"),
                                 torch.float16, None)
        assert out.shape == (6, 64) and out.dtype == torch.float16
    with pytest.raises(NotImplementedError):
        ops.per_token_quant_int8(torch.zeros(2, 16))


def test_linear_method_loads_a_checkpoint():
    from sglang_b200.int8 import W8A8Int8Config, W8A8Int8LinearMethod, quant_weight_int8

    cfg = W8A8Int8Config.from_config({"quant_method": "w8a8_int8", "ignore": ["lm_head"]})
    assert cfg.get_name() == "w8a8_int8" and cfg.is_layer_skipped("lm_head") and not cfg.is_layer_skipped("model.layers.0.mlp")
    with pytest.raises(NotImplementedError):
        W8A8Int8Config.from_config({"is_dynamic": False})
    method, layer = W8A8Int8LinearMethod(cfg), torch.nn.Module()
    method.create_weights(layer, 64, [32, 16], 64, 48, torch.bfloat16)
    with pytest.raises(AssertionError):
        method.process_weights_after_loading(layer)  # nothing loaded
    w = torch.randn(48, 64, generator=torch.Generator().manual_seed(0))
    q, s = quant_weight_int8(w)
    assert ((q.float() * s - w).abs() <= s / 2 * (1 + 2.0**-20)).all() and (q.abs().amax(1) == 127).all()
    layer.load_state_dict({"weight": q, "weight_scale": s})
    method.process_weights_after_loading(layer)
    assert torch.equal(layer.weight, q) and torch.equal(layer.weight_scale, s)


FAKE = 1 << 20  # an aligned address that no refused call reads


def mm(a=FAKE, lda=64, b=FAKE, ldb=64, sa=FAKE, sb=FAKE, c=FAKE, dtype=0, M=4, n=64, K=64, bias=0):
    return N.load().b200_int8_scaled_mm(a, lda, sa, b, ldb, sb, bias, c, dtype, M, n, K, None)


@pytest.mark.parametrize("kw,status", [
    (dict(a=None), N.E_BAD_ARG), (dict(sb=None), N.E_BAD_ARG), (dict(dtype=3), N.E_BAD_ARG), (dict(M=-1), N.E_BAD_ARG),
    (dict(K=0), N.E_BAD_ARG), (dict(lda=32), N.E_BAD_ARG), (dict(ldb=48), N.E_BAD_ARG), (dict(c=FAKE + 8), N.E_BAD_ARG), (dict(sa=FAKE + 2), N.E_BAD_ARG),
    (dict(bias=FAKE + 1), N.E_BAD_ARG), (dict(bias=FAKE + 2, dtype=2), N.E_BAD_ARG),
    (dict(K=72, lda=80, ldb=80), N.E_UNSUPPORTED), (dict(lda=72), N.E_UNSUPPORTED), (dict(ldb=65), N.E_UNSUPPORTED),
    (dict(a=FAKE + 8), N.E_UNSUPPORTED), (dict(b=FAKE + 1), N.E_UNSUPPORTED), (dict(n=65), N.E_UNSUPPORTED), (dict(n=4), N.E_UNSUPPORTED),
    (dict(K=131072, lda=131072, ldb=131072), N.E_UNSUPPORTED), (dict(M=1 << 40), N.E_UNSUPPORTED), (dict(M=0, a=None), 0), (dict(n=0), 0)])
def test_c_entry_of_the_product(kw, status):
    assert mm(**kw) == status, N.load().b200_last_error_detail()


def test_c_entries_of_the_row_kernels():
    lib = N.load()

    def norm(x=FAKE, r=0, w=FAKE, dtype=0, kind=0, q=FAKE, s=FAKE, ro=0, M=2, H=256):
        return lib.b200_rmsnorm_quant(x, H, r, H, w, dtype, kind, q, s, 2, 1, ro, M, H, 1e-6, None)

    bad = [dict(x=None), dict(w=None), dict(s=None), dict(dtype=4), dict(kind=3), dict(M=-1), dict(r=FAKE), dict(ro=FAKE), dict(kind=1, H=200),
           dict(kind=2, H=64), dict(x=FAKE + 1), dict(kind=1, q=FAKE + 8), dict(s=FAKE + 1)]
    assert [norm(**k) for k in bad] == [N.E_BAD_ARG] * len(bad)
    assert norm(H=(1 << 24) + 2) == N.E_UNSUPPORTED and norm(M=0) == 0 and norm(M=1 << 33) == N.E_UNSUPPORTED

    def quant(x=FAKE, dtype=0, q=FAKE, s=FAKE, M=2, K=256):
        return lib.b200_per_token_quant_int8(x, K, dtype, q, s, M, K, 0, None)

    bad = [dict(x=None), dict(q=None), dict(dtype=3), dict(K=-1), dict(x=FAKE + 1), dict(s=FAKE + 2)]
    assert [quant(**k) for k in bad] == [N.E_BAD_ARG] * len(bad)
    assert quant(K=(1 << 24) + 2) == N.E_UNSUPPORTED and quant(M=1 << 33) == N.E_UNSUPPORTED and quant(K=0) == 0


def test_codes_as_the_kernels_round_them():
    """The quotient by one residual step, and the whole number that adding 1.5 * 2^23 leaves, are the IEEE quotient's nearest integer:
    every pair of bf16 mantissas down to 1/512 of the row's largest magnitude."""
    import numpy as np

    f = np.float32
    m = (1 + np.arange(128) / 128).astype(f)
    small = np.concatenate([m * f(2.0**-e) for e in range(10)])
    for top in m:
        x = small[small <= top]
        s = f(top / f(127))
        r = f(1) / s
        fma = lambda a, b, c: (a.astype(np.float64) * np.float64(b) + c.astype(np.float64)).astype(f)  # noqa: E731
        q = (x * r).astype(f)
        rest = (x.astype(np.float64) - q.astype(np.float64) * np.float64(s)).astype(f)  # exact: the products have 48 bits
        q = fma(rest, r, q)
        whole = (q + f(12582912)).view(np.uint32).astype(np.uint8).view(np.int8)
        assert np.array_equal(whole, np.rint(x / s).astype(np.int8))


def test_plan():
    """Every size, known or odd, gets a kernel that can run it: no empty split, tiles within the kernels' limits, and few rows stream."""
    import random

    rng = random.Random(0)
    for _ in range(3000):
        M, n, K = (int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(3, 16)) // 8 * 8, int(2 ** rng.uniform(4, 17)) // 16 * 16)
        K = min(K, 131056)
        pl = N.plan_int8(M, n, K, rng.choice([148, 148, 132, 16, 1]))
        kbs = -(-K // 128)
        assert 1 <= pl.splits <= 8 and -(-kbs // -(-kbs // pl.splits)) == pl.splits, (M, n, K, pl)
        if pl.kernel != "stream":
            assert pl.tile in range(32, 257, 32) and pl.splits in (1, 2, 4) and M > 32
        else:
            assert pl.tile in range(16, 257, 16) and pl.tile < M + 16
    assert N.plan_int8(1, 4096, 4096, 148) == ("stream", 16, 4)
    assert N.plan_int8(8192, 28672, 4096, 148) == ("pair", 256, 1)
    with N.tuning(int8_tile=64, int8_splits=8):
        assert N.plan_int8(100, 4096, 256, 148) == ("stream", 64, 2)
    with N.tuning(int8_tile=1128, int8_splits=3):
        assert N.plan_int8(100, 4096, 4096, 148) == ("pair", 128, 1)
    with N.tuning(int8_tile=2224):
        assert N.plan_int8(100, 4096, 4096, 148) == ("swapped", 224, 1)
    assert N.load().b200_plan_int8(0, 8, 16, 148, None, None, None) == N.E_BAD_ARG
