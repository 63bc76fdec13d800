"""Norm and quantiser kernels against their definitions in 64 bits: codes, scales, the residual, rows of every width class.

Tolerances, from the arithmetic (u = 2^-24, the rounding of fp32):
  * h = x + r and h * w round once each; the sum of squares is a tree of at most 2^7 sequential additions and 10 levels, so
    rsqrt(mean) is off by at most 70 u + 2 ulp, and a scale by less than 2^-17 relative.
  * a code's quotient y / s is off by at most 8 u relative, as rsqrt(mean) is in both: an int8 code is within 0.5 + 127 * 2^-21
    of the quotient, an FP8 code within half of its step.
  * silu's exponential is off by |gate| * 2^-23 at most: 2^-16 for every gate whose silu is not lost beside the row's largest."""
import pytest
import torch

import sglang_b200 as S

pytestmark = pytest.mark.gpu
U = 2.0**-24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def draw(rows, width, dtype, seed, ld=None, outliers=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, ld or width, generator=g)
    if outliers:
        x[:, :: max(2, width // 7)] *= 20
    return x.to(dtype).cuda()[:, :width]


def normed(x, r, w, eps):
    h = x.double() if r is None else x.double() + r.double()
    return h * w.double() / (h.square().mean(-1, keepdim=True) + eps).sqrt(), h


def check_int8(q, s, y, extra=0.0):
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and s.shape == (*q.shape[:-1], 1)
    want = y.abs().amax(-1, keepdim=True).clamp_min(1e-10) / 127
    assert ((s.double() - want).abs() <= (2.0**-17 + extra) * want).all()
    off = (q.double() - y / want).abs()
    assert off.max() <= 0.5 + 127 * (2.0**-21 + extra), off.max()
    assert (q.abs().amax(-1) == 127).logical_or(want.squeeze(-1) <= 1e-12).all()


def check_residual(out, h, dtype):
    assert out.dtype == dtype
    assert ((out.double() - h).abs() <= (torch.finfo(dtype).eps / 2 + U) * h.abs() + 2.0**-25).all()


def half_step(v):
    return 2.0 ** (v.abs().clamp_min(2.0**-6).log2().floor() - 4)


def unpack(s, groups):
    b = ((s.long().unsqueeze(-1) >> torch.arange(0, 32, 8, device=s.device)) & 255).flatten(1)
    assert (b[:, groups:] == 0).all()
    return b[:, :groups].double() - 127


def check_fp8(q, s, y, ue8m0):
    rows, width = y.shape
    y = y.view(rows, -1, 128)
    want = y.abs().amax(-1).clamp_min(1e-10) / 448
    if ue8m0:
        e = unpack(s, width // 128)
        lo = (want * (1 - 2.0**-17)).log2().ceil()
        hi = (want * (1 + 2.0**-17)).log2().ceil()
        assert ((e == lo) | (e == hi)).all()
        scale = 2.0**e
    else:
        assert s.shape == want.shape and ((s.double() - want).abs() <= 2.0**-17 * want).all()
        scale = want
    v = (y / scale.unsqueeze(-1)).clamp(-448, 448)
    off = (q.double().view_as(y) - v).abs()
    assert (off <= half_step(v) * (1 + 2.0**-14) + 448 * 2.0**-21).all()


WIDTHS = [1, 2, 7, 8, 31, 100, 128, 255, 256, 520, 1000, 1024, 2048, 4096, 4104, 7168, 8192, 8193, 14336, 16384, 20000, 32768, 33000]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_int8(width, dtype):
    for rows, with_res in ((1, True), (3, False), (7, True)):
        x, w = draw(rows, width, dtype, width + rows), draw(1, width, dtype, 5, outliers=False)[0]
        r = draw(rows, width, dtype, width + rows + 9) if with_res else None
        q, s, *res = S.rmsnorm_quant_int8(x, w, 1e-6, residual=r)
        y, h = normed(x, r, w, 1e-6)
        check_int8(q, s, y)
        assert len(res) == int(with_res)
        if with_res:
            check_residual(res[0], h, dtype)


@pytest.mark.parametrize("width", [w for w in WIDTHS if w % 128 == 0] + [384, 5120, 24576])
@pytest.mark.parametrize("scales", ["row", "col", "aligned", "ue8m0"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_fp8(width, scales, dtype):
    for rows, with_res in ((1, False), (2, True), (5, True)):
        x, w = draw(rows, width, dtype, width + rows), draw(1, width, dtype, 5, outliers=False)[0]
        r = draw(rows, width, dtype, width + rows + 9) if with_res else None
        q, s, *res = S.rmsnorm_quant_fp8(x, w, 128, 1e-5, residual=r, column_major_scales=scales != "row",
                                         scale_tma_aligned=scales in ("aligned", "ue8m0"), scale_ue8m0=scales == "ue8m0")
        y, h = normed(x, r, w, 1e-5)
        assert q.dtype == torch.float8_e4m3fn
        if scales != "row" and rows > 1:
            assert s.stride(0) == 1 and (scales == "col" or s.stride(1) % 4 == 0)
        check_fp8(q.float(), s, y, scales == "ue8m0")
        if with_res:
            check_residual(res[0], h, dtype)


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quant_int8_is_the_ieee_quotient(width, dtype):
    """Bit for bit: scale and quotient are IEEE divisions, codes the nearest integers, ties to even."""
    for rows in (1, 5):
        x = draw(rows, width, dtype, width + rows)
        q, s = S.per_token_quant_int8(x)
        c = x.float().cpu()
        want = c.abs().amax(-1, keepdim=True).clamp_min(1e-10) / torch.tensor(127.0)
        assert torch.equal(s.cpu(), want)
        assert torch.equal(q.cpu(), (c / want).round().to(torch.int8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quant_int8_every_pair_of_mantissas(dtype):
    """Every mantissa of the row's largest magnitude against every mantissa of a value down to 1/512 of it."""
    bits = 7 if dtype == torch.bfloat16 else 10
    m = 1 + torch.arange(2**bits) / 2**bits
    small = torch.cat([m * 2.0**-e for e in range(10)])
    for top in m.split(64):
        x = small[None, :].repeat(len(top), 1)
        x[x > top[:, None]] = 0
        x = torch.cat([top[:, None], x, -x], 1).to(dtype)
        q, s = S.per_token_quant_int8(x.cuda())
        want = x.float().abs().amax(-1, keepdim=True) / torch.tensor(127.0)
        assert torch.equal(s.cpu(), want)
        assert torch.equal(q.cpu(), (x.float() / want).round().to(torch.int8))


@pytest.mark.parametrize("width", [64, 100, 4096])
def test_smallest_and_largest_values(width):
    """Rows of nothing but subnormal fp16 numbers, and of the largest that each type has."""
    g = torch.Generator().manual_seed(width)
    for dtype, size in ((torch.float16, 2.0**-17), (torch.float16, 60000.0), (torch.bfloat16, 3e38), (torch.float32, 3e38), (torch.bfloat16, 1e-9)):
        x = ((torch.rand(3, width, generator=g) * 2 - 1) * size).to(dtype)
        q, s = S.per_token_quant_int8(x.cuda())
        want = x.float().abs().amax(-1, keepdim=True).clamp_min(1e-10) / torch.tensor(127.0)
        assert torch.equal(s.cpu(), want) and torch.equal(q.cpu(), (x.float() / want).round().to(torch.int8))


@pytest.mark.parametrize("width", [1, 7, 8, 100, 128, 1000, 2048, 3584, 14336, 14337, 28672, 33000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_silu_quant_int8(width, dtype):
    for rows in (1, 4):
        x = draw(rows, 2 * width, dtype, width + rows)
        q, s = S.per_token_quant_int8(x, fuse_silu_and_mul=True)
        gate, up = x.double().chunk(2, -1)
        check_int8(q, s, gate / (1 + (-gate).exp()) * up, extra=2.0**-16)


@pytest.mark.parametrize("flag", [1, "gate"])
def test_any_true_value_fuses_the_gate(flag):
    x = draw(3, 512, torch.bfloat16, 4)
    assert all(torch.equal(a, b) for a, b in zip(S.per_token_quant_int8(x, fuse_silu_and_mul=flag), S.per_token_quant_int8(x, fuse_silu_and_mul=True)))


def test_leading_dimensions_and_empty_inputs():
    x, w = draw(6, 256, torch.bfloat16, 1).view(2, 3, 256), draw(1, 256, torch.bfloat16, 2)[0]
    q, s, r = S.rmsnorm_quant_int8(x, w, residual=x)
    q2, s2, r2 = S.rmsnorm_quant_int8(x.view(6, 256), w, residual=x.view(6, 256))
    assert q.shape == x.shape and s.shape == (2, 3, 1) and torch.equal(q.view(6, 256), q2) and torch.equal(r.view(6, 256), r2)
    q, s = S.rmsnorm_quant_fp8(x, w)
    assert q.shape == x.shape and s.shape == (2, 3, 2)
    q, s = S.per_token_quant_int8(x[0, 0])
    assert q.shape == (256,) and s.shape == (1,)
    for fn in (lambda t: S.rmsnorm_quant_int8(t, w, residual=t), lambda t: S.rmsnorm_quant_fp8(t, w, residual=t), S.per_token_quant_int8):
        out = fn(x.view(6, 256)[:0])
        assert all(t.shape[0] == 0 for t in out)


@pytest.mark.parametrize("offset", [0, 8, 16, 3])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_wider_tensors(offset, dtype):
    """Slices of wider rows, aligned to 16 bytes or not."""
    wide = draw(9, 2 * 1152 + 40, dtype, 3)
    x, r, w = wide[:, offset : offset + 1152], wide[:, offset + 1152 : offset + 2304], draw(1, 1152, dtype, 4)[0]
    y, h = normed(x, r, w, 1e-6)
    q, s, res = S.rmsnorm_quant_int8(x, w, residual=r)
    check_int8(q, s, y)
    check_residual(res, h, dtype)
    q, s, res = S.rmsnorm_quant_fp8(x, w, residual=r)
    check_fp8(q.float(), s, y, False)
    check_residual(res, h, dtype)
    for got, want in zip(S.per_token_quant_int8(x), S.per_token_quant_int8(x.contiguous())):
        assert torch.equal(got, want)
    gate, up = x.double().chunk(2, -1)
    check_int8(*S.per_token_quant_int8(x, fuse_silu_and_mul=True), gate / (1 + (-gate).exp()) * up, extra=2.0**-16)


@pytest.mark.parametrize("width", [128, 1000, 4096, 16384, 33024])
def test_zero_rows_nan_and_infinity(width):
    x = draw(6, width, torch.bfloat16, 8)
    x[0] = 0
    x[1, width // 2] = float("nan")
    x[2, 0] = float("inf")
    x[4, -1] = float("nan")
    w = draw(1, width, torch.bfloat16, 9, outliers=False)[0]
    clean = S.per_token_quant_int8(x[3:4].contiguous())
    q, s = S.per_token_quant_int8(x)
    assert (q[0] == 0).all() and s[0] == torch.tensor(1e-10) / torch.tensor(127.0)
    assert s[1].isnan() and s[4].isnan() and s[2].isinf()
    assert torch.equal(q[3], clean[0][0]) and torch.equal(s[3], clean[1][0])
    q, s = S.rmsnorm_quant_int8(x, w)
    assert (q[0] == 0).all() and s[0] > 0 and s[1].isnan() and s[2].isnan() and s[4].isnan() and s[3].isfinite() and s[5].isfinite()
    if width % 128 == 0:
        q, s = S.rmsnorm_quant_fp8(x, w)
        f = q.float()
        assert (f[0] == 0).all() and f[1].isnan().all() and f[4].isnan().all() and f[2, 0].isnan() and f[[3, 5]].isfinite().all()


@pytest.mark.parametrize("vectors", [1, 2, 4, 8])
@pytest.mark.parametrize("width", [8, 128, 264, 1024, 4096, 8192, 16384, 24576])
def test_every_number_of_vectors_per_thread(vectors, width):
    from sglang_b200 import _native as N

    x, r, w = draw(6, width, torch.bfloat16, 1), draw(6, width, torch.bfloat16, 2), draw(1, width, torch.bfloat16, 3)[0]
    y, h = normed(x, r, w, 1e-6)
    with N.tuning(row_vectors=vectors):
        q, s, res = S.rmsnorm_quant_int8(x, w, residual=r)
        check_int8(q, s, y)
        check_residual(res, h, torch.bfloat16)
        if width % 128 == 0:
            q, s, res = S.rmsnorm_quant_fp8(x, w, residual=r, column_major_scales=True)
            check_fp8(q.float(), s, y, False)
        gate, up = x.double().chunk(2, -1)
        if width % 16 == 0:
            check_int8(*S.per_token_quant_int8(x, fuse_silu_and_mul=True), gate / (1 + (-gate).exp()) * up, extra=2.0**-16)
        q, s = S.per_token_quant_int8(x)
    assert torch.equal(q.float().cpu(), (x.float().cpu() / s.cpu()).round())


def test_many_rows_and_repeats():
    """More rows than blocks fit the chip, the same bits on every run."""
    x, r, w = draw(5000, 1024, torch.bfloat16, 1), draw(5000, 1024, torch.bfloat16, 2), draw(1, 1024, torch.bfloat16, 3)[0]
    a, b = S.rmsnorm_quant_int8(x, w, residual=r), S.rmsnorm_quant_int8(x, w, residual=r)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    y, h = normed(x, r, w, 1e-6)
    check_int8(a[0], a[1], y)
    check_residual(a[2], h, torch.bfloat16)
    q, s = S.rmsnorm_quant_fp8(x, w, residual=r, column_major_scales=True)[:2]
    check_fp8(q.float(), s, y, False)


@pytest.mark.parametrize("rows,width,pad", [(19001, 1024, 0), (7105, 4096, 0), (7777, 4104, 24), (2500, 8192, 0), (1777, 14336, 0), (1801, 16384, 8),
                                            (3003, 20000, 0), (4000, 28672, 0), (1999, 2048, 0), (9400, 7168, 8)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_prefills(rows, width, pad, dtype):
    """Thousands of wide rows: plain ones bit for bit, gated ones by their definition."""
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    x = torch.randn(rows, width + pad, generator=g, device="cuda").to(dtype)[:, :width]
    x[rows // 2, width // 3], x[rows - 1] = float("nan"), 0
    q, s = S.per_token_quant_int8(x)
    f = x.float()
    want = f.abs().amax(-1, keepdim=True).clamp_min(1e-10) / torch.full((), 127.0, device="cuda")
    fine = ~want.isnan().squeeze(-1)
    assert s.isnan().sum() == 1 and torch.equal(s.isnan(), want.isnan()) and torch.equal(s[fine], want[fine])
    assert torch.equal(q[fine], (f / want).round()[fine].to(torch.int8))
    del f, want
    if width % 16 == 0:
        q, s = S.per_token_quant_int8(x, fuse_silu_and_mul=True)
        for part in torch.arange(rows, device="cuda")[fine].split(2000):
            gate, up = x[part].double().chunk(2, -1)
            check_int8(q[part], s[part], gate / (1 + (-gate).exp()) * up, extra=2.0**-16)


@pytest.mark.parametrize("width", [128, 512, 1024, 1152, 8192, 11904, 12032, 14336])
@pytest.mark.parametrize("dtype", DTYPES)
def test_unaligned_rows_of_every_width(width, dtype):
    """Rows that start off the 16-byte boundaries: narrow ones, those whose values are kept and those too wide for that."""
    wide = draw(3, 2 * width + 2, dtype, width)
    x, r, w = wide[:, 1 : 1 + width], wide[:, 1 + width : 1 + 2 * width], draw(1, width, dtype, 5, outliers=False)[0]
    y, h = normed(x, r, w, 1e-6)
    q, s, out = S.rmsnorm_quant_int8(x, w, 1e-6, residual=r)
    check_int8(q, s, y)
    check_residual(out, h, dtype)
    for ue8m0 in (False, True):
        q, s, out = S.rmsnorm_quant_fp8(x, w, 128, 1e-6, residual=r, column_major_scales=ue8m0, scale_tma_aligned=ue8m0, scale_ue8m0=ue8m0)
        check_fp8(q.float(), s, y, ue8m0)
        check_residual(out, h, dtype)
    q, s = S.per_token_quant_int8(wide[:, 1 : 1 + 2 * width], fuse_silu_and_mul=True)
    gate, up = x.double(), r.double()
    check_int8(q, s, gate / (1 + (-gate).exp()) * up, extra=2.0**-16)


def test_offsets_past_31_bits():
    """Rows that lie more than 2^31 elements into their tensors."""
    rows, width = 270000, 8192
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    x[-3:] = draw(3, width, torch.bfloat16, 5)
    w = draw(1, width, torch.bfloat16, 6, outliers=False)[0]
    q, s = S.per_token_quant_int8(x)
    assert torch.equal(q[-3:], S.per_token_quant_int8(x[-3:].contiguous())[0]) and (s[:-3] < 1e-11).all()
    del q, s
    q, s, r = S.rmsnorm_quant_fp8(x, w, residual=x, column_major_scales=True)
    q2, s2, r2 = S.rmsnorm_quant_fp8(x[-3:].contiguous(), w, residual=x[-3:].contiguous(), column_major_scales=True)
    assert torch.equal(q[-3:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[-3:], s2) and torch.equal(r[-3:], r2)


def test_nothing_is_written_behind_the_last_row():
    from sglang_b200 import _native as N

    lib, rows = N.load(), 5
    for width in (100, 1000, 1152, 4096, 33000):
        x, w = draw(rows, width, torch.bfloat16, 1), draw(1, width, torch.bfloat16, 2)[0]
        q = torch.full((rows + 1, width), 77, dtype=torch.int8, device="cuda")
        res = torch.full((rows + 1, width), 77, dtype=torch.bfloat16, device="cuda")
        s = torch.full((rows + 1,), 77.0, device="cuda")
        N.check(lib.b200_rmsnorm_quant(N.ptr(x), width, N.ptr(x), width, N.ptr(w), N.BF16, 0, N.ptr(q), N.ptr(s), 1, 0, N.ptr(res),
                                       rows, width, 1e-6, N.current_stream()), "rmsnorm_quant")
        assert (q[rows] == 77).all() and (res[rows] == 77).all() and s[rows] == 77
        N.check(lib.b200_per_token_quant_int8(N.ptr(x), width, N.BF16, N.ptr(q), N.ptr(s), rows, width, 0, N.current_stream()), "quant")
        assert (q[rows] == 77).all() and s[rows] == 77
