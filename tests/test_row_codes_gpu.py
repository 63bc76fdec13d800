"""One formula for every row: the 8-bit codes of the norms and of the gated quantiser do not depend on the alignment of the rows, on their
number or on how many vectors a thread takes, and those of the norms are what IEEE arithmetic in fp32 gives.

1/rms cancels in y / s, so the codes of a norm come from v = h * w alone (h and v rounded once each): e4m3(v * f), f = 448 / max|v| of the group
rounded once, and the whole number nearest to v / t, t = max|v| / 127 of the row, both quotients rounded once. Nothing in them depends on the order of the sum of
squares; it may move the last bits of the scales, by less than 2^-17 as everywhere."""
import pytest
import torch

import sglang_b200 as S
from sglang_b200 import _native as N

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
WIDTHS = [128, 640, 1024, 4096, 8192, 12032, 16384]


def rows_at(rows, width, dtype, seed, offset, scale=1.0):
    """The same rows, starting `offset` elements behind a boundary and an odd number of elements apart."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, width, generator=g, device="cuda") * scale
    x[:, :: max(2, width // 7)] *= 20
    x = x.to(dtype)
    if not offset:
        return x
    wide = torch.zeros(rows, width + offset + 9, dtype=dtype, device="cuda")
    wide[:, offset : offset + width] = x
    return wide[:, offset : offset + width]


def close(a, b):
    assert ((a.double() - b.double()).abs() <= 2.0**-17 * a.double().abs()).all()


def over(v, top):  # IEEE, not a product with a rounded reciprocal
    return torch.full_like(v, top) / v


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_of_the_norms_by_the_formula(width, dtype):
    for rows, with_res in ((3, True), (600, False)):
        x, w = rows_at(rows, width, dtype, 1, 0), rows_at(1, width, dtype, 2, 0)[0]
        r = rows_at(rows, width, dtype, 3, 0) if with_res else None
        v = (x.float() + r.float() if with_res else x.float()) * w.float()
        t = v.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device="cuda")
        assert torch.equal(S.rmsnorm_quant_int8(x, w, residual=r)[0], (v / t).round().to(torch.int8))
        g = v.view(rows, -1, 128)
        want = (g * over(g.abs().amax(-1, keepdim=True), 448.0)).to(torch.float8_e4m3fn).view(rows, width)
        assert torch.equal(S.rmsnorm_quant_fp8(x, w, residual=r)[0].view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_do_not_depend_on_alignment(width, dtype):
    for rows in (2, 700):
        x, r, w = (rows_at(n, width, dtype, k, 0) for n, k in ((rows, 4), (rows, 5), (1, 6)))
        x1, r1 = rows_at(rows, width, dtype, 4, 1), rows_at(rows, width, dtype, 5, 3)
        assert torch.equal(x, x1) and torch.equal(r, r1)
        for fn in (S.rmsnorm_quant_int8, S.rmsnorm_quant_fp8):
            (q, s, h), (q1, s1, h1) = fn(x, w[0], residual=r), fn(x1, w[0], residual=r1)
            assert torch.equal(q.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(h, h1)
            close(s, s1)
        q, s = S.per_token_quant_int8(x, fuse_silu_and_mul=True)
        q1, s1 = S.per_token_quant_int8(x1, fuse_silu_and_mul=True)
        assert torch.equal(s, s1) and torch.equal(q, q1)
        q, s = S.per_token_quant_int8(x)
        q1, s1 = S.per_token_quant_int8(x1)
        assert torch.equal(s, s1) and torch.equal(q, q1)


@pytest.mark.parametrize("width", [1024, 4096, 16384])
def test_codes_do_not_depend_on_the_batch(width):
    """A row alone, among few and among many, with every number of vectors per thread."""
    x, r, w = rows_at(3000, width, torch.bfloat16, 7, 0), rows_at(3000, width, torch.bfloat16, 8, 0), rows_at(1, width, torch.bfloat16, 9, 0)[0]
    calls = (lambda n: S.rmsnorm_quant_int8(x[:n], w, residual=r[:n]), lambda n: S.rmsnorm_quant_fp8(x[:n], w, residual=r[:n]),
             lambda n: S.per_token_quant_int8(x[:n], fuse_silu_and_mul=True))
    for k, call in enumerate(calls):
        want = call(3000)
        for n, vectors in ((1, -1), (5, -1), (600, -1), (9, 1), (9, 2), (9, 4), (9, 8)):
            with N.tuning(row_vectors=vectors):
                got = call(n)
            assert torch.equal(got[0].view(torch.uint8), want[0][:n].view(torch.uint8)), (k, n, vectors)
            if k == 2:
                assert torch.equal(got[1], want[1][:n])
            else:
                close(got[1], want[1][:n])


def test_rows_below_the_floor():
    """max|y| under 1e-10: the scale is that of the floor and the codes are y over it, zeros among them."""
    for offset in (0, 1):
        x = rows_at(4, 1024, torch.float32, 10, offset, scale=1e-14)
        x[1] = 0
        w = torch.ones(1024, device="cuda")
        y = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
        assert 1e-12 < y[0].abs().amax() < 1e-9
        for top, fn in ((127.0, S.rmsnorm_quant_int8), (448.0, S.rmsnorm_quant_fp8)):
            q, s = fn(x, w)
            g = y.view(4, -1, 128 if top == 448 else 1024)
            step = g.abs().amax(-1, keepdim=True).clamp_min(1e-10) / top
            assert ((s.double().view(step.shape) - step).abs() <= 2.0**-17 * step).all() and (q[1].float() == 0).all()
            off = (q.double().view(g.shape) - g / step).abs()
            half = 0.5 if top == 127 else 2.0 ** ((g / step).abs().clamp_min(2.0**-6).log2().floor() - 4)
            assert (off <= half * (1 + 2.0**-12) + top * 2.0**-17).all()


@pytest.mark.parametrize("width", [1024, 1023, 8192, 14336])
def test_ties_go_to_even(width):
    """Quotients that lie halfway between two whole numbers: max|v| = 127 * 2^k makes them exact."""
    g = torch.Generator(device="cuda").manual_seed(width)
    halves = torch.randint(-252, 253, (4, width), generator=g, device="cuda").float() / 2
    halves[:, width // 3] = 127
    want = halves.round().to(torch.int8)  # ties to even
    for dtype in DTYPES:
        x = (halves * torch.tensor([[1.0], [0.25], [8.0], [2.0**-7]], device="cuda")).to(dtype)
        assert torch.equal(x.float(), halves * torch.tensor([[1.0], [0.25], [8.0], [2.0**-7]], device="cuda"))
        w = torch.ones(width, dtype=dtype, device="cuda")
        assert torch.equal(S.rmsnorm_quant_int8(x, w)[0], want)
        assert torch.equal(S.rmsnorm_quant_int8(x, w, residual=torch.zeros_like(x))[0], want)
        assert torch.equal(S.per_token_quant_int8(x)[0], want)


def test_a_sum_past_the_largest_float_leaves_zeros():
    """mean(h^2) is infinite in fp32, so y is zero: codes are zeros and the scale is that of the floor, at every alignment."""
    for offset in (0, 1):
        x = rows_at(2, 1024, torch.bfloat16, 11, offset, scale=1e25)
        w = torch.ones(1024, dtype=torch.bfloat16, device="cuda")
        for top, fn in ((127.0, S.rmsnorm_quant_int8), (448.0, S.rmsnorm_quant_fp8)):
            q, s = fn(x, w)
            assert (q.float() == 0).all() and torch.equal(s, torch.full_like(s, 1e-10) / torch.full_like(s, top))
