"""The int8 product against exact sums in 64 bits.

Tolerance: the integer sums are exact; the conversion to fp32, the two scales and the addition of the bias round to 2^-24 each,
the result once to half a step of its type (below the normal range of fp16 2^-25)."""
import pytest
import torch

import sglang_b200 as S

pytestmark = pytest.mark.gpu
U = 2.0**-24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def operands(M, N, K, seed=0, lda=None, ldb=None):
    g = torch.Generator(device="cuda").manual_seed(seed + M * 7 + N * 3 + K)
    a = torch.randint(-128, 128, (M, lda or K), generator=g, device="cuda", dtype=torch.int8)[:, :K]
    b = torch.randint(-128, 128, (N, ldb or K), generator=g, device="cuda", dtype=torch.int8)[:, :K]
    sa = torch.rand(M, 1, generator=g, device="cuda") * 1e-3 + 1e-4
    sb = torch.rand(N, 1, generator=g, device="cuda") * 1e-3 + 1e-4
    return a, b, sa, sb, torch.randn(N, generator=g, device="cuda")


def check(out, a, b, sa, sb, bias):
    ref = (a.double() @ b.double().t()) * sa.double() * sb.double().t()
    room = 3 * U * ref.abs()
    if bias is not None:
        ref = ref + bias.double()
    half = torch.finfo(out.dtype).eps / 2
    room = room + (half + U) * ref.abs() + room * half + 2.0**-25 * (out.dtype == torch.float16)
    off = (out.double() - ref).abs()
    assert (off <= room).all(), (off / room.clamp_min(1e-30)).max()


SIZES = [(1, 8, 16), (1, 128, 128), (2, 136, 144), (3, 4096, 4096), (7, 264, 1040), (15, 512, 272), (16, 1280, 8192), (17, 2048, 528),
         (31, 8, 2048), (32, 1024, 14336), (33, 6144, 1024), (61, 1792, 8192), (64, 4096, 512), (65, 4096, 4096), (100, 24, 128),
         (127, 5120, 640), (128, 256, 16384), (129, 128, 4112), (200, 4096, 1792), (203, 1000, 4096), (256, 512, 256),
         (257, 2568, 784), (384, 8200, 32), (511, 1032, 2064), (640, 4096, 4096), (1027, 7168, 1024), (1500, 14336, 512),
         (2049, 2056, 2064), (4100, 520, 1040), (3000, 28672, 256)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_sizes(M, N, K):
    a, b, sa, sb, bias = operands(M, N, K)
    dtype = DTYPES[(M + N + K) % 2]
    check(S.int8_scaled_mm(a, b.t(), sa, sb, dtype), a, b, sa, sb, None)
    check(S.int8_scaled_mm(a, b.t(), sa, sb, dtype, bias.to(dtype)), a, b, sa, sb, bias.to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 9, 48, 130, 300, 1100])
def test_types(dtype, M):
    a, b, sa, sb, bias = operands(M, 1304, 1552)
    check(S.int8_scaled_mm(a, b.t(), sa, sb, dtype, bias.to(dtype)), a, b, sa, sb, bias.to(dtype))


@pytest.mark.parametrize("M", [1, 20, 70, 140, 600])
def test_rows_of_wider_tensors(M):
    a, b, sa, sb, _ = operands(M, 520, 1040, lda=1072, ldb=2080)
    got = S.int8_scaled_mm(a, b.t(), sa.view(-1), sb.view(-1), torch.bfloat16)
    assert torch.equal(got, S.int8_scaled_mm(a.contiguous(), b.contiguous().t(), sa, sb, torch.bfloat16))
    check(got, a, b, sa, sb, None)


@pytest.mark.parametrize("M", [1, 40, 128, 300])
def test_largest_sums(M):
    """K at its limit with every product at its largest: the sums are 2^14 K < 2^31."""
    K = 131056
    a = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    b = torch.full((256, K), -128, dtype=torch.int8, device="cuda")
    b[1::2] = 127
    one = torch.ones(max(M, 256), device="cuda")
    out = S.int8_scaled_mm(a, b.t(), one[:M].contiguous(), one[:256].contiguous(), torch.float32)
    assert (out[:, ::2].double() - 2.0**14 * K).abs().max() <= 2.0**14 * K * U
    assert (out[:, 1::2].double() + 128.0 * 127 * K).abs().max() <= 2.0**14 * K * U


@pytest.mark.parametrize("M", [1, 16, 61, 150, 700])
def test_scales_that_are_not_finite_stay_in_their_rows(M):
    a, b, sa, sb, _ = operands(M, 512, 512)
    want = S.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16)
    sa[M // 2], sb[5] = float("nan"), float("inf")
    out = S.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16)
    assert out[M // 2].isnan().all() and not out[:, 5].isfinite().any()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[M // 2], keep[:, 5] = False, False
    assert torch.equal(out[keep], want[keep])


def test_the_same_bits_on_every_run_and_for_every_batch():
    """Integer sums do not depend on the order of the additions, nor on the kernel that a batch takes."""
    a, b, sa, sb, bias = operands(1200, 1536, 4096)
    full = S.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16, bias.bfloat16())
    for m in (1, 5, 16, 17, 33, 64, 65, 128, 129, 200, 256, 300, 513, 1200):
        for _ in range(2):
            assert torch.equal(S.int8_scaled_mm(a[:m], b.t(), sa[:m], sb, torch.bfloat16, bias.bfloat16()), full[:m]), m


@pytest.mark.parametrize("tile", [16, 32, 48, 64, 96, 128, 208, 256, 1032, 1064, 1096, 1128, 1160, 1192, 1224, 1256, 2032, 2064, 2096, 2128, 2160, 2192, 2224, 2256])
@pytest.mark.parametrize("splits", [1, 2, 3, 4, 5, 7, 8])
def test_every_tile_and_split(tile, splits):
    """The kernels that the plan chooses from, each at sizes that it would not be chosen for, too."""
    from sglang_b200 import _native as N

    if tile > 256 and splits not in (1, 2, 4):
        pytest.skip("pairs split K by 2 or 4")
    for M, n, K in ((1, 136, 2064), (39, 1000, 1040), (130, 264, 272), (300, 520, 4096), (577, 2056, 144)):
        a, b, sa, sb, bias = operands(M, n, K)
        for dtype in (torch.bfloat16, torch.float32):
            with N.tuning(int8_tile=tile, int8_splits=splits):
                out = S.int8_scaled_mm(a, b.t(), sa, sb, dtype, bias.to(dtype))
            check(out, a, b, sa, sb, bias.to(dtype))


def test_empty():
    a, b, sa, sb, _ = operands(4, 64, 64)
    assert S.int8_scaled_mm(a[:0], b.t(), sa[:0], sb, torch.bfloat16).shape == (0, 64)
    assert S.int8_scaled_mm(a, b[:0].t(), sa, sb[:0], torch.bfloat16).shape == (4, 0)


def test_offsets_past_31_bits():
    """Operand and output rows that lie more than 2^31 bytes into their tensors."""
    M, N, K = 140000, 128, 16384
    a = torch.zeros(M, K, dtype=torch.int8, device="cuda")
    _, b, _, sb, _ = operands(1, N, K)
    a[-2:] = operands(2, 8, K)[0]
    sa = torch.full((M,), 1e-3, device="cuda")
    out = S.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16)
    assert (out[:-2] == 0).all()
    check(out[-2:], a[-2:], b, sa[-2:, None], sb, None)
    del a, out
    M, N, K = 80000, 28672, 32
    a, b, sa, sb, _ = operands(M, N, K)
    out = S.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16)
    for r in (0, M // 2 + 1, M - 3):
        check(out[r : r + 3], a[r : r + 3], b, sa[r : r + 3], sb, None)


def test_nothing_is_written_outside_the_output():
    from sglang_b200 import _native as N

    lib = N.load()
    for M, n, K in ((1, 136, 256), (17, 8, 64), (65, 1000, 512), (130, 392, 256), (300, 1160, 640)):
        a, b, sa, sb, _ = operands(M, n, K)
        for dtype in DTYPES:
            buf = torch.full(((M + 2) * n,), 77.0, dtype=dtype, device="cuda")
            N.check(lib.b200_int8_scaled_mm(N.ptr(a), K, N.ptr(sa), N.ptr(b), K, N.ptr(sb), 0, N.ptr(buf[n:]), N.DTYPE_CODE[dtype], M,
                                            n, K, N.current_stream()), "int8_scaled_mm")
            assert (buf[:n] == 77).all() and (buf[-n:] == 77).all()
            check(buf[n:-n].view(M, n), a, b, sa, sb, None)


def test_linear_is_quantiser_and_product():
    g = torch.Generator(device="cuda").manual_seed(3)
    for shape in ((1, 1024), (2, 5, 1024), (70, 1024), (600, 1024)):
        for dtype in (torch.bfloat16, torch.float16):
            x = torch.randn(*shape, generator=g, device="cuda").to(dtype)
            _, b, _, sb, bias = operands(1, 1536, 1024)
            q, s = S.per_token_quant_int8(x.view(-1, 1024))
            want = S.int8_scaled_mm(q, b.t(), s, sb, dtype, bias.to(dtype)).view(*shape[:-1], 1536)
            assert torch.equal(S.w8a8_int8_linear(x, b, sb, bias.to(dtype)), want)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("N,K", [(8, 16), (128, 128), (136, 272), (1000, 1040), (4096, 4096), (6144, 2064), (264, 14336), (28672, 512), (2048, 28672)])
def test_linear_in_one_launch_equals_two(M, N, K):
    from sglang_b200 import _native

    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    for dtype, splits in ((torch.bfloat16, 0), (torch.float16, 0), (torch.bfloat16, 1), (torch.bfloat16, 3), (torch.float16, 8)):
        wide = torch.randn(M, K + 64, generator=g, device="cuda").to(dtype)
        x = wide[:, 8 : 8 + K] if splits else wide[:, :K].contiguous()
        if M > 2:
            x[1, K // 2], x[2] = float("nan"), 0
        _, b, _, sb, bias = operands(1, N, K)
        with _native.tuning(int8_splits=splits, int8_tile=16 if splits else -1, int8_linear_fused=1):
            got = S.w8a8_int8_linear(x, b, sb, bias.to(dtype))
            with _native.tuning(int8_linear_fused=0):
                want = S.w8a8_int8_linear(x, b, sb, bias.to(dtype))
        assert torch.equal(got.nan_to_num(7e4), want.nan_to_num(7e4)) and torch.equal(got.isnan(), want.isnan())
        q, s = S.per_token_quant_int8(x)
        keep = [i for i in range(M) if M <= 2 or i != 1]
        check(got[keep], q[keep], b, s[keep], sb, bias.to(dtype))


def test_linear_rows_at_odd_addresses():
    x = torch.randn(3, 1032, device="cuda").bfloat16()[:, 3 : 3 + 1024]
    _, b, _, sb, _ = operands(1, 512, 1024)
    assert torch.equal(S.w8a8_int8_linear(x, b, sb), S.w8a8_int8_linear(x.contiguous(), b, sb))


def test_device_status_is_clear():
    from sglang_b200 import _native as N

    assert N.read_device_status() == 0
