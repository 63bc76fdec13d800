"""Norms and rotation of q and k, and the append to a paged cache, against their formulas in 64 bits.

Tolerance: half a step of the result's type for its one rounding, and the fp32 arithmetic in front of it. There a normed element has
the errors of a sum of D squares (each lane adds up to D / 32 * 2 of them, then five steps: below 40 roundings for D <= 512, halved by the
root), of the reciprocal root (2 steps) and of two products; the rotation adds three roundings of |a c| + |b s|. Together below
40 * 2^-24 of |a c| + |b s|."""
import itertools
import math

import pytest
import torch

import sglang_b200 as S

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
ARITHMETIC = 40 * 2.0**-24
SMALLEST = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-150, FP8: 2.0**-10}  # half of the smallest step


def table(rows, rotated, base=10000.0):
    rate = base ** (-torch.arange(rotated // 2, dtype=torch.float64, device="cuda") / max(1, rotated // 2))
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * rate
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def axis_map(pairs, section, interleaved):
    if section is None:
        return [0] * pairs
    if not interleaved:
        return [k for k, n in enumerate(section) for _ in range(n)]
    n = len(section)
    return [j % n if j % n and j < n * section[j % n] else 0 for j in range(pairs)]


def formula(x, weight, eps, positions, cos_sin, neox, section, interleaved):
    """[T, heads, D] -> (result, size of the terms it is a sum of), float64."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    out, size = y.clone(), y.abs()
    if positions is None:
        return out, size
    pairs = cos_sin.shape[1] // 2
    positions = positions.view(-1, x.shape[0]).long()
    for j, axis in enumerate(axis_map(pairs, section, interleaved)):
        at = positions[axis]
        known = (at >= 0) & (at < cos_sin.shape[0])
        line = cos_sin[at.clamp(0, cos_sin.shape[0] - 1)].double().masked_fill(~known[:, None], math.nan)
        c, s = line[:, j, None], line[:, pairs + j, None]
        a, b = (j, j + pairs) if neox else (2 * j, 2 * j + 1)
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
        size[..., a] = (y[..., a] * c).abs() + (y[..., b] * s).abs()
        size[..., b] = (y[..., b] * c).abs() + (y[..., a] * s).abs()
    return out, size


def check(got, want, size, scale=None):
    """``got`` against 64-bit values; an FP8 ``got`` holds ``want / scale``."""
    half = torch.finfo(got.dtype).eps / 2
    g = got.double()
    if got.dtype == FP8:
        if scale is not None:
            scale = scale.double().view(1, -1, 1)
            want, size = want / scale, size / scale
        want = want.clamp(-448, 448)
    bad = torch.isnan(want)
    assert torch.equal(torch.isnan(g), bad)
    bound = half * torch.maximum(want.abs(), g.abs()) + ARITHMETIC * size + SMALLEST[got.dtype]
    ok = ((g - want).abs() <= bound) | bad | (g == want)
    assert ok.all(), f"{(~ok).sum().item()} of {ok.numel()} off, worst {((g - want).abs() / bound)[~ok].max().item():.3f} of the bound"


def make_qkv(rows, heads, dim, dtype, seed=0, pitch=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, heads * dim + pitch, generator=g, device="cuda")
    x[:, :: 97] *= 20
    return x.to(dtype)[:, : heads * dim]


def weights(dim, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(dim, generator=g, device="cuda") * 0.2 + 1).to(dtype) for _ in range(2)]


def split(qkv, q, kv):
    return qkv.unflatten(1, (q + 2 * kv, -1)).split([q, kv, kv], 1)


SHAPES = [  # tokens, q heads, kv heads, dim, rotated
    (1, 1, 1, 64, 64), (1, 32, 8, 128, 128), (7, 8, 1, 128, 64), (3, 5, 5, 80, 80), (130, 6, 2, 96, 48), (2, 7, 1, 72, 32),
    (5, 4, 2, 256, 256), (9, 3, 3, 512, 512), (33, 2, 1, 192, 96), (4, 3, 1, 100, 50), (6, 2, 2, 37, 20), (700, 10, 2, 128, 128),
    (11, 2, 1, 8, 8), (3, 1, 1, 1, 0), (4, 2, 1, 66, 66), (5000, 3, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm_and_rotation(shape, neox, dtype):
    rows, q, kv, dim, rotated = shape
    qkv = make_qkv(rows, q + 2 * kv, dim, dtype)
    for norm, offset in itertools.product([True, False], [0, 1]):
        wq, wk = weights(dim, dtype) if norm else (None, None)
        x = qkv if not offset else make_qkv(rows, q + 2 * kv, dim, dtype, 3, pitch=8 + offset)
        pos = (torch.arange(rows, device="cuda") * 37 + 1000) % 4096 if rotated else None
        cs = table(4096, rotated) if rotated else None
        got = S.qk_norm_rope(x, q, kv, pos, cs, wq, wk, 1e-6, is_neox=neox)
        for g, part, w in zip(got, split(x, q, kv), (wq, wk)):
            assert g.shape == part.shape and g.is_contiguous() and g.dtype == dtype
            check(g, *formula(part, w, 1e-6, pos, cs, neox, None, False))


@pytest.mark.parametrize("section, interleaved", [([16, 24, 24], False), ([24, 20, 20], True), ([64], False), ([0, 64], False),
                                                  ([1, 0, 63], False), ([16, 16, 16, 16], False), ([16, 16, 16, 16], True), ([64, 0, 0], True)])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("rows", [1, 77])
def test_several_axes(rows, neox, section, interleaved):
    q, kv, dim = 6, 2, 160  # 128 of 160 elements turn
    x = make_qkv(rows, q + 2 * kv, dim, torch.bfloat16)
    wq, wk = weights(dim, torch.bfloat16)
    for dtype in (torch.int64, torch.int32):
        wide = torch.randint(0, 500, (len(section), rows + 3), device="cuda", dtype=dtype)
        pos = wide[:, 1 : rows + 1]
        got = S.qk_norm_rope(x, q, kv, pos, table(500, 128), wq, wk, 1e-5, neox, section, interleaved)
        for g, part, w in zip(got, split(x, q, kv), (wq, wk)):
            check(g, *formula(part, w, 1e-5, pos.contiguous(), table(500, 128), neox, section, interleaved))


def caches(pages, page, kv, dim, dtype, layout="plain", seed=5):
    """The two caches: alone, halves of one tensor, with heads before tokens, or off the 16-byte boundaries."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = {"plain": (2, pages, page, kv, dim), "joint": (pages, 2, page, kv, dim), "heads": (2, pages, kv, page, dim),
             "odd": (2, pages, page, kv, dim + 3)}[layout]
    t = torch.randn(shape, generator=g, device="cuda").to(dtype)
    k, v = t.unbind(1) if layout == "joint" else t.unbind(0)
    if layout == "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    if layout == "odd":
        k, v = k[..., 1 : dim + 1], v[..., 3:]
    return k, v


def bits(t):
    return t.view(torch.uint8 if t.element_size() == 1 else torch.int16 if t.element_size() == 2 else torch.int32)


def check_cache(cache, before, slots, want, size, scale):
    page = cache.shape[1]
    used = torch.zeros(cache.shape[0] * page, dtype=torch.bool, device="cuda")
    valid = (slots >= 0) & (slots < used.numel())
    at = slots[valid].long()
    used[at] = True
    flat = cache.reshape(-1, *cache.shape[2:])
    check(flat[at], want[valid], size[valid], scale)
    assert torch.equal(bits(flat[~used]), bits(before.reshape(flat.shape)[~used])), "a slot of no token was written"


@pytest.mark.parametrize("layout", ["plain", "joint", "heads", "odd"])
@pytest.mark.parametrize("page", [1, 16, 5])
@pytest.mark.parametrize("rows, q, kv, dim, rotated", [(1, 8, 2, 128, 128), (37, 4, 1, 64, 32), (300, 3, 3, 80, 80), (6, 2, 2, 50, 10)])
@pytest.mark.parametrize("dtype, held", [(torch.bfloat16, None), (torch.float16, None), (torch.bfloat16, FP8), (torch.float16, FP8),
                                         (torch.float32, None), (torch.float32, FP8)])
def test_append(dtype, held, rows, q, kv, dim, rotated, page, layout):
    pages = -(-rows // page) + 3
    g = torch.Generator().manual_seed(rows)
    slots = torch.randperm(pages * page, generator=g)[:rows].cuda()
    if rows > 4:
        slots[1], slots[4] = -1, pages * page  # padding, and a slot behind the cache
        slots[3] = -(2**40)
    x = make_qkv(rows, q + 2 * kv, dim, dtype, rows)
    pos, cs = torch.arange(rows, device="cuda", dtype=torch.int32), table(rows, rotated)
    wq, wk = weights(dim, dtype)
    part = split(x, q, kv)
    scales = [torch.rand(n, device="cuda") * 0.1 + 0.01 for n in (kv, 1)] if held else [None, None]
    for fused in (True, False):
        k, v = caches(pages, page, kv, dim, held or dtype, layout)
        old = k.clone(), v.clone()
        if fused:
            got = S.qk_norm_rope_append(x, q, kv, pos, cs, k, v, slots, wq, wk, 1e-6, k_scale=scales[0], v_scale=scales[1])
            check(got, *formula(part[0], wq, 1e-6, pos, cs, True, None, False))
        else:
            S.append_paged_kv(part[1], part[2], k, v, slots, pos, cs, k_scale=scales[0], v_scale=scales[1])
        check_cache(k, old[0], slots, *formula(part[1], wk if fused else None, 1e-6, pos, cs, True, None, False), scales[0])
        check_cache(v, old[1], slots, part[2].double(), torch.zeros_like(part[2], dtype=torch.double), scales[1])


def test_append_without_rotation_copies_bits():
    x = make_qkv(9, 4, 128, torch.bfloat16)
    _, k, v = split(x, 2, 1)
    kc, vc = caches(4, 4, 1, 128, torch.bfloat16)
    slots = torch.arange(9, device="cuda", dtype=torch.int32) + 3
    S.append_paged_kv(k, v, kc, vc, slots)
    assert torch.equal(kc.flatten(0, 1)[3:12], k) and torch.equal(vc.flatten(0, 1)[3:12], v)


def test_fp8_codes_are_those_of_the_ieee_quotient():
    """Every finite bf16 magnitude over scales whose reciprocal is inexact: the nearest code of the quotient, as the definition says."""
    x = torch.arange(0x7F80, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.cat([x, -x]).view(-1, 1, 128)
    kc, vc = (torch.zeros(x.shape[0], 1, 1, 128, device="cuda").to(FP8) for _ in range(2))
    for ks, vs in ((0.0107, 3.7), (1.0, 0.1), (7e-4, 11.0)):
        ks, vs = torch.tensor([ks], device="cuda"), torch.tensor([vs], device="cuda")
        S.append_paged_kv(x, x, kc, vc, torch.arange(x.shape[0], device="cuda"), k_scale=ks, v_scale=vs)
        for c, s in ((kc, ks), (vc, vs)):
            want = (x.float() / s).clamp(-448, 448).to(FP8)
            assert torch.equal(bits(c[:, 0]), bits(want))


def test_values_that_are_not_finite():
    x = make_qkv(4, 3, 128, torch.bfloat16)
    x[0, 5], x[1, 130], x[2, 300] = math.nan, math.inf, -math.inf  # in q, k and v
    pos, cs = torch.arange(4, device="cuda"), table(8, 64)
    q, k = S.qk_norm_rope(x, 1, 1, pos, cs)
    for got, part in zip((q, k), split(x, 1, 1)):
        check(got, *formula(part, None, 1e-6, pos, cs, True, None, False))
    # neighbours of an infinity that do not turn keep their bits
    x[3, 126] = math.inf
    for neox in (True, False):
        q, _ = S.qk_norm_rope(x, 1, 1, pos, cs, is_neox=neox)
        assert torch.equal(q[3, 0, 64:], x[3, 64:128])
    kc, vc = caches(1, 4, 1, 128, FP8)
    _, k, v = split(x, 1, 1)
    S.append_paged_kv(k, v, kc, vc, pos, k_scale=torch.ones(1, device="cuda"), v_scale=torch.full((1,), 0.5, device="cuda"))
    assert kc[0, 1, 0, 2].item() == 448 and vc[0, 2, 0, 44].item() == -448
    assert torch.isnan(kc.float()).sum() == 0
    S.append_paged_kv(x[:, :128].view(4, 1, 128), v, kc, vc, pos)
    assert torch.isnan(kc.float()).sum() == 1 and math.isnan(kc[0, 0, 0, 5].item())


def test_rows_of_zeros_and_positions_outside_the_table():
    x = make_qkv(6, 4, 128, torch.float16)
    x[2] = 0
    pos = torch.tensor([0, 7, 3, -1, 8, 2**40], device="cuda")
    wq, wk = weights(128, torch.float16)
    q, k = S.qk_norm_rope(x, 2, 1, pos, table(8, 64), wq, wk)
    for got, part, w in zip((q, k), split(x, 2, 1), (wq, wk)):
        check(got, *formula(part, w, 1e-6, pos, table(8, 64), True, None, False))
    assert not torch.isnan(q[:3]).any() and torch.isnan(q[3:, :, :64]).all() and not torch.isnan(q[..., 64:]).any()
    assert (q[2] == 0).all()


def test_far_positions_of_a_large_table_and_cache():
    """Offsets past 32 bits: the last rows of a table of 2^31 bytes and more, and of a cache of more than 2^32."""
    rows = (1 << 23) + 5
    cs = torch.zeros(rows, 128, device="cuda")
    cs[:, :64] = 1
    cs[rows - 1, 64:] = 0.5
    pages = (1 << 32) // (64 * 128) + 2
    kc, vc = (torch.zeros(pages, 64, 1, 128, dtype=torch.uint8, device="cuda").view(FP8) for _ in range(2))
    x = make_qkv(2, 3, 128, torch.bfloat16)
    pos, slots = torch.tensor([rows - 1, 0], device="cuda"), torch.tensor([pages * 64 - 1, 0], device="cuda")
    wq, wk = weights(128, torch.bfloat16)
    q = S.qk_norm_rope_append(x, 1, 1, pos, cs, kc, vc, slots, wq, wk)
    _, k, v = split(x, 1, 1)
    check(q, *formula(x[:, :128].view(2, 1, 128), wq, 1e-6, pos, cs, True, None, False))
    flat = torch.stack([kc[-1, -1], kc[0, 0]])
    check(flat, *formula(k, wk, 1e-6, pos, cs, True, None, False), torch.ones(1, device="cuda"))
    check(torch.stack([vc[-1, -1], vc[0, 0]]), v.double(), torch.zeros_like(v, dtype=torch.double))


@pytest.mark.parametrize("rows", [0, 1, 50])
def test_graph_and_side_stream(rows):
    x = make_qkv(rows, 12, 128, torch.bfloat16)
    pos, cs = torch.arange(rows, device="cuda"), table(64, 128)
    kc, vc = caches(8, 8, 2, 128, FP8)
    wq, wk = weights(128, torch.bfloat16)
    slots = torch.arange(rows, device="cuda")
    want = S.qk_norm_rope_append(x, 8, 2, pos, cs, kc, vc, slots, wq, wk)
    after = kc.clone(), vc.clone()
    kc2, vc2 = caches(8, 8, 2, 128, FP8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            got = S.qk_norm_rope_append(x, 8, 2, pos, cs, kc2, vc2, slots, wq, wk)
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert got.shape == (rows, 8, 128) and torch.equal(got, want)
    assert torch.equal(bits(kc2), bits(after[0])) and torch.equal(bits(vc2), bits(after[1]))


def test_tokens_behind_a_kernel_that_still_writes_them():
    """Chained launches on one stream: every call reads what the one before it left."""
    x = make_qkv(64, 12, 128, torch.bfloat16)
    pos, cs = torch.arange(64, device="cuda"), table(64, 128)
    y = x.clone()
    for _ in range(20):
        q, k = S.qk_norm_rope(y, 8, 2, pos, cs)
        y[:, : 8 * 128] = q.flatten(1)
        y[:, 8 * 128 : 10 * 128] = k.flatten(1)
    z = x.clone()
    for _ in range(20):
        q, k = S.qk_norm_rope(z, 8, 2, pos, cs)
        torch.cuda.synchronize()
        z[:, : 8 * 128] = q.flatten(1)
        z[:, 8 * 128 : 10 * 128] = k.flatten(1)
        torch.cuda.synchronize()
    assert torch.equal(y, z)


@pytest.mark.parametrize("scale", [2.0**-60, 1.3e-19, 2.0**-126, 1.9e-38, 2.0**-129, 3e-39, 2.0**-140, 2.0**-149, 1.7e38])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_fp8_codes_of_any_scale(dtype, scale):
    """Scales whose reciprocal is infinite or not a normal number, values from the smallest to the largest: the codes of the IEEE quotient."""
    x = torch.arange(0x7F80, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.cat([x, -x]).view(-1, 1, 128).to(dtype)
    s = torch.tensor([scale], device="cuda")
    assert s.item() > 0
    # (the quotient in 64 bits, rounded to 32: PyTorch's own 32-bit division may flush what is not normal)
    want = (x.double() / s.double()).float().clamp(-448, 448).to(FP8)
    for pad in (0, 1):  # whole vectors, and elements one by one
        kc, vc = (torch.zeros(x.shape[0], 1, 1, 128 + pad, device="cuda").to(FP8)[..., pad:] for _ in range(2))
        S.append_paged_kv(x, x, kc, vc, torch.arange(x.shape[0], device="cuda"), k_scale=s, v_scale=s)
        for c in (kc, vc):
            assert torch.equal(bits(c[:, 0].contiguous()), bits(want))
