"""The FP8 norm in front of the block-FP8 linears, layer after layer without a pause: every kernel is resident before the one ahead of it
has finished, and the blocks of the scales are given out again at once. The same bits as with a synchronisation behind every operator,
so no kernel reads what its predecessor has not written yet or what a line of an earlier call still holds."""
import pytest
import torch

import sglang_b200 as S
from sglang_b200.int8 import quant_weight_int8
from sglang_b200.weight_quant import block_quant_weight_fp8, requant_weight_ue8m0

pytestmark = pytest.mark.gpu
H = 1024


def weights(n, k, count=3):
    g = torch.Generator(device="cuda").manual_seed(n + k)
    return [block_quant_weight_fp8((0.03 * torch.randn(n, k, generator=g, device="cuda")).bfloat16()) for _ in range(count)]


def start(rows):
    g = torch.Generator(device="cuda").manual_seed(rows)
    return [torch.randn(rows, H, generator=g, device="cuda").bfloat16() for _ in range(2)]


def same_as_step_by_step(run, repeats=4):
    want = run(torch.cuda.synchronize)
    assert all(t.isfinite().all() for t in want)
    for _ in range(repeats):
        assert all(torch.equal(a, b) for a, b in zip(run(lambda: None), want))


@pytest.mark.parametrize("layout", ["row", "col", "aligned", "ue8m0"])
@pytest.mark.parametrize("rows", [1, 3, 12, 17, 61, 130, 300, 1100])
def test_norm_and_block_gemm(rows, layout):
    norm = (1 + 0.1 * torch.randn(H, generator=torch.Generator().manual_seed(1))).bfloat16().cuda()
    ws = weights(H, H)
    if layout == "ue8m0":
        ws = [requant_weight_ue8m0(w, s, [128, 128]) for w, s in ws]

    def run(pause):
        x, r = start(rows)
        for k in range(60):
            q, s, r = S.rmsnorm_quant_fp8(x, norm, residual=r, column_major_scales=layout != "row",
                                          scale_tma_aligned=layout in ("aligned", "ue8m0"), scale_ue8m0=layout == "ue8m0")
            pause()
            w, sw = ws[k % 3]
            x = S.w8a8_block_fp8_matmul(q, w, s, sw, [128, 128], torch.bfloat16)
            pause()
        return x, r

    same_as_step_by_step(run)


@pytest.mark.parametrize("rows", [1, 4, 16, 40, 300])
def test_operators_that_signal_early_in_front_of_the_ones_that_read_16_bits(rows):
    """Norms, int8 products and quantisers let their successors in at once: a quantising linear, a group quantiser and a product that read
    their 16-bit outputs."""
    norm = torch.ones(H, device="cuda").bfloat16()
    fp8 = weights(H, H)
    int8 = [quant_weight_int8(0.03 * torch.randn(H, H, generator=torch.Generator().manual_seed(i)).cuda()) for i in range(3)]

    def run(pause):
        x, r = start(rows)
        for k in range(40):
            (w, ws), (v, vs) = fp8[k % 3], int8[k % 3]
            q, s, r = S.rmsnorm_quant_int8(x, norm, residual=r)
            pause()
            x = S.int8_scaled_mm(q, v.t(), s, vs, torch.bfloat16)
            pause()
            x = S.w8a8_block_fp8_linear(x, w, [128, 128], ws)
            pause()
            q, s = S.per_token_group_quant_fp8(r, 128, column_major_scales=True)
            pause()
            x = x + S.w8a8_block_fp8_matmul(q, w, s, ws, [128, 128], torch.bfloat16)
            x = x / x.float().abs().amax().bfloat16()
            pause()
            x = S.w8a8_int8_linear(x, v, vs)
            pause()
        return x, r

    same_as_step_by_step(run)


def test_device_status_is_clear():
    from sglang_b200 import _native as N

    assert N.read_device_status() == 0
