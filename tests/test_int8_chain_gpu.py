"""The int8 and norm operators together, as a decoder layer's MLP runs them, and under everything that a server does to a call:
graphs, side streams, threads, dispatcher ops.

Against its definition the chain is checked link by link, every operator on what the one before it gave, at that operator's own
tolerance. Its end has none that would be worth testing: a 16-bit intermediate value that lies on a rounding border may go
either way, and where it is the largest of its row the row's scale moves by 2^-8 and every code of the row is rounded anew, half a
step at random, which is several percent of the output's rms."""
import threading

import pytest
import torch

import sglang_b200 as S
from test_int8_gpu import check as check_product
from test_row_quant_gpu import check_int8, check_residual, normed
from sglang_b200.int8 import W8A8Int8Config, W8A8Int8LinearMethod, quant_weight_int8

pytestmark = pytest.mark.gpu


class MLP:
    def __init__(self, hidden, inter, dtype, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = dtype
        self.norm = (1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(dtype)
        self.w1, self.s1 = quant_weight_int8(0.02 * torch.randn(2 * inter, hidden, generator=g, device="cuda"))
        self.w2, self.s2 = quant_weight_int8(0.02 * torch.randn(hidden, inter, generator=g, device="cuda"))

    def __call__(self, x, r):
        q, s, r = S.rmsnorm_quant_int8(x, self.norm, 1e-6, residual=r)
        mid = S.int8_scaled_mm(q, self.w1.t(), s, self.s1, self.dtype)
        q, s = S.per_token_quant_int8(mid, fuse_silu_and_mul=True)
        return S.int8_scaled_mm(q, self.w2.t(), s, self.s2, self.dtype), r


def inputs(rows, hidden, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(rows, hidden, generator=g, device="cuda").to(dtype) for _ in range(2)]


@pytest.mark.parametrize("rows", [1, 4, 17, 130, 600])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_mlp(rows, dtype):
    mlp = MLP(1024, 1408, dtype)
    x, r = inputs(rows, 1024, dtype, rows)
    out, res = mlp(x, r)
    y, h = normed(x, r, mlp.norm, 1e-6)
    q, s, res2 = S.rmsnorm_quant_int8(x, mlp.norm, 1e-6, residual=r)
    check_int8(q, s, y)
    check_residual(res, h, dtype)
    mid = S.int8_scaled_mm(q, mlp.w1.t(), s, mlp.s1, dtype)
    check_product(mid, q, mlp.w1, s, mlp.s1, None)
    gate, up = mid.double().chunk(2, -1)
    q, s = S.per_token_quant_int8(mid, fuse_silu_and_mul=True)
    check_int8(q, s, gate / (1 + (-gate).exp()) * up, extra=2.0**-16)
    check_product(out, q, mlp.w2, s, mlp.s2, None)
    assert torch.equal(res, res2)


def test_fp8_norm_feeds_the_block_gemm():
    """The norm's FP8 rows and scales in every layout are what the block GEMM takes."""
    import oracle as O

    g = torch.Generator().manual_seed(1)
    wq, ws = O.block_quant_weight_fp8((torch.randn(512, 1024, generator=g) * 0.02).bfloat16())
    x, r = inputs(40, 1024, torch.bfloat16, 2)
    norm = torch.ones(1024, device="cuda").bfloat16()
    outs = []
    for col, aligned in ((False, False), (True, False), (True, True)):
        q, s, res = S.rmsnorm_quant_fp8(x, norm, residual=r, column_major_scales=col, scale_tma_aligned=aligned)
        outs.append(S.w8a8_block_fp8_matmul(q, wq.cuda(), s, ws.cuda(), [128, 128], torch.bfloat16))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    h = x.float() + r.float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6)
    rq, rs = O.per_token_group_quant_fp8(y.cpu(), 128)
    ref = O.w8a8_block_fp8_matmul(rq, wq, rs, ws, [128, 128], torch.float32)
    assert O.rel_frobenius(outs[0].float().cpu(), ref) < 1e-2


def capture(fn, stream=None):
    stream = stream or torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        fn()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = fn()
    torch.cuda.synchronize()
    return graph, out


@pytest.mark.parametrize("rows", [1, 61, 700])
def test_replays(rows):
    mlp = MLP(1024, 768, torch.bfloat16)
    x, r = inputs(rows, 1024, torch.bfloat16, 1)
    graph, out = capture(lambda: mlp(x, r))
    for seed in (2, 3):
        for t, new in zip((x, r), inputs(rows, 1024, torch.bfloat16, seed)):
            t.copy_(new)
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, mlp(x, r)))


def test_two_graphs_of_one_stream_replayed_at_once():
    """Linears captured on the same stream share nothing: replayed on two streams at once each gives its own result."""
    stream, runs = torch.cuda.Stream(), []
    for i, rows in enumerate((40, 40)):
        w, s = quant_weight_int8(torch.randn(4096, 4096, generator=torch.Generator().manual_seed(i)).cuda())
        x = inputs(rows, 4096, torch.bfloat16, i)[0]
        graph, out = capture(lambda: [S.w8a8_int8_linear(x, w, s) for _ in range(20)], stream)
        runs.append((graph, out, S.w8a8_int8_linear(x, w, s), (x, w, s)))  # the graph reads its inputs where they are
    sides = [torch.cuda.Stream() for _ in runs]
    for _ in range(5):
        for (graph, *_), side in zip(runs, sides):
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _ in runs:
        assert all(torch.equal(o, want) for o in out)


def test_side_stream_waits_for_its_inputs():
    """Inputs written on another stream just before the call, weights too: an event is all that orders them."""
    mlp, other = MLP(2048, 1024, torch.bfloat16), torch.cuda.Stream()
    x, r = inputs(30, 2048, torch.bfloat16, 4)
    want = mlp(x, r)
    w1, w2 = mlp.w1.clone(), mlp.w2.clone()
    xs, rs = x.clone(), r.clone()
    for _ in range(10):
        for t in (xs, rs, mlp.w1, mlp.w2):
            t.zero_()
        torch.cuda._sleep(200000)
        for t, v in ((xs, x), (rs, r), (mlp.w1, w1), (mlp.w2, w2)):
            t.copy_(v)
        event = torch.cuda.Event()
        event.record()
        with torch.cuda.stream(other):
            other.wait_event(event)
            got = mlp(xs, rs)
        torch.cuda.current_stream().wait_stream(other)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("rows", [1, 3, 40, 300])
def test_long_chain_equals_step_by_step(rows):
    """Layer after layer without a pause, every kernel resident before the one ahead has finished and buffers given out again at once:
    the same bits as with a synchronisation behind every operator."""
    mlps = [MLP(1024, 640, torch.bfloat16, seed=i) for i in range(3)]
    lin = [quant_weight_int8(0.05 * torch.randn(1024, 1024, generator=torch.Generator().manual_seed(i)).cuda()) for i in range(3)]

    def run(pause):
        x, r = inputs(rows, 1024, torch.bfloat16, 9)
        for k in range(60):
            m, (w, s) = mlps[k % 3], lin[k % 3]
            q, sc, r = S.rmsnorm_quant_int8(x, m.norm, 1e-6, residual=r)
            pause()
            mid = S.int8_scaled_mm(q, m.w1.t(), sc, m.s1, m.dtype)
            pause()
            q, sc = S.per_token_quant_int8(mid, fuse_silu_and_mul=True)
            pause()
            x = S.int8_scaled_mm(q, m.w2.t(), sc, m.s2, m.dtype)
            pause()
            x = S.w8a8_int8_linear(x, w, s)
            pause()
        return x, r

    want = run(torch.cuda.synchronize)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(run(lambda: None), want))


@pytest.mark.parametrize("rows", [1, 40])
def test_threads_share_a_stream(rows):
    mlps = [MLP(1024, 512, torch.bfloat16, seed=i) for i in range(4)]
    ins = [inputs(rows, 1024, torch.bfloat16, i) for i in range(4)]
    want = [m(*i) for m, i in zip(mlps, ins)]
    w, s = quant_weight_int8(torch.randn(512, 1024, device="cuda"))
    lin = [S.w8a8_int8_linear(i[0], w, s) for i in ins]
    wrong = []

    def work(k):
        for _ in range(100):
            if not all(torch.equal(a, b) for a, b in zip(mlps[k](*ins[k]), want[k])) or not torch.equal(S.w8a8_int8_linear(ins[k][0], w, s), lin[k]):
                wrong.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_linear_method():
    method, layer = W8A8Int8LinearMethod(W8A8Int8Config()), torch.nn.Module()
    method.create_weights(layer, 512, [256, 128], 512, 384, torch.bfloat16, device="cuda")
    w, s = quant_weight_int8(torch.randn(384, 512, device="cuda"))
    layer.load_state_dict({"weight": w, "weight_scale": s})
    method.process_weights_after_loading(layer)
    x = torch.randn(2, 9, 512, device="cuda").bfloat16()
    bias = torch.randn(384, device="cuda").bfloat16()
    want = S.w8a8_int8_linear(x, w, s, bias)
    assert want.shape == (2, 9, 384) and torch.equal(method.apply(layer, x, bias), want)
    assert torch.equal(method.apply(layer, S.per_token_quant_int8(x), bias), want)
    norm = torch.ones(512, device="cuda").bfloat16()
    assert method.apply(layer, S.rmsnorm_quant_int8(x, norm, residual=x)).shape == (2, 9, 384)


def test_dispatcher_ops_equal_direct_calls():
    ops, mlp = torch.ops.sglang_b200, MLP(512, 384, torch.float16)
    x, r = inputs(21, 512, torch.float16, 5)

    def chain(x, r):
        q, s, r = ops.rmsnorm_quant_int8(x, mlp.norm, 1e-6, r)
        mid = ops.int8_scaled_mm(q, mlp.w1.t(), s, mlp.s1, torch.float16, None)
        q, s = ops.per_token_quant_int8(mid, True)
        return ops.int8_scaled_mm(q, mlp.w2.t(), s, mlp.s2, torch.float16, None), r

    want = mlp(x, r)
    for fn in (chain, torch.compile(chain, backend="eager", fullgraph=True)):
        assert all(torch.equal(a, b) for a, b in zip(fn(x, r), want))
    a, b = ops.rmsnorm_quant_fp8(x, mlp.norm, 128, 1e-6, None, True, True, True), S.rmsnorm_quant_fp8(
        x, mlp.norm, 128, 1e-6, column_major_scales=True, scale_tma_aligned=True, scale_ue8m0=True)
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


def test_subclasses_and_parameters_take_the_general_path():
    """What the native host path does not take (a tensor subclass) gives the same bits through the general one."""
    class Sub(torch.Tensor):
        pass

    mlp = MLP(512, 256, torch.bfloat16)
    x, r = inputs(5, 512, torch.bfloat16, 6)
    w = torch.nn.Parameter(mlp.w1, requires_grad=False)
    q, s = S.per_token_quant_int8(x)
    sub = x.as_subclass(Sub)
    for a, b in ((S.per_token_quant_int8(sub), (q, s)), (S.rmsnorm_quant_int8(sub, mlp.norm, residual=r), S.rmsnorm_quant_int8(x, mlp.norm, residual=r)),
                 (S.rmsnorm_quant_fp8(sub, mlp.norm), S.rmsnorm_quant_fp8(x, mlp.norm)), ([S.w8a8_int8_linear(sub, w, mlp.s1)], [S.w8a8_int8_linear(x, w, mlp.s1)]),
                 ([S.int8_scaled_mm(q.as_subclass(Sub), w.t(), s, mlp.s1, torch.float32)], [S.int8_scaled_mm(q, w.t(), s, mlp.s1, torch.float32)])):
        assert all(torch.equal(u.float(), v.float()) for u, v in zip(a, b))


def test_device_status_is_clear():
    from sglang_b200 import _native as N

    assert N.read_device_status() == 0
