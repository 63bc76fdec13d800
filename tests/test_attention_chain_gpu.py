"""A decoder layer's attention block as it is run: norm into FP8, qkv linear, norm and rotation of the heads with the append to the cache, attention over
the cache, o_proj linear, for prompts, single tokens and trees of drafted ones; and under what a server does to a call.

Link by link: every operator is tested on what the one before it gave, at that operator's own tolerance."""
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import sglang_b200 as S
from sglang_b200.weight_quant import block_quant_weight_fp8
from test_rotary_gpu import bits, check, check_cache, formula, split, table, weights
from test_tree_attention_gpu import Case

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
HEADS, KV, DIM, HIDDEN, PAGE, PAGES = 8, 2, 128, 1024, 16, 60


class Block:
    def __init__(self, held, seed=0, axes=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        linear = lambda n, k: block_quant_weight_fp8((torch.randn(n, k, generator=g, device="cuda") * 0.02).bfloat16())  # noqa: E731
        self.qkv, self.o = linear((HEADS + 2 * KV) * DIM, HIDDEN), linear(HIDDEN, HEADS * DIM)
        self.norm = (1 + 0.1 * torch.randn(HIDDEN, generator=g, device="cuda")).bfloat16()
        self.wq, self.wk = weights(DIM, torch.bfloat16)
        self.cs, self.axes = table(2048, DIM), axes
        self.kc, self.vc = (torch.zeros(PAGES, PAGE, KV, DIM, device="cuda").to(held) for _ in range(2))
        self.scale = torch.tensor([0.02], device="cuda") if held == FP8 else None

    def __call__(self, x, positions, slots, pages, lens, starts, mask=None):
        q8, s8 = S.rmsnorm_quant_fp8(x, self.norm, column_major_scales=True)
        qkv = S.w8a8_block_fp8_matmul(q8, self.qkv[0], s8, self.qkv[1], [128, 128], torch.bfloat16)
        q = S.qk_norm_rope_append(qkv, HEADS, KV, positions, self.cs, self.kc, self.vc, slots, self.wq, self.wk, mrope_section=self.axes,
                                  k_scale=self.scale, v_scale=self.scale)
        out = S.tree_attention(q, self.kc, self.vc, pages, lens, starts, mask, k_scale=self.scale, v_scale=self.scale)
        return qkv, q, out, S.w8a8_block_fp8_linear(out.flatten(1), self.o[0], [128, 128], self.o[1])


class Sequences:
    """Pages, lengths and positions of a batch whose contexts grow step by step."""

    def __init__(self, n):
        self.pages = torch.randperm(PAGES, generator=torch.Generator().manual_seed(n))[: n * (PAGES // n)].view(n, -1).to(torch.int32).cuda()
        self.lens = [0] * n

    def step(self, counts):
        at, slots = [], []
        for b, n in enumerate(counts):
            for j in range(self.lens[b], self.lens[b] + n):
                at.append(j)
                slots.append(int(self.pages[b, j // PAGE]) * PAGE + j % PAGE)
            self.lens[b] += n
        to = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        return to(at), to(slots), to(self.lens), to([sum(counts[:b]) for b in range(len(counts) + 1)])


@pytest.mark.parametrize("held", [torch.bfloat16, FP8])
@pytest.mark.parametrize("axes", [None, [16, 24, 24]])
def test_prompt_then_tokens_then_trees(held, axes):
    block, seqs = Block(held, axes=axes), Sequences(3)
    g = torch.Generator(device="cuda").manual_seed(1)
    for counts, tree in (([130, 40, 7], False), ([1, 1, 1], False), ([8, 6, 8], True), ([1, 0, 2], False)):
        x = torch.randn(sum(counts), HIDDEN, generator=g, device="cuda").bfloat16()
        positions, slots, lens, starts = seqs.step(counts)
        if axes:
            positions = torch.stack([positions, positions // 3, positions % 5])
        mask = None
        if tree:
            mask = (torch.rand(sum(counts), max(counts), device="cuda") < 0.5) | torch.cat([torch.eye(max(counts), device="cuda")[:n] for n in counts]).bool()
        old = block.kc.clone(), block.vc.clone()
        qkv, q, out, y = block(x, positions, slots, seqs.pages, lens, starts, mask)
        parts = split(qkv, HEADS, KV)
        check(q, *formula(parts[0], block.wq, 1e-6, positions, block.cs, True, axes, False))
        check_cache(block.kc, old[0], slots, *formula(parts[1], block.wk, 1e-6, positions, block.cs, True, axes, False), block.scale)
        check_cache(block.vc, old[1], slots, parts[2].double(), torch.zeros_like(parts[2], dtype=torch.double), block.scale)
        c = Case([1], [1], HEADS, KV, DIM)
        c.lens, c.counts, c.page, c.held, c.q, c.kc, c.vc, c.table = list(seqs.lens), counts, PAGE, held, q, block.kc, block.vc, seqs.pages
        c.starts, c.mask, c.ks, c.vs = starts, mask, block.scale, block.scale
        c.check(out)
        assert torch.equal(y, S.w8a8_block_fp8_linear(out.flatten(1).contiguous(), block.o[0], [128, 128], block.o[1]))


def test_a_captured_step_serves_growing_contexts():
    """A decode step captured once, its inputs refilled: what a server does. Padded to four rows, the last of which belongs to no sequence."""
    block, seqs = Block(FP8), Sequences(3)
    eager = Block(FP8)
    x = torch.randn(177, HIDDEN, device="cuda").bfloat16()
    positions, slots, lens, starts = seqs.step([130, 40, 7])
    for b in (block, eager):
        b(x, positions, slots, seqs.pages, lens, starts)
    static = dict(x=torch.zeros(4, HIDDEN, device="cuda").bfloat16(), positions=torch.zeros(4, dtype=torch.int32, device="cuda"),
                  slots=torch.full((4,), -1, dtype=torch.int32, device="cuda"), pages=seqs.pages, lens=lens.clone(),
                  starts=torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda"))
    block(**static)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = block(**static)
    for _ in range(4):
        x = torch.randn(3, HIDDEN, device="cuda").bfloat16()
        positions, slots, lens, starts = seqs.step([1, 1, 1])
        static["x"][:3], static["positions"][:3], static["slots"][:3] = x, positions, slots
        static["lens"].copy_(lens)
        graph.replay()
        want = eager(**{n: t.clone() for n, t in static.items()})
        for g, w in zip(got, want):
            assert torch.equal(g[:3], w[:3])  # (the fourth belongs to no sequence)
        assert torch.equal(bits(block.kc), bits(eager.kc)) and torch.equal(bits(block.vc), bits(eager.vc))


def test_threads_on_streams_of_their_own():
    cases = [Case([900 + 37 * i, 300], [3, 1], 8, 2, 128, torch.bfloat16, FP8, 16, True, seed=i) for i in range(4)]
    want = [c() for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def run(c, w):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not torch.equal(c(), w):
                    wrong.append(c)

    threads = [threading.Thread(target=run, args=a) for a in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_dispatcher_ops_give_the_same_bits():
    ops = torch.ops.sglang_b200
    x = torch.randn(20, 12 * DIM, device="cuda").bfloat16()
    pos, cs = torch.arange(20, device="cuda"), table(64, DIM)
    wq, wk = weights(DIM, torch.bfloat16)
    for a, b in zip(ops.qk_norm_rope(x, 8, 2, pos, cs, wq, wk, 1e-6), S.qk_norm_rope(x, 8, 2, pos, cs, wq, wk)):
        assert torch.equal(a, b)
    caches = [torch.zeros(4, 8, 2, DIM, device="cuda").to(FP8) for _ in range(6)]
    q1 = ops.qk_norm_rope_append(x, 8, 2, pos, cs, caches[0], caches[1], pos, wq, wk)
    q2 = S.qk_norm_rope_append(x, 8, 2, pos, cs, caches[2], caches[3], pos, wq, wk)
    _, k, v = split(x, 8, 2)
    ops.append_paged_kv(k, v, caches[4], caches[5], pos)
    assert torch.equal(q1, q2) and all(torch.equal(bits(a), bits(b)) for a, b in zip(caches[:2], caches[2:4]))
    assert torch.equal(bits(caches[5]), bits(caches[1]))
    c = Case([100, 40], [3, 2], 8, 2, 128, mask=True)
    assert torch.equal(ops.tree_attention(c.q, c.kc, c.vc, c.table, c.seq_lens, c.starts, c.mask), c())


def test_native_and_general_host_path_agree():
    """A call with return_lse, or through a subclass, takes the general path of Python: the same bits."""
    c = Case([700, 40, 129], [6, 2, 1], 8, 2, 128, torch.float16, FP8, 16, True)
    assert torch.equal(c(), c(return_lse=True)[0])
    x = torch.randn(9, 12 * DIM, device="cuda").half()
    sub = torch.nn.Parameter(x, requires_grad=False)
    pos, cs = torch.stack([torch.arange(9, device="cuda")] * 3), table(64, DIM)
    for inter, section in ((False, [16, 24, 24]), (True, [24, 20, 20])):
        for a, b in zip(S.qk_norm_rope(x, 8, 2, pos, cs, None, None, 1e-6, False, section, inter),
                        S.qk_norm_rope(sub, 8, 2, pos, cs, None, None, 1e-6, False, tuple(section), inter)):
            assert torch.equal(a, b)


def test_a_first_call_may_be_a_captured_one():
    """A process whose first calls of the operators are captured: what they set up once must not need the stream."""
    code = """
import torch, sglang_b200 as S
x = torch.randn(5, 12 * 128, device='cuda').bfloat16()
at = torch.arange(5, device='cuda', dtype=torch.int32)
kc, vc = (torch.zeros(2, 16, 2, 128, device='cuda', dtype=torch.bfloat16) for _ in range(2))
cs = torch.randn(9, 128, device='cuda')
pages, lens, starts = (torch.tensor(t, device='cuda', dtype=torch.int32) for t in ([[0]], [5], [0, 5]))
torch.cuda.synchronize()
def step():
    q = S.qk_norm_rope_append(x, 8, 2, at, cs, kc, vc, at)
    return q, S.tree_attention(q, kc, vc, pages, lens, starts)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
got = [t.clone() for t in got]
assert got[1].abs().sum() > 0 and all(torch.equal(a, b) for a, b in zip(got, step()))
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=Path(__file__).resolve().parent.parent)
