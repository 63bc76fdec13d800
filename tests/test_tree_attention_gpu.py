"""Attention of the newest tokens over a paged cache against its definition in 64 bits.

Tolerance. With h half a step of the 16-bit type (relative), weights p rounded to p (1 + d), |d| <= h, and exponents off by e (fp32 sums of D
exact products, added in an order and with a rounding that is not specified: D steps of 2^-23 of the terms' size; the exponential itself 2^-21 and
the rounding of exponents of size t, t 2^-23):
    |o' - o| <= h |o'| + 2 (h + e) A,   A = sum p |v| / sum p
and for fp16, whose weights below 2^-14 are rounded to multiples of 2^-24, L 2^-25 max |v| more, as the sum of the weights is at least 1. Errors of
single weights have no common sign: the whole result is tested for twice h times (its size + that of the weights' errors) in the root mean square."""
import math

import pytest
import torch

import sglang_b200 as S

pytestmark = pytest.mark.gpu
BF, HF, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


class Case:
    """Sequences of ``lens`` keys with ``counts`` new tokens each."""

    def __init__(self, lens, counts, q_heads, kv_heads, dim, dtype=BF, held=None, page=16, mask=False, seed=0, spread=1.5, extra_rows=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.counts, self.page, self.dim = lens, counts, page, dim
        self.q_heads, self.kv_heads, self.dtype, self.held = q_heads, kv_heads, dtype, held or dtype
        T = sum(counts) + extra_rows
        self.q = (torch.randn(T, q_heads, dim, generator=g, device="cuda") * spread).to(dtype)
        need = [-(-max(n, 0) // page) for n in lens]
        pages = sum(need) + 2
        k, v = (torch.randn(pages, page, kv_heads, dim, generator=g, device="cuda") for _ in range(2))
        self.ks = self.vs = None
        if self.held == FP8:
            k, v = (k * 90).clamp(-448, 448), (v * 70).clamp(-448, 448)
            self.ks = (torch.rand(kv_heads, generator=g, device="cuda") + 0.5) / 90
            self.vs = (torch.rand(1, generator=g, device="cuda") + 0.5) / 70
        self.kc, self.vc = k.to(self.held), v.to(self.held)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), max(need + [1])), 2**31 - 1, dtype=torch.int32, device="cuda")  # what no key asks for is not read
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at : at + n]
            at += n
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.starts = torch.tensor([sum(counts[:b]) for b in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        self.mask = None
        if mask:
            width = max(counts)
            self.mask = torch.rand(T, width, generator=g, device="cuda") < 0.5
            for b, n in enumerate(counts):
                at = int(self.starts[b])
                if n:
                    self.mask[at : at + n, :n] |= torch.eye(n, dtype=torch.bool, device="cuda")

    def __call__(self, **kw):
        return S.tree_attention(self.q, self.kc, self.vc, self.table, self.seq_lens, self.starts, self.mask, k_scale=self.ks, v_scale=self.vs, **kw)

    def visible(self, b):
        n, length = self.counts[b], self.lens[b]
        j = torch.arange(length, device="cuda") - (length - n)  # index among the new tokens
        i = torch.arange(n, device="cuda")[:, None]
        if self.mask is None:
            return j <= i
        rows = self.mask[int(self.starts[b]) : int(self.starts[b]) + n]
        known = (j >= 0) & (j < rows.shape[1])
        return (j < 0) | (known & rows[:, j.clamp(0, max(0, rows.shape[1] - 1))]) if rows.shape[1] else (j < 0).expand(n, -1)

    def keys(self, b):
        j = torch.arange(self.lens[b], device="cuda")
        page = self.table[b].long()[j // self.page] if self.lens[b] else j
        k, v = self.kc[page, j % self.page].double(), self.vc[page, j % self.page].double()
        if self.ks is not None:
            k, v = k * self.ks.double().view(1, -1, 1), v * self.vs.double().view(1, -1, 1)
        return k, v

    def check(self, out, lse=None, scale=None):
        scale = self.dim**-0.5 if scale is None else scale
        half = torch.finfo(self.dtype).eps / 2
        group = self.q_heads // self.kv_heads
        off = size = 0.0
        for b, n in enumerate(self.counts):
            if n == 0:
                continue
            at = int(self.starts[b])
            k, v = (t.transpose(0, 1).repeat_interleave(group, 0) for t in self.keys(b))  # [heads, L, dim]
            q = self.q[at : at + n].double().transpose(0, 1)
            sees = self.visible(b)
            s = (q @ k.transpose(1, 2)) * scale
            terms = (q.abs() @ k.abs().transpose(1, 2)) * scale
            e = (terms * (self.dim * 2.0**-23) + s.abs() * 2.0**-21).masked_fill(~sees, 0).amax(-1, keepdim=True) + 2.0**-20 if self.lens[b] else 0
            s = s.masked_fill(~sees, -math.inf)
            top = s.amax(-1, keepdim=True) if self.lens[b] else s.new_full((*s.shape[:2], 1), -math.inf)
            p = torch.exp(s - top.masked_fill(top == -math.inf, 0))
            total = p.sum(-1, keepdim=True)
            w = p / total.clamp(min=1e-300)
            vis_v = v.masked_fill(~sees.any(0)[None, :, None], 0) if self.lens[b] else v
            want = w @ vis_v
            bound = 2 * (half + e) * (w @ vis_v.abs()) + (self.lens[b] * 2.0**-25 * vis_v.abs().amax() if self.dtype == HF and self.lens[b] else 0)
            got = out[at : at + n].double().transpose(0, 1)
            bound = bound + half * torch.maximum(got.abs(), want.abs()) + 2.0**-25
            err = (got - want).abs()
            assert not torch.isnan(got).any()
            assert (err <= bound).all(), f"sequence {b}: {(err / bound).max().item():.2f} of the bound"
            off += (err**2).sum().item()
            size += (want**2).sum().item() + ((w**2) @ (vis_v**2)).sum().item()
            if lse is not None:
                ref = (top + total.log()).squeeze(-1).transpose(0, 1)
                none = ~sees.any(-1) if self.lens[b] else torch.ones(n, dtype=torch.bool, device="cuda")
                assert (lse[at : at + n][none] == -math.inf).all()
                d = (lse[at : at + n].double() - ref)[~none].abs()
                assert (d <= (half + 2 * e.max()) + ref[~none].abs() * 2.0**-22).all() if d.numel() else True
        if size:
            assert math.sqrt(off) <= 2 * half * math.sqrt(size), f"root mean square {math.sqrt(off / size) / half:.2f} half steps"


def test_one_key():
    c = Case([1], [1], 1, 1, 64)
    c.check(*c(return_lse=True))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype, held", [(BF, None), (HF, None), (BF, FP8), (HF, FP8)])
def test_one_tile(dim, dtype, held):
    c = Case([50], [1], 4, 1, dim, dtype, held)
    c.check(*c(return_lse=True))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype, held", [(BF, None), (HF, None), (BF, FP8), (HF, FP8)])
@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 127, 128, 129, 255, 257, 640, 1031])
def test_one_token_of_every_length(length, dtype, held, dim):
    c = Case([length], [1], 8, 2, dim, dtype, held, seed=length)
    c.check(*c(return_lse=True))


@pytest.mark.parametrize("page", [1, 2, 5, 16, 64, 100, 256])
@pytest.mark.parametrize("held", [None, FP8])
def test_ragged_batch(held, page):
    lens = [700, 1, 128, 33, 5000, 129, 64, 2, 300, 1024, 4097]
    c = Case(lens, [1] * len(lens), 8, 2, 128, BF, held, page)
    c.check(*c(return_lse=True))


@pytest.mark.parametrize("group, kv", [(1, 8), (1, 1), (4, 2), (5, 3), (7, 1), (16, 1), (64, 1), (128, 1), (200, 1)])
@pytest.mark.parametrize("mask", [False, True])
def test_groups(group, kv, mask):
    c = Case([300, 170, 9], [6, 1, 9], group * kv, kv, 64, BF, None, 16, mask)
    c.check(*c(return_lse=True))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("held", [None, FP8])
@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("lens, counts", [([40], [40]), ([129, 200], [7, 64]), ([2000, 1, 130, 0, 128], [33, 1, 3, 0, 128]),
                                          ([500, 900], [300, 140]), ([130, 131], [2, 3])])
def test_trees_and_chains(lens, counts, mask, held, dim):
    c = Case(lens, counts, 4, 2, dim, BF, held, 32, mask)
    c.check(*c(return_lse=True))


def test_a_long_context_is_cut_over_all_sms():
    for dim, dtype, held, counts in ((128, BF, None, [1]), (128, HF, FP8, [20]), (64, HF, None, [4]), (256, BF, FP8, [3])):
        c = Case([70001], counts, 8, 1, dim, dtype, held, 64, counts[0] > 1)
        c.check(*c(return_lse=True))


def test_many_sequences():
    g = torch.Generator().manual_seed(0)
    lens = [int(x) for x in torch.randint(1, 400, (1000,), generator=g)]
    counts = [min(n, int(x)) for n, x in zip(lens, torch.randint(0, 4, (1000,), generator=g))]
    c = Case(lens, counts, 2, 1, 64, BF, None, 8)
    c.check(*c(return_lse=True))


def test_sequences_without_tokens_at_either_end():
    c = Case([9, 300, 0, 50, 77], [0, 5, 0, 2, 0], 4, 2, 128)
    c.check(*c(return_lse=True))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_that_see_nothing(dim):
    # fewer keys than tokens, no keys at all, a mask without a bit
    c = Case([3, 0, 20], [5, 2, 4], 4, 2, dim)
    c.check(*c(return_lse=True))
    c = Case([4, 140], [4, 140], 4, 2, dim, mask=True)
    c.mask[1] = False
    c.mask[50:60] = False
    out, lse = c(return_lse=True)
    c.check(out, lse)
    assert (out[1] == 0).all() and (out[50:60] == 0).all() and (lse[50:60] == -math.inf).all()


def test_a_mask_narrower_than_the_tree():
    c = Case([200, 50], [10, 3], 4, 2, 128, mask=True)
    c.mask = c.mask[:, :6]
    c.check(*c(return_lse=True))
    c.mask = c.mask[:, :0]
    c.check(*c(return_lse=True))
    c.mask = torch.ones(13, 40, dtype=torch.bool, device="cuda")[:, 3:30]
    c.check(*c(return_lse=True))


def test_no_starts_means_a_token_each():
    c = Case([100, 7, 300], [1, 1, 1], 8, 2, 128)
    a = c()
    b = S.tree_attention(c.q, c.kc, c.vc, c.table, c.seq_lens)
    assert torch.equal(a, b)


def test_rows_behind_the_last_sequence_stay():
    c = Case([100, 300], [3, 1], 8, 2, 128, extra_rows=5)
    out = torch.full_like(c.q, 7)
    assert c(out=out) is out
    c.check(out)
    assert (out[4:] == 7).all()


@pytest.mark.parametrize("scale", [1.0, 0.01, 3.0])
def test_scale_and_sharp_rows(scale):
    c = Case([600, 90], [4, 2], 4, 2, 128, mask=True, spread=3.0)
    c.check(*c(scale=scale, return_lse=True), scale=scale)


def test_growing_scores_move_the_reference():
    """Keys that grow along the sequence, so that the largest score rises tile after tile."""
    for dtype in (BF, HF):
        c = Case([1500], [2], 8, 1, 128, dtype, page=16)
        flat = torch.arange(1500, device="cuda")
        ramp = (flat / 1500 * 12).to(dtype)
        direction = c.q[0, 0] / c.q[0, 0].float().norm()
        c.kc[c.table[0].long()[flat // 16], flat % 16, 0] = (ramp[:, None] * direction).to(dtype)
        c.check(*c(return_lse=True))


def test_layouts():
    """Caches as halves of one tensor and with heads before tokens; queries as a slice of the qkv linear's rows."""
    c = Case([100, 333], [2, 5], 8, 2, 128, mask=True)
    want = c()
    joint = torch.stack([c.kc, c.vc], 1)
    c.kc, c.vc = joint.unbind(1)
    assert torch.equal(c(), want)
    c.kc, c.vc = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.kc, c.vc))
    assert torch.equal(c(), want)
    wide = torch.zeros(7, 12 * 128, dtype=BF, device="cuda")
    wide[:, : 8 * 128] = c.q.flatten(1)
    c.q = wide[:, : 8 * 128].unflatten(1, (8, 128))
    assert not c.q.is_contiguous() and torch.equal(c(), want)
    c.table = torch.cat([torch.full_like(c.table, -5), c.table, c.table], 1)[:, c.table.shape[1] : 2 * c.table.shape[1]]
    assert torch.equal(c(), want)


def test_distances_that_lead_nowhere():
    """One token of rows whose length is no multiple of 16 bytes, one kv head, one page of one token."""
    c = Case([1], [1], 4, 1, 64, page=1)
    c.kc, c.vc = c.kc[int(c.table[0, 0])][None], c.vc[int(c.table[0, 0])][None]
    c.table = torch.zeros_like(c.table)
    want = c()
    c.check(want)
    c.q = c.q.as_strided(c.q.shape, (4 * 64 + 3, 64, 1))
    c.kc, c.vc = (t.as_strided(t.shape, (3, 5, 7, 1)) for t in (c.kc, c.vc))
    assert c.q.stride(0) % 8 and torch.equal(c(), want) and torch.equal(c(return_lse=True)[0], want)


def test_what_no_row_sees_does_not_matter():
    """Garbage behind the last key of a page, in pages of no sequence."""
    for held in (None, FP8):
        c = Case([100, 33], [3, 1], 4, 2, 128, BF, held, mask=True)
        used = torch.zeros(c.kc.shape[:2], dtype=torch.bool, device="cuda")
        for b, n in enumerate(c.lens):
            j = torch.arange(n, device="cuda")
            used[c.table[b].long()[j // 16], j % 16] = True
        want = c()
        for t in (c.kc, c.vc):
            t.view(torch.uint8 if held else torch.int16)[~used] = 0x7F if held else 0x7FFF  # the types' NaN
        assert torch.equal(c(), want)


def test_pages_that_the_cache_does_not_have():
    c = Case([100, 40, 200], [1, 1, 1], 4, 2, 128)
    want = c()
    c.table[1, 1] = c.kc.shape[0]
    c.table[2, 0] = -1
    out = c()
    assert torch.equal(out[0], want[0]) and torch.isnan(out[1:]).all()


def test_lengths_past_the_page_table_are_cut():
    c = Case([64, 40], [1, 1], 4, 2, 128)
    want = c()
    c.seq_lens[0] = 2**31 - 1
    assert torch.equal(c(), want)
    c.seq_lens[0] = -4
    out = c()
    assert (out[0] == 0).all() and torch.equal(out[1], want[1])


def test_an_infinite_score_is_nan_and_stays_in_its_row():
    c = Case([100, 40], [2, 1], 4, 2, 128)
    want = c()
    c.q[0, 0, 0] = math.inf
    out = c()
    assert torch.isnan(out[0, 0]).all() and torch.equal(out[0, 1:], want[0, 1:]) and torch.equal(out[1:], want[1:])


def test_same_bits_every_time_on_any_stream_and_in_graphs():
    c = Case([9000, 300, 12000], [4, 2, 6], 8, 2, 128, BF, FP8, mask=True)
    want = c()
    for _ in range(10):
        assert torch.equal(c(), want)
    graphs = []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            out = c()
        graphs.append((graph, out, side))
    for _ in range(5):
        for graph, out, side in graphs:  # at the same time: each has a workspace of its own
            with torch.cuda.stream(side):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out, _ in graphs)


def test_lengths_of_a_captured_call_may_change():
    c = Case([400, 900], [3, 3], 8, 2, 128, mask=True)
    graph = torch.cuda.CUDAGraph()
    c()
    with torch.cuda.graph(graph):
        out = c()
    for lens in ([400, 900], [3, 17], [129, 128]):
        c.lens = lens
        c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        c.check(out)


def test_far_pages():
    """Offsets past 32 bits in a cache of more than 2^32 elements."""
    pages = (1 << 32) // (16 * 2 * 128) + 40
    kc, vc = (torch.zeros(pages, 16, 2, 128, dtype=torch.uint8, device="cuda").view(FP8) for _ in range(2))
    c = Case([600], [4], 4, 2, 128, BF, FP8, 16)
    n = c.kc.shape[0]
    want = c()
    for far, near in ((kc, c.kc), (vc, c.vc)):
        far[-n:] = near
    c.table += pages - n
    c.kc, c.vc = kc, vc
    assert torch.equal(c(), want)


def test_device_status_is_clean():
    from sglang_b200 import _native as N

    assert N.read_device_status() == 0


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("held", [None, FP8])
@pytest.mark.parametrize("lens, counts, heads", [([140], [12], 1), ([300, 9], [20, 9], 8), ([70, 1300], [5, 130], 2)])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(lens, counts, heads, held, dim):
    """A drafted token whose value has NaN or infinities: rows whose mask hides it are what they were, the others get those elements alone."""
    for mask in (True, False):
        c = Case(lens, counts, 2 * heads, 2, dim, BF, held, 16, mask)
        want, lse = c(return_lse=True)
        for b, (length, n) in enumerate(zip(lens, counts)):
            own = n - 2  # (its index among the new tokens)
            j = length - n + own
            row = c.vc[int(c.table[b, j // 16]), j % 16, 1]
            if held:
                row.view(torch.uint8)[5], row.view(torch.uint8)[dim - 1] = 0x7F, 0xFF
            else:
                row[5], row[dim - 1], row[8] = math.nan, math.inf, -math.inf
        got, lse2 = c(return_lse=True)
        assert torch.equal(lse, lse2)
        for b, (length, n) in enumerate(zip(lens, counts)):
            at, own = int(c.starts[b]), n - 2
            sees = c.visible(b)[:, length - n + own]
            for i in range(n):
                g, w = got[at + i], want[at + i]
                assert torch.equal(g[:heads], w[:heads])  # the other kv head's
                odd = torch.zeros(dim, dtype=torch.bool, device="cuda")
                if sees[i]:
                    odd[[5, dim - 1] if held else [5, dim - 1, 8]] = True
                    assert torch.isnan(g[heads:, 5]).all()
                    if not held:
                        assert (g[heads:, dim - 1] == math.inf).all() and (g[heads:, 8] == -math.inf).all()
                    else:
                        assert torch.isnan(g[heads:, dim - 1]).all()
                # the other elements lose nothing but what the taken-out ones did not add
                assert torch.equal(g[heads:, ~odd], w[heads:, ~odd])


def test_short_sequences_of_very_different_queries():
    """Row tiles of a single tile of keys one after the other, the power of two that scales their queries another for each."""
    for group in (1, 4, 8):
        lens = [20 + 7 * b % 110 for b in range(900)]
        c = Case(lens, [1] * len(lens), 2 * group, 2, 128, BF, FP8)
        c.q = (c.q.float() * torch.pow(4.0, (torch.arange(900, device="cuda") % 5 - 4).float())[:, None, None]).to(BF)
        want = c()
        c.check(want)
        for _ in range(5):
            assert torch.equal(c(), want)


@pytest.mark.parametrize("held", [None, FP8])
@pytest.mark.parametrize("mask", [False, True])
def test_many_masked_tiles_of_partly_filled_row_tiles(mask, held):
    """Row tiles of 128 with 4, 20, 60 and 92 rows at the end of every sequence, up to eight tiles of keys that not every row sees one after the other in
    the same CTA: the definition, and the same bits every time."""
    counts = [288 + (b * 37) % 11 * 32 + [1, 5, 15, 23][b % 4] for b in range(64)]
    assert {n * 4 % 128 for n in counts} == {4, 20, 60, 92} and max(counts) < 700
    lens = [n + [0, 100, 61][b % 3] for b, n in enumerate(counts)]
    c = Case(lens, counts, 8, 2, 128, BF, held, 16, mask)
    want, lse = c(return_lse=True)
    c.check(want, lse)
    for _ in range(40):
        assert torch.equal(c(), want)


def test_masked_tiles_in_the_first_places_of_a_piece():
    """Nothing but masked tiles: a drafted tree, or a chain, of 9 to 12 tokens of eight heads across a multiple of 128 keys."""
    for mask in (False, True):
        lens = [128 * (1 + b % 3) + 1 + b % 8 for b in range(296)]
        counts = [9 + b % 4 for b in range(296)]
        c = Case(lens, counts, 8, 1, 128, BF, FP8, 16, mask)
        want, lse = c(return_lse=True)
        c.check(want, lse)
        for _ in range(100):
            assert torch.equal(c(), want)


@pytest.mark.parametrize("held", [None, FP8])
@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("dim, group", [(64, 1), (128, 1), (128, 3), (128, 16), (256, 2)])
def test_many_values_that_are_not_finite(dim, group, mask, held):
    """A third of the own values are NaN or infinite: every row takes what it sees, the other elements keep their bits."""
    lens, counts = [300, 40, 700], [150, 33, 21]
    c = Case(lens, counts, 2 * group, 2, dim, BF, held, 16, mask)
    if mask:
        c.mask[torch.rand(c.mask.shape, device="cuda") < 0.7] = False
    want = c()
    g = torch.Generator(device="cuda").manual_seed(3)
    expected = []
    for b, (length, n) in enumerate(zip(lens, counts)):
        kind = torch.randint(0, 9, (n, 2, dim), generator=g, device="cuda")  # 0: NaN, 1, 2: infinities, others stay
        j = torch.arange(length - n, length, device="cuda")
        page = c.table[b].long()[j // 16]
        v = c.vc[page, j % 16]
        if held:
            v = v.view(torch.uint8).masked_fill(kind < 3, 0x7F).view(FP8)
        else:
            v = v.masked_fill(kind == 0, math.nan).masked_fill(kind == 1, math.inf).masked_fill(kind == 2, -math.inf)
        bits = torch.uint8 if held else torch.int16
        c.vc.view(bits)[page, j % 16] = v.view(bits)
        sees = c.visible(b)[:, length - n :].float()
        met = [torch.einsum("ij,jhd->ihd", sees, (kind == k).float()) > 0 for k in range(3)]
        nan = met[0] | met[1] | met[2] if held else met[0] | (met[1] & met[2])
        expected.append(torch.where(nan, 3, torch.where(met[1], 1, torch.where(met[2], 2, 0))).repeat_interleave(group, 1))
    got, kind = c(), torch.cat(expected)
    assert torch.equal(torch.isnan(got), kind == 3)
    assert torch.equal(got == math.inf, kind == 1) and torch.equal(got == -math.inf, kind == 2)
    assert torch.equal(got[kind == 0], want[kind == 0])


@pytest.mark.parametrize("held", [None, FP8])
def test_a_long_prompt_of_values_that_are_not_finite(held):
    """What they cost must stay below what the kernel's other warps wait for, whose waits end."""
    from sglang_b200 import _native as N

    n = 32768
    c = Case([n], [n], 1, 1, 64, BF, held, 64)
    want = c()
    j = torch.arange(n, device="cuda")
    rows = c.vc.view(torch.uint8 if held else BF)
    page = c.table[0].long()[j // 64]
    if held:
        rows[page, j % 64, 0, 5] = 0x7F
        rows[page[1000:], j[1000:] % 64, 0, 9] = 0xFF
    else:
        rows[page, j % 64, 0, 5] = math.nan
        rows[page[1000:], j[1000:] % 64, 0, 9] = math.inf
        rows[page[10], 10, 0, 12], rows[page[20000], 20000 % 64, 0, 12] = math.inf, -math.inf
    got = c()[:, 0]
    assert N.read_device_status() == 0
    assert torch.isnan(got[:, 5]).all()
    assert torch.equal(got[:1000, 9], want[:1000, 0, 9])
    assert torch.isnan(got[1000:, 9]).all() if held else (got[1000:, 9] == math.inf).all()
    if not held:
        assert torch.equal(got[:10, 12], want[:10, 0, 12]) and (got[10:20000, 12] == math.inf).all() and torch.isnan(got[20000:, 12]).all()
    others = [d for d in range(64) if d not in (5, 9, 12)]
    assert torch.equal(got[:, others], want[:, 0, others])


@pytest.mark.parametrize("dtype, held", [(BF, FP8), (HF, FP8), (HF, None), (BF, None)])
@pytest.mark.parametrize("dim, group, n", [(64, 1, 1), (128, 8, 1), (128, 8, 4), (64, 8, 8), (128, 8, 16), (256, 4, 8)])
def test_one_large_key_above_a_long_flat_context(dim, group, n, dtype, held):
    """A key whose weight is 2^26 times that of every other, 131072 of them: together 2^-9 of the result, which fp16 weights of the largest key's
    size would lose. The largest weight is 2^7 or more and steps are 2^-24, so a weight is off by 2^-32 of it at most."""
    L = 131072
    c = Case([L] * 3, [n] * 3, group, 1, dim, dtype, held, 64)
    c.ks = c.vs = None
    c.q.zero_()
    c.q[:, :, 0] = dim**0.5  # 18 * 1.4427 = 25.97 powers of two for a key of 18
    score = float(c.q[0, 0, 0]) * 18 * dim**-0.5  # (the query as its type holds it)
    for t in (c.kc, c.vc):
        t.view(torch.uint8 if held else torch.int16).zero_()
    v = torch.tensor([1.0, -2.0, 0.5, 0.0], device="cuda").repeat(dim // 4)
    c.vc.copy_(v.to(c.held).expand(c.vc.shape))
    for b, j in enumerate((3, L // 2 + 77, L - n - 1)):
        page = int(c.table[b, j // 64])
        c.kc[page, j % 64, 0, 0] = 18.0
        c.vc[page, j % 64] = torch.zeros(dim, device="cuda").to(c.held)
    out, lse = c(return_lse=True)
    half = torch.finfo(dtype).eps / 2
    weight = math.exp(-score)
    for b in range(3):
        for i in range(n):
            others = L - n + i  # (without the large one)
            total = 1 + others * weight
            want = others * weight / total * v.double()
            got = out[b * n + i].double()
            # one rounding of the result, twice the weights' and the exponentials' (scores are exact but for the scale: 2^-22 of 26), and what fp16 loses
            bound = (3 * half + 2.0**-15) * want.abs() + L * 2.0**-32 * v.double().abs()
            assert ((got - want).abs() <= bound).all(), (b, i, got[0, :4], want[:4])
            assert (lse[b * n + i].double() - (score + math.log(total))).abs().max() <= 18 * 2.0**-21 + 2.0**-15


def test_weights_at_the_top_of_fp16():
    """Scores that rise by just less than what moves a reference: weights up to 2^15, and sums of them."""
    for held in (None, FP8):
        for group, n in ((1, 1), (8, 4), (8, 8), (8, 16)):
            c = Case([3000], [n], group, 1, 64, HF, held)
            c.ks = c.vs = None
            c.q.zero_()
            c.q[:, :, 0] = 8
            c.kc.view(torch.uint8 if held else torch.int16).zero_()
            j = torch.arange(3000, device="cuda")
            c.kc[c.table[0].long()[j // 16], j % 16, 0, 0] = ((j >= 200).float() * 5.5).to(c.held)  # 7.93 powers of two
            c.check(*c(return_lse=True))


@pytest.mark.parametrize("group, n", [(1, 1), (8, 4), (8, 8), (8, 16)])
@pytest.mark.parametrize("power", [115, 117, 121, 125])
def test_queries_at_the_end_of_bf16_over_an_fp8_cache(power, group, n):
    """Rows of up to 2^128 whose scores a small scale (a normal number even so) makes ordinary ones: the bits of rows of ordinary size."""
    c = Case([700, 130], [n, n], 2 * group, 2, 64, BF, FP8)
    c.kc = (c.kc.float() * 2.0**-10).to(FP8)
    c.ks = torch.ones(1, device="cuda")
    want = c(scale=2.0)
    c.check(want, scale=2.0)
    c.q = c.q * 2.0**power
    assert torch.isfinite(c.q).all()
    assert torch.equal(c(scale=2.0 * 2.0**-power), want)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("group, n", [(1, 1), (8, 4), (8, 8), (8, 16)])
def test_scales_whose_product_is_nothing(group, n, dtype):
    """Scores that vanish altogether: every key that a row sees counts alike, the others not at all."""
    for mask in (False, True):
        c = Case([700, n], [n, n], 2 * group, 2, 64, dtype, FP8, mask=mask)
        c.ks = torch.full((2,), 1e-12, device="cuda")
        c.check(*c(scale=1e-38, return_lse=True), scale=1e-38)


@pytest.mark.parametrize("held", [None, FP8])
@pytest.mark.parametrize("group, n", [(1, 1), (8, 4), (8, 8), (8, 16)])
@pytest.mark.parametrize("sequences", [1, 300])
def test_a_value_that_is_not_a_number_shows_whatever_its_weight(sequences, group, n, held):
    """NaN among the values that every row sees, its key 2^230 below another: in the other group's tile, in the other half of a tile, in another piece."""
    for bad, large in ((5, 130), (5, 70), (70, 5), (130, 5)):
        c = Case([200 + n] * sequences, [n] * sequences, group, 1, 64, BF, held)
        c.ks = c.vs = None
        c.q.zero_()
        c.q[:, :, 0] = 64
        c.kc.view(torch.uint8 if held else torch.int16).zero_()
        c.kc[c.table[:, large // 16].long(), large % 16, 0, 0] = 20.0
        where = c.table[:, bad // 16].long(), torch.tensor(bad % 16, device="cuda"), torch.tensor(0, device="cuda"), torch.tensor(7, device="cuda")
        want = c()
        assert torch.isfinite(want).all()
        bits = torch.uint8 if held else torch.int16
        c.vc.view(bits)[where] = 0x7F if held else 0x7FC0
        out = c()
        assert torch.isnan(out[..., 7]).all(), (bad, large)
        others = [d for d in range(64) if d != 7]
        assert torch.equal(out[..., others], want[..., others])


@pytest.mark.parametrize("dtype, held", [(BF, FP8), (HF, FP8), (HF, None), (BF, None)])
@pytest.mark.parametrize("dim, group, n", [(64, 1, 1), (128, 8, 1), (128, 8, 4), (64, 8, 8), (128, 8, 16), (256, 4, 8)])
def test_one_large_key_in_front_of_a_long_flat_context(dim, group, n, dtype, held):
    """As above, in so many sequences (over the same pages) that all keys of one are taken against the same reference: cut over many CTAs, only the piece
    with the large key would lose its others."""
    L, B = 131072, 300
    c = Case([L], [n], group, 1, dim, dtype, held, 64)
    c.q = (torch.zeros_like(c.q) + torch.eye(1, dim, dtype=dtype, device="cuda") * dim**0.5).repeat(B, 1, 1)
    score = float(c.q[0, 0, 0]) * 18 * dim**-0.5
    c.kc.view(torch.uint8 if held else torch.int16).zero_()
    v = torch.tensor([1.0, -2.0, 0.5, 0.0], device="cuda").repeat(dim // 4)
    c.vc.copy_(v.to(c.held).expand(c.vc.shape))
    page = int(c.table[0, 0])
    c.kc[page, 3, 0, 0] = 18.0
    c.vc[page, 3] = torch.zeros(dim, device="cuda").to(c.held)
    c.table, c.seq_lens = c.table.repeat(B, 1), c.seq_lens.repeat(B)
    c.starts = torch.arange(B + 1, dtype=torch.int32, device="cuda") * n
    c.ks = c.vs = None
    out = c().view(B, n, group, dim).double()
    half, weight = torch.finfo(dtype).eps / 2, math.exp(-score)
    others = (L - n + torch.arange(n, device="cuda", dtype=torch.float64)).view(1, n, 1, 1)
    want = others * weight / (1 + others * weight) * v.double()
    bound = (3 * half + 2.0**-15) * want.abs() + L * 2.0**-32 * v.double().abs()
    assert ((out - want).abs() <= bound).all(), (out[0, 0, 0, :4], want[0, 0, 0, :4])


@pytest.mark.parametrize("held", [None, FP8])
@pytest.mark.parametrize("group, n", [(4, 1), (8, 16)])
def test_the_longest_line_of_a_page_table(group, n, held):
    """2^31 - 256 keys, the most that a line may name: one page again and again, so the result is that page's. fp32 sums of up to 2^17 tiles a CTA may be off by
    2^17 half steps, the weights' and the values' both."""
    c = Case([256], [n], group, 1, 64, BF, held, 256)
    page = c.table[:, :1].clone()
    k, v = c.keys(0)
    s = torch.einsum("thd,kd->thk", c.q.double(), k[:, 0]) * 64**-0.5
    want = torch.softmax(s, -1) @ v[:, 0]
    c.table, c.seq_lens = page.repeat(1, 0x7FFFFF00 // 256), torch.full_like(c.seq_lens, 2**31 - 1)
    out, lse = c(return_lse=True)
    size = torch.softmax(s, -1) @ v[:, 0].abs()
    assert ((out.double() - want).abs() <= 2.0**-9 * want.abs() + (2 * 2.0**-7 + 2.0**-8 + 2.0**-12) * size).all()
    assert ((lse.double() - (torch.logsumexp(s, -1) + math.log(0x7FFFFF00 / 256))).abs() <= 2.0**-7 + 2.0**-12).all()


def test_nothing_to_attend_to():
    c = Case([100], [2], 4, 2, 64)
    assert S.tree_attention(c.q[:0], c.kc, c.vc, c.table, c.seq_lens, torch.zeros_like(c.starts)).shape == (0, 4, 64)
    out = torch.full_like(c.q, 3)
    got = S.tree_attention(c.q, c.kc, c.vc, c.table[:0], c.seq_lens[:0], c.starts[:1], out=out)
    assert got is out and (out == 3).all()
    got = S.tree_attention(c.q, c.kc, c.vc, c.table[:, :0], c.seq_lens, c.starts)  # no page at all
    assert (got == 0).all()
