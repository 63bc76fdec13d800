"""Performance cases of the operators between a decoder layer's qkv linear and its o_proj linear: what an inference server has
them do.

``norm_rope``  RMSNorm of every head of q and k (where the model has one) and the rotation by position, q and k as new tensors.
``append``     keys, rotated on the way, and values into the pages of a cache, in 16 bits or in FP8 with a scale.
``layer``      both at once, as a layer does it behind its qkv linear: q as a new tensor, k and v into the cache.
``attend``     attention of the newest tokens of every sequence (one, or a tree of drafted ones) over the paged cache.

Head counts are those of the benchmark configurations of this repository (qkv widths of ``sglang_b200.synthetic``), their
tensor-parallel shards and generic ones; row counts run from one decoded token to a full prefill chunk, contexts from a few
tokens to 131072.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn}
EPS = 1e-6  # of the norm
BASE = 500000.0  # of the angles
MAX_ROWS = 16384 * 80 * 128  # elements of the largest chunk's q and k
MAX_KV = 640 << 20  # elements of keys and values that one attention pass may read


def _heads(rows, q, kv, dim):
    return {"rows": rows, "q_heads": q, "kv_heads": kv, "dim": dim}


def _rope(op, name, heads, dtype, rotated, halves=True, norm=True, axes=1, mixed=False, cache="", page=0, table=32768):
    """``rotated``: elements of a head that rotate; ``mixed``: axes alternate over the frequencies instead of in runs;
    ``table``: positions that the angles are tabulated for."""
    return {"name": name, "op": op, **heads, "dtype": dtype, "rotated": rotated, "halves": halves, "norm": norm, "axes": axes,
            "mixed": mixed, "cache": cache, "page": page, "table": table}


def _attend(name, seqs, longest, drafted, q, kv, dim, dtype, cache, page, tree=True):
    return {"name": name, "op": "attend", "seqs": seqs, "longest": longest, "drafted": drafted, "q_heads": q, "kv_heads": kv,
            "dim": dim, "dtype": dtype, "cache": cache, "page": page, "tree": tree}


def listed():
    return [
        # one user decoding far into a document: latency of one launch
        _rope("norm_rope", "norm_rope_decode_1", _heads(1, 32, 8, 128), "bf16", 128, table=131072),
        # a short prompt of an fp16 model without norms of q and k, whose heads rotate by half, as neighbouring pairs
        _rope("norm_rope", "norm_rope_203_fp16", _heads(203, 32, 8, 128), "fp16", 64, halves=False, norm=False),
        # the largest prefill chunk, images among the text: positions of time, height and width
        _rope("norm_rope", "norm_rope_axes_16384", _heads(16384, 64, 8, 128), "bf16", 128, axes=3),
        # a decode batch into an FP8 cache whose pages hold one token
        _rope("append", "append_decode_61_fp8", _heads(61, 64, 8, 128), "bf16", 128, norm=False, cache="fp8", page=1),
        # a ragged prefill chunk into a 16-bit cache
        _rope("append", "append_prefill_8191", _heads(8191, 64, 8, 128), "bf16", 128, norm=False, cache="bf16", page=64),
        # a decode batch of a layer with normed heads
        _rope("layer", "layer_decode_16", _heads(16, 32, 8, 128), "bf16", 128, cache="bf16", page=64),
        # a prefill chunk of a model for images, axes alternating over the frequencies, into an FP8 cache
        _rope("layer", "layer_axes_8192_fp8", _heads(8192, 32, 8, 128), "bf16", 128, axes=3, mixed=True, cache="fp8", page=64),
        # one user decoding in a short conversation, fp16 model
        _attend("attend_decode_1", 1, 1171, 1, 32, 8, 128, "fp16", "fp16", 16),
        # a decode batch, ragged contexts, one token per page
        _attend("attend_decode_128", 128, 8192, 1, 32, 8, 128, "bf16", "bf16", 1),
        # one user with a tree of drafted tokens on one rank of eight, FP8 cache, a long document
        _attend("attend_tree_1_fp8", 1, 131072, 32, 8, 1, 128, "bf16", "fp8", 64),
        # a batch of users, each with a small tree
        _attend("attend_tree_16", 16, 16384, 8, 64, 8, 128, "bf16", "bf16", 64),
        # a larger batch of trees on one rank of eight, FP8 cache
        _attend("attend_tree_61_fp8", 61, 32768, 16, 8, 1, 128, "bf16", "fp8", 32),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "layer", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    group, kv = rng.choice([1, 2, 4, 5, 7, 8, 16]), rng.choice([1, 2, 4, 8])
    cache = rng.choice([dtype, "fp8"])
    page = rng.choice([1, 16, 24, 32, 64, 128])
    if op == "attend":
        dim = rng.choice([64, 128, 128, 128, 256])
        seqs, longest = _log_int(rng, 1, 200), _log_int(rng, 8, 131072)
        drafted = 1 if rng.random() < 0.4 else min(_log_int(rng, 2, 64), longest)
        longest = max(8, drafted, min(longest, int(MAX_KV / (seqs * kv * dim) / max(1, drafted * group / 32))))
        c = _attend("", seqs, longest, drafted, group * kv, kv, dim, dtype, cache, page, rng.random() < 0.8)
    else:
        dim = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
        rotated = rng.choice([dim, dim, dim // 2 // 16 * 16])
        axes = rng.choice([1, 1, 3])
        rows = min(_log_int(rng, 1, 16384), MAX_ROWS // ((group + 2) * kv * dim))
        c = _rope(op, "", _heads(rows, group * kv, kv, dim), dtype, rotated, rng.random() < 0.7, op != "append" and rng.random() < 0.7,
                  axes, axes > 1 and rng.random() < 0.5, "" if op == "norm_rope" else cache, 0 if op == "norm_rope" else page)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------------------ inputs

def _sections(case):
    """Frequency pairs per axis: a quarter or so for time, the rest for height and width alike."""
    pairs = case["rotated"] // 2
    if case["axes"] == 1:
        return None
    side = pairs * 5 // 16 if case["mixed"] else pairs * 3 // 8
    return [pairs - 2 * side, side, side]


def _lengths(case):
    """Context lengths of the sequences, the drafted tokens among them: the longest first, the others spread below it."""
    low = max(1, case["drafted"])
    return [max(low, int(case["longest"] * (1 - (b * 0.6180339887) % 1.0))) for b in range(case["seqs"])]


def _drafted(case):
    """Newest tokens per sequence: trees are cut to different sizes."""
    return [max(1, case["drafted"] - b % 3) if case["tree"] else case["drafted"] for b in range(case["seqs"])]


def _table(case):
    pairs = case["rotated"] // 2
    rate = BASE ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    angle = torch.arange(case["table"], dtype=torch.float64, device="cuda")[:, None] * rate
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _to_cache(x, case):
    return x.to(DTYPES[case["cache"]]) if case["cache"] != "fp8" else (x * 80).clamp(-448, 448).to(DTYPES["fp8"])


def _prepare_rope(case, g):
    rows, q, kv, dim = case["rows"], case["q_heads"], case["kv_heads"], case["dim"]
    dtype, op = DTYPES[case["dtype"]], case["op"]
    s = dict(case, dtype=dtype, eps=EPS, sections=_sections(case))
    x = _normal(g, rows, (q + 2 * kv) * dim)
    x[:, torch.randperm(x.shape[1], generator=g, device="cuda")[: x.shape[1] // 100]] *= 20  # outlier channels
    x = x.to(dtype)
    if op == "append":  # slices of the qkv linear's rows
        s["k"], s["v"] = (t.unflatten(1, (kv, dim)) for t in x[:, q * dim :].chunk(2, 1))
    else:
        s["qkv"] = x
        s["wq"], s["wk"] = ((_normal(g, dim) * 0.1 + 1).to(dtype) if case["norm"] else None for _ in range(2))
    # consecutive tokens of one prompt, or anywhere for a decode batch; height and width within an image of 64 x 64
    first = torch.randint(0, case["table"] - rows, (1,), generator=g, device="cuda")
    text = first + torch.arange(rows, device="cuda") if rows > 256 else torch.randint(0, case["table"], (rows,), generator=g, device="cuda")
    if case["axes"] > 1:
        s["positions"] = torch.stack([text] + [(text // 64 ** i) % 64 + text // 4096 for i in range(case["axes"] - 1)])
    else:
        s["positions"] = text
    s["cos_sin"] = _table(case)
    if op != "norm_rope":
        pages = -(-rows // case["page"]) + 5
        shape = (pages, case["page"], kv, dim)
        s["kc"], s["vc"] = (_to_cache(_normal(g, *shape), case) for _ in range(2))
        at = torch.randperm(pages, generator=g, device="cuda")[: -(-rows // case["page"])]
        slots = (at[:, None] * case["page"] + torch.arange(case["page"], device="cuda")).flatten()
        s["slots"] = slots[:rows].contiguous()
        s["sk"], s["sv"] = (torch.rand(kv, generator=g, device="cuda") * 0.02 + 0.02 if case["cache"] == "fp8" else None
                            for _ in range(2))
    return s


def _trees(drafted, g):
    """``[tokens, widest]``: every token of a sequence's tree sees itself and the tokens on its way to the root."""
    width = max(drafted)
    mask = torch.eye(width, dtype=torch.bool).repeat(len(drafted), 1, 1)
    at = torch.arange(len(drafted))
    for i in range(1, width):  # parents are among the last few tokens, as in trees of a few branches
        parent = i - 1 - (torch.rand(len(drafted), generator=g) * min(i, 4)).long()
        mask[:, i] |= mask[at, parent]
    return torch.cat([mask[b, :n] for b, n in enumerate(drafted)])


def _prepare_attend(case, g, seed):
    seqs, q, kv, dim, page = case["seqs"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    lengths, drafted = _lengths(case), _drafted(case)
    s = dict(case, dtype=dtype, lengths=lengths, counts=drafted, scale=dim**-0.5)
    tokens = sum(drafted)
    s["q"] = (_normal(g, tokens, q, dim) * 1.5).to(dtype)
    need = [-(-n // page) for n in lengths]
    pages, fp8 = sum(need) + 3, case["cache"] == "fp8"
    s["kc"], s["vc"] = (torch.empty(pages, page, kv, dim, dtype=DTYPES[case["cache"]], device="cuda") for _ in range(2))
    step = max(1, (64 << 20) // (page * kv * dim))
    for cache in (s["kc"], s["vc"]):
        for i in range(0, pages, step):
            cache[i : i + step] = _to_cache(_normal(g, *cache[i : i + step].shape), case)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table, at = torch.zeros(seqs, max(need), dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    s["pages"] = table
    s["lens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    starts = [sum(drafted[:b]) for b in range(seqs + 1)]
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["mask"] = _trees(drafted, torch.Generator().manual_seed(seed)).cuda() if case["tree"] and case["drafted"] > 1 else None
    s["sk"], s["sv"] = ((torch.rand(kv, generator=g, device="cuda") * 0.2 + 0.9) / 80 if fp8 else None for _ in range(2))
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_attend(case, g, seed) if case["op"] == "attend" else _prepare_rope(case, g)


# -------------------------------------------------------------------------------------------------------- plain forms

def _axis_of_pair(pairs, sections, mixed):
    if sections is None:
        return [0] * pairs
    if mixed:
        n = len(sections)
        return [j % n if j < n * sections[j % n] else 0 for j in range(pairs)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


def _normed(x, weight, eps):
    x = x.float()
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.float()


def _rotated(x, s):
    """``x`` [rows, heads, dim] in 32 bits, its first ``rotated`` elements turned by the positions' angles."""
    n = s["rotated"]
    pairs = n // 2
    at = s["positions"].reshape(-1, x.shape[0])[_axis_of_pair(pairs, s["sections"], s["mixed"])].t()  # [rows, pairs]
    pair = torch.arange(pairs, device=x.device)
    c, d = s["cos_sin"][at, pair][:, None], s["cos_sin"][at, pairs + pair][:, None]
    a, b = (x[..., :pairs], x[..., pairs:n]) if s["halves"] else (x[..., 0:n:2], x[..., 1:n:2])
    a, b = a * c - b * d, b * c + a * d
    turned = torch.cat([a, b], -1) if s["halves"] else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., n:]], -1)


def _put(cache, slots, x, scale):
    """``x`` [rows, heads, dim] in 32 bits into the cache's slots."""
    if scale is not None:
        x = (x / scale[:, None]).clamp(-448, 448)
    cache.view(torch.uint8 if cache.element_size() == 1 else torch.int16).flatten(0, 1)[slots] = x.to(cache.dtype).view(
        torch.uint8 if cache.element_size() == 1 else torch.int16)


def _plain_rope(s):
    op, dtype = s["op"], s["dtype"]
    if op == "append":
        _put(s["kc"], s["slots"], _rotated(s["k"].float(), s), s["sk"])
        _put(s["vc"], s["slots"], s["v"].float(), s["sv"])
        return {"kc": s["kc"], "vc": s["vc"]}
    q, k, v = s["qkv"].unflatten(1, (-1, s["dim"])).split([s["q_heads"], s["kv_heads"], s["kv_heads"]], 1)
    q, k = _rotated(_normed(q, s["wq"], s["eps"]), s), _rotated(_normed(k, s["wk"], s["eps"]), s)
    if op == "norm_rope":
        return {"q": q.to(dtype), "k": k.to(dtype)}
    _put(s["kc"], s["slots"], k, s["sk"])
    _put(s["vc"], s["slots"], v.float(), s["sv"])
    return {"q": q.to(dtype), "kc": s["kc"], "vc": s["vc"]}


def _plain_attend(s):
    out = torch.empty_like(s["q"])
    group, page, at = s["q_heads"] // s["kv_heads"], s["page"], 0
    for b, (length, n) in enumerate(zip(s["lengths"], s["counts"])):
        pages = s["pages"][b, : -(-length // page)]
        k, v = (c[pages].flatten(0, 1)[:length].float().transpose(0, 1) for c in (s["kc"], s["vc"]))  # [kv heads, length, dim]
        if s["sk"] is not None:
            k, v = k * s["sk"][:, None, None], v * s["sv"][:, None, None]
        q = s["q"][at : at + n].float().unflatten(1, (-1, group)).permute(1, 2, 0, 3).flatten(1, 2)  # [kv heads, group * n, dim]
        seen = torch.ones(n, length, dtype=torch.bool, device=q.device)
        seen[:, length - n :] = torch.ones(n, n, dtype=torch.bool, device=q.device).tril() if s["mask"] is None else s["mask"][at : at + n, :n]
        score = (q @ k.transpose(1, 2) * s["scale"]).unflatten(1, (group, n)).masked_fill(~seen, -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = (p.flatten(1, 2) @ v).unflatten(1, (group, n)).permute(2, 0, 1, 3)
        out[at : at + n] = o.flatten(1, 2).to(out.dtype)
        at += n
    return out


# ------------------------------------------------------------------------------------------------- the framework's own

def _own(s):
    import sglang_b200 as sb

    op = s["op"]
    if op == "attend":
        return sb.tree_attention(s["q"], s["kc"], s["vc"], s["pages"], s["lens"], s["starts"], s["mask"], scale=s["scale"],
                                 k_scale=s["sk"], v_scale=s["sv"])
    rope = dict(is_neox=s["halves"], mrope_section=s["sections"], mrope_interleaved=s["mixed"])
    if op == "append":
        sb.append_paged_kv(s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["positions"], s["cos_sin"], k_scale=s["sk"],
                           v_scale=s["sv"], **rope)
        return {"kc": s["kc"], "vc": s["vc"]}
    if op == "norm_rope":
        q, k = sb.qk_norm_rope(s["qkv"], s["q_heads"], s["kv_heads"], s["positions"], s["cos_sin"], s["wq"], s["wk"], s["eps"], **rope)
        return {"q": q, "k": k}
    q = sb.qk_norm_rope_append(s["qkv"], s["q_heads"], s["kv_heads"], s["positions"], s["cos_sin"], s["kc"], s["vc"], s["slots"],
                               s["wq"], s["wk"], s["eps"], k_scale=s["sk"], v_scale=s["sv"], **rope)
    return {"q": q, "kc": s["kc"], "vc": s["vc"]}


def run(state):
    if own:
        return _own(state)
    return _plain_attend(state) if state["op"] == "attend" else _plain_rope(state)


def work(case):
    q, kv, dim = case["q_heads"], case["kv_heads"], case["dim"]
    held = 1 if case["cache"] == "fp8" else 2
    if case["op"] == "attend":
        lengths, drafted = _lengths(case), _drafted(case)
        tokens = sum(drafted)
        pages = sum(-(-n // case["page"]) for n in lengths)
        mask = sum(n * n for n in drafted) if case["tree"] and case["drafted"] > 1 else 0
        return {"bytes": sum(lengths) * kv * dim * 2 * held + tokens * q * dim * 4 + 4 * pages + 8 * case["seqs"] + mask,
                "flops": sum(4 * a * b for a, b in zip(lengths, drafted)) * q * dim}
    rows, op = case["rows"], case["op"]
    turned = kv if op == "append" else q + kv
    read = 2 * kv if op == "append" else q + kv if op == "norm_rope" else q + 2 * kv
    written = 2 * kv * held if op == "append" else 2 * (q + kv) if op == "norm_rope" else 2 * q + 2 * kv * held
    # rows in and out, angles, positions and slots
    b = rows * (dim * (2 * read + written) + 4 * case["rotated"] + 8 * case["axes"] + (0 if op == "norm_rope" else 8))
    return {"bytes": b + (4 * dim if case["norm"] else 0), "flops": rows * turned * (3 * case["rotated"] + (4 * dim if case["norm"] else 0))}


# ------------------------------------------------------------------------------------------------------ in 64 bits

def _e4m3(y):
    """Nearest value of 4 exponent and 3 mantissa bits, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def _exact_rope(case, s):
    d = torch.float64
    rows, dim, pairs = case["rows"], case["dim"], case["rotated"] // 2
    axis = []
    for j in range(pairs):
        if case["axes"] == 1:
            axis.append(0)
        elif case["mixed"]:
            a = j % case["axes"]
            axis.append(a if a and j < case["axes"] * s["sections"][a] else 0)
        else:
            axis.append(next(a for a in range(case["axes"]) if j < sum(s["sections"][: a + 1])))
    positions = s["positions"].view(case["axes"], rows)
    angles = torch.empty(rows, pairs, dtype=torch.complex128, device="cuda")
    for j, a in enumerate(axis):
        line = s["cos_sin"][positions[a]]
        angles[:, j] = torch.complex(line[:, j].to(d), line[:, pairs + j].to(d))

    def turn(x, weight):
        x = x.to(d)
        if weight is not None:
            x = x / ((x * x).sum(-1, keepdim=True) / dim + EPS).sqrt() * weight.to(d)
        out = x.clone()
        first, second = (slice(0, pairs), slice(pairs, 2 * pairs)) if case["halves"] else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * angles[:, None]
        out[..., first], out[..., second] = z.real, z.imag
        return out

    def held(cache, x, scale):
        out = cache.to(d).flatten(0, 1).clone()
        out[s["slots"]] = x if scale is None else _e4m3(x / scale.to(d).view(1, -1, 1))
        return out.view(cache.shape)

    if case["op"] == "append":
        return {"kc": held(s["kc"], turn(s["k"], None), s["sk"]), "vc": held(s["vc"], s["v"].to(d), s["sv"])}
    q, kv = case["q_heads"] * dim, case["kv_heads"] * dim
    heads = [s["qkv"][:, a:b].reshape(rows, -1, dim) for a, b in ((0, q), (q, q + kv), (q + kv, q + 2 * kv))]
    out = {"q": turn(heads[0], s["wq"])}
    k = turn(heads[1], s["wk"])
    if case["op"] == "norm_rope":
        return {**out, "k": k}
    return {**out, "kc": held(s["kc"], k, s["sk"]), "vc": held(s["vc"], heads[2].to(d), s["sv"])}


def _exact_attend(case, s):
    d = torch.float64
    out = torch.zeros(s["q"].shape, dtype=d, device="cuda")
    group = case["q_heads"] // case["kv_heads"]
    at = 0
    for b, (length, n) in enumerate(zip(s["lengths"], s["counts"])):
        where = torch.arange(length, device="cuda")
        where = s["pages"][b].long()[where // case["page"]], where % case["page"]
        hidden = torch.zeros(n, length, dtype=torch.bool, device="cuda")
        for i in range(n):
            for_i = torch.arange(n, device="cuda") > i if s["mask"] is None else ~s["mask"][at + i, :n]
            hidden[i, length - n :] = for_i
        for h in range(case["kv_heads"]):
            k, v = s["kc"][where[0], where[1], h].to(d), s["vc"][where[0], where[1], h].to(d)
            if s["sk"] is not None:
                k, v = k * s["sk"][h].to(d), v * s["sv"][h].to(d)
            for g in range(group):
                score = torch.matmul(s["q"][at : at + n, h * group + g].to(d), k.t()) / math.sqrt(case["dim"])
                out[at : at + n, h * group + g] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
        at += n
    return out


def exact(case, seed):
    """The same outputs by the definitions in 64 bits: rotations as products of complex numbers, attention query head by query
    head with every key by its own slot."""
    s = prepare(case, seed)
    return _exact_attend(case, s) if case["op"] == "attend" else _exact_rope(case, s)
