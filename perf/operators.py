"""Performance cases of the W8A8 operators around the linear layers: what an inference server has them do.

``norm_fp8``    RMSNorm of the hidden states, with the residual's addition, into FP8 rows and their block scales: the input
                of a block-FP8 linear.
``norm_int8``   the same into 8-bit integers with one scale per token.
``quant_int8``  one scale per token for activations that no norm precedes, optionally with SiLU and the product in front.
``mm``          product of 8-bit integers with scales per token and per output channel.
``linear``      quantiser and product: one int8 linear layer on 16-bit activations.
``mlp``         all of them as a decoder layer's MLP runs them: norm, gate and up projection, SiLU and product, down
                projection; 16-bit tensors in between.

Widths are the benchmark configurations of this repository (``sglang_b200.synthetic``), their tensor-parallel shards and
generic ones; row counts run from one decoded token to a full prefill chunk.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6  # of the norm
# hidden size, rows of qkv, intermediate size
DENSE = {"llama3_8b": (4096, 6144, 14336), "llama3_70b": (8192, 10240, 28672)}
HIDDEN = (4096, 7168, 8192)
MAX_FLOPS = 2.0 * 8192 * 28672 * 4096


def _norm_fp8(name, rows, hidden, residual, scales="col", dtype="bf16"):
    return {"name": name, "op": "norm_fp8", "rows": rows, "hidden": hidden, "residual": residual, "scales": scales, "dtype": dtype}


def _norm_int8(name, rows, hidden, residual, dtype="bf16"):
    return {"name": name, "op": "norm_int8", "rows": rows, "hidden": hidden, "residual": residual, "dtype": dtype}


def _quant(name, rows, width, silu, dtype="bf16"):
    return {"name": name, "op": "quant_int8", "rows": rows, "width": width, "silu": silu, "dtype": dtype}


def _mm(name, rows, n, k, bias=False, dtype="bf16", op="mm"):
    return {"name": name, "op": op, "rows": rows, "n": n, "k": k, "bias": bias, "dtype": dtype}


def _mlp(name, model, tp, rows, dtype="bf16"):
    return {"name": name, "op": "mlp", "model": model, "tp": tp, "rows": rows, "dtype": dtype}


def listed():
    return [
        # one user decoding: a single row, where the launch and the host's time count
        _norm_fp8("norm_fp8_decode_1", 1, 8192, True),
        # a ragged prefill chunk of an expert model, whose scales are powers of two, packed as exponent bytes
        _norm_fp8("norm_fp8_ue8m0_3001", 3001, 7168, True, "ue8m0"),
        # the largest prefill chunk
        _norm_fp8("norm_fp8_prefill_16384", 16384, 8192, True),
        # the first norm of a model, which has no residual yet, on a short prompt, fp16 model
        _norm_int8("norm_int8_203_fp16", 203, 4096, False, "fp16"),
        # a decode batch in front of the down projection
        _quant("quant_int8_decode_16", 16, 14336, False),
        # the same for a prefill chunk: whole rows of the intermediate size
        _quant("quant_int8_prefill_8192", 8192, 14336, False),
        # a larger decode batch on one rank of four (gate and up projection), fp16 model
        _mm("mm_decode_61_tp4_fp16", 61, 14336, 8192, dtype="fp16"),
        # a short prompt, or a decode batch mixed with a piece of one; a layer with a bias
        _mm("mm_mixed_203_bias", 203, 4096, 14336, bias=True),
        # the largest prefill chunk through the widest projection
        _mm("mm_prefill_8192", 8192, 28672, 4096),
        # one user decoding through one linear layer
        _mm("linear_decode_1", 1, 6144, 4096, op="linear"),
        # one user decoding through an MLP: four launches in a chain
        _mlp("mlp_decode_1", "llama3_8b", 1, 1),
        # an ordinary prefill chunk through the MLP of one rank of eight, ragged as prompts are
        _mlp("mlp_prefill_1027_tp8", "llama3_70b", 8, 1027),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, step, lo, hi):
    return max(step, _log_int(rng, lo, hi) // step * step)


def draw(rng):
    op = rng.choice(["norm_fp8", "norm_fp8", "norm_int8", "quant_int8", "mm", "mm", "mm", "linear", "mlp"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("norm_fp8", "norm_int8"):
        hidden = rng.choice(HIDDEN) if rng.random() < 0.5 else _width(rng, 128, 512, 16384)
        rows = min(_log_int(rng, 1, 16384), 16384 * 8192 // hidden)
        residual = rng.random() < 0.7
        c = (_norm_fp8("", rows, hidden, residual, rng.choice(["row", "col", "ue8m0"]), dtype) if op == "norm_fp8"
             else _norm_int8("", rows, hidden, residual, dtype))
    elif op == "quant_int8":
        width = _width(rng, rng.choice([128, 16, 1]), 256, 28672)
        c = _quant("", min(_log_int(rng, 1, 16384), 16384 * 8192 // width // 2), width, rng.random() < 0.4, dtype)
    elif op == "mlp":
        model, tp = rng.choice(sorted(DENSE)), rng.choice([1, 2, 4, 8])
        h, _, i = DENSE[model]
        c = _mlp("", model, tp, min(_log_int(rng, 1, 8192), int(MAX_FLOPS / (6 * h * i / tp))), dtype)
    else:
        if rng.random() < 0.5:
            h, qkv, i = DENSE[rng.choice(sorted(DENSE))]
            tp = rng.choice([1, 2, 4, 8])
            n, k = rng.choice([(qkv // tp, h), (h, h // tp), (2 * i // tp, h), (h, i // tp)])
        else:
            n, k = _width(rng, 8, 256, 28672), _width(rng, 16, 256, 16384)
        c = _mm("", min(_log_int(rng, 1, 8192), int(MAX_FLOPS / (2 * n * k))), n, k, rng.random() < 0.3, dtype, op)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------------------ inputs

def _activation(g, rows, width, dtype):
    """N(0, 1) with one channel in a hundred twenty times as large."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    x[:, torch.randperm(width, generator=g, device="cuda")[: max(1, width // 100)]] *= 20
    return x.to(dtype)


def _int8(g, rows, width):
    """Rows as a quantiser leaves normal values: a standard deviation of 32 steps."""
    return torch.randn(rows, width, generator=g, device="cuda").mul_(32).round_().clamp_(-127, 127).to(torch.int8)


def _scales(g, rows, size):
    return torch.rand(rows, 1, generator=g, device="cuda").mul_(size).add_(0.5 * size)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op, rows = DTYPES[case["dtype"]], case["op"], case["rows"]
    s = dict(case, dtype=dtype)
    if op in ("norm_fp8", "norm_int8", "mlp"):
        hidden = DENSE[case["model"]][0] if op == "mlp" else case["hidden"]
        s["x"] = _activation(g, rows, hidden, dtype)
        s["weight"] = torch.randn(hidden, generator=g, device="cuda").mul_(0.1).add_(1).to(dtype)
        s["res"] = _activation(g, rows, hidden, dtype) if op == "mlp" or case["residual"] else None
    if op == "mlp":
        inter = DENSE[case["model"]][2] // case["tp"]
        s["w1"], s["s1"] = _int8(g, 2 * inter, hidden), _scales(g, 2 * inter, 6e-4)
        s["w2"], s["s2"] = _int8(g, hidden, inter), _scales(g, hidden, 6e-4)
    elif op == "quant_int8":
        s["x"] = _activation(g, rows, case["width"] * (2 if case["silu"] else 1), dtype)
    elif op in ("mm", "linear"):
        n, k = case["n"], case["k"]
        if op == "mm":
            s["a"], s["sa"] = _int8(g, rows, k), _scales(g, rows, 0.03)
        else:
            s["x"] = _activation(g, rows, k, dtype)
        s["w"], s["sw"] = _int8(g, n, k), _scales(g, n, 6e-4)
        s["b"] = torch.randn(n, generator=g, device="cuda").to(dtype) if case["bias"] else None
    return s


# -------------------------------------------------------------------------------------------------------- plain forms

def _norm(x, res, weight, f):
    """Unrounded RMSNorm of ``x + res`` and that sum, in type ``f``."""
    h = x.to(f) if res is None else x.to(f) + res.to(f)
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * weight.to(f), h


def _over(v, top):
    return v / torch.full((), top, dtype=v.dtype, device=v.device)


def _int8_rows(y):
    s = _over(y.abs().amax(-1, keepdim=True).clamp_min(1e-10), 127.0)
    return (y / s).round().clamp(-127, 127), s


def _fp8_rows(y, ue8m0):
    v = y.unflatten(-1, (-1, 128))
    s = _over(v.abs().amax(-1, keepdim=True).clamp_min(1e-10), 448.0)
    if ue8m0:
        s = torch.exp2(torch.ceil(torch.log2(s)))
    return (v / s).clamp(-448, 448).flatten(-2).to(torch.float8_e4m3fn), s.squeeze(-1)


def _silu_mul(x, f):
    gate, up = x.to(f).chunk(2, -1)
    return gate / (1 + torch.exp(-gate)) * up


def _product(q, s, w, sw, bias, dtype, f):
    c = (q.to(f) @ w.to(f).t()) * s.to(f) * sw.to(f).t()
    return (c if bias is None else c + bias.to(f)).to(dtype)


def _formula(s, f, dtype):
    """One pass from the definitions, in type ``f``; 16-bit results become ``dtype``. The scales of ``ue8m0`` are held in 8
    bits: what they stand for is in the rows' values."""
    op = s["op"]
    if op == "norm_fp8":
        y, h = _norm(s["x"], s["res"], s["weight"], f)
        q, sc = _fp8_rows(y, s["scales"] == "ue8m0")
        out = {"q": q} if s["scales"] == "ue8m0" else {"q": q, "s": sc}
        return out if s["res"] is None else {**out, "res": h.to(dtype)}
    if op == "norm_int8":
        y, h = _norm(s["x"], s["res"], s["weight"], f)
        q, sc = _int8_rows(y)
        out = {"y": (q * sc).to(dtype), "s": sc}
        return out if s["res"] is None else {**out, "res": h.to(dtype)}
    if op == "quant_int8":
        if s["silu"]:
            q, sc = _int8_rows(_silu_mul(s["x"], f))
            return {"y": (q * sc).to(dtype), "s": sc}
        q, sc = _int8_rows(s["x"].to(f))
        return {"q": q.to(torch.int8), "s": sc}
    if op == "mm":
        return _product(s["a"], s["sa"], s["w"], s["sw"], s["b"], dtype, f)
    if op == "linear":
        return _product(*_int8_rows(s["x"].to(f)), s["w"], s["sw"], s["b"], dtype, f)
    # 16-bit tensors between the operators
    y, h = _norm(s["x"], s["res"], s["weight"], f)
    mid = _product(*_int8_rows(y), s["w1"], s["s1"], None, s["dtype"], f)
    return {"out": _product(*_int8_rows(_silu_mul(mid, f)), s["w2"], s["s2"], None, dtype, f), "res": h.to(dtype)}


# ------------------------------------------------------------------------------------------------- the framework's own

def _values(q, s, dtype):
    return torch.mul(q, s, out=torch.empty(q.shape, dtype=dtype, device=q.device))


def _own(s):
    import sglang_b200 as sb

    op, dtype = s["op"], s["dtype"]
    if op == "norm_fp8":
        ue8m0 = s["scales"] == "ue8m0"
        q, sc, *res = sb.rmsnorm_quant_fp8(s["x"], s["weight"], 128, EPS, residual=s["res"], column_major_scales=s["scales"] != "row",
                                           scale_tma_aligned=ue8m0, scale_ue8m0=ue8m0)
        out = {"q": q} if ue8m0 else {"q": q, "s": sc}
        return {**out, "res": res[0]} if res else out
    if op == "norm_int8":
        q, sc, *res = sb.rmsnorm_quant_int8(s["x"], s["weight"], EPS, residual=s["res"])
        out = {"y": _values(q, sc, dtype), "s": sc}
        return {**out, "res": res[0]} if res else out
    if op == "quant_int8":
        q, sc = sb.per_token_quant_int8(s["x"], fuse_silu_and_mul=s["silu"])
        return {"y": _values(q, sc, dtype), "s": sc} if s["silu"] else {"q": q, "s": sc}
    if op == "mm":
        return sb.int8_scaled_mm(s["a"], s["w"].t(), s["sa"], s["sw"], dtype, s["b"])
    if op == "linear":
        return sb.w8a8_int8_linear(s["x"], s["w"], s["sw"], s["b"])
    q, sc, res = sb.rmsnorm_quant_int8(s["x"], s["weight"], EPS, residual=s["res"])
    mid = sb.int8_scaled_mm(q, s["w1"].t(), sc, s["s1"], dtype)
    q, sc = sb.per_token_quant_int8(mid, fuse_silu_and_mul=True)
    return {"out": sb.int8_scaled_mm(q, s["w2"].t(), sc, s["s2"], dtype), "res": res}


def run(state):
    if own:
        return _own(state)
    return _formula(state, torch.float32, state["dtype"])


def work(case):
    rows, op = case["rows"], case["op"]

    def norm(hidden, residual, scale_bytes):
        n = rows * hidden
        return n * (2 + 1 + (4 if residual else 0)) + 2 * hidden + rows * scale_bytes, n * 6

    def mm(n, k, bias=False):
        return rows * k + n * k + 2 * rows * n + 4 * (rows + n) + (2 * n if bias else 0), 2 * rows * n * k

    if op == "norm_fp8":
        b, f = norm(case["hidden"], case["residual"], case["hidden"] // 128 * (1 if case["scales"] == "ue8m0" else 4))
    elif op == "norm_int8":
        b, f = norm(case["hidden"], case["residual"], 4)
    elif op == "quant_int8":
        n = rows * case["width"]
        b, f = n * (5 if case["silu"] else 3) + 4 * rows, n * (8 if case["silu"] else 3)
    elif op == "mm":
        b, f = mm(case["n"], case["k"], case["bias"])
    elif op == "linear":
        b, f = mm(case["n"], case["k"], case["bias"])
        b += rows * case["k"]  # 16-bit rows in
    else:
        h, _, i = DENSE[case["model"]]
        i //= case["tp"]
        # the weights, the rows and the residual in, the result and the residual out
        b, f = 3 * h * i + 4 * (2 * i + h) + rows * h * 8 + 2 * h, rows * 6 * h * i
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    """The same outputs by the definitions in 64 bits, row by row: norm with a plain sum of squares, scales from the largest
    magnitude, codes as the nearest of the type's values, products of whole numbers."""
    s, d = prepare(case, seed), torch.float64
    op = case["op"]

    def normed():
        h = s["x"].to(d) if s["res"] is None else s["x"].to(d) + s["res"].to(d)
        return h / ((h * h).sum(-1, keepdim=True) / h.shape[-1] + EPS).sqrt() * s["weight"].to(d), h

    def whole(y):
        step = y.abs().amax(-1, keepdim=True).clamp(min=1e-10) / 127
        return torch.round(y / step).clamp(-127, 127), step

    def silu(x):
        gate, up = x[:, : x.shape[1] // 2].to(d), x[:, x.shape[1] // 2 :].to(d)
        return gate * torch.sigmoid(gate) * up

    def e4m3(y, top):
        """Nearest value of 4 exponent and 3 mantissa bits, ties to even."""
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
        return (torch.round(y / step) * step).clamp(-top, top)

    def rows_of(q, step, w, sw, bias):
        out = torch.matmul(q, w.to(d).transpose(0, 1)) * step * sw.to(d).view(1, -1)
        return out if bias is None else out + bias.to(d)

    if op == "norm_fp8":
        y, h = normed()
        y = y.view(y.shape[0], -1, 128)
        step = y.abs().amax(-1, keepdim=True).clamp(min=1e-10) / 448
        if case["scales"] == "ue8m0":
            step = 2.0 ** torch.ceil(torch.log2(step))
        out = {"q": e4m3(y / step, 448.0).reshape(h.shape)}
        if case["scales"] != "ue8m0":
            out["s"] = step.squeeze(-1)
        return {**out, "res": h} if s["res"] is not None else out
    if op == "norm_int8":
        y, h = normed()
        q, step = whole(y)
        return {"y": q * step, "s": step, **({"res": h} if s["res"] is not None else {})}
    if op == "quant_int8":
        if case["silu"]:
            q, step = whole(silu(s["x"]))
            return {"y": q * step, "s": step}
        return {"q": None, "s": whole(s["x"].to(d))[1]}
    if op == "mm":
        return rows_of(s["a"].to(d), s["sa"].to(d), s["w"], s["sw"], s["b"])
    if op == "linear":
        return rows_of(*whole(s["x"].to(d)), s["w"], s["sw"], s["b"])
    y, h = normed()
    mid = rows_of(*whole(y), s["w1"], s["s1"], None).to(s["dtype"])  # a 16-bit tensor between two operators
    return {"out": rows_of(*whole(silu(mid)), s["w2"], s["s2"], None), "res": h}
