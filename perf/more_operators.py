"""Cases of the dense steps around a served block: norms, 8-bit rows, projections and the draw of a token.

Four operators:

* ``norm``      the residual's addition and the root-mean-square norm of its
                rows, written in the input's type, in 8 bits with a scale a
                row, or both;
* ``quantize``  rows to 8 bits with a scale each (an attention's output on its
                way into an 8-bit product, a weight when it is laid out);
* ``linear``    ``act(x W^T + bias) + residual`` of bfloat16 rows and weights,
                or of 8-bit ones with a scale a row;
* ``sample``    one token a row of logits by temperature, top-k, top-p and
                min-p, from a given uniform number a row.

Codes are compared as the values that they stand for, so the 8-bit cases read
their codes back (``dequantize_rows``) within the pass.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TINY = 2.0 ** -100  # least magnitude a row's scale is made for
KINDS = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # the norm before a layer of one decoded token: latency
        {"name": "norm 1 x 2048", "op": "norm", "rows": 1, "dim": 2048, "type": "bf16", "weight": "bf16",
         "residual": "bf16", "offset": False, "kind": "none", "keep": True, "pad": 0},
        # the 5,000-token prefill chunk: bfloat16 rows for the router and 8-bit rows for a projection from one pass
        {"name": "norm 5000 x 2048 int8", "op": "norm", "rows": 5000, "dim": 2048, "type": "bf16", "weight": "bf16",
         "residual": "bf16", "offset": True, "kind": "int8", "keep": True, "pad": 0},
        # attention outputs (16 heads of 256) of the 64-token batch before an 8-bit output projection
        {"name": "quantize 64 x 4096 e4m3", "op": "quantize", "rows": 64, "dim": 4096, "type": "bf16", "kind": "e4m3",
         "pad": 0},
        # a float32 weight of odd sizes laid out in 8 bits
        {"name": "quantize 5003 x 2561 int8", "op": "quantize", "rows": 5003, "dim": 2561, "type": "f32", "kind": "int8",
         "pad": 0},
        # the fused query, key and value projection of one decoded token (16 + 2 x 2 heads of 256)
        {"name": "linear 1 x 2048 > 5120", "op": "linear", "m": 1, "k": 2048, "n": 5120, "kind": "bf16", "bias": "bf16",
         "act": "none", "residual": "none", "out": "bf16", "pad": 0},
        # the attention's output projection in 8 bits for the 64-token batch, added to a float32 residual
        {"name": "linear 64 x 4096 > 2048 int8", "op": "linear", "m": 64, "k": 4096, "n": 2048, "kind": "int8",
         "bias": "none", "act": "none", "residual": "f32", "out": "f32", "pad": 0},
        # the head of a 16-sequence decode step: float32 logits over a large vocabulary
        {"name": "linear 16 x 2048 > 131072", "op": "linear", "m": 16, "k": 2048, "n": 131072, "kind": "bf16",
         "bias": "none", "act": "none", "residual": "none", "out": "f32", "pad": 0},
        # a ragged chunk through an odd 8-bit layer, input rows cut from wider ones
        {"name": "linear 1237 x 2576 > 5003 e4m3", "op": "linear", "m": 1237, "k": 2576, "n": 5003, "kind": "e4m3",
         "bias": "f32", "act": "gelu", "residual": "bf16", "out": "bf16", "pad": 48},
        # the 5,000-token prefill chunk through a bfloat16 layer
        {"name": "linear 5000 x 2048 > 5120", "op": "linear", "m": 5000, "k": 2048, "n": 5120, "kind": "bf16",
         "bias": "bf16", "act": "silu", "residual": "none", "out": "bf16", "pad": 0},
        # one user's next token, with the usual filters: latency
        {"name": "sample 1 x 131072", "op": "sample", "rows": 1, "vocab": 131072, "type": "f32", "form": "usual",
         "masked": 0.0, "pad": 0},
        # the 64-token batch, every request with settings of its own
        {"name": "sample 64 x 131072 mixed", "op": "sample", "rows": 64, "vocab": 131072, "type": "f32", "form": "mixed",
         "masked": 0.0, "pad": 0},
        # many rows of bfloat16 logits over an odd vocabulary, part of it masked by a grammar
        {"name": "sample 300 x 32003 bf16", "op": "sample", "rows": 300, "vocab": 32003, "type": "bf16", "form": "top_p",
         "masked": 0.3, "pad": 61},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "linear", "sample", "sample"])
    c = {"op": op}
    if op in ("norm", "quantize"):
        dim = _log(rng, 16, 16384)
        c.update(rows=_log(rng, 1, max(1, 10_000_000 // dim)), dim=dim, type=rng.choice(["bf16", "f32"]),
                 pad=rng.choice([0, 0, 8, rng.randint(1, 100)]), kind=rng.choice(["int8", "e4m3"]))
        if op == "norm":
            kind = rng.choice(["none", c["kind"]])
            c.update(weight=rng.choice(["bf16", "f32"]), residual=rng.choice(["none", "bf16", "f32"]),
                     offset=rng.random() < 0.3, kind=kind, keep=kind == "none" or rng.random() < 0.5)
        return c
    if op == "linear":
        kind = rng.choice(["bf16", "bf16", "int8", "e4m3"])
        step = 8 if kind == "bf16" else 16
        m = rng.choice([_log(rng, 1, 64), _log(rng, 1, 5000)])
        k = step * max(1, _log(rng, 64, 8192) // step)
        n = _log(rng, 16, min(131072, 5000 * 2048 * 5120 // (m * k), 2 ** 28 // k, 2 ** 25 // m))
        out = rng.choice(["bf16", "f32"])
        return dict(c, m=m, k=k, n=n, kind=kind, bias=rng.choice(["none", "bf16", "f32"]),
                    act=rng.choice(["none", "silu", "gelu", "relu"]), residual=rng.choice(["none", "bf16", "f32"]),
                    out=out, pad=step * rng.choice([0, 0, rng.randint(1, 20)]))
    vocab = _log(rng, 16, 131072)
    return dict(c, rows=_log(rng, 1, min(512, 64 * 131072 // vocab)), vocab=vocab, type=rng.choice(["bf16", "f32"]),
                form=rng.choice(["temperature", "usual", "top_p", "top_k", "mixed", "mixed"]),
                masked=rng.choice([0.0, 0.0, rng.uniform(0.05, 0.95)]), pad=rng.choice([0, 0, rng.randint(1, 100)]))


# ---- inputs ----


def _slice(x, pad):
    """``x`` as the first columns of rows that are ``pad`` wider."""
    if not pad:
        return x
    wide = x.new_zeros((x.shape[0], x.shape[1] + pad)) if x.element_size() > 1 else \
        torch.zeros((x.shape[0], x.shape[1] + pad), dtype=torch.uint8, device=x.device).view(x.dtype)
    wide[:, : x.shape[1]] = x
    return wide[:, : x.shape[1]]


def _codes(x, kind):
    """Codes and scales of x's rows, as a program has them in hand."""
    dtype, top = KINDS[kind]
    scale = x.abs().amax(1).clamp_min(TINY) / top
    y = (x / scale[:, None]).clamp(-top, top)
    return (y.round() if kind == "int8" else y).to(dtype), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    op = case["op"]
    s = {"op": op}
    if op in ("norm", "quantize"):
        rows, dim = case["rows"], case["dim"]
        # hidden states: rows of different sizes, a few channels far above the others
        gain = torch.exp(0.5 * randn(dim))
        gain[torch.randint(dim, (max(1, dim // 256),), device="cuda", generator=g)] *= 12.0
        x = randn(rows, dim) * gain * torch.exp(0.3 * randn(rows, 1))
        s["kind"] = case["kind"]
        s["x"] = _slice(x.to(TYPES[case["type"]]), case["pad"])
        if op == "norm":
            s.update(offset=case["offset"], keep=case["keep"], residual=None)
            s["weight"] = ((0.0 if case["offset"] else 1.0) + 0.2 * randn(dim)).to(TYPES[case["weight"]])
            if case["residual"] != "none":
                s["residual"] = (randn(rows, dim) * 3.0 * gain).to(TYPES[case["residual"]])
        return s
    if op == "linear":
        m, k, n, kind = case["m"], case["k"], case["n"], case["kind"]
        x = randn(m, k) * torch.exp(0.5 * randn(k))
        w = randn(n, k) * (k ** -0.5) * torch.exp(0.2 * randn(n, 1))
        s.update(kind=kind, act=case["act"], out=case["out"], x_scale=None, weight_scale=None, bias=None, residual=None)
        if kind == "bf16":
            x, s["weight"] = x.bfloat16(), w.bfloat16()
        else:
            x, s["x_scale"] = _codes(x, kind)
            s["weight"], s["weight_scale"] = _codes(w, kind)
        del w
        s["x"] = _slice(x, case["pad"])
        if case["bias"] != "none":
            s["bias"] = (0.5 * randn(n)).to(TYPES[case["bias"]])
        if case["residual"] != "none":
            s["residual"] = randn(m, n).to(TYPES[case["residual"]])
        return s
    rows, vocab = case["rows"], case["vocab"]
    x = 2.5 * randn(rows, vocab)
    # a few likely continuations stand out
    few = torch.randint(vocab, (rows, min(12, vocab)), device="cuda", generator=g)
    x.scatter_add_(1, few, 9.0 * torch.rand(few.shape, device="cuda", generator=g))
    if case["masked"]:
        off = torch.rand(rows, vocab, device="cuda", generator=g) < case["masked"]
        off.scatter_(1, few, False)
        x.masked_fill_(off, -math.inf)
    s["logits"] = _slice(x.to(TYPES[case["type"]]), case["pad"])
    s["u"] = torch.rand(rows, device="cuda", generator=g)
    form = case["form"]
    if form == "mixed":
        i = torch.arange(rows, device="cuda")
        s["temperature"] = torch.where(i % 5 == 4, 0.0, 0.4 + torch.rand(rows, device="cuda", generator=g))
        s["top_k"] = torch.where(i % 3 == 0, 0, torch.randint(1, 200, (rows,), device="cuda", generator=g)).to(torch.int32)
        s["top_p"] = torch.where(i % 4 == 0, 1.0, 0.5 + 0.5 * torch.rand(rows, device="cuda", generator=g))
        s["min_p"] = torch.where(i % 2 == 0, 0.0, 0.2 * torch.rand(rows, device="cuda", generator=g))
    else:
        s["temperature"] = 0.8
        s["top_k"] = {"usual": 50, "top_k": 20}.get(form, 0)
        s["top_p"] = {"usual": 0.95, "top_p": 0.9}.get(form, 1.0)
        s["min_p"] = 0.02 if form == "usual" else 0.0
    return s


# ---- the plain forms ----


def _plain_rows(y, kind):
    """The values that y's 8-bit codes stand for."""
    codes, scale = _codes(y, kind)
    return (codes.float() * scale[:, None]).bfloat16()


def _plain_norm(s):
    x = s["x"].float()
    got = {}
    if s["residual"] is not None:
        x = x + s["residual"].float()
        got["residual"] = x.to(s["residual"].dtype)
    w = s["weight"].float() + (1.0 if s["offset"] else 0.0)
    y = x * (1.0 / (x.square().mean(1, keepdim=True) + EPS).sqrt()) * w
    if s["keep"]:
        got["y"] = y.to(s["x"].dtype)
    if s["kind"] != "none":
        got["values"] = _plain_rows(y, s["kind"])
    return got


def _plain_linear(s):
    y = s["x"].float() @ s["weight"].float().T
    if s["x_scale"] is not None:
        y *= s["x_scale"][:, None]
        y *= s["weight_scale"]
    if s["bias"] is not None:
        y += s["bias"].float()
    act = s["act"]
    if act == "silu":
        y = y / (1.0 + (-y).exp())
    elif act == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * 0.5 ** 0.5))
    elif act == "relu":
        y = torch.where(y > 0, y, 0.0)
    if s["residual"] is not None:
        y += s["residual"].float()
    return y.to(TYPES[s["out"]])


def _plain_sample(s):
    z = s["logits"].double()
    rows, vocab = z.shape
    dev = z.device

    def column(v, dtype):
        return v.to(dtype)[:, None] if isinstance(v, torch.Tensor) else torch.full((rows, 1), v, dtype=dtype, device=dev)

    t, p, least = (column(s[k], torch.float32).double() for k in ("temperature", "top_p", "min_p"))
    k = column(s["top_k"], torch.int64)
    z, order = z.sort(dim=1, descending=True, stable=True)
    x = (z - z[:, :1]) / torch.where(t > 0, t, 1.0)
    w = x.exp()
    at = torch.arange(vocab, device=dev)
    w = torch.where((k <= 0) | (at < k), w, 0.0)
    before = w.cumsum(1) - w
    w = torch.where((p >= 1.0) | (before < p * w.sum(1, keepdim=True)) | (at == 0), w, 0.0)
    w = torch.where((w >= least) & ((t > 0) | (at == 0)), w, 0.0)
    total = w.sum(1, keepdim=True)
    cdf = torch.zeros_like(w).scatter_(1, order, w).cumsum(1)
    token = torch.searchsorted(cdf, s["u"].double()[:, None] * total, right=True).clamp_max(vocab - 1)
    place = (order == token).to(torch.int8).argmax(1, keepdim=True)
    return {"token": token[:, 0], "logprob": (x.gather(1, place) - total.log())[:, 0].float()}


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "macqwen-releases_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from flashnext_b200 import dense, sampling

    return dense, sampling


def run(s):
    op = s["op"]
    if not own:
        if op == "quantize":
            return _plain_rows(s["x"].float(), s["kind"])
        return {"norm": _plain_norm, "linear": _plain_linear, "sample": _plain_sample}[op](s)
    dense, sampling = _framework()
    if op == "sample":
        token, logprob = sampling.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        return {"token": token, "logprob": logprob}
    if op == "linear":
        return dense.linear(s["x"], s["weight"], s["bias"], activation=None if s["act"] == "none" else s["act"],
                            residual=s["residual"], x_scale=s["x_scale"], weight_scale=s["weight_scale"],
                            out_dtype=TYPES[s["out"]])
    if op == "quantize":
        return dense.dequantize_rows(*dense.quantize_rows(s["x"], KINDS[s["kind"]][0]))
    kind = s["kind"]
    r = dense.add_rms_norm(s["x"], s["weight"], s["residual"], EPS, unit_offset=s["offset"],
                           codes=None if kind == "none" else KINDS[kind][0], keep=s["keep"])
    got = {}
    if r.residual is not None:
        got["residual"] = r.residual
    if r.y is not None:
        got["y"] = r.y
    if r.codes is not None:
        got["values"] = dense.dequantize_rows(r.codes, r.scales)
    return got


def work(case):
    op = case["op"]
    size = {"bf16": 2, "f32": 4, "none": 0, "int8": 1, "e4m3": 1}
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size[case["type"]] + case["rows"] * 32, "flops": 4 * n}
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        b = (m + n) * k * size[case["kind"]] + m * n * (size[case["out"]] + size[case["residual"]]) + n * size[case["bias"]]
        return {"bytes": b + (0 if case["kind"] == "bf16" else 4 * (m + n)), "flops": 2 * m * k * n}
    n = case["rows"] * case["dim"]
    read_back = 0 if case["kind"] == "none" else n * (1 + 1 + 2) + 8 * case["rows"]  # codes out, in, their values out
    if op == "quantize":
        return {"bytes": n * size[case["type"]] + read_back, "flops": 4 * n}
    per = size[case["type"]] * (2 if case["keep"] else 1) + 2 * size[case["residual"]]
    return {"bytes": n * per + read_back + case["dim"] * size[case["weight"]], "flops": 8 * n}


# ---- 64 bits ----


def _nearest(y, kind):
    """The nearest code's value, ties to even, of each element of a float64 tensor."""
    top = KINDS[kind][1]
    if kind == "int8":
        return torch.round(y).clamp(-top, top)
    mantissa, exponent = torch.frexp(y.abs())
    step = torch.ldexp(torch.ones_like(y), exponent.clamp_min(-5) - 4)  # 2^-9 below the normal range
    return torch.copysign((torch.round(y.abs() / step) * step).clamp_max(top), y)


def _exact_rows(y, kind):
    scale = y.abs().max(1, keepdim=True).values.clamp_min(TINY) / KINDS[kind][1]
    return _nearest(y / scale, kind) * scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_rows(s["x"].double(), case["kind"])
    if op == "norm":
        v = s["x"].double()
        got = {}
        if s["residual"] is not None:
            got["residual"] = v = v + s["residual"].double()
        length = torch.linalg.vector_norm(v, dim=1, keepdim=True)
        gain = s["weight"].double()
        y = v / torch.sqrt(length ** 2 / v.shape[1] + EPS) * (gain + 1.0 if s["offset"] else gain)
        if s["keep"]:
            got["y"] = y
        if case["kind"] != "none":
            got["values"] = _exact_rows(y, case["kind"])
        return got
    if op == "linear":
        m, n = case["m"], case["n"]
        out = torch.empty(m, n, dtype=torch.float64, device="cuda")
        x = s["x"].to(torch.float32).double()
        if s["x_scale"] is not None:
            x = x * s["x_scale"].double()[:, None]
        step = max(1, (1 << 27) // case["k"])
        for at in range(0, n, step):
            w = s["weight"][at:at + step].to(torch.float32).double()
            if s["weight_scale"] is not None:
                w = w * s["weight_scale"][at:at + step].double()[:, None]
            y = torch.einsum("mk,nk->mn", x, w)
            if s["bias"] is not None:
                y = y + s["bias"][at:at + step].double()
            if case["act"] == "silu":
                y = y * torch.sigmoid(y)
            elif case["act"] == "gelu":
                y = y * torch.special.ndtr(y)
            elif case["act"] == "relu":
                y = y.clamp_min(0.0)
            if s["residual"] is not None:
                y = y + s["residual"][:, at:at + step].double()
            out[:, at:at + step] = y
        return out
    logits = s["logits"].double().cpu().numpy()
    u = s["u"].cpu().numpy().astype(np.float64)
    rows, vocab = logits.shape

    def setting(name, i):
        v = s[name]
        return v[i].item() if isinstance(v, torch.Tensor) else (v if name == "top_k" else float(np.float32(v)))

    tokens, logprobs = np.zeros(rows, dtype=np.int64), np.zeros(rows)
    for i in range(rows):
        z, t, k = logits[i], setting("temperature", i), setting("top_k", i)
        best = int(np.argmax(z))
        if t <= 0:
            tokens[i] = best
            continue
        weight = np.exp((z - z[best]) / t)
        ranked = np.lexsort((np.arange(vocab), -z))
        if 0 < k < vocab:
            ranked = ranked[:k]
        p = setting("top_p", i)
        if p < 1.0:
            mass = np.cumsum(weight[ranked])
            ranked = ranked[: max(1, int(np.searchsorted(mass[:-1], p * mass[-1], side="left")) + 1)]
        chosen = np.sort(ranked)
        chosen = chosen[weight[chosen] >= setting("min_p", i)]
        mass = np.cumsum(weight[chosen])
        tokens[i] = chosen[min(int(np.searchsorted(mass, u[i] * mass[-1], side="right")), len(chosen) - 1)]
        logprobs[i] = (z[tokens[i]] - z[best]) / t - math.log(mass[-1])
    return {"token": torch.from_numpy(tokens), "logprob": torch.from_numpy(logprobs)}
