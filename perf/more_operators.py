"""Operators of language models on 4-bit microscaled matrices, as programs call them.

A matrix in this form (MX4 below) has, for each 32 neighbouring values of a row, one
power of two and 32 values of 4 bits. Four families: rounding to it and back, the
product of two such matrices, the linear layer on it (with its gradients), and a
mixture-of-experts layer for a few tokens whose experts' weights are held in it. A
plain form in elementary 32-bit torch operations stands beside the library's calls.
"""
from __future__ import annotations

import math

import torch

own = False

_CTX = None
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_BITS = 4.25 / 8  # bytes to a value, its share of the scale with it


def listed():
    return [
        # Weights of odd sizes after an optimizer's step, for both products of a training step.
        {"name": "round_ragged", "kind": "round", "type": "f32", "rows": 1000, "cols": 1101},
        # The same for a large layer's weights.
        {"name": "round_weights", "kind": "round", "type": "bf16", "rows": 8192, "cols": 8192},
        # A short prompt's rows, rounded once, through two layers of odd sizes that read them.
        {"name": "product_ragged", "kind": "product", "type": "f16", "tokens": 300, "outs": 1101, "ins": 903},
        # A long prompt through the two first layers of a gated block.
        {"name": "product_prompt", "kind": "product", "type": "bf16", "tokens": 8192, "outs": 8192, "ins": 8192},
        # One token through a linear layer: the weights are read once.
        {"name": "linear_one_token", "kind": "linear", "train": False, "type": "bf16", "tokens": 1, "outs": 8192,
         "ins": 8192, "bias": False},
        # A batch of requests, one token each, through the same layer.
        {"name": "linear_requests", "kind": "linear", "train": False, "type": "f16", "tokens": 48, "outs": 8192,
         "ins": 4096, "bias": True},
        # A training step of a layer: its weights rounded, the product, the gradients of input, weights and bias.
        {"name": "linear_train", "kind": "linear", "train": True, "type": "bf16", "tokens": 4096, "outs": 4096,
         "ins": 4096, "bias": True},
        # The same at odd sizes in single precision.
        {"name": "linear_train_ragged", "kind": "linear", "train": True, "type": "f32", "tokens": 500, "outs": 701,
         "ins": 611, "bias": True},
        # One token of one answer: eight experts of 128 are read.
        {"name": "experts_one_token", "kind": "experts", "type": "bf16", "tokens": 1, "experts": 128, "top": 8,
         "width": 4096, "inner": 1536, "normalize": True},
        # Five answers at once in a small model of odd sizes.
        {"name": "experts_ragged", "kind": "experts", "type": "f32", "tokens": 5, "experts": 12, "top": 3,
         "width": 1101, "inner": 701, "normalize": False},
        # A batch of requests, one token each: nearly all experts are read.
        {"name": "experts_requests", "kind": "experts", "type": "bf16", "tokens": 64, "experts": 128, "top": 8,
         "width": 4096, "inner": 1536, "normalize": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["round", "product", "linear", "linear", "linear", "experts", "experts"])
    case = {"kind": kind, "type": rng.choice(["f32", "f16", "bf16"])}
    if kind == "round":
        return case | {"rows": _log(rng, 1, 8192), "cols": _log(rng, 1, 8192)}
    if kind == "product":
        return case | {"tokens": _log(rng, 1, 8192), "outs": _log(rng, 64, 8192), "ins": _log(rng, 64, 8192)}
    if kind == "linear":
        train = rng.random() < 0.5
        top = 4096 if train else 8192
        return case | {"train": train, "tokens": _log(rng, 1, 4096), "outs": _log(rng, 64, top),
                       "ins": _log(rng, 64, top), "bias": rng.random() < 0.5}
    experts = _log(rng, 4, 256)
    inner = _log(rng, 64, 2048)
    width = _log(rng, 64, min(4096, (128 * 1536 * 4096) // (experts * inner)))
    return case | {"tokens": _log(rng, 1, 64), "experts": experts, "top": rng.randint(1, 8 if experts >= 8 else 4),
                   "width": width, "inner": inner, "normalize": rng.random() < 0.5}


# ---- what a program has in hand ---------------------------------------------------


class _Draws:
    """Seeded normal draws on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda")

    def below(self, high, *shape):
        return torch.randint(high, shape, generator=self.g, device="cuda")


def _activations(d, tokens, dim):
    """Rows of unit scale in which a few channels are much larger than the others."""
    x = d.normal(tokens, dim)
    x[:, d.below(dim, max(1, dim // 500))] *= 8.0
    return x


def _weights(d, outs, ins):
    """Weights as checkpoints hold them: rows of 4-bit codes, two to a byte (the first in the low bits), and of
    exponents, one to 32 values."""
    w = torch.nn.functional.pad(d.normal(outs, ins) / math.sqrt(ins), (0, -ins % 32)).view(outs, -1, 32)
    exponent = torch.frexp(w.abs().amax(2, keepdim=True)).exponent - 3
    y = torch.ldexp(w, -exponent)
    step = torch.where(y.abs() < 2, 2.0, torch.where(y.abs() < 4, 1.0, 0.5))
    level = (torch.round(y.abs() * step) / step).clamp_(max=6.0)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    code = (torch.bucketize(level, edges) + 8 * (y < 0)).view(outs, -1).to(torch.uint8)
    return code[:, ::2][:, :(ins + 1) // 2] | code[:, 1::2][:, :(ins + 1) // 2] << 4, (exponent + 127).view(outs, -1).to(torch.uint8)


def prepare(case, seed):
    d, t = _Draws(seed), _TYPES[case["type"]]
    s = {"case": case}
    if case["kind"] == "round":
        s["x"] = (d.normal(case["rows"], case["cols"]) / math.sqrt(case["cols"])).to(t)
    elif case["kind"] == "product":
        s["x"] = _activations(d, case["tokens"], case["ins"]).to(t)
        s["w"] = [_weights(d, case["outs"], case["ins"]) for _ in range(2)]
    elif case["kind"] == "linear":
        s["x"] = _activations(d, case["tokens"], case["ins"]).to(t)
        s["bias"] = d.normal(case["outs"]) if case["bias"] else None
        if case["train"]:
            s["w"] = (d.normal(case["outs"], case["ins"]) / math.sqrt(case["ins"])).to(t)
            s["dy"] = d.normal(case["tokens"], case["outs"]).to(t)
        else:
            s["w"] = _weights(d, case["outs"], case["ins"])
    else:
        experts, width, inner = case["experts"], case["width"], case["inner"]
        s["x"] = _activations(d, case["tokens"], width).to(t)
        s["router"] = (d.normal(experts, width) * 1.5 / math.sqrt(width)).to(t)
        for name, outs, ins in (("gate", inner, width), ("up", inner, width), ("down", width, inner)):
            each = [_weights(d, outs, ins) for _ in range(experts)]
            s[name] = tuple(torch.stack(part) for part in zip(*each))
    # the library's stream does not wait for torch's: the inputs are ready first
    torch.cuda.synchronize()
    return s


# ---- the plain form ------------------------------------------------------------------


def _rounded(v):
    """v's rows as MX4 holds them: blocks of 32 values with one power of two (NaN where a value is not finite)."""
    rows, cols = v.shape
    y = torch.nn.functional.pad(v, (0, -cols % 32)).view(rows, -1, 32)
    amax = y.abs().amax(2, keepdim=True)
    # the power of two that takes the largest value between 4 and 8, of which 6 is the largest that 4 bits hold
    exponent = torch.clamp(torch.frexp(amax).exponent - 3, min=-127)
    y = torch.ldexp(y, -exponent)
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.clamp(torch.round(a / step) * step, max=6.0)
    y = torch.ldexp(torch.copysign(a, y), exponent)
    return torch.where(torch.isfinite(amax), y, torch.full_like(y, math.nan)).view(rows, -1)[:, :cols]


def _values(w, cols):
    """The 32-bit values of codes and exponents; any leading dimensions."""
    data, exponent = w
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=data.device)
    levels = torch.cat([levels, -levels])
    code = torch.stack([data & 15, data >> 4], -1).flatten(-2)[..., :cols].int()
    scale = torch.ldexp(torch.ones_like(exponent, dtype=torch.float32), exponent.int() - 127)
    return levels[code] * scale.repeat_interleave(32, -1)[..., :cols]


def _plain_linear(s):
    case, t = s["case"], s["x"].dtype
    x = s["x"].float()
    w = s["w"].float() if case["train"] else None
    out = _rounded(x) @ (_rounded(w) if case["train"] else _values(s["w"], case["ins"])).t()
    if s["bias"] is not None:
        out = out + s["bias"]
    got = {"out": out.to(t)}
    if case["train"]:
        dy = s["dy"].float()
        got["dx"] = (_rounded(dy) @ _rounded(w.t()).t()).to(t)
        got["dw"] = _rounded(dy.t()) @ _rounded(x.t()).t()
        if s["bias"] is not None:
            got["dbias"] = dy.sum(0)
    return got


def _plain_experts(s):
    case, t = s["case"], s["x"].dtype
    tokens, experts, top = case["tokens"], case["experts"], case["top"]
    x = s["x"].float()
    # the scores in 64 bits: two experts whose scores are next to each other must not change places
    logits = (s["x"].double() @ s["router"].double().t()).float()
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
    chosen = logits.gather(1, ids)
    p = torch.exp(chosen - logits.amax(1, keepdim=True))
    total = p if case["normalize"] else torch.exp(logits - logits.amax(1, keepdim=True))
    weights = p / total.sum(1, keepdim=True)
    if tokens * top < experts:
        # the chosen experts, once for each token that chose them
        row, use = torch.arange(tokens, device=x.device).repeat_interleave(top), ids.flatten()
        gate, up, down = ((w[0][use], w[1][use]) for w in (s["gate"], s["up"], s["down"]))
        g = torch.bmm(_values(gate, case["width"]), x[row][:, :, None])
        u = torch.bmm(_values(up, case["width"]), x[row][:, :, None])
        y = torch.bmm(_values(down, case["inner"]), g * torch.sigmoid(g) * u)[:, :, 0]
        out = (y.view(tokens, top, -1) * weights[:, :, None]).sum(1)
    else:
        # every expert on every token, those that the token did not choose with no weight
        share = torch.zeros(tokens, experts, device=x.device).scatter_(1, ids, weights)
        xt = x.t().contiguous().expand(experts, -1, -1)
        g, u = torch.bmm(_values(s["gate"], case["width"]), xt), torch.bmm(_values(s["up"], case["width"]), xt)
        h = g * torch.sigmoid(g) * u * share.t()[:, None, :]
        out = torch.bmm(_values(s["down"], case["inner"]), h).sum(0).t()
    return {"out": out.to(t), "ids": ids.to(torch.int32), "weights": weights}


def _plain(s):
    case, t = s["case"], s["x"].dtype
    if case["kind"] == "linear":
        return _plain_linear(s)
    if case["kind"] == "experts":
        return _plain_experts(s)
    x = s["x"].float()
    if case["kind"] == "round":
        return {"rows": _rounded(x).to(t), "columns": _rounded(x.t()).to(t)}
    a = _rounded(x)
    first, second = s["w"]
    return {"first": (a @ _values(first, case["ins"]).t()).to(t), "second": (a @ _values(second, case["ins"]).t()).to(t)}


# ---- the library's calls -----------------------------------------------------------------


def _context():
    """One context per program, as a program that serves a model holds it."""
    global _CTX
    if _CTX is None:
        import rns8_amd

        _CTX = rns8_amd.Context(0)
    return _CTX


def _laid_out(ops, ctx, w, rows, cols):
    """Weights from a checkpoint's rows in the library's layout, as a program keeps them."""
    data, exponent = w
    q = torch.empty(ops.mx4_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    ops.PackMx4(ctx, data=data, scale=exponent, q=q, cols=cols)(torch.cuda.current_stream().cuda_stream)
    return q


def _calls(s):
    """The calls of one pass with their arguments and outputs in place, as a program that repeats them keeps them."""
    from rns8_amd import operators as ops

    case, ctx = s["case"], _context()
    t = _TYPES[case["type"]]
    empty = lambda *shape, dtype=t: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    mx4 = lambda rows, cols: empty(ops.mx4_bytes(rows, cols), dtype=torch.uint8)  # noqa: E731
    if case["kind"] == "round":
        rows, cols = case["rows"], case["cols"]
        q, qt = mx4(rows, cols), mx4(cols, rows)
        out = {"rows": empty(rows, cols), "columns": empty(cols, rows)}
        return [ops.QuantizeMx4(ctx, x=s["x"], q=q, q_t=qt), ops.DequantizeMx4(ctx, q=q, out=out["rows"]),
                ops.DequantizeMx4(ctx, q=qt, out=out["columns"])], out
    if case["kind"] == "product":
        tokens, outs, ins = case["tokens"], case["outs"], case["ins"]
        a = mx4(tokens, ins)
        out = {"first": empty(tokens, outs), "second": empty(tokens, outs)}
        return [ops.QuantizeMx4(ctx, x=s["x"], q=a)] + [
            ops.GemmMx4(ctx, a=a, b=_laid_out(ops, ctx, w, outs, ins), k=ins, out=out[name])
            for name, w in zip(out, s["w"])], out
    if case["kind"] == "linear":
        tokens, outs, ins = case["tokens"], case["outs"], case["ins"]
        out = {"out": empty(tokens, outs)}
        if not case["train"]:
            return [ops.LinearMx4(ctx, x=s["x"], w=_laid_out(ops, ctx, s["w"], outs, ins), bias=s["bias"],
                                  out=out["out"])], out
        w, w_t = mx4(outs, ins), mx4(ins, outs)
        out |= {"dx": empty(tokens, ins), "dw": empty(outs, ins, dtype=torch.float32)}
        if case["bias"]:
            out["dbias"] = empty(outs, dtype=torch.float32)
        return [ops.QuantizeMx4(ctx, x=s["w"], q=w, q_t=w_t),
                ops.LinearMx4(ctx, x=s["x"], w=w, bias=s["bias"], out=out["out"]),
                ops.LinearMx4Backward(ctx, dy=s["dy"], x=s["x"], w_t=w_t, dx=out["dx"], dw=out["dw"],
                                      dbias=out.get("dbias"))], out
    tokens, experts, width, inner = case["tokens"], case["experts"], case["width"], case["inner"]
    held = {}
    for name, rows, cols in (("gate", inner, width), ("up", inner, width), ("down", width, inner)):
        data, exponent = s[name]
        held[name] = torch.stack([_laid_out(ops, ctx, w, rows, cols) for w in zip(data, exponent)])
    out = {"out": empty(tokens, width), "ids": empty(tokens, case["top"], dtype=torch.int32),
           "weights": empty(tokens, case["top"], dtype=torch.float32)}
    return [ops.ExpertsMx4(ctx, x=s["x"], router=s["router"], **held, inner=inner, normalize=case["normalize"],
                           **out)], out


def run(state):
    if not own:
        return _plain(state)
    if "calls" not in state:
        state["calls"], state["out"] = _calls(state)
    stream = torch.cuda.current_stream().cuda_stream
    for call in state["calls"]:
        call(stream)
    return state["out"]


# ---- what a pass cannot do without ---------------------------------------------------


def work(case):
    size = _SIZE[case["type"]]
    if case["kind"] == "round":
        # the values read, both forms written and read, the values of both written
        cells = case["rows"] * case["cols"]
        return {"bytes": cells * (3 * size + 4 * _BITS), "flops": 8 * cells}
    tokens = case["tokens"]
    if case["kind"] == "product":
        outs, ins = case["outs"], case["ins"]
        return {"bytes": tokens * (ins + 2 * outs) * size + 2 * outs * ins * _BITS, "flops": 4 * tokens * outs * ins}
    if case["kind"] == "linear":
        outs, ins = case["outs"], case["ins"]
        if not case["train"]:
            return {"bytes": tokens * (ins + outs) * size + outs * ins * _BITS + 4 * outs,
                    "flops": 2 * tokens * outs * ins}
        return {"bytes": 2 * tokens * (ins + outs) * size + outs * ins * (size + 4) + 8 * outs,
                "flops": 6 * tokens * outs * ins}
    experts, top, width, inner = case["experts"], case["top"], case["width"], case["inner"]
    read = experts * (1 - (1 - top / experts) ** tokens)  # experts that some token chooses, if all are as likely
    return {"bytes": 3 * read * width * inner * _BITS + (experts + 2 * tokens) * width * size + 8 * tokens * top,
            "flops": 6 * tokens * top * width * inner + 2 * tokens * experts * width}


# ---- the definition in 64 bits ----------------------------------------------------------


def _nearest(v):
    """The definition of the rounding: in each block of 32 along a row the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6, the
    one with an even code where two are as near, times the largest power of two that is at most a quarter of the
    block's largest value."""
    rows, cols = v.shape
    blocks = torch.nn.functional.pad(v, (0, -cols % 32)).reshape(rows, -1, 32)
    top = torch.linalg.vector_norm(blocks, ord=math.inf, dim=2, keepdim=True)
    unit = torch.exp2(torch.clamp(torch.floor(torch.log2(top)) - 2, min=-127.0))
    y = blocks.abs() / unit
    level = 0.5 * ((y > 0.25).double() + (y >= 0.75).double() + (y > 1.25).double() + (y >= 1.75).double())
    level += (y > 2.5).double() + (y >= 3.5).double() + 2.0 * (y > 5.0).double()
    return (torch.sign(blocks) * level * unit).reshape(rows, -1)[:, :cols]


def _decoded(w, cols):
    """The values of one matrix's codes and exponents."""
    data, exponent = w
    code = torch.empty(data.shape[0], 2 * data.shape[1], dtype=torch.int64, device=data.device)
    code[:, 0::2], code[:, 1::2] = data.long() % 16, data.long() // 16
    code = code[:, :cols]
    size, high = code % 8, code % 8 // 2
    level = torch.where(high == 0, 0.5 * size, torch.exp2(high.double() - 1) * (1 + 0.5 * (size % 2)))
    unit = torch.exp2(exponent.double() - 127)
    block = torch.arange(cols, device=data.device) // 32
    return torch.where(code >= 8, -level, level) * unit[:, block]


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["kind"] == "round":
        return {"rows": _nearest(x), "columns": _nearest(x.t().contiguous())}
    if case["kind"] == "product":
        a = _nearest(x)
        return {name: torch.mm(a, _decoded(w, case["ins"]).t().contiguous()) for name, w in zip(("first", "second"), s["w"])}
    if case["kind"] == "linear":
        w = s["w"].double() if case["train"] else None
        weights = _nearest(w) if case["train"] else _decoded(s["w"], case["ins"])
        out = {"out": torch.mm(_nearest(x), weights.t().contiguous())}
        if case["bias"]:
            out["out"] += s["bias"].double()
        if case["train"]:
            dy = s["dy"].double()
            out["dx"] = torch.mm(_nearest(dy), _nearest(w.t().contiguous()).t().contiguous())
            out["dw"] = torch.mm(_nearest(dy.t().contiguous()), _nearest(x.t().contiguous()).t().contiguous())
            if case["bias"]:
                out["dbias"] = dy.sum(0)
        return out
    logits = torch.mm(x, s["router"].double().t().contiguous()).float().double()
    probability = torch.softmax(logits, 1)
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :case["top"]]
    weights = probability.gather(1, ids)
    if case["normalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    out = torch.zeros_like(x)
    for e in range(case["experts"]):
        token, slot = (ids == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        gate, up, down = ((s[k][0][e], s[k][1][e]) for k in ("gate", "up", "down"))
        mine = x[token].t().contiguous()
        hidden = torch.nn.functional.silu(torch.mm(_decoded(gate, case["width"]), mine))
        hidden = hidden * torch.mm(_decoded(up, case["width"]), mine)
        out[token] += torch.mm(_decoded(down, case["inner"]), hidden).t() * weights[token, slot][:, None]
    return {"out": out, "ids": ids.to(torch.int32), "weights": weights}
