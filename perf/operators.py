"""Operators of language models around the 8-bit matrix product, as programs call them.

Three families: the linear layer in 8-bit integers with a scale for each token
and channel (with its gradients), the norms around a residual block (which may
write the 8-bit rows that a linear layer reads), and the log-probabilities of
given tokens with entropy and top alternatives (with their gradient). A plain
form in elementary 32-bit torch operations stands beside the library's calls.
"""
from __future__ import annotations

import math

import torch

own = False

_CTX = None
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-6
_TINY = 2.0 ** -100  # rows below this quantize to zero


def listed():
    return [
        # One token between two blocks while a model answers: latency alone.
        {"name": "norm_one_token", "kind": "norm", "train": False, "type": "bf16", "tokens": 1, "dim": 4096,
         "gate": "row"},
        # A small training batch of odd sizes in single precision.
        {"name": "norm_train_ragged", "kind": "norm", "train": True, "type": "f32", "tokens": 1000, "dim": 1101,
         "gate": "token"},
        # A training batch: both norms, gate and residual forward, then their gradients.
        {"name": "norm_train", "kind": "norm", "train": True, "type": "bf16", "tokens": 8192, "dim": 4096,
         "gate": "row"},
        # One token through a linear layer: the weights are read once.
        {"name": "linear_one_token", "kind": "linear", "train": False, "type": "bf16", "tokens": 1, "outs": 8192,
         "ins": 8192, "bias": False},
        # A batch of requests, one token each, through the same layer.
        {"name": "linear_requests", "kind": "linear", "train": False, "type": "f16", "tokens": 48, "outs": 8192,
         "ins": 4096, "bias": True},
        # A short prompt through a layer of odd sizes.
        {"name": "linear_ragged", "kind": "linear", "train": False, "type": "f16", "tokens": 1000, "outs": 1101,
         "ins": 903, "bias": True},
        # A long prompt: the block's norm writes the 8-bit rows, the product reads them.
        {"name": "norm_linear", "kind": "norm_linear", "type": "bf16", "tokens": 8192, "outs": 8192, "ins": 8192,
         "gate": "row"},
        # A training step of a layer: the product, then the gradients of its input, weights and bias.
        {"name": "linear_train", "kind": "linear", "train": True, "type": "bf16", "tokens": 4096, "outs": 4096,
         "ins": 4096, "bias": True},
        # The same at odd sizes in single precision.
        {"name": "linear_train_ragged", "kind": "linear", "train": True, "type": "f32", "tokens": 500, "outs": 701,
         "ins": 611, "bias": True},
        # Four requests' next-token scores over a large vocabulary, a tenth of it ruled out.
        {"name": "score_requests", "kind": "score", "train": False, "type": "bf16", "tokens": 4, "vocab": 131072,
         "top": 20, "banned": True},
        # The log-probabilities of a prompt's own tokens, from single-precision logits.
        {"name": "score_prompt", "kind": "score", "train": False, "type": "f32", "tokens": 1000, "vocab": 50001,
         "top": 5, "banned": False},
        # A training loss over the vocabulary and its gradient.
        {"name": "score_train", "kind": "score", "train": True, "type": "bf16", "tokens": 4096, "vocab": 32768,
         "top": 0, "banned": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "linear", "linear", "linear", "norm_linear", "score", "score"])
    train = rng.random() < 0.5
    if kind == "norm":
        return {"kind": kind, "train": train, "type": rng.choice(["f32", "f16", "bf16"]),
                "tokens": _log(rng, 1, 8192), "dim": _log(rng, 64, 4096), "gate": rng.choice(["row", "token", "none"])}
    if kind == "linear":
        top = 4096 if train else 8192
        return {"kind": kind, "train": train, "type": rng.choice(["f32", "f16", "bf16"]),
                "tokens": _log(rng, 1, 4096), "outs": _log(rng, 64, top), "ins": _log(rng, 64, top),
                "bias": rng.random() < 0.5}
    if kind == "norm_linear":
        return {"kind": kind, "type": rng.choice(["f16", "bf16"]), "tokens": _log(rng, 1, 8192),
                "outs": _log(rng, 64, 8192), "ins": _log(rng, 64, 8192), "gate": rng.choice(["row", "token", "none"])}
    vocab = _log(rng, 500, 131072)
    return {"kind": kind, "train": train, "type": rng.choice(["f32", "f16", "bf16"]),
            "tokens": _log(rng, 1, min(4096, (1 << 27) // vocab)), "vocab": vocab, "top": rng.choice([0, 1, 5, 20]),
            "banned": rng.random() < 0.5}


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
    """Quantized weights and their channels' scales."""
    q = (d.normal(outs, ins) * 30.0).round_().clamp_(-127, 127).to(torch.int8)
    return q, torch.exp(0.2 * d.normal(outs)) / (30.0 * math.sqrt(ins))


def _norm_inputs(d, s, case, tokens, dim):
    t = _TYPES[case["type"]]
    s["x"] = _activations(d, tokens, dim).to(t)
    s["residual"] = (2.0 * d.normal(tokens, dim)).to(t)
    s["gate"] = None
    if case["gate"] != "none":
        s["gate"] = torch.sigmoid(d.normal(*([dim] if case["gate"] == "row" else [tokens, dim]))).to(t)
    s["post_weight"] = (1.0 + 0.2 * d.normal(dim)).to(t)
    s["pre_weight"] = (1.0 + 0.2 * d.normal(dim)).to(t)
    s["branch_scale"], s["residual_scale"] = 0.5, 1.0


def prepare(case, seed):
    d, t = _Draws(seed), _TYPES[case["type"]]
    s = {"case": case}
    if case["kind"] == "norm":
        _norm_inputs(d, s, case, case["tokens"], case["dim"])
        if case["train"]:
            s["dy"] = d.normal(case["tokens"], case["dim"]).to(t)
            s["dh"] = d.normal(case["tokens"], case["dim"]).to(t)
    elif case["kind"] == "linear":
        s["x"] = _activations(d, case["tokens"], case["ins"]).to(t)
        s["w"], s["w_scale"] = _weights(d, case["outs"], case["ins"])
        s["bias"] = d.normal(case["outs"]) if case["bias"] else None
        if case["train"]:
            s["dy"] = d.normal(case["tokens"], case["outs"]).to(t)
    elif case["kind"] == "norm_linear":
        _norm_inputs(d, s, case, case["tokens"], case["ins"])
        s["w"], s["w_scale"] = _weights(d, case["outs"], case["ins"])
    else:
        z = 2.5 * d.normal(case["tokens"], case["vocab"])
        s["targets"] = d.below(case["vocab"], case["tokens"])
        if case["banned"]:
            z.masked_fill_(d.below(10, case["vocab"]) == 0, -math.inf)
            # a given token is one that the model may say
            z.scatter_(1, s["targets"][:, None], 1.0)
        s["logits"] = z.to(t)
        if case["train"]:
            s["dlogp"] = -torch.rand(case["tokens"], generator=d.g, device="cuda") / case["tokens"]
            s["dentropy"] = 0.01 * d.normal(case["tokens"]) / case["tokens"]
    # the library's stream does not wait for torch's: the inputs are ready first
    torch.cuda.synchronize()
    return s


# ---- the plain form ------------------------------------------------------------------


def _quantize(v, dim):
    """v in 8 bits with one scale along `dim` (zero below _TINY, NaN where a value is not finite)."""
    amax = v.abs().amax(dim, keepdim=True)
    most = torch.full_like(amax, 127.0)  # (a tensor: by a number torch multiplies with the reciprocal)
    live = amax >= _TINY
    fine = torch.isfinite(amax)
    scale = torch.where(fine, torch.where(live, amax / most, torch.zeros_like(amax)), torch.full_like(amax, math.nan))
    q = torch.round(v * torch.where(live & fine, most / amax, torch.zeros_like(amax)))
    return torch.where(live & fine, q, torch.zeros_like(q)), scale


def _plain_norm(s, to=torch.float32):
    x, residual = s["x"].to(to), s["residual"].to(to)
    gate = 1.0 if s["gate"] is None else s["gate"].to(to)
    post, pre = s["post_weight"].to(to), s["pre_weight"].to(to)
    r1 = torch.rsqrt((x * x).mean(1, keepdim=True) + _EPS)
    f = x * r1 * post
    h = s["residual_scale"] * residual + s["branch_scale"] * gate * f
    r2 = torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS)
    return {"x": x, "gate": gate, "post": post, "pre": pre, "r1": r1, "f": f, "h": h, "r2": r2, "y": h * r2 * pre}


def _plain_norm_backward(s, n, to=torch.float32):
    dy, t = s["dy"].to(to), s["x"].dtype
    x, h, r1, r2 = n["x"], n["h"], n["r1"], n["r2"]
    wdy = n["pre"] * dy
    dh = s["dh"].to(to) + r2 * wdy - h * (r2 ** 3 * (wdy * h).mean(1, keepdim=True))
    df = s["branch_scale"] * n["gate"] * dh
    wdf = n["post"] * df
    out = {"dx": (r1 * wdf - x * (r1 ** 3 * (wdf * x).mean(1, keepdim=True))).to(t),
           "dresidual": (s["residual_scale"] * dh).to(t),
           "dpost_weight": (df * x * r1).sum(0), "dpre_weight": (dy * h * r2).sum(0)}
    if s["gate"] is not None:
        dgate = s["branch_scale"] * n["f"] * dh
        out["dgate"] = dgate.sum(0) if s["gate"].dim() == 1 else dgate.to(t)
    return out


def _plain_linear(s):
    t = s["x"].dtype
    q, scale = _quantize(s["x"].float(), 1)
    out = (q @ s["w"].float().t()) * scale * s["w_scale"]
    if s["bias"] is not None:
        out = out + s["bias"]
    got = {"out": out.to(t)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        gq, g_scale = _quantize(dy * s["w_scale"], 1)
        hq, h_scale = _quantize(dy * scale, 0)
        got["dx"] = ((gq @ s["w"].float()) * g_scale).to(t)
        got["dw"] = (hq.t() @ q) * h_scale.t()
        if s["bias"] is not None:
            got["dbias"] = dy.sum(0)
    return got


def _plain_score(s):
    case, z = s["case"], s["logits"].float()
    top = z.amax(1, keepdim=True)
    logp = (z - top) - torch.log(torch.exp(z - top).sum(1, keepdim=True))
    p = torch.exp(logp)
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    entropy = -plogp.sum(1)
    got = {"logp": logp.gather(1, s["targets"][:, None])[:, 0], "entropy": entropy}
    if case["top"]:
        # one integer per logit whose order is the logits', then the lower index first
        bits = (z + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)
        index = torch.arange(case["vocab"], device=z.device)
        keys = torch.topk(order * 2 ** 32 + (2 ** 31 - 1 - index), case["top"], 1).values
        ids = 2 ** 31 - 1 - torch.remainder(keys, 2 ** 32)
        got["top_ids"], got["top_logp"] = ids.to(torch.int32), logp.gather(1, ids)
    if case["train"]:
        d = -s["dlogp"][:, None] * p - s["dentropy"][:, None] * (plogp + p * entropy[:, None])
        d.scatter_add_(1, s["targets"][:, None], s["dlogp"][:, None])
        got["dlogits"] = d.to(s["logits"].dtype)
    return got


def _plain(s):
    case = s["case"]
    if case["kind"] == "linear":
        return _plain_linear(s)
    if case["kind"] == "score":
        return _plain_score(s)
    n, t = _plain_norm(s), s["x"].dtype
    got = {"h": n["h"].to(t)}
    if case["kind"] == "norm":
        got["y"] = n["y"].to(t)
        return got | (_plain_norm_backward(s, n) if case["train"] else {})
    q, scale = _quantize(n["y"], 1)
    got["out"] = ((q @ s["w"].float().t()) * scale * s["w_scale"]).to(t)
    return got


# ---- the library's calls -----------------------------------------------------------------


def _context():
    """One context per program, as a program that serves a model holds it."""
    global _CTX
    if _CTX is None:
        import rns8_amd

        _CTX = rns8_amd.Context(0)
    return _CTX


def _calls(s):
    """The calls of one pass with their arguments and outputs in place, as a program that repeats them keeps them."""
    from rns8_amd import operators as ops

    case, ctx = s["case"], _context()
    t = _TYPES[case["type"]]
    empty = lambda *shape, dtype=t: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    f32 = torch.float32
    tokens = case["tokens"]
    if case["kind"] in ("norm", "norm_linear"):
        dim = s["x"].shape[1]
        block = dict(x=s["x"], residual=s["residual"], gate=s["gate"], post_weight=s["post_weight"],
                     pre_weight=s["pre_weight"], eps=_EPS, branch_scale=s["branch_scale"],
                     residual_scale=s["residual_scale"])
        out = {"h": empty(tokens, dim)}
        if case["kind"] == "norm_linear":
            q, scale = empty(tokens, ops.padded(dim), dtype=torch.int8), empty(tokens, dtype=f32)
            out["out"] = empty(tokens, case["outs"])
            return [ops.BlockNorm(ctx, **block, h=out["h"], q=q, q_scale=scale),
                    ops.GemmI8Scaled(ctx, a=q[:, :dim], b=s["w"], a_scale=scale, b_scale=s["w_scale"],
                                     out=out["out"])], out
        out["y"] = empty(tokens, dim)
        if not case["train"]:
            return [ops.BlockNorm(ctx, **block, h=out["h"], y=out["y"])], out
        rstd = empty(2, tokens, dtype=f32)
        out |= {"dx": empty(tokens, dim), "dresidual": empty(tokens, dim), "dpost_weight": empty(dim, dtype=f32),
                "dpre_weight": empty(dim, dtype=f32)}
        if s["gate"] is not None:
            out["dgate"] = empty(dim, dtype=f32) if s["gate"].dim() == 1 else empty(tokens, dim)
        return [ops.BlockNorm(ctx, **block, h=out["h"], y=out["y"], rstd=rstd),
                ops.BlockNormBackward(ctx, **block, rstd=rstd, dy=s["dy"], dh=s["dh"], dx=out["dx"],
                                      dresidual=out["dresidual"], dgate=out.get("dgate"),
                                      dpost_weight=out["dpost_weight"], dpre_weight=out["dpre_weight"])], out
    if case["kind"] == "linear":
        outs, ins = s["w"].shape
        out = {"out": empty(tokens, outs)}
        layer = dict(x=s["x"], w=s["w"], w_scale=s["w_scale"], bias=s["bias"], out=out["out"])
        if not case["train"]:
            return [ops.LinearI8(ctx, **layer)], out
        q, scale = empty(tokens, ops.padded(ins), dtype=torch.int8), empty(tokens, dtype=f32)
        out |= {"dx": empty(tokens, ins), "dw": empty(outs, ins, dtype=f32)}
        if case["bias"]:
            out["dbias"] = empty(outs, dtype=f32)
        return [ops.LinearI8(ctx, **layer, x_q=q, x_scale=scale),
                ops.LinearI8Backward(ctx, dy=s["dy"], x_q=q[:, :ins], x_scale=scale, w=s["w"], w_scale=s["w_scale"],
                                     dx=out["dx"], dw=out["dw"], dbias=out.get("dbias"))], out
    top = case["top"]
    out = {"logp": empty(tokens, dtype=f32), "entropy": empty(tokens, dtype=f32)}
    if top:
        out |= {"top_ids": empty(tokens, top, dtype=torch.int32), "top_logp": empty(tokens, top, dtype=f32)}
    given = dict(logits=s["logits"], targets=s["targets"])
    if not case["train"]:
        return [ops.TokenLogprobs(ctx, **given, **out)], out
    lse = empty(tokens, dtype=f32)
    forward = ops.TokenLogprobs(ctx, **given, **out, lse=lse)
    out["dlogits"] = torch.empty_like(s["logits"])
    return [forward, ops.TokenLogprobsBackward(ctx, **given, lse=lse, entropy=out["entropy"], dlogp=s["dlogp"],
                                               dentropy=s["dentropy"], dlogits=out["dlogits"])], out


def run(state):
    if not own:
        return _plain(state)
    if "calls" not in state:
        state["calls"], state["out"] = _calls(state)
    for call in state["calls"]:
        call()
    return state["out"]


# ---- what a pass cannot do without ---------------------------------------------------


def work(case):
    size, tokens = _SIZE[case["type"]], case["tokens"]
    if case["kind"] == "score":
        cells = tokens * case["vocab"]
        return {"bytes": cells * size * (2 if case["train"] else 1) + tokens * (24 + 8 * case["top"]),
                "flops": cells * (10 if case["train"] else 5)}
    if case["kind"] == "linear":
        outs, ins = case["outs"], case["ins"]
        moved = (tokens * ins + tokens * outs) * size + outs * ins + 8 * outs
        if not case["train"]:
            return {"bytes": moved, "flops": 2 * tokens * outs * ins}
        return {"bytes": 2 * (tokens * ins + tokens * outs) * size + 5 * outs * ins + 12 * outs,
                "flops": 6 * tokens * outs * ins}
    dim = case["dim"] if case["kind"] == "norm" else case["ins"]
    gates = {"row": 0, "token": 1, "none": 0}[case["gate"]]
    if case["kind"] == "norm":
        if case["train"]:
            return {"bytes": tokens * dim * size * (8 + 2 * gates) + 20 * dim, "flops": 40 * tokens * dim}
        return {"bytes": tokens * dim * size * (4 + gates) + 6 * dim, "flops": 12 * tokens * dim}
    outs = case["outs"]
    return {"bytes": (tokens * dim * (3 + gates) + tokens * outs) * size + outs * dim + 4 * outs,
            "flops": 2 * tokens * outs * dim + 14 * tokens * dim}


# ---- the definition in 64 bits ----------------------------------------------------------


def _rms(v):
    return 1.0 / torch.sqrt(torch.mean(v * v, dim=-1, keepdim=True) + _EPS)


def _eight_bits(v, dim):
    """What v is in 8 bits: the whole numbers and the scale (all rows of these cases are finite)."""
    top = torch.linalg.vector_norm(v, ord=math.inf, dim=dim, keepdim=True)
    step = top / 127.0
    return torch.where(top < _TINY, torch.zeros_like(v), torch.round(v / step)), torch.where(top < _TINY, 0.0 * top, step)


def _exact_norm(s):
    """The block's two norms with every gradient, by differentiation of the definition in 64 bits."""
    names = [k for k in ("x", "residual", "gate", "post_weight", "pre_weight") if s[k] is not None]
    v = {k: s[k].double().requires_grad_("dy" in s) for k in names}
    branch = v["x"] * _rms(v["x"]) * v["post_weight"]
    if "gate" in v:
        branch = branch * v["gate"]
    h = v["residual"] * s["residual_scale"] + branch * s["branch_scale"]
    y = h * _rms(h) * v["pre_weight"]
    out = {"h": h.detach(), "y": y.detach()}
    if "dy" in s:
        grads = torch.autograd.grad([y, h], [v[k] for k in names], [s["dy"].double(), s["dh"].double()])
        out |= {"d" + k: g for k, g in zip(names, grads)}
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("norm", "norm_linear"):
        out = _exact_norm(s)
        if case["kind"] == "norm_linear":
            q, step = _eight_bits(out.pop("y"), 1)
            out["out"] = torch.mm(q, s["w"].double().t().contiguous()) * (step * s["w_scale"].double())
        return out
    if case["kind"] == "linear":
        w, w_scale = s["w"].double(), s["w_scale"].double()
        q, step = _eight_bits(s["x"].double(), 1)
        out = {"out": torch.mm(q, w.t().contiguous()) * (step * w_scale)}
        if case["bias"]:
            out["out"] += s["bias"].double()
        if case["train"]:
            dy = s["dy"].double()
            g, g_step = _eight_bits(dy * w_scale, 1)
            out["dx"] = torch.mm(g, w) * g_step
            g, g_step = _eight_bits(dy * step, 0)
            out["dw"] = torch.mm(g.t().contiguous(), q) * g_step.t()
            if case["bias"]:
                out["dbias"] = dy.sum(0)
        return out
    parts = []
    rows = max(1, (1 << 25) // case["vocab"])
    for at in range(0, case["tokens"], rows):
        z, target = s["logits"][at:at + rows].double(), s["targets"][at:at + rows, None]
        logp = torch.log_softmax(z, 1)
        p = logp.exp()
        entropy = torch.special.entr(p).sum(1)
        part = {"logp": logp.gather(1, target)[:, 0], "entropy": entropy}
        if case["top"]:
            ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :case["top"]]
            part["top_ids"], part["top_logp"] = ids.to(torch.int32), logp.gather(1, ids)
        if case["train"]:
            g_logp, g_entropy = s["dlogp"][at:at + rows, None].double(), s["dentropy"][at:at + rows, None].double()
            hit = torch.zeros_like(p).scatter_(1, target, 1.0)
            spread = torch.where(p > 0, logp, torch.zeros_like(p)) + entropy[:, None]
            part["dlogits"] = g_logp * (hit - p) - g_entropy * p * spread
        parts.append(part)
    return {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
