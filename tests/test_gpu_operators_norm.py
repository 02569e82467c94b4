"""The norms after and before a block, with gate, residual and scales, against
the formula in 64 bits and its derivatives.

A value is a sum of products of at most eight 32-bit factors; a row's sum adds
at most 32 terms in one thread and 16 partial sums after them, so a factor is
off by at most 64 * 2^-24 of itself and a term by 128 * 2^-24 of its magnitude.
Sums over rows add at most 16 rows in a group and 80 groups after them: 256 *
2^-24 of the sum of magnitudes. On top comes the output's own rounding.
"""
import itertools

import pytest
import torch

import rns8_amd as r
from operator_cases import TYPES, U32, Guarded, assert_close, place
from rns8_amd import operators as ops

pytestmark = pytest.mark.gpu

EPS = 1e-5


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def ready():
    torch.cuda.synchronize()


def formula(v, flags, branch, keep):
    """h, y and the factors behind them, in the type of the values `v` (None where absent)."""
    x = v["x"]
    f, r1 = x, None
    if flags & ops.NORM_POST:
        r1 = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
        f = x * r1
        if v["post_weight"] is not None:
            f = f * v["post_weight"]
    h = branch * f if v["gate"] is None else branch * v["gate"] * f
    if v["residual"] is not None:
        h = h + keep * v["residual"]
    y = r2 = None
    if flags & ops.NORM_PRE:
        r2 = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
        y = h * r2 if v["pre_weight"] is None else h * r2 * v["pre_weight"]
    return h, y, r1, r2


def inputs(rows, cols, dtype, gate, residual, weights, pad=0, offset=0):
    v = {"x": place((3.0 * normal(1, rows, cols)).to(dtype), pad, offset), "residual": None, "gate": None,
         "post_weight": None, "pre_weight": None}
    if residual:
        v["residual"] = place(normal(2, rows, cols).to(dtype), pad, offset)
    if gate == "token":
        v["gate"] = place(normal(3, rows, cols).to(dtype), pad, offset)
    t = {k: None if g is None else g.t for k, g in v.items()}
    if gate == "row":
        t["gate"] = normal(3, cols).to(dtype)
    if weights:
        t["post_weight"], t["pre_weight"] = (1 + 0.3 * normal(4, cols)).to(dtype), (1 + 0.3 * normal(5, cols)).to(dtype)
    return t


def doubled(t):
    return {k: None if x is None else x.double() for k, x in t.items()}


def magnitude(t, flags, branch, keep):
    """Of h: the sum of its terms' magnitudes."""
    v = {k: None if x is None else x.abs() for k, x in doubled(t).items()}
    return formula(v, flags & ops.NORM_POST, abs(branch), abs(keep))[0]


SIZES = [(1, 1, 0, 0), (1, 4096, 0, 0), (3, 8, 1, 1), (5, 100, 3, 0), (7, 1101, 0, 0), (600, 63, 0, 1),
         (513, 2000, 8, 0), (530, 2056, 0, 0), (33, 8192, 0, 0), (520, 8200, 0, 0), (2, 32768, 0, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad,offset", SIZES)
@pytest.mark.parametrize("flags", [0, ops.NORM_POST, ops.NORM_PRE, ops.NORM_POST | ops.NORM_PRE])
@pytest.mark.parametrize("gate,residual,weights", [("row", True, True), ("token", True, False), (None, False, True)])
def test_forward(gpu_ctx, dtype, rows, cols, pad, offset, flags, gate, residual, weights):
    branch, keep = 0.75, -1.25
    t = inputs(rows, cols, dtype, gate, residual, weights, pad, offset)
    h, rstd = Guarded(rows, cols, dtype, pad, offset), torch.zeros(2, rows, device="cuda")
    more = {}
    if flags & ops.NORM_PRE:
        y, q = Guarded(rows, cols, dtype, pad, offset), Guarded(rows, ops.padded(cols), torch.int8, pad, offset)
        scale = torch.full((rows + 1,), 5.0, device="cuda")
        more = dict(y=y.t, q=q.t, q_scale=scale[:rows])
    ready()
    ops.BlockNorm(gpu_ctx, **t, h=h.t, rstd=rstd, flags=flags, eps=EPS, branch_scale=branch, residual_scale=keep,
                  **more)()
    ready()
    wh, wy, r1, r2 = formula(doubled(t), flags, branch, keep)
    mag = magnitude(t, flags, branch, keep)
    assert_close(h.t, wh, 128 * U32 * mag, "h")
    assert h.untouched()
    if flags & ops.NORM_POST:
        assert_close(rstd[0], r1[:, 0], 64 * U32 * r1[:, 0], "r1")
    if flags & ops.NORM_PRE:
        # h's own errors reach r2 through the mean of squares
        rel = 128 * U32 * ((mag * wh.abs()).mean(1, keepdim=True) * r2 * r2 + 1)
        assert_close(rstd[1], r2[:, 0], (rel * r2)[:, 0], "r2")
        w = 1.0 if t["pre_weight"] is None else t["pre_weight"].double().abs()
        off = 128 * U32 * mag * r2 * w + rel * wy.abs()
        assert_close(y.t, wy, off, "y")
        # the bytes: half a step, and what y and the scale may be off
        top = wy.abs().amax(1, keepdim=True)
        s = scale[:rows].double()[:, None]
        edge = off.amax(1, keepdim=True) + 4 * U32 * top
        assert ((s * 127 - top).abs() <= edge).all()
        assert ((q.t[:, :cols].double() * s - wy).abs() <= 0.5 * s + 2 * edge).all()
        assert not q.t[:, cols:].any()
        assert q.untouched() and y.untouched() and scale[rows] == 5.0


@pytest.mark.parametrize("into", ["x", "residual"])
def test_in_place(gpu_ctx, into):
    t = inputs(40, 777, torch.bfloat16, "row", True, True)
    apart = torch.empty_like(t["x"]).contiguous()
    y0, y1 = torch.empty(2, 40, 777, dtype=torch.bfloat16, device="cuda")
    ready()
    ops.BlockNorm(gpu_ctx, **t, h=apart, y=y0)()
    ready()
    ops.BlockNorm(gpu_ctx, **t, h=t[into], y=y1)()
    ready()
    assert torch.equal(t[into], apart) and torch.equal(y0, y1)


def test_rows_that_are_not_finite(gpu_ctx):
    """A NaN or an infinity stays in its row; a row of zeros gives zeros."""
    t = inputs(600, 100, torch.float32, "row", True, True)
    t["x"][3, 7], t["x"][4, 99], t["residual"][5, 0] = float("nan"), float("inf"), float("inf")
    t["x"][6], t["residual"][6] = 0.0, 0.0
    h, y = torch.empty(2, 600, 100, device="cuda")
    q, s = torch.ones(600, 112, dtype=torch.int8, device="cuda"), torch.empty(600, device="cuda")
    ready()
    ops.BlockNorm(gpu_ctx, **t, h=h, y=y, q=q, q_scale=s, eps=EPS)()
    ready()
    bad = torch.isnan(s)
    assert bad.nonzero().flatten().tolist() == [3, 4, 5] and not q[3:6].any()
    assert torch.isfinite(y[~bad]).all() and torch.isfinite(h[~bad]).all()
    assert not h[6].any() and not y[6].any() and s[6] == 0 and not q[6].any()


def exact_gradients(t, flags, branch, keep, dy, dh):
    names = [k for k in t if t[k] is not None]
    v = {k: None if t[k] is None else t[k].double().detach().requires_grad_() for k in t}
    h, y, _, _ = formula(v, flags, branch, keep)
    pairs = [(o, g.double()) for o, g in ((y, dy), (h, dh)) if g is not None and o is not None]
    grads = torch.autograd.grad([p[0] for p in pairs], [v[k] for k in names], [p[1] for p in pairs], allow_unused=True)
    return dict(zip(names, grads))


def gradient_magnitudes(t, flags, branch, keep, dy, dh):
    """The sums of the gradients' terms, each by its magnitude."""
    v = doubled(t)
    h, _, r1, r2 = formula(v, flags, branch, keep)
    mag = magnitude(t, flags, branch, keep)
    one = torch.ones_like(v["x"])
    r1 = torch.ones_like(one[:, :1]) if r1 is None else r1
    post = one if v["post_weight"] is None or not flags & ops.NORM_POST else v["post_weight"].abs() * one
    gate = one if v["gate"] is None else v["gate"].abs() * one
    d_h = torch.zeros_like(one) if dh is None else dh.double().abs()
    out = {}
    if dy is not None:
        wdy = dy.double().abs() * (one if v["pre_weight"] is None else v["pre_weight"].abs())
        # (r2 and the mean take the errors of h: its terms count in place of its value)
        grow = 1 + (mag * h.abs()).mean(1, keepdim=True) * r2 * r2
        d_h = d_h + grow * (r2 * wdy + 2 * mag * r2 ** 3 * (wdy * mag).mean(1, keepdim=True))
        out["pre_weight"] = (dy.double().abs() * mag * r2 * grow).sum(0)
    out["residual"] = abs(keep) * d_h
    f = v["x"].abs() * r1 * post
    out["gate"] = abs(branch) * f * d_h
    df = abs(branch) * gate * d_h
    out["post_weight"] = (df * v["x"].abs() * r1).sum(0)
    wdf = post * df
    out["x"] = r1 * wdf
    if flags & ops.NORM_POST:
        out["x"] = out["x"] + v["x"].abs() * r1 ** 3 * (wdf * v["x"].abs()).mean(1, keepdim=True)
    return out


BACK_SIZES = [(1, 1, 0, 0), (1, 4096, 0, 0), (3, 8, 1, 1), (9, 100, 3, 0), (70, 1101, 0, 0), (600, 63, 0, 1),
              (1030, 2000, 8, 0), (530, 2056, 0, 0), (17, 8192, 0, 0), (520, 8200, 0, 0), (2, 32768, 0, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad,offset", BACK_SIZES)
@pytest.mark.parametrize("flags", [0, ops.NORM_POST, ops.NORM_PRE, ops.NORM_POST | ops.NORM_PRE])
@pytest.mark.parametrize("gate,residual,weights,both", [
    ("row", True, True, True), ("token", True, False, False), (None, False, True, True)])
def test_gradients(gpu_ctx, dtype, rows, cols, pad, offset, flags, gate, residual, weights, both):
    branch, keep = 0.75, -1.25
    t = inputs(rows, cols, dtype, gate, residual, weights, pad, offset)
    pre = flags & ops.NORM_PRE
    dy = place(normal(8, rows, cols).to(dtype), pad, offset).t if pre else None
    dh = place(normal(9, rows, cols).to(dtype), pad, offset).t if both or not pre else None
    want = exact_gradients(t, flags, branch, keep, dy, dh)
    rstd = torch.zeros(2, rows, device="cuda")
    h = torch.empty(rows, cols, dtype=dtype, device="cuda")
    y = torch.empty(rows, cols, dtype=dtype, device="cuda") if pre else None
    settings = dict(flags=flags, eps=EPS, branch_scale=branch, residual_scale=keep)
    g = {k: Guarded(rows, cols, dtype, pad, offset) for k in ("x", "residual")}
    out = {"dx": g["x"].t}
    if residual:
        out["dresidual"] = g["residual"].t
    flat = {}
    if gate == "row":
        flat["gate"] = torch.full((cols + 1,), 6.0, device="cuda")
    elif gate == "token":
        g["gate"] = Guarded(rows, cols, dtype, pad, offset)
        out["dgate"] = g["gate"].t
    if weights and flags & ops.NORM_POST:
        flat["post_weight"] = torch.full((cols + 1,), 6.0, device="cuda")
    if weights and pre:
        flat["pre_weight"] = torch.full((cols + 1,), 6.0, device="cuda")
    ready()
    ops.BlockNorm(gpu_ctx, **t, h=h, y=y, rstd=rstd, **settings)()
    ops.BlockNormBackward(gpu_ctx, **t, rstd=rstd, dy=dy, dh=dh, **out, **settings,
                          **{"d" + k: x[:cols] for k, x in flat.items()})()
    ready()
    mags = gradient_magnitudes(t, flags, branch, keep, dy, dh)
    for k in out:
        assert_close(out[k], want[k[1:]], 128 * U32 * mags[k[1:]], k)
        assert g[k[1:]].untouched()
    for k, x in flat.items():
        mag = mags[k].sum(0) if mags[k].dim() == 2 else mags[k]
        assert_close(x[:cols], want[k], 256 * U32 * mag, "d" + k)
        assert x[cols] == 6.0


def test_gradients_against_differences(gpu_ctx):
    """The kernel's gradients along random directions against central differences of the formula in 64 bits."""
    rows, cols, flags = 6, 50, ops.NORM_POST | ops.NORM_PRE
    t = inputs(rows, cols, torch.float32, "row", True, True)
    t = {k: x.clone() for k, x in t.items()}
    dy, dh = normal(8, rows, cols), normal(9, rows, cols)
    rstd, h, y = torch.empty(2, rows, device="cuda"), *torch.empty(2, rows, cols, device="cuda")
    grads = {k: torch.empty_like(x) for k, x in t.items()}
    settings = dict(flags=flags, eps=EPS, branch_scale=0.5, residual_scale=2.0)
    ready()
    ops.BlockNorm(gpu_ctx, **t, h=h, y=y, rstd=rstd, **settings)()
    ops.BlockNormBackward(gpu_ctx, **t, rstd=rstd, dy=dy, dh=dh, **settings,
                          **{"d" + k: x for k, x in grads.items()})()
    ready()

    def loss(v):
        h, y, _, _ = formula(v, flags, 0.5, 2.0)
        return float((y * dy.double()).sum() + (h * dh.double()).sum())

    for seed, name in itertools.product(range(3), t):
        step = 1e-5 * normal(30 + seed, *t[name].shape).double()
        v = doubled(t)
        up, down = dict(v), dict(v)
        up[name], down[name] = v[name] + step, v[name] - step
        slope = (loss(up) - loss(down)) / 2
        got = float((grads[name].double() * step).sum())
        # differences: 64-bit cancellation and a third derivative times the step's cube; the gradient's own rounding
        size = float((grads[name].double().abs() * step.abs()).sum())
        assert abs(slope - got) <= 1e-4 * size + 1e-9, name


def test_no_rows(gpu_ctx):
    """Gradients that are sums over rows are zeros; nothing else is written."""
    e = torch.empty(0, 40, device="cuda")
    w = torch.ones(40, device="cuda")
    dw, dp, dg = torch.full((3, 40), 3.0, device="cuda")
    ready()
    ops.BlockNorm(gpu_ctx, x=e, post_weight=w, h=e, y=e)()
    ops.BlockNormBackward(gpu_ctx, x=e, rstd=torch.empty(2, 0, device="cuda"), gate=w, dy=e, dx=e, dgate=dg,
                          dpost_weight=dw, dpre_weight=dp)()
    ready()
    assert not dw.any() and not dp.any() and not dg.any()


def test_replayed_in_a_graph(gpu_ctx):
    from rns8_amd import hip

    t = inputs(520, 1101, torch.bfloat16, "row", True, True)
    dy = normal(8, 520, 1101).bfloat16()
    h, y, dx, dr = torch.empty(4, 520, 1101, dtype=torch.bfloat16, device="cuda")
    rstd, sums = torch.empty(2, 520, device="cuda"), torch.empty(3, 1101, device="cuda")
    calls = [ops.BlockNorm(gpu_ctx, **t, h=h, y=y, rstd=rstd),
             ops.BlockNormBackward(gpu_ctx, **t, rstd=rstd, dy=dy, dx=dx, dresidual=dr, dgate=sums[0],
                                   dpost_weight=sums[1], dpre_weight=sums[2])]
    ready()
    stream = hip.stream_create()
    try:
        hip.capture_begin(stream)
        for c in calls:
            c(stream)
        graph, exe = hip.capture_end(stream)
        try:
            for replay in range(3):
                t["x"].copy_(normal(50 + replay, 520, 1101))
                ready()
                hip.graph_launch(exe, stream)
                hip.stream_synchronize(stream)
                got = [v.clone() for v in (h, y, dx, dr, rstd, sums)]
                for v in (h, y, dx, dr, sums):
                    v.zero_()
                ready()
                for c in calls:
                    c()
                ready()
                assert all(torch.equal(a, b) for a, b in zip(got, (h, y, dx, dr, rstd, sums)))
        finally:
            hip.graph_destroy(graph, exe)
    finally:
        hip.stream_destroy(stream)


def test_refusals(gpu_ctx):
    x = torch.zeros(4, 32, device="cuda")
    big = torch.zeros(1, 32769, device="cuda")
    ready()
    for kwargs, status in (({"flags": 4, "y": x}, r.abi.INVALID_ARGUMENT), ({}, r.abi.INVALID_ARGUMENT),
                           ({"y": x, "eps": -1.0}, r.abi.INVALID_ARGUMENT),
                           ({"flags": ops.NORM_POST, "h": x, "y": x}, r.abi.INVALID_ARGUMENT),
                           ({"x": big, "h": big, "y": big}, r.abi.UNSUPPORTED_BACKEND)):
        with pytest.raises(r.Rns8Error) as e:
            ops.BlockNorm(gpu_ctx, **({"x": x} | kwargs))()
        assert e.value.status == status, kwargs
