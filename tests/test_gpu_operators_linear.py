"""8-bit quantization, the scaled product and the linear layer with its gradients.

Quantization has to give the very bytes and scales of the definition in 32-bit
operations. A product's sum is exact in integers: what is left is the rounding
of the sum to 32 bits, three 32-bit operations and the output's own rounding, so
|error| <= 4 * 2^-24 * (|sum * scales| + |bias|) + the output's unit of the
result.
"""
import pytest
import torch

import rns8_amd as r
from operator_cases import TYPES, U32, Guarded, assert_close, place, quantize
from rns8_amd import operators as ops

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def integers(seed, *shape, low=-128, high=128):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(low, high, shape, generator=g, device="cuda").to(torch.int8)


def ready():
    torch.cuda.synchronize()  # the library's stream does not wait for torch's


SPECIAL = [0.0, 1e-38, 2.0 ** -100, 2.0 ** -101, float("inf"), float("-inf"), float("nan")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad,offset", [
    (1, 1, 0, 0), (1, 7, 0, 1), (3, 64, 0, 0), (5, 100, 3, 1), (600, 63, 0, 0), (600, 2000, 0, 3), (513, 2049, 1, 0),
    (520, 8200, 8, 8), (9, 4096, 0, 0), (4, 16385, 0, 0), (2, 40001, 0, 1)])
@pytest.mark.parametrize("scaled", [False, True])
def test_rows_in_8_bits(gpu_ctx, dtype, rows, cols, pad, offset, scaled):
    v = normal(rows * 7 + cols, rows, cols).to(dtype)
    for i, value in enumerate(SPECIAL):  # rows of one special value among ordinary ones
        if i + 1 < rows:
            v[i + 1] = 0 if value < 1 else v[i + 1]
            v[i + 1, (3 * i) % cols] = value
    x = place(v, pad, offset)
    m = torch.exp(normal(5, cols)) if scaled else None
    wide = ops.padded(cols)
    q, scale = Guarded(rows, wide, torch.int8, pad, offset), torch.full((rows + 1,), 7.0, device="cuda")
    ready()
    ops.QuantizeRows(gpu_ctx, x=x.t, q=q.t, scale=scale[:rows], multiplier=m)()
    ready()
    want_q, want_s = quantize(v.float() * m if scaled else v.float(), 1)
    assert torch.equal(q.t[:, :cols], want_q)
    assert not q.t[:, cols:].any()
    assert torch.equal(scale[:rows].view(torch.int32)[~torch.isnan(want_s)],
                       want_s.view(torch.int32)[~torch.isnan(want_s)])
    assert torch.equal(torch.isnan(scale[:rows]), torch.isnan(want_s))
    assert q.untouched() and scale[rows] == 7.0


def test_rows_in_8_bits_without_room_for_zeros(gpu_ctx):
    v = normal(3, 6, 21)
    x, q = place(v), Guarded(6, 21, torch.int8)
    scale = torch.empty(6, device="cuda")
    ready()
    ops.QuantizeRows(gpu_ctx, x=x.t, q=q.t, scale=scale)()
    ready()
    assert torch.equal(q.t, quantize(v, 1)[0]) and q.untouched()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad,offset", [
    (0, 5, 0, 0), (1, 1, 0, 0), (5, 3, 2, 1), (64, 64, 0, 0), (100, 129, 0, 0), (1000, 257, 7, 3), (33, 1000, 0, 0),
    (2049, 70, 0, 0)])
@pytest.mark.parametrize("scaled", [False, True])
def test_columns_in_8_bits(gpu_ctx, dtype, rows, cols, pad, offset, scaled):
    v = normal(rows + cols, rows, cols).to(dtype)
    for i, value in enumerate(SPECIAL):
        if i + 1 < cols and rows:
            v[:, i + 1] = 0 if value < 1 else v[:, i + 1]
            v[(3 * i) % rows, i + 1] = value
    x = place(v, pad, offset)
    m = torch.exp(normal(5, rows)) if scaled else None
    wide = ops.padded(rows)
    q = Guarded(cols, wide, torch.int8, pad, offset)
    scale, sums = torch.full((2, cols + 1), 7.0, device="cuda")
    ready()
    ops.QuantizeColumns(gpu_ctx, x=x.t, q=q.t, scale=scale[:cols], multiplier=m, sums=sums[:cols])()
    ready()
    if rows:
        want_q, want_s = quantize(v.float() * m[:, None] if scaled else v.float(), 0)
    else:
        want_q, want_s = torch.zeros(0, cols, dtype=torch.int8, device="cuda"), torch.zeros(cols, device="cuda")
    assert torch.equal(q.t[:, :rows], want_q.t())
    assert not q.t[:, rows:].any()
    nan = torch.isnan(want_s)
    assert torch.equal(torch.isnan(scale[:cols]), nan) and torch.equal(scale[:cols][~nan], want_s[~nan])
    # a column's sum: chains of at most rows additions
    terms = v.double()
    assert_close(sums[:cols], terms.sum(0), rows * U32 * terms.abs().nan_to_num(0, 0, 0).sum(0), "sums")
    assert q.untouched() and scale[cols] == 7.0 and sums[cols] == 7.0


# ---- product -----------------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 64, 64), (1, 1000, 4096), (2, 17, 100), (5, 4099, 513), (16, 16, 16), (16, 300, 1024),
          (17, 33, 129), (33, 500, 2000), (48, 64, 640), (64, 64, 64), (65, 130, 192), (100, 257, 15), (128, 128, 4096),
          (130, 70, 300), (256, 256, 256), (300, 513, 1000), (513, 300, 128), (1000, 1101, 903), (3, 5, 0),
          (128, 256, 65536 + 100), (9, 40, 140000), (200, 136, 140001)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("layout", [ops.B_CHANNELS, ops.B_INNER])
@pytest.mark.parametrize("pads", [(0, 0, 0), (5, 3, 1), (-1, -1, 8)])
def test_product(gpu_ctx, m, n, k, layout, pads):
    dtype = TYPES[(m + n + k + layout) % 3]
    a = integers(m + k, m, k)
    b = integers(n + k + 1, *((k, n) if layout == ops.B_INNER else (n, k)))
    # -1: rows at the next multiple of 16 bytes, at an aligned address
    pad = [p if p >= 0 else -c % 16 for p, c in zip(pads, (a.shape[1], b.shape[1], 0))]
    offset = 0 if pads[0] < 1 else 3
    A, B = place(a, pad[0], offset), place(b, pad[1], 0 if pads[1] < 1 else 1)
    sa, sb, bias = torch.exp(normal(1, m)), torch.exp(normal(2, n)) / (k + 1), normal(3, n)
    some = (m + n) % 4
    use = dict(a_scale=sa if some != 1 else None, b_scale=sb if some != 2 else None, bias=bias if some != 3 else None)
    out = Guarded(m, n, dtype, pads[2], pads[2])
    ready()
    ops.GemmI8Scaled(gpu_ctx, a=A.t, b=B.t, out=out.t, layout=layout, **use)()
    ready()
    bt = b.double() if layout == ops.B_INNER else b.double().t().contiguous()
    want = a.double() @ bt  # exact: below 2^53
    if use["a_scale"] is not None:
        want = want * sa.double()[:, None]
    if use["b_scale"] is not None:
        want = want * sb.double()
    mag = want.abs()
    if use["bias"] is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    if dtype == torch.float16:
        want = torch.where(want.abs() >= 65520, torch.copysign(torch.full_like(want, float("inf")), want), want)
        near = want.abs().sub(65520).abs() < 1  # at the edge of the type either answer is right
        want, mag = torch.where(near, out.t.double(), want), torch.where(near, torch.zeros_like(mag), mag)
    assert_close(out.t, want, 4 * U32 * mag, "out")
    assert out.untouched()


@pytest.mark.parametrize("m,n", [(1, 40), (40, 33), (200, 136)])
@pytest.mark.parametrize("layout", [ops.B_CHANNELS, ops.B_INNER])
def test_product_of_the_largest_bytes(gpu_ctx, m, n, layout):
    """All -128: the sum passes 2^31 at k = 131072 and has to stay exact."""
    k = 140000
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((k, n) if layout == ops.B_INNER else (n, k), -128, dtype=torch.int8, device="cuda")
    out = torch.empty(m, n, device="cuda")
    ready()
    ops.GemmI8Scaled(gpu_ctx, a=a, b=b, out=out, layout=layout)()
    ready()
    assert (out == float(k * 16384)).all()


def test_product_of_nothing(gpu_ctx):
    e = lambda *s, t=torch.int8: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731
    ops.GemmI8Scaled(gpu_ctx, a=e(0, 5), b=e(7, 5), out=e(0, 7, t=torch.float32))()
    ops.GemmI8Scaled(gpu_ctx, a=e(3, 5), b=e(0, 5), out=e(3, 0, t=torch.float32))()
    ready()


def test_product_carries_nan_scales(gpu_ctx):
    a, b = integers(1, 40, 64), integers(2, 48, 64)
    sa, out = torch.ones(40, device="cuda"), torch.empty(40, 48, device="cuda")
    sa[7], a[7] = float("nan"), 0
    ready()
    ops.GemmI8Scaled(gpu_ctx, a=a, b=b, a_scale=sa, out=out)()
    ready()
    assert torch.isnan(out[7]).all() and not torch.isnan(out[6]).any() and not torch.isnan(out[8:]).any()


# ---- linear layer ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,pad", [
    (1, 1, 1, 0), (1, 256, 1024, 0), (1, 1000, 4100, 3), (7, 64, 77, 1), (16, 129, 512, 0), (40, 512, 1030, 0),
    (64, 256, 256, 0), (70, 300, 130, 0), (300, 257, 640, 16), (530, 130, 1000, 0)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("keep", [False, True])
def test_linear(gpu_ctx, dtype, m, n, k, pad, bias, keep):
    x, w = place(normal(m, m, k).to(dtype), pad, pad), place(integers(n, n, k), pad, pad)
    ws, b = torch.exp(normal(4, n)) / k, normal(5, n) if bias else None
    out = Guarded(m, n, dtype, pad, pad)
    more = {}
    if keep:
        kept, ks = Guarded(m, ops.padded(k), torch.int8), torch.empty(m, device="cuda")
        more = dict(x_q=kept.t, x_scale=ks)
    ready()
    call = ops.LinearI8(gpu_ctx, x=x.t, w=w.t, w_scale=ws, bias=b, out=out.t, **more)
    for _ in range(2):
        call()
    ready()
    q, s = quantize(x.t.float(), 1)
    if keep:
        assert torch.equal(kept.t[:, :k], q) and torch.equal(ks, s) and kept.untouched()
    want = (q.double() @ w.t.double().t().contiguous()) * s.double()[:, None] * ws.double()
    mag = want.abs() + (b.double().abs() if bias else 0)
    assert_close(out.t, want + b.double() if bias else want, 4 * U32 * mag, "out")
    assert out.untouched()


def test_linear_rows_that_are_not_finite(gpu_ctx):
    x, w = normal(1, 20, 96), integers(2, 40, 96)
    x[3, 5], x[4, 0], x[5] = float("inf"), float("nan"), 0.0
    ws, bias, out = torch.ones(40, device="cuda"), normal(3, 40), torch.empty(20, 40, device="cuda")
    ready()
    ops.LinearI8(gpu_ctx, x=x, w=w, w_scale=ws, bias=bias, out=out)()
    ready()
    nan = torch.isnan(out).all(1)
    assert nan.tolist() == [i in (3, 4) for i in range(20)] and not torch.isnan(out[~nan]).any()
    assert torch.equal(out[5], bias)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,pad", [
    (0, 8, 16, 0), (1, 1, 1, 0), (1, 64, 96, 0), (5, 33, 70, 1), (64, 64, 64, 0), (100, 130, 257, 0),
    (300, 257, 129, 5), (513, 256, 512, 0), (1030, 300, 200, 0)])
@pytest.mark.parametrize("wanted", ["all", "dx", "dw", "dbias"])
def test_linear_gradients(gpu_ctx, dtype, m, n, k, pad, wanted):
    dy = place(normal(m + 1, m, n).to(dtype), pad, pad)
    xq, xs = integers(k, m, k, low=-127), torch.exp(normal(6, m))
    w, ws = place(integers(n, n, k), pad, pad), torch.exp(normal(7, n))
    XQ = place(xq, -k % 16)
    dx, dw, db = Guarded(m, k, dtype, pad, pad), Guarded(n, k, torch.float32, pad), torch.full((n,), 9.0, device="cuda")
    outs = {"dx": dx.t, "dw": dw.t, "dbias": db}
    given = outs if wanted == "all" else {wanted: outs[wanted]}
    ready()
    ops.LinearI8Backward(gpu_ctx, dy=dy.t, x_q=XQ.t, x_scale=xs, w=w.t, w_scale=ws, **given)()
    ready()
    d = dy.t.float()
    assert dx.untouched() and dw.untouched()
    if "dx" in given:
        gq, gs = quantize(d * ws, 1)
        want = (gq.double() @ w.t.double()) * gs.double()[:, None]
        assert_close(dx.t, want, 4 * U32 * want.abs(), "dx")
        # against the product's own derivative: half a step for each weight
        true = (dy.t.double() * ws.double()) @ w.t.double()
        slack = 0.5001 * gs.double()[:, None] * w.t.double().abs().sum(0)
        assert_close(dx.t, true, slack, "dx against the derivative")
    if "dw" in given:
        if m:
            hq, hs = quantize(d * xs[:, None], 0)
            want = (hq.double().t().contiguous() @ xq.double()) * hs.double()[:, None]
            true = dy.t.double().t().contiguous() @ (xq.double() * xs.double()[:, None])
            slack = 0.5001 * hs.double()[:, None] * xq.double().abs().sum(0)
            assert_close(dw.t, true, slack, "dw against the derivative")
        else:
            want = torch.zeros(n, k, device="cuda", dtype=torch.float64)
        assert_close(dw.t, want, 4 * U32 * want.abs(), "dw")
    if "dbias" in given:
        assert_close(db, d.double().sum(0), m * U32 * d.double().abs().sum(0), "dbias")


def test_linear_replayed_in_a_graph(gpu_ctx):
    """The layer and its gradients, captured once and replayed on new inputs between eager work."""
    from rns8_amd import hip

    m, n, k = 130, 192, 256
    x, dy = normal(1, m, k), normal(2, m, n)
    w, ws = integers(3, n, k), torch.exp(normal(4, n))
    out, dx, dw, db = (torch.empty(s, device="cuda") for s in ((m, n), (m, k), (n, k), (n,)))
    xq, xs = torch.empty(m, k, dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
    calls = [ops.LinearI8(gpu_ctx, x=x, w=w, w_scale=ws, out=out, x_q=xq, x_scale=xs),
             ops.LinearI8Backward(gpu_ctx, dy=dy, x_q=xq, x_scale=xs, w=w, w_scale=ws, dx=dx, dw=dw, dbias=db)]
    ready()
    stream = hip.stream_create()
    try:
        hip.capture_begin(stream)
        for c in calls:
            c(stream)
        graph, exe = hip.capture_end(stream)
        try:
            for replay in range(3):
                x.copy_(normal(10 + replay, m, k))
                dy.copy_(normal(20 + replay, m, n))
                ready()
                hip.graph_launch(exe, stream)
                hip.stream_synchronize(stream)
                got = [t.clone() for t in (out, dx, dw, db, xq, xs)]
                for t in (out, dx, dw, db):
                    t.zero_()
                ready()
                for c in calls:
                    c()
                ready()
                assert all(torch.equal(a, b) for a, b in zip(got, (out, dx, dw, db, xq, xs)))
        finally:
            hip.graph_destroy(graph, exe)
    finally:
        hip.stream_destroy(stream)


def test_on_a_stream_of_torch(gpu_ctx):
    """On a stream of torch's the operator is ordered with torch's own work, with no synchronization between."""
    if len({line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line}) != 1:
        pytest.skip("torch was loaded after the library: two HIP runtimes, whose streams differ")
    x, w = normal(1, 64, 512), integers(2, 256, 512)
    ws, out = torch.ones(256, device="cuda"), torch.zeros(64, 256, device="cuda")
    call = ops.LinearI8(gpu_ctx, x=x, w=w, w_scale=ws, out=out)
    ready()
    stream, got = torch.cuda.Stream(), []
    with torch.cuda.stream(stream):
        for step in range(3):
            x.mul_(3.0).add_(step)
            call(stream.cuda_stream)
            got.append((x.clone(), out.clone()))
    ready()
    for step, (x, out) in enumerate(got):
        q, s = quantize(x, 1)
        want = (q.double() @ w.double().t().contiguous()) * s.double()[:, None]
        assert_close(out, want, 4 * U32 * want.abs(), f"step {step}")


@pytest.mark.parametrize("what", ["shape", "type", "host", "rows overlap", "workspace", "inner stride"])
def test_refused_before_anything_runs(gpu_ctx, what):
    x, w, ws = normal(1, 8, 64), integers(2, 16, 64), torch.ones(16, device="cuda")
    out = torch.full((8, 16), 5.0, device="cuda")
    args = dict(x=x, w=w, w_scale=ws, out=out)
    if what == "shape":
        args["out"] = out[:, :15]
    if what == "type":
        args["w_scale"] = ws.half()
    if what == "host":
        args["w"] = w.cpu()
    if what == "rows overlap":
        args["x"] = x[:1].expand(8, 64)
    if what == "inner stride":
        args["x"] = normal(1, 64, 8).t()
    if what == "workspace":
        args["workspace"] = torch.empty(16, dtype=torch.uint8, device="cuda")
        call = ops.LinearI8(gpu_ctx, **args)
        ready()
        with pytest.raises(r.Rns8Error) as e:
            call()
        assert e.value.status == r.abi.WORKSPACE_TOO_SMALL
    else:
        with pytest.raises(ValueError):
            ops.LinearI8(gpu_ctx, **args)
    ready()
    assert (out == 5.0).all()
