"""The language-model operators at sizes and arguments at the edge of what they take."""
import pytest
import torch

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


@pytest.mark.parametrize("m", [1, 2, 3, 70])
@pytest.mark.parametrize("k", [15, 64, 8192, 8200])
@pytest.mark.parametrize("keep", [False, True])
def test_a_layer_without_channels(gpu_ctx, m, k, keep):
    """There is no output; rows that are kept are the quantization's own."""
    x, nothing = normal(m + k, m, k).bfloat16(), torch.empty(0, device="cuda")
    more = {}
    if keep:
        kept, scale = Guarded(m, ops.padded(k), torch.int8), torch.empty(m, device="cuda")
        more = dict(x_q=kept.t, x_scale=scale)
    ready()
    ops.LinearI8(gpu_ctx, x=x, w=torch.empty(0, k, dtype=torch.int8, device="cuda"), w_scale=nothing,
                 out=torch.empty(m, 0, dtype=x.dtype, device="cuda"), **more)()
    ready()
    if keep:
        q, s = quantize(x.float(), 1)
        assert torch.equal(kept.t[:, :k], q) and torch.equal(scale, s) and kept.untouched()


def test_on_the_default_stream(gpu_ctx):
    """The handle that torch gives for its default stream: behind torch's work there, and before what follows."""
    if len({line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line}) != 1:
        pytest.skip("torch was loaded after the library: two HIP runtimes, whose streams differ")
    handle = torch.cuda.current_stream().cuda_stream
    assert handle == 0
    big = torch.randn(8192, 8192, device="cuda")
    x, scale = torch.zeros(300, 512, device="cuda"), torch.zeros(300, device="cuda")
    call = ops.QuantizeRows(gpu_ctx, x=x, q=torch.empty(300, 512, dtype=torch.int8, device="cuda"), scale=scale)
    big @ big
    ready()
    got = []
    for value in (3.0, 5.0, 7.0):
        for _ in range(4):  # some milliseconds
            big @ big
        x.fill_(value)
        call(handle)
        got.append(scale.clone())
    ready()
    for value, scale in zip((3.0, 5.0, 7.0), got):
        assert torch.equal(scale, torch.full_like(scale, value) / torch.full_like(scale, 127.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset,scale", [(0, 1.0), (50, 1.0), (100, 1.0), (1000, 1.0), (-1000, 0.5), (2000, 2.0),
                                          (4000, 1.0), (-4000, 1.0), (100000, 1.0)])
@pytest.mark.parametrize("rows,vocab", [(40, 1000), (3, 50001)])
@pytest.mark.parametrize("in_place", [False, True])
def test_gradient_of_logits_on_a_common_offset(gpu_ctx, dtype, offset, scale, rows, vocab, in_place):
    """An offset that all logits of a row share changes no probability, so it is no excuse for an error.

    With D = max |z - max z| and L = max -log p of a row, an exponential's argument is off by 2^-24 (4 (D + L)), lse by
    32 of these units at most where the row is not summed again (|lse| <= 64), the sum and its logarithm by 512."""
    v = (2.5 / scale * normal(rows, rows, vocab) + offset / scale).to(dtype)
    v[:, 7] = v.amax(1) + 1 / scale
    targets = torch.arange(rows, device="cuda")
    targets[1] = 7
    gl, ge = normal(3, rows), normal(4, rows)
    out = {k: torch.empty(rows, device="cuda") for k in ("logp", "entropy", "lse")}
    d, e_ = v.clone(), v.clone()
    ready()
    ops.TokenLogprobs(gpu_ctx, logits=v, targets=targets, scale=scale, **out)()
    more = dict(lse=out["lse"], scale=scale)
    ops.TokenLogprobsBackward(gpu_ctx, logits=d if in_place else v, targets=targets, dlogp=gl, dlogits=d, **more)()
    ops.TokenLogprobsBackward(gpu_ctx, logits=e_ if in_place else v, entropy=out["entropy"], dentropy=ge, dlogits=e_,
                              **more)()
    ready()
    z = v.double() * float(torch.tensor(scale))
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    entropy = -(p * logp).sum(1)
    size = (z.amax(1) - z.amin(1))[:, None]
    off = U32 * (4 * (size - logp.amin(1, keepdim=True)) + 32 + 512)
    given = logp.gather(1, targets[:, None])[:, 0]
    assert_close(out["logp"], given, off[:, 0], "logp")
    assert_close(out["entropy"], entropy, (2 * off * (1 + size))[:, 0], "entropy")
    want = -scale * gl.double()[:, None] * p
    slack = off * want.abs()
    hit = torch.zeros_like(p).scatter_(1, targets[:, None], 1.0)
    want, slack = want + scale * gl.double()[:, None] * hit, slack + 2 * U32 * scale * gl.double().abs()[:, None] * hit
    assert_close(d, want, slack, "dlogits of logp")
    terms = scale * ge.double().abs()[:, None] * p
    want = -scale * ge.double()[:, None] * p * (logp + entropy[:, None])
    assert_close(e_, want, terms * (off * (logp.abs() + entropy[:, None]) + 2 * off * (2 + size)), "dlogits of entropy")
    if dtype == torch.float32:  # what the target gains the others lose
        assert (d.double().sum(1).abs() <= scale * gl.double().abs() * (off[:, 0] + 4 * U32)).all()


@pytest.mark.parametrize("rows,cols", [(2**28 + 1000, 1), (2**30 + 1000, 1), (2, 2**24 + 50), (1, 2**28 + 50)])
def test_columns_past_the_workgroups_of_a_launch(gpu_ctx, rows, cols):
    """As many tiles, or strips of whole columns, as take more than one launch; whole numbers add up exactly in 32 bits."""
    x = torch.randint(-7, 8, (rows, cols), device="cuda", dtype=torch.int8)
    if cols == 1:
        x[::2, 0] = -x[1::2, 0]
        x[12345, 0], x[12344, 0] = 127, -127
    v = x.half()
    q = torch.full((cols, rows), 99, dtype=torch.int8, device="cuda")
    scale, sums = torch.empty(2, cols, device="cuda")
    ready()
    ops.QuantizeColumns(gpu_ctx, x=v, q=q, scale=scale, sums=sums)()
    ready()
    assert torch.equal(sums, x.sum(0).float())
    if cols == 1:
        assert scale.item() == 1.0 and torch.equal(q[0], x[:, 0])
    else:
        want, want_scale = quantize(v.float(), 0)
        assert torch.equal(scale, want_scale) and torch.equal(q, want.t())


@pytest.mark.parametrize("weight", [1.0, 2.0 ** 30, -(2.0 ** 66), 2.0 ** 116])
def test_large_weights_of_the_entropy_beside_masks(gpu_ctx, weight):
    """A ruled-out token gets 0 whatever the weight is; the others' gradients grow with it (a power of two times those of 1)."""
    v = normal(1, 5, 3000)
    v[:, ::3], v[1, 1::3], v[2, 4] = -float("inf"), torch.finfo(torch.float32).min, -500.0
    lse, entropy = torch.empty(2, 5, device="cuda")
    ready()
    ops.TokenLogprobs(gpu_ctx, logits=v, lse=lse, entropy=entropy)()
    got = []
    for w in (1.0, weight):
        d, g = torch.empty_like(v), torch.full((5,), w, device="cuda")
        ready()
        ops.TokenLogprobsBackward(gpu_ctx, logits=v, lse=lse, entropy=entropy, dentropy=g, dlogits=d)()
        ready()
        got.append(d)
    none = torch.softmax(v.double(), 1) < 2.0 ** -150
    assert none[:, ::3].all() and none[1, 1::3].all() and none[2, 4]
    assert not got[1][none].any()
    # (values that are denormal for a weight of 1 have lost digits that they keep for a large one)
    normal_ones = got[0].abs() > 2.0 ** -126
    assert torch.equal(got[1][normal_ones], got[0][normal_ones] * weight)


@pytest.mark.parametrize("size", [1e-18, 1e-15, 1e-13, 1e-10, 1.0, 1e10, 1e13, 1e14, 1e15, 1e17])
@pytest.mark.parametrize("flags", [ops.NORM_POST, ops.NORM_PRE])
@pytest.mark.parametrize("rows,cols", [(5, 200), (40, 5000)])
def test_norm_gradients_of_rows_of_any_size(gpu_ctx, size, flags, rows, cols):
    """Rows whose squares 32 bits hold: r, but not its cube. With n = x r, each of
    dx = r (w d - n mean(w d n)) and dw = sum d n is off by 128 (over rows 256) units of its terms, as any norm's gradients."""
    x, d, w = size * normal(1, rows, cols), normal(2, rows, cols), 1 + 0.3 * normal(3, cols)
    rstd, h, y, dx = torch.empty(2, rows, device="cuda"), *torch.empty(3, rows, cols, device="cuda")
    dw = torch.empty(cols, device="cuda")
    pre = flags == ops.NORM_PRE
    given = dict(x=x, flags=flags, eps=0.0, **({"pre_weight": w} if pre else {"post_weight": w}))
    ready()
    ops.BlockNorm(gpu_ctx, **given, h=h, y=y if pre else None, rstd=rstd)()
    ops.BlockNormBackward(gpu_ctx, **given, rstd=rstd, dx=dx, **(dict(dy=d, dpre_weight=dw) if pre else
                                                                 dict(dh=d, dpost_weight=dw)))()
    ready()
    r = x.double().square().mean(1, keepdim=True).rsqrt()
    n, wd = x.double() * r, w.double() * d.double()
    assert_close(dx, r * (wd - n * (wd * n).mean(1, keepdim=True)),
                 128 * U32 * r * (wd.abs() + n.abs() * (wd * n).abs().mean(1, keepdim=True)), "dx")
    terms = d.double() * n
    assert_close(dw, terms.sum(0), 256 * U32 * terms.abs().sum(0), "dw")


@pytest.mark.parametrize("flags", [0, ops.NORM_POST])
@pytest.mark.parametrize("cols", [100, 9000])
def test_gradients_past_infinite_values_that_no_norm_reads(gpu_ctx, flags, cols):
    """Without a norm of h, dresidual is residual_scale dh, and without one of x, dx is branch_scale gate dh: whatever the
    block's output and the residual hold."""
    x, res, gate, dh = (normal(i, 6, cols) for i in range(4))
    x[1, 3], x[2, 7], res[3, 5], res[4, 6] = float("inf"), float("nan"), -float("inf"), float("nan")
    rstd, h, dx, dres = torch.empty(2, 6, device="cuda"), *torch.empty(3, 6, cols, device="cuda")
    given = dict(x=x, residual=res, gate=gate, flags=flags, branch_scale=0.5, residual_scale=4.0)
    ready()
    ops.BlockNorm(gpu_ctx, **given, h=h, rstd=rstd)()
    ops.BlockNormBackward(gpu_ctx, **given, rstd=rstd, dh=dh, dx=dx, dresidual=dres)()
    ready()
    assert torch.equal(dres, 4.0 * dh)
    if not flags:
        assert torch.equal(dx, 0.5 * gate * dh)
    else:
        assert torch.isnan(dx).any(1).tolist() == [False, True, True, False, False, False]


# kept rows of the quantized activations: next to each other, at an odd address, with room for some of the zeros, and
# at a stride of whole 16 bytes from an address that is none
KEPT = [(0, 0), (0, 3), (5, 1), (None, 5)]


def kept_rows(values, m, k, pad, offset):
    pad = -k % 16 if pad is None else pad
    kept = Guarded(m, k, torch.int8, pad, offset, -99)
    if values is not None:
        kept.t.copy_(values)
        kept.was = kept.buf.clone()
    return kept


@pytest.mark.parametrize("m,n,k", [(1, 300, 1000), (2, 40, 70), (17, 300, 1000), (48, 130, 77), (64, 8200, 129),
                                   (70, 300, 130), (300, 257, 641), (530, 130, 1000), (300, 64, 15)])
@pytest.mark.parametrize("pad,offset", KEPT)
@pytest.mark.parametrize("w_pad", [0, 3])
def test_layers_that_keep_rows_at_any_alignment(gpu_ctx, m, n, k, pad, offset, w_pad):
    """A product's sum is exact: its scales and bias are three 32-bit operations, and the rounding of the sum one more."""
    dtype = TYPES[(m + k) % 3]
    x, w = normal(m, m, k).to(dtype), place(integers(n, n, k), w_pad, w_pad)
    ws, bias = torch.exp(normal(4, n)) / k, normal(5, n)
    kept, scale, out = kept_rows(None, m, k, pad, offset), torch.empty(m, device="cuda"), Guarded(m, n, dtype)
    ready()
    ops.LinearI8(gpu_ctx, x=x, w=w.t, w_scale=ws, bias=bias, out=out.t, x_q=kept.t, x_scale=scale)()
    ready()
    q, s = quantize(x.float(), 1)
    stop = min(kept.ld, ops.padded(k))
    rows = torch.as_strided(kept.buf, (m, stop), (kept.ld, 1), kept.at)
    assert torch.equal(rows[:, :k], q) and not rows[:, k:].any() and torch.equal(scale, s) and kept.untouched(stop)
    want = (q.double() @ w.t.double().t().contiguous()) * s.double()[:, None] * ws.double()
    assert_close(out.t, want + bias.double(), 4 * U32 * (want.abs() + bias.double().abs()), "out")
    assert out.untouched()


@pytest.mark.parametrize("m,n,k", [(1, 64, 97), (5, 33, 70), (100, 130, 257), (300, 257, 129), (513, 256, 520),
                                   (1030, 300, 200), (70, 40, 15)])
@pytest.mark.parametrize("pad,offset", KEPT)
@pytest.mark.parametrize("wanted", ["all", "dw"])
def test_gradients_from_kept_rows_at_any_alignment(gpu_ctx, m, n, k, pad, offset, wanted):
    """As the layer: exact sums, and the quantized gradients' own bytes and scales."""
    dtype = TYPES[(m + n) % 3]
    dy, xq, xs = normal(m + 1, m, n).to(dtype), integers(k, m, k), torch.exp(normal(6, m))
    w, ws, kept = place(integers(n, n, k), 1, 1), torch.exp(normal(7, n)), kept_rows(xq, m, k, pad, offset)
    dx, dw, db = Guarded(m, k, dtype), Guarded(n, k, torch.float32), torch.full((n,), 9.0, device="cuda")
    more = dict(dx=dx.t, dbias=db) if wanted == "all" else {}
    ready()
    ops.LinearI8Backward(gpu_ctx, dy=dy, x_q=kept.t, x_scale=xs, w=w.t, w_scale=ws, dw=dw.t, **more)()
    ready()
    d = dy.float()
    hq, hs = quantize(d * xs[:, None], 0)
    want = (hq.double().t().contiguous() @ xq.double()) * hs.double()[:, None]
    assert_close(dw.t, want, 4 * U32 * want.abs(), "dw")
    if wanted == "all":
        gq, gs = quantize(d * ws, 1)
        want = (gq.double() @ w.t.double()) * gs.double()[:, None]
        assert_close(dx.t, want, 4 * U32 * want.abs(), "dx")
        assert_close(db, d.double().sum(0), m * U32 * d.double().abs().sum(0), "dbias")
    assert kept.untouched() and dx.untouched() and dw.untouched()
    assert torch.equal(kept.t, xq)
