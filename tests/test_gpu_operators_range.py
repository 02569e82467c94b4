"""The language-model operators where their forms change and where offsets are large.

Products of few tokens with wide and narrow outputs, columns on both sides of
the lengths at which they are taken whole, launches that move enough for
their stores to pass the caches, and rows whose offsets pass 2^31 and 2^32
elements. Tolerances are those of the operators' own tests: a product's sum is
exact, so it is off by 4 * 2^-24 of itself and the output's rounding; others
are stated where they are used.
"""
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
    torch.cuda.synchronize()


def product(q, w):
    return q.double() @ w.double().t().contiguous()


@pytest.mark.parametrize("m", [2, 3, 15, 16, 17, 32, 33, 48, 49, 63, 64, 65])
@pytest.mark.parametrize("n,k,pad", [(40, 1000, 0), (300, 2048, 0), (1025, 4093, 3), (8192, 512, 0), (8200, 1031, 16),
                                     (16400, 70, 5)])
@pytest.mark.parametrize("keep", [False, True])
def test_few_tokens(gpu_ctx, m, n, k, pad, keep):
    dtype = TYPES[(m + n) % 3]
    x, w = place(normal(m, m, k).to(dtype), pad, pad), place(integers(n, n, k), pad, pad)
    ws, bias = torch.exp(normal(4, n)) / k, normal(5, n)
    out = Guarded(m, n, dtype, pad, pad)
    more = {}
    if keep:
        more = dict(x_q=torch.empty(m, ops.padded(k), dtype=torch.int8, device="cuda"), x_scale=torch.empty(m, device="cuda"))
    ready()
    ops.LinearI8(gpu_ctx, x=x.t, w=w.t, w_scale=ws, bias=bias, out=out.t, **more)()
    ready()
    q, s = quantize(x.t.float(), 1)
    want = product(q, w.t) * s.double()[:, None] * ws.double()
    assert_close(out.t, want + bias.double(), 4 * U32 * (want.abs() + bias.double().abs()), "out")
    assert out.untouched()
    # the same bytes from the two calls that it stands for
    apart = torch.empty_like(out.t)
    ready()
    ops.GemmI8Scaled(gpu_ctx, a=q, b=w.t, a_scale=s, b_scale=ws, bias=bias, out=apart)()
    ready()
    assert torch.equal(apart, out.t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [511, 512, 513, 1023, 1025])
@pytest.mark.parametrize("cols,pad", [(31, 0), (32, 0), (33, 1), (200, 0), (1000, 8)])
def test_columns_where_the_form_changes(gpu_ctx, dtype, rows, cols, pad):
    x = place(normal(rows + cols, rows, cols).to(dtype), pad)
    m = torch.exp(normal(5, rows))
    q = Guarded(cols, ops.padded(rows), torch.int8, pad)
    scale, sums = torch.empty(2, cols, device="cuda")
    ready()
    ops.QuantizeColumns(gpu_ctx, x=x.t, q=q.t, scale=scale, multiplier=m, sums=sums)()
    ready()
    want_q, want_s = quantize(x.t.float() * m[:, None], 0)
    assert torch.equal(q.t[:, :rows], want_q.t()) and not q.t[:, rows:].any() and q.untouched()
    assert torch.equal(scale, want_s)
    terms = x.t.double()
    assert_close(sums, terms.sum(0), rows * U32 * terms.abs().sum(0), "sums")


def test_norms_of_a_launch_past_the_caches(gpu_ctx):
    """300 MB and more in one call; a sum of 4096 squares is off by at most 4096 * 2^-24 of itself, its root by half."""
    rows, cols = 9001, 4096
    x, res = normal(1, rows, cols).bfloat16(), normal(2, rows, cols).bfloat16()
    h, y = torch.empty_like(x), torch.empty_like(x)
    rstd = torch.empty(2, rows, device="cuda")
    dy, dx, dres = normal(3, rows, cols).bfloat16(), torch.empty_like(x), torch.empty_like(x)
    ready()
    ops.BlockNorm(gpu_ctx, x=x, residual=res, h=h, y=y, rstd=rstd)()
    ops.BlockNormBackward(gpu_ctx, x=x, residual=res, rstd=rstd, dy=dy, dx=dx, dresidual=dres)()
    ready()
    part = slice(0, rows, 97)
    xs = x[part].double().requires_grad_()
    rs = res[part].double().requires_grad_()
    f = xs * (xs.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    hs = rs + f
    ys = hs * (hs.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    ys.backward(dy[part].double())
    e = 4096 * U32
    assert_close(h[part], hs.detach(), e * (hs.detach().abs() + f.detach().abs()), "h")
    assert_close(y[part], ys.detach(), 2 * e * (ys.detach().abs() + f.detach().abs()), "y")
    size = dy[part].double().abs().mean(1, keepdim=True) * 8
    assert_close(dres[part], rs.grad, 4 * e * (rs.grad.abs() + size), "dresidual")
    assert_close(dx[part], xs.grad, 8 * e * (xs.grad.abs() + size), "dx")


def test_gradient_of_logits_past_the_caches(gpu_ctx):
    """420 MB in one call, against the same rows in small calls: every value has one way to be computed."""
    rows, vocab = 2100, 50001
    v = normal(1, rows, vocab).half()
    targets = torch.randint(vocab, (rows,), device="cuda")
    lse, entropy, gl = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), normal(2, rows)
    d = torch.empty_like(v)
    ready()
    ops.TokenLogprobs(gpu_ctx, logits=v, lse=lse, entropy=entropy)()
    ops.TokenLogprobsBackward(gpu_ctx, logits=v, lse=lse, targets=targets, dlogp=gl, dlogits=d)()
    ready()
    for i in (0, 1049, 2099):
        one = torch.empty(1, vocab, dtype=v.dtype, device="cuda")
        ready()
        ops.TokenLogprobsBackward(gpu_ctx, logits=v[i:i + 1], lse=lse[i:i + 1], targets=targets[i:i + 1],
                                  dlogp=gl[i:i + 1], dlogits=one)()
        ready()
        assert torch.equal(one[0], d[i])
        z = v[i].double()
        p = torch.softmax(z, 0)
        want = -gl[i].double() * p
        want[targets[i]] += gl[i].double()
        # exp: 2^-23 (|z| + |lse|) + 4 units of itself; lse: 512 units at most
        slack = gl[i].double().abs() * p * U32 * (4 * (z.abs().max() + lse[i].double().abs()) + 1024)
        assert_close(d[i], want, slack + U32 * want.abs(), f"row {i}")


FAR = 2**31 + 64  # row stride: rows 1 and 2 lie past 2^31 and 2^32 elements


def far(values):
    """`values`, at most three rows, FAR apart."""
    rows, cols = values.shape
    t = torch.as_strided(torch.empty((rows - 1) * FAR + cols, dtype=values.dtype, device="cuda"), (rows, cols), (FAR, 1))
    t.copy_(values)
    return t


def test_far_rows_of_logits(gpu_ctx):
    v = normal(1, 3, 5000).bfloat16()
    targets = torch.tensor([1, 4999, 70], device="cuda")

    def results(logits, dlogits):
        out = {k: torch.empty(3, device="cuda") for k in ("logp", "entropy", "lse")}
        out |= dict(top_ids=torch.empty(3, 5, dtype=torch.int32, device="cuda"), top_logp=torch.empty(3, 5, device="cuda"))
        ready()
        ops.TokenLogprobs(gpu_ctx, logits=logits, targets=targets, **out)()
        ops.TokenLogprobsBackward(gpu_ctx, logits=logits, lse=out["lse"], entropy=out["entropy"], targets=targets,
                                  dlogp=torch.ones(3, device="cuda"), dentropy=torch.ones(3, device="cuda"),
                                  dlogits=dlogits)()
        ready()
        return [*out.values(), dlogits.clone()]

    near = results(v, torch.empty_like(v))
    assert all(torch.equal(a, b) for a, b in zip(near, results(far(v), far(torch.zeros_like(v)))))


def test_far_rows_of_a_norm(gpu_ctx):
    x, g, dy = (normal(i, 3, 1000).half() for i in range(3))

    def results(put):
        x_, g_, dy_ = put(x), put(g), put(dy)
        h, y, dx, dg = (put(torch.zeros_like(x)) for _ in range(4))
        rstd = torch.empty(2, 3, device="cuda")
        ready()
        ops.BlockNorm(gpu_ctx, x=x_, residual=dy_, gate=g_, h=h, y=y, rstd=rstd)()
        ops.BlockNormBackward(gpu_ctx, x=x_, residual=dy_, gate=g_, rstd=rstd, dy=dy_, dx=dx, dgate=dg)()
        ready()
        return [t.clone() for t in (h, y, dx, dg, rstd)]

    assert all(torch.equal(a, b) for a, b in zip(results(lambda t: t.clone()), results(far)))


def test_far_rows_of_a_linear_layer(gpu_ctx):
    """Activations and results far apart, and 8-bit rows at the longest stride: their offsets pass 2^32 bytes."""
    n, k, ld = 600, 64, 2**23 - 16
    x, w, ws = normal(1, 3, k).bfloat16(), integers(2, n, k), torch.exp(normal(3, n))
    spread = torch.as_strided(torch.empty((n - 1) * ld + k, dtype=torch.int8, device="cuda"), (n, k), (ld, 1))
    spread.copy_(w)
    near, away = torch.empty(3, n, dtype=x.dtype, device="cuda"), far(torch.zeros(3, n, device="cuda").bfloat16())
    dnear, daway = torch.empty(3, k, dtype=x.dtype, device="cuda"), far(torch.zeros(3, k, device="cuda").bfloat16())
    ready()
    ops.LinearI8(gpu_ctx, x=x, w=w, w_scale=ws, out=near)()
    ops.LinearI8(gpu_ctx, x=far(x), w=spread, w_scale=ws, out=away)()
    ops.LinearI8Backward(gpu_ctx, dy=near, w=w, w_scale=ws, dx=dnear)()
    ops.LinearI8Backward(gpu_ctx, dy=away, w=spread, w_scale=ws, dx=daway)()
    ready()
    assert torch.equal(near, away) and torch.equal(dnear, daway)
    # many rows of 8-bit operands on both sides of a tiled product
    out = torch.empty(n, n, device="cuda")
    for b, layout in ((spread, ops.B_CHANNELS), (w.t().contiguous(), ops.B_INNER)):
        ready()
        ops.GemmI8Scaled(gpu_ctx, a=spread, b=b, out=out, layout=layout)()
        ready()
        assert torch.equal(out.double(), product(w, w))


@pytest.mark.parametrize("what", ["norm x", "norm residual", "logits"])
def test_in_place_at_other_strides_is_refused(gpu_ctx, what):
    import rns8_amd as r

    buf = torch.zeros(4, 96, device="cuda")
    one, other = buf[:3, :64], torch.as_strided(buf, (3, 64), (80, 1))
    more, f = torch.zeros(3, 64, device="cuda"), torch.zeros(3, device="cuda")
    ready()
    with pytest.raises(r.Rns8Error) as e:
        if what == "norm x":
            ops.BlockNorm(gpu_ctx, x=one, h=other, y=more)()
        elif what == "norm residual":
            ops.BlockNorm(gpu_ctx, x=more, residual=one, h=other, y=torch.zeros_like(more))()
        else:
            ops.TokenLogprobsBackward(gpu_ctx, logits=one, lse=f, targets=f.long(), dlogp=f, dlogits=other)()
    assert e.value.status == r.abi.INVALID_ARGUMENT
