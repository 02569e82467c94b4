"""4-bit microscaled matrices on the GPU: rounding and back, products, linear layers and their gradients."""
import pytest
import torch

import mx4_cases as mx4
from operator_cases import TYPES, UNIT, Guarded, assert_close, place
from rns8_amd import operators as ops

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def ready():
    torch.cuda.synchronize()  # the library's stream does not wait for torch's


def empty_mx4(rows, cols, fill=0xAB):
    """A matrix's bytes between two guards."""
    buf = torch.full((ops.mx4_bytes(rows, cols) + 128,), fill, dtype=torch.uint8, device="cuda")
    return buf, buf[64:-64]


def guards_kept(buf, fill=0xAB):
    return bool((buf[:64] == fill).all() and (buf[-64:] == fill).all())


def awkward(seed, rows, cols, dtype):
    """Rows whose blocks differ in size by many powers of two, with ties, zeros, the smallest and largest values."""
    x = normal(seed, rows, cols)
    size = torch.randint(-14, 14, (rows, (cols + 31) // 32), generator=torch.Generator(device="cuda").manual_seed(seed + 1),
                         device="cuda")
    x = torch.ldexp(x, size.repeat_interleave(32, 1)[:, :cols])
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9375, -0.0, -0.25, -5.0], device="cuda")
    x[::3, :13] = ties[:min(13, cols)]
    x[1::5, :64] = 0.0
    x[2::7, 32:64] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps * 3  # below the normal values
    x[3::7, 64:70] = torch.finfo(dtype).max
    return x.to(dtype)


SHAPES = [(1, 1), (1, 32), (2, 31), (16, 256), (17, 257), (15, 1000), (130, 515), (257, 96), (300, 7), (512, 1024)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (5, 3)])
def test_rounding(gpu_ctx, dtype, rows, cols, pad, offset):
    """The bytes of both forms, in one call and in two, zeros past the matrix with them."""
    x = place(awkward(rows + cols, rows, cols, dtype), pad, offset)
    want, _ = mx4.matrix(x.t)
    want_t, _ = mx4.matrix(x.t.t())
    for both in (True, False):
        buf, q = empty_mx4(rows, cols)
        buf_t, q_t = empty_mx4(cols, rows)
        ready()
        if both:
            ops.QuantizeMx4(gpu_ctx, x=x.t, q=q, q_t=q_t)()
        else:
            ops.QuantizeMx4(gpu_ctx, x=x.t, q=q)()
            ops.QuantizeMx4(gpu_ctx, x=x.t, q_t=q_t)()
        ready()
        assert torch.equal(q, want) and guards_kept(buf)
        assert torch.equal(q_t, want_t) and guards_kept(buf_t)
        assert x.untouched()


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_that_are_not_finite(gpu_ctx, dtype):
    x = normal(1, 40, 300).to(dtype)
    x[3, 5], x[3, 40], x[20, 299], x[39, 0] = float("nan"), float("inf"), -float("inf"), float("nan")
    want, values = mx4.matrix(x)
    want_t, _ = mx4.matrix(x.t())
    (_, q), (_, q_t) = empty_mx4(40, 300), empty_mx4(300, 40)
    back = torch.empty(40, 300, device="cuda")
    ready()
    ops.QuantizeMx4(gpu_ctx, x=x, q=q, q_t=q_t)()
    ops.DequantizeMx4(gpu_ctx, q=q, out=back)()
    ready()
    assert torch.equal(q, want) and torch.equal(q_t, want_t)
    assert torch.isnan(back[3, :64]).all() and torch.isnan(back[20, 288:]).all() and torch.isnan(back[39, :32]).all()
    assert torch.isnan(back).sum() == 64 + 12 + 32
    assert_close(back, values, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_back_to_values(gpu_ctx, dtype, rows, cols):
    """Every value that a matrix holds; a second rounding changes none of them."""
    q, values = mx4.matrix(awkward(rows, rows, cols, torch.float32))
    out = Guarded(rows, cols, dtype, pad=3, offset=1)
    full = torch.empty(rows, cols, device="cuda")
    _, again = empty_mx4(rows, cols)
    once_more = torch.empty(rows, cols, device="cuda")
    ready()
    ops.DequantizeMx4(gpu_ctx, q=q, out=out.t)()
    ops.DequantizeMx4(gpu_ctx, q=q, out=full)()
    ops.QuantizeMx4(gpu_ctx, x=full, q=again)()
    ops.DequantizeMx4(gpu_ctx, q=again, out=once_more)()
    ready()
    assert torch.equal(full.double(), values)
    assert torch.equal(out.t, full.to(dtype)) and out.untouched()
    assert torch.equal(once_more, full)


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_packing_of_rows(gpu_ctx, rows, cols):
    """All codes and all scales, at any stride; the half byte after an odd row's end is not taken."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    blocks = (cols + 31) // 32
    code = torch.randint(0, 16, (rows, blocks * 32), generator=g, device="cuda")
    scale = torch.randint(0, 256, (rows, blocks), generator=g, device="cuda")
    data = place((code[:, ::2] | code[:, 1::2] << 4)[:, :(cols + 1) // 2].to(torch.uint8).view(torch.int8), 3, 1)
    exponents = place(scale.to(torch.uint8).view(torch.int8), 2, 5)
    code[:, cols:] = 0
    buf, q = empty_mx4(rows, cols)
    ready()
    ops.PackMx4(gpu_ctx, data=data.t.view(torch.uint8), scale=exponents.t.view(torch.uint8), q=q, cols=cols)()
    ready()
    assert torch.equal(q, mx4.buffer_of(code.reshape(rows, blocks, 32), scale, cols)) and guards_kept(buf)


PRODUCTS = [(1, 1, 1), (1, 40, 300), (5, 17, 256), (16, 8200, 512), (17, 100, 777), (33, 64, 4096), (48, 130, 1000),
            (64, 300, 2048), (65, 64, 256), (70, 500, 300), (128, 128, 4096), (130, 257, 1300), (300, 1101, 903),
            (513, 300, 2100), (1000, 700, 64), (1030, 1300, 513), (2048, 2048, 512)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("bias", [False, True])
def test_products_are_exact_where_32_bits_hold_the_sums(gpu_ctx, m, n, k, bias):
    """Sums of multiples of 2^-4 below 2^20, in whatever order: not a bit is lost before the output's rounding."""
    (a, av), (b, bv) = mx4.exact_matrix(m, m, k), mx4.exact_matrix(n + 7, n, k)
    want = torch.mm(av, bv.t().contiguous())
    vector = torch.randint(-64, 64, (n,), device="cuda").float() if bias else None
    if bias:
        want = want + vector
    for dtype, pad in ((torch.float32, 0), (torch.bfloat16, 5), (torch.float16, 1)):
        out = Guarded(m, n, dtype, pad=pad, offset=pad)
        ready()
        ops.GemmMx4(gpu_ctx, a=a, b=b, k=k, out=out.t, bias=vector)()
        ready()
        assert torch.equal(out.t, want.float().to(dtype)) and out.untouched()


def product_limit(a, b, k):
    """|error| of k products added in 32 bits, each addition off by at most one step (2^-23) of a sum below sum |a b|,
    and up to 64 more additions of partial sums and a bias."""
    return (k + 64) * 2.0 ** -23 * torch.mm(a.abs(), b.abs().t().contiguous())


@pytest.mark.parametrize("m,n,k", [(3, 50, 700), (40, 60, 5000), (200, 300, 9000)])
def test_products_of_blocks_of_any_size(gpu_ctx, m, n, k):
    a, av = mx4.matrix(awkward(1, m, k, torch.bfloat16).clamp(-1e6, 1e6))
    b, bv = mx4.matrix(awkward(2, n, k, torch.bfloat16).clamp(-1e6, 1e6))
    out = torch.empty(m, n, device="cuda")
    ready()
    ops.GemmMx4(gpu_ctx, a=a, b=b, k=k, out=out)()
    ready()
    assert_close(out, torch.mm(av, bv.t().contiguous()), product_limit(av, bv, k))


@pytest.mark.parametrize("m", [3, 40, 200])
def test_products_with_blocks_that_are_not_finite(gpu_ctx, m):
    """A block without a finite scale makes its row of the result NaN, or its column, and nothing else."""
    x, w = normal(1, m, 600), normal(2, 90, 600)
    x[2, 599], w[33, 0] = float("nan"), float("inf")
    (a, av), (b, bv) = mx4.matrix(x), mx4.matrix(w)
    out = torch.empty(m, 90, device="cuda")
    ready()
    ops.GemmMx4(gpu_ctx, a=a, b=b, k=600, out=out)()
    ready()
    bad = torch.isnan(out)
    assert bad[2].all() and bad[:, 33].all() and bad.sum() == 90 + m - 1
    assert_close(out, torch.mm(av, bv.t().contiguous()), product_limit(av.nan_to_num(), bv.nan_to_num(), 600))


def test_sums_of_nothing(gpu_ctx):
    nothing = torch.empty(0, dtype=torch.uint8, device="cuda")
    bias = normal(3, 70)
    for m in (1, 64, 300):
        out, zeros = torch.empty(m, 70, device="cuda"), torch.full((m, 70), 7.0, dtype=torch.bfloat16, device="cuda")
        ready()
        ops.GemmMx4(gpu_ctx, a=nothing, b=nothing, k=0, out=out, bias=bias)()
        ops.GemmMx4(gpu_ctx, a=nothing, b=nothing, k=0, out=zeros)()
        ready()
        assert torch.equal(out, bias.expand(m, -1)) and not zeros.any()
    ops.GemmMx4(gpu_ctx, a=nothing, b=mx4.matrix(normal(1, 70, 40))[0], k=40, out=torch.empty(0, 70, device="cuda"))()
    ready()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 70, 33), (1, 8200, 1000), (2, 64, 8192), (16, 300, 515), (17, 300, 515),
                                   (64, 1000, 700), (65, 33, 64), (300, 200, 1101)])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_layers(gpu_ctx, dtype, m, n, k, bias):
    x = place(normal(m, m, k).to(dtype), 3, 1)
    x.t[0, :3] *= 40
    w, wv = mx4.matrix(normal(n, n, k))
    _, xv = mx4.matrix(x.t)
    vector = normal(5, n) if bias else None
    out = Guarded(m, n, dtype, pad=2, offset=3)
    ready()
    ops.LinearMx4(gpu_ctx, x=x.t, w=w, bias=vector, out=out.t)()
    ready()
    want = torch.mm(xv, wv.t().contiguous()) + (vector.double() if bias else 0.0)
    limit = product_limit(xv, wv, k) + (vector.abs().double() * 2.0 ** -23 if bias else 0.0)
    assert_close(out.t, want, limit)
    assert out.untouched() and x.untouched()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 40, 50), (33, 64, 300), (70, 35, 118), (500, 701, 611), (1300, 100, 257)])
def test_gradients_of_linear_layers(gpu_ctx, dtype, m, n, k):
    """Against the formulas; all at once and each by itself."""
    dy, x = place(normal(m, m, n).to(dtype), 1, 1), place(normal(k, m, k).to(dtype), 2, 5)
    w = normal(n, n, k)
    w_t, wv = mx4.matrix(w.t())
    _, gv = mx4.matrix(dy.t)
    _, gtv = mx4.matrix(dy.t.t())
    _, xtv = mx4.matrix(x.t.t())
    want_dx, want_dw, want_db = torch.mm(gv, wv.t().contiguous()), torch.mm(gtv, xtv.t().contiguous()), dy.t.double().sum(0)
    for wanted in ({"dx", "dw", "dbias"}, {"dx"}, {"dw"}, {"dbias"}, {"dx", "dbias"}):
        dx, dw = Guarded(m, k, dtype, pad=3, offset=1), Guarded(n, k, torch.float32, pad=1, offset=2)
        db = torch.empty(n, device="cuda")
        given = {"dx": dict(dx=dx.t, w_t=w_t), "dw": dict(dw=dw.t, x=x.t), "dbias": dict(dbias=db)}
        more = {}
        for name in wanted:
            more |= given[name]
        ready()
        ops.LinearMx4Backward(gpu_ctx, dy=dy.t, **more)()
        ready()
        if "dx" in wanted:
            assert_close(dx.t, want_dx, product_limit(gv, wv, n), "dx")
        if "dw" in wanted:
            assert_close(dw.t, want_dw, product_limit(gtv, xtv, m), "dw")
        if "dbias" in wanted:
            assert_close(db, want_db, (m + 8) * 2.0 ** -24 * dy.t.double().abs().sum(0), "dbias")
        assert dx.untouched() and dw.untouched() and dy.untouched() and x.untouched()


def test_gradients_without_rows(gpu_ctx):
    dw, db = torch.full((40, 50), 7.0, device="cuda"), torch.full((40,), 7.0, device="cuda")
    nothing = torch.empty(0, 40, device="cuda")
    ready()
    ops.LinearMx4Backward(gpu_ctx, dy=nothing, x=torch.empty(0, 50, device="cuda"), dw=dw, dbias=db)()
    ready()
    assert not dw.any() and not db.any()


def test_the_same_bytes_on_every_run(gpu_ctx):
    """Also where K is cut into slices."""
    (a, _), (b, _) = mx4.matrix(normal(1, 100, 30000)), mx4.matrix(normal(2, 200, 30000))
    outs = [torch.empty(100, 200, device="cuda") for _ in range(5)]
    ready()
    for out in outs:
        ops.GemmMx4(gpu_ctx, a=a, b=b, k=30000, out=out)()
    ready()
    assert all(torch.equal(out, outs[0]) for out in outs)
