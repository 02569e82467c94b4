"""Operators on 4-bit microscaled matrices where sizes, grids and uses meet their limits."""
import pytest
import torch

import mx4_cases as mx4
from operator_cases import TYPES, assert_close
from rns8_amd import operators as ops
from test_gpu_mx4 import normal, product_limit, ready

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(300, 300, 100), (65, 65, 65), (129, 700, 64), (128, 2000, 700), (1000, 130, 1025), (9000, 100, 90),
                                   (100, 9000, 90), (4096, 1024, 1024)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_in_one_launch(gpu_ctx, dtype, m, n, k):
    """Tiles of both products that are no multiple of the grid's eighths; each gradient as it is by itself."""
    dy, x = normal(1, m, n).to(dtype), normal(2, m, k).to(dtype)
    w_t, _ = mx4.matrix(normal(3, n, k).t())
    both = [torch.full((m, k), 7.0, dtype=dtype, device="cuda"), torch.full((n, k), 7.0, device="cuda"),
            torch.full((n,), 7.0, device="cuda")]
    alone = [torch.empty_like(t) for t in both]
    ready()
    ops.LinearMx4Backward(gpu_ctx, dy=dy, x=x, w_t=w_t, dx=both[0], dw=both[1], dbias=both[2])()
    ops.LinearMx4Backward(gpu_ctx, dy=dy, w_t=w_t, dx=alone[0])()
    ops.LinearMx4Backward(gpu_ctx, dy=dy, x=x, dw=alone[1])()
    ops.LinearMx4Backward(gpu_ctx, dy=dy, dbias=alone[2])()
    ready()
    assert torch.equal(both[2], alone[2])
    _, gv = mx4.matrix(dy)
    _, gtv = mx4.matrix(dy.t())
    _, xtv = mx4.matrix(x.t())
    wv = mx4.matrix(normal(3, n, k).t())[1]
    for got in (both, alone):
        assert_close(got[0], torch.mm(gv, wv.t().contiguous()), product_limit(gv, wv, n), "dx")
        assert_close(got[1], torch.mm(gtv, xtv.t().contiguous()), product_limit(gtv, xtv, m), "dw")
        assert_close(got[2], dy.double().sum(0), (m + 8) * 2.0 ** -24 * dy.double().abs().sum(0), "dbias")


@pytest.mark.parametrize("m,n,k", [(128, 2000, 64), (70, 3000, 70)])
def test_bias_gradients_wider_than_the_grid(gpu_ctx, m, n, k):
    """More columns than the waves of a launch whose last workgroups have no tile."""
    dy, x = normal(1, m, n), normal(2, m, k)
    w_t, _ = mx4.matrix(normal(3, n, k).t())
    dx, dw, db = torch.empty(m, k, device="cuda"), torch.empty(n, k, device="cuda"), torch.full((n,), 7.0, device="cuda")
    ready()
    ops.LinearMx4Backward(gpu_ctx, dy=dy, x=x, w_t=w_t, dx=dx, dw=dw, dbias=db)()
    ready()
    assert_close(db, dy.double().sum(0), (m + 8) * 2.0 ** -24 * dy.double().abs().sum(0))


def levels(seed, rows, cols):
    """Values that a rounding along rows or columns leaves as they are."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = mx4.LEVELS.cuda()[torch.randint(0, 8, (rows, cols), generator=g, device="cuda")]
    return torch.where(torch.randint(0, 2, (rows, cols), generator=g, device="cuda") == 1, v, -v).float()


@pytest.mark.parametrize("m,n,k", [(1, 40, 50), (16, 64, 100), (70, 130, 90), (300, 200, 333)])
def test_gradients_against_differences(gpu_ctx, m, n, k):
    """f = sum(g * (x w^T + b)) on values that no rounding changes: all its sums are exact in 32 bits, so its differences
    along x, w and b are the gradients' products with the steps to the last bit."""
    x, w, g = levels(1, m, k), levels(2, n, k), levels(3, m, n)
    b = levels(4, 1, n)[0]

    def f(x, w, b):
        q, _ = mx4.matrix(w)
        out = torch.empty(m, n, device="cuda")
        ready()
        ops.LinearMx4(gpu_ctx, x=x, w=q, bias=b, out=out)()
        ready()
        return (g.double() * out.double()).sum()

    q_t = torch.empty(ops.mx4_bytes(k, n), dtype=torch.uint8, device="cuda")
    dx, dw, db = torch.empty(m, k, device="cuda"), torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    ready()
    ops.QuantizeMx4(gpu_ctx, x=w, q_t=q_t)()
    ops.LinearMx4Backward(gpu_ctx, dy=g, x=x, w_t=q_t, dx=dx, dw=dw, dbias=db)()
    ready()
    start = f(x, w, b)
    for seed in (5, 6):
        x2, w2, b2 = levels(seed, m, k), levels(seed + 2, n, k), levels(seed + 4, 1, n)[0]
        assert f(x2, w, b) - start == (dx.double() * (x2 - x).double()).sum()
        assert f(x, w2, b) - start == (dw.double() * (w2 - w).double()).sum()
        assert f(x, w, b2) - start == (db.double() * (b2 - b).double()).sum()


def test_sums_of_nothing_of_many_rows(gpu_ctx):
    bias = normal(1, 3)
    out = torch.full((5_000_000, 3), 7.0, dtype=torch.bfloat16, device="cuda")
    nothing = torch.empty(0, dtype=torch.uint8, device="cuda")
    ready()
    ops.GemmMx4(gpu_ctx, a=nothing, b=nothing, k=0, out=out, bias=bias)()
    ready()
    assert torch.equal(out, bias.bfloat16().expand_as(out))


def group(q, g, cols):
    """16 rows of an MX4 matrix: one themselves."""
    size = ops.mx4_bytes(16, cols)
    return q[g * size:(g + 1) * size]


def test_rounding_past_32_bits(gpu_ctx):
    rows, cols = 70000, 65536
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    q = torch.empty(ops.mx4_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    q_t = torch.empty(ops.mx4_bytes(cols, rows), dtype=torch.uint8, device="cuda")
    ready()
    ops.QuantizeMx4(gpu_ctx, x=x, q=q, q_t=q_t)()
    ready()
    for g in (0, 2000, rows // 16 - 1):
        assert torch.equal(group(q, g, cols), mx4.matrix(x[16 * g:16 * g + 16])[0])
    for g in (0, cols // 16 - 1):
        assert torch.equal(group(q_t, g, rows), mx4.matrix(x[:, 16 * g:16 * g + 16].t())[0])
    want = mx4.matrix(x[-16:])[1]
    ready()
    ops.DequantizeMx4(gpu_ctx, q=q, out=x)()
    ready()
    assert torch.equal(x[-16:].double(), want)


@pytest.mark.parametrize("m", [3, 40, 100])
def test_products_of_operands_past_32_bits(gpu_ctx, m):
    n, k = 140000, 65536
    a, av = mx4.matrix(normal(1, m, k))
    b = torch.empty(ops.mx4_bytes(n, k), dtype=torch.uint8, device="cuda")
    step = ops.mx4_bytes(10000, k)
    for i in range(14):
        part = normal(i, 10000, k).bfloat16()
        ready()
        ops.QuantizeMx4(gpu_ctx, x=part, q=b[i * step:(i + 1) * step])()
        ready()
    out = torch.full((m, n), 7.0, device="cuda")
    ready()
    ops.GemmMx4(gpu_ctx, a=a, b=b, k=k, out=out)()
    ready()
    for g in (0, 4000, 8191, n // 16 - 1):
        bv = torch.empty(16, k, device="cuda")
        ready()
        ops.DequantizeMx4(gpu_ctx, q=group(b, g, k), out=bv)()
        ready()
        bv = bv.double()
        assert_close(out[:, 16 * g:16 * g + 16], av @ bv.t().contiguous(), product_limit(av, bv, k), f"channels {16 * g}")


def test_results_past_32_bits(gpu_ctx):
    n, k = 66000, 64
    (a, av), (b, bv) = mx4.exact_matrix(1, n, k), mx4.exact_matrix(2, n, k)
    out = torch.full((n, n), 7.0, device="cuda")
    ready()
    ops.GemmMx4(gpu_ctx, a=a, b=b, k=k, out=out)()
    ready()
    for rows in (slice(0, 100), slice(33000, 33100), slice(n - 100, n)):
        assert torch.equal(out[rows].double(), av[rows] @ bv.t().contiguous())


@pytest.mark.parametrize("tokens", [2, 20])
def test_experts_past_32_bits(gpu_ctx, tokens):
    """1024 experts of 4.4 MB a matrix: the same bytes as of those experts alone."""
    width, inner, some = 4096, 2048, [0, 500, 1000, 1023]
    g = torch.Generator(device="cuda").manual_seed(1)
    weights = {}
    for name, rows, cols in (("gate", inner, width), ("up", inner, width), ("down", width, inner)):
        q = torch.randint(0, 256, (1024, ops.mx4_bytes(rows, cols)), generator=g, device="cuda", dtype=torch.uint8)
        q.view(-1, ops.mx4_bytes(1, 1))[:, 2048:] = 120
        weights[name] = q
    few = {name: q[some].clone() for name, q in weights.items()}
    ids = torch.randint(0, 4, (tokens, 2), generator=g, device="cuda", dtype=torch.int32)
    x, w = normal(2, tokens, width).bfloat16(), normal(3, tokens, 2)
    outs = [torch.empty_like(x) for _ in range(2)]
    ready()
    ops.ExpertsMx4(gpu_ctx, x=x, **weights, inner=inner, out=outs[0], ids=torch.tensor(some, device="cuda").int()[ids.long()], weights=w)()
    ops.ExpertsMx4(gpu_ctx, x=x, **few, inner=inner, out=outs[1], ids=ids, weights=w)()
    ready()
    assert torch.equal(outs[0], outs[1]) and outs[0].any(1).all() and torch.isfinite(outs[0]).all()
