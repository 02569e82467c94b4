"""Workspaces of the operators on 4-bit matrices: of exactly the bytes that a query answers, at the least alignment, whatever
they held before."""
import pytest
import torch

import mx4_cases as mx4
from operator_cases import TYPES
from rns8_amd import operators as ops
from test_gpu_mx4 import normal, ready
from test_gpu_mx4_experts import Experts

pytestmark = pytest.mark.gpu


def outputs_of(make):
    """make(**more) gives (call, outputs): the call is made with a workspace of its own and in guarded ones."""
    call, outputs = make()
    ready()
    call()
    ready()
    want = [t.clone() for t in outputs]
    size = call.workspace_bytes
    for fill in (0xFF, 0x00, 0x3C):  # (as floats NaN, 0 and small numbers)
        buf = torch.full((size + 16 + 512,), fill, dtype=torch.uint8, device="cuda")
        for t in outputs:
            t.fill_(7)
        call, outputs = make(workspace=buf[16:16 + size])
        assert call.workspace_bytes == size and call.args.workspace % 32 == 16
        ready()
        call()
        ready()
        assert all(torch.equal(a, b) for a, b in zip(outputs, want))
        assert (buf[:16] == fill).all() and (buf[16 + size:] == fill).all()
    return size


def empty(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


@pytest.mark.parametrize("m,n,k", [(65, 64, 5000), (100, 200, 30000), (70, 513, 9000), (300, 300, 20000)])
def test_products_in_slices(gpu_ctx, m, n, k):
    (a, _), (b, _) = mx4.matrix(normal(1, m, k)), mx4.matrix(normal(2, n, k))
    out = empty(m, n)
    assert outputs_of(lambda **more: (ops.GemmMx4(gpu_ctx, a=a, b=b, k=k, out=out, **more), [out])) > 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(17, 40, 300), (65, 70, 3000), (300, 130, 1101)])
def test_linear_layers(gpu_ctx, dtype, m, n, k):
    x, (w, _) = normal(1, m, k).to(dtype), mx4.matrix(normal(2, n, k))
    out = empty(m, n, dtype=dtype)
    assert outputs_of(lambda **more: (ops.LinearMx4(gpu_ctx, x=x, w=w, out=out, **more), [out])) >= ops.mx4_bytes(m, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(300, 200, 333), (500, 701, 611), (40, 30, 50), (70, 65, 9000), (3000, 100, 90)])
@pytest.mark.parametrize("wanted", ["all", "dx", "dw", "dbias"])
def test_gradients(gpu_ctx, dtype, m, n, k, wanted):
    """In one launch and apart, each alone, cut into slices or not."""
    dy, x = normal(1, m, n).to(dtype), normal(2, m, k).to(dtype)
    w_t, _ = mx4.matrix(normal(3, k, n))
    given = {"dx": dict(dx=empty(m, k, dtype=dtype), w_t=w_t), "dw": dict(dw=empty(n, k), x=x), "dbias": dict(dbias=empty(n))}
    args = {}
    for name, some in given.items():
        if wanted in ("all", name):
            args |= some
    results = [args[name] for name in given if name in args]
    assert outputs_of(lambda **more: (ops.LinearMx4Backward(gpu_ctx, dy=dy, **args, **more), results)) > 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,top,width,inner", [(1, 8, 2, 64, 100), (5, 12, 3, 1101, 701), (16, 16, 16, 100, 300),
                                                            (17, 6, 2, 100, 300), (64, 70, 8, 264, 272), (40, 3, 2, 520, 2600)])
@pytest.mark.parametrize("chosen", [False, True])
def test_experts(gpu_ctx, dtype, tokens, experts, top, width, inner, chosen):
    layer = Experts(width, experts, width, inner)
    x, out = normal(1, tokens, width).to(dtype), empty(tokens, width, dtype=dtype)
    args = dict(x=x, **layer.bytes, inner=inner, out=out)
    results = [out]
    if chosen:
        args |= dict(ids=torch.randint(-1, experts, (tokens, top), device="cuda").int(), weights=normal(3, tokens, top))
    else:
        args |= dict(router=normal(2, experts, width).to(dtype), ids=torch.empty(tokens, top, dtype=torch.int32, device="cuda"),
                     weights=empty(tokens, top))
        results += [args["ids"], args["weights"]]
    assert outputs_of(lambda **more: (ops.ExpertsMx4(gpu_ctx, **args, **more), results)) > 0
