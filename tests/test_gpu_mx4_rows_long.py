"""Products of few rows over sums so long that every wave's ring of chunks goes round, exactly: a chunk that is left out,
taken twice or read before it has come shows."""
import pytest
import torch

import mx4_cases as mx4
from operator_cases import TYPES, Guarded
from rns8_amd import operators as ops
from test_gpu_mx4 import ready

pytestmark = pytest.mark.gpu


def small(seed, rows, cols):
    """An MX4 matrix of multiples of 1/4 up to 6. Products are multiples of 1/16 up to 36: sums of at most 29000 of them stay
    below 2^20, and 32 bits hold them in any order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = (cols + 31) // 32
    code = torch.randint(0, 16, (rows, blocks * 32), generator=g, device="cuda")
    code[:, cols:] = 0
    code = code.reshape(rows, blocks, 32)
    scale = torch.randint(126, 128, (rows, blocks), generator=g, device="cuda")
    return mx4.buffer_of(code, scale, cols), mx4.values(code, scale, cols)


# 16, 32, 48 and 64 rows to a workgroup, 16 channels and 32
@pytest.mark.parametrize("m,n,k", [(5, 100, 16384), (16, 8200, 20000), (20, 100, 16384), (20, 8200, 12000), (33, 70, 12300),
                                   (40, 8200, 12000), (64, 40, 9000), (64, 8200, 9000), (3, 33, 29000)])
def test_products(gpu_ctx, m, n, k):
    (a, av), (b, bv) = small(m, m, k), small(n + 7, n, k)
    want = torch.mm(av, bv.t().contiguous())
    for dtype, pad in ((torch.float32, 0), (torch.bfloat16, 5), (torch.float16, 1)):
        out = Guarded(m, n, dtype, pad=pad, offset=pad)
        ready()
        ops.GemmMx4(gpu_ctx, a=a, b=b, k=k, out=out.t)()
        ready()
        assert torch.equal(out.t, want.float().to(dtype)) and out.untouched()


# one and two tokens, then up to 16; 16 channels to a workgroup and 32; whole chunks and a cut one at the end
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 64, 16384), (2, 64, 9000), (1, 8200, 20000), (2, 8200, 20001), (3, 64, 8192), (3, 8200, 4700),
                                   (16, 300, 8192), (16, 300, 13000), (16, 8200, 6003), (9, 8200, 12288)])
def test_linear_layers(gpu_ctx, dtype, m, n, k):
    """Floating rows that a rounding leaves as they are."""
    (_, xv), (w, wv) = small(m, m, k), small(n + 7, n, k)
    assert torch.equal(mx4.matrix(xv)[1], xv)
    x, out = xv.to(dtype), Guarded(m, n, dtype, pad=2, offset=3)
    ready()
    ops.LinearMx4(gpu_ctx, x=x, w=w, out=out.t)()
    ready()
    assert torch.equal(out.t, torch.mm(xv, wv.t().contiguous()).float().to(dtype)) and out.untouched()
