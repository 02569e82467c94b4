"""A stack of matrices whose rows are a multiple of 16 is one matrix: packed, rounded and read back in one call."""
import pytest
import torch

from operator_cases import TYPES
from rns8_amd import operators as ops
from test_gpu_mx4 import normal, ready

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count,rows,cols", [(3, 16, 33), (5, 48, 300), (7, 32, 1024)])
def test_packing(gpu_ctx, count, rows, cols):
    g = torch.Generator(device="cuda").manual_seed(cols)
    data = torch.randint(0, 256, (count, rows, (cols + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = torch.randint(0, 256, (count, rows, (cols + 31) // 32), generator=g, device="cuda", dtype=torch.uint8)
    one, each = (torch.full((count, ops.mx4_bytes(rows, cols)), 7, dtype=torch.uint8, device="cuda") for _ in range(2))
    ready()
    ops.PackMx4(gpu_ctx, data=data.flatten(0, 1), scale=scale.flatten(0, 1), q=one, cols=cols)()
    for i in range(count):
        ops.PackMx4(gpu_ctx, data=data[i], scale=scale[i], q=each[i], cols=cols)()
    ready()
    assert torch.equal(one, each)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,rows,cols", [(3, 16, 33), (5, 48, 300)])
def test_rounding_and_back(gpu_ctx, dtype, count, rows, cols):
    x = normal(1, count, rows, cols).to(dtype)
    one, each = (torch.full((count, ops.mx4_bytes(rows, cols)), 7, dtype=torch.uint8, device="cuda") for _ in range(2))
    back, back_each = torch.empty_like(x), torch.empty_like(x)
    ready()
    ops.QuantizeMx4(gpu_ctx, x=x.flatten(0, 1), q=one)()
    ops.DequantizeMx4(gpu_ctx, q=one, out=back.flatten(0, 1))()
    for i in range(count):
        ops.QuantizeMx4(gpu_ctx, x=x[i], q=each[i])()
        ops.DequantizeMx4(gpu_ctx, q=each[i], out=back_each[i])()
    ready()
    assert torch.equal(one, each) and torch.equal(back, back_each)
