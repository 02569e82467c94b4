"""The experts' layer at the limits of its sizes and of what a workgroup holds."""
import pytest
import torch

import mx4_cases as mx4  # noqa: F401
from operator_cases import TYPES, Guarded, assert_close
from rns8_amd import operators as ops
from test_gpu_mx4_experts import Experts, normal, ready

pytestmark = pytest.mark.gpu


def check(ctx, dtype, tokens, experts, top, width, inner):
    layer = Experts(width, experts, width, inner)
    x = normal(1, tokens, width).to(dtype)
    g = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.stack([torch.randperm(experts, generator=g, device="cuda")[:top] for _ in range(tokens)]).int()
    weights = normal(3, tokens, top)
    out = Guarded(tokens, width, dtype, pad=3, offset=1)
    ready()
    ops.ExpertsMx4(ctx, x=x, **layer.bytes, inner=inner, out=out.t, ids=ids, weights=weights)()
    ready()
    want, limit = layer.expected(x, ids, weights)
    assert_close(out.t, want, limit)
    assert out.untouched()


# what a workgroup of the kernels for few pairs holds, filled to its last byte and passed by one block or one token
@pytest.mark.parametrize("dtype,tokens,experts,top,width,inner", [
    (torch.bfloat16, 16, 4, 2, 2048, 768), (torch.bfloat16, 16, 4, 2, 2049, 768), (torch.bfloat16, 16, 4, 2, 2048, 769),
    (torch.bfloat16, 17, 4, 2, 1024, 256), (torch.float16, 16, 4, 2, 1024, 768), (torch.float32, 16, 4, 2, 512, 512),
    (torch.float32, 2, 4, 2, 5376, 4096), (torch.float32, 2, 4, 2, 5377, 300)])
def test_few_pairs(gpu_ctx, dtype, tokens, experts, top, width, inner):
    check(gpu_ctx, dtype, tokens, experts, top, width, inner)


# rows that LDS does not hold at once
@pytest.mark.parametrize("dtype,tokens,width,inner", [
    (torch.bfloat16, 20, 40000, 40), (torch.bfloat16, 20, 40, 17000), (torch.float32, 19, 12000, 40),
    (torch.float32, 5, 40, 12000), (torch.float16, 18, 17000, 33), (torch.float32, 1, 65536, 16),
    (torch.bfloat16, 2, 16, 65536)])
def test_wide_rows(gpu_ctx, dtype, tokens, width, inner):
    check(gpu_ctx, dtype, tokens, 3, 2, width, inner)


@pytest.mark.parametrize("dtype", TYPES)
def test_most_tokens_and_slots(gpu_ctx, dtype):
    check(gpu_ctx, dtype, 64, 16, 16, 70, 50)
    check(gpu_ctx, dtype, 64, 17, 16, 40, 300)


@pytest.mark.parametrize("tokens", [3, 40])
@pytest.mark.parametrize("normalize", [True, False])
def test_scores_that_are_not_finite(gpu_ctx, tokens, normalize):
    """A NaN or infinite score of a token is its own; -infinity beside finite scores is an expert that gets nothing."""
    layer = Experts(1, 6, 64, 48)
    x = normal(2, tokens, 64)
    x[:, 0], x[:, 1] = 0.0, 0.0
    router = normal(3, 6, 64)
    clean, out = torch.empty(2, tokens, 64, device="cuda")
    ids, weights = torch.empty(tokens, 6, dtype=torch.int32, device="cuda"), torch.empty(tokens, 6, device="cuda")
    args = dict(router=router, **layer.bytes, inner=48, normalize=normalize, top=6)
    ready()
    ops.ExpertsMx4(gpu_ctx, x=x, out=clean, **args)()
    ready()
    x[1, 5] = float("nan")
    ready()
    ops.ExpertsMx4(gpu_ctx, x=x, out=out, ids=ids, weights=weights, **args)()
    ready()
    rest = [t for t in range(tokens) if t != 1]
    assert torch.equal(out[rest], clean[rest]) and torch.isnan(out[1]).all() and torch.isnan(weights[1]).all()
    assert ids[1].tolist() == [0, 1, 2, 3, 4, 5]
    # an expert's score of -infinity: the largest negative numbers times a large one
    x[1, 5], x[:, 0] = 0.0, 1e30
    router[:, 0], router[2, 0] = 0.0, -3e38
    lowest = x.clone()
    lowest[:, 0] = 1e30
    ready()
    ops.ExpertsMx4(gpu_ctx, x=lowest, out=out, ids=ids, weights=weights, **args)()
    ready()
    assert (ids[:, 5] == 2).all() and not weights[:, 5].any() and torch.isfinite(weights).all()
    # each weight is off by a step for each unit of the scores' spread (below 100), and 22 more
    assert ((weights.double().sum(1) - 1).abs() < 128 * 2.0 ** -23).all()
