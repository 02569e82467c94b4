"""The experts' layer where experts have as many tokens as a batch holds, one more, and far more: on weights that pick
single values, exactly."""
import pytest
import torch

from operator_cases import TYPES, Guarded
from rns8_amd import operators as ops
from test_gpu_mx4 import normal, ready
from test_gpu_mx4_experts_bits import picking

pytestmark = pytest.mark.gpu


def check(gpu_ctx, dtype, counts, width, inner, scattered=True):
    """counts: how many tokens each expert has. An output is 32 times one value of the token, times its expert's factor of
    one or two bits."""
    experts, tokens = len(counts), sum(counts)
    gen = torch.Generator(device="cuda").manual_seed(width + inner)
    ids = torch.arange(experts, device="cuda").repeat_interleave(torch.tensor(counts, device="cuda"))
    if scattered:
        ids = ids[torch.randperm(tokens, generator=gen, device="cuda")]
    x = normal(tokens, tokens, width).to(dtype)
    x[:, 0] = 32.0
    of_x = torch.randint(1, width, (inner,), generator=gen, device="cuda")
    of_h = torch.randint(0, inner, (width,), generator=gen, device="cuda")
    gate = picking(inner, width, [(i, 0, 1.0) for i in range(inner)])
    up = picking(inner, width, [(i, c, 1.0) for i, c in enumerate(of_x.tolist())])
    scale = [1.0, 2.0, 3.0, 4.0, 6.0, 0.5, 1.5]
    down = [picking(width, inner, [(c, i, scale[e % 7]) for c, i in enumerate(of_h.tolist())]) for e in range(min(experts, 7))]
    out = Guarded(tokens, width, dtype, pad=3, offset=1)
    ready()
    ops.ExpertsMx4(gpu_ctx, x=x, gate=gate.expand(experts, -1).contiguous(), up=up.expand(experts, -1).contiguous(),
                   down=torch.stack([down[e % 7] for e in range(experts)]), inner=inner, out=out.t,
                   ids=ids.int()[:, None].contiguous(), weights=torch.ones(tokens, 1, device="cuda"))()
    ready()
    factor = 32 * torch.tensor(scale, dtype=torch.float64, device="cuda")[ids % 7]
    want = x[:, of_x][:, of_h].double() * factor[:, None]
    if dtype != torch.float32:
        assert torch.equal(out.t, want.to(dtype))  # (11 bits times two are exact in 32)
    else:
        # three parts of 8 bits, each times two bits exactly, added: two roundings
        assert ((out.t.double() - want).abs() <= 2 * 2.0 ** -24 * want.abs()).all()
    assert out.untouched()


# three parts: 5 tokens are one MFMA's columns, 10 two's; two parts: 8 and 16; one: 16
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts", [[1, 5, 6, 10, 11, 7], [8, 9, 0, 16, 17], [20, 21, 0, 0, 22], [64], [0, 0, 33, 31], [17, 47]])
@pytest.mark.parametrize("width,inner", [(300, 520), (70, 40)])
def test_tokens_of_an_expert(gpu_ctx, dtype, counts, width, inner):
    check(gpu_ctx, dtype, counts, width, inner)


# rows of which LDS holds a few, one, or part of one, hidden and down
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,width,inner", [([3, 4, 7, 8, 9], 4096, 40), ([2, 3, 5, 6, 9], 40, 2600), ([1, 2, 3, 14], 12000, 40),
                                                ([1, 2, 3, 14], 40, 12000), ([40, 24], 4096, 300)])
def test_long_rows(gpu_ctx, dtype, counts, width, inner):
    check(gpu_ctx, dtype, counts, width, inner, scattered=False)


# every token's expert its own; experts without tokens between
def test_many_experts(gpu_ctx):
    check(gpu_ctx, torch.bfloat16, [1] * 64, 2100, 1030)
    check(gpu_ctx, torch.float32, [0, 1, 0, 2] * 21, 600, 520)


# what the down kernel for few pairs holds, to its last whole row, and one block more
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,inner", [([2, 3], 4352), ([2, 3], 4353), ([16], 1280), ([16], 1281), ([1], 21760), ([1], 21761)])
def test_few_pairs(gpu_ctx, dtype, counts, inner):
    check(gpu_ctx, dtype, counts, 40, inner)
