"""How many bits the experts' layer keeps of its tokens and of its hidden values: on weights that pick single values, so
that every sum is one term or a difference that is exact, and nothing is allowed for."""
import pytest
import torch

import mx4_cases as mx4
from operator_cases import TYPES, Guarded
from rns8_amd import operators as ops
from test_gpu_mx4 import normal, ready

pytestmark = pytest.mark.gpu

# a token to a workgroup's table, several, and more than the kernels for few pairs take
TOKENS = [1, 5, 17, 40]


def picking(rows, cols, at):
    """A matrix of zeros with the given values (row, column, value): what MX4 holds as it is."""
    v = torch.zeros(rows, cols, device="cuda")
    for r, c, value in at:
        v[r, c] = value
    return mx4.matrix(v)[0]


def layer(gpu_ctx, x, gate, up, down, inner, ids, weights):
    """The layer on three experts with the same weights each."""
    out = Guarded(x.shape[0], x.shape[1], x.dtype, pad=3, offset=1)
    held = {name: q.expand(3, -1).contiguous() for name, q in (("gate", gate), ("up", up), ("down", down))}
    ready()
    ops.ExpertsMx4(gpu_ctx, x=x, **held, inner=inner, out=out.t, ids=ids, weights=weights)()
    ready()
    assert out.untouched()
    return out.t


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("width,inner", [(64, 40), (300, 520)])
def test_values_keep_their_bits(gpu_ctx, dtype, tokens, width, inner):
    """g = 32, so that silu(g) is g to the last bit; u is one value of the token, an output one hidden value: 32 times a
    value, exactly, whatever its type. A part of a value that is left out shows."""
    x = normal(tokens, tokens, width).to(dtype)
    x[:, 0] = 32.0
    gen = torch.Generator(device="cuda").manual_seed(width)
    of_x = torch.randint(1, width, (inner,), generator=gen, device="cuda").tolist()
    of_h = torch.randint(0, inner, (width,), generator=gen, device="cuda").tolist()
    gate = picking(inner, width, [(i, 0, 1.0) for i in range(inner)])
    up = picking(inner, width, [(i, c, 1.0) for i, c in enumerate(of_x)])
    down = picking(width, inner, [(c, i, 1.0) for c, i in enumerate(of_h)])
    ids = (torch.arange(tokens, device="cuda") % 3).int()[:, None].contiguous()
    out = layer(gpu_ctx, x, gate, up, down, inner, ids, torch.ones(tokens, 1, device="cuda"))
    want = 32 * x[:, torch.tensor(of_x, device="cuda")][:, torch.tensor(of_h, device="cuda")]
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("width,inner", [(64, 40), (300, 520)])
def test_differences_of_hidden_values(gpu_ctx, dtype, tokens, width, inner):
    """Hidden values 32 (1 + 2^-8 + 2^-d) and 32 (1 + 2^-8), one less the other: 2^(5 - d) to the last bit, for every d
    that 24 bits hold beside 1. Every type holds 2^-d, and the difference."""
    x = torch.zeros(tokens, width, dtype=dtype, device="cuda")
    d = torch.arange(tokens, device="cuda") * 5 % 23 + 1
    if tokens == 1:
        d[0] = 23
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = 1.0, torch.exp2(-d.double()).to(dtype), 32.0, 2.0 ** -8
    first, second = 0, inner - 1
    gate = picking(inner, width, [(first, 2, 1.0), (second, 2, 1.0)])
    up = picking(inner, width, [(first, 0, 1.0), (first, 3, 1.0), (first, 1, 1.0), (second, 0, 1.0), (second, 3, 1.0)])
    down = picking(width, inner, [at for c in range(width) for at in ((c, first, 1.0), (c, second, -1.0))])
    ids = torch.stack([torch.arange(tokens, device="cuda") % 3, (torch.arange(tokens, device="cuda") + 1) % 3], 1).int()
    weights = torch.tensor([1.0, -0.5], device="cuda").expand(tokens, 2).contiguous()
    out = layer(gpu_ctx, x, gate, up, down, inner, ids, weights)
    assert torch.equal(out.double(), torch.exp2(4 - d.double())[:, None].expand(tokens, width))
