"""The experts' layer for few tokens on the GPU, against its definition in 64 bits."""
import pytest
import torch

import mx4_cases as mx4
from operator_cases import TYPES, Guarded, assert_close, place
from rns8_amd import operators as ops

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def ready():
    torch.cuda.synchronize()  # the library's stream does not wait for torch's


class Experts:
    """Weights of every expert, as matrices' bytes and as values in 64 bits."""

    def __init__(self, seed, experts, width, inner):
        self.inner = inner
        self.bytes, self.value = {}, {}
        for at, (name, rows, cols) in enumerate((("gate", inner, width), ("up", inner, width), ("down", width, inner))):
            each = [mx4.matrix(normal(seed + 1000 * at + e, rows, cols) / cols ** 0.5) for e in range(experts)]
            self.bytes[name] = torch.stack([q for q, _ in each])
            self.value[name] = torch.stack([v for _, v in each])

    def expected(self, x, ids, weights):
        """The layer's result and what 32-bit sums, hidden values of 16 bits (24) and exponentials may be off."""
        gate, up, down = (self.value[n] for n in ("gate", "up", "down"))
        x64, out = x.double(), torch.zeros(*x.shape, dtype=torch.float64, device="cuda")
        limit = torch.zeros_like(out)
        kept = STEP if x.dtype == torch.float32 else 2.0 ** -16
        for e in range(gate.shape[0]):
            for slot in range(ids.shape[1]):
                t = (ids[:, slot] == e).nonzero()[:, 0]
                if t.numel() == 0:
                    continue
                xt = x64[t].t().contiguous()
                w = weights[t, slot].double()
                g, u = gate[e] @ xt, up[e] @ xt
                off = (x.shape[1] + 64) * STEP
                dg, du = off * (gate[e].abs() @ xt.abs()), off * (up[e].abs() @ xt.abs())
                silu = g * torch.sigmoid(g)
                h = silu * u
                # |silu'| < 1.1; an exponential, a division and products: sixteen steps
                dh = 1.1 * dg * u.abs() + silu.abs() * du + 1.1 * dg * du + (16 * STEP + kept) * h.abs()
                out[t] += ((down[e] @ h) * w).t()
                sums = (self.inner * ids.shape[1] + 64) * STEP
                limit[t] += ((down[e].abs() @ (dh + sums * (h.abs() + dh))) * w.abs()).t()
        return out, limit


def chosen(scores, top, normalize):
    """Experts and weights, from scores in 32 bits."""
    ids = torch.sort(scores, dim=1, descending=True, stable=True).indices[:, :top]
    p = torch.softmax(scores.double(), 1)
    weights = p.gather(1, ids)
    return ids, weights / weights.sum(1, keepdim=True) if normalize else weights


CASES = [(1, 1, 1, 1, 1), (1, 8, 2, 64, 100), (1, 128, 8, 512, 256), (2, 5, 5, 33, 17), (3, 100, 16, 300, 70),
         (5, 12, 3, 1101, 701), (16, 4, 1, 256, 512), (17, 6, 2, 100, 300), (40, 3, 2, 520, 260), (64, 2, 2, 100, 40),
         (64, 70, 8, 264, 272), (64, 1024, 4, 40, 24)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,top,width,inner", CASES)
@pytest.mark.parametrize("normalize", [True, False])
def test_layer_with_router(gpu_ctx, dtype, tokens, experts, top, width, inner, normalize):
    layer = Experts(width, experts, width, inner)
    x = place(normal(tokens, tokens, width).to(dtype), 3, 1)
    router = place((2 * normal(5, experts, width) / width ** 0.5).to(dtype), 1, 3)
    out = Guarded(tokens, width, dtype, pad=5, offset=1)
    ids = torch.full((tokens, top), -7, dtype=torch.int32, device="cuda")
    weights = torch.full((tokens, top), 7.0, device="cuda")
    call = ops.ExpertsMx4(gpu_ctx, x=x.t, router=router.t, **layer.bytes, inner=inner, out=out.t, ids=ids, weights=weights,
                          normalize=normalize)
    scores = (x.t.double() @ router.t.double().t()).float()
    want_ids, want_weights = chosen(scores, top, normalize)
    ready()
    call()
    ready()
    assert torch.equal(ids.long(), want_ids)
    # an exponential's argument is off by one step of the largest score difference, its sum by `experts` steps
    spread = (scores.amax(1) - scores.amin(1)).double()[:, None]
    assert ((weights - want_weights).abs() <= (spread + experts + 16) * STEP * want_weights).all()
    want, limit = layer.expected(x.t, want_ids, weights)
    assert_close(out.t, want, limit)
    assert out.untouched() and x.untouched() and router.untouched()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 9, 64])
def test_layer_with_ids_of_its_own(gpu_ctx, dtype, tokens):
    """Slots elsewhere, experts twice, tokens without any expert, weights of any sign and size."""
    layer = Experts(3, 7, 300, 130)
    x = normal(tokens, tokens, 300).to(dtype)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    ids = torch.randint(-2, 9, (tokens, 4), generator=g, device="cuda").int()
    ids[tokens // 2] = torch.tensor([3, 3, 5, 3])
    if tokens > 1:
        ids[1] = torch.tensor([-1, 7, 2 ** 31 - 1, -2 ** 31])
    weights = 3 * normal(2, tokens, 4)
    kept = ids.clone(), weights.clone()
    out = Guarded(tokens, 300, dtype, pad=1)
    ready()
    ops.ExpertsMx4(gpu_ctx, x=x, **layer.bytes, inner=130, out=out.t, ids=ids, weights=weights)()
    ready()
    want, limit = layer.expected(x, ids, weights)
    assert_close(out.t, want, limit)
    if tokens > 1:
        assert not out.t[1].any()
    assert out.untouched() and torch.equal(ids, kept[0]) and torch.equal(weights, kept[1])


def test_equal_scores_go_to_the_lower_index(gpu_ctx):
    layer = Experts(3, 9, 64, 32)
    x = torch.zeros(3, 64, device="cuda")
    x[0, 0], x[1, 1] = 1.0, -1.0
    router = torch.zeros(9, 64, device="cuda")
    router[:, 0] = torch.tensor([0.0, 2, -0.0, 2, 1, 2, 0, 1, 2])
    router[:, 1] = torch.tensor([5.0, 5, 5, 5, 5, 5, 5, 4, 5])
    ids, out = torch.zeros(3, 6, dtype=torch.int32, device="cuda"), torch.zeros(3, 64, device="cuda")
    ready()
    ops.ExpertsMx4(gpu_ctx, x=x, router=router, **layer.bytes, inner=32, out=out, ids=ids)()
    ready()
    assert ids.tolist() == [[1, 3, 5, 8, 4, 7], [7, 0, 1, 2, 3, 4], [0, 1, 2, 3, 4, 5]]


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(gpu_ctx, dtype):
    """A token's own row, or the rows that read an expert's bad block; no other."""
    layer = Experts(3, 5, 300, 130)
    x = normal(4, 20, 300).to(dtype)
    ids = (torch.arange(20, device="cuda")[:, None] + torch.arange(2, device="cuda")).remainder(4).int()
    weights = torch.full((20, 2), 0.5, device="cuda")
    clean, out = torch.empty(20, 300, dtype=dtype, device="cuda"), torch.empty(20, 300, dtype=dtype, device="cuda")
    ready()
    ops.ExpertsMx4(gpu_ctx, x=x, **layer.bytes, inner=130, out=clean, ids=ids, weights=weights)()
    ready()
    x[6, 299], x[11, 0] = float("nan"), float("inf")
    ready()
    ops.ExpertsMx4(gpu_ctx, x=x, **layer.bytes, inner=130, out=out, ids=ids, weights=weights)()
    ready()
    rest = [t for t in range(20) if t not in (6, 11)]
    assert torch.isnan(out[6]).all() and not torch.isfinite(out[11]).any()
    assert torch.equal(out[rest], clean[rest])
    for name, of in (("gate", (130, 300)), ("down", (300, 130))):
        held = {k: v.clone() for k, v in layer.bytes.items()}
        v = layer.value[name][2].clone()
        v[9, 40] = float("nan")
        held[name][2] = mx4.matrix(v)[0]
        x[6], x[11] = 1.0, 2.0
        ready()
        ops.ExpertsMx4(gpu_ctx, x=x, **held, inner=130, out=out, ids=ids, weights=weights)()
        ready()
        uses = (ids == 2).any(1)
        bad = torch.isnan(out)
        if name == "gate":
            assert torch.equal(bad, uses[:, None].expand(20, 300))
        else:
            assert bad[uses, 9].all() and bad.sum() == uses.sum()


def test_the_same_bytes_on_every_run_and_in_any_batch(gpu_ctx):
    layer = Experts(3, 16, 1000, 500)
    x, router = normal(1, 33, 1000).bfloat16(), normal(2, 16, 1000).bfloat16()
    outs = [torch.empty(33, 1000, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    ids = torch.empty(33, 4, dtype=torch.int32, device="cuda")
    alone = torch.empty(1, 4, dtype=torch.int32, device="cuda")
    ready()
    for out in outs:
        ops.ExpertsMx4(gpu_ctx, x=x, router=router, **layer.bytes, inner=500, out=out, ids=ids)()
    ready()
    assert all(torch.equal(out, outs[0]) for out in outs)
    for t in (0, 32):
        one = torch.empty(1, 1000, dtype=torch.bfloat16, device="cuda")
        ops.ExpertsMx4(gpu_ctx, x=x[t:t + 1], router=router, **layer.bytes, inner=500, out=one, ids=alone)()
        ready()
        assert torch.equal(alone[0], ids[t])
