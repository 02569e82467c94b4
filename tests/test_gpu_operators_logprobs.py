"""Token log-probabilities, entropy, top alternatives and their gradient against the definition in 64 bits.

z - m is one 32-bit difference of |z| and the maximum, so an exponential is off
by 2^-23 (|z| + |m|) + 4 * 2^-24 of itself; sums add at most 256 terms of a
thread's own and 64 partial sums. With R = |z| + |m| over the row: logp and lse
are off by at most 2^-24 (4 R + 512 + |log S|).
"""
import pytest
import torch

import rns8_amd as r
from operator_cases import TYPES, U32, Guarded, assert_close, place
from rns8_amd import operators as ops

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def ready():
    torch.cuda.synchronize()


def definition(logits, targets, scale, top):
    z = logits.double() * scale
    lse = torch.logsumexp(z, 1)
    logp = z - lse[:, None]
    p = logp.exp()
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(1)
    empty = (logits == -float("inf")).all(1)
    entropy[empty] = 0
    asked = (targets >= 0) & (targets < logits.shape[1])
    given = logp.gather(1, targets.clamp(0, logits.shape[1] - 1)[:, None])[:, 0]
    given = torch.where(empty, torch.full_like(given, -float("inf")), given)
    ids = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :top]
    best = logp.gather(1, ids)
    best[empty] = -float("inf")
    return dict(lse=lse, logp=torch.where(asked, given, torch.zeros_like(given)), entropy=entropy, top_ids=ids.int(),
                top_logp=best, all=logp, p=p)


def run(ctx, logits, targets, scale=1.0, top=0):
    rows = logits.shape[0]
    out = {k: torch.full((rows,), 9.0, device="cuda") for k in ("logp", "entropy", "lse")}
    if top:
        out |= {"top_ids": torch.full((rows, top), -7, dtype=torch.int32, device="cuda"),
                "top_logp": torch.full((rows, top), 9.0, device="cuda")}
    ready()
    ops.TokenLogprobs(ctx, logits=logits, targets=targets, scale=scale, **out)()
    ready()
    return out


def check(got, want, logits, scale):
    z = torch.where(torch.isfinite(logits), logits, torch.zeros_like(logits)).double().abs() * scale
    size = 2 * z.amax(1)
    slack = U32 * (4 * size + 512 + want["lse"].abs().nan_to_num(0, 0, 0))
    assert_close(got["lse"], want["lse"], slack, "lse")
    assert_close(got["logp"], want["logp"], slack, "logp")
    # W / S: every term d e^d is off by its exponential's error and d's own
    assert_close(got["entropy"], want["entropy"], 2 * slack * (1 + size), "entropy")
    if "top_ids" in got:
        assert torch.equal(got["top_ids"], want["top_ids"])
        assert_close(got["top_logp"], want["top_logp"], slack[:, None], "top_logp")


SIZES = [(1, 1, 0, 0), (1, 131072, 0, 0), (2, 7, 0, 1), (3, 1000, 3, 0), (4, 50001, 0, 1), (7, 8192, 0, 0),
         (600, 513, 7, 0), (300, 4099, 0, 0), (2, 300000, 0, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,pad,offset", SIZES)
@pytest.mark.parametrize("scale,top,banned", [(1.0, 0, False), (0.7, 1, True), (1.0, 5, True), (3.0, 20, False),
                                              (1.0, 64, True)])
def test_forward(gpu_ctx, dtype, rows, vocab, pad, offset, scale, top, banned):
    top = min(top, vocab)
    v = 3.0 * normal(rows + vocab, rows, vocab)
    if banned:
        v[:, 1::3] = -float("inf")
    logits = place(v.to(dtype), pad, offset).t
    targets = torch.randint(vocab, (rows,), device="cuda")
    targets[::5] = 0
    if rows > 2:
        targets[1], targets[2] = -100, vocab
    got = run(gpu_ctx, logits, targets, scale, top)
    check(got, definition(logits, targets, scale, top), logits, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 1000, 70000])
def test_ties_and_special_rows(gpu_ctx, dtype, vocab):
    """Equal logits go to the lower index; the type's lowest value is a number; rows with nothing left."""
    low = torch.finfo(dtype).min
    v = torch.zeros(10, vocab, device="cuda").to(dtype)
    v[0] = 1.5                                     # all equal
    v[1, ::2] = -0.0                               # 0 and -0 are equal
    v[2] = -float("inf")                           # nothing left
    v[3] = low                                     # the lowest value everywhere
    v[4] = low
    v[4, vocab - 1] = 1.0                          # all but one masked by it
    v[5] = -float("inf")
    v[5, vocab // 2] = -3.0                        # one token left
    v[6] = torch.arange(vocab, device="cuda").remainder(5).to(dtype)  # many equal ones
    v[7] = torch.arange(vocab, device="cuda").to(dtype)   # rising: the best are next to each other
    v[8] = -torch.arange(vocab, device="cuda").to(dtype)
    v[9, vocab - 20:] = 2.0
    targets = torch.zeros(10, dtype=torch.int64, device="cuda")
    targets[4], targets[5] = vocab - 1, vocab // 2
    if dtype == torch.float16 and vocab > 60000:
        v[7], v[8] = v[7].clamp(max=60000), v[8].clamp(min=-60000)
    got = run(gpu_ctx, v, targets, 1.0, 20)
    want = definition(v, targets, 1.0, 20)
    for k in ("lse", "logp", "entropy", "top_logp"):
        assert not torch.isnan(got[k]).any(), k
    z = v.double()
    fine = torch.where(torch.isfinite(z), z, torch.zeros_like(z)).abs().amax(1) < 1e30
    assert torch.equal(got["top_ids"], want["top_ids"])
    check({k: x[fine] for k, x in got.items()}, {k: x[fine] for k, x in want.items()}, v[fine], 1.0)
    # rows of the lowest value: differences of equal numbers are exact
    n = torch.log(torch.tensor(float(vocab)))
    assert abs(got["entropy"][3].item() - n.item()) < 1e-5 and abs(got["logp"][3].item() + n.item()) < 1e-5
    assert got["logp"][4] == 0 and got["entropy"][4] == 0 and got["logp"][2] == -float("inf")
    assert got["entropy"][2] == 0 and got["lse"][2] == -float("inf")


@pytest.mark.parametrize("rows", [1, 3, 130, 700])
@pytest.mark.parametrize("vocab", [511, 512, 513, 1543, 2041, 2057, 8200, 12969, 14847, 17493])
@pytest.mark.parametrize("top", [1, 5, 20, 64])
def test_alternatives_of_short_and_ragged_parts(gpu_ctx, rows, vocab, top):
    logits = (3.0 * normal(rows + vocab, rows, vocab)).bfloat16()
    if rows > 2:
        logits[1, 40:] = -float("inf")
        logits[2, : vocab - 10] = -float("inf")
    targets = torch.randint(vocab, (rows,), device="cuda")
    check(run(gpu_ctx, logits, targets, 1.0, top), definition(logits, targets, 1.0, top), logits, 1.0)


def test_not_finite(gpu_ctx):
    v = normal(1, 6, 3000)
    v[1, 2999], v[2, 5], v[3, 100] = float("nan"), float("inf"), -float("inf")
    v[4] = float("nan")
    got = run(gpu_ctx, v, torch.zeros(6, dtype=torch.int64, device="cuda"), 1.0, 3)
    bad = torch.tensor([False, True, True, False, True, False], device="cuda")
    for k in ("lse", "logp", "entropy"):
        assert torch.equal(torch.isnan(got[k]), bad), k
    assert got["top_ids"][1, 0] == 2999 and got["top_ids"][2, 0] == 5 and got["top_ids"][4].tolist() == [0, 1, 2]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,pad,offset", SIZES)
@pytest.mark.parametrize("scale,parts,banned", [(1.0, "both", True), (0.7, "logp", False), (2.0, "entropy", True)])
def test_gradient(gpu_ctx, dtype, rows, vocab, pad, offset, scale, parts, banned):
    v = 3.0 * normal(rows + vocab, rows, vocab)
    if banned:
        v[:, 1::3] = -float("inf")
    if rows > 6:
        v[4] = -float("inf")
    logits = place(v.to(dtype), pad, offset).t
    targets = torch.randint(vocab, (rows,), device="cuda")
    if rows > 2:
        targets[1], targets[2] = -100, vocab
    want = definition(logits, targets, scale, 0)
    gl, ge = normal(3, rows), normal(4, rows)
    use = {}
    if parts != "entropy":
        use |= dict(dlogp=gl, targets=targets)
    out = Guarded(rows, vocab, dtype, pad, offset)
    fwd = run(gpu_ctx, logits, targets, scale)
    if parts != "logp":
        use |= dict(dentropy=ge, entropy=fwd["entropy"])
    ops.TokenLogprobsBackward(gpu_ctx, logits=logits, lse=fwd["lse"], dlogits=out.t, scale=scale, **use)()
    ready()
    gone = logits == -float("inf")
    z = torch.where(gone, torch.zeros_like(logits), logits).double()
    z = (z * scale).detach().requires_grad_()
    masked = torch.where(gone, torch.full_like(z, -float("inf")), z)
    # the definition's derivative: softmax terms written out, ruled-out tokens and empty rows without any
    p = torch.where(gone, torch.zeros_like(z), want["p"])
    logp = torch.where(p == 0, torch.zeros_like(z), masked.detach() - want["lse"][:, None])
    asked = (targets >= 0) & (targets < vocab)
    hit = torch.zeros_like(p).scatter_(1, targets.clamp(0, vocab - 1)[:, None], asked.double()[:, None])
    terms = []
    if parts != "entropy":
        g = (gl.double() * asked)[:, None]
        terms += [g * hit, -g * p]
    if parts != "logp":
        terms += [-ge.double()[:, None] * p * logp, -ge.double()[:, None] * p * want["entropy"][:, None]]
    d = torch.where(gone, torch.zeros_like(p), scale * sum(terms))
    size = 2 * (z.detach().abs().amax(1) + want["lse"].abs().nan_to_num(0, 0, 0))
    e = U32 * (4 * size + 512)[:, None]
    mag = scale * sum(t.abs() for t in terms)
    # an error of lse or entropy shifts every term it is in
    shift = scale * p * (ge.double().abs()[:, None] * 2 * e * (2 + size[:, None])) if parts != "logp" else 0
    assert_close(out.t, d, torch.where(gone, torch.zeros_like(mag), e * mag + shift), "dlogits")
    assert out.untouched()


def test_gradient_against_differences(gpu_ctx):
    rows, vocab, scale = 4, 60, 0.8
    v = normal(1, rows, vocab)
    targets = torch.tensor([3, 59, -1, 0], device="cuda")
    gl, ge = normal(2, rows), normal(3, rows)
    fwd = run(gpu_ctx, v, targets, scale)
    d = torch.empty_like(v)
    ops.TokenLogprobsBackward(gpu_ctx, logits=v, lse=fwd["lse"], entropy=fwd["entropy"], targets=targets, dlogp=gl,
                              dentropy=ge, dlogits=d, scale=scale)()
    ready()

    def loss(x):
        w = definition(x, targets, scale, 0)
        return float((w["logp"] * gl.double()).sum() + (w["entropy"] * ge.double()).sum())

    for seed in range(5):
        step = 1e-5 * normal(10 + seed, rows, vocab).double()
        slope = (loss(v.double() + step) - loss(v.double() - step)) / 2
        size = float((d.double().abs() * step.abs()).sum())
        assert abs(slope - float((d.double() * step).sum())) <= 1e-4 * size + 1e-9


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_beside_masks_of_the_lowest_value(gpu_ctx, dtype, in_place):
    """A row of nothing but the type's lowest value spreads evenly; one left beside such a mask takes it all."""
    vocab, low = 20000, torch.finfo(dtype).min
    v = torch.full((3, vocab), low, device="cuda").to(dtype)
    v[1, 777], v[2, 5:9] = 2.0, -60.0
    targets, gl, ge = torch.tensor([9, 777, 6], device="cuda"), torch.ones(3, device="cuda"), torch.ones(3, device="cuda")
    fwd = run(gpu_ctx, v, targets)
    d = v if in_place else torch.empty_like(v)
    ops.TokenLogprobsBackward(gpu_ctx, logits=v, lse=fwd["lse"], entropy=fwd["entropy"], targets=targets, dlogp=gl,
                              dentropy=ge, dlogits=d)()
    ready()
    want = torch.zeros(3, vocab, dtype=torch.float64, device="cuda")
    want[0] = -1 / vocab
    want[0, 9] += 1
    want[2, 5:9] = -0.25
    want[2, 6] += 1
    # log p and entropy, both near 10 at most, each off by a few of their 32-bit steps, which p multiplies
    assert_close(d, want, 128 * U32 * (want.abs() + 1.0 / vocab), "dlogits")


def test_gradient_in_place(gpu_ctx):
    v = normal(1, 20, 3001).bfloat16()
    targets, gl = torch.arange(20, device="cuda"), normal(2, 20)
    fwd = run(gpu_ctx, v, targets)
    apart = torch.empty_like(v)
    ready()
    for out in (apart, v):
        ops.TokenLogprobsBackward(gpu_ctx, logits=v, lse=fwd["lse"], targets=targets, dlogp=gl, dlogits=out)()
    ready()
    assert torch.equal(apart, v)


def test_same_bytes_every_time_and_in_a_graph(gpu_ctx):
    from rns8_amd import hip

    v = normal(1, 5, 90001)
    targets = torch.arange(5, device="cuda")
    out = {k: torch.empty(5, device="cuda") for k in ("logp", "entropy", "lse")}
    out |= {"top_ids": torch.empty(5, 10, dtype=torch.int32, device="cuda"), "top_logp": torch.empty(5, 10, device="cuda")}
    call = ops.TokenLogprobs(gpu_ctx, logits=v, targets=targets, **out)
    ready()
    stream = hip.stream_create()
    try:
        hip.capture_begin(stream)
        call(stream)
        graph, exe = hip.capture_end(stream)
        try:
            for replay in range(4):
                v.copy_(normal(40 + replay // 2, 5, 90001))
                ready()
                hip.graph_launch(exe, stream)
                hip.stream_synchronize(stream)
                got = {k: x.clone() for k, x in out.items()}
                for x in out.values():
                    x.zero_()
                ready()
                call()
                ready()
                assert all(torch.equal(got[k], out[k]) for k in out)
        finally:
            hip.graph_destroy(graph, exe)
    finally:
        hip.stream_destroy(stream)


def test_refusals(gpu_ctx):
    v = torch.zeros(3, 50, device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    f = torch.zeros(3, device="cuda")
    ready()
    for kwargs in ({}, {"logp": f}, {"logp": f, "targets": t, "scale": 0.0}, {"lse": f, "scale": float("inf")},
                   {"top_logp": torch.zeros(3, 65, device="cuda")}, {"top_logp": torch.zeros(3, 51, device="cuda")}):
        with pytest.raises(r.Rns8Error) as e:
            ops.TokenLogprobs(gpu_ctx, logits=v, **kwargs)()
        assert e.value.status == r.abi.INVALID_ARGUMENT, kwargs
    with pytest.raises(r.Rns8Error):
        ops.TokenLogprobsBackward(gpu_ctx, logits=v, lse=f, dlogits=v)()


# masks' values and scales for which scale * value lies on both sides of 2^20 / log2(e), up to the type's limits
LARGE = [(-1e5, 1.0), (-7e5, 1.0), (-7.5e5, 1.0), (-1e6, 1.0), (-1e9, 1.0), (-1e10, 0.7), (-1e20, 1.0), (-1e36, 1000.0),
         (3e5, 1.0), (1e10, 1.0), (3e38, 1.0), (3e38, 0.5), (-3e4, 40.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value,scale", LARGE)
@pytest.mark.parametrize("vocab", [700, 70000])
def test_rows_of_one_large_value(gpu_ctx, dtype, value, scale, vocab):
    """Equal logits spread evenly however large they are; one that stands out by 2^-4 of the value takes everything.

    Differences of equal numbers are exact, so the logarithm of vocab (below 12, log2 below 17) is off by the sum's
    and the logarithm's few steps alone; lse has six roundings of |z| (scale's own among them)."""
    v = torch.full((3, vocab), value, device="cuda").to(dtype)
    v[1, vocab - 3] = value * (1 - 2.0 ** -4) if value < 0 else value
    if value > 0:
        v[1, :vocab - 3], v[1, vocab - 2:] = value * (1 - 2.0 ** -4), -value
    v[2, ::2] = -float("inf")
    targets = torch.tensor([7, vocab - 3, 1], device="cuda")
    fwd = run(gpu_ctx, v, targets, scale, 3)
    n = torch.log(torch.tensor([vocab, 1.0, vocab / 2], dtype=torch.float64))
    assert_close(fwd["logp"].cpu(), -n, 128 * U32, "logp")
    assert_close(fwd["entropy"].cpu(), n, 128 * U32, "entropy")
    z = v.double().amax(1).cpu() * scale
    fits = z.abs() < 3.4e38
    assert ((fwd["lse"].cpu().double() - z - n).abs() <= 8 * U32 * z.abs() + 128 * U32)[fits].all()
    assert fwd["top_ids"].tolist() == [[0, 1, 2], [vocab - 3, 0, 1], [1, 3, 5]]
    assert (fwd["top_logp"][:, 0].cpu().double() + n).abs().max() <= 128 * U32
    if not fits.all():
        return
    ones, d = torch.ones(3, device="cuda"), torch.empty_like(v)
    ops.TokenLogprobsBackward(gpu_ctx, logits=v, lse=fwd["lse"], entropy=fwd["entropy"], targets=targets, dlogp=ones,
                              dentropy=ones, dlogits=d, scale=scale)()
    ready()
    want = torch.zeros(3, vocab, dtype=torch.float64, device="cuda")
    want[0], want[2, 1::2] = -scale / vocab, -2 * scale / vocab
    want[0, 7] += scale
    want[2, 1] += scale
    p = torch.zeros_like(want)
    p[0], p[1, vocab - 3], p[2, 1::2] = 1 / vocab, 1.0, 2 / vocab
    # log p, entropy and p itself, each off as above
    assert_close(d, want, 3 * 128 * U32 * scale * p + U32 * want.abs(), "dlogits")


def test_maxima_that_rise_past_the_fused_range(gpu_ctx):
    """Logits that rise from -1e10 to 1e10 along a row: each part's sums follow maxima of every size."""
    up = torch.logspace(0, 10, 4500, device="cuda", dtype=torch.float64).float()
    v = torch.cat((-up.flip(0), up, up[-1:]))[None].repeat(2, 1)
    v[1] = v[1].flip(0)
    top = torch.tensor([9000, 1], device="cuda")
    fwd = run(gpu_ctx, v, top, 1.0, 3)
    assert (fwd["logp"].double() + torch.log(torch.tensor(2.0))).abs().max() <= 128 * U32
    assert (fwd["entropy"].double() - torch.log(torch.tensor(2.0))).abs().max() <= 128 * U32
    assert fwd["top_ids"].tolist() == [[8999, 9000, 8998], [0, 1, 2]]
