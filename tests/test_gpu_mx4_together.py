"""Operators on 4-bit microscaled matrices together: a decoding step, a training step, graphs and streams."""
import pytest
import torch

import mx4_cases as mx4
from operator_cases import TYPES, U32, assert_close
from rns8_amd import operators as ops
from test_gpu_mx4 import normal, product_limit, ready
from test_gpu_mx4_experts import Experts, chosen

pytestmark = pytest.mark.gpu


def empty(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def one_runtime():
    if len({line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line}) != 1:
        pytest.skip("torch was loaded after the library: two HIP runtimes, whose streams differ")


class Decode:
    """A block's last half and the answer: norm, experts, residual and norm, the vocabulary's layer, log-probabilities."""

    def __init__(self, ctx, tokens, dtype, width=512, inner=256, vocab=1000):
        self.layer = Experts(3, 8, width, inner)
        self.head, self.head_value = mx4.matrix(normal(9, vocab, width) / width ** 0.5)
        self.vocab = vocab
        self.h, self.router = normal(1, tokens, width).to(dtype), (normal(2, 8, width) / width ** 0.5).to(dtype)
        self.weight = (1 + 0.1 * normal(4, width)).to(dtype)
        self.y, self.mixed, self.sum, self.last = (empty(tokens, width, dtype=dtype) for _ in range(4))
        self.logits, self.logp, self.lse = empty(tokens, vocab, dtype=dtype), empty(tokens), empty(tokens)
        self.ids, self.gates = torch.empty(tokens, 2, dtype=torch.int32, device="cuda"), empty(tokens, 2)
        self.targets = torch.arange(tokens, device="cuda")
        norm = dict(flags=ops.NORM_PRE, eps=1e-6, pre_weight=self.weight)
        self.calls = [
            ops.BlockNorm(ctx, x=self.h, y=self.y, **norm),
            ops.ExpertsMx4(ctx, x=self.y, router=self.router, **self.layer.bytes, inner=inner, out=self.mixed, ids=self.ids,
                           weights=self.gates),
            ops.BlockNorm(ctx, x=self.mixed, residual=self.h, h=self.sum, y=self.last, **norm),
            ops.LinearMx4(ctx, x=self.last, w=self.head, out=self.logits),
            ops.TokenLogprobs(ctx, logits=self.logits, targets=self.targets, logp=self.logp, lse=self.lse)]
        self.results = (self.y, self.mixed, self.sum, self.last, self.logits, self.logp, self.lse, self.ids, self.gates)

    def run(self, stream=None):
        for call in self.calls:
            call(stream) if stream is not None else call()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 7, 40])
def test_a_decoding_step(gpu_ctx, dtype, tokens):
    d = Decode(gpu_ctx, tokens, dtype)
    ready()
    d.run()
    ready()
    scores = (d.y.double() @ d.router.double().t()).float()
    ids, _ = chosen(scores, 2, True)
    assert torch.equal(d.ids.long(), ids)
    want, limit = d.layer.expected(d.y, ids, d.gates)
    assert_close(d.mixed, want, limit, "experts")
    _, rows = mx4.matrix(d.last)
    assert_close(d.logits, rows @ d.head_value.t().contiguous(), product_limit(rows, d.head_value, rows.shape[1]), "logits")
    z = d.logits.double()
    logp = torch.log_softmax(z, 1).gather(1, d.targets[:, None])[:, 0]
    # an exponential's argument is off by four units of the logits' spread, the sum and its logarithm by 544
    assert_close(d.logp, logp, U32 * (4 * (z.amax(1) - z.amin(1) - logp) + 544), "log-probabilities")
    one_by_one = [t.clone() for t in d.results]
    for t in d.results:
        t.zero_()
    ready()
    for call in d.calls:
        call()
        ready()
    assert all(torch.equal(a, b) for a, b in zip(one_by_one, d.results))


class Train:
    """A step of a layer under cross-entropy, its weights kept in floats and rounded anew."""

    def __init__(self, ctx, tokens, dtype, width=300, vocab=700):
        self.x, self.w, self.b = normal(1, tokens, width).to(dtype), normal(2, vocab, width) / width ** 0.5, normal(3, vocab)
        self.targets = torch.arange(tokens, device="cuda") % vocab
        self.q, self.q_t = (torch.empty(ops.mx4_bytes(*s), dtype=torch.uint8, device="cuda") for s in
                            ((vocab, width), (width, vocab)))
        self.logits, self.dlogits = empty(tokens, vocab, dtype=dtype), empty(tokens, vocab, dtype=dtype)
        self.logp, self.lse = empty(tokens), empty(tokens)
        self.dlogp = torch.full((tokens,), -1.0 / tokens, device="cuda")
        self.dx, self.dw, self.db = empty(tokens, width, dtype=dtype), empty(vocab, width), empty(vocab)
        self.calls = [
            ops.QuantizeMx4(ctx, x=self.w, q=self.q, q_t=self.q_t),
            ops.LinearMx4(ctx, x=self.x, w=self.q, bias=self.b, out=self.logits),
            ops.TokenLogprobs(ctx, logits=self.logits, targets=self.targets, logp=self.logp, lse=self.lse),
            ops.TokenLogprobsBackward(ctx, logits=self.logits, targets=self.targets, lse=self.lse, dlogp=self.dlogp,
                                      dlogits=self.dlogits),
            ops.LinearMx4Backward(ctx, dy=self.dlogits, x=self.x, w_t=self.q_t, dx=self.dx, dw=self.dw, dbias=self.db)]
        self.results = (self.q, self.q_t, self.logits, self.logp, self.dlogits, self.dx, self.dw, self.db)

    run = Decode.run


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 64, 500])
def test_a_training_step(gpu_ctx, dtype, tokens):
    t = Train(gpu_ctx, tokens, dtype)
    ready()
    t.run()
    ready()
    (q, wv), (q_t, wtv) = mx4.matrix(t.w), mx4.matrix(t.w.t())
    assert torch.equal(t.q, q) and torch.equal(t.q_t, q_t)
    xv, gv = mx4.matrix(t.x)[1], mx4.matrix(t.dlogits)[1]
    xtv, gtv = mx4.matrix(t.x.t())[1], mx4.matrix(t.dlogits.t())[1]
    width, vocab = t.x.shape[1], t.b.numel()
    off = product_limit(xv, wv, width) + 2.0 ** -23 * t.b.double().abs()
    assert_close(t.logits, xv @ wv.t().contiguous() + t.b.double(), off, "logits")
    assert_close(t.dx, gv @ wtv.t().contiguous(), product_limit(gv, wtv, vocab), "dx")
    assert_close(t.dw, gtv @ xtv.t().contiguous(), product_limit(gtv, xtv, tokens), "dw")
    assert_close(t.db, t.dlogits.double().sum(0), (tokens + 8) * 2.0 ** -24 * t.dlogits.double().abs().sum(0), "dbias")


@pytest.mark.parametrize("make", [lambda c: Decode(c, 1, torch.bfloat16), lambda c: Decode(c, 40, torch.bfloat16),
                                  lambda c: Train(c, 300, torch.bfloat16), lambda c: Train(c, 3000, torch.float32)],
                         ids=["decode1", "decode40", "train300", "train3000"])
def test_captured_steps(gpu_ctx, make):
    """Two graphs, replayed in turn with eager steps and waits between, on inputs that change."""
    one_runtime()
    steps = make(gpu_ctx), make(gpu_ctx)
    stream = torch.cuda.Stream()
    graphs = []
    ready()
    for step in steps:
        step.run(stream.cuda_stream)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    for turn in range(4):
        for step, graph in zip(steps, graphs):
            source = step.h if isinstance(step, Decode) else step.x
            source.copy_(normal(100 + turn, *source.shape))
            for t in step.results:
                t.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in step.results]
            for t in step.results:
                t.zero_()
            torch.cuda.synchronize()
            step.run()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, step.results))
            assert all(t.any() for t in got)


def test_steps_on_two_streams_at_once(gpu_ctx):
    one_runtime()
    steps = [Decode(gpu_ctx, 16, torch.bfloat16), Train(gpu_ctx, 500, torch.bfloat16)]
    want = []
    ready()
    for step in steps:
        step.run()
        ready()
        want.append([t.clone() for t in step.results])
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(20):
        for step, stream in zip(steps, streams):
            step.run(stream.cuda_stream)
    torch.cuda.synchronize()
    for step, values in zip(steps, want):
        assert all(torch.equal(a, b) for a, b in zip(step.results, values))


def test_on_the_default_stream(gpu_ctx):
    """Behind torch's work there and before what follows."""
    one_runtime()
    step = Decode(gpu_ctx, 5, torch.bfloat16)
    big = torch.randn(8192, 8192, device="cuda")
    big @ big
    first = step.h.clone()
    ready()
    step.run()
    ready()
    want = [t.clone() for t in step.results]
    step.h.zero_()
    for _ in range(4):  # some milliseconds
        big @ big
    step.h.copy_(first)
    step.run(torch.cuda.current_stream().cuda_stream)
    got = [t.clone() for t in step.results]
    ready()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
