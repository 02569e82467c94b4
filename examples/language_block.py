"""The language-model operators together: a small model trained in 8-bit products, then used token by token.

    python examples/language_block.py [steps]

The model reads one token and predicts the next: an embedding, a norm, one
8-bit linear layer as the residual block, the norms after and before a block,
and an 8-bit linear layer into the vocabulary. Its data is a rule,
next = (5 token + 3) mod vocab, so the result can be checked: the loss falls to
near zero, and decoding follows the rule. Master weights and their gradients are
32-bit tensors that torch's optimizer steps; rns8_mi355x_quantize_rows turns them
into 8-bit weights after each step. Everything runs on one stream, and training
steps and decoding make the same calls again and again on memory of their own.
"""
import sys
from pathlib import Path

import torch  # before the library loads: both then share one HIP runtime

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import rns8_amd  # noqa: E402
from rns8_amd import operators as ops  # noqa: E402

VOCAB, WIDTH, BATCH = 1000, 256, 500
DTYPE = torch.bfloat16


def rule(token):
    return (5 * token + 3) % VOCAB


class Weights:
    """32-bit master weights and what the operators read: 8-bit rows with a scale each, norm weights in bf16."""

    def __init__(self, ctx, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape):
            return torch.randn(*shape, generator=gen, device="cuda")

        self.embedding = normal(VOCAB, WIDTH).to(DTYPE)
        self.master = {"block": normal(WIDTH, WIDTH) / WIDTH**0.5, "head": normal(VOCAB, WIDTH) / WIDTH**0.5}
        self.norms = {name: torch.ones(WIDTH, device="cuda") for name in ("first", "post", "pre", "gate")}
        self.parameters = [*self.master.values(), *self.norms.values()]
        for p in self.parameters:
            p.grad = torch.zeros_like(p)
        self.q, self.scale, self.low, self.calls = {}, {}, {}, []
        for name, w in self.master.items():
            q = torch.empty(w.shape[0], ops.padded(w.shape[1]), dtype=torch.int8, device="cuda")
            self.scale[name] = torch.empty(w.shape[0], device="cuda")
            self.q[name] = q[:, : w.shape[1]]
            self.calls.append(ops.QuantizeRows(ctx, x=w, q=q, scale=self.scale[name]))
        for name, w in self.norms.items():
            self.low[name] = w.to(DTYPE)

    def refresh(self, stream):
        """The operators' weights from the master weights."""
        for call in self.calls:
            call(stream)
        for name, w in self.norms.items():
            self.low[name].copy_(w)


class Model:
    """The calls for `rows` tokens at a time, on buffers that they share."""

    def __init__(self, ctx, weights, rows, top=0, train=False):
        def empty(*shape, dtype=DTYPE):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        w, f32 = weights, torch.float32
        self.weights = w
        self.tokens, self.targets = (empty(rows, dtype=torch.int64) for _ in range(2))
        self.stream_in, y0, u, h, y1 = (empty(rows, WIDTH) for _ in range(5))
        logits = empty(rows, VOCAB)
        rstd0, rstd1 = empty(2 * rows, dtype=f32), empty(2 * rows, dtype=f32)
        q0, q1 = (empty(rows, ops.padded(WIDTH), dtype=torch.int8)[:, :WIDTH] for _ in range(2))
        s0, s1 = empty(rows, dtype=f32), empty(rows, dtype=f32)
        self.logp, self.entropy, lse = (empty(rows, dtype=f32) for _ in range(3))
        self.top_ids = empty(rows, top, dtype=torch.int32) if top else None
        around = dict(residual=self.stream_in, gate=w.low["gate"], post_weight=w.low["post"], pre_weight=w.low["pre"])
        saved0, saved1 = (dict(x_q=q0, x_scale=s0), dict(x_q=q1, x_scale=s1)) if train else ({}, {})
        self.forward = [
            ops.BlockNorm(ctx, x=self.stream_in, pre_weight=w.low["first"], y=y0, rstd=rstd0, flags=ops.NORM_PRE),
            ops.LinearI8(ctx, x=y0, w=w.q["block"], w_scale=w.scale["block"], out=u, **saved0),
            ops.BlockNorm(ctx, x=u, h=h, y=y1, rstd=rstd1, **around),
            ops.LinearI8(ctx, x=y1, w=w.q["head"], w_scale=w.scale["head"], out=logits, **saved1),
            ops.TokenLogprobs(ctx, logits=logits, targets=self.targets, logp=self.logp, entropy=self.entropy, lse=lse,
                              top_ids=self.top_ids),
        ]
        self.backward = []
        if train:
            dlogits, dy1, du, dy0 = empty(rows, VOCAB), empty(rows, WIDTH), empty(rows, WIDTH), empty(rows, WIDTH)
            dlogp = torch.full((rows,), -1.0 / rows, device="cuda")  # the loss is the mean of -logp
            grad = {name: p.grad for name, p in (w.master | w.norms).items()}
            self.backward = [
                ops.TokenLogprobsBackward(ctx, logits=logits, lse=lse, targets=self.targets, dlogp=dlogp,
                                          dlogits=dlogits),
                ops.LinearI8Backward(ctx, dy=dlogits, x_q=q1, x_scale=s1, w=w.q["head"], w_scale=w.scale["head"],
                                     dx=dy1, dw=grad["head"]),
                ops.BlockNormBackward(ctx, x=u, rstd=rstd1, dy=dy1, dx=du, dgate=grad["gate"],
                                      dpost_weight=grad["post"], dpre_weight=grad["pre"], **around),
                ops.LinearI8Backward(ctx, dy=du, x_q=q0, x_scale=s0, w=w.q["block"], w_scale=w.scale["block"], dx=dy0,
                                     dw=grad["block"]),
                ops.BlockNormBackward(ctx, x=self.stream_in, rstd=rstd0, pre_weight=w.low["first"], dy=dy0,
                                      dpre_weight=grad["first"], flags=ops.NORM_PRE),
            ]

    def __call__(self, tokens, stream):
        self.tokens.copy_(tokens)
        torch.index_select(self.weights.embedding, 0, self.tokens, out=self.stream_in)
        for call in self.forward + self.backward:
            call(stream)


def train(ctx, weights, steps, stream, report=None):
    """The loss of every step."""
    model = Model(ctx, weights, BATCH, train=True)
    optimizer = torch.optim.Adam(weights.parameters, lr=0.01)
    gen = torch.Generator(device="cuda").manual_seed(1)
    losses = []
    for step in range(steps):
        weights.refresh(stream)
        tokens = torch.randint(VOCAB, (BATCH,), generator=gen, device="cuda")
        model.targets.copy_(rule(tokens))
        model(tokens, stream)
        losses.append(-model.logp.mean())
        optimizer.step()
        if report and step % 20 == 0:
            report(f"step {step}: loss {losses[-1].item():.4f}")
    weights.refresh(stream)
    return [float(x) for x in losses]


def decode(ctx, weights, first, count, stream):
    """The most likely continuation of one token: one-token calls, each from what the last one wrote."""
    model = Model(ctx, weights, 1, top=4)
    token = torch.tensor([first], device="cuda")
    model.targets.fill_(-1)  # no token's log-probability is asked for
    out = []
    for _ in range(count):
        model(token, stream)
        token = model.top_ids[:, 0].long()
        out.append(token)
    return torch.cat(out).tolist()


def main(steps=200, report=None):
    """(losses, decoded tokens, the rule's tokens)"""
    ctx = rns8_amd.Context(0)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        weights = Weights(ctx, 0)
        losses = train(ctx, weights, steps, stream.cuda_stream, report)
        decoded = decode(ctx, weights, 7, 12, stream.cuda_stream)
    stream.synchronize()
    expected, token = [], 7
    for _ in range(12):
        token = rule(token)
        expected.append(token)
    return losses, decoded, expected


if __name__ == "__main__":
    losses, decoded, expected = main(int(sys.argv[1]) if len(sys.argv) > 1 else 200, print)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.4f}")
    print("decoded ", *decoded)
    print("the rule", *expected)
