"""Shared pieces of the operator tests: device tensors with guarded surroundings, the definitions in 64 bits, tolerances."""
import torch

U32 = 2.0 ** -24
UNIT = {torch.float32: U32, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# the least spacing of a type: what an underflowing result may be off
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


class Guarded:
    """rows x cols elements at a stride and an offset inside a buffer of a known filling, which has to survive."""

    def __init__(self, rows, cols, dtype, pad=0, offset=0, fill=77):
        self.rows, self.cols, self.ld, self.at = rows, cols, cols + pad, 64 + offset
        self.buf = torch.full((self.at + rows * self.ld + 64,), fill, dtype=dtype, device="cuda")
        self.was = self.buf.clone()
        self.t = torch.as_strided(self.buf, (rows, cols), (self.ld, 1), self.at)

    def untouched(self, cols=None):
        """Whether nothing outside the first `cols` columns of the rows changed."""
        now = self.buf.clone()
        kept = torch.as_strided(now, (self.rows, cols or self.cols), (self.ld, 1), self.at)
        kept.copy_(torch.as_strided(self.was, kept.shape, kept.stride(), self.at))
        return torch.equal(now.view(torch.uint8), self.was.view(torch.uint8))


def place(values, pad=0, offset=0):
    """`values` in a guarded buffer whose surroundings hold NaN (or -99 for bytes): reads outside would show."""
    fill = -99 if values.dtype == torch.int8 else float("nan")
    g = Guarded(values.shape[0], values.shape[1], values.dtype, pad, offset, fill)
    g.t.copy_(values)
    g.was = g.buf.clone()
    return g


def quantize(v, dim):
    """The definition of the 8-bit form in 32-bit operations, which round the same way everywhere: bytes and scales."""
    amax = v.abs().amax(dim, keepdim=True)
    most = torch.full_like(amax, 127.0)  # (a tensor: by a number torch multiplies with the reciprocal)
    fine, live = torch.isfinite(amax), amax >= 2.0 ** -100
    inverse = torch.where(fine & live, most / amax, torch.zeros_like(amax))
    q = torch.where(inverse == 0, torch.zeros_like(v), torch.round(v * inverse))
    scale = torch.where(fine, torch.where(live, amax / most, torch.zeros_like(amax)), torch.full_like(amax, float("nan")))
    return q.to(torch.int8), scale.squeeze(dim)


def assert_close(got, want, slack, what=""):
    """|got - want| within got's rounding of `want` plus `slack` (both in 64 bits); NaN and infinity where `want` has them."""
    g, w = got.double(), want.double()
    assert torch.equal(torch.isnan(g), torch.isnan(w)), f"{what}: NaN in other places"
    limit = UNIT[got.dtype] * 1.01 * w.abs() + slack * (1 + UNIT[got.dtype]) + TINY[got.dtype]
    fine = torch.isfinite(w)
    assert torch.equal(g[~fine & ~torch.isnan(w)], w[~fine & ~torch.isnan(w)]), f"{what}: other infinities"
    over = ((g - w).abs() > limit) & fine
    if over.any():
        at = int(over.flatten().nonzero()[0])
        raise AssertionError(f"{what}: {int(over.sum())} of {w.numel()} values off, first at {at}: "
                             f"{g.flatten()[at].item()} for {w.flatten()[at].item()}")
