"""The language-model operators at sizes and arguments at the edge of what they take."""
import pytest
import torch

from operator_cases import Guarded, quantize
from rns8_amd import operators as ops

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def ready():
    torch.cuda.synchronize()  # the library's stream does not wait for torch's


@pytest.mark.parametrize("m", [1, 2, 3, 70])
@pytest.mark.parametrize("k", [15, 64, 8192, 8200])
@pytest.mark.parametrize("keep", [False, True])
def test_a_layer_without_channels(gpu_ctx, m, k, keep):
    """There is no output; rows that are kept are the quantization's own."""
    x, nothing = normal(m + k, m, k).bfloat16(), torch.empty(0, device="cuda")
    more = {}
    if keep:
        kept, scale = Guarded(m, ops.padded(k), torch.int8), torch.empty(m, device="cuda")
        more = dict(x_q=kept.t, x_scale=scale)
    ready()
    ops.LinearI8(gpu_ctx, x=x, w=torch.empty(0, k, dtype=torch.int8, device="cuda"), w_scale=nothing,
                 out=torch.empty(m, 0, dtype=x.dtype, device="cuda"), **more)()
    ready()
    if keep:
        q, s = quantize(x.float(), 1)
        assert torch.equal(kept.t[:, :k], q) and torch.equal(scale, s) and kept.untouched()


def test_on_the_default_stream(gpu_ctx):
    """The handle that torch gives for its default stream: behind torch's work there, and before what follows."""
    if len({line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line}) != 1:
        pytest.skip("torch was loaded after the library: two HIP runtimes, whose streams differ")
    handle = torch.cuda.current_stream().cuda_stream
    assert handle == 0
    big = torch.randn(8192, 8192, device="cuda")
    x, scale = torch.zeros(300, 512, device="cuda"), torch.zeros(300, device="cuda")
    call = ops.QuantizeRows(gpu_ctx, x=x, q=torch.empty(300, 512, dtype=torch.int8, device="cuda"), scale=scale)
    big @ big
    ready()
    got = []
    for value in (3.0, 5.0, 7.0):
        for _ in range(4):  # some milliseconds
            big @ big
        x.fill_(value)
        call(handle)
        got.append(scale.clone())
    ready()
    for value, scale in zip((3.0, 5.0, 7.0), got):
        assert torch.equal(scale, torch.full_like(scale, value) / torch.full_like(scale, 127.0))
