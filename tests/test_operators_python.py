"""The operators' Python classes without a device: what they check of tensors, and the strides that they hand on."""
from pathlib import Path

import pytest

from rns8_amd import abi

torch = pytest.importorskip("torch")

if not (Path(__file__).resolve().parent.parent / "rns8_amd" / "librns8.so").exists():
    pytest.skip("librns8.so not built (run __graft_entry__.build())", allow_module_level=True)

from rns8_amd import operators as ops  # noqa: E402


class Device:
    """A tensor of host memory that says it is in device memory."""

    is_cuda = True

    def __init__(self, t, index=0):
        self.t = t
        self.device = type("device", (), {"index": index})()

    def __getattr__(self, name):
        return getattr(self.t, name)


class Context:
    ptr = None

    def device_info(self):
        return type("Info", (), {"device_id": 0})()


def quantized(q, rows, cols, kind="rows"):
    """The stride that a call hands on for its quantized rows `q`."""
    f32 = Device(torch.zeros(rows, cols))
    scale = Device(torch.zeros(rows))
    q = Device(q)
    if kind == "rows":
        return ops.QuantizeRows(Context(), x=f32, q=q, scale=scale).args.ldq
    if kind == "columns":
        columns = Device(torch.zeros(cols, rows))
        return ops.QuantizeColumns(Context(), x=columns, q=q, scale=scale, workspace=scale).args.ldq
    if kind == "norm":
        return ops.BlockNorm(Context(), x=f32, q=q, q_scale=scale).args.ldq
    w, out = Device(torch.zeros(8, cols, dtype=torch.int8)), Device(torch.zeros(rows, 8))
    return ops.LinearI8(Context(), x=f32, w=w, w_scale=Device(torch.zeros(8)), out=out, x_q=q, x_scale=scale,
                        workspace=scale).args.ldq


def buffer(*shape):
    return torch.zeros(*shape, dtype=torch.int8)


@pytest.mark.parametrize("kind", ["rows", "columns", "norm", "linear"])
def test_zeros_after_quantized_rows_stay_in_the_storage(kind):
    """They go on to 16 bytes or the next row, also past the columns of a view; the last row's may have no room."""
    assert quantized(buffer(5, 16), 5, 6, kind) == 16
    assert quantized(buffer(5, 16)[:, :6], 5, 6, kind) == 16
    assert quantized(buffer(5, 6), 5, 6, kind) == 6
    assert quantized(buffer(5, 20)[:, 4:10], 5, 6, kind) == 20
    assert quantized(buffer(6, 16)[:5, 10:], 5, 6, kind) == 16
    with pytest.raises(ValueError, match="zeros"):
        quantized(buffer(5, 16)[:, 10:], 5, 6, kind)
    with pytest.raises(ValueError, match="zeros"):
        quantized(buffer(5, 20)[:, 8:14], 5, 6, kind)
    # one row has no next: it keeps its room, or does without
    assert quantized(buffer(1, 16)[:, :6], 1, 6, kind) == 16
    assert quantized(buffer(5, 16)[4:, 10:], 1, 6, kind) == 6
    assert quantized(buffer(6).as_strided((1, 6), (1000, 1)), 1, 6, kind) == 6


def test_rows_that_are_only_read_need_no_room():
    dy, w = Device(torch.zeros(5, 8)), Device(torch.zeros(8, 6, dtype=torch.int8))
    call = ops.LinearI8Backward(Context(), dy=dy, x_q=Device(buffer(5, 16)[:, 10:]), x_scale=Device(torch.zeros(5)), w=w,
                                w_scale=Device(torch.zeros(8)), dw=Device(torch.zeros(8, 6)),
                                workspace=Device(torch.zeros(1)))
    assert call.args.ldq == 16 and call.args.dtype == abi.F32


@pytest.mark.parametrize("what", ["device", "host", "strides"])
def test_workspaces_that_a_call_cannot_use(what):
    x, w = Device(torch.zeros(70, 64)), Device(torch.zeros(80, 64, dtype=torch.int8))
    layer = dict(x=x, w=w, w_scale=Device(torch.zeros(80)), out=Device(torch.zeros(70, 80)))
    given = {"device": Device(torch.zeros(1 << 16), index=1), "host": torch.zeros(1 << 16),
             "strides": Device(torch.zeros(1 << 16, 2)[:, 0])}[what]
    with pytest.raises(ValueError, match="workspace"):
        ops.LinearI8(Context(), **layer, workspace=given)
    ops.LinearI8(Context(), **layer, workspace=Device(torch.zeros(1 << 16)))
