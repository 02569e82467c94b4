"""The operators on 4-bit microscaled matrices without a device: structs against the header, refusals and workspaces."""
from __future__ import annotations

import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

from rns8_amd import abi

ROOT = Path(__file__).resolve().parent.parent
STRUCTS = {"mx4": abi.Mx4Args, "pack_mx4": abi.PackMx4Args, "gemm_mx4": abi.GemmMx4Args, "linear_mx4": abi.LinearMx4Args,
           "linear_mx4_backward": abi.LinearMx4BackwardArgs, "experts_mx4": abi.ExpertsMx4Args}


def test_structs_mirror_the_header(tmp_path):
    compiler = shutil.which("g++")
    if not compiler:
        pytest.skip("no host compiler")
    lines, want = [], []
    for name, mirror in STRUCTS.items():
        c = f"rns8_mi355x_{name}_args"
        lines.append(f'std::printf("{name} %zu\\n", sizeof({c}));')
        want.append(f"{name} {C.sizeof(mirror)}")
        for field, *_ in mirror._fields_:
            d = getattr(mirror, field)
            lines.append(f'std::printf("{name}.{field} %zu %zu\\n", offsetof({c}, {field}), sizeof({c}::{field}));')
            want.append(f"{name}.{field} {d.offset} {d.size}")
    for rows, cols in ((0, 5), (1, 1), (16, 256), (17, 257), (2**31 - 300, 2**31 - 300)):
        lines.append(f'std::printf("bytes %llu\\n", (unsigned long long)RNS8_MI355X_MX4_BYTES({rows}ll, {cols}ll));')
        want.append(f"bytes {-(-rows // 16) * -(-cols // 256) * 2176}")
    lines.append('std::printf("%d %u\\n", RNS8_MI355X_MX4_UNIT, RNS8_MI355X_EXPERTS_NORMALIZE);')
    want.append(f"{abi.MX4_UNIT} {abi.EXPERTS_NORMALIZE}")
    source = tmp_path / "layout.cpp"
    source.write_text("#include <cstddef>\n#include <cstdio>\n#include \"rns8_mi355x.h\"\nint main() {\n" + "\n".join(lines) + "\n}\n")
    subprocess.run([compiler, "-std=c++17", f"-I{ROOT / 'include'}", str(source), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split("\n")
    assert [line for line in got if line] == want


@pytest.fixture(scope="module")
def lib():
    if not (ROOT / "rns8_amd" / "librns8.so").exists():
        pytest.skip("librns8.so not built (run __graft_entry__.build())")
    import rns8_amd

    return rns8_amd.lib()


P = 1 << 20  # an address that nothing here reads
GEMM = dict(dtype=abi.F32, m=300, n=500, k=256, a=P, b=P, out=P, ldo=500)
LINEAR = dict(dtype=abi.BF16, m=300, n=500, k=256, x=P, ldx=256, w=P, out=P, ldo=500)
BACK = dict(dtype=abi.F16, m=300, n=500, k=256, dy=P, lddy=500, x=P, ldx=256, w_t=P, dx=P, lddx=256, dw=P, lddw=256, dbias=P)
EXPERTS = dict(dtype=abi.BF16, tokens=20, experts=8, width=512, inner=256, top=2, x=P, ldx=512, router=P, ldrouter=512, gate=P,
               up=P, down=P, out=P, ldo=512, ids=P, weights=P)
CALLS = {"gemm_mx4": (abi.GemmMx4Args, GEMM), "linear_mx4": (abi.LinearMx4Args, LINEAR),
         "linear_mx4_backward": (abi.LinearMx4BackwardArgs, BACK), "experts_mx4": (abi.ExpertsMx4Args, EXPERTS)}


def query(lib, name, **change):
    struct, fields = CALLS[name]
    args = abi.new_struct(struct)
    for k, v in (fields | change).items():
        setattr(args, k, v)
    need = C.c_uint64(77)
    return getattr(lib, f"rns8_mi355x_{name}_workspace")(C.byref(args), C.byref(need)), need.value


@pytest.mark.parametrize("name", CALLS)
def test_queries_answer(lib, name):
    status, need = query(lib, name)
    assert status == abi.SUCCESS and need < 2**26
    assert query(lib, name) == (status, need)


@pytest.mark.parametrize("name,change", [
    ("gemm_mx4", dict(dtype=3)), ("gemm_mx4", dict(abi_version=0)), ("gemm_mx4", dict(struct_size=8)), ("gemm_mx4", dict(m=-1)),
    ("gemm_mx4", dict(n=-1)), ("gemm_mx4", dict(k=-1)), ("gemm_mx4", dict(a=0)), ("gemm_mx4", dict(b=P + 8)),
    ("gemm_mx4", dict(out=0)), ("gemm_mx4", dict(ldo=499)), ("gemm_mx4", dict(out=P + 2)), ("gemm_mx4", dict(bias=P + 3)),
    ("linear_mx4", dict(k=0)), ("linear_mx4", dict(x=0)), ("linear_mx4", dict(x=P + 1)), ("linear_mx4", dict(ldx=255)),
    ("linear_mx4", dict(w=0)), ("linear_mx4", dict(w=P + 2)), ("linear_mx4", dict(ldo=2**62)),
    ("linear_mx4_backward", dict(n=0)), ("linear_mx4_backward", dict(k=0)), ("linear_mx4_backward", dict(dx=0, dw=0, dbias=0)),
    ("linear_mx4_backward", dict(x=0)), ("linear_mx4_backward", dict(w_t=0)), ("linear_mx4_backward", dict(dy=0)),
    ("linear_mx4_backward", dict(dw=P + 2)), ("linear_mx4_backward", dict(lddw=255)), ("linear_mx4_backward", dict(dbias=P + 1)),
    ("experts_mx4", dict(top=0)), ("experts_mx4", dict(top=9)), ("experts_mx4", dict(flags=2)), ("experts_mx4", dict(tokens=-1)),
    ("experts_mx4", dict(experts=0)), ("experts_mx4", dict(width=0)), ("experts_mx4", dict(inner=0)),
    ("experts_mx4", dict(router=0, ids=0)), ("experts_mx4", dict(router=0, weights=0)), ("experts_mx4", dict(gate=0)),
    ("experts_mx4", dict(up=P + 4)), ("experts_mx4", dict(down=0)), ("experts_mx4", dict(ids=P + 2)),
    ("experts_mx4", dict(ldrouter=511)), ("experts_mx4", dict(x=0))])
def test_invalid_arguments(lib, name, change):
    status, need = query(lib, name, **change)
    assert status == abi.INVALID_ARGUMENT and need in (0, 77)


@pytest.mark.parametrize("name,change", [
    ("gemm_mx4", dict(k=2**23 + 1)), ("gemm_mx4", dict(m=2**31 - 256)), ("gemm_mx4", dict(n=2**31, ldo=2**31)),
    ("linear_mx4", dict(k=2**23 + 1, ldx=2**23 + 1)), ("linear_mx4", dict(m=2**31)),
    ("linear_mx4_backward", dict(m=2**23 + 1)), ("linear_mx4_backward", dict(n=2**23 + 1, lddy=2**23 + 1)),
    ("linear_mx4_backward", dict(k=2**31, ldx=2**31, lddx=2**31, lddw=2**31)),
    ("experts_mx4", dict(tokens=65)), ("experts_mx4", dict(experts=1025)), ("experts_mx4", dict(top=17, experts=20)),
    ("experts_mx4", dict(width=65537, ldx=65537, ldo=65537, ldrouter=65537)), ("experts_mx4", dict(inner=65537))])
def test_sizes_past_the_limits(lib, name, change):
    assert query(lib, name, **change)[0] == abi.UNSUPPORTED_BACKEND


@pytest.mark.parametrize("name,change", [
    ("gemm_mx4", dict(k=2**23)), ("gemm_mx4", dict(m=2**31 - 257)), ("gemm_mx4", dict(m=0, a=0)), ("gemm_mx4", dict(k=0, a=0, b=0)),
    ("gemm_mx4", dict(n=0, b=0, out=0, ldo=0)), ("linear_mx4", dict(m=0, x=0, out=0)), ("linear_mx4", dict(m=1)),
    ("linear_mx4_backward", dict(m=0, dy=0, x=0, dx=0)), ("linear_mx4_backward", dict(dx=0, w_t=0, m=2**23)),
    ("linear_mx4_backward", dict(dw=0, x=0, dbias=0, m=2**23 + 1)), ("experts_mx4", dict(tokens=0, x=0, out=0, ids=0, weights=0)),
    ("experts_mx4", dict(ids=0, weights=0)), ("experts_mx4", dict(router=0)),
    ("experts_mx4", dict(tokens=64, experts=1024, top=16, width=65536, inner=65536, ldx=65536, ldo=65536, ldrouter=65536))])
def test_sizes_within_the_limits(lib, name, change):
    assert query(lib, name, **change)[0] == abi.SUCCESS


@pytest.mark.parametrize("m", [1, 16, 17, 64, 65, 300, 5000])
@pytest.mark.parametrize("n", [1, 700, 8200])
@pytest.mark.parametrize("k", [1, 256, 70001])
def test_workspaces_of_layers(lib, m, n, k):
    """No larger than the rounded operands and 32-bit sums of a few hundred tiles of 256 x 256."""
    limit = 32 * 256 * 256 * 256 * 4 + 65536
    status, need = query(lib, "linear_mx4", m=m, n=n, k=k, ldx=k, ldo=n)
    assert status == abi.SUCCESS and need <= 2 * (m + 16) * (k + 256) + limit
    status, need = query(lib, "linear_mx4_backward", m=m, n=n, k=k, lddy=n, ldx=k, lddx=k, lddw=k)
    assert status == abi.SUCCESS and need <= 4 * (m + 256) * (n + k + 512) + 2 * limit


@pytest.mark.parametrize("name", [*CALLS, "quantize_mx4", "dequantize_mx4", "pack_mx4"])
def test_null_arguments(lib, name):
    struct = {"quantize_mx4": abi.Mx4Args, "dequantize_mx4": abi.Mx4Args, "pack_mx4": abi.PackMx4Args}.get(name)
    args = abi.new_struct(struct or CALLS[name][0])
    assert getattr(lib, f"rns8_mi355x_{name}")(None, C.byref(args), None) == abi.INVALID_ARGUMENT
    if not struct:
        need = C.c_uint64()
        fn = getattr(lib, f"rns8_mi355x_{name}_workspace")
        assert fn(None, C.byref(need)) == abi.INVALID_ARGUMENT
        assert fn(C.byref(args), None) == abi.INVALID_ARGUMENT


class NoContext:
    def device_info(self):
        return type("Info", (), {"device_id": 0})()


def test_python_refuses_host_tensors(lib):
    torch = pytest.importorskip("torch")
    from rns8_amd import operators as ops

    x, q = torch.zeros(4, 32), torch.zeros(ops.mx4_bytes(4, 32), dtype=torch.uint8)
    w = torch.zeros(ops.mx4_bytes(8, 32), dtype=torch.uint8)
    for call in (lambda: ops.QuantizeMx4(NoContext(), x=x, q=q), lambda: ops.DequantizeMx4(NoContext(), q=q, out=x),
                 lambda: ops.GemmMx4(NoContext(), a=q, b=w, k=32, out=torch.zeros(4, 8)),
                 lambda: ops.LinearMx4(NoContext(), x=x, w=w, out=torch.zeros(4, 8)),
                 lambda: ops.PackMx4(NoContext(), data=torch.zeros(4, 16, dtype=torch.uint8),
                                     scale=torch.zeros(4, 1, dtype=torch.uint8), q=q, cols=32)):
        with pytest.raises(ValueError, match="device memory"):
            call()


class Tensor:
    """What the checks look at of a tensor in device memory."""

    is_cuda = True
    device = type("Device", (), {"index": 0})()

    def __init__(self, shape, dtype="float32", strides=None, address=P):
        self.shape, self.dtype, self.address = tuple(shape), f"torch.{dtype}", address
        dense = [1]
        for size in reversed(self.shape[1:]):
            dense.insert(0, dense[0] * size)
        self.dense, self.strides = tuple(dense), tuple(strides or dense)

    def stride(self, d):
        return self.strides[d]

    def numel(self):
        n = 1
        for size in self.shape:
            n *= size
        return n

    def is_contiguous(self):
        return self.strides == self.dense

    def data_ptr(self):
        return self.address


@pytest.mark.parametrize("call,match", [
    (lambda o, c: o.QuantizeMx4(c, x=Tensor((4, 32)), q=Tensor((2175,), "uint8")), "2176 bytes"),
    (lambda o, c: o.QuantizeMx4(c, x=Tensor((4, 32)), q=Tensor((2176,), "int8")), "uint8 is wanted"),
    (lambda o, c: o.QuantizeMx4(c, x=Tensor((4, 32), "float64"), q=Tensor((2176,), "uint8")), "float64"),
    (lambda o, c: o.QuantizeMx4(c, x=Tensor((4, 32), strides=(1, 4)), q=Tensor((2176,), "uint8")), "next to each other"),
    (lambda o, c: o.GemmMx4(c, a=Tensor((2176,), "uint8"), b=Tensor((4352,), "uint8"), k=32, out=Tensor((4, 8))), "2176 bytes"),
    (lambda o, c: o.GemmMx4(c, a=Tensor((2176,), "uint8"), b=Tensor((2176,), "uint8", strides=(2,)), k=32, out=Tensor((4, 8))),
     "next to each other"),
    (lambda o, c: o.LinearMx4(c, x=Tensor((4, 32)), w=Tensor((2176,), "uint8"), out=Tensor((5, 8))), "wanted"),
    (lambda o, c: o.LinearMx4(c, x=Tensor((4, 32)), w=Tensor((2176,), "uint8"), out=Tensor((4, 8), "float16")), "float32 is wanted"),
    (lambda o, c: o.LinearMx4(c, x=Tensor((4, 32)), w=Tensor((2176,), "uint8"), out=Tensor((4, 8)), bias=Tensor((7,))), "8 values"),
    (lambda o, c: o.LinearMx4Backward(c, dy=Tensor((4, 8)), x=Tensor((4, 32)), dw=Tensor((8, 33))), "wanted"),
    (lambda o, c: o.ExpertsMx4(c, x=Tensor((4, 32)), gate=Tensor((3, 2176), "uint8"), up=Tensor((3, 2176), "uint8"),
                               down=Tensor((3, 2176), "uint8"), inner=16, out=Tensor((4, 32)), ids=Tensor((4, 2), "int64"),
                               weights=Tensor((4, 2))), "wanted"),
    (lambda o, c: o.ExpertsMx4(c, x=Tensor((4, 32)), gate=Tensor((3, 2176), "uint8"), up=Tensor((2, 2176), "uint8"),
                               down=Tensor((3, 2176), "uint8"), inner=16, out=Tensor((4, 32)), ids=Tensor((4, 2), "int32"),
                               weights=Tensor((4, 2))), "up has shape")])
def test_python_refuses_operands_that_do_not_fit(lib, call, match):
    from rns8_amd import operators as ops

    with pytest.raises(ValueError, match=match):
        call(ops, NoContext())
