"""The language-model operators without a device: argument structs against the header, refusals and workspace queries."""
from __future__ import annotations

import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

from rns8_amd import abi

ROOT = Path(__file__).resolve().parent.parent
STRUCTS = {"quantize": abi.QuantizeArgs, "gemm_i8": abi.GemmI8Args, "linear_i8": abi.LinearI8Args,
           "linear_i8_backward": abi.LinearI8BackwardArgs, "block_norm": abi.BlockNormArgs,
           "block_norm_backward": abi.BlockNormBackwardArgs, "logprobs": abi.LogprobsArgs,
           "logprobs_backward": abi.LogprobsBackwardArgs}


def test_structs_mirror_the_header(tmp_path):
    compiler = shutil.which("g++")
    if not compiler:
        pytest.skip("no host compiler")
    lines = []
    for name, mirror in STRUCTS.items():
        c = f"rns8_mi355x_{name}_args"
        lines.append(f'std::printf("{name} %zu\\n", sizeof({c}));')
        lines += [f'std::printf("{name}.{f[0]} %zu %zu\\n", offsetof({c}, {f[0]}), sizeof({c}::{f[0]}));'
                  for f in mirror._fields_]
    source = tmp_path / "layout.cpp"
    source.write_text("#include <cstddef>\n#include <cstdio>\n#include \"rns8_mi355x.h\"\nint main() {\n" +
                      "\n".join(lines) + "\n}\n")
    subprocess.run([compiler, "-std=c++17", f"-I{ROOT / 'include'}", str(source), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split("\n")
    want = []
    for name, mirror in STRUCTS.items():
        want.append(f"{name} {C.sizeof(mirror)}")
        for f in mirror._fields_:
            d = getattr(mirror, f[0])
            want.append(f"{name}.{f[0]} {d.offset} {d.size}")
    assert [line for line in got if line] == want


@pytest.fixture(scope="module")
def lib():
    if not (ROOT / "rns8_amd" / "librns8.so").exists():
        pytest.skip("librns8.so not built (run __graft_entry__.build())")
    import rns8_amd

    return rns8_amd.lib()


P = 1 << 20  # an address that nothing here reads


def query(lib, name, struct, **fields):
    args = abi.new_struct(struct)
    for k, v in fields.items():
        setattr(args, k, v)
    need = C.c_uint64(77)
    return getattr(lib, f"rns8_mi355x_{name}_workspace")(C.byref(args), C.byref(need)), need.value


LINEAR = dict(dtype=abi.BF16, m=300, n=500, k=256, x=P, ldx=256, w=P, ldw=256, w_scale=P, out=P, ldo=500)
GEMM = dict(dtype=abi.F32, m=300, n=500, k=256, a=P, lda=256, b=P, ldb=256, out=P, ldo=500)
BACK = dict(dtype=abi.F16, m=300, n=500, k=256, dy=P, lddy=500, x_q=P, ldq=256, x_scale=P, w=P, ldw=256, w_scale=P,
            dx=P, lddx=256, dw=P, lddw=256, dbias=P)
NORM = dict(dtype=abi.BF16, rows=50, cols=700, flags=3, eps=1e-6, branch_scale=1.0, residual_scale=1.0, x=P, ldx=700,
            residual=P, ldresidual=700, rstd=P, dy=P, lddy=700, dx=P, lddx=700, dpost_weight=P, dpre_weight=P)
LOGPROBS = dict(dtype=abi.BF16, rows=4, vocab=131072, logits=P, ldl=131072, targets=P, scale=1.0, logp=P, top=5,
                top_ids=P)
COLUMNS = dict(dtype=abi.F32, rows=1000, cols=300, x=P, ldx=300, q=P, ldq=1008, scale=P)
CALLS = {"linear_i8": (abi.LinearI8Args, LINEAR), "gemm_i8_scaled": (abi.GemmI8Args, GEMM),
         "linear_i8_backward": (abi.LinearI8BackwardArgs, BACK),
         "block_norm_backward": (abi.BlockNormBackwardArgs, NORM), "token_logprobs": (abi.LogprobsArgs, LOGPROBS),
         "quantize_columns": (abi.QuantizeArgs, COLUMNS)}


@pytest.mark.parametrize("name", CALLS)
def test_queries_answer(lib, name):
    struct, fields = CALLS[name]
    status, need = query(lib, name, struct, **fields)
    assert status == abi.SUCCESS and need < 2**32
    assert query(lib, name, struct, **fields) == (status, need)


@pytest.mark.parametrize("name,change", [
    ("linear_i8", dict(dtype=3)), ("linear_i8", dict(abi_version=0)), ("linear_i8", dict(struct_size=8)),
    ("linear_i8", dict(m=-1)), ("linear_i8", dict(k=0)), ("linear_i8", dict(x=0)), ("linear_i8", dict(ldx=255)),
    ("linear_i8", dict(ldw=255)), ("linear_i8", dict(ldo=499)), ("linear_i8", dict(x=P + 1)),
    ("linear_i8", dict(w_scale=P + 2)), ("linear_i8", dict(w_scale=0)), ("linear_i8", dict(x_q=P, ldq=256)),
    ("linear_i8", dict(x_scale=P)), ("gemm_i8_scaled", dict(b_layout=2)), ("gemm_i8_scaled", dict(reserved=1)),
    ("gemm_i8_scaled", dict(b_layout=1)), ("gemm_i8_scaled", dict(k=-1)), ("gemm_i8_scaled", dict(bias=P + 3)),
    ("linear_i8_backward", dict(n=0)), ("linear_i8_backward", dict(dx=0, dw=0, dbias=0)),
    ("linear_i8_backward", dict(x_q=0)), ("linear_i8_backward", dict(w=0)), ("linear_i8_backward", dict(dw=P + 2)),
    ("block_norm_backward", dict(flags=4)), ("block_norm_backward", dict(eps=-1.0)),
    ("block_norm_backward", dict(eps=float("nan"))), ("block_norm_backward", dict(branch_scale=float("inf"))),
    ("block_norm_backward", dict(rstd=0)), ("block_norm_backward", dict(dgate=P)),
    ("block_norm_backward", dict(flags=1)), ("block_norm_backward", dict(cols=0)),
    ("token_logprobs", dict(top=65)), ("token_logprobs", dict(vocab=3, ldl=3)), ("token_logprobs", dict(targets=0)),
    ("token_logprobs", dict(scale=0.0)), ("token_logprobs", dict(scale=float("nan"))),
    ("token_logprobs", dict(top=0)), ("token_logprobs", dict(logp=0, top=0, top_ids=0)),
    ("token_logprobs", dict(targets=P + 4)), ("quantize_columns", dict(cols=0)), ("quantize_columns", dict(ldq=999)),
    ("quantize_columns", dict(rows=-1))])
def test_invalid_arguments(lib, name, change):
    struct, fields = CALLS[name]
    status, need = query(lib, name, struct, **(fields | change))
    assert status == abi.INVALID_ARGUMENT and need in (0, 77)


@pytest.mark.parametrize("name,change", [
    ("linear_i8", dict(k=2**23, ldx=2**23, ldw=2**23)), ("gemm_i8_scaled", dict(lda=2**23)),
    ("gemm_i8_scaled", dict(ldb=2**23)), ("linear_i8_backward", dict(ldw=2**23)),
    ("linear_i8", dict(m=2**31)), ("block_norm_backward", dict(cols=32769, ldx=32769, ldresidual=32769, lddy=32769,
                                                               lddx=32769)),
    ("token_logprobs", dict(vocab=2**31, ldl=2**31)), ("quantize_columns", dict(rows=2**31, ldq=2**31))])
def test_sizes_past_the_limits(lib, name, change):
    struct, fields = CALLS[name]
    assert query(lib, name, struct, **(fields | change))[0] == abi.UNSUPPORTED_BACKEND


def test_offsets_past_64_bits(lib):
    status, _ = query(lib, "token_logprobs", abi.LogprobsArgs, **(LOGPROBS | dict(ldl=2**62)))
    assert status == abi.INVALID_ARGUMENT


@pytest.mark.parametrize("name", CALLS)
def test_null_arguments(lib, name):
    need = C.c_uint64()
    fn = getattr(lib, f"rns8_mi355x_{name}_workspace")
    args = abi.new_struct(CALLS[name][0])
    assert fn(None, C.byref(need)) == abi.INVALID_ARGUMENT
    assert fn(C.byref(args), None) == abi.INVALID_ARGUMENT
    assert getattr(lib, f"rns8_mi355x_{name}")(None, C.byref(args), None) == abi.INVALID_ARGUMENT


@pytest.mark.parametrize("m", [1, 2, 17, 64, 65, 300, 1797])
@pytest.mark.parametrize("n", [1, 40, 8200])
@pytest.mark.parametrize("k", [1, 100, 4096, 70001])
def test_workspaces_of_linear_layers(lib, m, n, k):
    """Any sizes and alignments have a workspace no larger than a few copies of the operands and 32-bit partial sums."""
    for at in (P, P + 3):
        status, need = query(lib, "linear_i8", abi.LinearI8Args, dtype=abi.F32, m=m, n=n, k=k, x=P, ldx=k, w=at, ldw=k,
                             w_scale=P, out=P, ldo=n)
        assert status == abi.SUCCESS
        assert need <= 3 * (m + 64) * (k + 64) + 2 * (n + 64) * (k + 64) + 4 * 1024 * 256 * 256 + 65536


def test_python_refuses_host_tensors(lib):
    torch = pytest.importorskip("torch")
    from rns8_amd import operators as ops

    class NoContext:
        def device_info(self):
            return type("Info", (), {"device_id": 0})()

    x = torch.zeros(4, 32)
    with pytest.raises(ValueError, match="device memory"):
        ops.LinearI8(NoContext(), x=x, w=torch.zeros(8, 32, dtype=torch.int8), w_scale=torch.ones(8), out=torch.zeros(4, 8))
    with pytest.raises(ValueError, match="float64"):
        ops.TokenLogprobs(NoContext(), logits=x.double(), lse=torch.zeros(4))
    assert ops.padded(1) == 16 and ops.padded(16) == 16 and ops.padded(17) == 32
