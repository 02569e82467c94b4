"""What calls of the operators on 4-bit microscaled matrices enqueue, without a device (tests/mx4_host_check.cpp).

Every kernel is one that some call launches, a refused call launches nothing, and a call needs the workspace that its
query answers to the last byte."""
from __future__ import annotations

import itertools
import shutil
import subprocess

import pytest

from rns8_amd import abi
from test_mx4_abi import BACK, EXPERTS, GEMM, LINEAR, P
from test_operators_host import CSRC, OBJS, ROOT, Answer

QUANTIZE = dict(dtype=abi.BF16, rows=300, cols=500, x=P, ldx=500, q=P, q_t=P)
BACKWARDS = dict(dtype=abi.BF16, rows=300, cols=500, x=P, ldx=500, q=P)
PACK = dict(rows=300, cols=500, data=P, ldd=250, scale=P, lds=16, q=P)


@pytest.fixture(scope="module")
def enqueued(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    if not all(p.is_file() for p in OBJS):
        pytest.skip("library objects missing: run __graft_entry__.build()")
    exe = tmp_path_factory.mktemp("mx4") / "mx4_host_check"
    subprocess.run([gxx, "-std=c++17", "-isystem", "/opt/rocm/include", "-I", str(CSRC), "-I", str(ROOT / "include"),
                    str(ROOT / "tests" / "mx4_host_check.cpp"), *map(str, OBJS), "-L/opt/rocm/lib",
                    "-Wl,-rpath,/opt/rocm/lib", "-lamdhip64", "-pthread", "-o", str(exe)], check=True)

    def run(*calls):
        """Answers to (name, arguments), and how often each kernel was launched."""
        lines = [" ".join([name, *(f"{k} {v}" for k, v in fields.items())]) for name, fields in calls]
        res = subprocess.run([str(exe)], input="\n".join([*lines, "kernels"]) + "\n", capture_output=True, text=True,
                             timeout=120, check=True).stdout.splitlines()
        return ([Answer(*map(int, line.split())) for line in res[:len(calls)]],
                {k: int(n) for k, n in map(str.split, res[len(calls):-1])})

    return run


def linear(m, n, k, dtype):
    return LINEAR | dict(dtype=dtype, m=m, n=n, k=k, ldx=k, ldo=n)


def backward(m, n, k, dtype, **more):
    return BACK | dict(dtype=dtype, m=m, n=n, k=k, lddy=n, ldx=k, lddx=k, lddw=k) | more


def experts(tokens, count, top, width, inner, dtype, **more):
    return EXPERTS | dict(dtype=dtype, tokens=tokens, experts=count, top=top, width=width, inner=inner, ldx=width, ldo=width,
                          ldrouter=width) | more


TYPES = (abi.F32, abi.F16, abi.BF16)
LAYERS = [(1, 1, 1, 1, 1), (1, 128, 8, 4096, 1536), (2, 1024, 16, 2048, 256), (16, 4, 2, 2048, 768), (16, 16, 16, 100, 300),
          (17, 4, 2, 100, 300), (64, 128, 8, 4096, 1536), (64, 1024, 16, 65536, 65536)]


def many_calls():
    """Calls of every operator over types and sizes on both sides of each rule (rows shorter than 16 bytes: 3 values, 5)."""
    for dtype in TYPES:
        for rows, cols in itertools.product((1, 100, 2000, 9000), (1, 5, 300, 5000)):
            for given in (dict(q=P), dict(q_t=P), dict(q=P, q_t=P)):
                yield "quantize_mx4", dict(dtype=dtype, rows=rows, cols=cols, x=P, ldx=cols) | given
            yield "dequantize_mx4", dict(dtype=dtype, rows=rows, cols=cols, x=P, ldx=cols, q=P)
        for m, n, k in itertools.product((1, 2, 16, 17, 40, 64, 65, 300, 4096), (3, 5, 300, 4096, 8200), (64, 900, 8192)):
            yield "gemm_mx4", GEMM | dict(dtype=dtype, m=m, n=n, k=k, ldo=n)
            yield "linear_mx4", linear(m, n, k, dtype)
            for some in ({}, dict(dw=0, dbias=0), dict(dx=0), dict(dx=0, dw=0)):
                yield "linear_mx4_backward", backward(m, n, k, dtype, **some)
        for layer in LAYERS:
            yield "experts_mx4", experts(*layer, dtype)
            yield "experts_mx4", experts(*layer, dtype, router=0)
    yield "gemm_mx4", GEMM | dict(k=0)
    yield "pack_mx4", PACK


KERNELS = ("quantize_mx4_kernel", "quantize_narrow_kernel", "sum_narrow_kernel", "sum_partials_kernel", "dequantize_mx4_kernel",
           "pack_mx4_kernel", "mx4_rows_kernel", "mx4_linear_rows_kernel", "mx4_tiles_kernel", "mx4_join_kernel",
           "experts_stage_kernel", "experts_choose_kernel", "experts_hidden_few_kernel", "experts_many_kernel",
           "experts_down_few_kernel", "experts_combine_kernel")


def test_every_kernel_is_reached(enqueued):
    """No instantiation is left that no call takes; no launch has 2^32 threads."""
    answers, kernels = enqueued(*many_calls())
    assert all(a.query == a.status == abi.SUCCESS and a.launches and a.blocks < 2**32 // 1024 for a in answers)
    mine = {k: n for k, n in kernels.items() if any(f"{len(name)}{name}" in k for name in KERNELS)}
    assert all(any(f"{len(name)}{name}" in k for k in mine) for name in KERNELS)
    unreached = [k for k, n in mine.items() if n == 0]
    assert not unreached, "\n".join(unreached)


SIZED = [("gemm_mx4", GEMM | dict(m=100, n=200, k=30000, ldo=200)), ("linear_mx4", linear(17, 40, 300, abi.F32)),
         ("linear_mx4", linear(300, 500, 70000, abi.BF16)), ("linear_mx4_backward", backward(300, 500, 256, abi.F16)),
         ("linear_mx4_backward", backward(1, 40, 50, abi.F16, dx=0, dw=0)), ("linear_mx4_backward", backward(3000, 100, 90, abi.F32)),
         ("experts_mx4", experts(1, 8, 2, 64, 100, abi.BF16)), ("experts_mx4", experts(64, 8, 2, 640, 1000, abi.F32)),
         ("experts_mx4", experts(64, 8, 2, 640, 1000, abi.F16, router=0))]


@pytest.mark.parametrize("name,fields", SIZED)
def test_workspaces_to_the_last_byte(enqueued, name, fields):
    (enough, short), _ = enqueued((name, fields), (name, fields | dict(less=1)))
    assert enough.query == enough.status == abi.SUCCESS and enough.bytes and enough.launches
    assert short[:4] == (abi.SUCCESS, enough.bytes, abi.WORKSPACE_TOO_SMALL, 0)


@pytest.mark.parametrize("name,fields", [
    ("quantize_mx4", dict(rows=-1)), ("quantize_mx4", dict(cols=0)), ("quantize_mx4", dict(q=0, q_t=0)),
    ("quantize_mx4", dict(x=0)), ("quantize_mx4", dict(ldx=499)), ("quantize_mx4", dict(q=P + 8)),
    ("quantize_mx4", dict(q_t=P + 1)), ("quantize_mx4", dict(dtype=3)), ("quantize_mx4", dict(x=P + 1)),
    ("dequantize_mx4", dict(q=0)), ("dequantize_mx4", dict(q_t=P)), ("dequantize_mx4", dict(x=0)),
    ("pack_mx4", dict(dtype=1)), ("pack_mx4", dict(data=0)), ("pack_mx4", dict(ldd=249)), ("pack_mx4", dict(lds=15)),
    ("pack_mx4", dict(scale=0)), ("pack_mx4", dict(q=P + 4)), ("gemm_mx4", dict(a=0)), ("gemm_mx4", dict(ldo=499)),
    ("linear_mx4", dict(x=0)), ("linear_mx4", dict(w=P + 2)), ("linear_mx4_backward", dict(dx=0, dw=0, dbias=0)),
    ("linear_mx4_backward", dict(w_t=0)), ("experts_mx4", dict(top=9)), ("experts_mx4", dict(flags=2)),
    ("experts_mx4", dict(router=0, ids=0)), ("experts_mx4", dict(down=0)), ("experts_mx4", dict(ldo=511))])
def test_refused_calls_launch_nothing(enqueued, name, fields):
    whole = {"quantize_mx4": QUANTIZE, "dequantize_mx4": BACKWARDS, "pack_mx4": PACK, "gemm_mx4": GEMM, "linear_mx4": LINEAR,
             "linear_mx4_backward": BACK, "experts_mx4": EXPERTS}[name]
    (fine, refused), _ = enqueued((name, whole), (name, whole | fields))
    assert fine.status == abi.SUCCESS and fine.launches
    assert refused.status == abi.INVALID_ARGUMENT and refused.launches == 0


@pytest.mark.parametrize("name,fields", [
    ("quantize_mx4", dict(rows=2**31 - 256)), ("dequantize_mx4", dict(cols=2**31, ldx=2**31)),
    ("pack_mx4", dict(rows=2**31)), ("gemm_mx4", dict(k=2**23 + 1)), ("linear_mx4", dict(m=2**31)),
    ("linear_mx4_backward", dict(m=2**23 + 1)), ("experts_mx4", dict(tokens=65)), ("experts_mx4", dict(inner=65537))])
def test_sizes_past_the_limits_launch_nothing(enqueued, name, fields):
    whole = {"quantize_mx4": QUANTIZE, "dequantize_mx4": BACKWARDS, "pack_mx4": PACK, "gemm_mx4": GEMM, "linear_mx4": LINEAR,
             "linear_mx4_backward": BACK, "experts_mx4": EXPERTS}[name]
    (refused,), _ = enqueued((name, whole | fields))
    assert refused.status == abi.UNSUPPORTED_BACKEND and refused.launches == 0


@pytest.mark.parametrize("name,fields", [
    ("quantize_mx4", dict(rows=0, x=0, q=0, q_t=0)), ("dequantize_mx4", dict(rows=0, x=0, q=0)),
    ("pack_mx4", dict(rows=0, data=0, scale=0, q=0)), ("gemm_mx4", dict(m=0, a=0, out=0)), ("linear_mx4", dict(m=0, x=0, out=0)),
    ("experts_mx4", dict(tokens=0, x=0, out=0, ids=0, weights=0))])
def test_calls_without_rows(enqueued, name, fields):
    whole = {"quantize_mx4": QUANTIZE, "dequantize_mx4": BACKWARDS, "pack_mx4": PACK, "gemm_mx4": GEMM, "linear_mx4": LINEAR,
             "experts_mx4": EXPERTS}[name]
    (got,), _ = enqueued((name, whole | fields))
    assert got[:4] == (abi.SUCCESS, 0, abi.SUCCESS, 0)
