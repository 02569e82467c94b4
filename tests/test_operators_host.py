"""What calls of the language-model operators enqueue, without a device.

tests/operators_host_check.cpp runs the entry points on the library's own
objects with HIP's launch functions replaced by ones that only take notes. A
call gets a workspace of the size that its query answers, so a launch that such
a call cannot feed shows here, and so does one before a refusal.
"""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path
from typing import NamedTuple

import pytest

from rns8_amd import abi

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "rns8_amd" / "csrc"
OBJS = [ROOT / "rns8_amd" / "_build" / f"{p.stem}.o" for p in sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.cpp")])]


class Answer(NamedTuple):
    query: int
    bytes: int
    status: int
    launches: int
    blocks: int  # of the largest launch
    stream: int


@pytest.fixture(scope="module")
def enqueued(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    if not all(p.is_file() for p in OBJS):
        pytest.skip("library objects missing: run __graft_entry__.build()")
    exe = tmp_path_factory.mktemp("operators") / "operators_host_check"
    subprocess.run([gxx, "-std=c++17", "-isystem", "/opt/rocm/include", "-I", str(CSRC), "-I", str(ROOT / "include"),
                    str(ROOT / "tests" / "operators_host_check.cpp"), *map(str, OBJS), "-L/opt/rocm/lib",
                    "-Wl,-rpath,/opt/rocm/lib", "-lamdhip64", "-pthread", "-o", str(exe)], check=True)

    def run(what, *calls):
        text = "\n".join(" ".join([what, *(f"{k} {v}" for k, v in c.items())]) for c in calls) + "\n"
        res = subprocess.run([str(exe)], input=text, capture_output=True, text=True, timeout=60, check=True)
        return [Answer(*map(int, line.split())) for line in res.stdout.splitlines()]

    return run


P = 1 << 20  # an address that nothing reads


def linear(m, n, k, keep=False, **more):
    """A linear layer's arguments; operands without elements are NULL, as those of empty tensors are."""
    c = dict(dtype=abi.BF16, m=m, n=n, k=k, x=P if m else 0, ldx=k, w=P if n else 0, ldw=k, w_scale=P if n else 0,
             out=P if m and n else 0, ldo=max(n, 1))
    if keep:
        c |= dict(x_q=P, ldq=k, x_scale=P)
    return c | more


@pytest.mark.parametrize("k", [1, 15, 16, 64, 8192, 8193, 16384, 16385, 70001])
@pytest.mark.parametrize("m", [1, 2, 3, 17, 64, 65, 300])
def test_a_layer_without_channels(enqueued, m, k):
    """Nothing is left to do but the 8-bit rows, where the caller keeps them: these take no workspace."""
    without, kept = enqueued("linear_i8", linear(m, 0, k), linear(m, 0, k, keep=True))
    assert without[:4] == (abi.SUCCESS, 0, abi.SUCCESS, 0)
    assert kept[:4] == (abi.SUCCESS, 0, abi.SUCCESS, 1)


@pytest.mark.parametrize("n", [0, 1, 500])
@pytest.mark.parametrize("keep", [False, True])
def test_a_layer_without_tokens(enqueued, n, keep):
    (got,) = enqueued("linear_i8", linear(0, n, 64, keep))
    assert got[:4] == (abi.SUCCESS, 0, abi.SUCCESS, 0)


def test_streams(enqueued):
    """No stream is the context's own (4096 here), the default stream's name is the default stream."""
    calls = [linear(300, 500, 64, stream=s) for s in (0, abi.DEFAULT_STREAM, 8192)]
    assert [a.stream for a in enqueued("linear_i8", *calls)] == [4096, 0, 8192]


def test_python_handles(monkeypatch):
    """A call without a stream names none; a handle of 0 is the default stream's."""
    from rns8_amd import operators

    seen = []
    call = object.__new__(operators.QuantizeRows)
    call.ctx = type("Context", (), {"ptr": None})()
    call._ref = None
    call._fn = lambda ctx, args, stream: seen.append(stream) or abi.SUCCESS
    call(), call(None), call(0), call(8192)
    assert seen == [None, None, abi.DEFAULT_STREAM, 8192]
