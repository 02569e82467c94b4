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

    def run_all(lines):
        res = subprocess.run([str(exe)], input="\n".join([*lines, "kernels"]) + "\n", capture_output=True, text=True,
                             timeout=120, check=True)
        answers, names = res.stdout.splitlines()[:len(lines)], res.stdout.splitlines()[len(lines):]
        return [Answer(*map(int, line.split())) for line in answers], {k: int(n) for k, n in map(str.split, names[:-1])}

    def run(what, *calls):
        text = "\n".join(" ".join([what, *(f"{k} {v}" for k, v in c.items())]) for c in calls) + "\n"
        res = subprocess.run([str(exe)], input=text, capture_output=True, text=True, timeout=60, check=True)
        return [Answer(*map(int, line.split())) for line in res.stdout.splitlines()]

    run.all = run_all
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


# ---- limits ---------------------------------------------------------------------------------


def columns(rows, cols):
    return dict(dtype=abi.F16, rows=rows, cols=cols, x=P if rows else 0, ldx=cols, q=P if rows else 0, ldq=max(rows, 1),
                scale=P, sums=P)


@pytest.mark.parametrize("rows,cols", [(2**20 + 1, 32768), (2**31 - 1, 1), (2**28 + 1000, 100), (0, 2**31 - 1),
                                       (1, 2**31 - 1), (2, 2**24 + 50), (512, 2**26), (513, 2**28), (600, 2**22 + 1)])
def test_columns_of_any_size_that_is_promised(enqueued, rows, cols):
    """Strips of 32 whole columns or, past 512 rows, partials and then tiles of 128 x 128: no launch is refused, and none
    has 2^32 threads."""
    (got,) = enqueued("quantize_columns", columns(rows, cols))
    assert got[:3:2] == (abi.SUCCESS, abi.SUCCESS) and got.blocks < 2**32 // 256
    units = -(-cols // 32) if 0 < rows <= 512 else max(1, -(-rows // 128)) * -(-cols // 128)
    launches = -(-units // 2**23) + (0 if 0 < rows <= 512 else 1)
    assert got.launches == launches


LONGEST = 2**23 - 16  # a row of 8-bit operands


def product(m, n, k, layout=abi.B_CHANNELS, pad=1):
    return dict(dtype=abi.F32, m=m, n=n, k=k, a=P, lda=k + pad, b=P, ldb=(n if layout else k) + pad, b_layout=layout, out=P,
                ldo=n)


@pytest.mark.parametrize("call,refused", [
    (product(300, 500, LONGEST), False), (product(300, 500, LONGEST, pad=0), False), (product(300, 500, LONGEST + 1), True),
    (product(300, 500, 2**23 - 1, pad=0), True), (product(300, LONGEST, 500, abi.B_INNER), False),
    (product(300, LONGEST + 1, 500, abi.B_INNER), True), (product(1, 2**31 - 257, 1), False),
    (product(1, 2**31 - 256, 1), True), (product(2**31 - 1, 1, 1), False)])
def test_limits_of_products(enqueued, call, refused):
    (got,) = enqueued("gemm_i8_scaled", call)
    if refused:
        assert got[:4] == (abi.UNSUPPORTED_BACKEND, 0, abi.UNSUPPORTED_BACKEND, 0)
    else:
        assert got.query == got.status == abi.SUCCESS and got.launches >= 1


def gradients(m, n, k, pad=1, **more):
    c = dict(dtype=abi.F32, m=m, n=n, k=k, dy=P, lddy=n, x_q=P, ldq=k + pad, x_scale=P, w=P, ldw=k + pad, w_scale=P, dx=P,
             lddx=k, dw=P, lddw=k, dbias=P)
    return c | more


@pytest.mark.parametrize("call,refused", [
    (gradients(300, 500, LONGEST), False), (gradients(300, 500, LONGEST + 1), True),
    (gradients(300, 500, LONGEST + 1, dx=0), True), (gradients(300, 500, LONGEST + 1, dw=0), True),
    (gradients(300, 500, LONGEST + 1, dx=0, dw=0), False), (gradients(LONGEST - 1, 500, 20), False),
    (gradients(LONGEST, 500, 20), True), (gradients(300, LONGEST, 20), True), (gradients(300, LONGEST - 1, 20), False)])
def test_limits_of_gradients(enqueued, call, refused):
    (got,) = enqueued("linear_i8_backward", call)
    if refused:
        assert got[:4] == (abi.UNSUPPORTED_BACKEND, 0, abi.UNSUPPORTED_BACKEND, 0)
    else:
        assert got.query == got.status == abi.SUCCESS and got.launches >= 1


def test_limits_of_layers(enqueued):
    fits = [linear(1, 2**31 - 257, 1), linear(300, 500, LONGEST - 1), linear(300, 2**31 - 257, 20)]
    over = [linear(1, 2**31 - 256, 1), linear(300, 500, LONGEST), linear(300, 2**31 - 256, 20)]
    assert all(a.query == a.status == abi.SUCCESS and a.launches for a in enqueued("linear_i8", *fits))
    refused = (abi.UNSUPPORTED_BACKEND, 0, abi.UNSUPPORTED_BACKEND, 0)
    assert all(a[:4] == refused for a in enqueued("linear_i8", *over))


@pytest.mark.parametrize("m,n,k", [(70, 300, 130), (300, 257, 641), (530, 130, 1000), (300, 64, 15)])
def test_layers_copy_what_they_cannot_read_in_place(enqueued, m, n, k):
    """Kept rows, weights, both or neither: each copy is a launch, or part of the quantization's where it is the weights'."""
    at = dict(ldq=-(-k // 16) * 16, ldw=-(-k // 16) * 16)
    none, rows, weights, both = enqueued("linear_i8", *(linear(m, n, k, keep=True, **(at | c)) for c in (
        {}, {"x_q": P + 1}, {"w": P + 1}, {"x_q": P + 1, "w": P + 1})))
    assert {a.status for a in (none, rows, weights, both)} == {abi.SUCCESS}
    assert [a.launches - none.launches for a in (rows, weights, both)] == [1, 0, 2]
    assert none.bytes < weights.bytes < both.bytes and none.bytes < rows.bytes < both.bytes


# ---- kernels ---------------------------------------------------------------------------------

OPERATOR_KERNELS = ("quantize_rows_kernel", "prepare_kernel", "quantize_columns_kernel", "copy_rows_kernel",
                    "scaled_tiles_kernel", "join_slices_kernel", "scaled_rows_kernel", "block_norm_kernel",
                    "block_norm_backward_kernel", "sum_groups_kernel", "logprobs_kernel", "join_parts_kernel",
                    "logprobs_backward_kernel")


def many_calls():
    """Calls of every operator over types, sizes on both sides of each rule, and options."""
    def line(what, **fields):
        return " ".join([what, *(f"{k} {v}" for k, v in fields.items())])

    for dtype in (abi.F32, abi.F16, abi.BF16):
        for rows in (1, 40, 600):
            for cols in (5, 500, 1000, 1100, 2000, 3000, 4096, 5000, 8000, 9000, 16000, 17000, 30000, 40000):
                for multiplier in (0, P):
                    yield line("quantize_rows", dtype=dtype, rows=rows, cols=cols, x=P, ldx=cols, multiplier=multiplier,
                               q=P, ldq=cols, scale=P)
                if cols > 32768:
                    continue
                for ldgate in (0, cols):
                    norm = dict(dtype=dtype, rows=rows, cols=cols, flags=3, branch_scale=1, residual_scale=1, x=P,
                                ldx=cols, gate=P, ldgate=ldgate)
                    yield line("block_norm", **norm, h=P, ldh=cols, y=P, ldy=cols)
                    yield line("block_norm_backward", **norm, rstd=P, dy=P, lddy=cols, dx=P, lddx=cols, dpre_weight=P)
        for rows in (1, 5, 600):
            for vocab in (100, 2500, 7000, 30000, 50000, 130000):
                for top in (0, 5):
                    yield line("token_logprobs", dtype=dtype, rows=rows, vocab=vocab, logits=P, ldl=vocab, scale=1,
                               lse=P, top=top, top_ids=P if top else 0)
                yield line("token_logprobs_backward", dtype=dtype, rows=rows, vocab=vocab, logits=P, ldl=vocab, targets=P,
                           scale=1, lse=P, dlogp=P, dlogits=P, lddl=vocab)
        for m in (1, 2, 16, 17, 40, 60, 100, 300, 1000, 4096):
            for n in (40, 300, 1100, 4096, 8200):
                for k in (10, 64, 900, 1500, 3000, 8000, 12000):
                    yield line("linear_i8", **(linear(m, n, k) | dict(dtype=dtype)))
                    yield line("linear_i8", **(linear(m, n, k, keep=True, ldw=k + 1) | dict(dtype=dtype)))
        for m in (40, 600, 1500):
            for n in (40, 700, 1100, 3000, 5000, 9000):
                for k in (64, 1000, 4096):
                    for some in ({}, {"dw": 0, "dbias": 0}, {"dx": 0}):
                        yield line("linear_i8_backward", **(gradients(m, n, k) | dict(dtype=dtype) | some))
    for layout in (abi.B_CHANNELS, abi.B_INNER):
        for m in (64, 256, 500, 1000, 2048, 4096, 8192):
            for n in (64, 128, 300, 1000, 2048, 4096, 8192):
                for k in (64, 1000, 4096, 30000, 200000):
                    yield line("gemm_i8_scaled", **product(m, n, k, layout))
        for m, n, k in ((277, 40555, 721), (1362, 5607, 2070)):
            yield line("gemm_i8_scaled", **product(m, n, k, layout))
    for rows in (0, 100, 600, 20000):
        for dtype in (abi.F32, abi.F16, abi.BF16):
            yield line("quantize_columns", **(columns(rows, 300) | dict(dtype=dtype)))


def test_every_kernel_is_reached(enqueued):
    """No instantiation of an operator's kernel is left that no call takes."""
    answers, kernels = enqueued.all(list(many_calls()))
    assert all(a.query == a.status == abi.SUCCESS and a.launches for a in answers)
    mine = {k: n for k, n in kernels.items() if any(f"{len(name)}{name}" in k for name in OPERATOR_KERNELS)}
    assert all(any(f"{len(name)}{name}" in k for k in mine) for name in OPERATOR_KERNELS)
    unreached = [k for k, n in mine.items() if n == 0]
    assert not unreached, "\n".join(unreached)
