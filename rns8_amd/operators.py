"""Operators of language models around the 8-bit product, on device tensors.

Each class here is one call of the C entry point of the same name
(include/rns8_mi355x.h, which states what it computes): it takes its operands
and outputs once, checks that their shapes, types and strides fit together,
and keeps them with the call's workspace, as a C program keeps its argument
struct. Calling the object enqueues the operator on the context's stream, or on
the stream given:

    layer = operators.LinearI8(ctx, x=x, w=w, w_scale=s, out=y)
    layer()            # on the context's stream
    layer(stream)      # on a stream handle (an integer)

Operands are tensors in device memory: any objects with torch's data_ptr(),
shape, stride(), dtype and is_cuda. Rows may be strided; the elements of a row
are next to each other. Quantized rows that a call writes are followed by zeros up
to padded(cols) or the next row, whichever is first, also where q is a view that
ends before them (q[:, :cols] of a padded buffer). A torch.cuda.Stream is passed as its cuda_stream (in a
process that imports torch before this library is loaded: both then share one
HIP runtime). Torch's default stream has the handle 0: it runs the operator on
that stream, in order with torch's work there. The context's own stream waits for
no other, so a program that leaves the stream out synchronizes between the two. A
workspace is allocated when the object is made, unless one is given, and the
object must outlive its calls on the GPU.
"""
from __future__ import annotations

import ctypes as C

from . import abi, check, hip, lib
from .abi import B_CHANNELS, B_INNER, NORM_POST, NORM_PRE  # noqa: F401  (re-exported constants)

_DTYPES = {"float32": abi.F32, "float16": abi.F16, "bfloat16": abi.BF16}


def padded(cols: int) -> int:
    """The row length, in bytes, of quantized rows that products read in place."""
    return (cols + 15) // 16 * 16


def _name(t) -> str:
    return str(t.dtype).rsplit(".", 1)[-1]


class _Operands:
    """Checks operands against one another and fills the argument struct from them."""

    def __init__(self, ctx, args, first):
        self.args, self.keep = args, []
        self.device = ctx.device_info().device_id
        kind = _name(first)
        if kind not in _DTYPES:
            raise ValueError(f"operands of type {kind}: float32, float16 or bfloat16 are wanted")
        self.kind = kind
        args.dtype = _DTYPES[kind]

    def _on_device(self, what, t):
        if not getattr(t, "is_cuda", False):
            raise ValueError(f"{what} is not in device memory")
        if t.device.index not in (None, self.device):
            raise ValueError(f"{what} is on device {t.device.index}, the context on {self.device}")

    def _pointer(self, what, t, kind):
        self._on_device(what, t)
        if _name(t) != kind:
            raise ValueError(f"{what} is of type {_name(t)}: {kind} is wanted")
        self.keep.append(t)
        return t.data_ptr() or None

    def matrix(self, field, ld, t, rows, cols, kind=None, wider=False, padding=False):
        """A rows x cols operand into args.<field> and its row stride into args.<ld>.

        padding: bytes that are written with zeros after each row, up to its stride (padded(cols) at most)."""
        if t is None:
            setattr(self.args, ld, cols)
            return
        shape = tuple(t.shape)
        if len(shape) != 2 or shape[0] != rows or not (shape[1] == cols or (wider and shape[1] > cols)):
            raise ValueError(f"{field} has shape {shape}: ({rows}, {cols}) is wanted")
        if shape[1] > 1 and t.stride(1) != 1:
            raise ValueError(f"{field}: the elements of a row have to be next to each other")
        stride = t.stride(0) if rows > 1 else max(t.stride(0), shape[1])
        if stride < shape[1]:
            raise ValueError(f"{field}: rows overlap")
        if padding and rows and not self._has_room(t, (rows - 1) * stride + min(stride, padded(cols))):
            if rows > 1:
                raise ValueError(f"{field}: its storage ends before the zeros after the last row")
            stride = shape[1]
        setattr(self.args, field, self._pointer(field, t, kind or self.kind))
        setattr(self.args, ld, stride)

    @staticmethod
    def _has_room(t, length):
        """Whether `length` bytes from t's first on are in its storage (of tensors that have one)."""
        if not hasattr(t, "untyped_storage"):
            return True
        return t.storage_offset() + length <= t.untyped_storage().nbytes()

    def vector(self, field, t, count, kind="float32"):
        if t is None:
            return
        if t.numel() != count or not t.is_contiguous():
            raise ValueError(f"{field} has shape {tuple(t.shape)}: {count} values next to each other are wanted")
        setattr(self.args, field, self._pointer(field, t, kind))


class _Call:
    """An operator's call with its arguments in place."""

    _entry = ""
    _args = None
    _query = None

    def _begin(self, ctx, first):
        self.ctx = ctx
        self.args = abi.new_struct(self._args)
        self._own = 0
        return _Operands(ctx, self.args, first)

    def _finish(self, operands, workspace=None):
        self._keep = operands.keep
        self._fn = getattr(lib(), self._entry)
        self._ref = C.byref(self.args)
        if self._query:
            need = C.c_uint64()
            check(getattr(lib(), self._query)(self._ref, C.byref(need)), self._query)
            self.workspace_bytes = need.value
            if workspace is not None:
                operands._on_device("the workspace", workspace)
                if not workspace.is_contiguous():
                    raise ValueError("the workspace has to be contiguous")
                self._keep.append(workspace)
                self.args.workspace = workspace.data_ptr()
                self.args.workspace_bytes = workspace.numel() * workspace.element_size()
            elif need.value:
                hip.set_device(operands.device)
                self._own = hip.malloc(need.value)
                self.args.workspace, self.args.workspace_bytes = self._own, need.value

    def __call__(self, stream: int | None = None) -> None:
        # (the C interface reads a handle of 0 as none)
        status = self._fn(self.ctx.ptr, self._ref, abi.DEFAULT_STREAM if stream == 0 else stream)
        if status:
            check(status, self._entry)

    def __del__(self):
        own, self._own = getattr(self, "_own", 0), 0
        if own:
            try:
                hip.free(own)
            except Exception:
                pass


class QuantizeRows(_Call):
    """Rows of x in 8 bits with a scale each (rns8_mi355x_quantize_rows)."""

    _entry, _args = "rns8_mi355x_quantize_rows", abi.QuantizeArgs

    def __init__(self, ctx, *, x, q, scale, multiplier=None):
        o = self._begin(ctx, x)
        rows, cols = x.shape
        self.args.rows, self.args.cols = rows, cols
        o.matrix("x", "ldx", x, rows, cols)
        o.matrix("q", "ldq", q, rows, cols, "int8", wider=True, padding=True)
        o.vector("scale", scale, rows)
        o.vector("multiplier", multiplier, cols)
        self._finish(o)


class QuantizeColumns(_Call):
    """Columns of x in 8 bits with a scale each, transposed (rns8_mi355x_quantize_columns)."""

    _entry, _args = "rns8_mi355x_quantize_columns", abi.QuantizeArgs
    _query = "rns8_mi355x_quantize_columns_workspace"

    def __init__(self, ctx, *, x, q, scale, multiplier=None, sums=None, workspace=None):
        o = self._begin(ctx, x)
        rows, cols = x.shape
        self.args.rows, self.args.cols = rows, cols
        o.matrix("x", "ldx", x, rows, cols)
        o.matrix("q", "ldq", q, cols, rows, "int8", wider=True, padding=True)
        o.vector("scale", scale, cols)
        o.vector("multiplier", multiplier, rows)
        o.vector("sums", sums, cols)
        self._finish(o, workspace)


class GemmI8Scaled(_Call):
    """The product of 8-bit matrices with scales (rns8_mi355x_gemm_i8_scaled).

    b is n x k, or k x n with layout=B_INNER."""

    _entry, _args = "rns8_mi355x_gemm_i8_scaled", abi.GemmI8Args
    _query = "rns8_mi355x_gemm_i8_scaled_workspace"

    def __init__(self, ctx, *, a, b, out, a_scale=None, b_scale=None, bias=None, layout=B_CHANNELS, workspace=None):
        o = self._begin(ctx, out)
        (m, k), n = a.shape, b.shape[1 if layout == B_INNER else 0]
        self.args.m, self.args.n, self.args.k, self.args.b_layout = m, n, k, layout
        o.matrix("a", "lda", a, m, k, "int8")
        o.matrix("b", "ldb", b, *((k, n) if layout == B_INNER else (n, k)), "int8")
        o.matrix("out", "ldo", out, m, n)
        o.vector("a_scale", a_scale, m)
        o.vector("b_scale", b_scale, n)
        o.vector("bias", bias, n)
        self._finish(o, workspace)


class LinearI8(_Call):
    """A linear layer: x's rows in 8 bits times 8-bit weights (rns8_mi355x_linear_i8)."""

    _entry, _args = "rns8_mi355x_linear_i8", abi.LinearI8Args
    _query = "rns8_mi355x_linear_i8_workspace"

    def __init__(self, ctx, *, x, w, w_scale, out, bias=None, x_q=None, x_scale=None, workspace=None):
        o = self._begin(ctx, x)
        (m, k), n = x.shape, w.shape[0]
        self.args.m, self.args.n, self.args.k = m, n, k
        o.matrix("x", "ldx", x, m, k)
        o.matrix("w", "ldw", w, n, k, "int8")
        o.vector("w_scale", w_scale, n)
        o.vector("bias", bias, n)
        o.matrix("out", "ldo", out, m, n)
        o.matrix("x_q", "ldq", x_q, m, k, "int8", wider=True, padding=True)
        o.vector("x_scale", x_scale, m)
        self._finish(o, workspace)


class LinearI8Backward(_Call):
    """The linear layer's gradients (rns8_mi355x_linear_i8_backward)."""

    _entry, _args = "rns8_mi355x_linear_i8_backward", abi.LinearI8BackwardArgs
    _query = "rns8_mi355x_linear_i8_backward_workspace"

    def __init__(self, ctx, *, dy, x_q=None, x_scale=None, w=None, w_scale=None, dx=None, dw=None, dbias=None,
                 workspace=None):
        o = self._begin(ctx, dy)
        m, n = dy.shape
        shaped = next((t for t in (dx, dw, w, x_q) if t is not None), None)
        k = shaped.shape[1] if shaped is not None else 1
        self.args.m, self.args.n, self.args.k = m, n, k
        o.matrix("dy", "lddy", dy, m, n)
        o.matrix("x_q", "ldq", x_q, m, k, "int8", wider=True)
        o.vector("x_scale", x_scale, m)
        o.matrix("w", "ldw", w, n, k, "int8")
        o.vector("w_scale", w_scale, n)
        o.matrix("dx", "lddx", dx, m, k)
        o.matrix("dw", "lddw", dw, n, k, "float32")
        o.vector("dbias", dbias, n)
        self._finish(o, workspace)


def _norm_inputs(o, args, x, residual, gate, post_weight, pre_weight, flags, eps, branch_scale, residual_scale):
    rows, cols = x.shape
    args.rows, args.cols, args.flags, args.eps = rows, cols, flags, eps
    args.branch_scale, args.residual_scale = branch_scale, residual_scale
    o.matrix("x", "ldx", x, rows, cols)
    o.matrix("residual", "ldresidual", residual, rows, cols)
    if gate is not None and len(gate.shape) == 1:
        o.vector("gate", gate, cols, o.kind)
        args.ldgate = 0
    else:
        o.matrix("gate", "ldgate", gate, rows, cols)
    o.vector("post_weight", post_weight, cols, o.kind)
    o.vector("pre_weight", pre_weight, cols, o.kind)
    return rows, cols


class BlockNorm(_Call):
    """The norms after and before a residual block (rns8_mi355x_block_norm).

    gate is one row (cols) or one for each token (rows x cols). flags: which of
    the two norms run (both by default)."""

    _entry, _args = "rns8_mi355x_block_norm", abi.BlockNormArgs

    def __init__(self, ctx, *, x, residual=None, gate=None, post_weight=None, pre_weight=None, h=None, y=None, q=None,
                 q_scale=None, rstd=None, flags=NORM_POST | NORM_PRE, eps=1e-6, branch_scale=1.0, residual_scale=1.0):
        o = self._begin(ctx, x)
        rows, cols = _norm_inputs(o, self.args, x, residual, gate, post_weight, pre_weight, flags, eps, branch_scale,
                                  residual_scale)
        o.matrix("h", "ldh", h, rows, cols)
        o.matrix("y", "ldy", y, rows, cols)
        o.matrix("q", "ldq", q, rows, cols, "int8", wider=True, padding=True)
        o.vector("q_scale", q_scale, rows)
        o.vector("rstd", rstd, 2 * rows)
        self._finish(o)


class BlockNormBackward(_Call):
    """The gradients of the norms around a block (rns8_mi355x_block_norm_backward)."""

    _entry, _args = "rns8_mi355x_block_norm_backward", abi.BlockNormBackwardArgs
    _query = "rns8_mi355x_block_norm_backward_workspace"

    def __init__(self, ctx, *, x, rstd, residual=None, gate=None, post_weight=None, pre_weight=None, dy=None, dh=None,
                 dx=None, dresidual=None, dgate=None, dpost_weight=None, dpre_weight=None, flags=NORM_POST | NORM_PRE,
                 eps=1e-6, branch_scale=1.0, residual_scale=1.0, workspace=None):
        o = self._begin(ctx, x)
        rows, cols = _norm_inputs(o, self.args, x, residual, gate, post_weight, pre_weight, flags, eps, branch_scale,
                                  residual_scale)
        o.vector("rstd", rstd, 2 * rows)
        o.matrix("dy", "lddy", dy, rows, cols)
        o.matrix("dh", "lddh", dh, rows, cols)
        o.matrix("dx", "lddx", dx, rows, cols)
        o.matrix("dresidual", "lddresidual", dresidual, rows, cols)
        if gate is not None and len(gate.shape) == 1:
            o.vector("dgate", dgate, cols)
        else:
            o.matrix("dgate", "lddgate", dgate, rows, cols)
        o.vector("dpost_weight", dpost_weight, cols)
        o.vector("dpre_weight", dpre_weight, cols)
        self._finish(o, workspace)


class TokenLogprobs(_Call):
    """Log-probabilities of given tokens, entropy and top alternatives (rns8_mi355x_token_logprobs)."""

    _entry, _args = "rns8_mi355x_token_logprobs", abi.LogprobsArgs
    _query = "rns8_mi355x_token_logprobs_workspace"

    def __init__(self, ctx, *, logits, targets=None, logp=None, entropy=None, lse=None, top_ids=None, top_logp=None,
                 scale=1.0, workspace=None):
        o = self._begin(ctx, logits)
        rows, vocab = logits.shape
        top = next((t.shape[1] for t in (top_ids, top_logp) if t is not None), 0)
        self.args.rows, self.args.vocab, self.args.scale, self.args.top = rows, vocab, scale, top
        o.matrix("logits", "ldl", logits, rows, vocab)
        o.vector("targets", targets, rows, "int64")
        o.vector("logp", logp, rows)
        o.vector("entropy", entropy, rows)
        o.vector("lse", lse, rows)
        o.vector("top_ids", top_ids, rows * top, "int32")
        o.vector("top_logp", top_logp, rows * top)
        self._finish(o, workspace)


class TokenLogprobsBackward(_Call):
    """The gradient of log-probabilities and entropy (rns8_mi355x_token_logprobs_backward)."""

    _entry, _args = "rns8_mi355x_token_logprobs_backward", abi.LogprobsBackwardArgs

    def __init__(self, ctx, *, logits, lse, dlogits, targets=None, entropy=None, dlogp=None, dentropy=None, scale=1.0):
        o = self._begin(ctx, logits)
        rows, vocab = logits.shape
        self.args.rows, self.args.vocab, self.args.scale = rows, vocab, scale
        o.matrix("logits", "ldl", logits, rows, vocab)
        o.matrix("dlogits", "lddl", dlogits, rows, vocab)
        o.vector("targets", targets, rows, "int64")
        o.vector("lse", lse, rows)
        o.vector("entropy", entropy, rows)
        o.vector("dlogp", dlogp, rows)
        o.vector("dentropy", dentropy, rows)
        self._finish(o)
