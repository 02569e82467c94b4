// C entry points of the language-model operators (include/rns8_mi355x.h):
// argument checks, workspaces and the order of each operator's launches.
#include "operator_checks.hpp"

#include <cmath>

namespace rns8x {
namespace {

constexpr int64_t kMaxByteStride = int64_t{1} << 23;  // lda, ldb of 8-bit operands

// ---- quantization ------------------------------------------------------------------
rns8_status check_quantize(const rns8_mi355x_quantize_args& a, bool columns) {
  if (a.rows < 0 || a.cols < 1) return RNS8_INVALID_ARGUMENT;
  if (a.rows > kMaxSize || a.cols > kMaxSize) return RNS8_UNSUPPORTED_BACKEND;
  if (!operand_ok(a.x, a.rows, a.cols, a.ldx, element_size(a.dtype))) return RNS8_INVALID_ARGUMENT;
  const int64_t out_rows = columns ? a.cols : a.rows, out_cols = columns ? a.rows : a.cols;
  if (!operand_ok(a.q, out_rows, out_cols, a.ldq, 1) || !floats_ok(a.scale, out_rows)) return RNS8_INVALID_ARGUMENT;
  if (a.multiplier && !floats_ok(a.multiplier, columns ? a.rows : a.cols)) return RNS8_INVALID_ARGUMENT;
  if (a.sums && (!columns || !floats_ok(a.sums, a.cols))) return RNS8_INVALID_ARGUMENT;
  return RNS8_SUCCESS;
}

// ---- product ---------------------------------------------------------------------------
rns8_status check_gemm(const rns8_mi355x_gemm_i8_args& a) {
  if (a.m < 0 || a.n < 0 || a.k < 0 || a.reserved != 0) return RNS8_INVALID_ARGUMENT;
  if (a.b_layout != RNS8_MI355X_B_CHANNELS && a.b_layout != RNS8_MI355X_B_INNER) return RNS8_INVALID_ARGUMENT;
  const bool inner = a.b_layout == RNS8_MI355X_B_INNER;
  if (!operand_ok(a.a, a.m, a.k, a.lda, 1) || !operand_ok(a.b, inner ? a.k : a.n, inner ? a.n : a.k, a.ldb, 1) ||
      !operand_ok(a.out, a.m, a.n, a.ldo, element_size(a.dtype)))
    return RNS8_INVALID_ARGUMENT;
  if ((a.a_scale && !floats_ok(a.a_scale, a.m)) || (a.b_scale && !floats_ok(a.b_scale, a.n)) ||
      (a.bias && !floats_ok(a.bias, a.n)))
    return RNS8_INVALID_ARGUMENT;
  if (a.m > kMaxSize || a.n > (inner ? kMaxByteRow : kMaxProductCols) || a.k > kMaxByteRow || a.lda >= kMaxByteStride ||
      a.ldb >= kMaxByteStride)
    return RNS8_UNSUPPORTED_BACKEND;
  return RNS8_SUCCESS;
}

// ---- linear layer ------------------------------------------------------------------------
// The forward pass's workspace: the quantized rows and their scales where the
// caller keeps none, then the product's own.
struct LinearParts {
  rns8_mi355x_quantize_args quantize{};
  rns8_mi355x_gemm_i8_args gemm{};
  bool zero_filled = false;  // the quantized rows end in the zeros that the product may read
  bool fragments = false;    // the quantized rows, the caller wants none, are in fragment order
  uint64_t bytes = 0;
};

// Which way a call goes, for its workspace and for its launches alike: no
// outputs and no rows to keep, one kernel for all of it, or the parts below.
bool linear_is_empty(const rns8_mi355x_linear_i8_args& a) { return a.m == 0 || (a.n == 0 && !a.x_q); }
bool linear_in_one_kernel(const rns8_mi355x_linear_i8_args& a) {
  return a.m > 0 && a.n > 0 && linear_rows_takes(a.m, a.n, a.k);
}

// Quantized rows that a product may read whole 16-byte chunks of.
int64_t padded_row(int64_t cols) { return static_cast<int64_t>(round_up(static_cast<uint64_t>(cols), 16)); }

void linear_parts(const rns8_mi355x_linear_i8_args& a, LinearParts& p) {
  uint8_t* at = static_cast<uint8_t*>(a.workspace);
  auto take = [&](uint64_t bytes) {
    uint8_t* const got = at ? at + p.bytes : nullptr;
    p.bytes += round_up(bytes, 256);
    return got;
  };
  p.gemm.dtype = a.dtype;
  p.gemm.m = a.m;
  p.gemm.n = a.n;
  p.gemm.k = a.k;
  p.gemm.b = a.w;
  p.gemm.ldb = a.ldw;
  p.gemm.b_layout = RNS8_MI355X_B_CHANNELS;
  p.gemm.b_scale = a.w_scale;
  p.gemm.bias = a.bias;
  p.gemm.out = a.out;
  p.gemm.ldo = a.ldo;
  p.gemm.lda = padded_row(a.k);
  p.quantize.dtype = a.dtype;
  p.quantize.rows = a.m;
  p.quantize.cols = a.k;
  p.quantize.x = a.x;
  p.quantize.ldx = a.ldx;
  if (a.x_q) {
    p.quantize.q = a.x_q;
    p.quantize.ldq = a.ldq;
    p.quantize.scale = a.x_scale;
  } else {
    p.fragments = gemm_i8_takes_fragments(p.gemm);
    p.quantize.ldq = padded_row(a.k);
    const uint64_t bytes = p.fragments ? fragment_bytes(a.m, a.k)
                                       : static_cast<uint64_t>(a.m) * static_cast<uint64_t>(p.quantize.ldq);
    p.quantize.q = reinterpret_cast<int8_t*>(take(bytes));
    p.quantize.scale = reinterpret_cast<float*>(take(static_cast<uint64_t>(a.m) * sizeof(float)));
  }
  p.gemm.a = p.quantize.q;
  p.gemm.lda = p.quantize.ldq;
  p.gemm.a_scale = p.quantize.scale;
  if (p.fragments) return;  // (the kernel for few tokens needs no more)
  p.zero_filled = p.quantize.ldq >= padded_row(a.k);
  const uint64_t bytes = gemm_i8_bytes(p.gemm, p.zero_filled);
  p.gemm.workspace = take(bytes);
  p.gemm.workspace_bytes = bytes;
}

// The copies that can be made before the rows are quantized: the weights'. (Where
// the rows, too, would be copied, the product makes both copies itself.)
int weight_copies(const rns8_mi355x_gemm_i8_args& g, bool zero_filled, OperandCopy* copies) {
  const int count = gemm_i8_copies(g, zero_filled, copies);
  return count == 1 && copies[0].src == g.b ? 1 : 0;
}

rns8_status check_linear(const rns8_mi355x_linear_i8_args& a) {
  if (a.m < 0 || a.n < 0 || a.k < 1) return RNS8_INVALID_ARGUMENT;
  const uint64_t size = element_size(a.dtype);
  if (!operand_ok(a.x, a.m, a.k, a.ldx, size) || !operand_ok(a.w, a.n, a.k, a.ldw, 1) ||
      !operand_ok(a.out, a.m, a.n, a.ldo, size) || !floats_ok(a.w_scale, a.n) ||
      (a.bias && !floats_ok(a.bias, a.n)))
    return RNS8_INVALID_ARGUMENT;
  if (!a.x_q != !a.x_scale) return RNS8_INVALID_ARGUMENT;
  if (a.x_q && (!operand_ok(a.x_q, a.m, a.k, a.ldq, 1) || !floats_ok(a.x_scale, a.m))) return RNS8_INVALID_ARGUMENT;
  if (a.m > kMaxSize || a.n > kMaxProductCols || a.k >= kMaxByteRow || a.ldw >= kMaxByteStride ||
      (a.x_q && a.ldq >= kMaxByteStride))
    return RNS8_UNSUPPORTED_BACKEND;
  return RNS8_SUCCESS;
}

// The backward pass's workspace: dy in 8 bits by rows and, transposed, by
// columns, the column pass's partials and the products' own.
struct BackwardParts {
  rns8_mi355x_quantize_args rows{}, columns{};
  rns8_mi355x_gemm_i8_args dx{}, dw{};
  uint64_t bytes = 0;
};

// (n and k are at least 1)
bool both_products(const rns8_mi355x_linear_i8_backward_args& a) { return a.dx && a.dw && a.m > 0; }

void backward_parts(const rns8_mi355x_linear_i8_backward_args& a, BackwardParts& p) {
  uint8_t* at = static_cast<uint8_t*>(a.workspace);
  auto take = [&](uint64_t bytes) {
    uint8_t* const got = at ? at + p.bytes : nullptr;
    p.bytes += round_up(bytes, 256);
    return got;
  };
  if (a.dx) {
    p.rows.dtype = a.dtype;
    p.rows.rows = a.m;
    p.rows.cols = a.n;
    p.rows.x = a.dy;
    p.rows.ldx = a.lddy;
    p.rows.multiplier = a.w_scale;
    p.rows.ldq = padded_row(a.n);
    p.rows.q = reinterpret_cast<int8_t*>(take(static_cast<uint64_t>(a.m) * static_cast<uint64_t>(p.rows.ldq)));
    p.rows.scale = reinterpret_cast<float*>(take(static_cast<uint64_t>(a.m) * sizeof(float)));
    p.dx.dtype = a.dtype;
    p.dx.m = a.m;
    p.dx.n = a.k;
    p.dx.k = a.n;
    p.dx.a = p.rows.q;
    p.dx.lda = p.rows.ldq;
    p.dx.b = a.w;
    p.dx.ldb = a.ldw;
    p.dx.b_layout = RNS8_MI355X_B_INNER;
    p.dx.a_scale = p.rows.scale;
    p.dx.out = a.dx;
    p.dx.ldo = a.lddx;
  }
  if (a.dw || a.dbias) {
    p.columns.dtype = a.dtype;
    p.columns.rows = a.m;
    p.columns.cols = a.n;
    p.columns.x = a.dy;
    p.columns.ldx = a.lddy;
    p.columns.multiplier = a.dw ? a.x_scale : nullptr;
    p.columns.ldq = padded_row(a.m);
    p.columns.q = reinterpret_cast<int8_t*>(take(static_cast<uint64_t>(a.n) * static_cast<uint64_t>(p.columns.ldq)));
    p.columns.scale = reinterpret_cast<float*>(take(static_cast<uint64_t>(a.n) * sizeof(float)));
    p.columns.sums = a.dbias;
    p.columns.workspace_bytes = quantize_columns_bytes(a.m, a.n);
    p.columns.workspace = take(p.columns.workspace_bytes);
    p.dw.dtype = RNS8_MI355X_F32;
    p.dw.m = a.n;
    p.dw.n = a.k;
    p.dw.k = a.m;
    p.dw.a = p.columns.q;
    p.dw.lda = p.columns.ldq;
    p.dw.b = a.x_q;
    p.dw.ldb = a.ldq;
    p.dw.b_layout = RNS8_MI355X_B_INNER;
    p.dw.a_scale = p.columns.scale;
    p.dw.out = a.dw;
    p.dw.ldo = a.lddw;
  }
  uint64_t bytes[2] = {};
  if (both_products(a)) {
    gemm_i8_pair_bytes(p.dx, p.dw, bytes);
  } else {
    if (a.dx) bytes[0] = gemm_i8_bytes(p.dx, true);
    if (a.dw) bytes[1] = gemm_i8_bytes(p.dw, true);
  }
  p.dx.workspace_bytes = bytes[0];
  p.dx.workspace = take(bytes[0]);
  p.dw.workspace_bytes = bytes[1];
  p.dw.workspace = take(bytes[1]);
}

rns8_status check_linear_backward(const rns8_mi355x_linear_i8_backward_args& a) {
  if (a.m < 0 || a.n < 1 || a.k < 1 || (a.m > 0 && !a.dx && !a.dw && !a.dbias)) return RNS8_INVALID_ARGUMENT;
  const uint64_t size = element_size(a.dtype);
  if (!operand_ok(a.dy, a.m, a.n, a.lddy, size)) return RNS8_INVALID_ARGUMENT;
  if (a.dx && (!operand_ok(a.dx, a.m, a.k, a.lddx, size) || !operand_ok(a.w, a.n, a.k, a.ldw, 1) ||
               !floats_ok(a.w_scale, a.n)))
    return RNS8_INVALID_ARGUMENT;
  if (a.dw && (!operand_ok(a.dw, a.n, a.k, a.lddw, sizeof(float)) || !operand_ok(a.x_q, a.m, a.k, a.ldq, 1) ||
               !floats_ok(a.x_scale, a.m)))
    return RNS8_INVALID_ARGUMENT;
  if (a.dbias && !floats_ok(a.dbias, a.n)) return RNS8_INVALID_ARGUMENT;
  if (a.k > ((a.dx || a.dw) ? kMaxByteRow : kMaxSize) || (a.dx && (a.n >= kMaxByteRow || a.ldw >= kMaxByteStride)) ||
      ((a.dw || a.dbias) && (a.m >= kMaxByteRow || a.n > kMaxSize)) || (a.dw && a.ldq >= kMaxByteStride) ||
      a.m > kMaxSize)
    return RNS8_UNSUPPORTED_BACKEND;
  return RNS8_SUCCESS;
}

// ---- block norm ---------------------------------------------------------------------------
template <typename A>
rns8_status check_norm_inputs(const A& a) {
  if (a.rows < 0 || a.cols < 1 || (a.flags & ~(RNS8_MI355X_NORM_POST | RNS8_MI355X_NORM_PRE)) != 0)
    return RNS8_INVALID_ARGUMENT;
  if (!(a.eps >= 0.0f) || !std::isfinite(a.eps) || !std::isfinite(a.branch_scale) || !std::isfinite(a.residual_scale))
    return RNS8_INVALID_ARGUMENT;
  const uint64_t size = element_size(a.dtype);
  if (!operand_ok(a.x, a.rows, a.cols, a.ldx, size) || !optional_ok(a.residual, a.rows, a.cols, a.ldresidual, size) ||
      !optional_ok(a.post_weight, 1, a.cols, a.cols, size) || !optional_ok(a.pre_weight, 1, a.cols, a.cols, size))
    return RNS8_INVALID_ARGUMENT;
  if (a.gate && !(a.ldgate == 0 ? operand_ok(a.gate, 1, a.cols, a.cols, size)
                                : operand_ok(a.gate, a.rows, a.cols, a.ldgate, size)))
    return RNS8_INVALID_ARGUMENT;
  return RNS8_SUCCESS;
}

rns8_status check_norm(const rns8_mi355x_block_norm_args& a) {
  const rns8_status st = check_norm_inputs(a);
  if (st != RNS8_SUCCESS) return st;
  const bool pre = (a.flags & RNS8_MI355X_NORM_PRE) != 0;
  const uint64_t size = element_size(a.dtype);
  if (!optional_ok(a.h, a.rows, a.cols, a.ldh, size) || !optional_ok(a.y, a.rows, a.cols, a.ldy, size) ||
      !optional_ok(a.q, a.rows, a.cols, a.ldq, 1))
    return RNS8_INVALID_ARGUMENT;
  if (!in_place_ok(a.x, a.ldx, a.h, a.ldh, a.rows) || !in_place_ok(a.residual, a.ldresidual, a.h, a.ldh, a.rows))
    return RNS8_INVALID_ARGUMENT;
  if (!a.q != !a.q_scale) return RNS8_INVALID_ARGUMENT;
  if (a.rows > 0 && (pre ? !a.y && !a.q : !a.h)) return RNS8_INVALID_ARGUMENT;
  if (!pre && (a.y || a.q)) return RNS8_INVALID_ARGUMENT;
  if ((a.q_scale && !floats_ok(a.q_scale, a.rows)) || (a.rstd && !floats_ok(a.rstd, a.rows)))
    return RNS8_INVALID_ARGUMENT;
  return a.rows > kMaxSize || a.cols > kMaxNormCols ? RNS8_UNSUPPORTED_BACKEND : RNS8_SUCCESS;
}

rns8_status check_norm_backward(const rns8_mi355x_block_norm_backward_args& a) {
  const rns8_status st = check_norm_inputs(a);
  if (st != RNS8_SUCCESS) return st;
  const bool pre = (a.flags & RNS8_MI355X_NORM_PRE) != 0;
  const uint64_t size = element_size(a.dtype);
  if (a.rows > 0 && ((!a.dy && !a.dh) || !floats_ok(a.rstd, a.rows))) return RNS8_INVALID_ARGUMENT;
  if (!pre && (a.dy || a.dpre_weight)) return RNS8_INVALID_ARGUMENT;
  if (!optional_ok(a.dy, a.rows, a.cols, a.lddy, size) || !optional_ok(a.dh, a.rows, a.cols, a.lddh, size) ||
      !optional_ok(a.dx, a.rows, a.cols, a.lddx, size) ||
      !optional_ok(a.dresidual, a.rows, a.cols, a.lddresidual, size))
    return RNS8_INVALID_ARGUMENT;
  if (a.dpost_weight && (!(a.flags & RNS8_MI355X_NORM_POST) || !floats_ok(a.dpost_weight, a.cols)))
    return RNS8_INVALID_ARGUMENT;
  if (a.dpre_weight && !floats_ok(a.dpre_weight, a.cols)) return RNS8_INVALID_ARGUMENT;
  if (a.dgate && (!a.gate || !(a.ldgate == 0 ? floats_ok(a.dgate, a.cols)
                                             : operand_ok(a.dgate, a.rows, a.cols, a.lddgate, size))))
    return RNS8_INVALID_ARGUMENT;
  if (a.rows > 0 && !a.dx && !a.dresidual && !a.dgate && !a.dpost_weight && !a.dpre_weight) return RNS8_INVALID_ARGUMENT;
  return a.rows > kMaxSize || a.cols > kMaxNormCols ? RNS8_UNSUPPORTED_BACKEND : RNS8_SUCCESS;
}

// ---- token log-probabilities ------------------------------------------------------------------
bool ids_ok(const void* p, int64_t rows) { return operand_ok(p, 1, rows, rows, sizeof(int64_t)); }

rns8_status check_logprobs(const rns8_mi355x_logprobs_args& a) {
  if (a.rows < 0 || a.vocab < 1 || !(a.scale > 0.0f) || !std::isfinite(a.scale)) return RNS8_INVALID_ARGUMENT;
  if (!operand_ok(a.logits, a.rows, a.vocab, a.ldl, element_size(a.dtype))) return RNS8_INVALID_ARGUMENT;
  if ((a.logp && (!floats_ok(a.logp, a.rows) || !ids_ok(a.targets, a.rows))) ||
      (a.entropy && !floats_ok(a.entropy, a.rows)) || (a.lse && !floats_ok(a.lse, a.rows)))
    return RNS8_INVALID_ARGUMENT;
  if (a.top > kMaxTop || static_cast<int64_t>(a.top) > a.vocab) return RNS8_INVALID_ARGUMENT;
  if (a.top == 0 ? a.top_ids || a.top_logp : a.rows > 0 && !a.top_ids && !a.top_logp) return RNS8_INVALID_ARGUMENT;
  if (!optional_ok(a.top_ids, a.rows, a.top, a.top, sizeof(int32_t)) ||
      !optional_ok(a.top_logp, a.rows, a.top, a.top, sizeof(float)))
    return RNS8_INVALID_ARGUMENT;
  if (a.rows > 0 && !a.logp && !a.entropy && !a.lse && a.top == 0) return RNS8_INVALID_ARGUMENT;
  return a.rows > kMaxSize || a.vocab > kMaxSize ? RNS8_UNSUPPORTED_BACKEND : RNS8_SUCCESS;
}

rns8_status check_logprobs_backward(const rns8_mi355x_logprobs_backward_args& a) {
  if (a.rows < 0 || a.vocab < 1 || !(a.scale > 0.0f) || !std::isfinite(a.scale) || a.reserved != 0)
    return RNS8_INVALID_ARGUMENT;
  const uint64_t size = element_size(a.dtype);
  if (!operand_ok(a.logits, a.rows, a.vocab, a.ldl, size) || !operand_ok(a.dlogits, a.rows, a.vocab, a.lddl, size) ||
      !floats_ok(a.lse, a.rows))
    return RNS8_INVALID_ARGUMENT;
  if (!in_place_ok(a.logits, a.ldl, a.dlogits, a.lddl, a.rows)) return RNS8_INVALID_ARGUMENT;
  if (a.rows > 0 && !a.dlogp && !a.dentropy) return RNS8_INVALID_ARGUMENT;
  if (a.dlogp && (!floats_ok(a.dlogp, a.rows) || !ids_ok(a.targets, a.rows))) return RNS8_INVALID_ARGUMENT;
  if (a.dentropy && (!floats_ok(a.dentropy, a.rows) || !floats_ok(a.entropy, a.rows))) return RNS8_INVALID_ARGUMENT;
  return a.rows > kMaxSize || a.vocab > kMaxSize ? RNS8_UNSUPPORTED_BACKEND : RNS8_SUCCESS;
}

uint64_t linear_bytes(rns8_mi355x_linear_i8_args a) {
  if (linear_is_empty(a) || linear_in_one_kernel(a)) return 0;
  a.workspace = nullptr;
  LinearParts p;
  linear_parts(a, p);
  return p.bytes;
}

uint64_t linear_backward_bytes(rns8_mi355x_linear_i8_backward_args a) {
  a.workspace = nullptr;
  BackwardParts p;
  backward_parts(a, p);
  return p.bytes;
}

}  // namespace
}  // namespace rns8x

using namespace rns8x;

extern "C" {

rns8_status rns8_mi355x_quantize_rows(rns8_context* ctx, const rns8_mi355x_quantize_args* args, void* stream) {
  return run_operator(
      ctx, args, stream, [](const rns8_mi355x_quantize_args& a) { return check_quantize(a, false); },
      no_workspace<rns8_mi355x_quantize_args>, launch_quantize_rows);
}

rns8_status rns8_mi355x_quantize_columns(rns8_context* ctx, const rns8_mi355x_quantize_args* args, void* stream) {
  return run_operator(
      ctx, args, stream, [](const rns8_mi355x_quantize_args& a) { return check_quantize(a, true); },
      [](const rns8_mi355x_quantize_args& a) {
        return check_workspace(a.workspace, a.workspace_bytes, quantize_columns_bytes(a.rows, a.cols));
      },
      launch_quantize_columns);
}

rns8_status rns8_mi355x_quantize_columns_workspace(const rns8_mi355x_quantize_args* args, uint64_t* bytes) {
  return workspace_query(
      args, bytes, [](const rns8_mi355x_quantize_args& a) { return check_quantize(a, true); },
      [](const rns8_mi355x_quantize_args& a) { return quantize_columns_bytes(a.rows, a.cols); });
}

rns8_status rns8_mi355x_gemm_i8_scaled(rns8_context* ctx, const rns8_mi355x_gemm_i8_args* args, void* stream) {
  return run_operator(
      ctx, args, stream, check_gemm,
      [](const rns8_mi355x_gemm_i8_args& a) {
        return check_workspace(a.workspace, a.workspace_bytes, gemm_i8_bytes(a, false));
      },
      [](const rns8_mi355x_gemm_i8_args& a, hipStream_t s) { return launch_gemm_i8(a, false, false, s); });
}

rns8_status rns8_mi355x_gemm_i8_scaled_workspace(const rns8_mi355x_gemm_i8_args* args, uint64_t* bytes) {
  return workspace_query(args, bytes, check_gemm,
                         [](const rns8_mi355x_gemm_i8_args& a) { return gemm_i8_bytes(a, false); });
}

rns8_status rns8_mi355x_linear_i8(rns8_context* ctx, const rns8_mi355x_linear_i8_args* args, void* stream) {
  return run_operator(
      ctx, args, stream, check_linear,
      [](const rns8_mi355x_linear_i8_args& a) {
        return check_workspace(a.workspace, a.workspace_bytes, linear_bytes(a));
      },
      [](const rns8_mi355x_linear_i8_args& a, hipStream_t s) {
        if (linear_is_empty(a)) return hipSuccess;
        if (linear_in_one_kernel(a)) return launch_linear_rows(a, s);
        LinearParts p;
        linear_parts(a, p);
        if (p.fragments) {
          const hipError_t e = launch_quantize_fragments(p.quantize, s);
          return e != hipSuccess ? e : launch_gemm_i8_fragments(p.gemm, s);
        }
        OperandCopy copies[2];
        const int count = weight_copies(p.gemm, p.zero_filled, copies);
        const hipError_t e = count ? launch_prepare(&p.quantize, nullptr, copies, count, s)
                                   : launch_quantize_rows(p.quantize, s);
        return e != hipSuccess ? e : launch_gemm_i8(p.gemm, p.zero_filled, count != 0, s);
      });
}

rns8_status rns8_mi355x_linear_i8_workspace(const rns8_mi355x_linear_i8_args* args, uint64_t* bytes) {
  return workspace_query(args, bytes, check_linear, linear_bytes);
}

rns8_status rns8_mi355x_linear_i8_backward(rns8_context* ctx, const rns8_mi355x_linear_i8_backward_args* args,
                                           void* stream) {
  return run_operator(
      ctx, args, stream, check_linear_backward,
      [](const rns8_mi355x_linear_i8_backward_args& a) {
        return check_workspace(a.workspace, a.workspace_bytes, linear_backward_bytes(a));
      },
      [](const rns8_mi355x_linear_i8_backward_args& a, hipStream_t s) {
        BackwardParts p;
        backward_parts(a, p);
        const bool columns = a.dw || a.dbias;
        OperandCopy copies[4];
        int count = a.dx ? gemm_i8_copies(p.dx, true, copies) : 0;
        if (a.dw) count += gemm_i8_copies(p.dw, true, copies + count);
        hipError_t e = launch_prepare(a.dx ? &p.rows : nullptr, columns ? &p.columns : nullptr, copies, count, s);
        if (e == hipSuccess && columns) e = launch_quantize_columns_rest(p.columns, s);
        if (both_products(a)) return e != hipSuccess ? e : launch_gemm_i8_pair(p.dx, p.dw, s);
        if (e == hipSuccess && a.dx) e = launch_gemm_i8(p.dx, true, true, s);
        if (e == hipSuccess && a.dw) e = launch_gemm_i8(p.dw, true, true, s);
        return e;
      });
}

rns8_status rns8_mi355x_linear_i8_backward_workspace(const rns8_mi355x_linear_i8_backward_args* args,
                                                     uint64_t* bytes) {
  return workspace_query(args, bytes, check_linear_backward, linear_backward_bytes);
}

rns8_status rns8_mi355x_block_norm(rns8_context* ctx, const rns8_mi355x_block_norm_args* args, void* stream) {
  return run_operator(ctx, args, stream, check_norm, no_workspace<rns8_mi355x_block_norm_args>, launch_block_norm);
}

rns8_status rns8_mi355x_block_norm_backward(rns8_context* ctx, const rns8_mi355x_block_norm_backward_args* args,
                                            void* stream) {
  return run_operator(
      ctx, args, stream, check_norm_backward,
      [](const rns8_mi355x_block_norm_backward_args& a) {
        return check_workspace(a.workspace, a.workspace_bytes, block_norm_backward_bytes(a));
      },
      launch_block_norm_backward);
}

rns8_status rns8_mi355x_block_norm_backward_workspace(const rns8_mi355x_block_norm_backward_args* args,
                                                      uint64_t* bytes) {
  return workspace_query(args, bytes, check_norm_backward, block_norm_backward_bytes);
}

rns8_status rns8_mi355x_token_logprobs(rns8_context* ctx, const rns8_mi355x_logprobs_args* args, void* stream) {
  return run_operator(
      ctx, args, stream, check_logprobs,
      [](const rns8_mi355x_logprobs_args& a) {
        return check_workspace(a.workspace, a.workspace_bytes, logprobs_bytes(a));
      },
      launch_logprobs);
}

rns8_status rns8_mi355x_token_logprobs_workspace(const rns8_mi355x_logprobs_args* args, uint64_t* bytes) {
  return workspace_query(args, bytes, check_logprobs, logprobs_bytes);
}

rns8_status rns8_mi355x_token_logprobs_backward(rns8_context* ctx, const rns8_mi355x_logprobs_backward_args* args,
                                                void* stream) {
  return run_operator(ctx, args, stream, check_logprobs_backward, no_workspace<rns8_mi355x_logprobs_backward_args>,
                      launch_logprobs_backward);
}

}  // extern "C"
