// C entry points of the operators on 4-bit microscaled matrices
// (include/rns8_mi355x.h): argument checks, workspaces and the order of launches.
#include "mx4.hpp"
#include "operator_checks.hpp"

namespace rns8x {
namespace {

// An MX4 operand; one without elements may be NULL.
bool mx4_ok(const uint8_t* p, int64_t rows, int64_t cols) {
  return rows == 0 || cols == 0 || (p && reinterpret_cast<uintptr_t>(p) % 16 == 0);
}

// ---- rounding and back ---------------------------------------------------------------
rns8_status check_mx4(const rns8_mi355x_mx4_args& a, bool back) {
  if (a.rows < 0 || a.cols < 1 || (back ? a.q_t != nullptr : a.rows > 0 && !a.q && !a.q_t)) return RNS8_INVALID_ARGUMENT;
  if (!operand_ok(a.x, a.rows, a.cols, a.ldx, element_size(a.dtype)) ||
      ((back || a.q) && !mx4_ok(a.q, a.rows, a.cols)) || (a.q_t && !mx4_ok(a.q_t, a.cols, a.rows)))
    return RNS8_INVALID_ARGUMENT;
  return a.rows > kMaxMx4Size || a.cols > kMaxMx4Size ? RNS8_UNSUPPORTED_BACKEND : RNS8_SUCCESS;
}

rns8_status check_pack(const rns8_mi355x_pack_mx4_args& a) {
  if (a.dtype != 0 || a.rows < 0 || a.cols < 1) return RNS8_INVALID_ARGUMENT;
  if (a.rows > kMaxMx4Size || a.cols > kMaxMx4Size) return RNS8_UNSUPPORTED_BACKEND;
  return operand_ok(a.data, a.rows, (a.cols + 1) / 2, a.ldd, 1) && operand_ok(a.scale, a.rows, (a.cols + 31) / 32, a.lds, 1) &&
                 mx4_ok(a.q, a.rows, a.cols)
             ? RNS8_SUCCESS
             : RNS8_INVALID_ARGUMENT;
}

// ---- product ---------------------------------------------------------------------------
rns8_status check_gemm(const rns8_mi355x_gemm_mx4_args& a) {
  if (a.m < 0 || a.n < 0 || a.k < 0) return RNS8_INVALID_ARGUMENT;
  if (!mx4_ok(a.a, a.m, a.k) || !mx4_ok(a.b, a.n, a.k) || !operand_ok(a.out, a.m, a.n, a.ldo, element_size(a.dtype)) ||
      (a.bias && !floats_ok(a.bias, a.n)))
    return RNS8_INVALID_ARGUMENT;
  return a.m > kMaxMx4Size || a.n > kMaxMx4Size || a.k > kMaxMx4Sum ? RNS8_UNSUPPORTED_BACKEND : RNS8_SUCCESS;
}

Mx4Gemm gemm_of(int64_t m, int64_t n, int64_t k, const void* a, const uint8_t* b, const float* bias, void* out, int64_t ldo,
                uint32_t dtype) {
  Mx4Gemm g{};
  g.m = m;
  g.n = n;
  g.k = k;
  g.a = static_cast<const uint8_t*>(a);
  g.b = b;
  g.bias = bias;
  g.out = out;
  g.ldo = ldo;
  g.dtype = dtype;
  return g;
}

// A workspace's parts, one after the other; addresses are NULL where it has none yet.
struct Parts {
  uint8_t* at;
  uint64_t bytes = 0;
  uint8_t* take(uint64_t size) {
    uint8_t* const got = at ? at + bytes : nullptr;
    bytes += round_up(size, 256);
    return got;
  }
};

// ---- linear layer --------------------------------------------------------------------------
rns8_status check_linear(const rns8_mi355x_linear_mx4_args& a) {
  if (a.m < 0 || a.n < 0 || a.k < 1) return RNS8_INVALID_ARGUMENT;
  const uint64_t size = element_size(a.dtype);
  if (!operand_ok(a.x, a.m, a.k, a.ldx, size) || !mx4_ok(a.w, a.n, a.k) || !operand_ok(a.out, a.m, a.n, a.ldo, size) ||
      (a.bias && !floats_ok(a.bias, a.n)))
    return RNS8_INVALID_ARGUMENT;
  return a.m > kMaxMx4Size || a.n > kMaxMx4Size || a.k > kMaxMx4Sum ? RNS8_UNSUPPORTED_BACKEND : RNS8_SUCCESS;
}

struct LinearParts {
  uint8_t *rows = nullptr, *gemm = nullptr;
  uint64_t bytes = 0;
};
LinearParts linear_parts(const rns8_mi355x_linear_mx4_args& a, void* workspace) {
  LinearParts p;
  if (a.m == 0 || a.n == 0 || linear_mx4_in_one_kernel(a.m, a.n)) return p;
  Parts parts{static_cast<uint8_t*>(workspace)};
  p.rows = parts.take(mx4_bytes(a.m, a.k));
  p.gemm = parts.take(gemm_mx4_bytes(a.m, a.n, a.k));
  p.bytes = parts.bytes;
  return p;
}
uint64_t linear_bytes(const rns8_mi355x_linear_mx4_args& a) { return linear_parts(a, nullptr).bytes; }

hipError_t enqueue_linear(const rns8_mi355x_linear_mx4_args& a, hipStream_t s) {
  if (a.m == 0 || a.n == 0) return hipSuccess;
  const LinearParts p = linear_parts(a, a.workspace);
  Mx4Gemm g = gemm_of(a.m, a.n, a.k, p.rows, a.w, a.bias, a.out, a.ldo, a.dtype);
  if (linear_mx4_in_one_kernel(a.m, a.n)) {
    g.x = a.x;
    g.ldx = a.ldx;
    return launch_gemm_mx4(g, nullptr, s);
  }
  const Mx4Quantize rows{a.x, a.m, a.k, a.ldx, p.rows, nullptr, nullptr};
  const hipError_t e = launch_quantize_mx4(&rows, 1, a.dtype, s);
  return e != hipSuccess ? e : launch_gemm_mx4(g, p.gemm, s);
}

// ---- its gradients ---------------------------------------------------------------------------
rns8_status check_linear_backward(const rns8_mi355x_linear_mx4_backward_args& a) {
  if (a.m < 0 || a.n < 1 || a.k < 1 || (a.m > 0 && !a.dx && !a.dw && !a.dbias)) return RNS8_INVALID_ARGUMENT;
  const uint64_t size = element_size(a.dtype);
  if (!operand_ok(a.dy, a.m, a.n, a.lddy, size)) return RNS8_INVALID_ARGUMENT;
  if (a.dx && (!operand_ok(a.dx, a.m, a.k, a.lddx, size) || !mx4_ok(a.w_t, a.k, a.n))) return RNS8_INVALID_ARGUMENT;
  if (a.dw && (!operand_ok(a.dw, a.n, a.k, a.lddw, sizeof(float)) || !operand_ok(a.x, a.m, a.k, a.ldx, size)))
    return RNS8_INVALID_ARGUMENT;
  if (a.dbias && !floats_ok(a.dbias, a.n)) return RNS8_INVALID_ARGUMENT;
  return a.m > (a.dw ? kMaxMx4Sum : kMaxMx4Size) || a.n > (a.dx ? kMaxMx4Sum : kMaxMx4Size) || a.k > kMaxMx4Size
             ? RNS8_UNSUPPORTED_BACKEND
             : RNS8_SUCCESS;
}

struct BackwardParts {
  uint8_t *dy = nullptr, *dy_t = nullptr, *x_t = nullptr;
  Mx4Sums sums{};
  Mx4Gemm products[2] = {};  // dx and dw, empty where not wanted
  void* workspaces[2] = {};
  uint64_t bytes = 0;
};

BackwardParts backward_parts(const rns8_mi355x_linear_mx4_backward_args& a, void* workspace) {
  BackwardParts p;
  Parts parts{static_cast<uint8_t*>(workspace)};
  if (a.dx) {
    p.dy = parts.take(mx4_bytes(a.m, a.n));
    p.products[0] = gemm_of(a.m, a.k, a.n, p.dy, a.w_t, nullptr, a.dx, a.lddx, a.dtype);
  }
  if (a.dw) {
    p.dy_t = parts.take(mx4_bytes(a.n, a.m));
    p.x_t = parts.take(mx4_bytes(a.k, a.m));
    p.products[1] = gemm_of(a.n, a.k, a.m, p.dy_t, p.x_t, nullptr, a.dw, a.lddw, RNS8_MI355X_F32);
  }
  if (a.dbias) {
    p.sums.count = (a.m + 127) / 128;
    p.sums.cols = a.n;
    p.sums.out = a.dbias;
    p.sums.partials = reinterpret_cast<const float*>(
        parts.take(static_cast<uint64_t>(p.sums.count) * static_cast<uint64_t>(a.n) * sizeof(float)));
  }
  uint64_t bytes[2];
  gemm_mx4_pair_bytes(p.products, bytes);
  for (int i = 0; i < 2; ++i) p.workspaces[i] = parts.take(bytes[i]);
  p.bytes = parts.bytes;
  return p;
}
uint64_t backward_bytes(const rns8_mi355x_linear_mx4_backward_args& a) { return backward_parts(a, nullptr).bytes; }

hipError_t enqueue_backward(const rns8_mi355x_linear_mx4_backward_args& a, hipStream_t s) {
  const BackwardParts p = backward_parts(a, a.workspace);
  if (a.m > 0) {
    const Mx4Quantize jobs[2] = {{a.dy, a.m, a.n, a.lddy, p.dy, p.dy_t, const_cast<float*>(p.sums.partials)},
                                 {a.x, a.m, a.k, a.ldx, nullptr, p.x_t, nullptr}};
    const hipError_t e = launch_quantize_mx4(jobs, a.dw ? 2 : 1, a.dtype, s);
    if (e != hipSuccess) return e;
  }
  return launch_gemm_mx4_pair(p.products, p.workspaces, p.sums, s);
}

// ---- experts ---------------------------------------------------------------------------------
rns8_status check_experts(const rns8_mi355x_experts_mx4_args& a) {
  if (a.tokens < 0 || a.experts < 1 || a.width < 1 || a.inner < 1 || a.top < 1 || (a.flags & ~RNS8_MI355X_EXPERTS_NORMALIZE) != 0 ||
      static_cast<int64_t>(a.top) > a.experts)
    return RNS8_INVALID_ARGUMENT;
  if (a.tokens > kMaxExpertTokens || a.experts > kMaxExperts || a.top > kMaxExpertTop || a.width > kMaxExpertSize ||
      a.inner > kMaxExpertSize)
    return RNS8_UNSUPPORTED_BACKEND;
  const uint64_t size = element_size(a.dtype);
  if (!operand_ok(a.x, a.tokens, a.width, a.ldx, size) || !operand_ok(a.out, a.tokens, a.width, a.ldo, size) ||
      !optional_ok(a.router, a.experts, a.width, a.ldrouter, size))
    return RNS8_INVALID_ARGUMENT;
  if (!mx4_ok(a.gate, a.inner, a.width) || !mx4_ok(a.up, a.inner, a.width) || !mx4_ok(a.down, a.width, a.inner))
    return RNS8_INVALID_ARGUMENT;
  const int64_t pairs = a.tokens * a.top;
  if (!a.router && pairs > 0 && (!a.ids || !a.weights)) return RNS8_INVALID_ARGUMENT;
  return optional_ok(a.ids, 1, pairs, pairs, sizeof(int32_t)) && optional_ok(a.weights, 1, pairs, pairs, sizeof(float))
             ? RNS8_SUCCESS
             : RNS8_INVALID_ARGUMENT;
}

}  // namespace
}  // namespace rns8x

using namespace rns8x;

extern "C" {

rns8_status rns8_mi355x_quantize_mx4(rns8_context* ctx, const rns8_mi355x_mx4_args* args, void* stream) {
  return run_operator(
      ctx, args, stream, [](const rns8_mi355x_mx4_args& a) { return check_mx4(a, false); },
      no_workspace<rns8_mi355x_mx4_args>, [](const rns8_mi355x_mx4_args& a, hipStream_t s) {
        if (a.rows == 0) return hipSuccess;
        const Mx4Quantize job{a.x, a.rows, a.cols, a.ldx, a.q, a.q_t, nullptr};
        return launch_quantize_mx4(&job, 1, a.dtype, s);
      });
}

rns8_status rns8_mi355x_dequantize_mx4(rns8_context* ctx, const rns8_mi355x_mx4_args* args, void* stream) {
  return run_operator(
      ctx, args, stream, [](const rns8_mi355x_mx4_args& a) { return check_mx4(a, true); },
      no_workspace<rns8_mi355x_mx4_args>, launch_dequantize_mx4);
}

rns8_status rns8_mi355x_pack_mx4(rns8_context* ctx, const rns8_mi355x_pack_mx4_args* args, void* stream) {
  return run_operator(ctx, args, stream, check_pack, no_workspace<rns8_mi355x_pack_mx4_args>, launch_pack_mx4);
}

rns8_status rns8_mi355x_gemm_mx4(rns8_context* ctx, const rns8_mi355x_gemm_mx4_args* args, void* stream) {
  return run_operator(
      ctx, args, stream, check_gemm,
      [](const rns8_mi355x_gemm_mx4_args& a) {
        return check_workspace(a.workspace, a.workspace_bytes, gemm_mx4_bytes(a.m, a.n, a.k));
      },
      [](const rns8_mi355x_gemm_mx4_args& a, hipStream_t s) {
        return launch_gemm_mx4(gemm_of(a.m, a.n, a.k, a.a, a.b, a.bias, a.out, a.ldo, a.dtype), a.workspace, s);
      });
}

rns8_status rns8_mi355x_gemm_mx4_workspace(const rns8_mi355x_gemm_mx4_args* args, uint64_t* bytes) {
  return workspace_query(args, bytes, check_gemm,
                         [](const rns8_mi355x_gemm_mx4_args& a) { return gemm_mx4_bytes(a.m, a.n, a.k); });
}

rns8_status rns8_mi355x_linear_mx4(rns8_context* ctx, const rns8_mi355x_linear_mx4_args* args, void* stream) {
  return run_operator(
      ctx, args, stream, check_linear,
      [](const rns8_mi355x_linear_mx4_args& a) { return check_workspace(a.workspace, a.workspace_bytes, linear_bytes(a)); },
      enqueue_linear);
}

rns8_status rns8_mi355x_linear_mx4_workspace(const rns8_mi355x_linear_mx4_args* args, uint64_t* bytes) {
  return workspace_query(args, bytes, check_linear, linear_bytes);
}

rns8_status rns8_mi355x_linear_mx4_backward(rns8_context* ctx, const rns8_mi355x_linear_mx4_backward_args* args,
                                            void* stream) {
  return run_operator(
      ctx, args, stream, check_linear_backward,
      [](const rns8_mi355x_linear_mx4_backward_args& a) {
        return check_workspace(a.workspace, a.workspace_bytes, backward_bytes(a));
      },
      enqueue_backward);
}

rns8_status rns8_mi355x_linear_mx4_backward_workspace(const rns8_mi355x_linear_mx4_backward_args* args, uint64_t* bytes) {
  return workspace_query(args, bytes, check_linear_backward, backward_bytes);
}

rns8_status rns8_mi355x_experts_mx4(rns8_context* ctx, const rns8_mi355x_experts_mx4_args* args, void* stream) {
  return run_operator(
      ctx, args, stream, check_experts,
      [](const rns8_mi355x_experts_mx4_args& a) {
        return check_workspace(a.workspace, a.workspace_bytes, experts_mx4_bytes(a));
      },
      launch_experts_mx4);
}

rns8_status rns8_mi355x_experts_mx4_workspace(const rns8_mi355x_experts_mx4_args* args, uint64_t* bytes) {
  return workspace_query(args, bytes, check_experts, experts_mx4_bytes);
}

}  // extern "C"
