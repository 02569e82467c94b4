// The product of 8-bit matrices with a scale for each row and each column
// (gfx950): operands that the kernels cannot read in place are copied first,
// then the kernel of the product's shape runs.
#include <algorithm>

#include "operand_copy.hpp"
#include "scaled_gemm.hpp"

namespace rns8x {
namespace {

__global__ __launch_bounds__(256) void copy_rows_kernel(OperandCopy a) { copy_rows(a, blockIdx.x, gridDim.x); }

hipError_t launch_copy_rows(const OperandCopy& a, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  hipLaunchKernelGGL(copy_rows_kernel, dim3(operand_copy_blocks(a)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

bool in_place(const int8_t* p, int64_t ld) { return ld % 16 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// The workspace: copies of the operands that need one, then the partial sums.
struct Plan {
  bool few_rows;  // the kernel for few tokens (any alignment, no workspace) where it is predicted to be faster
  bool copy_a, copy_b;
  int64_t lda, ldb, b_rows, b_cols;
  uint64_t a_at, b_at, sums_at, bytes;
  TileShape tiles;
};

// fragments: for the choice, a as it would be in fragment order. tiles: how the
// tile kernel splits it, where that is settled already.
Plan make_plan(const rns8_mi355x_gemm_i8_args& g, bool a_zero_filled, bool fragments = false,
               const TileShape* tiles = nullptr) {
  Plan p{};
  const bool inner = g.b_layout == RNS8_MI355X_B_INNER;
  p.lda = g.lda;
  p.ldb = g.ldb;
  p.tiles = tiles ? *tiles : choose_tile_shape(g.m, g.n, g.k);
  p.b_rows = inner ? g.k : g.n;
  p.b_cols = inner ? g.n : g.k;
  p.copy_a = g.k > 0 && !in_place(g.a, g.lda);
  p.copy_b = g.k > 0 && !in_place(g.b, g.ldb);
  // where b is n x k and k ends inside a chunk, one of the two has to end in
  // zeros there, as copies do: the other's bytes then do not matter
  if (!inner && g.k % 16 != 0 && !a_zero_filled && !p.copy_a && !p.copy_b) (g.m <= g.n ? p.copy_a : p.copy_b) = true;
  if (scaled_rows_takes(g.m, g.n, g.k, inner)) {
    // a copy: a launch, and its bytes read and written
    const double copies = (p.copy_a ? 2.0 + static_cast<double>(g.m) * static_cast<double>(g.k) / 2.5e6 : 0.0) +
                          (p.copy_b ? 2.0 + static_cast<double>(g.n) * static_cast<double>(g.k) / 2.5e6 : 0.0);
    p.few_rows = scaled_rows_cost(g.m, g.n, g.k, fragments) <= p.tiles.cost + copies;
    if (p.few_rows) {
      p.copy_a = p.copy_b = false;
      return p;
    }
  }
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t got = at;
    at += round_up(bytes, 256);
    return got;
  };
  p.lda = p.copy_a ? static_cast<int64_t>(round_up(static_cast<uint64_t>(g.k), 16)) : g.lda;
  p.ldb = p.copy_b ? static_cast<int64_t>(round_up(static_cast<uint64_t>(p.b_cols), 16)) : g.ldb;
  if (p.copy_a) p.a_at = take(static_cast<uint64_t>(g.m) * static_cast<uint64_t>(p.lda));
  if (p.copy_b) p.b_at = take(static_cast<uint64_t>(p.b_rows) * static_cast<uint64_t>(p.ldb));
  p.sums_at = take(p.tiles.bytes);
  p.bytes = at;
  return p;
}

ScaledGemm planned(const rns8_mi355x_gemm_i8_args& g, const Plan& p) {
  int8_t* const ws = static_cast<int8_t*>(g.workspace);
  ScaledGemm s{g.m, g.n, g.k, g.a, g.b, p.lda, p.ldb, g.b_layout == RNS8_MI355X_B_INNER, g.a_scale, g.b_scale, g.bias,
               g.out, g.ldo, g.dtype};
  if (p.copy_a) s.a = ws + p.a_at;
  if (p.copy_b) s.b = ws + p.b_at;
  if (g.k == 0) {  // no operand is read (their buffers are empty): any aligned address will do
    s.a = s.b = static_cast<const int8_t*>(g.out) - reinterpret_cast<uintptr_t>(g.out) % 16;
    s.lda = 0;
    s.ldb = s.inner ? static_cast<int64_t>(round_up(static_cast<uint64_t>(g.n), 16)) : 0;
  }
  return s;
}

int32_t* sums_of(const rns8_mi355x_gemm_i8_args& g, const Plan& p) {
  return reinterpret_cast<int32_t*>(static_cast<int8_t*>(g.workspace) + p.sums_at);
}

bool pair_shapes(const rns8_mi355x_gemm_i8_args& x, const rns8_mi355x_gemm_i8_args& y, TileShape (&shapes)[2]) {
  return choose_pair_shapes({x.m, y.m}, {x.n, y.n}, {x.k, y.k}, shapes);
}

}  // namespace

uint64_t gemm_i8_bytes(const rns8_mi355x_gemm_i8_args& g, bool a_zero_filled) {
  return g.m == 0 || g.n == 0 ? 0u : make_plan(g, a_zero_filled).bytes;
}

int gemm_i8_copies(const rns8_mi355x_gemm_i8_args& g, bool a_zero_filled, OperandCopy* copies) {
  if (g.m == 0 || g.n == 0) return 0;
  const Plan p = make_plan(g, a_zero_filled);
  int8_t* const ws = static_cast<int8_t*>(g.workspace);
  int count = 0;
  if (p.copy_a) copies[count++] = {g.a, g.m, g.k, g.lda, ws + p.a_at, p.lda};
  if (p.copy_b) copies[count++] = {g.b, p.b_rows, p.b_cols, g.ldb, ws + p.b_at, p.ldb};
  return count;
}

// More than one tile of tokens is read by every workgroup: 48 tokens by 8192 x
// 4096 13.1 us from rows, 10.7 in fragment order.
bool gemm_i8_takes_fragments(const rns8_mi355x_gemm_i8_args& g) {
  return g.m > 16 && g.n > 0 && make_plan(g, true, true).few_rows;
}

hipError_t launch_gemm_i8_fragments(const rns8_mi355x_gemm_i8_args& g, hipStream_t stream) {
  ScaledGemm s{g.m, g.n, g.k, g.a, g.b, g.lda, g.ldb, false, g.a_scale, g.b_scale, g.bias, g.out, g.ldo, g.dtype};
  s.fragments = true;
  return launch_scaled_rows(s, stream);
}

hipError_t launch_gemm_i8(const rns8_mi355x_gemm_i8_args& g, bool a_zero_filled, bool copied, hipStream_t stream) {
  if (g.m == 0 || g.n == 0) return hipSuccess;
  const Plan p = make_plan(g, a_zero_filled);
  const ScaledGemm s = planned(g, p);
  if (p.few_rows) return launch_scaled_rows(s, stream);
  if (!copied) {
    OperandCopy copies[2];
    const int count = gemm_i8_copies(g, a_zero_filled, copies);
    for (int i = 0; i < count; ++i) {
      const hipError_t e = launch_copy_rows(copies[i], stream);
      if (e != hipSuccess) return e;
    }
  }
  int32_t* const sums = sums_of(g, p);
  return launch_scaled_tiles(&s, &p.tiles, &sums, 1, stream);
}

void gemm_i8_pair_bytes(const rns8_mi355x_gemm_i8_args& x, const rns8_mi355x_gemm_i8_args& y, uint64_t (&bytes)[2]) {
  TileShape shapes[2];
  pair_shapes(x, y, shapes);
  bytes[0] = make_plan(x, true, false, &shapes[0]).bytes;
  bytes[1] = make_plan(y, true, false, &shapes[1]).bytes;
}

hipError_t launch_gemm_i8_pair(const rns8_mi355x_gemm_i8_args& x, const rns8_mi355x_gemm_i8_args& y,
                               hipStream_t stream) {
  TileShape shapes[2];
  const bool one_launch = pair_shapes(x, y, shapes);
  const Plan p[2] = {make_plan(x, true, false, &shapes[0]), make_plan(y, true, false, &shapes[1])};
  const ScaledGemm s[2] = {planned(x, p[0]), planned(y, p[1])};
  int32_t* const sums[2] = {sums_of(x, p[0]), sums_of(y, p[1])};
  if (one_launch) return launch_scaled_tiles(s, shapes, sums, 2, stream);
  const hipError_t e = launch_scaled_tiles(&s[0], &shapes[0], &sums[0], 1, stream);
  return e != hipSuccess ? e : launch_scaled_tiles(&s[1], &shapes[1], &sums[1], 1, stream);
}

}  // namespace rns8x
