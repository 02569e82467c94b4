// The product of 8-bit matrices with a scale for each row and each column
// (gfx950): operands that the kernels cannot read in place are copied first,
// then the kernel of the product's shape runs.
#include <algorithm>

#include "elements.hpp"
#include "scaled_gemm.hpp"

namespace rns8x {
namespace {

// Copies rows of `cols` bytes at any address and stride to rows at stride ldd
// (cols rounded up to 16) and fills them up with zeros.
struct CopyArgs {
  const int8_t* src;
  int64_t rows, cols, lds;
  int8_t* dst;
  int64_t ldd;
};

// Four rows to a wave, 16 bytes of each to a lane at a time, all four loads in
// flight. The chunk that a row's end cuts comes from the row's last 16 bytes.
__global__ __launch_bounds__(256) void copy_rows_kernel(CopyArgs a) {
  const int lane = threadIdx.x & 63;
  const uint32_t cols = static_cast<uint32_t>(a.cols), padded = static_cast<uint32_t>(a.ldd);
  for (int64_t row = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * 4; row < a.rows;
       row += static_cast<int64_t>(gridDim.x) * 16) {
    const int64_t rows = a.rows - row;
    for (uint32_t c = 16 * (64 * blockIdx.y + lane); c < padded; c += 16 * 64 * gridDim.y) {
      u32x4 w[4];
      const bool whole = c + 16 <= cols;
      const uint32_t at = whole ? c : cols - 16, drop = whole ? 0 : c + 16 - cols;
#pragma unroll
      for (int r = 0; r < 4; ++r) __builtin_memcpy(&w[r], a.src + (row + min<int64_t>(r, rows - 1)) * a.lds + at, 16);
#pragma unroll
      for (int r = 0; r < 4; ++r) w[r] = drop_bytes(w[r], drop);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r < rows) __builtin_memcpy(a.dst + (row + r) * a.ldd + c, &w[r], 16);
    }
  }
}

// Rows below 16 bytes: one to a thread.
__global__ __launch_bounds__(256) void copy_short_rows_kernel(CopyArgs a) {
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; row < a.rows;
       row += static_cast<int64_t>(gridDim.x) * 256) {
    uint32_t w[4] = {};
#pragma unroll
    for (int i = 0; i < 15; ++i)
      if (i < a.cols)
        w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(a.src[row * a.lds + i])) << (8 * (i & 3));
    __builtin_memcpy(a.dst + row * a.ldd, w, 16);
  }
}

hipError_t launch_copy_rows(const CopyArgs& a, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  if (a.cols < 16) {
    const int64_t blocks = std::min<int64_t>((a.rows + 255) / 256, 1 << 16);
    hipLaunchKernelGGL(copy_short_rows_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  const int64_t blocks = (a.rows + 15) / 16;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(blocks, 1 << 16)),
                  static_cast<unsigned>(std::min<int64_t>((a.ldd + 1023) / 1024, 64)));
  hipLaunchKernelGGL(copy_rows_kernel, grid, dim3(256), 0, stream, a);
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

Plan make_plan(const rns8_mi355x_gemm_i8_args& g, bool a_zero_filled) {
  Plan p{};
  const bool inner = g.b_layout == RNS8_MI355X_B_INNER;
  p.lda = g.lda;
  p.ldb = g.ldb;
  p.tiles = choose_tile_shape(g.m, g.n, g.k);
  p.b_rows = inner ? g.k : g.n;
  p.b_cols = inner ? g.n : g.k;
  // where b is n x k, a's chunks are read whole: they have to end in zeros
  p.copy_a = g.k > 0 && !(in_place(g.a, g.lda) && (inner || a_zero_filled || g.k % 16 == 0));
  p.copy_b = g.k > 0 && !in_place(g.b, g.ldb);
  if (scaled_rows_takes(g.m, g.n, g.k, inner)) {
    // a copy: a launch, and its bytes read and written
    const double copies = (p.copy_a ? 2.0 + static_cast<double>(g.m) * static_cast<double>(g.k) / 2.5e6 : 0.0) +
                          (p.copy_b ? 2.0 + static_cast<double>(g.n) * static_cast<double>(g.k) / 2.5e6 : 0.0);
    p.few_rows = scaled_rows_cost(g.m, g.n, g.k) <= p.tiles.cost + copies;
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

}  // namespace

uint64_t gemm_i8_bytes(const rns8_mi355x_gemm_i8_args& g, bool a_zero_filled) {
  return g.m == 0 || g.n == 0 ? 0u : make_plan(g, a_zero_filled).bytes;
}

hipError_t launch_gemm_i8(const rns8_mi355x_gemm_i8_args& g, bool a_zero_filled, hipStream_t stream) {
  if (g.m == 0 || g.n == 0) return hipSuccess;
  const Plan p = make_plan(g, a_zero_filled);
  uint8_t* const ws = static_cast<uint8_t*>(g.workspace);
  ScaledGemm s{g.m, g.n, g.k, g.a, g.b, p.lda, p.ldb, g.b_layout == RNS8_MI355X_B_INNER, g.a_scale, g.b_scale, g.bias,
               g.out, g.ldo, g.dtype};
  if (p.few_rows) return launch_scaled_rows(s, stream);
  if (p.copy_a) {
    int8_t* const to = reinterpret_cast<int8_t*>(ws + p.a_at);
    const hipError_t e = launch_copy_rows({g.a, g.m, g.k, g.lda, to, p.lda}, stream);
    if (e != hipSuccess) return e;
    s.a = to;
  }
  if (p.copy_b) {
    int8_t* const to = reinterpret_cast<int8_t*>(ws + p.b_at);
    const hipError_t e = launch_copy_rows({g.b, p.b_rows, p.b_cols, g.ldb, to, p.ldb}, stream);
    if (e != hipSuccess) return e;
    s.b = to;
  }
  if (g.k == 0) {  // no operand is read (their buffers are empty): any aligned address will do
    s.a = s.b = static_cast<const int8_t*>(g.out) - reinterpret_cast<uintptr_t>(g.out) % 16;
    s.lda = 0;
    s.ldb = s.inner ? static_cast<int64_t>(round_up(static_cast<uint64_t>(g.n), 16)) : 0;
  }
  return launch_scaled_tiles(s, p.tiles, reinterpret_cast<int32_t*>(ws + p.sums_at), stream);
}

}  // namespace rns8x
