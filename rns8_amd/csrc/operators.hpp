// Host-side launchers of the language-model operators (defined in the .hip
// files). The C entry points (api_operators.cpp) check the arguments; the
// launchers check what their own grids and index arithmetic assume and return
// hipErrorInvalidValue otherwise.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "rns8_mi355x.h"

namespace rns8x {

inline uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// Whether an output's stores pass the caches by: a launch that moves as many bytes
// as the Infinity Cache holds (256 MB) leaves it full of dirty lines, little of
// which survives to be read and whose way out competes with the next kernel's
// reads. Norm gradients of 8192 x 4096 93 us with ordinary stores, 74 past the
// caches; the loss over 4096 x 32768 reads its logits in 78 us after ordinary
// stores of the last gradient, in 50 after these. Rows of 16-byte aligned
// vectors only.
inline bool streams(int64_t bytes_moved, const void* p, int64_t ld, uint32_t dtype) {
  return bytes_moved >= (int64_t{256} << 20) && reinterpret_cast<uintptr_t>(p) % 16 == 0 &&
         ld * (dtype == RNS8_MI355X_F32 ? 4 : 2) % 16 == 0;
}

// ---- quantization (quantize.hip) -------------------------------------------------
hipError_t launch_quantize_rows(const rns8_mi355x_quantize_args& a, hipStream_t stream);
// Rows in fragment order, as the matrix cores take them: blocks of 64 columns;
// in each, tiles of 16 rows of 1024 bytes, chunk g (16 columns) of row r at 256 g
// + 16 r. Zeros up to whole blocks. A product of few tokens then reads its rows
// in whole cache lines.
inline __host__ __device__ int64_t fragment_offset(int64_t row, int64_t col, uint32_t tiles) {
  return ((col / 64) * tiles + row / 16) * 1024 + (col % 64) / 16 * 256 + row % 16 * 16 + col % 16;
}
inline uint64_t fragment_bytes(int64_t rows, int64_t cols) {
  return static_cast<uint64_t>((rows + 15) / 16) * static_cast<uint64_t>((cols + 63) / 64) * 1024u;
}
hipError_t launch_quantize_fragments(const rns8_mi355x_quantize_args& a, hipStream_t stream);
uint64_t quantize_columns_bytes(int64_t rows, int64_t cols);
hipError_t launch_quantize_columns(const rns8_mi355x_quantize_args& a, hipStream_t stream);

// A copy of rows of `cols` bytes at any address and stride to rows at stride
// ldd (cols rounded up to 16), filled up with zeros (operand_copy.hpp).
struct OperandCopy {
  const int8_t* src;
  int64_t rows, cols, lds;
  int8_t* dst;
  int64_t ldd;
};
inline uint32_t operand_copy_blocks(const OperandCopy& a) {
  const int64_t units = a.cols < 16 ? (a.rows + 255) / 256 : (a.rows + 15) / 16 * ((a.ldd + 1023) / 1024);
  return static_cast<uint32_t>(units < (1 << 16) ? units : 1 << 16);
}

// What a linear layer's products wait for, in one launch: rows to quantize,
// columns' partial maxima and sums, and operand copies (any of them NULL or 0).
// launch_quantize_columns_rest then finishes the columns.
hipError_t launch_prepare(const rns8_mi355x_quantize_args* rows, const rns8_mi355x_quantize_args* columns,
                          const OperandCopy* copies, int copy_count, hipStream_t stream);
hipError_t launch_quantize_columns_rest(const rns8_mi355x_quantize_args& a, hipStream_t stream);

// ---- scaled product (scaled_gemm.hip) ----------------------------------------------
// a_zero_filled: a's rows hold zeros from k up to the next multiple of 16 (and
// their stride reaches it), as quantized rows do: the product may read them.
uint64_t gemm_i8_bytes(const rns8_mi355x_gemm_i8_args& a, bool a_zero_filled);
// The copies (at most two) that the product needs of its operands, into its
// workspace; launch_gemm_i8 makes them itself unless `copied`.
int gemm_i8_copies(const rns8_mi355x_gemm_i8_args& a, bool a_zero_filled, OperandCopy* copies);
hipError_t launch_gemm_i8(const rns8_mi355x_gemm_i8_args& a, bool a_zero_filled, bool copied, hipStream_t stream);
// Two products with rows in each, both with b k x n, zero-filled rows of a and their
// copies made: in one launch where that is faster. Their workspaces are apart.
void gemm_i8_pair_bytes(const rns8_mi355x_gemm_i8_args& x, const rns8_mi355x_gemm_i8_args& y, uint64_t (&bytes)[2]);
hipError_t launch_gemm_i8_pair(const rns8_mi355x_gemm_i8_args& x, const rns8_mi355x_gemm_i8_args& y,
                               hipStream_t stream);
// Whether the product would rather have its rows in fragment order, and the product of such rows.
bool gemm_i8_takes_fragments(const rns8_mi355x_gemm_i8_args& a);
hipError_t launch_gemm_i8_fragments(const rns8_mi355x_gemm_i8_args& a, hipStream_t stream);
// What the product's kernels take: rows of 8-bit operands whose copies, at a
// multiple of 16 bytes, stay below 2^23, and columns whose tiles end below 2^31.
constexpr int64_t kMaxByteRow = (int64_t{1} << 23) - 16;
constexpr int64_t kMaxProductCols = 0x7FFFFFFF - 256;

// The linear layer for one or two tokens in one kernel (scaled_rows.hip).
bool linear_rows_takes(int64_t m, int64_t n, int64_t k);
hipError_t launch_linear_rows(const rns8_mi355x_linear_i8_args& a, hipStream_t stream);

// ---- block norm (block_norm.hip) ------------------------------------------------------
constexpr int64_t kMaxNormCols = 32768;
hipError_t launch_block_norm(const rns8_mi355x_block_norm_args& a, hipStream_t stream);
uint64_t block_norm_backward_bytes(const rns8_mi355x_block_norm_backward_args& a);
hipError_t launch_block_norm_backward(const rns8_mi355x_block_norm_backward_args& a, hipStream_t stream);

// ---- token log-probabilities (logprobs.hip) ----------------------------------------------
constexpr uint32_t kMaxTop = 64;
uint64_t logprobs_bytes(const rns8_mi355x_logprobs_args& a);
hipError_t launch_logprobs(const rns8_mi355x_logprobs_args& a, hipStream_t stream);
hipError_t launch_logprobs_backward(const rns8_mi355x_logprobs_backward_args& a, hipStream_t stream);

}  // namespace rns8x
