// Internal interface of the scaled 8-bit product's kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "operators.hpp"

namespace rns8x {

// Operands as the kernels read them: 16-byte aligned rows at strides that are
// multiples of 16 below 2^23. `k` may end inside a 16-byte chunk: where b is n x
// k, a's or b's bytes from k to the chunk's end are zeros and the other's may hold
// anything.
struct ScaledGemm {
  int64_t m, n, k;
  const int8_t *a, *b;
  int64_t lda, ldb;
  bool inner;  // b is k x n
  const float *a_scale, *b_scale, *bias;
  void* out;
  int64_t ldo;
  uint32_t dtype;
  bool fragments = false;  // a in fragment order (launch_scaled_rows only)
};

// How the tile kernel splits a product: slices == 1 writes the output, more
// leave int32 partial sums [slices][m][ldp], which launch_scaled_tiles adds in a
// second launch.
struct TileShape {
  uint32_t bm, bn;  // the tile
  uint32_t slices;
  int64_t k_slice;  // a multiple of 128 where slices > 1
  int64_t ldp;
  uint64_t bytes;
  double cost;  // predicted us
};
TileShape choose_tile_shape(int64_t m, int64_t n, int64_t k);
// Shapes for two products with b stored k x n, and whether one launch takes both.
bool choose_pair_shapes(const int64_t (&m)[2], const int64_t (&n)[2], const int64_t (&k)[2], TileShape (&shapes)[2]);
// One product, or two of one tile with b stored k x n.
hipError_t launch_scaled_tiles(const ScaledGemm* g, const TileShape* shapes, int32_t* const* partials, int count,
                               hipStream_t stream);

// Few tokens (scaled_rows.hip): operands at any alignment, no workspace.
bool scaled_rows_takes(int64_t m, int64_t n, int64_t k, bool inner);
double scaled_rows_cost(int64_t m, int64_t n, int64_t k, bool fragments);  // predicted us
hipError_t launch_scaled_rows(const ScaledGemm& g, hipStream_t stream);

// What operands read once arrive at, for the predicted times: bytes per us.
constexpr double kBytesPerUs = 5.5e6;

// Products of at most this many bytes in one int32 sum: |a b| <= 2^14.
constexpr int64_t kExactK = 131071;

}  // namespace rns8x
