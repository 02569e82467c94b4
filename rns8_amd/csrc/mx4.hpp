// 4-bit microscaled ("MX4") matrices: their layout (include/rns8_mi355x.h), the
// rounding of a block, and the launchers of their operators.
//
// A unit is 16 rows x 256 columns: two fragments of 1 KB, each what a wave hands
// to v_mfma_scale_f32_16x16x128_f8f6f4 (lane L has the 16 bytes of block L / 16 of
// row L % 16), then 128 bytes with lane L's two scales next to each other, so
// that one 16-bit load serves both fragments and the instruction picks its byte.
// Fragments are read in whole lines, at any matrix size and without a swizzle; the
// 17 lines of a unit and its neighbours along a row are one stream in HBM.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "elements.hpp"
#include "rns8_mi355x.h"

namespace rns8x {

constexpr int kMx4Unit = RNS8_MI355X_MX4_UNIT, kMx4Scales = 2048;
constexpr int64_t kMaxMx4Size = 0x7FFFFFFF - 256;
constexpr int64_t kMaxMx4Sum = int64_t{1} << 23;

inline __host__ __device__ int64_t mx4_chunks(int64_t cols) { return (cols + 255) / 256; }
inline __host__ __device__ int64_t mx4_groups(int64_t rows) { return (rows + 15) / 16; }
// Bytes from 16 rows to the next 16.
inline __host__ __device__ int64_t mx4_stride(int64_t cols) { return mx4_chunks(cols) * kMx4Unit; }
inline uint64_t mx4_bytes(int64_t rows, int64_t cols) {
  return static_cast<uint64_t>(mx4_groups(rows)) * static_cast<uint64_t>(mx4_stride(cols));
}

// ---- rounding -----------------------------------------------------------------------
struct Mx4Scale {
  uint32_t code;  // the scale's byte
  float scale;    // the same as a float, as the conversions take it
  bool bad;       // the block has no finite scale: its codes are zeros
};
// Of a block whose largest magnitude has these bits (as a float): its exponent less
// two, at least 2^-127, which is below the normal floats.
__device__ __forceinline__ Mx4Scale mx4_scale(uint32_t amax_bits) {
  const uint32_t exponent = amax_bits & 0x7F800000u;
  const int32_t scale = max(static_cast<int32_t>(exponent) - 0x01000000, 0x00400000);
  const bool bad = exponent == 0x7F800000u;
  return {bad ? 255u : static_cast<uint32_t>(scale) >> 23, as_float(static_cast<uint32_t>(scale)), bad};
}

typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// Two values as codes into byte kByte of `word`.
template <int kByte>
__device__ __forceinline__ uint32_t mx4_codes(uint32_t word, float a, float b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, a, b, scale, kByte);
}
// Two neighbouring 16-bit values of type T.
template <int kByte, typename T>
__device__ __forceinline__ uint32_t mx4_codes(uint32_t word, uint32_t pair, float scale) {
  if constexpr (std::is_same_v<T, bf16>)
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, __builtin_bit_cast(bf16x2, pair), scale, kByte);
  else
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, __builtin_bit_cast(f16x2, pair), scale, kByte);
}

// Magnitudes as bits, whose order is the values', infinity and NaN above all:
// one to a word (float) or two (16-bit types).
template <typename T>
__device__ __forceinline__ uint32_t magnitudes(uint32_t word) {
  return word & (sizeof(T) == 4 ? 0x7FFFFFFFu : 0x7FFF7FFFu);
}
template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 4)
    return a > b ? a : b;
  else
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// A magnitude in the low bits of a word as a float's bits.
template <typename T>
__device__ __forceinline__ uint32_t float_bits(uint32_t magnitude) {
  if constexpr (sizeof(T) == 4)
    return magnitude;
  else if constexpr (std::is_same_v<T, bf16>)
    return magnitude << 16;
  else
    return as_uint(static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(magnitude))));
}

// ---- launchers ------------------------------------------------------------------------
// What a quantization reads and writes (mx4_quantize.hip). q: rows x cols, q_t: cols
// x rows, sums: of the columns for each 128 rows, [ceil(rows / 128)][cols]. Any may
// be NULL.
struct Mx4Quantize {
  const void* x;
  int64_t rows, cols, ldx;
  uint8_t *q, *q_t;
  float* sums;
};
// Up to two quantizations of one type in one launch.
hipError_t launch_quantize_mx4(const Mx4Quantize* jobs, int count, uint32_t dtype, hipStream_t stream);
// Partial sums [count][cols], added in a fixed order.
struct Mx4Sums {
  const float* partials;
  int64_t count, cols;
  float* out;  // or NULL: nothing to add
};
hipError_t launch_sum_partials(const Mx4Sums& s, hipStream_t stream);
hipError_t launch_dequantize_mx4(const rns8_mi355x_mx4_args& a, hipStream_t stream);
hipError_t launch_pack_mx4(const rns8_mi355x_pack_mx4_args& a, hipStream_t stream);

// Products (mx4_tiles.hip, which chooses between its tiles and mx4_rows.hip).
struct Mx4Gemm {
  int64_t m, n, k;
  const uint8_t *a, *b;
  const float* bias;
  void* out;
  int64_t ldo;
  uint32_t dtype;
  // the floating rows that `a` would be rounded from, where the kernel rounds them itself
  const void* x = nullptr;
  int64_t ldx = 0;
};
uint64_t gemm_mx4_bytes(int64_t m, int64_t n, int64_t k);
hipError_t launch_gemm_mx4(const Mx4Gemm& g, void* workspace, hipStream_t stream);

// Two products (empty ones among them) and partial sums to add up: in one launch where
// that is faster. Their workspaces are apart.
void gemm_mx4_pair_bytes(const Mx4Gemm (&g)[2], uint64_t (&bytes)[2]);
hipError_t launch_gemm_mx4_pair(const Mx4Gemm (&g)[2], void* const (&workspaces)[2], const Mx4Sums& sums, hipStream_t stream);

// How the tile kernel cuts a product.
struct Mx4Tiles {
  uint32_t bm, bn, slices;
  int64_t slice_chunks;
  int64_t ldp;
  uint64_t bytes;
  double cost;  // predicted us
};
Mx4Tiles choose_mx4_tiles(int64_t m, int64_t n, int64_t k);

// Few rows: m <= 64 (MX4), or m <= kMx4FusedRows of floating rows.
constexpr int64_t kMx4Rows = 64, kMx4FusedRows = 16;
// Whether a linear layer rounds its rows in the product's kernel.
bool linear_mx4_in_one_kernel(int64_t m, int64_t n);
hipError_t launch_mx4_rows(const Mx4Gemm& g, hipStream_t stream);

// ---- experts (mx4_experts.hip) ------------------------------------------------------------
constexpr int64_t kMaxExpertTokens = 64, kMaxExperts = 1024, kMaxExpertSize = 65536;
constexpr uint32_t kMaxExpertTop = 16;
uint64_t experts_mx4_bytes(const rns8_mi355x_experts_mx4_args& a);
hipError_t launch_experts_mx4(const rns8_mi355x_experts_mx4_args& a, hipStream_t stream);

}  // namespace rns8x
