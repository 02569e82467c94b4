// The scaled MFMA on MX4 fragments, the rounding of a lane's own block, and the sum of
// partial sums.
#pragma once

#include "elements.hpp"
#include "mx4.hpp"

namespace rns8x {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// What a lane has of a unit: a block of each fragment, and their scales (low byte
// the first's).
struct Mx4Unit {
  i32x4 codes[2];
  uint32_t scales;
};

__device__ __forceinline__ Mx4Unit load_unit(const uint8_t* unit, int lane) {
  Mx4Unit u;
  u.codes[0] = *reinterpret_cast<const i32x4*>(unit + 16 * lane);
  u.codes[1] = *reinterpret_cast<const i32x4*>(unit + 1024 + 16 * lane);
  u.scales = *reinterpret_cast<const uint16_t*>(unit + kMx4Scales + 2 * lane);
  return u;
}

// The same past the caches: for what is read once (a plain read of 1 GB of units runs
// at 6.2 TB/s, this one at 7.1).
__device__ __forceinline__ Mx4Unit stream_unit(const uint8_t* unit, int lane) {
  Mx4Unit u;
  u.codes[0] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(unit + 16 * lane));
  u.codes[1] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(unit + 1024 + 16 * lane));
  u.scales = __builtin_nontemporal_load(reinterpret_cast<const uint16_t*>(unit + kMx4Scales + 2 * lane));
  return u;
}

// acc[row of b][row of a] += sum over 128 columns; kByteB, kByteA: which bytes of the
// scales are this fragment's. Lane L then has rows 4 (L / 16) + e of b and row L % 16
// of a.
template <int kByteB, int kByteA>
__device__ __forceinline__ f32x4 mx4_mfma(i32x4 b, i32x4 a, f32x4 acc, uint32_t b_scales, uint32_t a_scales) {
  const i32x8 b8 = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 a8 = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  constexpr int kFp4 = 4;
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b8, a8, acc, kFp4, kFp4, kByteB, static_cast<int>(b_scales),
                                                          kByteA, static_cast<int>(a_scales));
}
// Both fragments of a unit.
__device__ __forceinline__ f32x4 mx4_mfma(const Mx4Unit& b, const Mx4Unit& a, f32x4 acc) {
  acc = mx4_mfma<0, 0>(b.codes[0], a.codes[0], acc, b.scales, a.scales);
  return mx4_mfma<1, 1>(b.codes[1], a.codes[1], acc, b.scales, a.scales);
}

// Adds up partial sums: sixteen columns to a wave, a quarter of the partials to each
// sixteen lanes; their order is the same whatever the grid.
__device__ __forceinline__ void add_partials(const Mx4Sums& s, uint32_t wave, uint32_t waves, int lane) {
  const int g = lane >> 4;
  for (int64_t c0 = static_cast<int64_t>(wave) * 16; c0 < s.cols; c0 += static_cast<int64_t>(waves) * 16) {
    const int64_t c = min(c0 + (lane & 15), s.cols - 1);
    float sum = 0.0f;
    for (int64_t i = g; i < s.count; i += 32) {
      float v[8];  // eight loads in flight
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = s.partials[min(i + 4 * j, s.count - 1) * s.cols + c];
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += i + 4 * j < s.count ? v[j] : 0.0f;
    }
    const auto a = __builtin_amdgcn_permlane16_swap(as_uint(sum), as_uint(sum), false, false);
    sum = as_float(a[0]) + as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(as_uint(sum), as_uint(sum), false, false);
    sum = as_float(b[0]) + as_float(b[1]);
    if (lane < 16 && c0 + lane < s.cols) s.out[c0 + lane] = sum;
  }
}

struct Mx4Block {
  i32x4 codes;
  uint32_t scale;
};

// A block's values as loaded.
template <typename T>
struct RawBlock {
  static constexpr int kWords = 8 * sizeof(T);
  uint32_t raw[kWords];
};

// Columns [c, c + 32) of a row of k values: all there, or zeros past its end.
template <typename T>
__device__ __forceinline__ void load_block(const T* row, uint32_t c, RawBlock<T>& b) {
  __builtin_memcpy(b.raw, row + c, sizeof(b.raw));
}
template <typename T>
__device__ __forceinline__ void load_cut_block(const T* row, uint32_t c, uint32_t k, RawBlock<T>& b) {
#pragma unroll
  for (uint32_t i = 0; i < 32; i += 8) {
    T t[8] = {};
    if (c + i + 8 <= k) {
      __builtin_memcpy(t, row + c + i, sizeof(t));
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e)
        if (c + i + e < k) t[e] = row[c + i + e];
    }
    __builtin_memcpy(b.raw + i * sizeof(T) / 4, t, sizeof(t));
  }
}

template <typename T>
__device__ __forceinline__ Mx4Block round_block(const RawBlock<T>& b) {
  constexpr int kWords = RawBlock<T>::kWords;
  const uint32_t (&raw)[kWords] = b.raw;
  uint32_t m = 0;
#pragma unroll
  for (int w = 0; w < kWords; ++w) m = larger<T>(m, magnitudes<T>(raw[w]));
  if constexpr (sizeof(T) == 2) m = larger<T>(m, m >> 16) & 0xFFFFu;
  const Mx4Scale s = mx4_scale(float_bits<T>(m));
  Mx4Block out;
  out.scale = s.code;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t codes = 0;
    auto pair = [&](auto byte) {
      constexpr int b = decltype(byte)::value;
      if constexpr (sizeof(T) == 4)
        codes = mx4_codes<b>(codes, as_float(raw[8 * q + 2 * b]), as_float(raw[8 * q + 2 * b + 1]), s.scale);
      else
        codes = mx4_codes<b, T>(codes, raw[4 * q + b], s.scale);
    };
    pair(std::integral_constant<int, 0>{});
    pair(std::integral_constant<int, 1>{});
    pair(std::integral_constant<int, 2>{});
    pair(std::integral_constant<int, 3>{});
    out.codes[q] = s.bad ? 0 : static_cast<int>(codes);
  }
  return out;
}

}  // namespace rns8x
