// Element types of the floating operands (float, half, bfloat16) and the
// reductions over a row that the operators' kernels share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace rns8x {

using f16 = _Float16;
using bf16 = __bf16;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float as_float(uint32_t x) { return __builtin_bit_cast(float, x); }
__device__ __forceinline__ uint32_t as_uint(float x) { return __builtin_bit_cast(uint32_t, x); }

// Eight consecutive elements, as floats. Rows may start at any element: the
// copy compiles to 16-byte loads that need no alignment (gfx9-family global
// memory instructions take any address).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  T t[8];
  __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(t[i]);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = static_cast<T>(v[i]);  // to nearest even
  __builtin_memcpy(p, t, sizeof(t));
}

// Past the caches, to a 16-byte aligned address.
template <typename T>
__device__ __forceinline__ void stream8(T* p, const float (&v)[8]) {
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = static_cast<T>(v[i]);
  u32x4 w[sizeof(t) / 16];
  __builtin_memcpy(w, t, sizeof(t));
#pragma unroll
  for (unsigned i = 0; i < sizeof(t) / 16; ++i) __builtin_nontemporal_store(w[i], reinterpret_cast<u32x4*>(p) + i);
}

// The first `n` (at most 8) of eight elements; the others read `other` and are not written.
template <typename T>
__device__ __forceinline__ void load_upto8(const T* p, int64_t n, float (&v)[8], float other) {
  if (n >= 8) {
    load8(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? static_cast<float>(p[i]) : other;
}

template <typename T>
__device__ __forceinline__ void store_upto8(T* p, int64_t n, const float (&v)[8]) {
  if (n >= 8) {
    store8(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = static_cast<T>(v[i]);
}

// ---- rows in registers -------------------------------------------------------------
// Eight consecutive elements as loaded.
template <typename T>
struct Packed8 {
  static constexpr int kWords = 2 * sizeof(T);
  u32x4 q[kWords / 4];
  __device__ __forceinline__ uint32_t word(int i) const { return q[i >> 2][i & 3]; }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) {
      return as_float(word(i));
    } else if constexpr (std::is_same_v<T, bf16>) {
      return as_float(i & 1 ? word(i >> 1) & 0xFFFF0000u : word(i >> 1) << 16);
    } else {
      return static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(word(i >> 1) >> (16 * (i & 1)))));
    }
  }
  __device__ __forceinline__ void fill(T v) {
    uint32_t w;
    if constexpr (sizeof(T) == 4)
      w = __builtin_bit_cast(uint32_t, v);
    else
      w = __builtin_bit_cast(uint16_t, v) * 0x10001u;
#pragma unroll
    for (auto& x : q) x = u32x4{w, w, w, w};
  }
  // Drops the first k (0 to 7) elements: the others move down, zeros follow.
  __device__ __forceinline__ void drop(uint32_t k) {
    uint32_t w[kWords + 4] = {};
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = word(i);
#pragma unroll
    for (int step = kWords / 2; step >= 1; step /= 2) {
      const bool on = k & (step * 4 / sizeof(T));
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = on ? (i + step < kWords ? w[i + step] : 0u) : w[i];
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = k & 1 ? w[i] >> 16 | w[i + 1] << 16 : w[i];
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) q[i >> 2][i & 3] = w[i];
  }
};

// Sixteen bytes without the first n (0 to 15), zeros after them.
__device__ __forceinline__ u32x4 drop_bytes(u32x4 w, uint32_t n) {
  const uint64_t lo = static_cast<uint64_t>(w[1]) << 32 | w[0], hi = static_cast<uint64_t>(w[3]) << 32 | w[2];
  const uint32_t bits = 8 * n & 63;
  const uint64_t a = n & 8 ? hi : lo, b = n & 8 ? 0 : hi;
  const uint64_t x = a >> bits | (b << 1) << (63 - bits), y = b >> bits;
  return u32x4{static_cast<uint32_t>(x), static_cast<uint32_t>(x >> 32), static_cast<uint32_t>(y),
               static_cast<uint32_t>(y >> 32)};
}

// kVectors vectors of 8 consecutive elements of a row for each of kThreads
// threads, vector j of thread t at column 8 (j kThreads + t), as loaded: all
// loads of a row (and of the rows beside it) are issued before the first
// conversion waits for one.
template <typename T, int kVectors>
struct RawRow {
  Packed8<T> v[kVectors];
};

template <int kThreads>
__device__ __forceinline__ uint32_t column_of(int vector, int lane) {
  return 8 * (static_cast<uint32_t>(vector) * kThreads + static_cast<uint32_t>(lane));
}

// Element `at` of a row below 2^32 bytes, as the row's (uniform) address and a 32-bit offset.
template <typename T>
__device__ __forceinline__ T* element(T* row, uint32_t at) {
  using Byte = std::conditional_t<std::is_const_v<T>, const char, char>;
  return reinterpret_cast<T*>(reinterpret_cast<Byte*>(row) + static_cast<uint32_t>(at * sizeof(T)));
}

// Elements past the row are zeros. One load to a vector: lanes past the row
// read its start, the lane that the row's end cuts reads the row's last eight
// and drops those that are others'. Rows below eight are read by elements.
template <int kThreads, typename T, int kVectors>
__device__ __forceinline__ void load_row(const T* row, uint32_t cols, int lane, RawRow<T, kVectors>& r) {
  if (cols < 8) {
#pragma unroll
    for (int j = 0; j < kVectors; ++j) r.v[j].fill(static_cast<T>(0.0f));
    if (lane == 0) {
      T t[8] = {};
      for (uint32_t i = 0; i < 8; ++i)
        if (i < cols) t[i] = row[i];
      __builtin_memcpy(r.v[0].q, t, sizeof(t));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kVectors; ++j) {
    const uint32_t c = column_of<kThreads>(j, lane);
    const uint32_t at = c + 8 <= cols ? c : c < cols ? cols - 8 : 0;
    __builtin_memcpy(r.v[j].q, element(row, at), sizeof(r.v[j].q));
  }
  if (cols == 8 * kThreads * kVectors) return;
#pragma unroll
  for (int j = 0; j < kVectors; ++j) {
    const uint32_t c = column_of<kThreads>(j, lane);
    if (cols % 8 != 0) r.v[j].drop(c < cols && c + 8 > cols ? c + 8 - cols : 0u);
    if (c >= cols) r.v[j].fill(static_cast<T>(0.0f));
  }
}

template <int kThreads, typename T, int kVectors>
__device__ __forceinline__ void store_vector(T* row, uint32_t cols, int vector, int lane, const float (&v)[8],
                                             bool streamed) {
  const uint32_t c = column_of<kThreads>(vector, lane);
  if (streamed && c + 8 <= cols)
    stream8(element(row, c), v);
  else if (c < cols)
    store_upto8(element(row, c), static_cast<int64_t>(cols - c), v);
}

// ---- reductions over a wave: every lane ends with the result --------------------
// Within each 16-lane row by rotations, then across rows by lane swaps.
template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_move(uint32_t x) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(x), kCtrl, 0xF, 0xF, false));
}
constexpr int kRowRotate = 0x120;

template <typename Op>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t x, Op op) {
  x = op(x, dpp_move<kRowRotate + 8>(x));
  x = op(x, dpp_move<kRowRotate + 4>(x));
  x = op(x, dpp_move<kRowRotate + 2>(x));
  x = op(x, dpp_move<kRowRotate + 1>(x));
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = op(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return op(b[0], b[1]);
}

struct AddF {
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const {
    return as_uint(as_float(a) + as_float(b));
  }
};
struct MaxU {
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};

// A reduction over the kThreads threads that share a row: a whole number of
// waves, all in one workgroup. `scratch` holds a word for each wave and is used
// by one reduction at a time; more than one wave means a barrier of the whole
// workgroup, so every thread of it takes part.
template <int kThreads, typename Op>
__device__ __forceinline__ uint32_t row_reduce(uint32_t x, Op op, uint32_t* scratch) {
  x = wave_reduce(x, op);
  if constexpr (kThreads > 64) {
    constexpr int kWaves = kThreads / 64;
    const int wave = static_cast<int>(threadIdx.x) >> 6;
    if ((threadIdx.x & 63u) == 0) scratch[wave] = x;
    __syncthreads();
    x = scratch[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) x = op(x, scratch[w]);
    __syncthreads();
  }
  return x;
}
template <int kThreads>
__device__ __forceinline__ float row_sum(float x, uint32_t* scratch) {
  return as_float(row_reduce<kThreads>(as_uint(x), AddF{}, scratch));
}

// ---- 8-bit quantization of a row ---------------------------------------------------
// |v| is compared as its bits, whose order is that of the values, infinity and
// then the NaNs above all: a row's largest says whether any value is not finite.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return as_uint(v) & 0x7FFFFFFFu; }

struct RowScale {
  float inverse;  // 127 / amax, or 0: every byte is zero
  float scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  const float amax = as_float(amax_bits);
  if (amax_bits >= 0x7F800000u) return {0.0f, __builtin_nanf("")};
  if (amax < 0x1p-100f) return {0.0f, 0.0f};
  return {127.0f / amax, amax / 127.0f};
}
__device__ __forceinline__ uint32_t quantize_byte(float v, float inverse) {
  return inverse == 0.0f ? 0u : static_cast<uint32_t>(static_cast<int>(__builtin_rintf(v * inverse))) & 0xFFu;
}
// Eight values as eight bytes.
__device__ __forceinline__ uint64_t quantize8(const float (&v)[8], float inverse) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i >> 2] |= quantize_byte(v[i], inverse) << (8 * (i & 3));
  return static_cast<uint64_t>(w[1]) << 32 | w[0];
}
// Bytes [c, c + 8) of a quantized row of `cols` values whose zeros run on to `stop`.
__device__ __forceinline__ void store_bytes8(int8_t* row, int64_t c, int64_t stop, uint64_t w) {
  if (c + 8 <= stop) {
    __builtin_memcpy(row + c, &w, 8);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < stop) row[c + i] = static_cast<int8_t>(w >> (8 * i));
}

// Where a quantized row's zeros end: min(ld, cols rounded up to 16).
inline int64_t quantized_stop(int64_t cols, int64_t ld) {
  const int64_t padded = (cols + 15) / 16 * 16;
  return padded < ld ? padded : ld;
}

}  // namespace rns8x
