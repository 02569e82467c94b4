// Scales, bias and rounding of the scaled 8-bit product.
#pragma once

#include "elements.hpp"

namespace rns8x {

// A sum with its scales and bias, in 32 bits. Every kernel of the product ends in
// this, so a token's results do not depend on which of them its batch takes. (Left
// alone, the compiler joins the last step and the conversion to 16 bits in some
// kernels, which rounds once instead of twice.)
template <typename S>
__device__ __forceinline__ float scaled_value(S sum, float a_scale, float b_scale, float bias) {
  float v = fmaf(static_cast<float>(sum) * a_scale, b_scale, bias);
  asm("" : "+v"(v));  // (no instruction: the value as 32 bits hold it)
  return v;
}

// Four neighbouring outputs of a row (`n` of them inside it).
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t n, const float (&v)[4]) {
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = static_cast<T>(v[i]);
  if (n >= 4) {
    __builtin_memcpy(p, t, sizeof(t));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) p[i] = t[i];
}

// Four values of a vector of length n from i on; `absent` past its end or where there is none.
__device__ __forceinline__ void load4_or(const float* base, int64_t i, int64_t n, float absent, float (&v)[4]) {
  if (base && i + 4 <= n) {
    __builtin_memcpy(v, base + i, 16);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = base && i + e < n ? base[i + e] : absent;
}

}  // namespace rns8x
