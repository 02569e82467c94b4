// Copies of 8-bit operands whose rows the matrix kernels cannot read in place.
#pragma once

#include "elements.hpp"
#include "operators.hpp"

namespace rns8x {

// Four rows to a wave, 16 bytes of each to a lane at a time, all four loads in
// flight. The chunk that a row's end cuts comes from the row's last 16 bytes.
// Rows below 16 bytes: one to a thread. `block` of `blocks` workgroups of 256.
__device__ __forceinline__ void copy_rows(const OperandCopy& a, uint32_t block, uint32_t blocks) {
  if (a.cols < 16) {
    for (int64_t row = static_cast<int64_t>(block) * 256 + threadIdx.x; row < a.rows;
         row += static_cast<int64_t>(blocks) * 256) {
      uint32_t w[4] = {};
#pragma unroll 1
      for (int i = 0; i < a.cols; ++i) {
        const uint32_t b = static_cast<uint32_t>(static_cast<uint8_t>(a.src[row * a.lds + i])) << (8 * (i & 3));
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] |= (i >> 2) == k ? b : 0u;
      }
      __builtin_memcpy(a.dst + row * a.ldd, w, 16);
    }
    return;
  }
  const int lane = threadIdx.x & 63;
  const uint32_t cols = static_cast<uint32_t>(a.cols), padded = static_cast<uint32_t>(a.ldd);
  // units: (16 rows, 1024 bytes of each); a wave of the workgroup has four of the rows
  const uint32_t strips = (padded + 1023) / 1024;
  const int64_t units = (a.rows + 15) / 16 * strips;
  for (int64_t u = block; u < units; u += blocks) {
    const int64_t group = u / strips;
    const uint32_t c = 1024 * static_cast<uint32_t>(u - group * strips) + 16 * lane;
    const int64_t row = 16 * group + 4 * (threadIdx.x >> 6), rows = a.rows - row;
    if (rows <= 0 || c >= padded) continue;
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

}  // namespace rns8x
