// How a kernel that keeps a row in registers spreads it over threads.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace rns8x {

// Threads per row (64: a wave, four rows to a workgroup; 128 to 1024: the
// workgroup) and 8-element vectors per thread (1, 2 or 4).
struct RowShape {
  int threads, vectors;
};
constexpr bool row_is_shared(int threads) { return threads > 64; }  // by the waves of a workgroup
constexpr int row_block(int threads) { return row_is_shared(threads) ? threads : 256; }

// The fewest threads that hold a row in `most` vectors each (more where 1024
// threads are not enough).
inline RowShape row_shape(int64_t cols, int most) {
  const int64_t vectors = (cols + 7) / 8;
  for (const int threads : {64, 128, 256, 512, 1024}) {
    const int64_t v = (vectors + threads - 1) / threads;
    if (v <= most || threads == 1024) return RowShape{threads, v <= 1 ? 1 : v <= 2 ? 2 : 4};
  }
  return RowShape{1024, 4};
}

// Two vectors of 16 bytes each where there are rows enough to fill the chip;
// one vector where they are few and a row's own latency is what counts.
inline RowShape choose_row_shape(int64_t rows, int64_t cols, int element_size) {
  return row_shape(cols, rows < 512 || element_size == 4 ? 1 : 2);
}

// The shapes that choose_row_shape gives for elements of this size.
template <int kElementSize>
struct ChosenShapes {
  static constexpr bool has(int threads, int vectors) {
    return vectors == 1 || threads == 1024 || (vectors == 2 && kElementSize < 4);
  }
};

// f(threads, vectors) with the shape, one that Shapes has, as compile-time constants.
template <typename Shapes, typename F>
hipError_t with_row_shape(RowShape s, F&& f) {
  auto vectors = [&](auto threads) {
    constexpr int kThreads = decltype(threads)::value;
    if constexpr (Shapes::has(kThreads, 1)) {
      if (s.vectors == 1) return f(threads, std::integral_constant<int, 1>{});
    }
    if constexpr (Shapes::has(kThreads, 2)) {
      if (s.vectors == 2) return f(threads, std::integral_constant<int, 2>{});
    }
    if constexpr (Shapes::has(kThreads, 4)) {
      if (s.vectors == 4) return f(threads, std::integral_constant<int, 4>{});
    }
    return hipErrorInvalidValue;
  };
  if (s.threads == 64) return vectors(std::integral_constant<int, 64>{});
  if (s.threads == 128) return vectors(std::integral_constant<int, 128>{});
  if (s.threads == 256) return vectors(std::integral_constant<int, 256>{});
  if (s.threads == 512) return vectors(std::integral_constant<int, 512>{});
  return vectors(std::integral_constant<int, 1024>{});
}

// A launch holds fewer than 2^32 threads; larger row counts are walked.
constexpr int64_t kMaxBlocks = int64_t{1} << 21;

inline dim3 row_grid(int threads, int64_t rows) {
  const int64_t blocks = row_is_shared(threads) ? rows : (rows + 3) / 4;
  return dim3(static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks));
}

// body(row, thread of the row) for this workgroup's (row_is_shared) or this
// wave's rows. Waves of a workgroup that own rows of their own may run
// different counts: such a body has no barrier.
template <int kThreads, typename F>
__device__ __forceinline__ void for_rows(int64_t rows, F&& body) {
  constexpr bool shared = row_is_shared(kThreads);
  const int lane = shared ? threadIdx.x : threadIdx.x & 63;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (shared ? 1 : 4);
  for (int64_t r = shared ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); r < rows; r += step)
    body(r, lane);
}

}  // namespace rns8x
