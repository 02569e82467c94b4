// Rows, weights and the walk over rows that the block norm's kernels share.
#pragma once

#include "elements.hpp"
#include "operators.hpp"
#include "row_shape.hpp"

namespace rns8x {

// The same value everywhere where there is no row to load.
template <int kThreads, typename T, int kVectors>
__device__ __forceinline__ void load_row_or(const void* base, int64_t at, int64_t cols, int lane, float absent,
                                            RawRow<T, kVectors>& r) {
  if (base) {
    load_row<kThreads>(static_cast<const T*>(base) + at, cols, lane, r);
  } else {
#pragma unroll
    for (int j = 0; j < kVectors; ++j) r.v[j].fill(static_cast<T>(absent));
  }
}

// What a workgroup (or wave) keeps over its rows: the weights and a one-row gate.
template <typename T, int kVectors>
struct Weights {
  RawRow<T, kVectors> gate, post, pre;
};
template <int kThreads, typename T, int kVectors, typename A>
__device__ __forceinline__ void load_weights(const A& a, int lane, Weights<T, kVectors>& w) {
  load_row_or<kThreads>(a.ldgate == 0 ? a.gate : nullptr, 0, a.cols, lane, 1.0f, w.gate);
  load_row_or<kThreads>(a.has_post ? a.post : nullptr, 0, a.cols, lane, 1.0f, w.post);
  load_row_or<kThreads>(a.has_pre ? a.pre : nullptr, 0, a.cols, lane, 1.0f, w.pre);
}

template <bool kGates, typename Rows, typename W>
__device__ __forceinline__ float gate_at(const Rows& r, const W& w, int j, int i) {
  if constexpr (kGates) return r.gate.v[j].at(i);
  else return w.gate.v[j].at(i);
}

// body(row, its loaded rows) over this group's rows, the next row's loads in
// flight beside each body where the registers hold two rows. (Waves of a
// workgroup that own rows of their own may run different counts: no barrier is
// between them.)
template <int kThreads, bool kAhead, typename Rows, typename Load, typename Body>
__device__ __forceinline__ void walk_rows(int64_t rows, Load&& load, Body&& body) {
  constexpr bool shared = row_is_shared(kThreads);
  const int64_t group = shared ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (shared ? 1 : 4);
  Rows now;
  if constexpr (kAhead) {
    Rows next;
    if (group < rows) load(group, now);
    for (int64_t row = group; row < rows; row += step) {
      load(row + step < rows ? row + step : row, next);
      body(row, now);
      now = next;
    }
  } else {
    for (int64_t row = group; row < rows; row += step) {
      load(row, now);
      body(row, now);
    }
  }
}

// f(T{}) for the element type of `dtype`.
template <typename F>
hipError_t of_dtype(uint32_t dtype, F&& f) {
  switch (dtype) {
    case RNS8_MI355X_F32: return f(float{});
    case RNS8_MI355X_F16: return f(f16{});
    case RNS8_MI355X_BF16: return f(bf16{});
    default: return hipErrorInvalidValue;
  }
}

}  // namespace rns8x
