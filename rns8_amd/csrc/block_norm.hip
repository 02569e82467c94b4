// The norms after and before a residual block, fused with gate, residual and
// scales (gfx950). For each row:
//   f = x r1 w_post, r1 = 1/sqrt(mean x^2 + eps)
//   h = residual_scale residual + branch_scale gate f
//   y = h r2 w_pre,  r2 = 1/sqrt(mean h^2 + eps)      (in dtype, or in 8 bits)
//
// Bound by HBM: a row is read once into registers, crosses one reduction for each
// norm (and one for its 8-bit form) and is written once, while the next row is on
// its way. The weights and a one-row gate stay in registers over a workgroup's rows.
// bf16, 8192 x 4096 50 us (268 MB: 5.3 TB/s); 8192 x 8192 with h and 8-bit rows 91 us
// (470 MB: 5.1 TB/s); one token of 4096 3.5 us. Rows past 16384 (four vectors to each
// of 1024 threads) keep more than a CU's registers hold, and spill.
#include <algorithm>

#include "block_norm.hpp"

namespace rns8x {
namespace {

struct NormArgs {
  const void *x, *residual, *gate, *post, *pre;
  int64_t rows, cols, ldx, ldresidual, ldgate;
  float eps, branch, keep;
  uint32_t has_post, has_pre;
  void *h, *y;
  int64_t ldh, ldy;
  int8_t* q;
  int64_t ldq, stop;
  float *q_scale, *rstd;
  uint32_t stream_h, stream_y;  // stores pass the caches by
};

__device__ __forceinline__ float inverse_rms(float sum_sq, int64_t cols, float eps) {
  return 1.0f / sqrtf(sum_sq / static_cast<float>(cols) + eps);
}

// kGates: a row of the gate for each token.
template <typename T, int kThreads, int kVectors, bool kGates>
__global__ __launch_bounds__(row_block(kThreads)) void block_norm_kernel(NormArgs a) {
  __shared__ uint32_t scratch[16];
  using Raw = RawRow<T, kVectors>;
  struct Rows {
    Raw x, res;
    RawRow<T, kGates ? kVectors : 1> gate;
  };
  const int lane = row_is_shared(kThreads) ? threadIdx.x : threadIdx.x & 63;
  Weights<T, kVectors> w;
  load_weights<kThreads>(a, lane, w);
  auto load = [&](int64_t row, Rows& r) {
    load_row<kThreads>(static_cast<const T*>(a.x) + row * a.ldx, a.cols, lane, r.x);
    load_row_or<kThreads>(a.residual, row * a.ldresidual, a.cols, lane, 0.0f, r.res);
    if constexpr (kGates) load_row<kThreads>(static_cast<const T*>(a.gate) + row * a.ldgate, a.cols, lane, r.gate);
  };
  walk_rows<kThreads, (kThreads < 1024), Rows>(a.rows, load, [&](int64_t row, const Rows& r) {
    float sum = 0.0f;
    float r1 = 1.0f;
    if (a.has_post) {
#pragma unroll
      for (int j = 0; j < kVectors; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += r.x.v[j].at(i) * r.x.v[j].at(i);
      r1 = inverse_rms(row_sum<kThreads>(sum, scratch), a.cols, a.eps);
    }
    float h[kVectors][8];
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // (columns past the row are 0: x and the residual are 0 there)
        const float f = r.x.v[j].at(i) * r1 * w.post.v[j].at(i);
        h[j][i] = a.keep * r.res.v[j].at(i) + a.branch * gate_at<kGates>(r, w, j, i) * f;
        sum += h[j][i] * h[j][i];
      }
      if (a.h) store_vector<kThreads, T, kVectors>(static_cast<T*>(a.h) + row * a.ldh, a.cols, j, lane, h[j], a.stream_h);
    }
    if (!a.has_pre) {
      if (a.rstd && lane == 0) a.rstd[row] = r1;
      return;
    }
    const float r2 = inverse_rms(row_sum<kThreads>(sum, scratch), a.cols, a.eps);
    if (a.rstd && lane == 0) {
      a.rstd[row] = r1;
      a.rstd[a.rows + row] = r2;
    }
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[j][i] = h[j][i] * r2 * w.pre.v[j].at(i);
        // (a NaN row: columns past it hold 0 * NaN, in its scale already)
        const uint32_t m = magnitude_bits(h[j][i]);
        amax = amax > m ? amax : m;
      }
      if (a.y) store_vector<kThreads, T, kVectors>(static_cast<T*>(a.y) + row * a.ldy, a.cols, j, lane, h[j], a.stream_y);
    }
    if (a.q) {
      const RowScale s = row_scale(row_reduce<kThreads>(amax, MaxU{}, scratch));
      if (lane == 0) a.q_scale[row] = s.scale;
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        const uint32_t c = column_of<kThreads>(j, lane);
        if (c < a.stop) store_bytes8(a.q + row * a.ldq, c, a.stop, quantize8(h[j], s.inverse));
      }
    }
  });
}

// As many workgroups as stay on the chip at once (by registers, 1536 threads to
// a CU with one vector each, 1024 with two): each walks its rows.
dim3 forward_grid(int threads, int vectors, int64_t rows) {
  const int64_t groups = threads == 64 ? (rows + 3) / 4 : rows;
  const int64_t per_cu = std::max(1, (vectors == 1 ? 1536 : 1024) / row_block(threads));
  return dim3(static_cast<unsigned>(std::min<int64_t>(groups, 256 * per_cu)));
}

}  // namespace

hipError_t launch_block_norm(const rns8_mi355x_block_norm_args& g, hipStream_t stream) {
  if (g.rows == 0) return hipSuccess;
  if (g.cols > kMaxNormCols) return hipErrorInvalidValue;
  NormArgs a{};
  a.x = g.x;
  a.residual = g.residual;
  a.gate = g.gate;
  a.post = g.post_weight;
  a.pre = g.pre_weight;
  a.rows = g.rows;
  a.cols = g.cols;
  a.ldx = g.ldx;
  a.ldresidual = g.ldresidual;
  a.ldgate = g.ldgate;
  a.eps = g.eps;
  a.branch = g.branch_scale;
  a.keep = g.residual_scale;
  a.has_post = g.flags & RNS8_MI355X_NORM_POST;
  a.has_pre = g.flags & RNS8_MI355X_NORM_PRE;
  a.h = g.h;
  a.ldh = g.ldh;
  a.y = g.y;
  a.ldy = g.ldy;
  a.q = g.q;
  a.ldq = g.ldq;
  a.stop = quantized_stop(g.cols, g.ldq);
  a.q_scale = g.q_scale;
  a.rstd = g.rstd;
  const int64_t rows_moved = 1 + (g.residual ? 1 : 0) + (g.gate && g.ldgate != 0 ? 1 : 0) + (g.h ? 1 : 0) + (g.y ? 1 : 0);
  const int64_t moved = rows_moved * g.rows * g.cols * (g.dtype == RNS8_MI355X_F32 ? 4 : 2);
  a.stream_h = streams(moved, g.h, g.ldh, g.dtype);
  a.stream_y = streams(moved, g.y, g.ldy, g.dtype);
  return of_dtype(g.dtype, [&](auto t) {
    return with_row_shape<ChosenShapes<sizeof(t)>>(choose_row_shape(g.rows, g.cols, sizeof(t)), [&](auto threads, auto vectors) {
      constexpr int kThreads = decltype(threads)::value;
      const dim3 grid = forward_grid(kThreads, decltype(vectors)::value, a.rows), block(row_block(kThreads));
      if (a.gate && a.ldgate != 0)
        hipLaunchKernelGGL((block_norm_kernel<decltype(t), kThreads, decltype(vectors)::value, true>), grid, block, 0,
                           stream, a);
      else
        hipLaunchKernelGGL((block_norm_kernel<decltype(t), kThreads, decltype(vectors)::value, false>), grid, block, 0,
                           stream, a);
      return hipGetLastError();
    });
  });
}

}  // namespace rns8x
