// The norms after and before a residual block, fused with gate, residual and
// scales, and their gradients (gfx950).
//
// Forward, for each row:
//   f = x r1 w_post, r1 = 1/sqrt(mean x^2 + eps)
//   h = residual_scale residual + branch_scale gate f
//   y = h r2 w_pre,  r2 = 1/sqrt(mean h^2 + eps)      (in dtype, or in 8 bits)
// Backward, with dH the whole gradient of h:
//   dH = dh + r2 w_pre dy - h r2^3 mean(w_pre dy h)
//   dresidual = residual_scale dH,  dgate = branch_scale f dH,  df = branch_scale gate dH
//   dx = r1 w_post df - x r1^3 mean(w_post df x)
//   dw_pre = sum_rows dy h r2,  dw_post = sum_rows df x r1
//
// Both are bound by HBM: each row is read once into registers, crosses one
// reduction for each norm, and is written once.
#include <algorithm>

#include "elements.hpp"
#include "operators.hpp"
#include "row_shape.hpp"

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
};

__device__ __forceinline__ float inverse_rms(float sum_sq, int64_t cols, float eps) {
  return 1.0f / sqrtf(sum_sq / static_cast<float>(cols) + eps);
}

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

template <typename T, int kThreads, int kVectors>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads) void block_norm_kernel(NormArgs a) {
  __shared__ uint32_t scratch[16];
  using Raw = RawRow<T, kVectors>;
  for_rows<kThreads>(a.rows, [&](int64_t row, int lane) {
    Raw x, res, gate, post, pre;
    load_row<kThreads>(static_cast<const T*>(a.x) + row * a.ldx, a.cols, lane, x);
    load_row_or<kThreads>(a.residual, row * a.ldresidual, a.cols, lane, 0.0f, res);
    load_row_or<kThreads>(a.gate, row * a.ldgate, a.cols, lane, 1.0f, gate);
    load_row_or<kThreads>(a.has_post ? a.post : nullptr, 0, a.cols, lane, 1.0f, post);
    float sum = 0.0f;
    float r1 = 1.0f;
    if (a.has_post) {
#pragma unroll
      for (int j = 0; j < kVectors; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = x.v[j].at(i);
          sum += v * v;
        }
      r1 = inverse_rms(row_sum<kThreads>(sum, scratch), a.cols, a.eps);
    }
    load_row_or<kThreads>(a.has_pre ? a.pre : nullptr, 0, a.cols, lane, 1.0f, pre);
    float h[kVectors][8];
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // (columns past the row are 0: x and the residual are 0 there)
        const float f = x.v[j].at(i) * r1 * post.v[j].at(i);
        h[j][i] = a.keep * res.v[j].at(i) + a.branch * gate.v[j].at(i) * f;
        sum += h[j][i] * h[j][i];
      }
      if (a.h) store_vector<kThreads, T, kVectors>(static_cast<T*>(a.h) + row * a.ldh, a.cols, j, lane, h[j]);
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
        h[j][i] = h[j][i] * r2 * pre.v[j].at(i);
        // (a NaN row: columns past it hold 0 * NaN, in its scale already)
        const uint32_t m = magnitude_bits(h[j][i]);
        amax = amax > m ? amax : m;
      }
      if (a.y) store_vector<kThreads, T, kVectors>(static_cast<T*>(a.y) + row * a.ldy, a.cols, j, lane, h[j]);
    }
    if (a.q) {
      const RowScale s = row_scale(row_reduce<kThreads>(amax, MaxU{}, scratch));
      if (lane == 0) a.q_scale[row] = s.scale;
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        const int64_t c = column_of<kThreads>(j, lane);
        if (c < a.stop) store_bytes8(a.q + row * a.ldq, c, a.stop, quantize8(h[j], s.inverse));
      }
    }
  });
}

// ---- backward -------------------------------------------------------------------------
// Sums over rows (the gradients of the weights and of a one-row gate) stay in
// registers over the rows that a row group walks and are then written as
// partial rows, which a second kernel adds in their order.
struct NormBackArgs {
  const void *x, *residual, *gate, *post, *pre, *dy, *dh;
  int64_t rows, cols, ldx, ldresidual, ldgate, lddy, lddh;
  float branch, keep;
  uint32_t has_post, has_pre;
  const float* rstd;
  void *dx, *dresidual, *dgate_rows;
  int64_t lddx, lddresidual, lddgate;
  float *part_post, *part_pre, *part_gate;  // [groups][cols], or NULL
};

template <typename T, int kThreads, int kVectors>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads) void block_norm_backward_kernel(NormBackArgs a) {
  __shared__ uint32_t scratch[16];
  using Raw = RawRow<T, kVectors>;
  struct Rows {
    Raw x, res, gate, dy, dh;
  };
  float sum_post[kVectors][8] = {}, sum_pre[kVectors][8] = {}, sum_gate[kVectors][8] = {};
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  auto load = [&](int64_t row, int lane, Rows& r) {
    load_row<kThreads>(static_cast<const T*>(a.x) + row * a.ldx, a.cols, lane, r.x);
    load_row_or<kThreads>(a.residual, row * a.ldresidual, a.cols, lane, 0.0f, r.res);
    load_row_or<kThreads>(a.gate, row * a.ldgate, a.cols, lane, 1.0f, r.gate);
    load_row_or<kThreads>(a.dy, row * a.lddy, a.cols, lane, 0.0f, r.dy);
    load_row_or<kThreads>(a.dh, row * a.lddh, a.cols, lane, 0.0f, r.dh);
  };
  auto work = [&](int64_t row, int lane, const Rows& r) {
    const float r1 = a.has_post ? a.rstd[row] : 1.0f;
    const float r2 = a.has_pre ? a.rstd[a.rows + row] : 0.0f;
    Raw post, pre;
    load_row_or<kThreads>(a.has_post ? a.post : nullptr, 0, a.cols, lane, 1.0f, post);
    load_row_or<kThreads>(a.has_pre ? a.pre : nullptr, 0, a.cols, lane, 1.0f, pre);
    float h[kVectors][8];
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < kVectors; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = r.x.v[j].at(i) * r1 * post.v[j].at(i);
        const float dy = r.dy.v[j].at(i);
        h[j][i] = a.keep * r.res.v[j].at(i) + a.branch * r.gate.v[j].at(i) * f;
        dot += pre.v[j].at(i) * dy * h[j][i];
        sum_pre[j][i] += dy * (h[j][i] * r2);
      }
    float k2 = 0.0f;
    if (a.has_pre) k2 = r2 * r2 * r2 * (row_sum<kThreads>(dot, scratch) * inv_cols);
    dot = 0.0f;
    // h becomes w_post df
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        h[j][i] = r.dh.v[j].at(i) +
                  r2 * (pre.v[j].at(i) * r.dy.v[j].at(i)) - h[j][i] * k2;
      if (a.dresidual) {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = a.keep * h[j][i];
        store_vector<kThreads, T, kVectors>(static_cast<T*>(a.dresidual) + row * a.lddresidual, a.cols, j, lane, out);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float xr = r.x.v[j].at(i) * r1, w = post.v[j].at(i);
        const float dgate = a.branch * (xr * w) * h[j][i];
        const float df = a.branch * r.gate.v[j].at(i) * h[j][i];
        out[i] = dgate;
        sum_gate[j][i] += dgate;
        sum_post[j][i] += df * xr;
        h[j][i] = w * df;
        dot += h[j][i] * r.x.v[j].at(i);
      }
      if (a.dgate_rows)
        store_vector<kThreads, T, kVectors>(static_cast<T*>(a.dgate_rows) + row * a.lddgate, a.cols, j, lane, out);
    }
    if (!a.dx) return;
    float k1 = 0.0f;
    if (a.has_post) k1 = r1 * r1 * r1 * (row_sum<kThreads>(dot, scratch) * inv_cols);
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = r1 * h[j][i] - r.x.v[j].at(i) * k1;
      store_vector<kThreads, T, kVectors>(static_cast<T*>(a.dx) + row * a.lddx, a.cols, j, lane, out);
    }
  };
  const bool shared = kThreads >= 256;
  const int lane = shared ? threadIdx.x : threadIdx.x & 63;
  const int64_t group = shared ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t step = static_cast<int64_t>(gridDim.x) * (shared ? 1 : 4);
  // the next row's loads are in flight while a row is worked on (waves of a
  // workgroup that own rows of their own may run different counts: no barrier
  // is between them)
  Rows now;
  if constexpr (kThreads < 1024) {
    Rows next;
    if (group < a.rows) load(group, lane, now);
    for (int64_t row = group; row < a.rows; row += step) {
      load(row + step < a.rows ? row + step : row, lane, next);
      work(row, lane, now);
      now = next;
    }
  } else {  // (no registers for two rows)
    for (int64_t row = group; row < a.rows; row += step) {
      load(row, lane, now);
      work(row, lane, now);
    }
  }
#pragma unroll
  for (int j = 0; j < kVectors; ++j) {
    const int64_t c = 8 * (static_cast<int64_t>(j) * kThreads + lane);
    if (c >= a.cols) continue;
    const int64_t at = group * a.cols + c, n = a.cols - c;
    if (a.part_post) store_upto8(a.part_post + at, n, sum_post[j]);
    if (a.part_pre) store_upto8(a.part_pre + at, n, sum_pre[j]);
    if (a.part_gate) store_upto8(a.part_gate + at, n, sum_gate[j]);
  }
}

struct SumArgs {
  const float* part[3];  // [groups][cols]
  float* out[3];
  int64_t groups, cols;
};

// 32 columns of one sum to a workgroup: 32 threads of consecutive columns for
// each of 32 groups at a time, four loads in flight, then across.
__global__ __launch_bounds__(1024) void sum_groups_kernel(SumArgs a) {
  __shared__ float part[32][33];
  const float* const src = a.part[blockIdx.y];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sum = 0.0f;
  if (c < a.cols) {
    int64_t g = sub;
    for (; g + 96 < a.groups; g += 128) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = src[(g + 32 * i) * a.cols + c];
      sum += (v[0] + v[1]) + (v[2] + v[3]);
    }
    for (; g < a.groups; g += 32) sum += src[g * a.cols + c];
  }
  part[sub][lane] = sum;
  __syncthreads();
  // row `sub` of the transposed tile: column `sub`'s 32 sums, one to a lane
  float v = part[lane][sub];
#pragma unroll
  for (int d = 1; d < 32; d *= 2) v += __shfl_xor(v, d, 32);
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + sub;
  if (lane == 0 && col < a.cols) a.out[blockIdx.y][col] = v;
}

// One vector per thread as far as that goes: sums and two rows stay in registers.
RowShape backward_shape(int64_t cols) { return row_shape(cols, cols <= 4096 ? 1 : 2); }

// Row groups of a backward launch: enough to fill the chip, few enough that
// their partial sums stay small beside the rows.
dim3 backward_grid(int64_t rows, int threads) {
  const int64_t most = threads <= 256 ? 1024 : threads == 512 ? 512 : 256;
  const int64_t groups = threads == 64 ? (rows + 3) / 4 : rows;
  return dim3(static_cast<unsigned>(std::min(groups, threads == 64 ? most / 2 : most)));
}
int64_t partial_rows(int64_t rows, int threads) {
  const int64_t blocks = backward_grid(rows, threads).x;
  return threads == 64 ? 4 * blocks : blocks;
}

template <typename F>
hipError_t of_dtype(uint32_t dtype, F&& f) {
  switch (dtype) {
    case RNS8_MI355X_F32: return f(float{});
    case RNS8_MI355X_F16: return f(f16{});
    case RNS8_MI355X_BF16: return f(bf16{});
    default: return hipErrorInvalidValue;
  }
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
  return of_dtype(g.dtype, [&](auto t) {
    return with_row_shape(choose_row_shape(g.rows, g.cols), [&](auto threads, auto vectors) {
      constexpr int kThreads = decltype(threads)::value;
      hipLaunchKernelGGL((block_norm_kernel<decltype(t), kThreads, decltype(vectors)::value>),
                         row_grid(kThreads, a.rows), dim3(kThreads < 256 ? 256 : kThreads), 0, stream, a);
      return hipGetLastError();
    });
  });
}

uint64_t block_norm_backward_bytes(const rns8_mi355x_block_norm_backward_args& g) {
  if (g.rows == 0) return 0;
  const int sums = (g.dpost_weight ? 1 : 0) + (g.dpre_weight ? 1 : 0) + (g.dgate && g.ldgate == 0 ? 1 : 0);
  const int threads = backward_shape(g.cols).threads;
  return round_up(static_cast<uint64_t>(sums) * static_cast<uint64_t>(partial_rows(g.rows, threads)) *
                      static_cast<uint64_t>(g.cols) * sizeof(float),
                  256);
}

hipError_t launch_block_norm_backward(const rns8_mi355x_block_norm_backward_args& g, hipStream_t stream) {
  if (g.cols > kMaxNormCols) return hipErrorInvalidValue;
  const RowShape shape = backward_shape(g.cols);
  const int64_t groups = g.rows > 0 ? partial_rows(g.rows, shape.threads) : 0;
  SumArgs sums{};
  unsigned count = 0;
  float* next = static_cast<float*>(g.workspace);
  auto part_of = [&](float* out) -> float* {
    if (!out) return nullptr;
    float* const part = next;
    sums.part[count] = part;
    sums.out[count++] = out;
    next += groups * g.cols;
    return part;
  };
  sums.groups = groups;
  sums.cols = g.cols;
  NormBackArgs a{};
  a.x = g.x;
  a.residual = g.residual;
  a.gate = g.gate;
  a.post = g.post_weight;
  a.pre = g.pre_weight;
  a.dy = g.dy;
  a.dh = g.dh;
  a.rows = g.rows;
  a.cols = g.cols;
  a.ldx = g.ldx;
  a.ldresidual = g.ldresidual;
  a.ldgate = g.ldgate;
  a.lddy = g.lddy;
  a.lddh = g.lddh;
  a.branch = g.branch_scale;
  a.keep = g.residual_scale;
  a.has_post = g.flags & RNS8_MI355X_NORM_POST;
  a.has_pre = g.flags & RNS8_MI355X_NORM_PRE;
  a.rstd = g.rstd;
  a.dx = g.dx;
  a.lddx = g.lddx;
  a.dresidual = g.dresidual;
  a.lddresidual = g.lddresidual;
  a.dgate_rows = g.ldgate != 0 ? g.dgate : nullptr;
  a.lddgate = g.lddgate;
  a.part_post = part_of(g.dpost_weight);
  a.part_pre = part_of(g.dpre_weight);
  a.part_gate = part_of(g.ldgate == 0 ? static_cast<float*>(g.dgate) : nullptr);
  if (g.rows > 0) {
    const hipError_t e = of_dtype(g.dtype, [&](auto t) {
      return with_row_shape(shape, [&](auto threads, auto vectors) {
        constexpr int kThreads = decltype(threads)::value;
        hipLaunchKernelGGL((block_norm_backward_kernel<decltype(t), kThreads, decltype(vectors)::value>),
                           backward_grid(g.rows, kThreads), dim3(kThreads < 256 ? 256 : kThreads), 0, stream, a);
        return hipGetLastError();
      });
    });
    if (e != hipSuccess) return e;
  }
  if (count == 0) return hipSuccess;
  hipLaunchKernelGGL(sum_groups_kernel, dim3(static_cast<unsigned>((g.cols + 31) / 32), count), dim3(1024), 0, stream,
                     sums);
  return hipGetLastError();
}

}  // namespace rns8x
