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

// Eight values of a row, or of a row that is the same everywhere.
template <typename T>
__device__ __forceinline__ void load_or(const void* base, int64_t at, int64_t n, float (&v)[8], float absent) {
  if (base) {
    load_upto8(static_cast<const T*>(base) + at, n, v, absent);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = absent;
  }
}

template <typename T, int kThreads, int kVectors>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads) void block_norm_kernel(NormArgs a) {
  __shared__ uint32_t scratch[16];
  for_rows<kThreads>(a.rows, [&](int64_t row, int lane) {
    float v[kVectors][8];  // x, then h
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      const int64_t c = 8 * (static_cast<int64_t>(j) * kThreads + lane);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = 0.0f;
      if (c < a.cols) load_upto8(static_cast<const T*>(a.x) + row * a.ldx + c, a.cols - c, v[j], 0.0f);
    }
    float r1 = 1.0f;
    if (a.has_post) {
#pragma unroll
      for (int j = 0; j < kVectors; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[j][i] * v[j][i];
      r1 = inverse_rms(row_sum<kThreads>(sum, scratch), a.cols, a.eps);
    }
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      const int64_t c = 8 * (static_cast<int64_t>(j) * kThreads + lane);
      if (c >= a.cols) continue;
      const int64_t n = a.cols - c;
      float w[8], g[8], res[8];
      load_or<T>(a.has_post ? a.post : nullptr, c, n, w, 1.0f);
      load_or<T>(a.gate, row * a.ldgate + c, n, g, 1.0f);
      load_or<T>(a.residual, row * a.ldresidual + c, n, res, 0.0f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // (columns past the row keep 0: x is 0 there, and so is the residual)
        const float f = v[j][i] * r1 * w[i];
        const float kept = a.residual ? a.keep * res[i] : 0.0f;
        v[j][i] = kept + a.branch * g[i] * f;
        sum += v[j][i] * v[j][i];
      }
      if (a.h) store_upto8(static_cast<T*>(a.h) + row * a.ldh + c, n, v[j]);
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
      const int64_t c = 8 * (static_cast<int64_t>(j) * kThreads + lane);
      if (c >= a.cols) continue;
      float w[8];
      load_or<T>(a.pre, c, a.cols - c, w, 1.0f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[j][i] = v[j][i] * r2 * w[i];
        // (a NaN row: columns past it hold 0 * NaN, in its scale already)
        const uint32_t m = magnitude_bits(v[j][i]);
        amax = amax > m ? amax : m;
      }
      if (a.y) store_upto8(static_cast<T*>(a.y) + row * a.ldy + c, a.cols - c, v[j]);
    }
    if (a.q) {
      const RowScale s = row_scale(row_reduce<kThreads>(amax, MaxU{}, scratch));
      if (lane == 0) a.q_scale[row] = s.scale;
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        const int64_t c = 8 * (static_cast<int64_t>(j) * kThreads + lane);
        if (c < a.stop) store_bytes8(a.q + row * a.ldq, c, a.stop, quantize8(v[j], s.inverse));
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
  float sum_post[kVectors][8] = {}, sum_pre[kVectors][8] = {}, sum_gate[kVectors][8] = {};
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  for_rows<kThreads>(a.rows, [&](int64_t row, int lane) {
    const float r1 = a.has_post ? a.rstd[row] : 1.0f;
    const float r2 = a.has_pre ? a.rstd[a.rows + row] : 0.0f;
    float x[kVectors][8], h[kVectors][8], wdy[kVectors][8];
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      const int64_t c = 8 * (static_cast<int64_t>(j) * kThreads + lane);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[j][i] = h[j][i] = wdy[j][i] = 0.0f;
      if (c >= a.cols) continue;
      const int64_t n = a.cols - c;
      float g[8], w[8], res[8], dy[8];
      load_upto8(static_cast<const T*>(a.x) + row * a.ldx + c, n, x[j], 0.0f);
      load_or<T>(a.residual, row * a.ldresidual + c, n, res, 0.0f);
      load_or<T>(a.gate, row * a.ldgate + c, n, g, 1.0f);
      load_or<T>(a.has_post ? a.post : nullptr, c, n, w, 1.0f);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        h[j][i] = (a.residual ? a.keep * res[i] : 0.0f) + a.branch * g[i] * (x[j][i] * r1 * w[i]);
      if (a.has_pre) {
        load_or<T>(a.dy, row * a.lddy + c, n, dy, 0.0f);
        load_or<T>(a.pre, c, n, w, 1.0f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          wdy[j][i] = w[i] * dy[i];
          dot += wdy[j][i] * h[j][i];
          sum_pre[j][i] += dy[i] * (h[j][i] * r2);
        }
      }
    }
    float k2 = 0.0f;
    if (a.has_pre) k2 = r2 * r2 * r2 * (row_sum<kThreads>(dot, scratch) * inv_cols);
    dot = 0.0f;
    // h becomes dH, wdy becomes w_post df
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      const int64_t c = 8 * (static_cast<int64_t>(j) * kThreads + lane);
      if (c >= a.cols) continue;
      const int64_t n = a.cols - c;
      float dh[8], g[8], w[8], out[8];
      load_or<T>(a.dh, row * a.lddh + c, n, dh, 0.0f);
      load_or<T>(a.gate, row * a.ldgate + c, n, g, 1.0f);
      load_or<T>(a.has_post ? a.post : nullptr, c, n, w, 1.0f);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[j][i] = dh[i] + r2 * wdy[j][i] - h[j][i] * k2;
      if (a.dresidual) {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = a.keep * h[j][i];
        store_upto8(static_cast<T*>(a.dresidual) + row * a.lddresidual + c, n, out);
      }
      if (a.dgate_rows || a.part_gate) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          out[i] = a.branch * (x[j][i] * r1 * w[i]) * h[j][i];
          sum_gate[j][i] += out[i];
        }
        if (a.dgate_rows) store_upto8(static_cast<T*>(a.dgate_rows) + row * a.lddgate + c, n, out);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float df = a.branch * g[i] * h[j][i];
        sum_post[j][i] += df * (x[j][i] * r1);
        wdy[j][i] = w[i] * df;
        dot += wdy[j][i] * x[j][i];
      }
    }
    if (!a.dx) return;
    float k1 = 0.0f;
    if (a.has_post) k1 = r1 * r1 * r1 * (row_sum<kThreads>(dot, scratch) * inv_cols);
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      const int64_t c = 8 * (static_cast<int64_t>(j) * kThreads + lane);
      if (c >= a.cols) continue;
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = r1 * wdy[j][i] - x[j][i] * k1;
      store_upto8(static_cast<T*>(a.dx) + row * a.lddx + c, a.cols - c, out);
    }
  });
  const bool shared = kThreads >= 256;
  const int lane = shared ? threadIdx.x : threadIdx.x & 63;
  const int64_t group = shared ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
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

// 64 columns of one sum to a workgroup: 16 groups at a time, then across.
__global__ __launch_bounds__(1024) void sum_groups_kernel(SumArgs a) {
  __shared__ float part[16][64];
  const float* const src = a.part[blockIdx.y];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + (threadIdx.x & 63);
  const int sub = threadIdx.x >> 6;
  float sum = 0.0f;
  if (c < a.cols)
    for (int64_t g = sub; g < a.groups; g += 16) sum += src[g * a.cols + c];
  part[sub][threadIdx.x & 63] = sum;
  __syncthreads();
  if (sub == 0 && c < a.cols) {
#pragma unroll
    for (int s = 1; s < 16; ++s) sum += part[s][threadIdx.x];
    a.out[blockIdx.y][c] = sum;
  }
}

// Row groups of a backward launch: enough to fill the chip, few enough that
// their partial sums stay small beside the rows.
int64_t backward_groups(int64_t rows, int threads) {
  const int64_t most = threads == 64 ? 1024 : threads == 256 ? 512 : 256;
  return rows < most ? rows : most;
}
dim3 backward_grid(int64_t rows, int threads) {
  const int64_t groups = backward_groups(rows, threads);
  return dim3(static_cast<unsigned>(threads == 64 ? (groups + 3) / 4 : groups));
}
// (whole workgroups: partial rows past the last group's are zero)
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
  const int threads = choose_row_shape(g.rows, g.cols).threads;
  return round_up(static_cast<uint64_t>(sums) * static_cast<uint64_t>(partial_rows(g.rows, threads)) *
                      static_cast<uint64_t>(g.cols) * sizeof(float),
                  256);
}

hipError_t launch_block_norm_backward(const rns8_mi355x_block_norm_backward_args& g, hipStream_t stream) {
  if (g.cols > kMaxNormCols) return hipErrorInvalidValue;
  const RowShape shape = choose_row_shape(g.rows, g.cols);
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
  hipLaunchKernelGGL(sum_groups_kernel, dim3(static_cast<unsigned>((g.cols + 63) / 64), count), dim3(1024), 0, stream,
                     sums);
  return hipGetLastError();
}

}  // namespace rns8x
