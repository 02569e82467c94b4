// The gradients of the norms around a residual block (gfx950). With dH the whole
// gradient of h (block_norm.hip has the forward formulas):
//   dH = dh + r2 w_pre dy - h r2 r2 mean(w_pre dy h r2)
//   dresidual = residual_scale dH,  dgate = branch_scale f dH,  df = branch_scale gate dH
//   dx = r1 w_post df - x r1 r1 mean(w_post df x r1)
//   dw_pre = sum_rows dy h r2,  dw_post = sum_rows df x r1
// (h r2 and x r1 are near 1: r^3 leaves 32 bits for rows below 1e-13 and above 1e13)
//
// Bound by HBM: four rows are read into registers, cross one reduction for each
// norm and leave as two. The sums over rows take half of the registers, so the
// next row's loads are those of the CU's other workgroups (holding the next
// row beside this one left room for one workgroup of 512 to a CU: 8192 x 4096
// 114 us against 93). bf16, 8192 x 4096 76 us (335 MB: 4.4 TB/s) and 6 for the sums;
// f32, 1000 x 1101 with gates 14 and 4. Rows past 8192 spill (16384 f32 columns are
// 2 MB of row, weights and sums to a CU's 512 KB of registers).
#include <algorithm>

#include "block_norm.hpp"

namespace rns8x {
namespace {

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
  uint32_t stream_dx, stream_dresidual;  // stores pass the caches by
  float *part_post, *part_pre, *part_gate;  // [groups][cols], or NULL
};

template <typename T, int kThreads, int kVectors, bool kGates>
__global__ __launch_bounds__(row_block(kThreads)) void block_norm_backward_kernel(NormBackArgs a) {
  __shared__ uint32_t scratch[16];
  using Raw = RawRow<T, kVectors>;
  struct Rows {
    Raw x, res, dy, dh;
    RawRow<T, kGates ? kVectors : 1> gate;
  };
  float sum_post[kVectors][8] = {}, sum_pre[kVectors][8] = {}, sum_gate[kVectors][8] = {};
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  const int lane = row_is_shared(kThreads) ? threadIdx.x : threadIdx.x & 63;
  Weights<T, kVectors> w;
  load_weights<kThreads>(a, lane, w);
  auto load = [&](int64_t row, Rows& r) {
    load_row<kThreads>(static_cast<const T*>(a.x) + row * a.ldx, a.cols, lane, r.x);
    load_row_or<kThreads>(a.residual, row * a.ldresidual, a.cols, lane, 0.0f, r.res);
    if constexpr (kGates) load_row<kThreads>(static_cast<const T*>(a.gate) + row * a.ldgate, a.cols, lane, r.gate);
    load_row_or<kThreads>(a.dy, row * a.lddy, a.cols, lane, 0.0f, r.dy);
    load_row_or<kThreads>(a.dh, row * a.lddh, a.cols, lane, 0.0f, r.dh);
  };
  walk_rows<kThreads, false, Rows>(a.rows, load, [&](int64_t row, const Rows& r) {
    const float r1 = a.has_post ? a.rstd[row] : 1.0f;
    const float r2 = a.has_pre ? a.rstd[a.rows + row] : 0.0f;
    auto gate = [&](int j, int i) { return gate_at<kGates>(r, w, j, i); };
    float h[kVectors][8] = {};  // (without a norm of h nothing depends on it, also where it is infinite)
    float dot = 0.0f, k2 = 0.0f;
    if (a.has_pre) {
#pragma unroll
      for (int j = 0; j < kVectors; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = r.x.v[j].at(i) * r1 * w.post.v[j].at(i);
          const float dy = r.dy.v[j].at(i);
          h[j][i] = (a.keep * r.res.v[j].at(i) + a.branch * gate(j, i) * f) * r2;
          dot += w.pre.v[j].at(i) * dy * h[j][i];
          sum_pre[j][i] += dy * h[j][i];
        }
      k2 = r2 * (row_sum<kThreads>(dot, scratch) * inv_cols);
      dot = 0.0f;
    }
    // h, by r2 so far, becomes w_post df
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        h[j][i] = r.dh.v[j].at(i) +
                  r2 * (w.pre.v[j].at(i) * r.dy.v[j].at(i)) - h[j][i] * k2;
      if (a.dresidual) {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = a.keep * h[j][i];
        store_vector<kThreads, T, kVectors>(static_cast<T*>(a.dresidual) + row * a.lddresidual, a.cols, j, lane, out, a.stream_dresidual);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float xr = r.x.v[j].at(i) * r1, post = w.post.v[j].at(i);
        const float dgate = a.branch * (xr * post) * h[j][i];
        const float df = a.branch * gate(j, i) * h[j][i];
        out[i] = dgate;
        sum_gate[j][i] += dgate;
        sum_post[j][i] += df * xr;
        h[j][i] = post * df;
        dot += h[j][i] * xr;
      }
      if (a.dgate_rows)
        store_vector<kThreads, T, kVectors>(static_cast<T*>(a.dgate_rows) + row * a.lddgate, a.cols, j, lane, out, false);
    }
    if (!a.dx) return;
    if (a.has_post) {
      const float k1 = r1 * (row_sum<kThreads>(dot, scratch) * inv_cols);
#pragma unroll
      for (int j = 0; j < kVectors; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) h[j][i] = r1 * h[j][i] - r.x.v[j].at(i) * r1 * k1;
    }
#pragma unroll
    for (int j = 0; j < kVectors; ++j)
      store_vector<kThreads, T, kVectors>(static_cast<T*>(a.dx) + row * a.lddx, a.cols, j, lane, h[j], a.stream_dx);
  });
  const int64_t group = row_is_shared(kThreads) ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
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
struct BackwardShapes {
  static constexpr bool has(int threads, int vectors) {
    return threads < 512 ? vectors == 1 : threads == 512 ? vectors <= 2 : vectors >= 2;
  }
};

// Row groups of a backward launch: enough to fill the chip, few enough that their
// partial sums, written once and read once, stay small beside the rows, and all of
// equal length. Two rows to a group at least where that leaves enough of them: f32
// 1000 x 1101 17.5 us in 500 groups, 20.3 in 1000; bf16 2000 x 300 14.9 and 17.7; but
// 300 x 700 10.4 in 300, 11.9 in 256. Rows of more than one vector to a thread take a
// CU's registers: bf16 600 x 8000 28.4 in 256 groups, 34.5 in 512.
dim3 backward_grid(int64_t rows, RowShape shape) {
  const int threads = shape.threads;
  const int64_t most = shape.vectors > 1 ? 256 : threads <= 128 ? 2048 : threads == 256 ? 1024 : threads == 512 ? 512 : 256;
  const int64_t units = threads == 64 ? (rows + 3) / 4 : rows;
  const int64_t groups = std::min(units > 384 ? (units + 1) / 2 : units, threads == 64 ? most / 4 : most);
  const int64_t each = (units + groups - 1) / groups;
  return dim3(static_cast<unsigned>((units + each - 1) / each));
}
int64_t partial_rows(int64_t rows, RowShape shape) {
  const int64_t blocks = backward_grid(rows, shape).x;
  return shape.threads == 64 ? 4 * blocks : blocks;
}

}  // namespace

uint64_t block_norm_backward_bytes(const rns8_mi355x_block_norm_backward_args& g) {
  if (g.rows == 0) return 0;
  const int sums = (g.dpost_weight ? 1 : 0) + (g.dpre_weight ? 1 : 0) + (g.dgate && g.ldgate == 0 ? 1 : 0);
  const RowShape shape = backward_shape(g.cols);
  return round_up(static_cast<uint64_t>(sums) * static_cast<uint64_t>(partial_rows(g.rows, shape)) *
                      static_cast<uint64_t>(g.cols) * sizeof(float),
                  256);
}

hipError_t launch_block_norm_backward(const rns8_mi355x_block_norm_backward_args& g, hipStream_t stream) {
  if (g.cols > kMaxNormCols) return hipErrorInvalidValue;
  const RowShape shape = backward_shape(g.cols);
  const int64_t groups = g.rows > 0 ? partial_rows(g.rows, shape) : 0;
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
  const int64_t rows_moved = 1 + (g.residual ? 1 : 0) + (g.gate && g.ldgate != 0 ? 1 : 0) + (g.dy ? 1 : 0) +
                             (g.dh ? 1 : 0) + (g.dx ? 1 : 0) + (g.dresidual ? 1 : 0);
  const int64_t moved = rows_moved * g.rows * g.cols * (g.dtype == RNS8_MI355X_F32 ? 4 : 2);
  a.stream_dx = streams(moved, g.dx, g.lddx, g.dtype);
  a.stream_dresidual = streams(moved, g.dresidual, g.lddresidual, g.dtype);
  a.part_post = part_of(g.dpost_weight);
  a.part_pre = part_of(g.dpre_weight);
  a.part_gate = part_of(g.ldgate == 0 ? static_cast<float*>(g.dgate) : nullptr);
  if (g.rows > 0) {
    const hipError_t e = of_dtype(g.dtype, [&](auto t) {
      return with_row_shape<BackwardShapes>(shape, [&](auto threads, auto vectors) {
        constexpr int kThreads = decltype(threads)::value;
        const dim3 grid = backward_grid(g.rows, shape), block(row_block(kThreads));
        if (a.gate && a.ldgate != 0)
          hipLaunchKernelGGL((block_norm_backward_kernel<decltype(t), kThreads, decltype(vectors)::value, true>), grid,
                             block, 0, stream, a);
        else
          hipLaunchKernelGGL((block_norm_backward_kernel<decltype(t), kThreads, decltype(vectors)::value, false>), grid,
                             block, 0, stream, a);
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
