// Quantization of token rows and of gradient columns to 8 bits (gfx950).
//
//   amax = max |v|, scale = amax / 127, q = round_to_even(v * (127 / amax)),
// over rows (v = x * multiplier of the column) or over columns (v = x *
// multiplier of the row, q written transposed). Both are bound by HBM: rows
// are read once and stay in registers between the maximum and the bytes;
// columns are read twice (their maxima need every row), the second time mostly
// from the Infinity Cache.
#include "elements.hpp"
#include "operators.hpp"
#include "row_shape.hpp"

namespace rns8x {
namespace {

struct RowsArgs {
  const void* x;
  int64_t rows, cols, ldx;
  const float* multiplier;
  int8_t* q;
  int64_t ldq, stop;
  float* scale;
};

// kThreads threads hold a row in kVectors vectors each (0: the row is read
// again instead of held).
template <typename T, int kThreads, int kVectors, bool kMul>
__device__ __forceinline__ void quantize_row(const RowsArgs& a, int64_t row, int lane, uint32_t* scratch) {
  const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
  int8_t* const q = a.q + row * a.ldq;
  uint32_t amax = 0;
  auto take = [&](const float (&u)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t m = magnitude_bits(u[i]);
      amax = amax > m ? amax : m;
    }
  };
  if constexpr (kVectors > 0) {
    RawRow<T, kVectors> raw;
    RawRow<float, kVectors> mul;
    load_row<kThreads>(x, a.cols, lane, raw);
    if constexpr (kMul) load_row<kThreads>(a.multiplier, a.cols, lane, mul);
    float v[kVectors][8];
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[j][i] = raw.v[j].at(i);
        if constexpr (kMul) v[j][i] *= mul.v[j].at(i);
      }
      take(v[j]);
    }
    const RowScale s = row_scale(row_reduce<kThreads>(amax, MaxU{}, scratch));
    if (lane == 0) a.scale[row] = s.scale;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      const int64_t c = column_of<kThreads>(j, lane);
      if (c < a.stop) store_bytes8(q, c, a.stop, quantize8(v[j], s.inverse));
    }
  } else {
    auto load = [&](int64_t c, float (&v)[8]) {
      load_upto8(x + c, a.cols - c, v, 0.0f);
      if constexpr (kMul) {
        float m[8];
        load_upto8(a.multiplier + c, a.cols - c, m, 0.0f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= m[i];
      }
    };
    float v[8];
    for (int64_t c = 8 * lane; c < a.cols; c += 8 * kThreads) {
      load(c, v);
      take(v);
    }
    const RowScale s = row_scale(row_reduce<kThreads>(amax, MaxU{}, scratch));
    if (lane == 0) a.scale[row] = s.scale;
    for (int64_t c = 8 * lane; c < a.stop; c += 8 * kThreads) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
      if (c < a.cols) load(c, v);
      store_bytes8(q, c, a.stop, quantize8(v, s.inverse));
    }
  }
}

template <typename T, int kThreads, int kVectors, bool kMul>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads) void quantize_rows_kernel(RowsArgs a) {
  __shared__ uint32_t scratch[16];
  for_rows<kThreads>(a.rows, [&](int64_t row, int lane) {
    quantize_row<T, kThreads, kVectors, kMul>(a, row, lane, scratch);
  });
}

template <typename T, int kThreads, int kVectors>
hipError_t launch_rows(const RowsArgs& a, hipStream_t stream) {
  const dim3 grid = row_grid(kThreads, a.rows), block(kThreads < 256 ? 256 : kThreads);
  if (a.multiplier)
    hipLaunchKernelGGL((quantize_rows_kernel<T, kThreads, kVectors, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((quantize_rows_kernel<T, kThreads, kVectors, false>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_rows_of(const RowsArgs& a, hipStream_t stream) {
  if (a.cols > 32768) return launch_rows<T, 1024, 0>(a, stream);
  return with_row_shape(choose_row_shape(a.rows, a.cols), [&](auto threads, auto vectors) {
    return launch_rows<T, decltype(threads)::value, decltype(vectors)::value>(a, stream);
  });
}

// ---- columns ----------------------------------------------------------------------
// A first kernel leaves every column's largest magnitude (and sum) over each
// of `chunks` groups of rows; the second joins a column's chunks in their
// order, quantizes 64 x 64 tiles and turns them over in LDS.
constexpr int kTile = 64;
constexpr int64_t kMaxChunks = 64;

struct ColsArgs {
  const void* x;
  int64_t rows, cols, ldx;
  const float* multiplier;
  int8_t* q;
  int64_t ldq, stop;
  float* scale;
  float* sums;
  uint32_t* amax_part;  // [chunks][cols]
  float* sum_part;      // [chunks][cols]
  int64_t chunks, chunk_rows;
  int64_t tiles_c;
};

int64_t column_chunks(int64_t rows, int64_t cols) {
  const int64_t col_blocks = (cols + 255) / 256;
  int64_t chunks = (1024 + col_blocks - 1) / col_blocks;
  if (chunks > (rows + 15) / 16) chunks = (rows + 15) / 16;
  return chunks < 1 ? 1 : chunks > kMaxChunks ? kMaxChunks : chunks;
}

// 256 threads: 32 vectors of 8 columns by 8 rows at a time.
template <typename T>
__global__ __launch_bounds__(256) void column_partials_kernel(ColsArgs a) {
  __shared__ uint32_t amax_lds[8][256];
  __shared__ float sum_lds[8][256];
  const int vec = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + 8 * vec;
  const int64_t first = static_cast<int64_t>(blockIdx.y) * a.chunk_rows;
  const int64_t last = first + a.chunk_rows < a.rows ? first + a.chunk_rows : a.rows;
  uint32_t amax[8] = {};
  float sum[8] = {};
  if (c < a.cols) {
    for (int64_t r = first + sub; r < last; r += 8) {
      float v[8];
      load_upto8(static_cast<const T*>(a.x) + r * a.ldx + c, a.cols - c, v, 0.0f);
      const float m = a.multiplier ? a.multiplier[r] : 1.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum[i] += v[i];
        const uint32_t b = magnitude_bits(v[i] * m);
        amax[i] = amax[i] > b ? amax[i] : b;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    amax_lds[sub][8 * vec + i] = amax[i];
    sum_lds[sub][8 * vec + i] = sum[i];
  }
  __syncthreads();
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (col < a.cols) {
    uint32_t m = 0;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = amax_lds[j][threadIdx.x];
      m = m > b ? m : b;
      s += sum_lds[j][threadIdx.x];
    }
    a.amax_part[blockIdx.y * a.cols + col] = m;
    a.sum_part[blockIdx.y * a.cols + col] = s;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void quantize_columns_kernel(ColsArgs a) {
  __shared__ float inverse[kTile];
  __shared__ __attribute__((aligned(16))) uint8_t tile[kTile][kTile + 8];  // [column][row]
  const int64_t tile_r = blockIdx.x / a.tiles_c;
  const int64_t c0 = (blockIdx.x - tile_r * a.tiles_c) * kTile, r0 = tile_r * kTile;
  if (threadIdx.x < kTile) {
    const int64_t c = c0 + threadIdx.x;
    RowScale s{0.0f, 0.0f};
    if (c < a.cols) {
      uint32_t m = 0;
      for (int64_t k = 0; k < a.chunks; ++k) {
        const uint32_t b = a.amax_part[k * a.cols + c];
        m = m > b ? m : b;
      }
      s = row_scale(m);
      if (tile_r == 0) {
        a.scale[c] = s.scale;
        if (a.sums) {
          float sum = 0.0f;
          for (int64_t k = 0; k < a.chunks; ++k) sum += a.sum_part[k * a.cols + c];
          a.sums[c] = sum;
        }
      }
    }
    inverse[threadIdx.x] = s.inverse;
  }
  __syncthreads();
  // 8 vectors of 8 columns by 32 rows, twice
  const int vec = threadIdx.x & 7;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = (threadIdx.x >> 3) + 32 * half;
    const int64_t row = r0 + r, c = c0 + 8 * vec;
    float v[8] = {};
    if (row < a.rows && c < a.cols) {
      load_upto8(static_cast<const T*>(a.x) + row * a.ldx + c, a.cols - c, v, 0.0f);
      const float m = a.multiplier ? a.multiplier[row] : 1.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= m;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) tile[8 * vec + i][r] = static_cast<uint8_t>(quantize_byte(v[i], inverse[8 * vec + i]));
  }
  __syncthreads();
  const int vr = threadIdx.x & 7;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int c = (threadIdx.x >> 3) + 32 * half;
    const int64_t col = c0 + c, r = r0 + 8 * vr;
    uint64_t w;
    __builtin_memcpy(&w, &tile[c][8 * vr], 8);
    if (col < a.cols && r < a.stop) store_bytes8(a.q + col * a.ldq, r, a.stop, w);
  }
}

template <typename T>
hipError_t launch_columns_of(const ColsArgs& a, hipStream_t stream) {
  const int64_t col_blocks = (a.cols + 255) / 256;
  const int64_t tiles_r = a.stop > 0 ? (a.stop + kTile - 1) / kTile : 1;  // no rows: scales and sums alone
  if (tiles_r > kMaxBlocks / a.tiles_c) return hipErrorInvalidValue;
  const dim3 part(static_cast<unsigned>(col_blocks), static_cast<unsigned>(a.chunks));
  hipLaunchKernelGGL((column_partials_kernel<T>), part, dim3(256), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((quantize_columns_kernel<T>), dim3(static_cast<unsigned>(tiles_r * a.tiles_c)), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize_rows(const rns8_mi355x_quantize_args& g, hipStream_t stream) {
  if (g.rows == 0) return hipSuccess;
  const RowsArgs a{g.x, g.rows, g.cols, g.ldx, g.multiplier, g.q, g.ldq, quantized_stop(g.cols, g.ldq), g.scale};
  switch (g.dtype) {
    case RNS8_MI355X_F32: return launch_rows_of<float>(a, stream);
    case RNS8_MI355X_F16: return launch_rows_of<f16>(a, stream);
    case RNS8_MI355X_BF16: return launch_rows_of<bf16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

uint64_t quantize_columns_bytes(int64_t rows, int64_t cols) {
  return round_up(static_cast<uint64_t>(column_chunks(rows, cols)) * static_cast<uint64_t>(cols) * 8u, 256);
}

hipError_t launch_quantize_columns(const rns8_mi355x_quantize_args& g, hipStream_t stream) {
  ColsArgs a{};
  a.x = g.x;
  a.rows = g.rows;
  a.cols = g.cols;
  a.ldx = g.ldx;
  a.multiplier = g.multiplier;
  a.q = g.q;
  a.ldq = g.ldq;
  a.stop = quantized_stop(g.rows, g.ldq);
  a.scale = g.scale;
  a.sums = g.sums;
  a.chunks = column_chunks(g.rows, g.cols);
  a.chunk_rows = (g.rows + a.chunks - 1) / a.chunks;
  a.amax_part = static_cast<uint32_t*>(g.workspace);
  a.sum_part = reinterpret_cast<float*>(a.amax_part + a.chunks * a.cols);
  a.tiles_c = (g.cols + kTile - 1) / kTile;
  switch (g.dtype) {
    case RNS8_MI355X_F32: return launch_columns_of<float>(a, stream);
    case RNS8_MI355X_F16: return launch_columns_of<f16>(a, stream);
    case RNS8_MI355X_BF16: return launch_columns_of<bf16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace rns8x
