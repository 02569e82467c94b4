// Quantization of token rows and of gradient columns to 8 bits (gfx950).
//
//   amax = max |v|, scale = amax / 127, q = round_to_even(v * (127 / amax)),
// over rows (v = x * multiplier of the column) or over columns (v = x *
// multiplier of the row, q written transposed). Both are bound by HBM: rows
// are read once and stay in registers between the maximum and the bytes;
// columns are read twice (their maxima need every row), the second time mostly
// from the Infinity Cache. bf16, 4096 x 4096: rows 13.4 us (3.8 TB/s); rows and the
// columns' partials in one launch 22 us, the columns' tiles 20 us. A column of at
// most 512 rows is held whole: 500 x 701 f32, rows and columns in one launch, 8.4 us.
#include <algorithm>

#include "elements.hpp"
#include "operand_copy.hpp"
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
  uint32_t fragments;  // tiles of 16 rows: q in fragment order (operators.hpp); 0: in rows
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
      const uint32_t c = column_of<kThreads>(j, lane);
      if (c >= a.stop) continue;
      const uint64_t w = quantize8(v[j], s.inverse);
      if (a.fragments)
        *reinterpret_cast<uint64_t*>(a.q + fragment_offset(row, c, a.fragments)) = w;
      else
        store_bytes8(q, c, a.stop, w);
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
      const uint64_t w = quantize8(v, s.inverse);
      if (a.fragments)
        *reinterpret_cast<uint64_t*>(a.q + fragment_offset(row, c, a.fragments)) = w;
      else
        store_bytes8(q, c, a.stop, w);
    }
  }
}

template <typename T, int kThreads, int kVectors, bool kMul>
__global__ __launch_bounds__(row_block(kThreads)) void quantize_rows_kernel(RowsArgs a) {
  __shared__ uint32_t scratch[16];
  for_rows<kThreads>(a.rows, [&](int64_t row, int lane) {
    quantize_row<T, kThreads, kVectors, kMul>(a, row, lane, scratch);
  });
}

template <typename T, int kThreads, int kVectors>
hipError_t launch_rows(const RowsArgs& a, hipStream_t stream) {
  const dim3 grid = row_grid(kThreads, a.rows), block(row_block(kThreads));
  if (a.multiplier)
    hipLaunchKernelGGL((quantize_rows_kernel<T, kThreads, kVectors, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((quantize_rows_kernel<T, kThreads, kVectors, false>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_rows_of(const RowsArgs& a, hipStream_t stream) {
  if (a.cols > 32768) return launch_rows<T, 1024, 0>(a, stream);
  return with_row_shape<ChosenShapes<sizeof(T)>>(choose_row_shape(a.rows, a.cols, sizeof(T)), [&](auto threads, auto vectors) {
    return launch_rows<T, decltype(threads)::value, decltype(vectors)::value>(a, stream);
  });
}

// ---- columns ----------------------------------------------------------------------
// A first kernel leaves every column's largest magnitude (and sum) over each
// of `chunks` groups of rows; the second joins a column's chunks in their
// order, quantizes 128 x 128 tiles and turns them over in LDS.
constexpr int kTile = 128;
constexpr int kPitch = kTile / 4 + 1;  // words of four rows' bytes to a column of the turned tile

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
  int64_t tiles, tiles_c;
  int64_t first;  // the first tile of this launch
};

// Tiles or strips of columns to a launch: workgroups of 256 threads, with room for
// what else it does below 2^32 threads. More of them take more launches (walked in
// the kernels, they would cost every call registers: 8192 x 8192 75 us for 67).
constexpr int64_t kMaxUnits = int64_t{1} << 23;

// About 1024 workgroups of 256 columns, at least 16 rows each, and few enough
// that joining them is a small part of the second kernel: 4096 x 4096 26.8 us in 32
// chunks, 27.9 in 64; 16384 x 2048 44.7 and 41.3.
int64_t column_chunks(int64_t rows, int64_t cols) {
  const int64_t col_blocks = (cols + 255) / 256;
  return std::max<int64_t>(1, std::min({(1024 + col_blocks - 1) / col_blocks, (rows + 15) / 16, int64_t{rows > 8192 ? 64 : 32}}));
}

// Eight columns from column c on of four rows `step` apart and their factors,
// all loads issued before any is looked at: rows past the last and columns past
// the row read others in their place, which are then dropped.
template <typename T>
struct FourRows {
  Packed8<T> p[4];
  float m[4];
  __device__ __forceinline__ void load(const ColsArgs& a, int64_t row, int64_t step, int64_t last, int64_t c) {
    const T* const x = static_cast<const T*>(a.x);
    const int64_t cols = a.cols;
    if (cols >= 8) {
      const int64_t at = c + 8 <= cols ? c : c < cols ? cols - 8 : 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t r = min(row + k * step, last - 1);
        __builtin_memcpy(p[k].q, x + r * a.ldx + at, sizeof(p[k].q));
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t r = min(row + k * step, last - 1);
        T t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = c + i < cols ? x[r * a.ldx + c + i] : static_cast<T>(0.0f);
        __builtin_memcpy(p[k].q, t, sizeof(t));
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) m[k] = a.multiplier ? a.multiplier[min(row + k * step, last - 1)] : 1.0f;
  }
  __device__ __forceinline__ void settle(const ColsArgs& a, int64_t row, int64_t step, int64_t last, int64_t c) {
    if (a.cols >= 8 && a.cols % 8 != 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) p[k].drop(c < a.cols && c + 8 > a.cols ? static_cast<uint32_t>(c + 8 - a.cols) : 0u);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (row + k * step >= last || c >= a.cols) p[k].fill(static_cast<T>(0.0f));
  }
};

// 256 threads: 32 vectors of 8 columns by 8 rows, four rows in flight each.
template <typename T>
__device__ __forceinline__ void column_partials(const ColsArgs& a, int64_t strip, int64_t chunk) {
  __shared__ uint32_t amax_lds[8][256];
  __shared__ float sum_lds[8][256];
  const int vec = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const int64_t c = strip * 256 + 8 * vec;
  const int64_t first = chunk * a.chunk_rows;
  const int64_t last = first + a.chunk_rows < a.rows ? first + a.chunk_rows : a.rows;
  uint32_t amax[8] = {};
  float sum[8] = {};
  for (int64_t r = first + sub; r < last; r += 32) {
    FourRows<T> rows;
    rows.load(a, r, 8, last, c);
    rows.settle(a, r, 8, last, c);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = rows.p[k].at(i);
        sum[i] += v;
        // (a row that is not there: 0 times a factor that may be infinite counts as 0)
        const uint32_t b = r + 8 * k < last ? magnitude_bits(v * rows.m[k]) : 0u;
        amax[i] = amax[i] > b ? amax[i] : b;
      }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    amax_lds[sub][8 * vec + i] = amax[i];
    sum_lds[sub][8 * vec + i] = sum[i];
  }
  __syncthreads();
  const int64_t col = strip * 256 + threadIdx.x;
  if (col < a.cols) {
    uint32_t m = 0;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = amax_lds[j][threadIdx.x];
      m = m > b ? m : b;
      s += sum_lds[j][threadIdx.x];
    }
    a.amax_part[chunk * a.cols + col] = m;
    a.sum_part[chunk * a.cols + col] = s;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void quantize_columns_kernel(ColsArgs a) {
  __shared__ float inverse[kTile];
  __shared__ uint32_t tile[kTile * kPitch];  // [column][four rows]
  __shared__ uint32_t amax_lds[kTile];
  __shared__ float sum_lds[kTile];
  const int64_t unit = a.first + blockIdx.x, tile_r = unit / a.tiles_c;
  const int64_t c0 = (unit - tile_r * a.tiles_c) * kTile, r0 = tile_r * kTile;
  const int vec = threadIdx.x & 15, quad = threadIdx.x >> 4;  // 16 vectors of 8 columns by 16 groups of four rows
  const int64_t c = c0 + 8 * vec;
  // the whole tile is on its way while the columns' scales are joined
  FourRows<T> rows[2];
  if (a.rows > 0) {
    rows[0].load(a, r0 + 4 * quad, 1, a.rows, c);
    rows[1].load(a, r0 + 64 + 4 * quad, 1, a.rows, c);
  }
  {
    // two threads to a column, one for even and one for odd chunks, 16 (and as
    // many sums) in flight: chunks past the last are read again and not counted
    const int col = threadIdx.x & (kTile - 1), half = threadIdx.x / kTile;
    const int64_t column = c0 + col;
    const uint32_t* const amax_at = a.amax_part + min(column, a.cols - 1);
    const float* const sum_at = a.sum_part + min(column, a.cols - 1);
    const bool summed = a.sums && tile_r == 0;
    uint32_t amax = 0;
    float sum = 0.0f;
    for (int64_t k = half; k < a.chunks; k += 32) {
      uint32_t v[16];
      float s[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = amax_at[min(k + 2 * i, a.chunks - 1) * a.cols];
      if (summed) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = sum_at[min(k + 2 * i, a.chunks - 1) * a.cols];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = amax > v[i] ? amax : v[i];
      if (summed) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += k + 2 * i < a.chunks ? s[i] : 0.0f;
      }
    }
    if (half) {
      amax_lds[col] = amax;
      sum_lds[col] = sum;
    }
    __syncthreads();
    if (!half) {
      const uint32_t b = amax_lds[col];
      const RowScale s = row_scale(amax > b ? amax : b);
      inverse[col] = s.inverse;
      if (tile_r == 0 && column < a.cols) {
        a.scale[column] = s.scale;
        if (summed) a.sums[column] = sum + sum_lds[col];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int64_t row = r0 + 64 * half + 4 * quad;
    rows[half].settle(a, row, 1, a.rows, c);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float inv = inverse[8 * vec + i];
      uint32_t w = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w |= (row + k < a.rows ? quantize_byte(rows[half].p[k].at(i) * rows[half].m[k], inv) : 0u) << (8 * k);
      tile[(8 * vec + i) * kPitch + 16 * half + quad] = w;
    }
  }
  __syncthreads();
  // 16 bytes of a column to a thread: 8 threads to a column, 32 columns at a time
  const int part = threadIdx.x & 7;
#pragma unroll
  for (int group = 0; group < kTile / 32; ++group) {
    const int col = (threadIdx.x >> 3) + 32 * group;
    const int64_t column = c0 + col, r = r0 + 16 * part;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = tile[col * kPitch + 4 * part + k];
    if (column < a.cols && r < a.stop) {
      int8_t* const q = a.q + column * a.ldq;
      if (r + 16 <= a.stop) {
        __builtin_memcpy(q + r, w, 16);
      } else {
        for (int i = 0; r + i < a.stop; ++i) q[r + i] = static_cast<int8_t>(w[i >> 2] >> (8 * (i & 3)));
      }
    }
  }
}

// ---- columns that a workgroup holds whole ------------------------------------------------
// At most kWholeRows rows: 32 columns to a workgroup, 4 vectors of 8 columns by
// 64 groups of four rows, twice, all of them in registers between the maxima and
// the bytes. One pass, no partials and no kernel of its own.
constexpr int kWholeRows = 512, kWholeCols = 32;
constexpr int kWholePitch = kWholeRows / 4 + 1;  // words of a column in LDS

struct WholeLds {
  uint32_t amax[64][kWholeCols + 1];
  float sum[64][kWholeCols + 1];
  float inverse[kWholeCols];
};
constexpr int kWholeBytes =
    sizeof(WholeLds) > kWholeCols * kWholePitch * 4 ? sizeof(WholeLds) : kWholeCols * kWholePitch * 4;

template <typename T>
__device__ __forceinline__ void quantize_whole_columns(const ColsArgs& a, int64_t strip, uint8_t* lds) {
  WholeLds& part = *reinterpret_cast<WholeLds*>(lds);
  uint32_t* const bytes = reinterpret_cast<uint32_t*>(lds);  // [column][four rows], after the parts
  const int vec = threadIdx.x & 3, sub = threadIdx.x >> 2;
  const int64_t c0 = kWholeCols * strip, c = c0 + 8 * vec;
  FourRows<T> rows[2];
#pragma unroll
  for (int r = 0; r < 2; ++r)
    if (256 * r < a.rows) rows[r].load(a, 256 * r + 4 * sub, 1, a.rows, c);
  uint32_t amax[8] = {};
  float sum[8] = {};
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t row = 256 * r + 4 * sub;
    rows[r].settle(a, row, 1, a.rows, c);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = rows[r].p[k].at(i);
        sum[i] += v;
        const uint32_t b = row + k < a.rows ? magnitude_bits(v * rows[r].m[k]) : 0u;
        amax[i] = amax[i] > b ? amax[i] : b;
      }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    part.amax[sub][8 * vec + i] = amax[i];
    part.sum[sub][8 * vec + i] = sum[i];
  }
  __syncthreads();
  // eight threads to a column, eight of its parts each
  {
    const int col = threadIdx.x >> 3, eighth = threadIdx.x & 7;
    uint32_t top = 0;
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t b = part.amax[8 * k + eighth][col];
      top = top > b ? top : b;
      total += part.sum[8 * k + eighth][col];
    }
#pragma unroll
    for (int d = 1; d < 8; d *= 2) {
      const uint32_t b = __shfl_xor(top, d);
      top = top > b ? top : b;
      total += __shfl_xor(total, d);
    }
    const RowScale s = row_scale(top);
    if (eighth == 0) {
      part.inverse[col] = s.inverse;
      if (c0 + col < a.cols) {
        a.scale[c0 + col] = s.scale;
        if (a.sums) a.sums[c0 + col] = total;
      }
    }
  }
  __syncthreads();
  float inv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) inv[i] = part.inverse[8 * vec + i];
  __syncthreads();  // the bytes take the parts' place
#pragma unroll
  for (int r = 0; r < 2; ++r)
    if (256 * r < a.rows) {
      const int64_t row = 256 * r + 4 * sub;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t w = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w |= (row + k < a.rows ? quantize_byte(rows[r].p[k].at(i) * rows[r].m[k], inv[i]) : 0u) << (8 * k);
        bytes[(8 * vec + i) * kWholePitch + 64 * r + sub] = w;
      }
    }
  __syncthreads();
  // 16 bytes of a column at a time
  const uint32_t stop = static_cast<uint32_t>(a.stop), chunks = (stop + 15) / 16;
  for (uint32_t e = threadIdx.x; e < chunks * kWholeCols; e += 256) {
    const uint32_t col = e / chunks, r = 16 * (e - col * chunks);
    if (c0 + col >= a.cols) break;  // (columns rise with e)
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = bytes[col * kWholePitch + r / 4 + k];
    int8_t* const to = a.q + (c0 + col) * a.ldq + r;
    if (r + 16 <= stop) {
      __builtin_memcpy(to, w, 16);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i)
        if (r + i < stop) to[i] = static_cast<int8_t>(w[i >> 2] >> (8 * (i & 3)));
    }
  }
}

template <typename T>
hipError_t launch_columns_rest(ColsArgs a, hipStream_t stream) {
  for (; a.first < a.tiles; a.first += kMaxUnits) {
    const dim3 grid(static_cast<unsigned>(std::min(a.tiles - a.first, kMaxUnits)));
    hipLaunchKernelGGL((quantize_columns_kernel<T>), grid, dim3(256), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// ---- rows, columns and copies in one launch -------------------------------------------
// Workgroups of 256 threads in three ranges: rows to quantize; columns, 32 of
// them whole or (256 columns, rows of a chunk) for their partials; copies. They
// share nothing: one launch costs less than three, and small ones fill the chip
// together.
struct PrepareArgs {
  RowsArgs rows;
  ColsArgs cols;
  OperandCopy copies[4];
  uint32_t row_blocks, col_blocks, col_strips;
  uint32_t copy_blocks[4];
};

// kThreads (64 or 256) to a row, as quantize_row.
template <typename T, int kThreads, int kVectors, bool kMul, bool kWhole>
__global__ __launch_bounds__(256) void prepare_kernel(PrepareArgs a) {
  __shared__ uint32_t scratch[4];
  __shared__ __attribute__((aligned(16))) uint8_t lds[kWhole ? kWholeBytes : 16];
  uint32_t block = blockIdx.x;
  if (block < a.row_blocks) {
    const int lane = kThreads == 64 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t first = kThreads == 64 ? 4 * static_cast<int64_t>(block) + (threadIdx.x >> 6) : block;
    for (int64_t row = first; row < a.rows.rows; row += static_cast<int64_t>(a.row_blocks) * (256 / kThreads))
      quantize_row<T, kThreads, kVectors, kMul>(a.rows, row, lane, scratch);
    return;
  }
  block -= a.row_blocks;
  if (block < a.col_blocks) {
    if constexpr (kWhole)
      quantize_whole_columns<T>(a.cols, block, lds);
    else
      column_partials<T>(a.cols, block % a.col_strips, block / a.col_strips);
    return;
  }
  block -= a.col_blocks;
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    if (block < a.copy_blocks[i]) {
      copy_rows(a.copies[i], block, a.copy_blocks[i]);
      return;
    }
    block -= a.copy_blocks[i];
  }
}

bool whole_columns(int64_t rows) { return rows > 0 && rows <= kWholeRows; }

template <typename T, int kThreads, int kVectors, bool kWhole>
hipError_t launch_prepare_as(const PrepareArgs& a, uint32_t blocks, hipStream_t stream) {
  if (a.rows.multiplier)
    hipLaunchKernelGGL((prepare_kernel<T, kThreads, kVectors, true, kWhole>), dim3(blocks), dim3(256), 0, stream, a);
  else if constexpr (!kWhole || (kThreads == 64 && kVectors == 1))
    hipLaunchKernelGGL((prepare_kernel<T, kThreads, kVectors, false, kWhole>), dim3(blocks), dim3(256), 0, stream, a);
  else  // rows beside columns are a gradient's, and have a multiplier
    return hipErrorInvalidValue;
  return hipGetLastError();
}

template <typename T, bool kWhole>
hipError_t launch_prepare_of(const PrepareArgs& a, uint32_t blocks, hipStream_t stream) {
  const int64_t cols = a.rows.cols;
  if (cols <= 512) return launch_prepare_as<T, 64, 1, kWhole>(a, blocks, stream);
  if (cols <= 1024) return launch_prepare_as<T, 64, 2, kWhole>(a, blocks, stream);
  if (cols <= 2048) return launch_prepare_as<T, 256, 1, kWhole>(a, blocks, stream);
  if (cols <= 4096) return launch_prepare_as<T, 256, 2, kWhole>(a, blocks, stream);
  if (cols <= 8192) return launch_prepare_as<T, 256, 4, kWhole>(a, blocks, stream);
  return launch_prepare_as<T, 256, 0, kWhole>(a, blocks, stream);
}

RowsArgs rows_args(const rns8_mi355x_quantize_args& g) {
  return {g.x, g.rows, g.cols, g.ldx, g.multiplier, g.q, g.ldq, quantized_stop(g.cols, g.ldq), g.scale, 0};
}

ColsArgs cols_args(const rns8_mi355x_quantize_args& g) {
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
  a.tiles = std::max<int64_t>(1, (a.stop + kTile - 1) / kTile) * a.tiles_c;  // no rows: scales and sums alone
  return a;
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

hipError_t launch_quantize_rows(const rns8_mi355x_quantize_args& g, hipStream_t stream) {
  if (g.rows == 0) return hipSuccess;
  return of_dtype(g.dtype, [&](auto t) { return launch_rows_of<decltype(t)>(rows_args(g), stream); });
}

hipError_t launch_quantize_fragments(const rns8_mi355x_quantize_args& g, hipStream_t stream) {
  if (g.rows == 0) return hipSuccess;
  RowsArgs a = rows_args(g);
  a.fragments = static_cast<uint32_t>((g.rows + 15) / 16);
  a.stop = (g.cols + 63) / 64 * 64;
  return of_dtype(g.dtype, [&](auto t) { return launch_rows_of<decltype(t)>(a, stream); });
}

uint64_t quantize_columns_bytes(int64_t rows, int64_t cols) {
  return round_up(static_cast<uint64_t>(column_chunks(rows, cols)) * static_cast<uint64_t>(cols) * 8u, 256);
}

hipError_t launch_prepare(const rns8_mi355x_quantize_args* rows, const rns8_mi355x_quantize_args* columns,
                          const OperandCopy* copies, int copy_count, hipStream_t stream) {
  PrepareArgs a{};
  uint32_t dtype = RNS8_MI355X_F32;
  uint64_t blocks = 0;
  int64_t col_units = 0;
  if (rows && rows->rows > 0) {
    dtype = rows->dtype;
    a.rows = rows_args(*rows);
    const int64_t wanted = rows->cols <= 1024 ? (rows->rows + 3) / 4 : rows->rows;
    a.row_blocks = static_cast<uint32_t>(std::min(wanted, kMaxBlocks / 4));
    blocks += a.row_blocks;
  }
  if (columns) {
    dtype = columns->dtype;
    a.cols = cols_args(*columns);
    const bool whole = whole_columns(columns->rows);
    const int64_t width = whole ? kWholeCols : 256, chunks = whole ? 1 : a.cols.chunks;
    const int64_t strips = (columns->cols + width - 1) / width;
    // (columns below 2^31: at most 2^26 strips of whole columns, and 2^23 units of
    // partials, which a launch holds: more than 2^12 strips are of one chunk each)
    col_units = strips * chunks;
    a.col_strips = static_cast<uint32_t>(strips);
    a.col_blocks = static_cast<uint32_t>(std::min(col_units, kMaxUnits));
    blocks += a.col_blocks;
  }
  if (copy_count > 4) return hipErrorInvalidValue;
  for (int i = 0; i < copy_count; ++i) {
    a.copies[i] = copies[i];
    a.copy_blocks[i] = operand_copy_blocks(copies[i]);
    blocks += a.copy_blocks[i];
  }
  if (blocks == 0) return hipSuccess;
  return of_dtype(dtype, [&](auto t) {
    if (!columns || !whole_columns(columns->rows))
      return launch_prepare_of<decltype(t), false>(a, static_cast<uint32_t>(blocks), stream);
    hipError_t e = launch_prepare_of<decltype(t), true>(a, static_cast<uint32_t>(blocks), stream);
    // columns past the first launch's: matrices of their own
    a.row_blocks = 0;
    std::fill_n(a.copy_blocks, 4, 0u);
    while (e == hipSuccess && (col_units -= kMaxUnits) > 0) {
      constexpr int64_t kDone = kMaxUnits * kWholeCols;
      a.cols.x = static_cast<const decltype(t)*>(a.cols.x) + kDone;
      a.cols.cols -= kDone;
      a.cols.q += kDone * a.cols.ldq;
      a.cols.scale += kDone;
      if (a.cols.sums) a.cols.sums += kDone;
      a.col_blocks = static_cast<uint32_t>(std::min(col_units, kMaxUnits));
      e = launch_prepare_of<decltype(t), true>(a, a.col_blocks, stream);
    }
    return e;
  });
}

hipError_t launch_quantize_columns_rest(const rns8_mi355x_quantize_args& g, hipStream_t stream) {
  if (whole_columns(g.rows)) return hipSuccess;  // done by launch_prepare
  return of_dtype(g.dtype, [&](auto t) { return launch_columns_rest<decltype(t)>(cols_args(g), stream); });
}

hipError_t launch_quantize_columns(const rns8_mi355x_quantize_args& g, hipStream_t stream) {
  const hipError_t e = launch_prepare(nullptr, &g, nullptr, 0, stream);
  return e != hipSuccess ? e : launch_quantize_columns_rest(g, stream);
}

}  // namespace rns8x
