// Rounding of floating rows to MX4 and back (gfx950). Bound by HBM: a value is
// read once and leaves as 0.53 bytes for each form.
//
//   * A lane holds 16 bytes (V = 4 or 8 columns) of each of its rows as loaded;
//     sixteen lanes a row's 64 or 128 columns, so loads are whole lines. A vector that
//     the row's end cuts is the row's last 16 bytes, moved down: no lane waits for single
//     elements (which took 15 us for a matrix of 1000 x 1101).
//   * q (blocks along a row): a block is 4 or 8 neighbouring lanes, its largest
//     magnitude two or three lane moves after the lane's own (as integers: two
//     16-bit values at a time); v_cvt_scalef32_pk_fp4_* divides by the power of two
//     and rounds two values, half to even, 6 at most.
//   * q_t (blocks along a column): a lane's 32 rows are a block of each of its V
//     columns, so both forms come from one read.
//   * Codes and scales are gathered in LDS as units and leave in whole lines. (A tile of
//     both forms has one fragment of q_t's units: its scales are every other byte of
//     lines that two workgroups share, and leave as bytes.)
//   * Sums of columns (a bias' gradient) in 32 bits for each 128 rows, in a fixed
//     order; a second kernel adds those.
// Measured at 8192 x 8192 in bf16: rows alone 33 us (5.1 TB/s), both forms 54 (3.8 TB/s),
// back to bf16 29 (5.9 TB/s).
#include <algorithm>
#include <type_traits>

#include "mx4.hpp"
#include "mx4_mfma.hpp"
#include "operators.hpp"
#include "row_shape.hpp"
#include "tables.hpp"

namespace rns8x {
namespace {

struct Jobs {
  Mx4Quantize job[2];
  uint32_t tiles[2];
  DivU31 chunks[2];  // of a row
  // both forms of a tile by workgroups of their own, which read it twice: where a SIMD
  // would have one wave or none (1024 x 1024 in bf16 9.2 us together, 6.2 apart)
  uint32_t apart;
};

__device__ __forceinline__ uint32_t div_u31(uint32_t n, DivU31 v) { return __umulhi(n << 1, v.mul) >> v.shift; }

constexpr int kQuadSwap1 = 0xB1, kQuadSwap2 = 0x4E, kHalfMirror = 0x141;  // DPP controls

// A workgroup's tile is 256 columns wide; kRows rows to a lane, of which a wave has
// four times as many. kTransposed: the tile is 128 rows high, a fragment of q_t's units.
template <typename T, bool kTransposed>
struct Shape {
  static constexpr int V = 16 / sizeof(T);
  static constexpr int kAcross = 16 / V;
  static constexpr int kRows = kTransposed ? 32 : 8;
  static constexpr int kDown = kTransposed ? 1 : 4 / kAcross;
  static constexpr int kThreads = 64 * kAcross * kDown;
  static constexpr int kHigh = 4 * kRows * kDown;
};

// A unit in LDS: its fragments with room after every block of 16 rows, then the
// scales, and room again, so that neither form's writes meet in a bank.
constexpr int kLdsFragment = 16 * 17 * 4, kLdsScales = 2 * kLdsFragment, kLdsUnit = kLdsScales + 128 + 32;
__device__ __forceinline__ int lds_place(int fragment, int block, int row) {
  return kLdsFragment * fragment + 16 * (17 * block + row);
}

// `count` units from LDS, `stride` bytes apart in memory.
template <int kThreads>
__device__ __forceinline__ void store_units(const uint8_t* lds, int64_t count, uint8_t* to, int64_t stride) {
  for (uint32_t i = threadIdx.x; i < 136 * count; i += kThreads) {
    const uint32_t unit = i / 136, v = i - 136 * unit;
    const uint32_t at = v < 128 ? lds_place(v / 64, v % 64 / 16, v % 16) : kLdsScales + 16 * (v - 128);
    *reinterpret_cast<u32x4*>(to + unit * stride + 16 * v) = *reinterpret_cast<const u32x4*>(lds + kLdsUnit * unit + at);
  }
}

// Fragment `fragment` of 16 units of q_t: the codes, then the scales, every other byte.
constexpr int kLdsColumns = kLdsFragment + 64 + 16;
template <int kThreads>
__device__ __forceinline__ void store_fragments(const uint8_t* lds, int64_t count, int fragment, uint8_t* to, int64_t stride) {
  for (uint32_t i = threadIdx.x; i < 64 * count; i += kThreads) {
    const uint32_t unit = i / 64, place = i % 64;
    *reinterpret_cast<u32x4*>(to + unit * stride + 1024 * fragment + 16 * place) =
        *reinterpret_cast<const u32x4*>(lds + kLdsColumns * unit + lds_place(0, place / 16, place % 16));
    to[unit * stride + kMx4Scales + 2 * place + fragment] = lds[kLdsColumns * unit + kLdsFragment + place];
  }
}

template <typename T, bool kTransposed>
__global__ __launch_bounds__((Shape<T, kTransposed>::kThreads)) void quantize_mx4_kernel(Jobs jobs) {
  using S = Shape<T, kTransposed>;
  constexpr int V = S::V, R = S::kRows;
  __shared__ __attribute__((aligned(16))) uint8_t row_units[S::kHigh / 16 * kLdsUnit];
  __shared__ __attribute__((aligned(16))) uint8_t column_units[kTransposed ? 16 * kLdsColumns : 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cl = lane & 15, g = lane >> 4;
  const int across = wave % S::kAcross, down = wave / S::kAcross;
  for (uint32_t turn = blockIdx.x; turn < (jobs.tiles[0] + jobs.tiles[1]) << jobs.apart; turn += gridDim.x) {
    const uint32_t tile = turn >> jobs.apart;
    const bool rows_here = !jobs.apart || (turn & 1) == 0, columns_here = !jobs.apart || (turn & 1) == 1;
    const bool second = tile >= jobs.tiles[0];
    const Mx4Quantize& job = jobs.job[second ? 1 : 0];
    const DivU31 chunks_of = jobs.chunks[second ? 1 : 0];
    const uint32_t at = second ? tile - jobs.tiles[0] : tile;
    const uint32_t tile_row = div_u31(at, chunks_of), chunk = at - tile_row * chunks_of.d;
    const int64_t chunks = chunks_of.d, rows = job.rows, cols = job.cols;
    const int wave_row = down * (4 * R), wave_col = across * (16 * V);
    const int64_t tile_r0 = static_cast<int64_t>(tile_row) * S::kHigh, wave_r0 = tile_r0 + wave_row;
    const int64_t wave_c0 = static_cast<int64_t>(chunk) * 256 + wave_col, c0 = wave_c0 + V * cl;
    // row i of this lane is row_of(i) of the tile: 32 neighbours, or every fourth row (a
    // wave's four are then 64 bytes of a fragment)
    constexpr int kRowStep = kTransposed ? 1 : 4;
    auto row_of = [&](int i) { return wave_row + (kTransposed ? g * R : g) + kRowStep * i; };
    const T* const x = static_cast<const T*>(job.x);
    const int64_t step = kRowStep * job.ldx;
    u32x4 raw[R];
    if (wave_r0 + 4 * R <= rows && wave_c0 + 16 * V <= cols) {
      const T* p = x + (tile_r0 + row_of(0)) * job.ldx + c0;
#pragma unroll
      for (int i = 0; i < R; ++i, p += step) __builtin_memcpy(&raw[i], p, 16);
    } else if (wave_r0 >= rows || wave_c0 >= cols) {
#pragma unroll
      for (int i = 0; i < R; ++i) raw[i] = u32x4{0, 0, 0, 0};
    } else {
      // rows past the last read it again
      const int64_t from = c0 + V <= cols ? c0 : cols - V;
      const uint32_t drop = static_cast<uint32_t>(min<int64_t>(c0 - from, V) * sizeof(T));
      const T* p = x + min(tile_r0 + row_of(0), rows - 1) * job.ldx + from;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        __builtin_memcpy(&raw[i], p, 16);
        if (tile_r0 + row_of(i + 1) < rows) p += step;
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const u32x4 cut = drop_bytes(raw[i], drop);
        raw[i] = drop < 16 && tile_r0 + row_of(i) < rows ? cut : u32x4{0, 0, 0, 0};
      }
    }
    // this lane's place in a unit of q: fragment, block of it, bytes of the block
    const int in_chunk = wave_col + V * cl;
    const int fragment = in_chunk / 128, block = in_chunk % 128 / 32;
    const bool makes_q = job.q && rows_here;
    if (makes_q) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        uint32_t m = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) m = larger<T>(m, magnitudes<T>(raw[i][w]));
        if constexpr (sizeof(T) == 2) m = larger<T>(m, m >> 16) & 0xFFFFu;
        m = larger<float>(m, dpp_move<kQuadSwap1>(m));
        m = larger<float>(m, dpp_move<kQuadSwap2>(m));
        if constexpr (sizeof(T) == 4) m = larger<float>(m, dpp_move<kHalfMirror>(m));
        const Mx4Scale s = mx4_scale(float_bits<T>(m));
        uint32_t codes = 0;
        if constexpr (sizeof(T) == 4) {
          codes = mx4_codes<0>(codes, as_float(raw[i][0]), as_float(raw[i][1]), s.scale);
          codes = mx4_codes<1>(codes, as_float(raw[i][2]), as_float(raw[i][3]), s.scale);
        } else {
          codes = mx4_codes<0, T>(codes, raw[i][0], s.scale);
          codes = mx4_codes<1, T>(codes, raw[i][1], s.scale);
          codes = mx4_codes<2, T>(codes, raw[i][2], s.scale);
          codes = mx4_codes<3, T>(codes, raw[i][3], s.scale);
        }
        if (s.bad) codes = 0;
        const int row = row_of(i) & 15;
        uint8_t* const unit = row_units + kLdsUnit * (row_of(i) >> 4);
        if constexpr (sizeof(T) == 4)
          *reinterpret_cast<uint16_t*>(unit + lds_place(fragment, block, row) + 2 * (cl & 7)) = static_cast<uint16_t>(codes);
        else
          *reinterpret_cast<uint32_t*>(unit + lds_place(fragment, block, row) + 4 * (cl & 3)) = codes;
        if (in_chunk % 32 == 0) unit[kLdsScales + 2 * (row + 16 * block) + fragment] = static_cast<uint8_t>(s.code);
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (all rows at once do not fit the registers)
      }
    }
    if constexpr (kTransposed) {
      if (columns_here && (job.q_t || job.sums)) {
        // 256 rows are a chunk of q_t, this tile one of its fragments, g the block of it
        uint32_t largest[4] = {};
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int w = 0; w < 4; ++w) largest[w] = larger<T>(largest[w], magnitudes<T>(raw[i][w]));
#pragma unroll
        for (int v = 0; v < V; ++v) {
          constexpr int kPer = 4 / sizeof(T);  // columns to a word
          const int w = v / kPer;
          const uint32_t m = sizeof(T) == 4 ? largest[w] : v & 1 ? largest[w] >> 16 : largest[w] & 0xFFFFu;
          const Mx4Scale s = mx4_scale(float_bits<T>(m));
          u32x4 out;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t codes = 0;
            auto pair = [&](auto byte) {
              constexpr int b = decltype(byte)::value;
              const uint32_t lo = raw[8 * k + 2 * b][w], hi = raw[8 * k + 2 * b + 1][w];
              if constexpr (sizeof(T) == 4)
                codes = mx4_codes<b>(codes, as_float(lo), as_float(hi), s.scale);
              else
                codes = mx4_codes<b, T>(codes, __builtin_amdgcn_perm(hi, lo, v & 1 ? 0x07060302u : 0x05040100u), s.scale);
            };
            pair(std::integral_constant<int, 0>{});
            pair(std::integral_constant<int, 1>{});
            pair(std::integral_constant<int, 2>{});
            pair(std::integral_constant<int, 3>{});
            out[k] = s.bad ? 0u : codes;
          }
          const int row = (in_chunk + v) & 15;
          uint8_t* const unit = column_units + kLdsColumns * ((in_chunk + v) >> 4);
          *reinterpret_cast<u32x4*>(unit + lds_place(0, g, row)) = out;
          unit[kLdsFragment + row + 16 * g] = static_cast<uint8_t>(s.code);
          __builtin_amdgcn_sched_barrier(0);
          if (job.sums) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i) {
              const uint32_t word = raw[i][w];
              if constexpr (sizeof(T) == 4)
                sum += as_float(word);
              else
                sum += static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(v & 1 ? word >> 16 : word)));
            }
            // over the four lane groups
            const auto a = __builtin_amdgcn_permlane16_swap(as_uint(sum), as_uint(sum), false, false);
            sum = as_float(a[0]) + as_float(a[1]);
            const auto b = __builtin_amdgcn_permlane32_swap(as_uint(sum), as_uint(sum), false, false);
            sum = as_float(b[0]) + as_float(b[1]);
            if (g == 0 && c0 + v < cols && wave_r0 < rows) job.sums[(wave_r0 >> 7) * cols + c0 + v] = sum;
          }
        }
      }
    }
    __syncthreads();
    if (makes_q) {
      const int64_t group = static_cast<int64_t>(tile_row) * (S::kHigh / 16);
      store_units<S::kThreads>(row_units, min<int64_t>(S::kHigh / 16, mx4_groups(rows) - group),
                               job.q + (group * chunks + chunk) * kMx4Unit, chunks * kMx4Unit);
    }
    if constexpr (kTransposed) {
      if (job.q_t && columns_here) {
        const int64_t group = static_cast<int64_t>(chunk) * 16, t_stride = mx4_stride(rows);
        store_fragments<S::kThreads>(column_units, min<int64_t>(16, mx4_groups(cols) - group), tile_row & 1,
                                     job.q_t + group * t_stride + static_cast<int64_t>(tile_row / 2) * kMx4Unit, t_stride);
      }
    }
    __syncthreads();
  }
}

// Rows shorter than a vector: a thread takes a block of 32 values and loads them one
// by one. kTransposed: the matrix is x's transpose.
template <typename T, bool kTransposed>
__global__ __launch_bounds__(64) void quantize_narrow_kernel(Mx4Quantize job) {
  const int64_t rows = kTransposed ? job.cols : job.rows, cols = kTransposed ? job.rows : job.cols;
  const int64_t chunks = mx4_chunks(cols), units = mx4_groups(rows) * chunks;
  const int lane = threadIdx.x;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int64_t group = u / chunks, chunk = u - group * chunks, r = group * 16 + (lane & 15);
    uint8_t* const unit = (kTransposed ? job.q_t : job.q) + u * kMx4Unit;
    uint32_t scales = 0;
    for (int f = 0; f < 2; ++f) {
      const int64_t c = chunk * 256 + 128 * f + 32 * (lane >> 4);
      float v[32];
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const int64_t at = kTransposed ? (c + e) * job.ldx + r : r * job.ldx + c + e;
        v[e] = r < rows && c + e < cols ? static_cast<float>(static_cast<const T*>(job.x)[at]) : 0.0f;
        bits = larger<float>(bits, magnitude_bits(v[e]));
      }
      const Mx4Scale s = mx4_scale(bits);
      scales |= s.code << (8 * f);
      u32x4 out;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t codes = mx4_codes<0>(0u, v[8 * q], v[8 * q + 1], s.scale);
        codes = mx4_codes<1>(codes, v[8 * q + 2], v[8 * q + 3], s.scale);
        codes = mx4_codes<2>(codes, v[8 * q + 4], v[8 * q + 5], s.scale);
        codes = mx4_codes<3>(codes, v[8 * q + 6], v[8 * q + 7], s.scale);
        out[q] = s.bad ? 0u : codes;
      }
      *reinterpret_cast<u32x4*>(unit + 1024 * f + 16 * lane) = out;
    }
    *reinterpret_cast<uint16_t*>(unit + kMx4Scales + 2 * lane) = static_cast<uint16_t>(scales);
  }
}

// Sums of 128 rows of a column to a thread.
template <typename T>
__global__ __launch_bounds__(64) void sum_narrow_kernel(Mx4Quantize job) {
  const int64_t parts = (job.rows + 127) / 128;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x; i < parts * job.cols;
       i += static_cast<int64_t>(gridDim.x) * 64) {
    const int64_t part = i / job.cols, c = i - part * job.cols;
    float sum = 0.0f;
#pragma unroll 16
    for (int64_t r = 128 * part; r < min(128 * part + 128, job.rows); ++r)
      sum += static_cast<float>(static_cast<const T*>(job.x)[r * job.ldx + c]);
    job.sums[i] = sum;
  }
}

__global__ __launch_bounds__(256) void sum_partials_kernel(Mx4Sums s) {
  add_partials(s, blockIdx.x * 4 + (threadIdx.x >> 6), gridDim.x * 4, threadIdx.x & 63);
}

// ---- back ------------------------------------------------------------------------------
struct DequantizeArgs {
  const uint8_t* q;
  int64_t rows, cols, ldx;
  void* x;
};

// A wave takes a unit: sixteen lanes the 128 columns of a row of one fragment, eight to a lane.
template <typename T>
__global__ __launch_bounds__(256) void dequantize_mx4_kernel(DequantizeArgs a) {
  const int lane = threadIdx.x & 63, cl = lane & 15, g = lane >> 4;
  const int64_t chunks = mx4_chunks(a.cols), units = mx4_groups(a.rows) * chunks;
  T* const x = static_cast<T*>(a.x);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); u < units; u += static_cast<int64_t>(gridDim.x) * 4) {
    const int64_t group = u / chunks, chunk = u - group * chunks;
    const uint8_t* const unit = a.q + u * kMx4Unit;
    uint32_t codes[8], scale[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int place = 4 * (i & 3) + g + 16 * (cl >> 2);
      codes[i] = *reinterpret_cast<const uint32_t*>(unit + 1024 * (i >> 2) + 16 * place + 4 * (cl & 3));
      scale[i] = unit[kMx4Scales + 2 * place + (i >> 2)];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t row = group * 16 + 4 * (i & 3) + g, c = chunk * 256 + 128 * (i >> 2) + 8 * cl;
      const float s = as_float(scale[i] ? scale[i] << 23 : 0x00400000u);
      float v[8];
      auto two = [&](auto byte) {
        constexpr int b = decltype(byte)::value;
        const auto f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], s, b);
        v[2 * b] = f[0];
        v[2 * b + 1] = f[1];
      };
      two(std::integral_constant<int, 0>{});
      two(std::integral_constant<int, 1>{});
      two(std::integral_constant<int, 2>{});
      two(std::integral_constant<int, 3>{});
      if (scale[i] == 255u) {
#pragma unroll
        for (float& f : v) f = __builtin_nanf("");
      }
      if (row < a.rows && c < a.cols) store_upto8(x + row * a.ldx + c, a.cols - c, v);
    }
  }
}

// A wave takes a unit, a lane one block of each fragment.
__global__ __launch_bounds__(256) void pack_mx4_kernel(rns8_mi355x_pack_mx4_args a) {
  const int lane = threadIdx.x & 63;
  const int64_t chunks = mx4_chunks(a.cols), units = mx4_groups(a.rows) * chunks;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); u < units; u += static_cast<int64_t>(gridDim.x) * 4) {
    const int64_t group = u / chunks, chunk = u - group * chunks;
    const int64_t row = group * 16 + (lane & 15);
    uint8_t* const unit = a.q + u * kMx4Unit;
    uint32_t scales = 0;
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int64_t c = chunk * 256 + 128 * f + 32 * (lane >> 4);
      u32x4 codes = {0, 0, 0, 0};
      if (row < a.rows && c < a.cols) {
        const uint8_t* const p = a.data + row * a.ldd + c / 2;
        if (c + 32 <= a.cols) {
          __builtin_memcpy(&codes, p, 16);
        } else {
          uint8_t t[16] = {};
          const int count = static_cast<int>(a.cols - c);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (2 * e < count) t[e] = 2 * e + 1 < count ? p[e] : p[e] & 15;
          __builtin_memcpy(&codes, t, 16);
        }
        scales |= static_cast<uint32_t>(a.scale[row * a.lds + c / 32]) << (8 * f);
      }
      *reinterpret_cast<u32x4*>(unit + 1024 * f + 16 * lane) = codes;
    }
    *reinterpret_cast<uint16_t*>(unit + kMx4Scales + 2 * lane) = static_cast<uint16_t>(scales);
  }
}

template <typename T, bool kTransposed>
hipError_t launch_jobs(const Mx4Quantize* jobs, int count, hipStream_t stream) {
  using S = Shape<T, kTransposed>;
  Jobs j{};
  int64_t tiles = 0;
  for (int i = 0; i < count; ++i) {
    // (of q_t whole units, which are two tiles high)
    const int64_t chunks = mx4_chunks(jobs[i].cols);
    const int64_t mine = (kTransposed ? 2 * mx4_chunks(jobs[i].rows) : (jobs[i].rows + S::kHigh - 1) / S::kHigh) * chunks;
    tiles += mine;
    if (tiles > 0x3FFFFFFF) return hipErrorInvalidValue;
    j.job[i] = jobs[i];
    j.tiles[i] = static_cast<uint32_t>(mine);
    j.chunks[i] = make_div_u31(static_cast<uint32_t>(chunks));
  }
  if (tiles == 0) return hipSuccess;
  bool both = false;
  for (int i = 0; i < count; ++i) both = both || (jobs[i].q && (jobs[i].q_t || jobs[i].sums));
  j.apart = both && tiles * (S::kThreads / 64) <= 1024;
  tiles <<= j.apart;
  hipLaunchKernelGGL((quantize_mx4_kernel<T, kTransposed>), dim3(static_cast<unsigned>(std::min(tiles, kMaxBlocks))),
                     dim3(S::kThreads), 0, stream, j);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_narrow(const Mx4Quantize& job, hipStream_t stream) {
  auto grid = [](int64_t blocks) { return dim3(static_cast<unsigned>(std::min(blocks, kMaxBlocks))); };
  if (job.rows == 0) return hipSuccess;
  if (job.q)
    hipLaunchKernelGGL((quantize_narrow_kernel<T, false>), grid(mx4_groups(job.rows)), dim3(64), 0, stream, job);
  if (job.q_t)
    hipLaunchKernelGGL((quantize_narrow_kernel<T, true>), grid(mx4_chunks(job.rows)), dim3(64), 0, stream, job);
  if (job.sums)
    hipLaunchKernelGGL(sum_narrow_kernel<T>, grid((job.rows + 127) / 128), dim3(64), 0, stream, job);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_typed(const Mx4Quantize* jobs, int count, hipStream_t stream) {
  Mx4Quantize wide[2];
  int n = 0;
  bool transposed = false;
  for (int i = 0; i < count; ++i) {
    if (jobs[i].cols < 16 / static_cast<int64_t>(sizeof(T))) {
      const hipError_t e = launch_narrow<T>(jobs[i], stream);
      if (e != hipSuccess) return e;
      continue;
    }
    wide[n++] = jobs[i];
    transposed = transposed || jobs[i].q_t || jobs[i].sums;
  }
  return transposed ? launch_jobs<T, true>(wide, n, stream) : launch_jobs<T, false>(wide, n, stream);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

unsigned unit_grid(int64_t rows, int64_t cols) {
  return static_cast<unsigned>(std::min((mx4_groups(rows) * mx4_chunks(cols) + 3) / 4, kMaxBlocks));
}

}  // namespace

hipError_t launch_quantize_mx4(const Mx4Quantize* jobs, int count, uint32_t dtype, hipStream_t stream) {
  if (count < 1 || count > 2) return hipErrorInvalidValue;
  for (int i = 0; i < count; ++i) {
    const Mx4Quantize& j = jobs[i];
    if (j.rows < 0 || j.cols < 1 || j.rows > kMaxMx4Size || j.cols > kMaxMx4Size || (!j.q && !j.q_t && !j.sums) ||
        !aligned16(j.q) || !aligned16(j.q_t))
      return hipErrorInvalidValue;
  }
  if (dtype == RNS8_MI355X_F32) return launch_typed<float>(jobs, count, stream);
  if (dtype == RNS8_MI355X_F16) return launch_typed<f16>(jobs, count, stream);
  if (dtype == RNS8_MI355X_BF16) return launch_typed<bf16>(jobs, count, stream);
  return hipErrorInvalidValue;
}

hipError_t launch_sum_partials(const Mx4Sums& s, hipStream_t stream) {
  if (s.cols < 1) return hipErrorInvalidValue;
  hipLaunchKernelGGL(sum_partials_kernel, dim3(static_cast<unsigned>(std::min((s.cols + 63) / 64, kMaxBlocks))), dim3(256), 0,
                     stream, s);
  return hipGetLastError();
}

hipError_t launch_dequantize_mx4(const rns8_mi355x_mx4_args& a, hipStream_t stream) {
  if (a.rows < 0 || a.cols < 1 || a.rows > kMaxMx4Size || a.cols > kMaxMx4Size || !aligned16(a.q)) return hipErrorInvalidValue;
  if (a.rows == 0) return hipSuccess;
  const DequantizeArgs d{a.q, a.rows, a.cols, a.ldx, a.x};
  const dim3 grid(unit_grid(a.rows, a.cols));
  if (a.dtype == RNS8_MI355X_F32)
    hipLaunchKernelGGL(dequantize_mx4_kernel<float>, grid, dim3(256), 0, stream, d);
  else if (a.dtype == RNS8_MI355X_F16)
    hipLaunchKernelGGL(dequantize_mx4_kernel<f16>, grid, dim3(256), 0, stream, d);
  else
    hipLaunchKernelGGL(dequantize_mx4_kernel<bf16>, grid, dim3(256), 0, stream, d);
  return hipGetLastError();
}

hipError_t launch_pack_mx4(const rns8_mi355x_pack_mx4_args& a, hipStream_t stream) {
  if (a.rows < 0 || a.cols < 1 || a.rows > kMaxMx4Size || a.cols > kMaxMx4Size || !aligned16(a.q)) return hipErrorInvalidValue;
  if (a.rows == 0) return hipSuccess;
  hipLaunchKernelGGL(pack_mx4_kernel, dim3(unit_grid(a.rows, a.cols)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace rns8x
