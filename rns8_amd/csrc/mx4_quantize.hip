// Rounding of floating rows to MX4 and back (gfx950). Bound by HBM: a value is
// read once and leaves as 0.53 bytes for each form.
//
//   * A lane holds 16 bytes (V = 4 or 8 columns) of each of its rows as loaded;
//     sixteen lanes a row's 64 or 128 columns, so loads are whole lines.
//   * q (blocks along a row): a block is 4 or 8 neighbouring lanes, its largest
//     magnitude two or three lane moves after the lane's own (as integers: two
//     16-bit values at a time); v_cvt_scalef32_pk_fp4_* divides by the power of two
//     and rounds two values, half to even, 6 at most.
//   * q_t (blocks along a column): a lane's 32 rows are a block of each of its V
//     columns, so both forms come from one read and without LDS.
//   * Scales are gathered in LDS and leave as whole lines with the unit's.
//   * Sums of columns (a bias' gradient) in 32 bits for each 128 rows, in a fixed
//     order; a second kernel adds those.
#include <algorithm>
#include <type_traits>

#include "mx4.hpp"
#include "operators.hpp"
#include "row_shape.hpp"

namespace rns8x {
namespace {

struct Jobs {
  Mx4Quantize job[2];
  int64_t blocks[2];  // workgroups' tiles
};

constexpr int kQuadSwap1 = 0xB1, kQuadSwap2 = 0x4E, kHalfMirror = 0x141;  // DPP controls

// A workgroup's tile is 256 columns wide; kRows rows to a lane, of which a wave has
// four times as many. kTransposed: the tile is 256 rows high and q_t may be wanted.
template <typename T, bool kTransposed>
struct Shape {
  static constexpr int V = 16 / sizeof(T);
  static constexpr int kAcross = 16 / V;
  static constexpr int kRows = kTransposed ? 32 : 8;
  static constexpr int kDown = kTransposed ? 2 : 4 / kAcross;
  static constexpr int kThreads = 64 * kAcross * kDown;
  static constexpr int kHigh = 4 * kRows * kDown;
};

template <typename T, bool kTransposed>
__global__ __launch_bounds__((Shape<T, kTransposed>::kThreads)) void quantize_mx4_kernel(Jobs jobs) {
  using S = Shape<T, kTransposed>;
  constexpr int V = S::V, R = S::kRows;
  __shared__ __attribute__((aligned(16))) uint8_t row_scales[S::kHigh / 16 * 128];
  __shared__ __attribute__((aligned(16))) uint8_t column_scales[kTransposed ? 2048 : 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cl = lane & 15, g = lane >> 4;
  const int across = wave % S::kAcross, down = wave / S::kAcross;
  for (int64_t tile = blockIdx.x; tile < jobs.blocks[0] + jobs.blocks[1]; tile += gridDim.x) {
    const bool second = tile >= jobs.blocks[0];
    const Mx4Quantize& job = jobs.job[second ? 1 : 0];
    const int64_t at = second ? tile - jobs.blocks[0] : tile;
    const int64_t chunks = mx4_chunks(job.cols), rows = job.rows, cols = job.cols;
    const int64_t tile_row = at / chunks, chunk = at - tile_row * chunks;
    const int64_t wave_r0 = tile_row * S::kHigh + down * (4 * R), wave_c0 = chunk * 256 + across * (16 * V);
    const int64_t r0 = wave_r0 + g * R, c0 = wave_c0 + V * cl;
    const T* const x = static_cast<const T*>(job.x);
    u32x4 raw[R];
    if (wave_r0 + 4 * R <= rows && wave_c0 + 16 * V <= cols) {
#pragma unroll
      for (int i = 0; i < R; ++i) __builtin_memcpy(&raw[i], x + (r0 + i) * job.ldx + c0, 16);
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        raw[i] = u32x4{0, 0, 0, 0};
        const T* const p = x + (r0 + i) * job.ldx + c0;
        if (r0 + i < rows && c0 + V <= cols) {
          __builtin_memcpy(&raw[i], p, 16);
        } else if (r0 + i < rows && c0 < cols) {
          T t[V] = {};
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (c0 + e < cols) t[e] = p[e];
          __builtin_memcpy(&raw[i], t, 16);
        }
      }
    }
    // this lane's place in a unit of q: fragment, block of it, bytes of the block
    const int in_chunk = across * 16 * V + V * cl;
    const int fragment = in_chunk / 128, block = in_chunk % 128 / 32;
    if (job.q) {
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
        if (s.code == 255u) codes = 0;
        const int64_t row = r0 + i;
        const int place = static_cast<int>(row & 15) + 16 * block;
        uint8_t* const unit = job.q + (row >> 4) * chunks * kMx4Unit + chunk * kMx4Unit;
        if constexpr (sizeof(T) == 4) {
          codes |= dpp_move<kQuadSwap1>(codes) << 16;  // two lanes' codes, of which the even one writes both
          if (row < mx4_groups(rows) * 16 && !(lane & 1))
            *reinterpret_cast<uint32_t*>(unit + 1024 * fragment + 16 * place + 2 * (cl & 7)) = codes;
        } else {
          if (row < mx4_groups(rows) * 16)
            *reinterpret_cast<uint32_t*>(unit + 1024 * fragment + 16 * place + 4 * (cl & 3)) = codes;
        }
        if (in_chunk % 32 == 0) {
          const int local = static_cast<int>(row - tile_row * S::kHigh) >> 4;
          row_scales[128 * local + 2 * place + fragment] = static_cast<uint8_t>(s.code);
        }
      }
    }
    if constexpr (kTransposed) {
      if (job.q_t || job.sums) {
        const int64_t t_stride = mx4_stride(rows);
        const int64_t t_chunk = tile_row;  // 256 rows are a chunk of q_t, `down` its fragment
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
            out[k] = s.code == 255u ? 0u : codes;
          }
          const int64_t column = c0 + v;
          const int place = static_cast<int>(column & 15) + 16 * g;
          if (job.q_t && column < mx4_groups(cols) * 16)
            *reinterpret_cast<u32x4*>(job.q_t + (column >> 4) * t_stride + t_chunk * kMx4Unit + 1024 * down + 16 * place) = out;
          column_scales[128 * ((in_chunk + v) >> 4) + 2 * place + down] = static_cast<uint8_t>(s.code);
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
            if (g == 0 && column < cols && wave_r0 < rows) job.sums[(wave_r0 >> 7) * cols + column] = sum;
          }
        }
      }
    }
    __syncthreads();
    const int t = threadIdx.x;
    if (job.q && t < S::kHigh / 16 * 8) {
      const int64_t group = tile_row * (S::kHigh / 16) + t / 8;
      if (group < mx4_groups(rows))
        *reinterpret_cast<u32x4*>(job.q + (group * chunks + chunk) * kMx4Unit + kMx4Scales + t % 8 * 16) =
            *reinterpret_cast<const u32x4*>(row_scales + 16 * t);
    }
    if constexpr (kTransposed) {
      if (job.q_t && t < 128) {
        const int64_t group = chunk * 16 + t / 8;
        if (group < mx4_groups(cols))
          *reinterpret_cast<u32x4*>(job.q_t + group * mx4_stride(rows) + tile_row * kMx4Unit + kMx4Scales + t % 8 * 16) =
              *reinterpret_cast<const u32x4*>(column_scales + 16 * t);
      }
    }
    __syncthreads();
  }
}

__global__ __launch_bounds__(256) void sum_partials_kernel(const float* partials, int64_t count, int64_t cols, float* sums) {
  for (int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + (threadIdx.x & 63); c - (threadIdx.x & 63) < cols;
       c += static_cast<int64_t>(gridDim.x) * 64) {
    // four waves share the partials of 64 columns
    __shared__ float part[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float sum = 0.0f;
    if (c < cols)
      for (int64_t i = wave; i < count; i += 4) sum += partials[i * cols + c];
    part[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && c < cols) sums[c] = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
    __syncthreads();
  }
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
  for (int i = 0; i < count; ++i) {
    j.job[i] = jobs[i];
    // (of q_t, whole chunks of rows; of q alone, whole units)
    j.blocks[i] = (jobs[i].rows + S::kHigh - 1) / S::kHigh * mx4_chunks(jobs[i].cols);
  }
  const int64_t blocks = j.blocks[0] + j.blocks[1];
  if (blocks == 0) return hipSuccess;
  hipLaunchKernelGGL((quantize_mx4_kernel<T, kTransposed>), dim3(static_cast<unsigned>(std::min(blocks, kMaxBlocks))),
                     dim3(S::kThreads), 0, stream, j);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_typed(const Mx4Quantize* jobs, int count, hipStream_t stream) {
  bool transposed = false;
  for (int i = 0; i < count; ++i) transposed = transposed || jobs[i].q_t || jobs[i].sums;
  return transposed ? launch_jobs<T, true>(jobs, count, stream) : launch_jobs<T, false>(jobs, count, stream);
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

hipError_t launch_sum_partials(const float* partials, int64_t count, int64_t cols, float* sums, hipStream_t stream) {
  if (cols < 1) return hipErrorInvalidValue;
  hipLaunchKernelGGL(sum_partials_kernel, dim3(static_cast<unsigned>(std::min((cols + 63) / 64, kMaxBlocks))), dim3(256), 0,
                     stream, partials, count, cols, sums);
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
