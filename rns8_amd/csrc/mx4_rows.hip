// The product of MX4 matrices for few rows of a (gfx950). Bound by reading b, the
// weights, once.
//
//   * A workgroup owns 16 or 32 channels, its eight waves a share of K each: a
//     wave streams whole units of b from HBM into the MFMA's registers (one 16-byte
//     load to a fragment, one 16-bit load for two fragments' scales), the next
//     group's loads issued before a group is multiplied. The waves' sums are added in
//     LDS, in a fixed order.
//   * Floating rows (a linear layer's, at most 16) are rounded here: a lane holds
//     a whole block of one row, so its largest value, its scale and its codes need no
//     other lane, and are the MFMA's operands. That is less than the launch of a
//     kernel of its own.
#include <algorithm>
#include <type_traits>

#include "mx4.hpp"
#include "mx4_mfma.hpp"
#include "scaled_epilogue.hpp"

namespace rns8x {
namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;

struct RowsArgs {
  const uint8_t *a, *b;
  const void* x;
  int64_t ldx;
  const float* bias;
  int64_t m, n, ldo;
  uint32_t k, chunks;
  void* out;
  uint32_t dtype;
};

// As many chunks as a wave has of 8192 columns, where the registers of two waves to a
// SIMD hold them.
template <int MB, int RB, typename T>
constexpr int ring_depth() {
  if constexpr (std::is_void_v<T>)
    return MB + RB <= 4 ? 4 : MB + RB <= 5 ? 3 : 2;
  else
    return sizeof(T) == 4 ? 2 : RB == 2 ? 3 : 4;
}

// T: the rows' type, or void where they are an MX4 matrix.
template <int kTokens16, int kChannels16, typename T>
__global__ __launch_bounds__(kThreads) void mx4_rows_kernel(RowsArgs a) {
  constexpr int MB = kTokens16, RB = kChannels16;
  constexpr bool kFused = !std::is_void_v<T>;
  constexpr int D = ring_depth<MB, RB, T>();  // chunks in flight
  __shared__ __attribute__((aligned(16))) f32x4 sums[kWaves][MB * RB][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * RB), m0 = static_cast<int64_t>(blockIdx.y) * (16 * MB);
  const uint32_t chunks = a.chunks;
  const uint32_t first = chunks * wave / kWaves, last = chunks * (wave + 1) / kWaves;
  const int64_t stride = static_cast<int64_t>(chunks) * kMx4Unit;

  const uint8_t* wrow[RB];
#pragma unroll
  for (int j = 0; j < RB; ++j) wrow[j] = a.b + min(n0 / 16 + j, mx4_groups(a.n) - 1) * stride;
  const uint8_t* arow[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) arow[i] = kFused ? nullptr : a.a + min(m0 / 16 + i, mx4_groups(a.m) - 1) * stride;

  using X = std::conditional_t<kFused, T, float>;
  struct Group {
    Mx4Unit w[RB], t[MB];
    RawBlock<X> x[kFused ? 2 : 1];
  };
  // a lane's row of floating x, its block of each fragment
  const int64_t mine = m0 + (lane & 15);
  const bool live = mine < a.m;
  const X* const row = static_cast<const X*>(a.x) + (live ? mine : 0) * a.ldx;
  auto load = [&](uint32_t c, Group& f) __attribute__((always_inline)) {
    // (past the wave's last chunk it is read again and not used)
    const uint32_t chunk = min(c, last - 1);
    const int64_t at = static_cast<int64_t>(chunk) * kMx4Unit;
    if constexpr (kFused) {
      // the rows first: loads return in order, and rounding them takes time
#pragma unroll
      for (int h = 0; h < 2; ++h) load_block(row, 256 * chunk + 128 * h + 32 * (lane >> 4), a.k, f.x[h]);
    }
#pragma unroll
    for (int j = 0; j < RB; ++j) f.w[j] = stream_unit(wrow[j] + at, lane);
    if constexpr (!kFused) {
#pragma unroll
      for (int i = 0; i < MB; ++i) f.t[i] = load_unit(arow[i] + at, lane);
    }
  };
  f32x4 acc[MB][RB] = {};
  auto multiply = [&](uint32_t c, Group& f) __attribute__((always_inline)) {
    if constexpr (kFused) {
      f.t[0].scales = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        cut_block(row, 256 * c + 128 * h + 32 * (lane >> 4), live ? a.k : 0, f.x[h]);
        const Mx4Block b = round_block(f.x[h]);
        f.t[0].codes[h] = b.codes;
        f.t[0].scales |= b.scale << (8 * h);
      }
    }
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < RB; ++j) {
        acc[i][j] = mx4_mfma<0>(f.w[j].codes[0], f.t[i].codes[0], acc[i][j], f.w[j].scales, f.t[i].scales);
        acc[i][j] = mx4_mfma<1>(f.w[j].codes[1], f.t[i].codes[1], acc[i][j], f.w[j].scales, f.t[i].scales);
      }
  };
  // a ring of D chunks' loads, without branches about them: a wait then counts them
  if (first < last) {
    Group ring[D];
#pragma unroll
    for (int d = 0; d < D; ++d) load(first + d, ring[d]);
    uint32_t c = first;
    for (; c + D < last; c += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        multiply(c + d, ring[d]);
        load(c + D + d, ring[d]);
      }
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (c + d < last) multiply(c + d, ring[d]);
  }
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < RB; ++j) sums[wave][i * RB + j][lane] = acc[i][j];
  __syncthreads();
  static_assert(MB * RB * 64 <= kThreads, "one quad of outputs to a thread");
  const int e = threadIdx.x;
  if (e >= MB * RB * 64) return;
  const int l = e & 63, block = e >> 6;
  const int64_t token = m0 + 16 * (block / RB) + (l & 15), channel = n0 + 16 * (block % RB) + 4 * (l >> 4);
  if (token >= a.m || channel >= a.n) return;
  f32x4 sum = sums[0][block][l];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) sum += sums[w][block][l];
  float bias[4], v[4];
  load4_or(a.bias, channel, a.n, 0.0f, bias);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = sum[i] + bias[i];
  const int64_t at = token * a.ldo + channel;
  if (a.dtype == RNS8_MI355X_F32)
    store4(static_cast<float*>(a.out) + at, a.n - channel, v);
  else if (a.dtype == RNS8_MI355X_F16)
    store4(static_cast<f16*>(a.out) + at, a.n - channel, v);
  else
    store4(static_cast<bf16*>(a.out) + at, a.n - channel, v);
}

template <int MB, typename T>
hipError_t launch_shape(const RowsArgs& a, hipStream_t stream) {
  const int64_t tokens = (a.m + 16 * MB - 1) / (16 * MB);
  // two groups of channels to a workgroup where that leaves one for each CU
  const bool wide = a.n >= 256 * 32 && MB * 2 <= 8;
  const int64_t blocks = (a.n + (wide ? 31 : 15)) / (wide ? 32 : 16);
  if (blocks > 0x7FFFFF || tokens > 65535 || blocks * tokens > 0x7FFFFF) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(tokens));
  if (wide)
    hipLaunchKernelGGL((mx4_rows_kernel<MB, 2, T>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((mx4_rows_kernel<MB, 1, T>), grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx4_rows(const Mx4Gemm& g, hipStream_t stream) {
  if (g.m < 1 || g.n < 1 || g.k < 0 || g.k > kMaxMx4Sum || g.dtype > RNS8_MI355X_BF16) return hipErrorInvalidValue;
  RowsArgs a{};
  a.a = g.a;
  a.b = g.b;
  a.x = g.x;
  a.ldx = g.ldx;
  a.bias = g.bias;
  a.m = g.m;
  a.n = g.n;
  a.ldo = g.ldo;
  a.k = static_cast<uint32_t>(g.k);
  a.chunks = static_cast<uint32_t>(mx4_chunks(g.k));
  a.out = g.out;
  a.dtype = g.dtype;
  if (g.x) {
    if (g.m > kMx4FusedRows) return hipErrorInvalidValue;
    if (g.dtype == RNS8_MI355X_F32) return launch_shape<1, float>(a, stream);
    if (g.dtype == RNS8_MI355X_F16) return launch_shape<1, f16>(a, stream);
    return launch_shape<1, bf16>(a, stream);
  }
  if (g.m <= 16) return launch_shape<1, void>(a, stream);
  if (g.m <= 32) return launch_shape<2, void>(a, stream);
  if (g.m <= 48) return launch_shape<3, void>(a, stream);
  return launch_shape<4, void>(a, stream);
}

}  // namespace rns8x
