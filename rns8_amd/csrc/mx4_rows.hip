// The product of MX4 matrices for few rows of a (gfx950). Bound by reading b, the
// weights, once.
//
//   * A workgroup owns 16 or 32 channels, its eight waves a share of K each: a
//     wave streams whole units of b into the MFMA's registers (one 16-byte
//     load to a fragment, one 16-bit load for two fragments' scales), a ring of chunks
//     ahead. The waves' sums are added in LDS, in a fixed order.
//   * Floating rows (a linear layer's, at most 16) are rounded here, which is less than
//     the launch of a kernel of its own: a wave rounds its share of each row, a block to
//     a lane, while its first weights are on their way, and hands the codes to the MFMA
//     through LDS of its own. (A lane that rounded its own operand, a row to each 16
//     lanes, would leave all but one of those idle where there is one row: 10.9 us for
//     8192 x 8192 in bf16.)
// Measured: 1 x 8192 x 8192 in bf16, floating row 8.4 us (4.2 TB/s) on the weights of 16
// layers in turn, which come from HBM, 5.4 on one layer's again and again (36 MB, which the
// 256 MB of cache beside HBM hold); 48 x 8192 x 4096 in f16 5.4 us on the same weights (3.3 TB/s:
// 48 rows' units come from the L2s for each 32 channels).
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

// The waves' sums of MB x RB blocks of 16 x 16 outputs, added, with bias, to memory.
template <int MB, int RB>
__device__ __forceinline__ void store_sums(const RowsArgs& a, const f32x4 (*sums)[MB * RB][64], int64_t m0, int64_t n0) {
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

template <int kTokens16, int kChannels16>
__global__ __launch_bounds__(kThreads) void mx4_rows_kernel(RowsArgs a) {
  constexpr int MB = kTokens16, RB = kChannels16;
  constexpr int D = MB + RB <= 4 ? 4 : MB + RB <= 5 ? 3 : 2;  // chunks in flight: what the registers hold
  __shared__ __attribute__((aligned(16))) f32x4 sums[kWaves][MB * RB][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * RB), m0 = static_cast<int64_t>(blockIdx.y) * (16 * MB);
  const uint32_t chunks = a.chunks;
  const uint32_t first = chunks * wave / kWaves, last = chunks * (wave + 1) / kWaves;
  const int64_t stride = static_cast<int64_t>(chunks) * kMx4Unit;
  const uint8_t *wrow[RB], *arow[MB];
#pragma unroll
  for (int j = 0; j < RB; ++j) wrow[j] = a.b + min(n0 / 16 + j, mx4_groups(a.n) - 1) * stride;
#pragma unroll
  for (int i = 0; i < MB; ++i) arow[i] = a.a + min(m0 / 16 + i, mx4_groups(a.m) - 1) * stride;
  struct Group {
    Mx4Unit w[RB], t[MB];
  };
  auto load = [&](uint32_t c, Group& f) __attribute__((always_inline)) {
    // (past the wave's last chunk it is read again and not used)
    const int64_t at = static_cast<int64_t>(min(c, last - 1)) * kMx4Unit;
#pragma unroll
    for (int j = 0; j < RB; ++j) f.w[j] = load_unit(wrow[j] + at, lane);
#pragma unroll
    for (int i = 0; i < MB; ++i) f.t[i] = load_unit(arow[i] + at, lane);
  };
  f32x4 acc[MB][RB] = {};
  auto multiply = [&](const Group& f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < RB; ++j) acc[i][j] = mx4_mfma(f.w[j], f.t[i], acc[i][j]);
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
        multiply(ring[d]);
        load(c + D + d, ring[d]);
      }
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (c + d < last) multiply(ring[d]);
  }
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < RB; ++j) sums[wave][i * RB + j][lane] = acc[i][j];
  __syncthreads();
  store_sums<MB, RB>(a, sums, m0, n0);
}

// At most kTokens (2 or 16) floating rows.
template <int kTokens, int kChannels16, typename T>
__global__ __launch_bounds__(kThreads) void mx4_linear_rows_kernel(RowsArgs a) {
  constexpr int RB = kChannels16;
  constexpr int D = kTokens == 2 ? 4 : 2;        // chunks rounded and multiplied together
  constexpr int R = (8 * D * kTokens + 63) / 64;  // blocks of them to a lane
  __shared__ __attribute__((aligned(16))) union {
    uint8_t units[kWaves][D][kMx4Unit];
    f32x4 sums[kWaves][RB][64];
  } lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * RB);
  const uint32_t chunks = a.chunks, m = static_cast<uint32_t>(a.m);
  const uint32_t first = chunks * wave / kWaves, last = chunks * (wave + 1) / kWaves;
  const int64_t stride = static_cast<int64_t>(chunks) * kMx4Unit;
  const uint8_t* wrow[RB];
#pragma unroll
  for (int j = 0; j < RB; ++j) wrow[j] = a.b + min(n0 / 16 + j, mx4_groups(a.n) - 1) * stride;
  // a wave's chunks whose columns are all there; one may follow that the rows' end cuts
  const uint32_t end = min(last, a.k / 256);

  // block i of a group of D chunks: row i / (8 D), and of its 8 D blocks that one
  auto row_of = [&](uint32_t i) { return static_cast<const T*>(a.x) + min(i / (8 * D), m - 1) * a.ldx; };
  RawBlock<T> x[R];
  Mx4Unit w[D][RB];
  // (rows past the last and chunks past the wave's last are others again, and not used)
  auto load_x = [&](uint32_t c) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t i = 64 * r + lane, j = i % (8 * D);
      load_block(row_of(i), 256 * min(c + j / 8, end - 1) + 32 * (j % 8), x[r]);
    }
  };
  auto load_w = [&](uint32_t c, Mx4Unit (&u)[RB]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < RB; ++j) u[j] = load_unit(wrow[j] + static_cast<int64_t>(min(c, end - 1)) * kMx4Unit, lane);
  };
  // The codes of row t's block j into the unit that the MFMA reads. (What no block fills
  // goes into columns of the product that are not stored.)
  auto put = [&](uint32_t i, const RawBlock<T>& x) __attribute__((always_inline)) {
    const uint32_t t = i / (8 * D), j = i % (8 * D);
    const Mx4Block b = round_block(x);
    if (t >= m) return;
    uint8_t* const unit = lds.units[wave][j / 8];
    const uint32_t place = t + 16 * (j % 4), fragment = j / 4 % 2;
    *reinterpret_cast<i32x4*>(unit + 1024 * fragment + 16 * place) = b.codes;
    unit[kMx4Scales + 2 * place + fragment] = static_cast<uint8_t>(b.scale);
  };
  f32x4 acc[RB] = {};
  auto multiply_chunk = [&](int d, const Mx4Unit (&w)[RB]) __attribute__((always_inline)) {
    const uint8_t* const unit = lds.units[wave][d];
    Mx4Unit t;
    t.codes[0] = *reinterpret_cast<const i32x4*>(unit + 16 * lane);
    t.codes[1] = *reinterpret_cast<const i32x4*>(unit + 1024 + 16 * lane);
    t.scales = *reinterpret_cast<const uint16_t*>(unit + kMx4Scales + 2 * lane);
#pragma unroll
    for (int j = 0; j < RB; ++j) acc[j] = mx4_mfma(w[j], t, acc[j]);
  };
  if (first < end) {
    // Rows before weights: loads return in order. No branches about them: a wait then
    // counts them.
    auto round = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int r = 0; r < R; ++r) put(64 * r + lane, x[r]);
      __builtin_amdgcn_wave_barrier();  // (LDS serves a wave in order)
    };
    load_x(first);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < D; ++d) load_w(first + d, w[d]);
    uint32_t c = first;
    for (; c + D < end; c += D) {
      round();
      load_x(c + D);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < D; ++d) {
        multiply_chunk(d, w[d]);
        load_w(c + D + d, w[d]);
      }
      __builtin_amdgcn_wave_barrier();
    }
    round();
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (c + d < end) multiply_chunk(d, w[d]);
    __builtin_amdgcn_wave_barrier();
  }
  if (end < last && first < last) {
#pragma unroll
    for (int j = 0; j < RB; ++j) w[0][j] = load_unit(wrow[j] + static_cast<int64_t>(last - 1) * kMx4Unit, lane);
    // one chunk: eight blocks to a row
    for (uint32_t i = lane; i < 8 * m; i += 64) {
      load_cut_block(static_cast<const T*>(a.x) + (i / 8) * a.ldx, 256 * (last - 1) + 32 * (i % 8), a.k, x[0]);
      put(i / 8 * (8 * D) + i % 8, x[0]);
    }
    __builtin_amdgcn_wave_barrier();
    multiply_chunk(0, w[0]);
  }
  __syncthreads();  // the units are read
#pragma unroll
  for (int j = 0; j < RB; ++j) lds.sums[wave][j][lane] = acc[j];
  __syncthreads();
  store_sums<1, RB>(a, lds.sums, 0, n0);
}

// Two groups of channels to a workgroup where that leaves one for each CU.
bool wide(int64_t n) { return n >= 256 * 32; }

template <int MB>
hipError_t launch_shape(const RowsArgs& a, hipStream_t stream) {
  const int64_t tokens = (a.m + 16 * MB - 1) / (16 * MB), blocks = (a.n + (wide(a.n) ? 31 : 15)) / (wide(a.n) ? 32 : 16);
  if (blocks > 0x7FFFFF) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(tokens));
  if (wide(a.n))
    hipLaunchKernelGGL((mx4_rows_kernel<MB, 2>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((mx4_rows_kernel<MB, 1>), grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

template <int kTokens, typename T>
hipError_t launch_linear(const RowsArgs& a, hipStream_t stream) {
  const int64_t blocks = (a.n + (wide(a.n) ? 31 : 15)) / (wide(a.n) ? 32 : 16);
  if (blocks > 0x7FFFFF) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (wide(a.n))
    hipLaunchKernelGGL((mx4_linear_rows_kernel<kTokens, 2, T>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((mx4_linear_rows_kernel<kTokens, 1, T>), grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_typed(const RowsArgs& a, hipStream_t stream) {
  return a.m <= 2 ? launch_linear<2, T>(a, stream) : launch_linear<16, T>(a, stream);
}

}  // namespace

hipError_t launch_mx4_rows(const Mx4Gemm& g, hipStream_t stream) {
  if (g.m < 1 || g.n < 1 || g.k < 1 || g.k > kMaxMx4Sum || g.dtype > RNS8_MI355X_BF16) return hipErrorInvalidValue;
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
    if (g.dtype == RNS8_MI355X_F32) return launch_typed<float>(a, stream);
    if (g.dtype == RNS8_MI355X_F16) return launch_typed<f16>(a, stream);
    return launch_typed<bf16>(a, stream);
  }
  if (g.m <= 16) return launch_shape<1>(a, stream);
  if (g.m <= 32) return launch_shape<2>(a, stream);
  if (g.m <= 48) return launch_shape<3>(a, stream);
  return launch_shape<4>(a, stream);
}

}  // namespace rns8x
