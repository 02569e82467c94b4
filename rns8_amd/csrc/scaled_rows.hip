// The scaled 8-bit product for few tokens (gfx950): at most 64 rows of a, b
// stored n x k. Bound by reading b (the weights) once.
//
//   * A workgroup owns 16 or 32 channels; its eight waves cut their K between
//     them, so that 8192 channels are 4096 waves with all of their loads in
//     flight, and add their int32 sums in LDS. No partial sum leaves the CU.
//   * b goes from HBM into the MFMA's registers: lane l loads 16 bytes of channel
//     l % 16 at 16 (l / 16) of each 64 of K (16 rows x 64 bytes to a load), at any
//     alignment. The next group's loads are issued before a group is multiplied.
//   * a (in 8 bits) is small and read the same way, from the caches; 32 channels
//     to a wave halve that traffic where there are more than 16 tokens, and the
//     linear layer then stores its rows in fragment order, whole cache lines to a
//     load.
//   * One or two tokens of a linear layer are quantized here, by every workgroup
//     into its LDS, while its first weights are on their way: less than the launch
//     of a kernel of its own.
// Measured: one token (bf16, quantized here) by 8192 x 8192 16.3 us with its launch
// (67 MB: 4.1 TB/s); 48 tokens by 8192 x 4096 in fragment order 10.4 us.
#include <algorithm>
#include <type_traits>

#include "scaled_epilogue.hpp"
#include "scaled_gemm.hpp"

namespace rns8x {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kWaves = 8, kThreads = 64 * kWaves;

struct RowsArgs {
  const int8_t* w;
  int64_t ldw;
  const int8_t* q;  // m x k; not fused
  int64_t ldq;
  const float *a_scale, *b_scale, *bias;
  int64_t m, n;
  uint32_t k;
  void* out;
  int64_t ldo;
  uint32_t dtype;
  // fused: the floating rows, and where their bytes and scales go if anywhere
  const void* x;
  int64_t ldx;
  int8_t* q_out;
  int64_t ldq_out, stop;
  float* scale_out;
};

// 16 bytes from byte c on of a row of k bytes (k >= 16) at any alignment, zeros past its end.
__device__ __forceinline__ v4i load_cut(const int8_t* row, uint32_t c, uint32_t k) {
  u32x4 w;
  const bool whole = c + 16 <= k;
  __builtin_memcpy(&w, row + (whole ? c : k - 16), 16);
  if (!whole) w = c < k ? drop_bytes(w, c + 16 - k) : u32x4{0, 0, 0, 0};
  return __builtin_bit_cast(v4i, w);
}

// kFragments: q in fragment order.
template <int kTokens16, int kChannels16, int kUnroll, bool kFused, bool kFragments, typename T>
__global__ __launch_bounds__(kThreads) void scaled_rows_kernel(RowsArgs a) {
  constexpr int MB = kTokens16, RB = kChannels16, U = kUnroll;
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];  // fused: m rows of k bytes; then the waves' sums
  __shared__ uint32_t amax_lds[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * RB);
  const uint32_t k = a.k, blocks = k / 64, tail = k % 64;
  const uint32_t first = blocks * wave / kWaves, last = blocks * (wave + 1) / kWaves;

  const int8_t* wrow[RB];
#pragma unroll
  for (int j = 0; j < RB; ++j) wrow[j] = a.w + min(n0 + 16 * j + r, a.n - 1) * a.ldw;
  const int8_t* qrow[MB];
  // (tokens past the last repeat it: their sums are not stored)
  const uint32_t pitch = (k + 63) / 64 * 64 + 16;  // fused: LDS rows
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int64_t t = min<int64_t>(16 * i + r, a.m - 1);
    qrow[i] = kFused ? lds + t * pitch : a.q + t * a.ldq;
  }
  auto fragment = [&](uint32_t block, int i) {
    return *reinterpret_cast<const v4i*>(a.q + (static_cast<uint64_t>(block) * MB + i) * 1024 + 16 * lane);
  };
  struct Group {
    v4i w[U][RB];
    v4i q[kFused ? 1 : U][MB];
  };
  auto load = [&](uint32_t b, Group& f) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (groups past the wave's last block read it again and are not used)
      const uint32_t c = 64 * min(b + u, last - 1) + 16 * g;
#pragma unroll
      for (int j = 0; j < RB; ++j) __builtin_memcpy(&f.w[u][j], wrow[j] + c, 16);
      if constexpr (!kFused) {
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if constexpr (kFragments)
            f.q[u][i] = fragment(min(b + u, last - 1), i);
          else
            __builtin_memcpy(&f.q[u][i], qrow[i] + c, 16);
        }
      }
    }
  };
  v4i acc[MB][RB] = {};
  auto multiply = [&](uint32_t b, const Group& f) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b + u >= last) break;  // the same in every lane
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        v4i q;
        if constexpr (kFused)
          q = *reinterpret_cast<const v4i*>(qrow[i] + 64 * (b + u) + 16 * g);
        else
          q = f.q[u][i];
#pragma unroll
        for (int j = 0; j < RB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.w[u][j], q, acc[i][j], 0, 0, 0);
      }
    }
  };
  Group now, next;
  if (first < last) load(first, now);
  // this thread's four outputs in the end, whose scales and biases are on their
  // way from here on: block (i, j), lane l of it
  static_assert(MB * RB * 64 <= kThreads, "one quad of outputs to a thread");
  const int e = threadIdx.x, l = e & 63, out_j = (e >> 6) % RB, out_i = (e >> 6) / RB;
  const bool writes = e < MB * RB * 64 && 16 * out_i + (l & 15) < a.m && n0 + 16 * out_j + 4 * (l >> 4) < a.n;
  const int64_t token = 16 * out_i + (l & 15), channel = n0 + 16 * out_j + 4 * (l >> 4);
  float sb[4], bias[4], token_scale = 1.0f;
  if (writes) {
    load4_or(a.b_scale, channel, a.n, 1.0f, sb);
    load4_or(a.bias, channel, a.n, 0.0f, bias);
    if (!kFused && a.a_scale) token_scale = a.a_scale[token];
  }
  float scale[2] = {1.0f, 1.0f};
  if constexpr (kFused) {
    // the tokens' maxima, then their bytes, zeros up to whole blocks
    if (threadIdx.x < 2) amax_lds[threadIdx.x] = 0;
    __syncthreads();
    const int tokens = static_cast<int>(a.m);
    for (int t = 0; t < tokens; ++t) {
      const T* const x = static_cast<const T*>(a.x) + t * a.ldx;
      uint32_t amax = 0;
      for (uint32_t c = 8 * threadIdx.x; c < k; c += 8 * kThreads) {
        float v[8];
        load_upto8(x + c, k - c, v, 0.0f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t m = magnitude_bits(v[i]);
          amax = amax > m ? amax : m;
        }
      }
      amax = wave_reduce(amax, MaxU{});
      if (lane == 0) atomicMax(&amax_lds[t], amax);
    }
    __syncthreads();
    for (int t = 0; t < tokens; ++t) {
      const T* const x = static_cast<const T*>(a.x) + t * a.ldx;
      const RowScale s = row_scale(amax_lds[t]);
      scale[t] = s.scale;
      const bool mine = blockIdx.x == 0 && a.q_out;
      if (mine && threadIdx.x == 0) a.scale_out[t] = s.scale;
      for (uint32_t c = 8 * threadIdx.x; c < (k + 63) / 64 * 64; c += 8 * kThreads) {
        float v[8] = {};
        if (c < k) load_upto8(x + c, k - c, v, 0.0f);
        const uint64_t w = quantize8(v, s.inverse);
        *reinterpret_cast<uint64_t*>(lds + t * pitch + c) = w;
        if (mine && c < a.stop) store_bytes8(a.q_out + t * a.ldq_out, c, a.stop, w);
      }
    }
    __syncthreads();
  }
  for (uint32_t b = first; b < last; b += U) {
    if (b + U < last) load(b + U, next);
    multiply(b, now);
    now = next;
  }
  if (tail && wave == kWaves - 1) {
    const uint32_t c = 64 * blocks + 16 * g;
    v4i w[RB];
#pragma unroll
    for (int j = 0; j < RB; ++j) w[j] = load_cut(wrow[j], c, k);
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      v4i q;
      if constexpr (kFused)
        q = *reinterpret_cast<const v4i*>(qrow[i] + c);
      else if constexpr (kFragments)
        q = fragment(blocks, i);
      else
        q = load_cut(qrow[i], c, k);
#pragma unroll
      for (int j = 0; j < RB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j], q, acc[i][j], 0, 0, 0);
    }
  }
  // the waves' sums: lane l holds token l % 16, channels 4 (l / 16) .. + 3 of a 16 x 16 block
  if constexpr (kFused) __syncthreads();  // (the rows in LDS are read)
  v4i* const sums = reinterpret_cast<v4i*>(lds);
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < RB; ++j) sums[((wave * MB + i) * RB + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  if (!writes) return;
  v4i sum = sums[e];
#pragma unroll
  for (int v = 1; v < kWaves; ++v) sum += sums[v * MB * RB * 64 + e];
  const float sa = kFused ? (token ? scale[1] : scale[0]) : token_scale;
  float f[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) f[x] = scaled_value(sum[x], sa, sb[x], bias[x]);
  const int64_t at = token * a.ldo + channel;
  if (a.dtype == RNS8_MI355X_BF16)
    store4(static_cast<bf16*>(a.out) + at, a.n - channel, f);
  else if (a.dtype == RNS8_MI355X_F16)
    store4(static_cast<f16*>(a.out) + at, a.n - channel, f);
  else
    store4(static_cast<float*>(a.out) + at, a.n - channel, f);
}

template <int MB, int RB, int U, bool kFused, bool kFragments, typename T>
hipError_t launch(const RowsArgs& a, hipStream_t stream) {
  const int64_t blocks = (a.n + 16 * RB - 1) / (16 * RB);
  if (blocks > 0x3FFFFF) return hipErrorInvalidValue;
  const size_t sums = static_cast<size_t>(kWaves) * MB * RB * 64 * sizeof(v4i);
  const size_t rows = kFused ? static_cast<size_t>(a.m) * ((a.k + 63) / 64 * 64 + 16) : 0;
  hipLaunchKernelGGL((scaled_rows_kernel<MB, RB, U, kFused, kFragments, T>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads),
                     static_cast<unsigned>(std::max(sums, rows)), stream, a);
  return hipGetLastError();
}

}  // namespace

bool scaled_rows_takes(int64_t m, int64_t n, int64_t k, bool inner) {
  return !inner && m <= 64 && k >= 16 && k <= kExactK && n <= (int64_t{1} << 25);
}

// A start, then the larger of a workgroup's own time (its K, read once for
// the weights and once for every 16 tokens) and the weights' from HBM beside
// what more than 16 tokens add, a quarter of it from fragment order. Fitted to 50
// shapes from 4 x 256 x 256 to 64 x 8192 x 8192, within 15% at each: 48 tokens by
// 8192 x 4096 14.9 us for 13.1 from rows and 10.4 for 9.7 in fragment order.
double scaled_rows_cost(int64_t m, int64_t n, int64_t k, bool fragments) {
  const double depth = static_cast<double>(k) / 8192, tokens16 = static_cast<double>((m + 15) / 16);
  const double more = (fragments ? 0.9 : 3.6) * depth * (tokens16 - 1), own = depth * 5.6 + more;
  return 3.4 + std::max(own, static_cast<double>(n) * static_cast<double>(k) / kBytesPerUs + more);
}

hipError_t launch_scaled_rows(const ScaledGemm& g, hipStream_t stream) {
  if (!scaled_rows_takes(g.m, g.n, g.k, g.inner) || g.m <= 0 || g.n <= 0) return hipErrorInvalidValue;
  RowsArgs a{};
  a.w = g.b;
  a.ldw = g.ldb;
  a.q = g.a;
  a.ldq = g.lda;
  a.a_scale = g.a_scale;
  a.b_scale = g.b_scale;
  a.bias = g.bias;
  a.m = g.m;
  a.n = g.n;
  a.k = static_cast<uint32_t>(g.k);
  a.out = g.out;
  a.ldo = g.ldo;
  a.dtype = g.dtype;
  // 32 channels to a workgroup read a half as often, 16 keep twice the workgroups
  // in flight: from a workgroup of 32 per CU on (and more than one token) the
  // former. In us, 16 / 32 channels: 8192 x 8192 with 1, 16, 48, 64 tokens 15.1 /
  // 15.6, 21.4 / 17.4, 36.8 / 25.6, 43.9 / 28.9; 4096 x 4096 6.5 / 8, 7.5 / 10,
  // 11.3 / 13.0, 13.1 / 15.1.
  const bool wide = g.m > 1 && g.n >= 32 * 256;
  if (g.m <= 16)
    return wide ? launch<1, 2, 4, false, false, float>(a, stream) : launch<1, 1, 4, false, false, float>(a, stream);
  auto tokens = [&](auto fragments) {
    constexpr bool kFragments = decltype(fragments)::value;
    if (g.m <= 32)
      return wide ? launch<2, 2, 4, false, kFragments, float>(a, stream)
                  : launch<2, 1, 4, false, kFragments, float>(a, stream);
    if (g.m <= 48)
      return wide ? launch<3, 2, 4, false, kFragments, float>(a, stream)
                  : launch<3, 1, 4, false, kFragments, float>(a, stream);
    return wide ? launch<4, 2, 4, false, kFragments, float>(a, stream)
                : launch<4, 1, 4, false, kFragments, float>(a, stream);
  };
  return g.fragments ? tokens(std::true_type{}) : tokens(std::false_type{});
}

// Two tokens at most, and no more bytes than the quantization is worth beside
// its own kernel.
bool linear_rows_takes(int64_t m, int64_t n, int64_t k) {
  return scaled_rows_takes(m, n, k, false) && m <= 2 && m * k <= 16384;
}

hipError_t launch_linear_rows(const rns8_mi355x_linear_i8_args& g, hipStream_t stream) {
  if (!linear_rows_takes(g.m, g.n, g.k) || g.m <= 0 || g.n <= 0) return hipErrorInvalidValue;
  RowsArgs a{};
  a.w = g.w;
  a.ldw = g.ldw;
  a.b_scale = g.w_scale;
  a.bias = g.bias;
  a.m = g.m;
  a.n = g.n;
  a.k = static_cast<uint32_t>(g.k);
  a.out = g.out;
  a.ldo = g.ldo;
  a.dtype = g.dtype;
  a.x = g.x;
  a.ldx = g.ldx;
  a.q_out = g.x_q;
  a.ldq_out = g.ldq;
  a.stop = quantized_stop(g.k, g.ldq);
  a.scale_out = g.x_scale;
  switch (g.dtype) {
    case RNS8_MI355X_F32: return launch<1, 1, 8, true, false, float>(a, stream);
    case RNS8_MI355X_F16: return launch<1, 1, 8, true, false, f16>(a, stream);
    case RNS8_MI355X_BF16: return launch<1, 1, 8, true, false, bf16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace rns8x
