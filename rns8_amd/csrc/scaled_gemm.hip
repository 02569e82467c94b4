// The product of 8-bit matrices with a scale for each row and each column
// (gfx950):
//   out[i][j] = a_scale[i] b_scale[j] sum_k a[i][k] b(k, j) + bias[j].
//
// 64 x 64 tiles, four waves; both operands are staged K-contiguous in LDS, 64
// of K at a time, and multiplied by v_mfma_i32_16x16x64_i8. Sums run in int32
// over blocks of 65536 K (|a b| <= 2^14: below 2^30) and are joined in 64 bits.
#include "elements.hpp"
#include "operators.hpp"

namespace rns8x {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

struct GemmI8Args {
  int64_t m, n, k;
  const int8_t *a, *b;
  int64_t lda, ldb;
  const float *a_scale, *b_scale, *bias;
  void* out;
  int64_t ldo;
  uint32_t tiles_n;
  uint32_t inner;
};

constexpr int kTile = 64, kStep = 64, kPitch = kStep + 16;

template <typename T>
__global__ __launch_bounds__(256) void gemm_i8_kernel(GemmI8Args g) {
  __shared__ __attribute__((aligned(16))) int8_t as[kTile * kPitch], bs[kTile * kPitch];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x / g.tiles_n) * kTile, n0 = static_cast<int64_t>(blockIdx.x % g.tiles_n) * kTile;
  int64_t total[4][4] = {};
  for (int64_t k0 = 0; k0 < g.k;) {
    const int64_t stop = k0 + 65536 < g.k ? k0 + 65536 : g.k;
    v4i acc[4] = {};
    for (; k0 < stop; k0 += kStep) {
      for (int e = threadIdx.x; e < kTile * kStep; e += 256) {
        const int r = e / kStep, c = e % kStep;
        const int64_t k = k0 + c;
        as[r * kPitch + c] = m0 + r < g.m && k < stop ? g.a[(m0 + r) * g.lda + k] : 0;
        if (!g.inner) bs[r * kPitch + c] = n0 + r < g.n && k < stop ? g.b[(n0 + r) * g.ldb + k] : 0;
        else bs[c * kPitch + r] = n0 + c < g.n && k0 + r < stop ? g.b[(k0 + r) * g.ldb + n0 + c] : 0;
      }
      __syncthreads();
      const v4i fa = *reinterpret_cast<const v4i*>(as + (16 * wave + (lane & 15)) * kPitch + 16 * (lane >> 4));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v4i fb = *reinterpret_cast<const v4i*>(bs + (16 * j + (lane & 15)) * kPitch + 16 * (lane >> 4));
        acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb, fa, acc[j], 0, 0, 0);
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) total[j][e] += acc[j][e];
  }
  const int64_t row = m0 + 16 * wave + (lane & 15);
  if (row >= g.m) return;
  const float sa = g.a_scale ? g.a_scale[row] : 1.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t col = n0 + 16 * j + 4 * (lane >> 4) + e;
      if (col >= g.n) continue;
      const float v = static_cast<float>(total[j][e]) * sa * (g.b_scale ? g.b_scale[col] : 1.0f);
      static_cast<T*>(g.out)[row * g.ldo + col] = static_cast<T>(v + (g.bias ? g.bias[col] : 0.0f));
    }
}

}  // namespace

uint64_t gemm_i8_bytes(const rns8_mi355x_gemm_i8_args&) { return 0; }

hipError_t launch_gemm_i8(const rns8_mi355x_gemm_i8_args& g, hipStream_t stream) {
  if (g.m == 0 || g.n == 0) return hipSuccess;
  const int64_t tiles_m = (g.m + kTile - 1) / kTile, tiles_n = (g.n + kTile - 1) / kTile;
  if (tiles_m > (int64_t{1} << 23) / tiles_n) return hipErrorInvalidValue;
  const GemmI8Args a{g.m, g.n, g.k, g.a, g.b, g.lda, g.ldb, g.a_scale, g.b_scale, g.bias, g.out, g.ldo,
                     static_cast<uint32_t>(tiles_n), g.b_layout == RNS8_MI355X_B_INNER};
  const dim3 grid(static_cast<unsigned>(tiles_m * tiles_n));
  switch (g.dtype) {
    case RNS8_MI355X_F32: hipLaunchKernelGGL(gemm_i8_kernel<float>, grid, dim3(256), 0, stream, a); break;
    case RNS8_MI355X_F16: hipLaunchKernelGGL(gemm_i8_kernel<f16>, grid, dim3(256), 0, stream, a); break;
    case RNS8_MI355X_BF16: hipLaunchKernelGGL(gemm_i8_kernel<bf16>, grid, dim3(256), 0, stream, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace rns8x
