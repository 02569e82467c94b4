// Log-probabilities of given tokens, entropy and top alternatives, and their
// gradient (gfx950).
//
// With z = scale * logit and a maximum m over the row:
//   S = sum exp(z - m),  W = sum exp(z - m) (z - m)
//   lse = m + log S,  logp = (z[target] - m) - log S,  entropy = log S - W / S
// S and W are kept for a running maximum: when it rises by d, S becomes
// S e^-d and W becomes (W - d S) e^-d, so one pass over the row is enough. The
// kernels are bound by reading the logits.
#include "elements.hpp"
#include "operators.hpp"
#include "row_shape.hpp"

namespace rns8x {
namespace {

constexpr int kThreads = 512;

// The sums of a part of a row. m = -infinity: nothing but ruled-out tokens yet.
struct Sums {
  float m, s, w;
};

__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return a.m != a.m || a.s != a.s ? a : b;
  const float da = a.m == -INFINITY ? 0.0f : a.m - m, db = b.m == -INFINITY ? 0.0f : b.m - m;
  const float ea = a.m == -INFINITY ? 0.0f : expf(da), eb = b.m == -INFINITY ? 0.0f : expf(db);
  // (a part without tokens has s = w = 0; a NaN stays in s. A part that the
  // maximum has left behind by more than floats hold adds nothing: its d s may
  // be infinite, as beside a mask of the type's lowest value)
  const float wa = ea > 0.0f ? (a.w + da * a.s) * ea : 0.0f, wb = eb > 0.0f ? (b.w + db * b.s) * eb : 0.0f;
  return {m, a.s * ea + b.s * eb, wa + wb};
}

struct Args {
  const void* logits;
  int64_t rows, vocab, ldl;
  const int64_t* targets;
  float scale;
  uint32_t top;
  float *logp, *entropy, *lse;
  int32_t* top_ids;
  float* top_logp;
};

// Order of the alternatives as one unsigned integer: the logit's order (NaNs
// above infinity, 0 and -0 equal) above the complement of the index.
__device__ __forceinline__ uint64_t rank_key(float z, uint32_t index) {
  const uint32_t b = as_uint(z + 0.0f);
  uint32_t order = b & 0x80000000u ? ~b : b | 0x80000000u;
  if (z != z) order = 0xFFFFFFFFu;
  return static_cast<uint64_t>(order) << 32 | static_cast<uint32_t>(~index);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Args a) {
  __shared__ Sums parts[kThreads / 64];
  __shared__ uint64_t keys[kThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const z = static_cast<const T*>(a.logits) + row * a.ldl;
    Sums t{-INFINITY, 0.0f, 0.0f};
    for (int64_t c = 8 * threadIdx.x; c < a.vocab; c += 8 * kThreads) {
      float v[8];
      load_upto8(z + c, a.vocab - c, v, -INFINITY);
      float m = t.m;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] *= a.scale;
        m = fmaxf(m, v[i]);
      }
      Sums u{m, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool out = v[i] == -INFINITY;
        const float d = out ? 0.0f : v[i] - m, e = out ? 0.0f : expf(d);
        u.s += e;
        u.w += e * d;
      }
      if (m != t.m) t = join({t.m, t.s, t.w}, {m, 0.0f, 0.0f});
      t.s += u.s;
      t.w += u.w;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const Sums o{__shfl_xor(t.m, d), __shfl_xor(t.s, d), __shfl_xor(t.w, d)};
      // (the same order of operands in both lanes: both get the same bits)
      t = lane & d ? join(o, t) : join(t, o);
    }
    if (lane == 0) parts[wave] = t;
    __syncthreads();
    t = parts[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) t = join(t, parts[w]);
    const float log_s = logf(t.s);
    const bool empty = t.m == -INFINITY && t.s == 0.0f;
    if (threadIdx.x == 0) {
      if (a.lse) a.lse[row] = empty ? -INFINITY : t.m + log_s;
      if (a.entropy) a.entropy[row] = empty ? 0.0f : log_s - t.w / t.s;
      if (a.logp) {
        const int64_t target = a.targets[row];
        const bool asked = target >= 0 && target < a.vocab;
        a.logp[row] = !asked ? 0.0f : empty ? -INFINITY : (static_cast<float>(z[target]) * a.scale - t.m) - log_s;
      }
    }
    // the alternatives, one pass for each
    uint64_t last = ~uint64_t{0};
    for (uint32_t k = 0; k < a.top; ++k) {
      uint64_t best = 0;
      for (int64_t c = threadIdx.x; c < a.vocab; c += kThreads) {
        const uint64_t key = rank_key(static_cast<float>(z[c]), static_cast<uint32_t>(c));
        if ((k == 0 || key < last) && key > best) best = key;
      }
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const uint64_t o = static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(best), d));
        best = best > o ? best : o;
      }
      if (lane == 0) keys[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kThreads / 64; ++w) best = best > keys[w] ? best : keys[w];
      __syncthreads();
      last = best;
      if (threadIdx.x == 0) {
        const uint32_t id = ~static_cast<uint32_t>(best);
        if (a.top_ids) a.top_ids[row * a.top + k] = static_cast<int32_t>(id);
        if (a.top_logp)
          a.top_logp[row * a.top + k] = empty ? -INFINITY : (static_cast<float>(z[id]) * a.scale - t.m) - log_s;
      }
    }
    __syncthreads();
  }
}

struct BackArgs {
  const void* logits;
  int64_t rows, vocab, ldl;
  const int64_t* targets;
  float scale;
  const float *lse, *entropy, *dlogp, *dentropy;
  void* dlogits;
  int64_t lddl;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_backward_kernel(BackArgs a) {
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const z = static_cast<const T*>(a.logits) + row * a.ldl;
    T* const out = static_cast<T*>(a.dlogits) + row * a.lddl;
    const float lse = a.lse[row];
    const int64_t target = a.dlogp ? a.targets[row] : -1;
    const bool asked = target >= 0 && target < a.vocab;
    const float gl = asked ? a.dlogp[row] : 0.0f;
    const float ge = a.dentropy ? a.dentropy[row] : 0.0f, entropy = a.dentropy ? a.entropy[row] : 0.0f;
    for (int64_t c = 8 * threadIdx.x; c < a.vocab; c += 8 * kThreads) {
      float v[8], d[8];
      load_upto8(z + c, a.vocab - c, v, -INFINITY);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool out_of = v[i] == -INFINITY;
        const float logp = out_of ? 0.0f : v[i] * a.scale - lse;
        const float p = out_of ? 0.0f : expf(logp);
        const float hit = asked && c + i == target ? 1.0f : 0.0f;
        d[i] = out_of ? 0.0f : a.scale * (gl * (hit - p) - (p == 0.0f ? 0.0f : ge * p * (logp + entropy)));
      }
      store_upto8(out + c, a.vocab - c, d);
    }
  }
}

dim3 grid_of(int64_t rows) { return dim3(static_cast<unsigned>(rows < kMaxBlocks ? rows : kMaxBlocks)); }

}  // namespace

uint64_t logprobs_bytes(const rns8_mi355x_logprobs_args&) { return 0; }

hipError_t launch_logprobs(const rns8_mi355x_logprobs_args& g, hipStream_t stream) {
  if (g.rows == 0) return hipSuccess;
  if (g.top > kMaxTop || g.vocab < 1 || g.vocab > 0x7FFFFFFF) return hipErrorInvalidValue;
  const bool wanted = g.top_ids || g.top_logp;
  const Args a{g.logits, g.rows, g.vocab, g.ldl, g.targets, g.scale, wanted ? g.top : 0u, g.logp, g.entropy, g.lse,
               g.top_ids, g.top_logp};
  switch (g.dtype) {
    case RNS8_MI355X_F32: hipLaunchKernelGGL(logprobs_kernel<float>, grid_of(g.rows), dim3(kThreads), 0, stream, a); break;
    case RNS8_MI355X_F16: hipLaunchKernelGGL(logprobs_kernel<f16>, grid_of(g.rows), dim3(kThreads), 0, stream, a); break;
    case RNS8_MI355X_BF16: hipLaunchKernelGGL(logprobs_kernel<bf16>, grid_of(g.rows), dim3(kThreads), 0, stream, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_logprobs_backward(const rns8_mi355x_logprobs_backward_args& g, hipStream_t stream) {
  if (g.rows == 0) return hipSuccess;
  const BackArgs a{g.logits, g.rows, g.vocab, g.ldl, g.targets, g.scale, g.lse, g.entropy, g.dlogp, g.dentropy,
                   g.dlogits, g.lddl};
  const dim3 grid = grid_of(g.rows), block(kThreads);
  switch (g.dtype) {
    case RNS8_MI355X_F32: hipLaunchKernelGGL(logprobs_backward_kernel<float>, grid, block, 0, stream, a); break;
    case RNS8_MI355X_F16: hipLaunchKernelGGL(logprobs_backward_kernel<f16>, grid, block, 0, stream, a); break;
    case RNS8_MI355X_BF16: hipLaunchKernelGGL(logprobs_backward_kernel<bf16>, grid, block, 0, stream, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace rns8x
