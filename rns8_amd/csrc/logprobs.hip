// Log-probabilities of given tokens, entropy and top alternatives, and their
// gradient (gfx950).
//
// With a maximum m over the row's logits, c = scale * log2(e) and d = c v - c m
// for each logit v:
//   S = sum 2^d,  W = sum 2^d d
//   lse = ln2 (c m + log2 S),  logp = ln2 (d[target] - log2 S),  entropy = ln2 (log2 S - W / S)
// S and W are kept for a running maximum: when c m rises by t, S becomes S 2^-t
// and W becomes (W - t S) 2^-t, so one pass over the row is enough. d is one
// fused multiply-add against the rounded c m, which is what lse starts from, so
// its error goes with its own size; where c m is so large that its rounding alone
// would be an exponent of its own (rows of nothing but a mask's value), v - m comes
// first instead. 32 bits hold every sum. Both kernels are bound by reading the logits (and writing
// their gradient): a logit costs about ten vector operations, the exponential
// counted as four, and the next loads are in flight beside them. bf16, 4096 x 32768
// 50 us (5.3 TB/s) and the gradient 84 (6.4 TB/s); f32, 1000 x 50001 with 5
// alternatives 43 us (4.6 TB/s); 4 x 131072 with 20 alternatives 7.5 and 4.9 for the
// join.
//
// Few long rows are cut into parts of 4096 logits or more, one workgroup each, whose
// sums and alternatives a second kernel joins: 4 rows of 131072 would occupy 4 of
// 256 CUs.
//
// Alternatives: the n-th largest of any n different threads' maxima is a lower
// bound of the part's n-th largest logit, so with 4 waves the least of the waves'
// ceil(n/4)-th largest lane maxima is one (in a part so short that not every wave
// has logits in all lanes: of the waves that do, which share n). Only threads whose maximum reaches it
// hold candidates: short parts keep their logits in registers for that look,
// longer ones read those threads' logits again (some tens of 256 threads). The
// candidates are ordered by counting; where too many are equal (a part of one
// value) the alternatives are taken one by one.
#include <algorithm>

#include "elements.hpp"
#include "operators.hpp"
#include "row_shape.hpp"

namespace rns8x {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kVector = 8;                     // logits of one load
constexpr int kStride = kThreads * kVector;    // logits of one round of a workgroup
constexpr int kHeldRounds = 4;                 // rounds that may stay in registers
constexpr int64_t kMaxParts = 64;              // a wave joins a row
constexpr uint32_t kMaxCandidates = 512;
constexpr float kLog2E = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The sums of a part of a row over its maximum m (a logit; -infinity: nothing
// but ruled-out tokens so far, s = w = 0). A NaN logit makes s NaN.
struct Sums {
  float m, s, w;
};

__device__ __forceinline__ bool is_empty(Sums t) { return t.m == -INFINITY && t.s == 0.0f; }

// d for a logit against the maximum m: c v - c m. Up to kFused the rounding of c m
// moves d by 2^-5 at most; beyond it that grows past any exponent (2^8 at 1e10),
// and c m may overflow: the difference comes first there, and the sums start from
// c m itself (m = -infinity: nothing but ruled-out tokens, d = -infinity).
constexpr float kFused = 0x1p20f;
__device__ __forceinline__ bool is_fused(float m, float c) { return fabsf(m * c) < kFused; }
__device__ __forceinline__ float exponent(float v, float m, float c) {
  if (is_fused(m, c)) return fmaf(v, c, -(m * c));
  return m == -INFINITY ? v : (v - m) * c;
}

// `a` for a maximum m >= a.m.
__device__ __forceinline__ Sums rescale(Sums a, float m, float c) {
  if (a.m == m || a.m == -INFINITY) return {m, a.s, a.w};
  const bool to_fused = is_fused(m, c);
  const float t = is_fused(a.m, c) ? (to_fused ? a.m * c - m * c : fmaf(-m, c, a.m * c))
                                   : (to_fused ? fmaf(a.m, c, -(m * c)) : (a.m - m) * c);
  const float e = exp2_fast(t);
  // (sums that the maximum has left behind by more than floats hold: t s may be infinite)
  return {m, a.s * e, e > 0.0f ? (a.w + t * a.s) * e : 0.0f};
}

struct MaxF {
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const {
    return as_uint(fmaxf(as_float(a), as_float(b)));
  }
};
__device__ __forceinline__ float wave_max(float x) { return as_float(wave_reduce(as_uint(x), MaxF{})); }
__device__ __forceinline__ float wave_sum(float x) { return as_float(wave_reduce(as_uint(x), AddF{})); }

__device__ __forceinline__ Sums wave_join(Sums t, float c) {
  t = rescale(t, wave_max(t.m), c);
  t.s = wave_sum(t.s);
  t.w = wave_sum(t.w);
  return t;
}

// The workgroup's sums from its waves'.
__device__ __forceinline__ Sums join_waves(const Sums* wave_sums, float c) {
  float m = wave_sums[0].m;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, wave_sums[w].m);
  Sums t = rescale(wave_sums[0], m, c);
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    const Sums u = rescale(wave_sums[w], m, c);
    t.s += u.s;
    t.w += u.w;
  }
  return t;
}

// Adds kCount logits. The decisions are the wave's, so that none of them costs
// more than a compare and a branch: a new maximum, a maximum past kFused, and
// ruled-out tokens, whose 2^d d is 0 times infinity: the chunk's own W is then
// NaN, its terms are taken again with d held above -200 (2^-200 is 0 in 32 bits,
// and so is its term), and so are those of the wave's later chunks at once
// (`held`: at first false).
template <int kCount>
__device__ __forceinline__ void add_logits(Sums& t, const float (&v)[kCount], float c, bool& held) {
  float m = t.m;
#pragma unroll
  for (int i = 0; i < kCount; ++i) m = fmaxf(m, v[i]);
  if (__any(m > t.m)) t = rescale(t, m, c);
  const float base = -(m * c);
  float s[2] = {0.0f, 0.0f}, w[2] = {0.0f, 0.0f};  // two chains of additions
  if (__any(!(fabsf(base) < kFused))) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const float d = exponent(v[i], m, c), e = exp2_fast(d);
      s[i & 1] += e;
      w[i & 1] = fmaf(e, fmaxf(d, -200.0f), w[i & 1]);
    }
  } else {
    if (!held) {
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        const float d = fmaf(v[i], c, base), e = exp2_fast(d);
        s[i & 1] += e;
        w[i & 1] = fmaf(e, d, w[i & 1]);
      }
      const float sum = w[0] + w[1];
      held = __any(sum != sum);
      if (held) s[0] = s[1] = w[0] = w[1] = 0.0f;
      if (!held) {
        t.s += s[0] + s[1];
        t.w += sum;
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const float d = fmaf(v[i], c, base), e = exp2_fast(d);
      s[i & 1] += e;
      w[i & 1] = fmaf(e, fmaxf(d, -200.0f), w[i & 1]);
    }
  }
  t.s += s[0] + s[1];
  t.w += w[0] + w[1];
}

// Order of the alternatives as one unsigned integer: the logit's order (NaNs
// above infinity, 0 and -0 equal) above the complement of the index. Neither 0 nor all ones.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t index) {
  const uint32_t b = as_uint(v + 0.0f);
  uint32_t order = b & 0x80000000u ? ~b : b | 0x80000000u;
  if (v != v) order = 0xFFFFFFFEu;
  return static_cast<uint64_t>(order) << 32 | static_cast<uint32_t>(~index);
}

// The logit that a key stands for (0 for -0, a NaN for any).
__device__ __forceinline__ float ranked_logit(uint64_t key) {
  const uint32_t order = static_cast<uint32_t>(key >> 32);
  return as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}

__device__ __forceinline__ uint64_t wave_max_key(uint64_t key) {
  const uint32_t hi = wave_reduce(static_cast<uint32_t>(key >> 32), MaxU{});
  const uint32_t lo = static_cast<uint32_t>(key >> 32) == hi ? static_cast<uint32_t>(key) : 0u;
  return static_cast<uint64_t>(hi) << 32 | wave_reduce(lo, MaxU{});
}

// How many of the keys come before `key` (eight loads in flight: one at a time, a
// list of 500 took 50 us).
__device__ __forceinline__ uint32_t rank_among(const uint64_t* keys, uint32_t n, uint64_t key) {
  uint32_t rank = 0;
#pragma unroll 8
  for (uint32_t j = 0; j < n; ++j) rank += keys[j] > key;
  return rank;
}

struct Args {
  const void* logits;
  int64_t rows, vocab, ldl;
  const int64_t* targets;
  float scale, c;
  uint32_t top;
  float *logp, *entropy, *lse;
  int32_t* top_ids;
  float* top_logp;
  int64_t parts, part_len;  // part_len: a multiple of 64 logits
  float* part_sums;         // [rows][parts][4]
  uint64_t* part_keys;      // [rows][parts][top]
};

// log(sum exp(scale (v - m))) from log_s = log2(S): the sums start from c m as it
// was rounded, this from m itself.
__device__ __forceinline__ float log_sum_over_max(Sums t, float c, float log_s) {
  return kLn2 * (is_fused(t.m, c) ? log_s - fmaf(t.m, c, -(t.m * c)) : log_s);
}
__device__ __forceinline__ float lse_of(Sums t, float scale, float c, float log_s) {
  const float over = log_sum_over_max(t, c, log_s);
  return t.m == -INFINITY ? over : fmaf(t.m, scale, over);  // rounded once where the maximum is the larger part
}

// The log-probability of a logit.
__device__ __forceinline__ float logp_of(float v, Sums t, float c) {
  return is_empty(t) ? -INFINITY : kLn2 * (exponent(v, t.m, c) - log2f(t.s));
}

// A row's results from its sums (one thread).
template <typename T>
__device__ __forceinline__ void write_row(const Args& a, int64_t row, Sums t) {
  const float log_s = log2f(t.s);
  if (a.lse) a.lse[row] = is_empty(t) ? -INFINITY : lse_of(t, a.scale, a.c, log_s);
  if (a.entropy) a.entropy[row] = is_empty(t) ? 0.0f : kLn2 * (log_s - t.w / t.s);
  if (a.logp) {
    const int64_t target = a.targets[row];
    const bool asked = target >= 0 && target < a.vocab;
    a.logp[row] = asked ? logp_of(static_cast<float>(static_cast<const T*>(a.logits)[row * a.ldl + target]), t, a.c) : 0.0f;
  }
}

__device__ __forceinline__ void write_alternative(const Args& a, int64_t row, uint32_t rank, uint64_t key, Sums t) {
  if (a.top_ids) a.top_ids[row * a.top + rank] = static_cast<int32_t>(~static_cast<uint32_t>(key));
  if (a.top_logp) a.top_logp[row * a.top + rank] = logp_of(ranked_logit(key), t, a.c);
}

template <typename T>
struct Held {
  T v[kVector];
};

// kRounds: rounds of a part held in registers (0: every part is read again for
// its alternatives, if any are asked for).
template <typename T, int kRounds>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(Args a) {
  __shared__ Sums wave_sums[kWaves];
  __shared__ float wave_least[kWaves];
  __shared__ uint64_t keys[kMaxCandidates];
  __shared__ uint32_t count, lane_count;
  __shared__ uint8_t lanes[kThreads];  // threads with candidates
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t unit = blockIdx.x; unit < a.rows * a.parts; unit += gridDim.x) {
    const int64_t row = unit / a.parts, part = unit - row * a.parts;
    const T* const z = static_cast<const T*>(a.logits) + row * a.ldl;
    const int64_t first = part * a.part_len, last = min(a.vocab, first + a.part_len);
    Sums t{-INFINITY, 0.0f, 0.0f};
    bool terms_held = false;
    constexpr int kHold = kRounds > 0 ? kRounds : 1;
    Held<T> held[kHold];
    auto load = [&](int64_t at, Held<T>& h) {
      if (at + kVector <= last) {
        __builtin_memcpy(h.v, z + at, sizeof(h.v));
      } else {
#pragma unroll
        for (int i = 0; i < kVector; ++i) h.v[i] = at + i < last ? z[at + i] : static_cast<T>(-INFINITY);
      }
    };
    auto floats = [&](const Held<T>& h, float (&v)[kVector]) {
#pragma unroll
      for (int i = 0; i < kVector; ++i) v[i] = static_cast<float>(h.v[i]);
    };
    float v[kVector];
    if constexpr (kRounds > 0) {
#pragma unroll
      for (int r = 0; r < kRounds; ++r) load(first + r * kStride + kVector * threadIdx.x, held[r]);
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        floats(held[r], v);
        add_logits(t, v, a.c, terms_held);
      }
    } else {
      // two vectors at a time, the next two in flight (the last are loaded twice)
      const int64_t at = first + kVector * threadIdx.x;
      const int64_t whole = last - at >= kVector ? (last - at - kVector) / kStride + 1 : 0;
      Held<T> x[2], y[2];
      auto load_pair = [&](int64_t i, Held<T> (&h)[2]) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          __builtin_memcpy(h[k].v, z + at + min(i + k, whole - 1) * kStride, sizeof(h[k].v));
      };
      auto add_pair = [&](int64_t i, const Held<T> (&h)[2]) {
        float u[2 * kVector];
#pragma unroll
        for (int k = 0; k < kVector; ++k) {
          u[k] = static_cast<float>(h[0].v[k]);
          u[kVector + k] = static_cast<float>(h[1].v[k]);
        }
        if (i + 1 >= whole) {  // the second was loaded twice
#pragma unroll
          for (int k = 0; k < kVector; ++k) u[kVector + k] = -INFINITY;
        }
        add_logits(t, u, a.c, terms_held);
      };
      if (whole > 0) {
        load_pair(0, x);
        for (int64_t i = 0; i < whole; i += 4) {
          load_pair(i + 2, y);
          add_pair(i, x);
          if (i + 2 >= whole) break;
          load_pair(i + 4, x);
          add_pair(i + 2, y);
        }
      }
      const int64_t rest = at + whole * kStride;
      if (rest < last) {  // the vector that the part's end cuts
        load(rest, held[0]);
        floats(held[0], v);
        add_logits(t, v, a.c, terms_held);
      }
    }
    const float lane_max = t.m;
    const bool lane_nan = t.s != t.s;  // a NaN among the lane's logits, which comes first
    t = wave_join(t, a.c);
    if (lane == 0) wave_sums[wave] = t;
    // waves with logits in every lane; without any, the part has few enough logits
    // for all of them to be candidates
    const uint32_t full = static_cast<uint32_t>(min<int64_t>((last - first) / (64 * kVector), kWaves));
    if (a.top && full) {
      float mine = lane_max, least = -INFINITY;
      for (uint32_t k = 0; k < (a.top + full - 1) / full; ++k) {
        least = wave_max(mine);
        const uint64_t who = __ballot(mine == least);
        if (lane == __ffsll(static_cast<unsigned long long>(who)) - 1) mine = -INFINITY;
      }
      if (lane == 0) wave_least[wave] = least;
    }
    if (threadIdx.x == 0) count = lane_count = 0;
    __syncthreads();
    t = join_waves(wave_sums, a.c);
    if (threadIdx.x == 0) {
      if (a.parts == 1) {
        write_row<T>(a, row, t);
      } else {
        const float w[4] = {t.m, t.s, t.w, 0.0f};
        __builtin_memcpy(a.part_sums + 4 * unit, w, 16);
      }
    }
    if (a.top) {
      float from = full ? wave_least[0] : -INFINITY;
#pragma unroll
      for (uint32_t w = 1; w < kWaves; ++w) from = w < full ? fminf(from, wave_least[w]) : from;
      auto gather = [&](int64_t at, const Held<T>& h) {
#pragma unroll
        for (int i = 0; i < kVector; ++i) {
          const float u = static_cast<float>(h.v[i]);
          if (!(u < from) && at + i < last) {
            const uint32_t slot = atomicAdd(&count, 1u);
            if (slot < kMaxCandidates) keys[slot] = rank_key(u, static_cast<uint32_t>(at + i));
          }
        }
      };
      const bool mine = !(lane_max < from) || lane_nan;
      const uint32_t rounds = static_cast<uint32_t>((last - first + kStride - 1) / kStride);
      // f on every vector of the threads with candidates
      auto each = [&](auto&& f) {
        if constexpr (kRounds > 0) {
          if (mine) {
#pragma unroll
            for (int r = 0; r < kRounds; ++r) f(first + r * kStride + kVector * threadIdx.x, held[r]);
          }
        } else {
          for (uint32_t i = threadIdx.x; i < lane_count * rounds; i += kThreads) {
            const uint32_t who = i / rounds;
            const int64_t at = first + static_cast<int64_t>(i - who * rounds) * kStride + kVector * lanes[who];
            if (at < last) {
              load(at, held[0]);
              f(at, held[0]);
            }
          }
        }
      };
      if constexpr (kRounds == 0) {
        if (mine) lanes[atomicAdd(&lane_count, 1u)] = static_cast<uint8_t>(threadIdx.x);
        __syncthreads();
      }
      each(gather);
      __syncthreads();
      auto put = [&](uint32_t rank, uint64_t key) {
        if (a.parts == 1)
          write_alternative(a, row, rank, key, t);
        else
          a.part_keys[unit * a.top + rank] = key;
      };
      const uint32_t n = count;
      if (n <= kMaxCandidates) {
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
          const uint64_t key = keys[i];
          const uint32_t rank = rank_among(keys, n, key);
          if (rank < a.top) put(rank, key);
        }
        // (a part shorter than `top`: its list ends in zeros, below every key)
        for (uint32_t i = n + threadIdx.x; i < a.top; i += kThreads) put(i, 0);
      } else {
        uint64_t before = ~uint64_t{0};
        for (uint32_t k = 0; k < a.top; ++k) {
          uint64_t best = 0;
          each([&](int64_t at, const Held<T>& h) {
#pragma unroll
            for (int i = 0; i < kVector; ++i) {
              const uint64_t key = rank_key(static_cast<float>(h.v[i]), static_cast<uint32_t>(at + i));
              if (at + i < last && key < before && key > best) best = key;
            }
          });
          best = wave_max_key(best);
          __syncthreads();  // (the last round's keys are read)
          if (lane == 0) keys[wave] = best;
          __syncthreads();
#pragma unroll
          for (int w = 0; w < kWaves; ++w) best = best > keys[w] ? best : keys[w];
          before = best;
          if (threadIdx.x == 0) put(k, best);
        }
      }
    }
    __syncthreads();  // the next unit writes the shared words
  }
}

// A workgroup loads a row's lists; its first wave joins the sums, lane p part p.
// The lists are in order: with each list's k-th key, k = ceil(top / parts), the
// ceil(top / k)-th largest of those has at least `top` keys at or above it. The keys
// from there on are gathered and ordered by counting, as within a part.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_parts_kernel(Args a) {
  __shared__ uint64_t keys[kMaxTop * kMaxTop];
  __shared__ uint64_t from;
  __shared__ uint32_t count;
  __shared__ Sums joined;
  const int lane = threadIdx.x & 63;
  const uint32_t parts = static_cast<uint32_t>(a.parts), total = parts * a.top;
  const uint32_t each = (a.top + parts - 1) / parts, enough = a.top ? (a.top + each - 1) / each : 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const uint64_t* const lists = a.part_keys + row * total;
    constexpr uint32_t kHeld = kMaxTop * kMaxTop / kThreads;  // 16: parts and top are at most 64
    uint64_t key[kHeld];
#pragma unroll
    for (uint32_t j = 0; j < kHeld; ++j) {
      key[j] = 0;
      if (j * kThreads < total) key[j] = lists[min(threadIdx.x + j * kThreads, total - 1)];
    }
    if (threadIdx.x < 64) {
      Sums t{-INFINITY, 0.0f, 0.0f};
      uint64_t head = 0;
      if (threadIdx.x < parts) {
        float w[4];
        __builtin_memcpy(w, a.part_sums + 4 * (row * a.parts + lane), 16);
        t = {w[0], w[1], w[2]};
        if (a.top) head = lists[lane * a.top + each - 1];
      }
      t = wave_join(t, a.c);
      if (lane == 0) {
        write_row<T>(a, row, t);
        joined = t;
        count = 0;
        from = 0;  // where lists end before their k-th key: every key
      }
      keys[lane] = head;
      __builtin_amdgcn_wave_barrier();
      if (head && rank_among(keys, parts, head) == enough - 1) from = head;
    }
    __syncthreads();
    if (a.top) {
      const uint64_t least = from;
      const Sums t = joined;
      __syncthreads();  // the heads are read
#pragma unroll
      for (uint32_t j = 0; j < kHeld; ++j)
        if (threadIdx.x + j * kThreads < total && key[j] >= least && key[j]) keys[atomicAdd(&count, 1u)] = key[j];
      __syncthreads();
      const uint32_t n = count;
      for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t mine = keys[i];
        const uint32_t rank = rank_among(keys, n, mine);
        if (rank < a.top) write_alternative(a, row, rank, mine, t);
      }
    }
    __syncthreads();  // the next row's shared words
  }
}

// ---- gradient --------------------------------------------------------------------------
// dlogit = -scale p (gl + ge (log p + entropy)), and scale gl more at the target,
// log p = scale v - lse. The rounding of lse to 32 bits is an error of every p of
// its row: up to kLargeLse 2^-19 of it at most, which is what the exponential of a
// log p of 20 is off by. Beyond (logits on a large common offset, rows of nothing
// but a mask's lowest value) the row's maximum and sum are computed again, and log p
// starts from the maximum, as in the forward pass: another read of the row by every
// workgroup that has a part of it (bf16, all rows such: 4096 x 32768 130 us for 84,
// 4 x 131072 in 32 parts 30 for 3; with the forward pass's four vectors in flight 119
// and 20, but 40 more registers, which cost f32 rows that need no such read 4%).
constexpr float kLargeLse = 64.0f;

struct BackArgs {
  const void* logits;
  int64_t rows, vocab, ldl;
  const int64_t* targets;
  float scale, c;
  const float *lse, *entropy, *dlogp, *dentropy;
  void* dlogits;
  int64_t lddl;
  int64_t parts, part_len;
  uint32_t streamed;  // stores pass the caches by
};

template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_backward_kernel(BackArgs a) {
  __shared__ Sums wave_sums[kWaves];
  for (int64_t unit = blockIdx.x; unit < a.rows * a.parts; unit += gridDim.x) {
    const int64_t row = unit / a.parts, part = unit - row * a.parts;
    const int64_t first = part * a.part_len, last = min(a.vocab, first + a.part_len);
    const T* const z = static_cast<const T*>(a.logits) + row * a.ldl;
    T* const out = static_cast<T*>(a.dlogits) + row * a.lddl;
    const int64_t target = a.dlogp ? a.targets[row] : -1;
    const bool asked = target >= 0 && target < a.vocab;
    const float gl = asked ? a.dlogp[row] : 0.0f;
    const float ge = a.dentropy ? a.dentropy[row] : 0.0f;
    const float rest = a.dentropy ? gl + ge * a.entropy[row] : gl;
    float from = 0.0f, log_s = a.lse[row];  // log p = scale (v - from) - log_s
    if (fabsf(log_s) > kLargeLse) {
      Sums t{-INFINITY, 0.0f, 0.0f};
      bool terms_held = false;
      for (int64_t at = kVector * threadIdx.x; at < a.vocab; at += kStride) {
        float v[kVector];
        load_upto8(z + at, a.vocab - at, v, -INFINITY);
        add_logits(t, v, a.c, terms_held);
      }
      t = wave_join(t, a.c);
      if ((threadIdx.x & 63) == 0) wave_sums[threadIdx.x >> 6] = t;
      __syncthreads();
      t = join_waves(wave_sums, a.c);
      // (where dlogits is logits: nothing is written before the whole row is read)
      __syncthreads();
      from = t.m == -INFINITY ? 0.0f : t.m;
      log_s = is_empty(t) ? 0.0f : log_sum_over_max(t, a.c, log2f(t.s));
    }
    auto grad = [&](int64_t at, float (&v)[kVector]) {
      float d[kVector];
#pragma unroll
      for (int i = 0; i < kVector; ++i) {
        const float logp = fmaf(v[i] - from, a.scale, -log_s), p = exp2_fast(logp * kLog2E);
        // (p is 0 in 32 bits below -104: its factor stays finite, also times a large ge)
        d[i] = -a.scale * p * fmaf(fmaxf(logp, -200.0f), ge, rest);
      }
      if (asked && static_cast<uint64_t>(target - at) < kVector) {
#pragma unroll
        for (int i = 0; i < kVector; ++i)
          if (at + i == target && v[i] != -INFINITY) d[i] += a.scale * gl;
      }
      if (a.streamed && at + kVector <= last)
        stream8(out + at, d);
      else
        store_upto8(out + at, last - at, d);
    };
    int64_t at = first + kVector * threadIdx.x;
    float v[kVector], w[kVector];
    for (; at + kStride + kVector <= last; at += 2 * kStride) {
      load8(z + at, v);
      load8(z + at + kStride, w);
      grad(at, v);
      grad(at + kStride, w);
    }
    for (; at < last; at += kStride) {
      load_upto8(z + at, last - at, v, -INFINITY);
      grad(at, v);
    }
  }
}

struct Cut {
  int64_t parts, len;
};

// A row in even parts, whole cache lines of whichever type.
Cut cut_row(int64_t vocab, int64_t parts) {
  const int64_t len = ((vocab + parts - 1) / parts + 63) / 64 * 64;
  return {(vocab + len - 1) / len, len};
}

// A second launch and its reads of what the first wrote cost 2 to 4 us. bf16, 20
// alternatives, one part against the number here: 4 rows of 131072 27 us and 12 (32
// parts), 64 rows 29 and 16 (8 parts), 16 rows of 50001 16 and 13; but 4 rows of
// 32768 12 both ways, and 400 rows of 100000 31 and 32 in two parts.
Cut forward_cut(int64_t rows, int64_t vocab) {
  if (vocab <= 32768) return cut_row(vocab, 1);
  return cut_row(vocab, std::max<int64_t>(1, std::min({512 / rows, vocab / 4096, kMaxParts})));
}

// The gradient: about 1024 workgroups, no fewer than two rounds each.
Cut backward_cut(int64_t rows, int64_t vocab) {
  const int64_t most = (vocab + 2 * kStride - 1) / (2 * kStride);
  return cut_row(vocab, std::max<int64_t>(1, std::min((1024 + rows - 1) / rows, most)));
}

dim3 grid_of(int64_t units) { return dim3(static_cast<unsigned>(std::min(units, kMaxBlocks))); }

template <typename T>
hipError_t launch_forward(const Args& a, hipStream_t stream) {
  const dim3 grid = grid_of(a.rows * a.parts), block(kThreads);
  const int64_t rounds = (a.part_len + kStride - 1) / kStride;
  if (a.top == 0 || rounds > kHeldRounds)
    hipLaunchKernelGGL((logprobs_kernel<T, 0>), grid, block, 0, stream, a);
  else if (rounds <= 1)
    hipLaunchKernelGGL((logprobs_kernel<T, 1>), grid, block, 0, stream, a);
  else if (rounds <= 2)
    hipLaunchKernelGGL((logprobs_kernel<T, 2>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((logprobs_kernel<T, kHeldRounds>), grid, block, 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.parts == 1) return e;
  hipLaunchKernelGGL((join_parts_kernel<T>), grid_of(a.rows), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
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

uint64_t logprobs_bytes(const rns8_mi355x_logprobs_args& g) {
  if (g.rows == 0) return 0;
  const int64_t parts = forward_cut(g.rows, g.vocab).parts;
  return parts == 1 ? 0u : static_cast<uint64_t>(g.rows) * static_cast<uint64_t>(parts) * (16u + 8u * g.top);
}

hipError_t launch_logprobs(const rns8_mi355x_logprobs_args& g, hipStream_t stream) {
  if (g.rows == 0) return hipSuccess;
  if (g.top > kMaxTop || g.vocab < 1 || g.vocab > 0x7FFFFFFF) return hipErrorInvalidValue;
  const Cut cut = forward_cut(g.rows, g.vocab);
  Args a{g.logits, g.rows, g.vocab, g.ldl, g.targets, g.scale, g.scale * kLog2E, g.top, g.logp, g.entropy, g.lse,
         g.top_ids, g.top_logp, cut.parts, cut.len, nullptr, nullptr};
  a.part_sums = static_cast<float*>(g.workspace);
  a.part_keys = reinterpret_cast<uint64_t*>(a.part_sums + 4 * g.rows * a.parts);
  return of_dtype(g.dtype, [&](auto t) { return launch_forward<decltype(t)>(a, stream); });
}

hipError_t launch_logprobs_backward(const rns8_mi355x_logprobs_backward_args& g, hipStream_t stream) {
  if (g.rows == 0) return hipSuccess;
  // in place a row's logits may be read twice: by the workgroup that writes them
  const Cut cut = g.dlogits == g.logits ? cut_row(g.vocab, 1) : backward_cut(g.rows, g.vocab);
  BackArgs a{g.logits, g.rows, g.vocab, g.ldl, g.targets, g.scale, g.scale * kLog2E, g.lse, g.entropy, g.dlogp,
             g.dentropy, g.dlogits, g.lddl, cut.parts, cut.len, 0};
  a.streamed = streams(2 * g.rows * g.vocab * (g.dtype == RNS8_MI355X_F32 ? 4 : 2), g.dlogits, g.lddl, g.dtype);
  return of_dtype(g.dtype, [&](auto t) {
    hipLaunchKernelGGL((logprobs_backward_kernel<decltype(t)>), grid_of(a.rows * a.parts), dim3(kThreads), 0, stream,
                       a);
    return hipGetLastError();
  });
}

}  // namespace rns8x
