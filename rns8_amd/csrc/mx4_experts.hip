// A mixture-of-experts layer for few tokens on MX4 weights (gfx950). Bound by
// reading the chosen experts' weights once.
//
// Four launches:
//   * stage: the router's scores, summed in 64 bits (two experts whose scores are next
//     to each other keep their order whatever the batch), and x as rows of bf16 parts
//     that add up to it exactly (bf16 1, half 2, float 3), zeros up to whole units;
//   * route: one workgroup chooses the experts and lists the (expert, token) pairs,
//     experts with a token first to last, each one's tokens in order;
//   * hidden: gate and up for 16 rows of one expert to a workgroup, its eight waves a
//     share of the width each; silu(gate) up times the token's weight goes to the
//     workspace, again as bf16 parts (two: 16 bits; float three);
//   * down: 16 channels to a workgroup, its waves a share of all experts' rows; a wave
//     adds an expert's result to its own table of tokens in LDS, the tables are added
//     in order.
// Weights go from HBM into registers as whole units, are turned to bf16 there (exact:
// v_cvt_scalef32_pk_bf16_fp4 applies the scale) and meet the tokens' parts in
// v_mfma_f32_16x16x32_bf16. The tokens of an expert are the MFMA's columns: an expert
// with few tokens costs few.
#include <algorithm>
#include <type_traits>

#include "mx4.hpp"
#include "mx4_mfma.hpp"
#include "operators.hpp"
#include "scaled_epilogue.hpp"

namespace rns8x {
namespace {

typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxPairs = kMaxExpertTokens * kMaxExpertTop;
constexpr int kMaxFrags = kMaxExpertTokens / 16;

// Who computes what: pairs sorted by expert, then token.
struct Routing {
  uint32_t active;  // experts with a token
  uint16_t expert[kMaxPairs], start[kMaxPairs + 1];  // of an active expert; its pairs are [start[i], start[i + 1])
  uint16_t token[kMaxPairs];
  float weight[kMaxPairs];
};

struct ExpertsArgs {
  const void *x, *router;
  int64_t ldx, ldrouter;
  const uint8_t *gate, *up, *down;
  void* out;
  int64_t ldo;
  int32_t* ids;
  float* weights;
  uint32_t tokens, experts, top, normalize, dtype;
  uint32_t width, inner, width_chunks, inner_chunks;
  float* scores;   // tokens x experts
  uint16_t* x_parts;  // [part][token][256 width_chunks]
  uint16_t* h_parts;  // [part][pair][256 inner_chunks]
  Routing* routing;
};

// v as bf16 parts whose sum is v to 8 kParts bits: its leading bits, then the leading
// bits of the rest (cut, not rounded: no part overflows).
template <int kParts>
__device__ __forceinline__ void split(float v, uint16_t (&part)[kParts]) {
  const bool finite = (as_uint(v) & 0x7F800000u) != 0x7F800000u;
  float rest = v;
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    const bool last = p == kParts - 1;
    const uint32_t cut = as_uint(rest) & 0xFFFF0000u;
    const bf16 rounded = static_cast<bf16>(rest);
    const uint16_t rounded_bits = __builtin_bit_cast(uint16_t, rounded);
    part[p] = !finite ? (p == 0 ? rounded_bits : uint16_t{0}) : last && p > 0 ? rounded_bits : static_cast<uint16_t>(cut >> 16);
    rest -= as_float(cut);
  }
}

// ---- stage ---------------------------------------------------------------------------------
constexpr int kScoreTokens = 8;

template <typename T, int kParts>
__global__ __launch_bounds__(256) void experts_stage_kernel(ExpertsArgs a, uint32_t score_blocks) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x < score_blocks) {
    const uint32_t per = (a.experts + 3) / 4;
    const uint32_t e = 4 * (blockIdx.x % per) + wave, t0 = kScoreTokens * (blockIdx.x / per);
    if (e >= a.experts) return;
    const T* const r = static_cast<const T*>(a.router) + e * a.ldrouter;
    const T* const x = static_cast<const T*>(a.x) + t0 * a.ldx;
    const uint32_t count = min(a.tokens - t0, static_cast<uint32_t>(kScoreTokens));
    double sum[kScoreTokens] = {};
    for (uint32_t c = 8 * lane; c < a.width; c += 512) {
      float w[8];
      load_upto8(r + c, a.width - c, w, 0.0f);
#pragma unroll
      for (uint32_t t = 0; t < kScoreTokens; ++t) {
        if (t >= count) break;
        float v[8];
        load_upto8(x + t * a.ldx + c, a.width - c, v, 0.0f);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[t] = fma(static_cast<double>(v[i]), static_cast<double>(w[i]), sum[t]);
      }
    }
#pragma unroll
    for (uint32_t t = 0; t < kScoreTokens; ++t) {
      if (t >= count) break;
#pragma unroll
      for (int step = 32; step >= 1; step /= 2) sum[t] += __shfl_xor(sum[t], step);
      if (lane == 0) a.scores[(t0 + t) * a.experts + e] = static_cast<float>(sum[t]);
    }
    return;
  }
  // x: 256 threads take eight values of a token each
  const uint32_t padded = 256 * a.width_chunks, per = (padded + 2047) / 2048;
  const uint32_t b = blockIdx.x - score_blocks, t = b / per, c = 2048 * (b % per) + 8 * threadIdx.x;
  if (t >= a.tokens || c >= padded) return;
  float v[8] = {};
  if (c < a.width) load_upto8(static_cast<const T*>(a.x) + t * a.ldx + c, a.width - c, v, 0.0f);
  uint16_t parts[8][kParts];
#pragma unroll
  for (int i = 0; i < 8; ++i) split<kParts>(v[i], parts[i]);
#pragma unroll
  for (int p = 0; p < kParts; ++p) {
    uint16_t out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = parts[i][p];
    __builtin_memcpy(a.x_parts + (static_cast<int64_t>(p) * a.tokens + t) * padded + c, out, 16);
  }
}

// ---- route -------------------------------------------------------------------------------------
constexpr int kRouteThreads = 512;

// Ordered as the scores are, NaN first.
__device__ __forceinline__ uint32_t score_key(float v) {
  const uint32_t bits = as_uint(v + 0.0f);  // (-0 is 0)
  if ((bits & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__global__ __launch_bounds__(kRouteThreads) void experts_route_kernel(ExpertsArgs a) {
  __shared__ uint32_t key[kMaxPairs];   // expert << 16 | pair, or ~0
  __shared__ float weight[kMaxPairs];
  __shared__ uint32_t sorted[kMaxPairs];
  __shared__ uint32_t firsts[kMaxPairs / 64 + 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t pairs = a.tokens * a.top;
  // each token's experts and weights
  if (a.router) {
    for (uint32_t t = wave; t < a.tokens; t += kRouteThreads / 64) {
      constexpr int kPer = kMaxExperts / 64;
      const float* const scores = a.scores + t * a.experts;
      uint32_t mine[kPer];
      float largest = 0.0f, total = 0.0f, chosen = 0.0f;
      uint32_t id = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) mine[i] = 64u * i + lane < a.experts ? score_key(scores[64 * i + lane]) : 0u;
      for (uint32_t s = 0; s < a.top; ++s) {
        uint32_t best = 0, at = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (mine[i] > best) {
            best = mine[i];
            at = 64u * i + lane;
          }
        const uint32_t top = wave_reduce(best, MaxU{});
        const uint32_t e = ~wave_reduce(best == top ? ~at : 0u, MaxU{});
        const float score = scores[e];
        if (s == 0) largest = score;
        if (lane == static_cast<int>(s)) {
          id = e;
          chosen = score;
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (64u * i + lane == e) mine[i] = 0;
      }
      const float p = static_cast<uint32_t>(lane) < a.top ? expf(chosen - largest) : 0.0f;
      if (a.normalize) {
        total = p;
      } else {
        for (uint32_t e = lane; e < a.experts; e += 64) total += expf(scores[e] - largest);
      }
      total = as_float(wave_reduce(as_uint(total), AddF{}));
      if (static_cast<uint32_t>(lane) < a.top) {
        const uint32_t pair = t * a.top + lane;
        key[pair] = id << 16 | pair;
        weight[pair] = p / total;
        if (a.ids) a.ids[pair] = static_cast<int32_t>(id);
        if (a.weights) a.weights[pair] = p / total;
      }
    }
  } else {
    for (uint32_t pair = threadIdx.x; pair < pairs; pair += kRouteThreads) {
      const int32_t id = a.ids[pair];
      const uint32_t first = pair - pair % a.top;
      bool counts = id >= 0 && id < static_cast<int32_t>(a.experts);
      float w = a.weights[pair];
      // an expert that the token has twice is one pair, the first
      for (uint32_t q = first; q < first + a.top; ++q) {
        if (q == pair || a.ids[q] != id) continue;
        counts = counts && q > pair;
        w += q > pair ? a.weights[q] : 0.0f;
      }
      key[pair] = counts ? static_cast<uint32_t>(id) << 16 | pair : 0xFFFFFFFFu;
      weight[pair] = w;
    }
  }
  __syncthreads();
  // sorted by counting the smaller keys
  for (uint32_t pair = threadIdx.x; pair < pairs; pair += kRouteThreads) {
    const uint32_t mine = key[pair];
    uint32_t rank = 0;
    for (uint32_t q = 0; q < pairs; ++q) rank += key[q] < mine || (key[q] == mine && q < pair);
    sorted[rank] = mine;
    if (mine != 0xFFFFFFFFu) {
      a.routing->token[rank] = static_cast<uint16_t>(pair / a.top);
      a.routing->weight[rank] = weight[pair];
    }
  }
  __syncthreads();
  // where experts begin
  const uint32_t rounds = (pairs + kRouteThreads - 1) / kRouteThreads;
  auto begins = [&](uint32_t r) {
    return r < pairs && sorted[r] != 0xFFFFFFFFu && (r == 0 || sorted[r - 1] >> 16 != sorted[r] >> 16);
  };
  for (uint32_t i = 0; i < rounds; ++i) {
    const uint32_t r = i * kRouteThreads + threadIdx.x;
    const uint64_t mask = __ballot(begins(r));
    if (lane == 0 && r / 64 < kMaxPairs / 64) firsts[r / 64] = static_cast<uint32_t>(__popcll(mask));
  }
  __syncthreads();
  for (uint32_t i = 0; i < rounds; ++i) {
    const uint32_t r = i * kRouteThreads + threadIdx.x;
    const uint64_t mask = __ballot(begins(r));
    uint32_t index = static_cast<uint32_t>(__popcll(mask & ((uint64_t{1} << lane) - 1)));
    for (uint32_t q = 0; q < r / 64; ++q) index += firsts[q];
    if (begins(r)) {
      a.routing->expert[index] = static_cast<uint16_t>(sorted[r] >> 16);
      a.routing->start[index] = static_cast<uint16_t>(r);
    }
  }
  if (threadIdx.x == 0) {
    uint32_t active = 0, count = 0;
    for (uint32_t q = 0; q < (pairs + 63) / 64; ++q) active += firsts[q];
    for (uint32_t q = 0; q < pairs; ++q) count += sorted[q] != 0xFFFFFFFFu;
    a.routing->active = active;
    a.routing->start[active] = static_cast<uint16_t>(count);
  }
}

// ---- products -----------------------------------------------------------------------------------
// A fragment's 32 codes of a lane's block as bf16: four operands of eight.
__device__ __forceinline__ void widen(i32x4 codes, uint32_t scale, bf16x8 (&w)[4]) {
  const float s = as_float(scale ? scale << 23 : 0x00400000u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t word = static_cast<uint32_t>(codes[i]);
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 0);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 2);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, s, 3);
    w[i] = bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
}

struct Quad {
  bf16x8 v[4];
};
// 32 values of a row of parts; zeros where there is no row.
__device__ __forceinline__ Quad load_quad(const uint16_t* p, bool there) {
  Quad q = {};
  if (there) {
#pragma unroll
    for (int i = 0; i < 4; ++i) q.v[i] = *reinterpret_cast<const bf16x8*>(p + 8 * i);
  }
  return q;
}

constexpr int kHiddenWaves = 8, kHiddenThreads = 64 * kHiddenWaves;

template <int kParts, int kHiddenParts>
__global__ __launch_bounds__(kHiddenThreads) void experts_hidden_kernel(ExpertsArgs a) {
  __shared__ __attribute__((aligned(16))) f32x4 sums[kHiddenWaves][2][kMaxFrags][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t groups = 16 * a.inner_chunks, real = (a.inner + 15) / 16;  // the last are zeros
  const uint32_t chunks = a.width_chunks, stride = chunks * kMx4Unit;
  const uint32_t first = chunks * wave / kHiddenWaves, last = chunks * (wave + 1) / kHiddenWaves;
  const int64_t x_part = static_cast<int64_t>(a.tokens) * 256 * chunks;
  const int64_t h_row = 256 * static_cast<int64_t>(a.inner_chunks), h_part = static_cast<int64_t>(a.tokens) * a.top * h_row;
  const uint32_t items = a.routing->active * groups;
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint32_t slot = item / groups, group = item - slot * groups;
    const uint32_t e = a.routing->expert[slot], start = a.routing->start[slot];
    const uint32_t count = a.routing->start[slot + 1] - start, frags = (count + 15) / 16;
    if (group < real) {
      const uint8_t* const gate = a.gate + (static_cast<uint64_t>(e) * real + group) * stride;
      const uint8_t* const up = a.up + (static_cast<uint64_t>(e) * real + group) * stride;
      const uint16_t* row[kMaxFrags];
      bool there[kMaxFrags];
#pragma unroll
      for (int f = 0; f < kMaxFrags; ++f) {
        const uint32_t r = 16 * f + (lane & 15);
        there[f] = r < count;
        row[f] = a.x_parts + static_cast<int64_t>(there[f] ? a.routing->token[start + r] : 0) * 256 * chunks;
      }
      f32x4 acc[2][kMaxFrags] = {};
      Mx4Unit g = {}, u = {};
      if (first < last) {
        g = load_unit(gate + first * kMx4Unit, lane);
        u = load_unit(up + first * kMx4Unit, lane);
      }
      for (uint32_t c = first; c < last; ++c) {
        const uint32_t ahead = min(c + 1, last - 1) * kMx4Unit;
        const Mx4Unit next_g = load_unit(gate + ahead, lane), next_u = load_unit(up + ahead, lane);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          bf16x8 wg[4], wu[4];
          widen(g.codes[h], g.scales >> (8 * h) & 0xFFu, wg);
          widen(u.codes[h], u.scales >> (8 * h) & 0xFFu, wu);
          const uint32_t k = 256 * c + 128 * h + 32 * (lane >> 4);
#pragma unroll
          for (int f = 0; f < kMaxFrags; ++f) {
            if (f >= static_cast<int>(frags)) break;
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
              const Quad q = load_quad(row[f] + p * x_part + k, there[f]);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                acc[0][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wg[i], q.v[i], acc[0][f], 0, 0, 0);
                acc[1][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wu[i], q.v[i], acc[1][f], 0, 0, 0);
              }
            }
          }
        }
        g = next_g;
        u = next_u;
      }
#pragma unroll
      for (int f = 0; f < kMaxFrags; ++f) {
        if (f >= static_cast<int>(frags)) break;
        sums[wave][0][f][lane] = acc[0][f];
        sums[wave][1][f][lane] = acc[1][f];
      }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 64 * frags; i += kHiddenThreads) {
      const uint32_t f = i / 64, l = i % 64, r = 16 * f + l % 16;
      if (r >= count) continue;
      f32x4 hidden = {0.0f, 0.0f, 0.0f, 0.0f};
      if (group < real) {
        f32x4 gv = sums[0][0][f][l], uv = sums[0][1][f][l];
#pragma unroll
        for (int w = 1; w < kHiddenWaves; ++w) {
          gv += sums[w][0][f][l];
          uv += sums[w][1][f][l];
        }
        const float weight = a.routing->weight[start + r];
#pragma unroll
        for (int v = 0; v < 4; ++v) hidden[v] = gv[v] / (1.0f + expf(-gv[v])) * uv[v] * weight;
      }
      uint16_t parts[4][kHiddenParts];
#pragma unroll
      for (int v = 0; v < 4; ++v) split<kHiddenParts>(hidden[v], parts[v]);
      uint16_t* const out = a.h_parts + (start + r) * h_row + 16 * group + 4 * (l / 16);
#pragma unroll
      for (int p = 0; p < kHiddenParts; ++p) {
        const uint16_t four[4] = {parts[0][p], parts[1][p], parts[2][p], parts[3][p]};
        __builtin_memcpy(out + p * h_part, four, 8);
      }
    }
    __syncthreads();
  }
}

constexpr int kDownWaves = 16, kDownThreads = 64 * kDownWaves;

template <int kHiddenParts, typename T>
__global__ __launch_bounds__(kDownThreads) void experts_down_kernel(ExpertsArgs a) {
  // [wave][token][16 channels]
  extern __shared__ __attribute__((aligned(16))) float table[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t chunks = a.inner_chunks, stride = chunks * kMx4Unit, groups = (a.width + 15) / 16;
  const uint32_t group = blockIdx.x, row = 16 * a.tokens;
  const int64_t h_row = 256 * static_cast<int64_t>(chunks), h_part = static_cast<int64_t>(a.tokens) * a.top * h_row;
  for (uint32_t i = threadIdx.x; i < kDownWaves * row; i += kDownThreads) table[i] = 0.0f;
  __syncthreads();
  const uint32_t units = a.routing->active * chunks;
  const uint32_t first = units * wave / kDownWaves, last = units * (wave + 1) / kDownWaves;
  auto unit_at = [&](uint32_t q) {
    const uint32_t slot = q / chunks, c = q - slot * chunks;
    return load_unit(a.down + (static_cast<uint64_t>(a.routing->expert[slot]) * groups + group) * stride + c * kMx4Unit, lane);
  };
  f32x4 acc[kMaxFrags] = {};
  Mx4Unit now = {};
  if (first < last) now = unit_at(first);
  for (uint32_t q = first; q < last; ++q) {
    const Mx4Unit next = unit_at(min(q + 1, last - 1));
    const uint32_t slot = q / chunks, c = q - slot * chunks;
    const uint32_t start = a.routing->start[slot], count = a.routing->start[slot + 1] - start, frags = (count + 15) / 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 w[4];
      widen(now.codes[h], now.scales >> (8 * h) & 0xFFu, w);
      const uint32_t k = 256 * c + 128 * h + 32 * (lane >> 4);
#pragma unroll
      for (int f = 0; f < kMaxFrags; ++f) {
        if (f >= static_cast<int>(frags)) break;
        const uint32_t r = 16 * f + (lane & 15);
#pragma unroll
        for (int p = 0; p < kHiddenParts; ++p) {
          const Quad v = load_quad(a.h_parts + p * h_part + (start + min(r, count - 1)) * h_row + k, r < count);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i], v.v[i], acc[f], 0, 0, 0);
        }
      }
    }
    if (c + 1 == chunks || q + 1 == last) {
      // the expert's share of its tokens (no token is twice in the list)
#pragma unroll
      for (int f = 0; f < kMaxFrags; ++f) {
        if (f >= static_cast<int>(frags)) break;
        const uint32_t r = 16 * f + (lane & 15);
        if (r < count) {
          f32x4* const at = reinterpret_cast<f32x4*>(table + wave * row + 16 * a.routing->token[start + r] + 4 * (lane >> 4));
          *at += acc[f];
        }
        acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    }
    now = next;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < row / 4; i += kDownThreads) {
    const uint32_t t = i / 4, channel = 16 * group + 4 * (i % 4);
    f32x4 sum = *reinterpret_cast<const f32x4*>(table + 4 * i);
#pragma unroll
    for (int w = 1; w < kDownWaves; ++w) sum += *reinterpret_cast<const f32x4*>(table + w * row + 4 * i);
    const float v[4] = {sum[0], sum[1], sum[2], sum[3]};
    if (channel < a.width) store4(static_cast<T*>(a.out) + t * a.ldo + channel, static_cast<int64_t>(a.width) - channel, v);
  }
}

int parts_of(uint32_t dtype) { return dtype == RNS8_MI355X_F32 ? 3 : dtype == RNS8_MI355X_F16 ? 2 : 1; }
int hidden_parts_of(uint32_t dtype) { return dtype == RNS8_MI355X_F32 ? 3 : 2; }

// The workspace: scores, the parts of x and of the hidden values, the lists.
uint64_t lay_out(const rns8_mi355x_experts_mx4_args& a, ExpertsArgs& e) {
  uint8_t* const at = static_cast<uint8_t*>(a.workspace);
  uint64_t bytes = 0;
  auto take = [&](uint64_t size) {
    uint8_t* const got = at ? at + bytes : nullptr;
    bytes += round_up(size, 256);
    return got;
  };
  const uint64_t tokens = static_cast<uint64_t>(a.tokens);
  e.scores = reinterpret_cast<float*>(take(a.router ? tokens * static_cast<uint64_t>(a.experts) * sizeof(float) : 0));
  e.x_parts = reinterpret_cast<uint16_t*>(
      take(static_cast<uint64_t>(parts_of(a.dtype)) * tokens * static_cast<uint64_t>(mx4_chunks(a.width)) * 512));
  e.h_parts = reinterpret_cast<uint16_t*>(
      take(static_cast<uint64_t>(hidden_parts_of(a.dtype)) * tokens * a.top * static_cast<uint64_t>(mx4_chunks(a.inner)) * 512));
  e.routing = reinterpret_cast<Routing*>(take(sizeof(Routing)));
  return bytes;
}

template <typename T, int kParts, int kHiddenParts>
hipError_t launch_typed(const ExpertsArgs& e, hipStream_t stream) {
  const uint32_t score_blocks = e.router ? (e.experts + 3) / 4 * ((e.tokens + kScoreTokens - 1) / kScoreTokens) : 0;
  const uint32_t x_blocks = e.tokens * ((256 * e.width_chunks + 2047) / 2048);
  hipLaunchKernelGGL((experts_stage_kernel<T, kParts>), dim3(score_blocks + x_blocks), dim3(256), 0, stream, e, score_blocks);
  hipLaunchKernelGGL(experts_route_kernel, dim3(1), dim3(kRouteThreads), 0, stream, e);
  const uint32_t most = std::min(e.experts, e.tokens * e.top) * 16 * e.inner_chunks;
  hipLaunchKernelGGL((experts_hidden_kernel<kParts, kHiddenParts>), dim3(std::min(most, 256u * 8)), dim3(kHiddenThreads), 0,
                     stream, e);
  hipLaunchKernelGGL((experts_down_kernel<kHiddenParts, T>), dim3((e.width + 15) / 16), dim3(kDownThreads),
                     kDownWaves * 16 * e.tokens * sizeof(float), stream, e);
  return hipGetLastError();
}

}  // namespace

uint64_t experts_mx4_bytes(const rns8_mi355x_experts_mx4_args& a) {
  if (a.tokens == 0) return 0;
  rns8_mi355x_experts_mx4_args sizes = a;
  sizes.workspace = nullptr;
  ExpertsArgs e{};
  return lay_out(sizes, e);
}

hipError_t launch_experts_mx4(const rns8_mi355x_experts_mx4_args& a, hipStream_t stream) {
  if (a.tokens == 0) return hipSuccess;
  if (a.tokens < 0 || a.tokens > kMaxExpertTokens || a.experts < 1 || a.experts > kMaxExperts || a.top < 1 ||
      a.top > kMaxExpertTop || a.width < 1 || a.width > kMaxExpertSize || a.inner < 1 || a.inner > kMaxExpertSize ||
      a.dtype > RNS8_MI355X_BF16)
    return hipErrorInvalidValue;
  ExpertsArgs e{};
  e.x = a.x;
  e.ldx = a.ldx;
  e.router = a.router;
  e.ldrouter = a.ldrouter;
  e.gate = a.gate;
  e.up = a.up;
  e.down = a.down;
  e.out = a.out;
  e.ldo = a.ldo;
  e.ids = a.ids;
  e.weights = a.weights;
  e.tokens = static_cast<uint32_t>(a.tokens);
  e.experts = static_cast<uint32_t>(a.experts);
  e.top = a.top;
  e.normalize = a.flags & RNS8_MI355X_EXPERTS_NORMALIZE;
  e.dtype = a.dtype;
  e.width = static_cast<uint32_t>(a.width);
  e.inner = static_cast<uint32_t>(a.inner);
  e.width_chunks = static_cast<uint32_t>(mx4_chunks(a.width));
  e.inner_chunks = static_cast<uint32_t>(mx4_chunks(a.inner));
  lay_out(a, e);
  if (a.dtype == RNS8_MI355X_F32) return launch_typed<float, 3, 3>(e, stream);
  if (a.dtype == RNS8_MI355X_F16) return launch_typed<f16, 2, 2>(e, stream);
  return launch_typed<bf16, 1, 2>(e, stream);
}

}  // namespace rns8x
