// A mixture-of-experts layer for few tokens on MX4 weights (gfx950). Bound by
// reading the chosen experts' weights once.
//
//   * stage: the router's scores, summed in 64 bits (two experts whose scores are next
//     to each other keep their order whatever the batch), and x as rows of bf16 parts
//     that add up to it exactly (bf16 1, half 2, float 3), zeros up to whole units.
//   * hidden: every workgroup lists the (expert, token) pairs for itself (in LDS: less than
//     a launch), experts with a token first to last, each one's tokens in order; of few
//     tokens it also chooses the experts. Then 16 rows of one expert's gate and up at a
//     time; silu(gate) up times the token's weight goes to the workspace, again as bf16
//     parts: three, the 24 bits of the 32-bit value.
//   * down, few pairs: 16 channels to a workgroup, its waves a share of all experts' rows,
//     the hidden values in LDS; a wave adds an expert's result to its own table of
//     tokens, the tables are added in order. Three launches.
//   * down, many pairs: 32 channels of one expert at a time, and its tokens' results go to
//     the workspace; a last kernel adds each token's, by its slots. Five launches with the
//     choice.
// Weights go from HBM into registers as whole units, are turned to bf16 there (exact:
// v_cvt_scalef32_pk_bf16_fp4 applies the scale) and meet the tokens' parts in
// v_mfma_f32_16x16x32_bf16. The tokens of an expert are the MFMA's columns: an expert
// with few tokens costs few. Sixteen rows are one wave's where there are many, and
// otherwise eight waves', each with a share of the sum. Loads return in order, and who
// waits for tokens from memory has waited for all weights asked for before: tokens lie
// in LDS, so that a wave always has the next units' weights in flight.
// Measured (1 token, 8 of 128 experts, 4096 -> 1536, bf16): stage 2.7 us, hidden 14.0
// (3.8 TB/s; some 4 of them before the first weights: lists and tokens), down 10.5 (2.5),
// on the same 80 MB again and again; hidden 14.8 and down 11.1 where other experts are chosen each
// time and their weights come from HBM.
#include <algorithm>
#include <cstddef>
#include <type_traits>

#include "mx4.hpp"
#include "mx4_mfma.hpp"
#include "operators.hpp"
#include "scaled_epilogue.hpp"

namespace rns8x {
namespace {

typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxPairs = kMaxExpertTokens * kMaxExpertTop;

// Who computes what: pairs sorted by expert, then token.
struct Routing {
  uint32_t active;      // experts with a token
  uint32_t batches[2];  // of all experts' tokens (hidden, down); many pairs
  uint16_t expert[kMaxPairs], start[kMaxPairs + 2];  // of an active expert; its pairs are [start[i], start[i + 1])
  uint16_t token[kMaxPairs];  // of a pair
  uint16_t place[kMaxPairs];  // of a token's slot: its pair, or kNone
  float weight[kMaxPairs];
};
constexpr uint32_t kNone = 0xFFFF;

// Many pairs: what LDS holds of an expert's tokens, `tokens` rows of `chunks` chunks (16
// bytes after each, so that sixteen rows' reads meet no bank twice). inverse: 2^16 /
// tokens and one.
struct Batches {
  uint32_t chunks, row, tokens, inverse;
};
// Whose a batch is: an index among the active experts and, in the low bits, its number
// among that one's.
constexpr uint32_t kBatchBits = 6;
static_assert(kMaxExpertTokens <= 1 << kBatchBits && kMaxExperts << kBatchBits <= 1 << 16, "an owner in 16 bits");


struct ExpertsArgs {
  const void *x, *router;
  int64_t ldx, ldrouter;
  const uint8_t *gate, *up, *down;
  void* out;
  int64_t ldo;
  int32_t* ids;
  float* weights;
  uint32_t tokens, experts, top, normalize;
  uint32_t width, inner, width_chunks, inner_chunks;
  int32_t* chosen;        // tokens x top: the caller's, or the choice where there are many pairs
  float* chosen_weights;
  float* scores;      // tokens x experts
  uint16_t* x_parts;  // [part][token][256 width_chunks]
  uint16_t* h_parts;  // [part][pair][256 inner_chunks]
  float* y;           // [pair][16 ceil(width / 16)]; many pairs
  Routing* routing;
  uint16_t* down_owner;  // of each of down's batches; many pairs
  Batches batches[2];  // hidden, down; many pairs
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
// The sum over a wave's lanes, in every lane.
template <int kCtrl>
__device__ __forceinline__ double add_moved(double x) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = dpp_move<kCtrl>(static_cast<uint32_t>(bits)), hi = dpp_move<kCtrl>(static_cast<uint32_t>(bits >> 32));
  return x + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double x) {
  x = add_moved<kRowRotate + 8>(x);
  x = add_moved<kRowRotate + 4>(x);
  x = add_moved<kRowRotate + 2>(x);
  x = add_moved<kRowRotate + 1>(x);
  auto swapped = [&](auto swap) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, x);
    const auto lo = swap(static_cast<uint32_t>(bits)), hi = swap(static_cast<uint32_t>(bits >> 32));
    x = __builtin_bit_cast(double, static_cast<uint64_t>(hi[0]) << 32 | lo[0]) +
        __builtin_bit_cast(double, static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
  };
  swapped([](uint32_t v) { return __builtin_amdgcn_permlane16_swap(v, v, false, false); });
  swapped([](uint32_t v) { return __builtin_amdgcn_permlane32_swap(v, v, false, false); });
  return x;
}

// Eight elements from column c on of a row of at least eight, zeros past its end.
template <typename T>
__device__ __forceinline__ Packed8<T> load_cut(const T* row, int32_t c, int32_t width) {
  Packed8<T> q;
  const int32_t at = min(c, width - 8);
  __builtin_memcpy(q.q, row + at, sizeof(q.q));
  if (c + 8 > width) {
    if (c < width)
      q.drop(static_cast<uint32_t>(c - at));
    else
      q.fill(static_cast<T>(0.0f));
  }
  return q;
}

// A workgroup takes the scores of kExperts experts and kTokens tokens, or 2048 values of
// a token of x.
template <typename T, int kParts, int kExperts, int kTokens>
__global__ __launch_bounds__(256) void experts_stage_kernel(ExpertsArgs a, uint32_t score_blocks) {
  __shared__ double sums[4][kExperts * kTokens];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x < score_blocks) {
    const uint32_t per = (a.experts + kExperts - 1) / kExperts;
    const uint32_t e0 = kExperts * (blockIdx.x % per), t0 = kTokens * (blockIdx.x / per);
    // (rows past the last read it again; their scores are not stored)
    const T *r[kExperts], *x[kTokens];
#pragma unroll
    for (uint32_t e = 0; e < kExperts; ++e) r[e] = static_cast<const T*>(a.router) + min(e0 + e, a.experts - 1) * a.ldrouter;
#pragma unroll
    for (uint32_t t = 0; t < kTokens; ++t) x[t] = static_cast<const T*>(a.x) + min(t0 + t, a.tokens - 1) * a.ldx;
    const int32_t width = static_cast<int32_t>(a.width);
    double sum[kExperts][kTokens] = {};
    constexpr int U = kTokens == 1 ? 2 : 1;  // loads in flight together
    for (int32_t c = 8 * threadIdx.x; c < width && width >= 8; c += 2048 * U) {
      Packed8<T> w[U][kExperts], v[U][kTokens];
#pragma unroll
      for (int i = 0; i < U; ++i) {
#pragma unroll
        for (int e = 0; e < kExperts; ++e) w[i][e] = load_cut(r[e], c + 2048 * i, width);
#pragma unroll
        for (int t = 0; t < kTokens; ++t) v[i][t] = load_cut(x[t], c + 2048 * i, width);
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          double we[kExperts];
#pragma unroll
          for (int e = 0; e < kExperts; ++e) we[e] = static_cast<double>(w[i][e].at(k));
#pragma unroll
          for (int t = 0; t < kTokens; ++t) {
            const double vt = static_cast<double>(v[i][t].at(k));
#pragma unroll
            for (int e = 0; e < kExperts; ++e) sum[e][t] = fma(we[e], vt, sum[e][t]);
          }
        }
    }
    if (width < 8 && static_cast<int32_t>(threadIdx.x) < width) {
#pragma unroll
      for (int e = 0; e < kExperts; ++e)
#pragma unroll
        for (int t = 0; t < kTokens; ++t)
          sum[e][t] = static_cast<double>(static_cast<float>(r[e][threadIdx.x])) * static_cast<double>(static_cast<float>(x[t][threadIdx.x]));
    }
#pragma unroll
    for (int e = 0; e < kExperts; ++e)
#pragma unroll
      for (int t = 0; t < kTokens; ++t) {
        const double all = wave_sum(sum[e][t]);
        if (lane == 0) sums[wave][e * kTokens + t] = all;
      }
    __syncthreads();
    if (threadIdx.x < kExperts * kTokens) {
      const uint32_t i = threadIdx.x, e = e0 + i / kTokens, t = t0 + i % kTokens;
      if (e < a.experts && t < a.tokens)
        a.scores[t * a.experts + e] = static_cast<float>((sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]));
    }
    return;
  }
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

// ---- choice of experts --------------------------------------------------------------------------
constexpr int kRouteThreads = 512, kRouteWaves = kRouteThreads / 64;

struct RouteScratch {
  uint16_t id[kMaxPairs];  // of a token's slot, or kNone
  float weight[kMaxPairs];
  uint32_t tokens[2][kMaxExperts];  // an expert's tokens, a bit each
  uint16_t start[kMaxExperts];
  uint32_t totals[kRouteWaves], batches[kRouteWaves];
};

// Ordered as the scores are, NaN first.
__device__ __forceinline__ uint32_t score_key(float v) {
  const uint32_t bits = as_uint(v + 0.0f);  // (-0 is 0)
  if ((bits & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ float score_of(uint32_t key) {
  return as_float(key == 0xFFFFFFFFu ? 0x7FC00000u : key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// A wave's choice for one token of at most 64 kPer experts, the largest left `top` times:
// put(slot, expert, weight) by the lanes that hold them.
template <int kPer, typename Put>
__device__ __forceinline__ void choose_of(const ExpertsArgs& a, uint32_t t, int lane, Put&& put) {
  const float* const scores = a.scores + t * a.experts;
  float score[kPer];
  uint32_t key[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t e = 64u * i + lane;
    score[i] = e < a.experts ? scores[e] : 0.0f;
    key[i] = e < a.experts ? score_key(score[i]) : 0u;
  }
  float largest = 0.0f, chosen = 0.0f;
  uint32_t id = 0;
  for (uint32_t n = 0; n < a.top; ++n) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
    const uint32_t top = wave_reduce(best, MaxU{});
    // the first of those that have it
    uint32_t e = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint64_t has = __ballot(key[i] == top);
      const bool here = !found && has != 0;
      e = here ? 64u * i + static_cast<uint32_t>(__builtin_ctzll(has)) : e;
      if (here && static_cast<uint32_t>(lane) == (e & 63u)) key[i] = 0;
      found = found || here;
    }
    const float value = score_of(top);
    if (n == 0) largest = value;
    if (lane == static_cast<int>(n)) {
      id = e;
      chosen = value;
    }
  }
  const bool holds = static_cast<uint32_t>(lane) < a.top;
  const float p = holds ? expf(chosen - largest) : 0.0f;
  float total = p;
  if (!a.normalize) {
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (64u * i + lane < a.experts) total += expf(score[i] - largest);
  }
  total = as_float(wave_reduce(as_uint(total), AddF{}));
  if (holds) put(static_cast<uint32_t>(lane), id, p / total);
}
template <typename Put>
__device__ __forceinline__ void choose(const ExpertsArgs& a, uint32_t t, int lane, Put&& put) {
  if (a.experts <= 128)
    choose_of<2>(a, t, lane, put);
  else if (a.experts <= 256)
    choose_of<4>(a, t, lane, put);
  else
    choose_of<kMaxExperts / 64>(a, t, lane, put);
}

// The choice alone, a token to a workgroup: where there are many, each workgroup of the
// next kernel would choose for eight tokens to a wave (64 tokens, 8 of 128: 27 us).
__global__ __launch_bounds__(64) void experts_choose_kernel(ExpertsArgs a) {
  const uint32_t t = blockIdx.x;
  choose(a, t, threadIdx.x, [&](uint32_t slot, uint32_t id, float weight) {
    const uint32_t pair = t * a.top + slot;
    a.chosen[pair] = static_cast<int32_t>(id);
    a.chosen_weights[pair] = weight;
    if (a.ids) a.ids[pair] = static_cast<int32_t>(id);
    if (a.weights) a.weights[pair] = weight;
  });
}

// The lists of at most 64 pairs, in LDS: one wave's work, a pair to a lane.
__device__ __forceinline__ void list_few(const ExpertsArgs& a, int lane, uint32_t id, float weight, Routing& r) {
  const uint32_t pairs = a.tokens * a.top, token = lane / a.top;
  const bool live = static_cast<uint32_t>(lane) < pairs;
  auto pair_id = [&](uint32_t q) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(id), static_cast<int>(q))); };
  // an expert that a token has twice is one pair, the first, with both weights
  bool counts = live && id != kNone;
  if (!a.router) {
    const uint32_t first = token * a.top, end = first + a.top;
    for (uint32_t q = 0; q < pairs; ++q) {
      const bool same = counts && pair_id(q) == id && q >= first && q < end;
      const float other = as_float(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(as_uint(weight)), static_cast<int>(q))));
      if (same && q > static_cast<uint32_t>(lane)) weight += other;
      if (same && q < static_cast<uint32_t>(lane)) counts = false;
    }
  }
  const uint64_t counted = __ballot(counts);
  const uint32_t key = counts ? id << 6 | lane : 0xFFFFFFFFu;  // (1024 experts, 64 pairs)
  uint32_t rank = 0, same_before = 0;
  for (uint32_t q = 0; q < pairs; ++q) {
    const uint32_t other = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(key), static_cast<int>(q)));
    rank += other < key;
    same_before += other < key && other >> 6 == id;
  }
  const uint64_t firsts = __ballot(counts && same_before == 0);
  // the experts before: the first pairs with a smaller key, whose ids are smaller then
  uint32_t index = 0;
  for (uint64_t left = firsts; left; left &= left - 1)
    index += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(key), __builtin_ctzll(left))) < key;
  if (counts) {
    r.token[rank] = static_cast<uint16_t>(token);
    r.weight[rank] = weight;
    if (same_before == 0) {
      r.expert[index] = static_cast<uint16_t>(id);
      r.start[index] = static_cast<uint16_t>(rank);
    }
  }
  if (live) r.place[lane] = static_cast<uint16_t>(counts ? rank : kNone);
  if (lane == 0) {
    r.active = static_cast<uint32_t>(__popcll(firsts));
    r.start[__popcll(firsts)] = static_cast<uint16_t>(__popcll(counted));
  }
}

// The lists, in LDS; all kRouteThreads threads. writes: this workgroup gives the
// next kernels the lists, and the caller its experts and weights where they are chosen
// here (kChooses: few pairs; otherwise `owner` receives the owners of hidden's batches).
template <bool kChooses>
__device__ __forceinline__ void route(const ExpertsArgs& a, bool writes, RouteScratch& s, Routing& r, uint16_t* owner) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t pairs = a.tokens * a.top, tid = threadIdx.x;
  auto give = [&]() {
    if (writes)
      for (uint32_t i = tid; i < sizeof(Routing) / 4; i += kRouteThreads)
        reinterpret_cast<uint32_t*>(a.routing)[i] = reinterpret_cast<const uint32_t*>(&r)[i];
  };
  if (kChooses && pairs <= 64) {
    if (a.router) {
      for (uint32_t t = wave; t < a.tokens; t += kRouteWaves)
        choose(a, t, lane, [&](uint32_t slot, uint32_t id, float weight) {
          const uint32_t pair = t * a.top + slot;
          s.id[pair] = static_cast<uint16_t>(id);
          s.weight[pair] = weight;
          if (writes && a.ids) a.ids[pair] = static_cast<int32_t>(id);
          if (writes && a.weights) a.weights[pair] = weight;
        });
      if (a.tokens > 1) __syncthreads();
    }
    if (wave == 0) {
      uint32_t id = kNone;
      float weight = 0.0f;
      if (static_cast<uint32_t>(lane) < pairs) {
        if (a.router) {
          id = s.id[lane];
          weight = s.weight[lane];
        } else {
          const int32_t given = a.chosen[lane];
          id = given >= 0 && given < static_cast<int32_t>(a.experts) ? static_cast<uint32_t>(given) : kNone;
          weight = a.chosen_weights[lane];
        }
      }
      list_few(a, lane, id, weight, r);
    }
    __syncthreads();
    give();
    return;
  }
  for (uint32_t e = tid; e < a.experts; e += kRouteThreads) s.tokens[0][e] = s.tokens[1][e] = 0;
  if (kChooses && a.router) {
    for (uint32_t t = wave; t < a.tokens; t += kRouteWaves)
      choose(a, t, lane, [&](uint32_t slot, uint32_t id, float weight) {
        const uint32_t pair = t * a.top + slot;
        s.id[pair] = static_cast<uint16_t>(id);
        s.weight[pair] = weight;
        if (writes && a.ids) a.ids[pair] = static_cast<int32_t>(id);
        if (writes && a.weights) a.weights[pair] = weight;
      });
  } else {
    for (uint32_t pair = tid; pair < pairs; pair += kRouteThreads) {
      const int32_t id = a.chosen[pair];
      s.id[pair] = id >= 0 && id < static_cast<int32_t>(a.experts) ? static_cast<uint16_t>(id) : static_cast<uint16_t>(kNone);
      s.weight[pair] = a.chosen_weights[pair];
    }
    if (!a.router) {
      // an expert that a token has twice is one pair, the first, with both weights
      __syncthreads();
      for (uint32_t t = tid; t < a.tokens; t += kRouteThreads)
        for (uint32_t n = t * a.top; n < (t + 1) * a.top; ++n)
          for (uint32_t q = t * a.top; q < n; ++q)
            if (s.id[q] == s.id[n] && s.id[n] != kNone) {
              s.weight[q] += s.weight[n];
              s.id[n] = static_cast<uint16_t>(kNone);
            }
    }
  }
  __syncthreads();
  for (uint32_t pair = tid; pair < pairs; pair += kRouteThreads) {
    const uint32_t t = pair / a.top;
    if (s.id[pair] != kNone) atomicOr(&s.tokens[t >> 5][s.id[pair]], 1u << (t & 31));
  }
  __syncthreads();
  // pairs (low half) and experts (high half) before each expert: two experts to a thread
  static_assert(kMaxExperts == 2 * kRouteThreads, "two experts to a thread");
  uint32_t mine[2];
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t e = 2 * tid + i;
    const uint32_t n = e < a.experts ? __popc(s.tokens[0][e]) + __popc(s.tokens[1][e]) : 0u;
    mine[i] = n ? n | 0x10000u : 0u;
  }
  // batches of hidden (low half) and of down (high half)
  uint32_t cut[2] = {};
  if constexpr (!kChooses) {
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i)
      for (uint32_t down = 0; down < 2; ++down)
        cut[i] |= ((mine[i] & 0xFFFFu) + a.batches[down].tokens - 1) * a.batches[down].inverse >> 16 << (16 * down);
  }
  uint32_t sum = mine[0] + mine[1], cuts = cut[0] + cut[1];
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    const uint32_t below = __shfl_up(sum, step);
    if (lane >= step) sum += below;
    if constexpr (!kChooses) {
      const uint32_t cuts_below = __shfl_up(cuts, step);
      if (lane >= step) cuts += cuts_below;
    }
  }
  if (lane == 63) {
    s.totals[wave] = sum;
    s.batches[wave] = cuts;
  }
  __syncthreads();
  uint32_t before = sum - mine[0] - mine[1], total = 0, cuts_before = cuts - cut[0] - cut[1], all_cuts = 0;
#pragma unroll
  for (int w = 0; w < kRouteWaves; ++w) {
    if (w < wave) {
      before += s.totals[w];
      cuts_before += s.batches[w];
    }
    total += s.totals[w];
    all_cuts += s.batches[w];
  }
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    if (!mine[i]) continue;
    const uint32_t at = i ? before + mine[0] : before;
    s.start[2 * tid + i] = static_cast<uint16_t>(at);
    r.expert[at >> 16] = static_cast<uint16_t>(2 * tid + i);
    r.start[at >> 16] = static_cast<uint16_t>(at);
    if constexpr (!kChooses) {
      const uint32_t first = i ? cuts_before + cut[0] : cuts_before, id = at >> 16 << kBatchBits;
      for (uint32_t n = 0; n < (cut[i] & 0xFFFFu); ++n) owner[(first & 0xFFFFu) + n] = static_cast<uint16_t>(id + n);
      for (uint32_t n = 0; writes && n < cut[i] >> 16; ++n) a.down_owner[(first >> 16) + n] = static_cast<uint16_t>(id + n);
    }
  }
  if (tid == 0) {
    r.batches[0] = all_cuts & 0xFFFFu;
    r.batches[1] = all_cuts >> 16;
    r.active = total >> 16;
    r.start[total >> 16] = static_cast<uint16_t>(total);
  }
  __syncthreads();
  for (uint32_t pair = tid; pair < pairs; pair += kRouteThreads) {
    const uint32_t t = pair / a.top, id = s.id[pair];
    uint32_t at = kNone;
    if (id != kNone) {
      const uint32_t lower = (1u << (t & 31)) - 1;
      at = s.start[id] + (t < 32 ? __popc(s.tokens[0][id] & lower)
                                 : __popc(s.tokens[0][id]) + __popc(s.tokens[1][id] & lower));
      r.token[at] = static_cast<uint16_t>(t);
      r.weight[at] = s.weight[pair];
    }
    r.place[pair] = static_cast<uint16_t>(at);
  }
  __syncthreads();
  give();
}

// ---- products -----------------------------------------------------------------------------------
// A fragment's 32 codes of a lane's block as bf16: four operands of eight.
template <int kFragment>
__device__ __forceinline__ void widen(const Mx4Unit& unit, bf16x8 (&w)[4]) {
  // the scale's byte as a float's exponent (2^-127 is below the normal floats)
  const float s = as_float(max(unit.scales << (23 - 8 * kFragment) & 0x7F800000u, 0x00400000u));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t word = static_cast<uint32_t>(unit.codes[kFragment][i]);
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
// 32 values of a row of parts: `row` is the same in every lane, `offset` (in bytes) a
// lane's own. Lanes past an expert's last token read that token's again: a column of
// the product that is not stored may hold anything.
__device__ __forceinline__ Quad load_quad(const uint16_t* row, uint32_t offset) {
  Quad q;
  const char* const p = reinterpret_cast<const char*>(row) + offset;
#pragma unroll
  for (int i = 0; i < 4; ++i) q.v[i] = *reinterpret_cast<const bf16x8*>(p + 16 * i);
  return q;
}
__device__ __forceinline__ f32x4 multiply(const bf16x8 (&w)[4], const Quad& q, f32x4 acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i], q.v[i], acc, 0, 0, 0);
  return acc;
}
// f(integral constant) for both fragments of a unit.
template <typename F>
__device__ __forceinline__ void both_fragments(F&& f) {
  f(std::integral_constant<int, 0>{});
  f(std::integral_constant<int, 1>{});
}

constexpr int kHiddenParts = 3;  // of a hidden value, whatever the type of x
constexpr int kHiddenWaves = kRouteWaves, kHiddenThreads = kRouteThreads;
constexpr uint32_t kLdsX = 32768;    // few tokens: values of x's parts that a workgroup holds
constexpr uint32_t kLdsH = 65536;    // and of the hidden values' (beside tables and lists all that LDS has)
constexpr uint32_t kFewTokens = 16;  // that the down kernel's tables hold
constexpr uint32_t kLdsRows = 65536;  // many: bytes of an expert's tokens

// Four hidden values of a pair as parts.
__device__ __forceinline__ void store_hidden(uint16_t* to, int64_t part, const float (&v)[4]) {
  uint16_t parts[4][kHiddenParts];
#pragma unroll
  for (int i = 0; i < 4; ++i) split<kHiddenParts>(v[i], parts[i]);
#pragma unroll
  for (int p = 0; p < kHiddenParts; ++p) {
    const uint16_t four[4] = {parts[0][p], parts[1][p], parts[2][p], parts[3][p]};
    __builtin_memcpy(to + p * part, four, 8);
  }
}

// silu(g) u weight.
__device__ __forceinline__ void gated(const f32x4& g, const f32x4& u, float weight, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = g[i] / (1.0f + expf(-g[i])) * u[i] * weight;
}

// ---- hidden, few pairs: eight waves to 16 rows, the tokens' parts in LDS ------------------------
template <int kParts>
__global__ __launch_bounds__(kHiddenThreads, 4) void experts_hidden_few_kernel(ExpertsArgs a) {
  constexpr int U = 2;  // chunks whose weights are in flight together
  __shared__ __attribute__((aligned(16))) union {
    RouteScratch route;
    f32x4 sums[kHiddenWaves][2][64];
  } scratch;
  __shared__ Routing lists;
  extern __shared__ __attribute__((aligned(16))) uint16_t lds_x[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t chunks = a.width_chunks, x_row = 256 * chunks, x_part = a.tokens * x_row;
  // (x's first values are on their way while the experts are chosen)
  const uint32_t mine = 8 * threadIdx.x;
  const u32x4 early = *reinterpret_cast<const u32x4*>(a.x_parts + min(mine, kParts * x_part - 8));
  route<true>(a, blockIdx.x == 0, scratch.route, lists, nullptr);
  if (mine < kParts * x_part) *reinterpret_cast<u32x4*>(lds_x + mine) = early;
  for (uint32_t i = mine + 8 * kHiddenThreads; i < kParts * x_part; i += 8 * kHiddenThreads)
    *reinterpret_cast<u32x4*>(lds_x + i) = *reinterpret_cast<const u32x4*>(a.x_parts + i);
  __syncthreads();
  const uint32_t groups = 16 * a.inner_chunks, real = (a.inner + 15) / 16;  // the last are zeros
  const uint32_t stride = chunks * kMx4Unit;
  const uint32_t first = chunks * wave / kHiddenWaves, last = chunks * (wave + 1) / kHiddenWaves;
  const int64_t h_row = 256 * static_cast<int64_t>(a.inner_chunks), h_part = static_cast<int64_t>(a.tokens) * a.top * h_row;
  const uint32_t items = lists.active * groups;
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const uint32_t slot = item / groups, group = item - slot * groups;
    const uint32_t e = lists.expert[slot], start = lists.start[slot], count = lists.start[slot + 1] - start;
    const uint8_t* const gate = a.gate + (static_cast<uint64_t>(e) * real + group) * stride;
    const uint8_t* const up = a.up + (static_cast<uint64_t>(e) * real + group) * stride;
    const uint32_t r = lane & 15;
    const uint32_t row = 2 * (lists.token[start + min(r, count - 1)] * x_row + 32 * (lane >> 4));
    f32x4 acc[2] = {};
    for (uint32_t c = first; c < (group < real ? last : first); c += U) {
      Mx4Unit g[U], u[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        // (past the last it is read again and not used)
        const uint32_t at = min(c + i, last - 1) * kMx4Unit;
        g[i] = stream_unit(gate + at, lane);
        u[i] = stream_unit(up + at, lane);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (c + i >= last) break;
        both_fragments([&](auto half) __attribute__((always_inline)) {
          constexpr int h = decltype(half)::value;
          bf16x8 wg[4], wu[4];
          widen<h>(g[i], wg);
          widen<h>(u[i], wu);
#pragma unroll
          for (int p = 0; p < kParts; ++p) {
            const Quad q = load_quad(lds_x + p * x_part + 256 * (c + i) + 128 * h, row);
            acc[0] = multiply(wg, q, acc[0]);
            acc[1] = multiply(wu, q, acc[1]);
          }
        });
      }
    }
    scratch.sums[wave][0][lane] = acc[0];
    scratch.sums[wave][1][lane] = acc[1];
    __syncthreads();
    if (wave == 0 && r < count) {
#pragma unroll
      for (int w = 1; w < kHiddenWaves; ++w) {
        acc[0] += scratch.sums[w][0][lane];
        acc[1] += scratch.sums[w][1][lane];
      }
      float v[4] = {};
      if (group < real) gated(acc[0], acc[1], lists.weight[start + r], v);
      store_hidden(a.h_parts + (start + r) * h_row + 16 * group + 4 * (lane >> 4), h_part, v);
    }
    __syncthreads();
  }
}

// What is the same in every lane, told so (LDS gives it to each): addresses from it are
// scalars.
__device__ __forceinline__ uint32_t same(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// ---- many pairs: a wave takes 32 rows of one expert's weights -----------------------------------
// (gate and up of 16 hidden values, or 32 channels of down.) The rows of all experts
// that have tokens are cut evenly over the workgroups, in blocks of eight, a wave each; an
// expert's tokens, as many as fit, lie in LDS while its rows stream by, two or three
// units' loads ahead. A further batch of tokens reads the weights again, as work of its
// own: behind the first in its workgroup it would be what the launch ends with (64 tokens,
// 8 of 128 experts, 4096 -> 1536, f32, whole layer 416 us, 569 that way; the most tokens of
// an expert were 10).
// Measured (the same in bf16): hidden 166 us, 5.1 TB/s of weights; down 90 us, 4.8 TB/s.

// A batch's lines, part by part and in each its tokens, are the columns of one or two
// MFMAs (three parts of up to five tokens are one's: down of the above 106 us with an MFMA
// for each part); here a token's are added, in the column of its number.
template <int kParts>
constexpr uint32_t kColumnGroups = kParts == 1 ? 1 : 2;
template <int kParts>
__device__ __forceinline__ void add_lines(f32x4 (&acc)[kColumnGroups<kParts>][2], uint32_t tokens, int lane) {
  f32x4 sum[2] = {acc[0][0], acc[0][1]};
#pragma unroll
  for (uint32_t p = 1; p < kParts; ++p) {
    const uint32_t line = p * tokens + (lane & 15);
    const int from = static_cast<int>((lane & 48) + (line & 15));
#pragma unroll
    for (uint32_t g = 0; g < kColumnGroups<kParts>; ++g) {
      if (g > 0 && kParts * tokens <= 16) break;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = __shfl(acc[g][j][e], from);
          sum[j][e] += line >> 4 == g ? v : 0.0f;
        }
    }
  }
  acc[0][0] = sum[0];
  acc[0][1] = sum[1];
}

template <bool kDown, int kParts>
__global__ __launch_bounds__(kHiddenThreads, 4) void experts_many_kernel(ExpertsArgs a) {
  constexpr uint32_t G = kColumnGroups<kParts>;
  constexpr int D = kParts == 1 ? 3 : 2;  // (three with more parts spill)
  __shared__ __attribute__((aligned(16))) union {
    RouteScratch route;
    uint8_t rows[kLdsRows];
  } lds;
  __shared__ Routing lists;
  __shared__ __attribute__((aligned(16))) uint16_t owner[kMaxPairs];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if constexpr (kDown) {
    // (of the lists what comes before the tokens)
    for (uint32_t i = threadIdx.x; i < offsetof(Routing, token) / 4; i += kHiddenThreads)
      reinterpret_cast<uint32_t*>(&lists)[i] = reinterpret_cast<const uint32_t*>(a.routing)[i];
    for (uint32_t i = threadIdx.x; i < sizeof(owner) / 4; i += kHiddenThreads)
      reinterpret_cast<uint32_t*>(owner)[i] = reinterpret_cast<const uint32_t*>(a.down_owner)[i];
  } else {
    route<false>(a, blockIdx.x == 0, lds.route, lists, owner);
  }
  __syncthreads();
  const uint32_t chunks = kDown ? a.inner_chunks : a.width_chunks, stride = chunks * kMx4Unit;
  const uint32_t groups = ((kDown ? a.width : a.inner) + 15) / 16;  // of 16 rows of a matrix
  const uint32_t per = kDown ? (groups + 1) / 2 : groups;           // a wave's turns to an expert
  const uint32_t in_row = 256 * chunks;
  const uint16_t* const in = kDown ? a.h_parts : a.x_parts;
  const int64_t in_part = static_cast<int64_t>(a.tokens) * (kDown ? a.top : 1) * in_row;
  const uint32_t out_row = kDown ? 16 * groups : 256 * a.inner_chunks;
  const int64_t h_part = static_cast<int64_t>(a.tokens) * a.top * out_row;
  const Batches& room = a.batches[kDown ? 1 : 0];
  const uint32_t held = room.chunks, lds_row = room.row, batch = room.tokens;

  // an item is eight turns of one expert for one batch of its tokens
  const uint32_t blocks = (per + kHiddenWaves - 1) / kHiddenWaves;
  const uint64_t items = static_cast<uint64_t>(same(lists.batches[kDown ? 1 : 0])) * blocks;
  // (where there are fewer than workgroups, an expert's batches meet in one XCD's L2 if its
  // blocks are a multiple of eight: 64 tokens, 4 of 16 experts, 2048 -> 1024, bf16, hidden 18.1 us, cut evenly 18.7)
  const uint64_t cut = max(items, static_cast<uint64_t>(gridDim.x));
  const uint32_t begin = static_cast<uint32_t>(min(cut * blockIdx.x / gridDim.x, items));
  const uint32_t end = static_cast<uint32_t>(min(cut * (blockIdx.x + 1) / gridDim.x, items));
  for (uint32_t item = begin; item < end;) {
    const uint32_t share = item / blocks, block = item - share * blocks, rounds = min(blocks - block, end - item);
    const uint32_t own = same(owner[share]), slot = own >> kBatchBits, r0 = (own & ((1u << kBatchBits) - 1)) * batch;
    item += rounds;
    const uint32_t from = block * kHiddenWaves, to = min(per, from + rounds * kHiddenWaves), steps = rounds * chunks;
    const uint32_t e = same(lists.expert[slot]), start = same(lists.start[slot]), count = same(lists.start[slot + 1]) - start;
    const uint32_t tokens = min(batch, count - r0), r = lane & 15, lines = kParts * tokens;
    uint32_t row[G];
#pragma unroll
    for (uint32_t g = 0; g < G; ++g) row[g] = min(16 * g + r, lines - 1) * lds_row + 64 * (lane >> 4);
    // Loads run D steps ahead, over rounds as well (past the last turn or step the
    // last row again), and have no branches: a wait in the loop then counts them.
    const uint64_t matrix = static_cast<uint64_t>(groups) * stride;
    const uint8_t* const base0 = (kDown ? a.down : a.gate) + e * matrix;
    const uint8_t* const base1 = (kDown ? a.down : a.up) + e * matrix;
    uint32_t ahead_chunk = 0, ahead_turn = from + wave;
    auto load = [&](Mx4Unit (&u)[2]) __attribute__((always_inline)) {
      const uint32_t t = min(ahead_turn, to - 1);
      // (an odd last group is read twice, its second results are not stored)
      const uint32_t g0 = kDown ? 2 * t : t, g1 = kDown ? min(2 * t + 1, groups - 1) : t;
      u[0] = stream_unit(base0 + static_cast<uint64_t>(g0) * stride + ahead_chunk * kMx4Unit, lane);
      u[1] = stream_unit(base1 + static_cast<uint64_t>(g1) * stride + ahead_chunk * kMx4Unit, lane);
      const bool wraps = ahead_chunk + 1 == chunks;
      ahead_turn += wraps ? kHiddenWaves : 0;
      ahead_chunk = wraps ? 0 : ahead_chunk + 1;
    };
    Mx4Unit w[D][2];
#pragma unroll
    for (int i = 0; i < D; ++i) load(w[i]);
    f32x4 acc[G][2] = {};
    uint32_t c = 0, held_at = 0, mine = from + wave;
    bool staged = false;
    for (uint32_t step = 0; step < steps; step += D) {
#pragma unroll
      for (int i = 0; i < D; ++i) {
        if (step + i < steps) {
          if (!staged || c - held_at >= held) {
            held_at = c;
            staged = true;
            const uint32_t now = min(held, chunks - c), vectors = 32 * now;
            __syncthreads();
            for (uint32_t v = threadIdx.x; v < lines * vectors; v += kHiddenThreads) {
              const uint32_t line = v / vectors, at = v - line * vectors, p = line / tokens, t = line - p * tokens;
              const uint32_t source = kDown ? start + r0 + t : lists.token[start + r0 + t];
              *reinterpret_cast<u32x4*>(lds.rows + line * lds_row + 16 * at) =
                  *reinterpret_cast<const u32x4*>(in + p * in_part + static_cast<int64_t>(source) * in_row + 256 * c + 8 * at);
            }
            __syncthreads();
          }
          both_fragments([&](auto half) __attribute__((always_inline)) {
            constexpr int h = decltype(half)::value;
            bf16x8 w0[4], w1[4];
            widen<h>(w[i][0], w0);
            widen<h>(w[i][1], w1);
#pragma unroll
            for (uint32_t g = 0; g < G; ++g) {
              if (g > 0 && lines <= 16) break;
              const Quad q = load_quad(reinterpret_cast<const uint16_t*>(lds.rows) + 256 * (c - held_at) + 128 * h, row[g]);
              acc[g][0] = multiply(w0, q, acc[g][0]);
              acc[g][1] = multiply(w1, q, acc[g][1]);
            }
          });
          if (++c == chunks) {
            add_lines<kParts>(acc, tokens, lane);
            const uint32_t pair = start + r0 + r;
            if (mine < to && r < tokens) {
              if constexpr (kDown) {
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j)
                  if (2 * mine + j < groups)
                    *reinterpret_cast<f32x4*>(a.y + static_cast<int64_t>(pair) * out_row + 16 * (2 * mine + j) + 4 * (lane >> 4)) = acc[0][j];
              } else {
                float v[4];
                gated(acc[0][0], acc[0][1], lists.weight[pair], v);
                uint16_t* const out = a.h_parts + static_cast<int64_t>(pair) * out_row + 4 * (lane >> 4);
                store_hidden(out + 16 * mine, h_part, v);
                // the zeros after the last
                const float zeros[4] = {};
                if (mine + 1 == groups)
                  for (uint32_t g = groups; g < 16 * a.inner_chunks; ++g) store_hidden(out + 16 * g, h_part, zeros);
              }
            }
#pragma unroll
            for (auto& group : acc) group[0] = group[1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            c = 0;
            mine += kHiddenWaves;
            if (held < chunks) staged = false;
          }
        }
        load(w[i]);
      }
    }
  }
}

// ---- down, few pairs ------------------------------------------------------------------------------
constexpr int kDownWaves = 16, kDownThreads = 64 * kDownWaves;

template <typename T>
__global__ __launch_bounds__(kDownThreads) void experts_down_few_kernel(ExpertsArgs a) {
  constexpr int U = 3;  // units in flight together
  __shared__ __attribute__((aligned(16))) float table[kDownWaves][kFewTokens][16];
  __shared__ __attribute__((aligned(16))) uint16_t lds_h[kLdsH];
  __shared__ Routing lists;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t chunks = a.inner_chunks, stride = chunks * kMx4Unit, groups = (a.width + 15) / 16, group = blockIdx.x;
  const uint32_t h_row = 256 * chunks, pairs = a.tokens * a.top, h_part = pairs * h_row;
  for (uint32_t i = threadIdx.x; i < offsetof(Routing, place) / 4; i += kDownThreads)
    reinterpret_cast<uint32_t*>(&lists)[i] = reinterpret_cast<const uint32_t*>(a.routing)[i];
  // The hidden values are asked for before the weights: loads return in order. (Pairs that
  // there are not hold anything, and meet no weights.)
  constexpr int kVectors = kLdsH / (8 * kDownThreads);
  u32x4 early[kVectors];
#pragma unroll
  for (int i = 0; i < kVectors; ++i)
    if (8u * kDownThreads * i < kHiddenParts * h_part)
      early[i] = *reinterpret_cast<const u32x4*>(a.h_parts + min(8 * (threadIdx.x + i * kDownThreads), kHiddenParts * h_part - 8));
  for (uint32_t i = threadIdx.x; i < kDownWaves * kFewTokens * 16; i += kDownThreads) (&table[0][0][0])[i] = 0.0f;
  __syncthreads();
  const uint32_t units = lists.active * chunks;
  const uint32_t first = units * wave / kDownWaves, last = units * (wave + 1) / kDownWaves;
  auto unit_at = [&](uint32_t q) {
    const uint32_t slot = q / chunks, c = q - slot * chunks;
    return stream_unit(a.down + (static_cast<uint64_t>(lists.expert[slot]) * groups + group) * stride + c * kMx4Unit, lane);
  };
  Mx4Unit w[U] = {};
  if (first < last) {
#pragma unroll
    for (int i = 0; i < U; ++i) w[i] = unit_at(min(first + i, last - 1));
  }
#pragma unroll
  for (int i = 0; i < kVectors; ++i) {
    const uint32_t at = 8 * (threadIdx.x + i * kDownThreads);
    if (at < kHiddenParts * h_part) *reinterpret_cast<u32x4*>(lds_h + at) = early[i];
  }
  __syncthreads();
  f32x4 acc = {};
  auto multiply_unit = [&](uint32_t q, const Mx4Unit& unit) __attribute__((always_inline)) {
    const uint32_t slot = q / chunks, c = q - slot * chunks;
    const uint32_t start = lists.start[slot], count = lists.start[slot + 1] - start, r = lane & 15;
    const uint32_t row = 2 * ((start + min(r, count - 1)) * h_row + 32 * (lane >> 4));
    both_fragments([&](auto half) __attribute__((always_inline)) {
      constexpr int h = decltype(half)::value;
      bf16x8 wide[4];
      widen<h>(unit, wide);
#pragma unroll
      for (int p = 0; p < kHiddenParts; ++p) acc = multiply(wide, load_quad(lds_h + p * h_part + 256 * c + 128 * h, row), acc);
    });
    if (c + 1 == chunks || q + 1 == last) {
      // the expert's share of its tokens (no token is twice in the list)
      if (r < count) {
        f32x4* const sum = reinterpret_cast<f32x4*>(&table[wave][lists.token[start + r]][4 * (lane >> 4)]);
        *sum += acc;
      }
      acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  };
  uint32_t base = first;
  for (; base + U < last; base += U) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      multiply_unit(base + i, w[i]);
      w[i] = unit_at(min(base + U + i, last - 1));
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (base + i < last) multiply_unit(base + i, w[i]);
  __syncthreads();
  const uint32_t i = threadIdx.x;
  if (i < 4 * a.tokens) {
    const uint32_t t = i / 4, channel = 16 * group + 4 * (i % 4);
    f32x4 sum = *reinterpret_cast<const f32x4*>(&table[0][t][4 * (i % 4)]);
#pragma unroll
    for (int v = 1; v < kDownWaves; ++v) sum += *reinterpret_cast<const f32x4*>(&table[v][t][4 * (i % 4)]);
    const float out[4] = {sum[0], sum[1], sum[2], sum[3]};
    if (channel < a.width) store4(static_cast<T*>(a.out) + t * a.ldo + channel, static_cast<int64_t>(a.width) - channel, out);
  }
}

// Each token's pairs, by its slots: four channels to a thread.
template <typename T>
__global__ __launch_bounds__(256) void experts_combine_kernel(ExpertsArgs a) {
  const uint32_t row = (a.width + 15) / 16 * 16, quads = (a.width + 3) / 4;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.tokens * quads) return;
  const uint32_t t = i / quads, channel = 4 * (i - t * quads);
  f32x4 v[kMaxExpertTop], sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (uint32_t n = 0; n < kMaxExpertTop; ++n) {
    v[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t place = n < a.top ? a.routing->place[t * a.top + n] : kNone;
    if (place != kNone) v[n] = *reinterpret_cast<const f32x4*>(a.y + static_cast<int64_t>(place) * row + channel);
  }
#pragma unroll
  for (uint32_t n = 0; n < kMaxExpertTop; ++n) sum += v[n];
  const float out[4] = {sum[0], sum[1], sum[2], sum[3]};
  store4(static_cast<T*>(a.out) + t * a.ldo + channel, static_cast<int64_t>(a.width) - channel, out);
}

int parts_of(uint32_t dtype) { return dtype == RNS8_MI355X_F32 ? 3 : dtype == RNS8_MI355X_F16 ? 2 : 1; }

// Whether x and the hidden values fit a workgroup's LDS, and the tokens its tables.
bool few(const rns8_mi355x_experts_mx4_args& a) {
  return a.tokens <= kFewTokens && parts_of(a.dtype) * a.tokens * mx4_chunks(a.width) * 256 <= kLdsX &&
         kHiddenParts * a.tokens * a.top * mx4_chunks(a.inner) * 256 <= kLdsH;
}

// The workspace: scores, the parts of x and of the hidden values, pairs' results, the lists.
uint64_t lay_out(const rns8_mi355x_experts_mx4_args& a, ExpertsArgs& e) {
  uint8_t* const at = static_cast<uint8_t*>(a.workspace);
  uint64_t bytes = 0;
  auto take = [&](uint64_t size) {
    uint8_t* const got = at ? at + bytes : nullptr;
    bytes += round_up(size, 256);
    return got;
  };
  const uint64_t tokens = static_cast<uint64_t>(a.tokens), pairs = tokens * a.top;
  e.scores = reinterpret_cast<float*>(take(a.router ? tokens * static_cast<uint64_t>(a.experts) * sizeof(float) : 0));
  e.x_parts = reinterpret_cast<uint16_t*>(
      take(static_cast<uint64_t>(parts_of(a.dtype)) * tokens * static_cast<uint64_t>(mx4_chunks(a.width)) * 512));
  e.h_parts = reinterpret_cast<uint16_t*>(
      take(static_cast<uint64_t>(kHiddenParts) * pairs * static_cast<uint64_t>(mx4_chunks(a.inner)) * 512));
  e.chosen = a.ids;
  e.chosen_weights = a.weights;
  if (a.router && !few(a)) {
    e.chosen = reinterpret_cast<int32_t*>(take(pairs * sizeof(int32_t)));
    e.chosen_weights = reinterpret_cast<float*>(take(pairs * sizeof(float)));
  }
  e.y = reinterpret_cast<float*>(take(few(a) ? 0 : pairs * static_cast<uint64_t>(mx4_groups(a.width)) * 64));
  e.routing = reinterpret_cast<Routing*>(take(sizeof(Routing)));
  e.down_owner = reinterpret_cast<uint16_t*>(take(few(a) ? 0 : kMaxPairs * sizeof(uint16_t)));
  return bytes;
}

template <typename T, int kParts>
hipError_t launch_typed(ExpertsArgs e, bool is_few, hipStream_t stream) {
  const uint32_t x_blocks = e.tokens * ((256 * e.width_chunks + 2047) / 2048);
  auto stage = [&](auto experts, auto tokens) {
    constexpr uint32_t kExperts = decltype(experts)::value, kTokens = decltype(tokens)::value;
    const uint32_t blocks = e.router ? (e.experts + kExperts - 1) / kExperts * ((e.tokens + kTokens - 1) / kTokens) : 0;
    hipLaunchKernelGGL((experts_stage_kernel<T, kParts, kExperts, kTokens>), dim3(blocks + x_blocks), dim3(256), 0, stream, e, blocks);
  };
  if (e.tokens <= 2)
    stage(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
  else
    stage(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{});
  const uint32_t active = std::min(e.experts, e.tokens * e.top), groups = (e.width + 15) / 16;
  const dim3 threads(kHiddenThreads);
  if (is_few) {
    hipLaunchKernelGGL(experts_hidden_few_kernel<kParts>, dim3(std::min(active * 16 * e.inner_chunks, 512u)), threads,
                       kParts * e.tokens * e.width_chunks * 512, stream, e);
    hipLaunchKernelGGL(experts_down_few_kernel<T>, dim3(groups), dim3(kDownThreads), 0, stream, e);
    return hipGetLastError();
  }
  if (e.router) hipLaunchKernelGGL(experts_choose_kernel, dim3(e.tokens), dim3(64), 0, stream, e);
  uint32_t grid[2];
  for (int down = 0; down < 2; ++down) {
    const uint32_t turns = down ? (groups + 1) / 2 : (e.inner + 15) / 16, parts = down ? kHiddenParts : kParts;
    const uint32_t blocks = (turns + kHiddenWaves - 1) / kHiddenWaves;
    Batches& b = e.batches[down];
    b.chunks = std::min(down ? e.inner_chunks : e.width_chunks, (kLdsRows / parts - 16) / 512);
    b.row = 512 * b.chunks + 16;
    b.tokens = std::min(kLdsRows / (parts * b.row), parts == 3 ? 10u : 16u);  // two MFMAs' columns
    b.inverse = 65536 / b.tokens + 1;  // (right for what it divides, below 80)
    const uint32_t batches = active + (e.tokens * e.top - active) / b.tokens;  // at most
    grid[down] = std::min(batches * blocks, 512u);  // two workgroups to a CU
  }
  hipLaunchKernelGGL((experts_many_kernel<false, kParts>), dim3(grid[0]), threads, 0, stream, e);
  hipLaunchKernelGGL((experts_many_kernel<true, kHiddenParts>), dim3(grid[1]), threads, 0, stream, e);
  hipLaunchKernelGGL(experts_combine_kernel<T>, dim3((e.tokens * ((e.width + 3) / 4) + 255) / 256), dim3(256), 0, stream, e);
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
  e.width = static_cast<uint32_t>(a.width);
  e.inner = static_cast<uint32_t>(a.inner);
  e.width_chunks = static_cast<uint32_t>(mx4_chunks(a.width));
  e.inner_chunks = static_cast<uint32_t>(mx4_chunks(a.inner));
  lay_out(a, e);
  if (a.dtype == RNS8_MI355X_F32) return launch_typed<float, 3>(e, few(a), stream);
  if (a.dtype == RNS8_MI355X_F16) return launch_typed<f16, 2>(e, few(a), stream);
  return launch_typed<bf16, 1>(e, few(a), stream);
}

}  // namespace rns8x
