// Tile kernels of the product of MX4 matrices (gfx950).
//
//   out[i][j] = sum_k a[i][k] b[j][k] + bias[j]
//
// Bound by the matrix cores where the product is large: v_mfma_scale_f32_16x16x128
// takes 128 columns of 4-bit codes in the time of 64 of bytes and applies both
// operands' scales itself.
//   * A persistent grid over output tiles (and slices of K), each XCD a contiguous
//     share of them, tiles in groups of rows for the L2.
//   * K in steps of 128 (a fragment, 1 KB for 16 rows) through a ring of four LDS
//     stages, filled by buffer-load DMA four steps ahead, also across tile
//     boundaries; one counted wait and one barrier per step. Fragments lie in memory
//     as a wave reads them, so the stages need no swizzle and no read conflicts.
//   * Scales of 256 columns (both fragments of a unit) come once for two steps into a
//     ring of two, and stay in registers for both; the MFMA picks its byte.
//   * A matrix ends with zeros in its units, and what lies past its last unit is past
//     the buffer and loads zero: nothing is masked.
//   * The next step's fragments are read beside a step's MFMAs.
//   * Few tiles: K is cut into slices of whole units, whose 32-bit sums go to the
//     workspace; a second kernel adds them in order.
//   * Both gradients of a linear layer are one launch where their tiles fit on the chip
//     at once: an eighth of each product to every XCD, the longer sums first. The gradient of
//     the bias, partial sums of rows, is added up there too, by waves that have asked for
//     their first tile. All gradients, with their roundings: 500 x 701 x 611 in f32 15.2
//     us instead of 23.8 (three launches), 2048^3 in bf16 31.7 instead of 38.6, 4096 x 1024
//     x 1024 30.0 instead of 32.2. Tiles that follow one another gain nothing (4096^3 in
//     one walk over both: 105 us, 86 apart).
// Measured on rounded normal values, bf16 outputs: 8192^3 257 us, 4.3 PFLOP/s; 4096^3
// 43 us, 3.2. Bare scaled MFMAs at one wave to a SIMD run at 5.3 PFLOP/s on random codes
// (6.8 on zeros: the clock gives way); eight waves of 128 x 64, two to a SIMD, issue them
// closer but read fragments more often: 8192^3 275 us.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dma.hpp"
#include "int_ops.hpp"
#include "kernels.hpp"
#include "mx4.hpp"
#include "mx4_mfma.hpp"
#include "scaled_epilogue.hpp"
#include "scaled_gemm.hpp"
#include "tables.hpp"

namespace rns8x {
namespace {

// kWaves waves (2 x WN) each own TM x TN blocks of 16 x 16 outputs: a tile of
// (32 TM) x (16 TN WN), kResident tiles to a CU.
template <int TM_, int TN_, int WN_, int kResident_>
struct Cfg {
  static constexpr int TM = TM_, TN = TN_, WN = WN_, kResident = kResident_;
  static constexpr int kWaves = 2 * WN, kThreads = 64 * kWaves;
  static constexpr int BM = 32 * TM, BN = 16 * TN * WN;
  static constexpr int kDmaA = BM / 16 / kWaves, kDmaB = BN / 16 / kWaves;  // fragments per wave and step
  static constexpr int kStageA = 64 * BM, kStage = 64 * (BM + BN), kStages = 4;
  static constexpr int kScaleSlot = 2048 * kWaves;  // 1 KB of each operand for a wave's DMA
  static constexpr int kLds = kStages * kStage + 2 * kScaleSlot;
  static constexpr int kGroupM = 1024 / BM;  // tile rows per L2 reuse group
  static_assert(kDmaA >= 1 && kDmaA <= 4 && kDmaB >= 1 && kDmaB <= 4, "DMA blocks");
  static_assert(TM % 2 == 0 && TN % 2 == 0 && kLds <= 160 * 1024, "tile config");
};

struct TileArgs {
  const uint8_t *a, *b;
  const float* bias;
  void* out;
  float* partials;  // [slices][m][ldp], or NULL
  int64_t ldo, ldp;
  uint32_t m, n, groups_m, groups_n;
  uint32_t chunks, stride;  // units of 16 rows, and their bytes
  uint32_t dtype;
  uint32_t units, tiles_m;  // slice-major, tiles in groups of kGroupM tile rows
  DivU31 tiles, group, rows, tail;
  uint32_t slice_chunks;
};

__device__ __forceinline__ uint32_t div_u31(uint32_t n, DivU31 v) { return __umulhi(n << 1, v.mul) >> v.shift; }

template <int kId, int kPer, int kReads>
__device__ __forceinline__ void sched_slots() {
  if constexpr (kReads > 0) {
    __builtin_amdgcn_sched_group_barrier(0x008, kPer, kId);  // MFMA
    __builtin_amdgcn_sched_group_barrier(0x100, 1, kId);     // DS read
    sched_slots<kId, kPer, kReads - 1>();
  }
}

// One product, or two, of each an eighth to every XCD and a unit to a workgroup.
struct OneProduct {
  TileArgs product[1];
};
struct TwoProducts {
  TileArgs product[2];
  Mx4Sums sums;
};

template <typename C, typename Products>
__global__ __launch_bounds__(C::kThreads, (C::kResident * C::kWaves / 4)) void mx4_tiles_kernel(Products p) {
  constexpr bool kTwo = std::is_same<Products, TwoProducts>::value;
  constexpr int TM = C::TM, TN = C::TN, BM = C::BM, BN = C::BN;
  __shared__ __attribute__((aligned(16))) int8_t lds[C::kLds];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave / C::WN, wave_n = wave % C::WN;

  uint32_t which = 0, u_first, u_step = 1, u_end;
  const uint32_t xcd = blockIdx.x & 7u, place = blockIdx.x >> 3;
  auto share = [&](uint32_t units, uint32_t x) { return static_cast<uint32_t>((static_cast<uint64_t>(x) * units) / 8); };
  if constexpr (kTwo) {
    const uint32_t first = share(p.product[0].units, xcd + 1) - share(p.product[0].units, xcd);
    which = place >= first ? 1 : 0;
    const uint32_t units = p.product[which].units;
    u_first = share(units, xcd) + place - (which ? first : 0);
    u_end = min(u_first + 1, share(units, xcd + 1));
  } else if ((gridDim.x & 7u) == 0u) {
    u_first = share(p.product[0].units, xcd) + place;
    u_end = share(p.product[0].units, xcd + 1);
    u_step = gridDim.x >> 3;
  } else {
    u_first = blockIdx.x;
    u_end = p.product[0].units;
    u_step = gridDim.x;
  }
  const TileArgs& args = p.product[which];
  u_first = __builtin_amdgcn_readfirstlane(u_first);
  u_end = __builtin_amdgcn_readfirstlane(u_end);
  // (a grid is whole multiples of eight: a workgroup may have no unit, but has its sums;
  // the last ones begin)
  auto add_sums = [&]() {
    if constexpr (kTwo) {
      if (p.sums.out) add_partials(p.sums, (gridDim.x - 1 - blockIdx.x) * C::kWaves + wave, gridDim.x * C::kWaves, lane);
    }
  };
  if (u_first >= u_end) {
    add_sums();
    return;
  }

  struct Unit {
    uint32_t slice, m0, n0, first, count;  // chunks
  };
  auto decode = [&](uint32_t u) {
    Unit U;
    U.slice = div_u31(u, args.tiles);
    const uint32_t pid = u - U.slice * args.tiles.d;
    const uint32_t group = div_u31(pid, args.group);
    const uint32_t first_m = group * C::kGroupM;
    const uint32_t rem = pid - group * args.group.d;
    const DivU31 rows = first_m + C::kGroupM <= args.tiles_m ? args.rows : args.tail;
    const uint32_t tn = div_u31(rem, rows);
    U.m0 = (first_m + rem - tn * rows.d) * BM;
    U.n0 = tn * BN;
    U.first = U.slice * args.slice_chunks;
    U.count = min(args.slice_chunks, args.chunks - U.first);
    return U;
  };

  // ---- global -> LDS by DMA -----------------------------------------------------------
  // The chunk whose DMA is issued next, two chunks ahead of the compute position;
  // past the last unit everything loads zero.
  struct Cursor {
    const uint8_t *a, *b;
    int32_t a_n, b_n;  // bytes from there to the end of the tile's last 16 rows
    uint32_t left, u;
  };
  auto cursor_of = [&](uint32_t u) {
    const bool live = u < u_end;
    const Unit U = decode(live ? u : u_end - 1);
    const uint32_t skip = U.first * kMx4Unit;
    Cursor c;
    c.a = args.a + static_cast<uint64_t>(U.m0 / 16) * args.stride + skip;
    c.b = args.b + static_cast<uint64_t>(U.n0 / 16) * args.stride + skip;
    const uint32_t ga = min(static_cast<uint32_t>(BM / 16), args.groups_m - U.m0 / 16);
    const uint32_t gb = min(static_cast<uint32_t>(BN / 16), args.groups_n - U.n0 / 16);
    c.a_n = live ? static_cast<int32_t>(ga * args.stride - skip) : 0;
    c.b_n = live ? static_cast<int32_t>(gb * args.stride - skip) : 0;
    c.left = live ? U.count : 0xFFFFFFFFu;
    c.u = u;
    return c;
  };
  Cursor cur = cursor_of(u_first);
  // (what is past the buffer's bytes reads as zero: offsets stay below 2^31)
  uint32_t a_voff[C::kDmaA], b_voff[C::kDmaB];
#pragma unroll
  for (int i = 0; i < C::kDmaA; ++i) a_voff[i] = static_cast<uint32_t>(wave * C::kDmaA + i) * args.stride + 16 * lane;
#pragma unroll
  for (int i = 0; i < C::kDmaB; ++i) b_voff[i] = static_cast<uint32_t>(wave * C::kDmaB + i) * args.stride + 16 * lane;
  // a wave's share of the scales: eight lanes to the 128 bytes of 16 rows
  const uint32_t row = lane >> 3, at = kMx4Scales + 16 * (lane & 7);
  const uint32_t as_voff = lane < 8 * C::kDmaA ? (wave * C::kDmaA + row) * args.stride + at : 0x80000000u;
  const uint32_t bs_voff = lane < 8 * C::kDmaB ? (wave * C::kDmaB + row) * args.stride + at : 0x80000000u;
  auto advance = [&]() {
    if (--cur.left == 0) {
      cur = cursor_of(cur.u + u_step);
      return;
    }
    const int32_t step = cur.a_n ? kMx4Unit : 0;
    cur.a += step;
    cur.b += step;
    cur.a_n -= step;
    cur.b_n -= step;
  };
  const uint32_t lds0 = lds_address(lds);
  const uint32_t lds_a = lds0 + static_cast<uint32_t>(wave * C::kDmaA * 1024);
  const uint32_t lds_b = lds0 + static_cast<uint32_t>(C::kStageA + wave * C::kDmaB * 1024);
  const uint32_t lds_s = lds0 + static_cast<uint32_t>(C::kStages * C::kStage + wave * 2048);
  auto dma_a = [&](v4i src, uint32_t stage, int half, int i) {
    dma16_block(__builtin_amdgcn_readfirstlane(lds_a + stage), i, a_voff[i] + 1024 * half, src);
  };
  auto dma_b = [&](v4i src, uint32_t stage, int half, int i) {
    dma16_block(__builtin_amdgcn_readfirstlane(lds_b + stage), i, b_voff[i] + 1024 * half, src);
  };
  auto dma_scales = [&](v4i sa, v4i sb, uint32_t slot) {
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds_s + slot);
    dma16_block(at, 0, as_voff, sa);
    dma16_block(at, 1, bs_voff, sb);
  };

  // ---- fragments and scales from LDS ---------------------------------------------------
  struct Frags {
    i32x4 a[TM];
    i32x4 b[TN];
  };
  struct Scales {  // both fragments' bytes
    uint32_t a[TM];
    uint32_t b[TN];
  };
  auto read_a = [&](uint32_t stage, int i) {
    return *reinterpret_cast<const i32x4*>(lds + stage + (wave_m * TM + i) * 1024 + 16 * lane);
  };
  auto read_b = [&](uint32_t stage, int j) {
    return *reinterpret_cast<const i32x4*>(lds + stage + C::kStageA + (wave_n * TN + j) * 1024 + 16 * lane);
  };
  auto scales_at = [&](uint32_t slot, int group, int per_wave, int operand) {
    return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(
        lds + C::kStages * C::kStage + slot + (group / per_wave) * 2048 + operand * 1024 + (group % per_wave) * 128 + 2 * lane));
  };
  auto read_sa = [&](uint32_t slot, int i) { return scales_at(slot, wave_m * TM + i, C::kDmaA, 0); };
  auto read_sb = [&](uint32_t slot, int j) { return scales_at(slot, wave_n * TN + j, C::kDmaB, 1); };

  f32x4 acc[TM][TN];
  auto mfma_half = [&](auto first, auto half_c, const Frags& f, const Scales& s, int i0) __attribute__((always_inline)) {
    constexpr int half = decltype(half_c)::value;
#pragma unroll
    for (int ii = 0; ii < TM / 2; ++ii)
#pragma unroll
      for (int jj = 0; jj < TN; ++jj) {
        const int i = i0 + ii, j = (ii & 1) ? TN - 1 - jj : jj;
        const f32x4 start = {0.0f, 0.0f, 0.0f, 0.0f};
        acc[i][j] = mx4_mfma<half, half>(f.b[j], f.a[i], decltype(first)::value ? start : acc[i][j], s.b[j], s.a[i]);
      }
  };
  constexpr int kMfma = TM / 2 * TN;
  auto schedule_region = [&](auto id, auto reads, int i0) __attribute__((always_inline)) {
    constexpr int kId = decltype(id)::value, kReads = decltype(reads)::value;
#pragma unroll
    for (int i = 0; i < TM / 2; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) asm volatile("" ::"a"(acc[i0 + i][j]));
    constexpr int kPerSlot = kMfma * 3 / 4 / kReads > 0 ? kMfma * 3 / 4 / kReads : 1;
    sched_slots<kId, kPerSlot, kReads>();
    if constexpr (kMfma > kPerSlot * kReads)
      __builtin_amdgcn_sched_group_barrier(0x008, kMfma - kPerSlot * kReads, kId);
    __builtin_amdgcn_sched_barrier(0);
  };

  // ---- epilogue: element e of acc[i][j] is row m0 + 16 (wave_m TM + i) + (lane & 15),
  // column n0 + 16 (wave_n TN + j) + 4 (lane >> 4) + e ------------------------------------
  const int frag_row = lane & 15, frag_col = lane >> 4;
  // (read in place by asm: left to itself the compiler moves all of them at once)
  auto sums = [&](int i, int j) {
    const Acc4 v = acc_read4(__builtin_bit_cast(v4i_acc, acc[i][j]));
    return f32x4{as_float(v.v[0]), as_float(v.v[1]), as_float(v.v[2]), as_float(v.v[3])};
  };
  auto epilogue = [&](const Unit& U) {
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");  // the reads below are asm: MFMA results settle first
    const int64_t row0 = static_cast<int64_t>(U.m0) + wave_m * (16 * TM) + frag_row;
    const int64_t col0 = static_cast<int64_t>(U.n0) + wave_n * (16 * TN);
    const int64_t m = args.m, n = args.n;
    if (args.partials) {
      float* const base = args.partials + (static_cast<int64_t>(U.slice) * m + row0) * args.ldp + col0 + 4 * frag_col;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const f32x4 v = sums(i, j);
          if (row0 + 16 * i < m && col0 + 16 * j + 4 * frag_col < args.ldp)
            *reinterpret_cast<f32x4*>(base + 16 * i * args.ldp + 16 * j) = v;
        }
      return;
    }
    auto write = [&](auto type) {
      using T = decltype(type);
      T* const out = static_cast<T*>(args.out);
#pragma unroll
      for (int j = 0; j < TN; j += 2) {
        float bias[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) load4_or(args.bias, col0 + 16 * (j + h) + 4 * frag_col, n, 0.0f, bias[h]);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int64_t row = row0 + 16 * i;
          float f[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const f32x4 v = sums(i, j + h);
#pragma unroll
            for (int e = 0; e < 4; ++e) f[h][e] = v[e] + bias[h][e];
          }
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int64_t c = col0 + 16 * (j + h) + 4 * frag_col;
              if (row < m && c < n) store4(out + row * args.ldo + c, n - c, f[h]);
            }
          } else {
            // Two blocks' 8-byte pieces: after swapping odd with even lane groups,
            // groups 0 and 2 hold block j's columns 0-7 and 8-15 of the row, groups 1
            // and 3 block j + 1's.
            uint32_t d[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              T t[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) t[e] = static_cast<T>(f[h][e]);
              __builtin_memcpy(d[h], t, 8);
            }
            const auto s0 = __builtin_amdgcn_permlane16_swap(d[0][0], d[1][0], false, false);
            const auto s1 = __builtin_amdgcn_permlane16_swap(d[0][1], d[1][1], false, false);
            const uint32_t w[4] = {s0[0], s1[0], s0[1], s1[1]};
            const int64_t c = col0 + 16 * (j + (frag_col & 1)) + 8 * (frag_col >> 1);
            if (row < m && c < n) {
              T* const p = out + row * args.ldo + c;
              if (c + 8 <= n) {
                __builtin_memcpy(p, w, 16);
              } else {
                T t[8];
                __builtin_memcpy(t, w, 16);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (c + e < n) p[e] = t[e];
              }
            }
          }
        }
      }
    };
    if (args.dtype == RNS8_MI355X_BF16)
      write(bf16{});
    else if (args.dtype == RNS8_MI355X_F16)
      write(f16{});
    else
      write(float{});
  };

  // ---- pipeline ---------------------------------------------------------------------------
  // Step t multiplies the fragments that step t - 1 read, reads those of t + 1 and
  // issues the DMA of t + 4 into the stage that t's came from; the scales of a chunk
  // go where the ones two chunks before were. At its end all but the DMA of the last
  // two steps (of which one has the scales) has landed: t + 2 may be read.
  constexpr int kDmaStep = C::kDmaA + C::kDmaB;
  using Half0 = std::integral_constant<int, 0>;
  using Half1 = std::integral_constant<int, 1>;
  Frags f0, f1;
  Scales now, next;
  uint32_t stage = 0;  // of an even step; the next is one further
  uint32_t slot = 0;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const v4i sa = buffer_rsrc(cur.a, cur.a_n), sb = buffer_rsrc(cur.b, cur.b_n);
    dma_scales(sa, sb, c * C::kScaleSlot);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int i = 0; i < C::kDmaA; ++i) dma_a(sa, (2 * c + half) * C::kStage, half, i);
#pragma unroll
      for (int i = 0; i < C::kDmaB; ++i) dma_b(sb, (2 * c + half) * C::kStage, half, i);
    }
    advance();
  }
  add_sums();
  __builtin_amdgcn_s_waitcnt(wait_vm(2 * kDmaStep + 2));  // chunk 0 landed
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    f0.a[i] = read_a(0, i);
    now.a[i] = read_sa(0, i);
  }
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    f0.b[j] = read_b(0, j);
    now.b[j] = read_sb(0, j);
  }
  __syncthreads();  // stage 0 and the scales are read: steps 4 and 5 may overwrite them
  auto step = [&](auto first, auto half_c, const Frags& f, Frags& fn) __attribute__((always_inline)) {
    constexpr int half = decltype(half_c)::value;
    constexpr int kLen = TM / 2 > TN / 2 ? (TM / 2 > 4 ? TM / 2 : 4) : (TN / 2 > 4 ? TN / 2 : 4);
    const uint32_t mine = stage + half * C::kStage;
    const uint32_t after = half ? stage ^ (2 * C::kStage) : stage + C::kStage;
    const uint32_t other = slot ^ C::kScaleSlot;
    const v4i sa = buffer_rsrc(cur.a, cur.a_n), sb = buffer_rsrc(cur.b, cur.b_n);
    if constexpr (half == 0) dma_scales(sa, sb, slot);
#pragma unroll
    for (int t = 0; t < kLen; ++t) {
      if (t < TM / 2) fn.a[t] = read_a(after, t);
      if (t < TN / 2) fn.b[t] = read_b(after, t);
      if constexpr (half == 1) {
        if (t < TM / 2) next.a[t] = read_sa(other, t);
        if (t < TN / 2) next.b[t] = read_sb(other, t);
      }
      if (t < C::kDmaA) dma_a(sa, mine, half, t);
    }
    constexpr int kReads = (TM / 2 + TN / 2) * (half + 1);
    mfma_half(first, half_c, f, now, 0);
    schedule_region(std::integral_constant<int, 1>{}, std::integral_constant<int, kReads>{}, 0);
#pragma unroll
    for (int t = 0; t < kLen; ++t) {
      if (t < TM / 2) fn.a[TM / 2 + t] = read_a(after, TM / 2 + t);
      if (t < TN / 2) fn.b[TN / 2 + t] = read_b(after, TN / 2 + t);
      if constexpr (half == 1) {
        if (t < TM / 2) next.a[TM / 2 + t] = read_sa(other, TM / 2 + t);
        if (t < TN / 2) next.b[TN / 2 + t] = read_sb(other, TN / 2 + t);
      }
      if (t < C::kDmaB) dma_b(sb, mine, half, t);
    }
    mfma_half(first, half_c, f, now, TM / 2);
    schedule_region(std::integral_constant<int, 2>{}, std::integral_constant<int, kReads>{}, TM / 2);
#pragma unroll
    for (int i = 0; i < TM; ++i) asm volatile("" ::"v"(fn.a[i]));
#pragma unroll
    for (int j = 0; j < TN; ++j) asm volatile("" ::"v"(fn.b[j]));
    if constexpr (half == 1) {
#pragma unroll
      for (int i = 0; i < TM; ++i) asm volatile("" ::"v"(next.a[i]));
#pragma unroll
      for (int j = 0; j < TN; ++j) asm volatile("" ::"v"(next.b[j]));
    }
    __builtin_amdgcn_s_waitcnt(wait_vm(2 * kDmaStep + 2));
    __syncthreads();
  };
  auto chunk = [&](auto first) __attribute__((always_inline)) {
    step(first, Half0{}, f0, f1);
    step(std::false_type{}, Half1{}, f1, f0);
    advance();
    now = next;
    stage ^= 2 * C::kStage;
    slot ^= C::kScaleSlot;
  };
  for (uint32_t u = u_first; u < u_end; u += u_step) {
    const Unit U = decode(u);
    chunk(std::true_type{});
    for (uint32_t left = U.count - 1; left; --left) chunk(std::false_type{});
    epilogue(U);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm(0));  // no DMA outlives the workgroup's LDS
}

// The slices' sums in order, and the bias: four columns to a thread.
struct JoinArgs {
  const float* partials;
  uint32_t slices;
  int64_t m, n, ldp, ldo;
  const float* bias;
  void* out;
  uint32_t dtype;
};

template <typename T>
__device__ __forceinline__ void join(const JoinArgs& a) {
  const int64_t quads = a.ldp / 4;
  for (int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; q < a.m * quads;
       q += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = q / quads, c = 4 * (q - row * quads);
    if (c >= a.n) continue;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    const float* const p = a.partials + row * a.ldp + c;
    for (uint32_t s = 0; s < a.slices; s += 8) {  // eight loads in flight
      f32x4 v[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        v[i] = *reinterpret_cast<const f32x4*>(p + static_cast<int64_t>(min(s + i, a.slices - 1)) * a.m * a.ldp);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        if (s + i < a.slices) sum += v[i];
    }
    float bias[4], f[4];
    load4_or(a.bias, c, a.n, 0.0f, bias);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = sum[e] + bias[e];
    store4(static_cast<T*>(a.out) + row * a.ldo + c, a.n - c, f);
  }
}

__global__ __launch_bounds__(256) void mx4_join_kernel(JoinArgs a) {
  if (a.dtype == RNS8_MI355X_F32)
    join<float>(a);
  else if (a.dtype == RNS8_MI355X_F16)
    join<f16>(a);
  else
    join<bf16>(a);
}

template <int TM, int TN, int WN, int kResident>
hipError_t launch_cfg(TwoProducts p, const uint32_t* slices, int count, hipStream_t stream) {
  using Cf = Cfg<TM, TN, WN, kResident>;
  uint64_t all = 0;
  for (int i = 0; i < count; ++i) {
    TileArgs& a = p.product[i];
    const uint32_t tiles_m = (a.m + Cf::BM - 1) / Cf::BM, tiles_n = (a.n + Cf::BN - 1) / Cf::BN;
    const uint64_t tiles = static_cast<uint64_t>(tiles_m) * tiles_n, units = tiles * slices[i];
    all += units;
    if (units == 0 || all > 0x7FFFFFFFull) return hipErrorInvalidValue;
    a.units = static_cast<uint32_t>(units);
    a.tiles_m = tiles_m;
    a.tiles = make_div_u31(static_cast<uint32_t>(tiles));
    a.group = make_div_u31(static_cast<uint32_t>(Cf::kGroupM) * tiles_n);
    a.rows = make_div_u31(Cf::kGroupM);
    a.tail = make_div_u31(tiles_m - (tiles_m - 1) / Cf::kGroupM * Cf::kGroupM);
  }
  const uint32_t grid = static_cast<uint32_t>(persistent_grid(all, static_cast<uint64_t>(device_cu_count()) * kResident));
  if (count == 1)
    hipLaunchKernelGGL((mx4_tiles_kernel<Cf, OneProduct>), dim3(grid), dim3(Cf::kThreads), 0, stream, OneProduct{{p.product[0]}});
  else if constexpr (kResident > 1)
    hipLaunchKernelGGL((mx4_tiles_kernel<Cf, TwoProducts>),
                       dim3((p.product[0].units + 7) / 8 * 8 + (p.product[1].units + 7) / 8 * 8), dim3(Cf::kThreads), 0, stream, p);
  return hipGetLastError();
}

// A tile's costs in us, fitted to launches of 16 shapes from 100^3 to 8192^3 (bf16
// outputs, 1 to 32 slices each; the choices are within 0.4% of the best of them): a
// start (launch, first loads, epilogue) and one chunk of 256 columns on a CU that holds
// one workgroup, where few CUs do (`alone`) and where all do (`full`: clock and memory
// are shared), and per workgroup where it holds more (`shared`).
struct TileCost {
  uint32_t bm, bn, resident;
  double start, alone, full, shared;
};
constexpr TileCost kTileCosts[] = {{256, 256, 1, 10.8, 1.05, 1.92, 1.92},
                                   {128, 128, 2, 5.18, 0.47, 0.53, 0.58},
                                   {64, 64, 4, 4.16, 0.28, 0.31, 0.21}};

double tile_cost(const TileCost& c, int64_t m, int64_t n, int64_t k, double units, int64_t slice_chunks) {
  const double per_cu = std::ceil(units / 256);
  double chunk = c.alone + (c.full - c.alone) * std::min(1.0, units / 256);
  if (per_cu > 1) chunk = std::max(chunk, c.shared * per_cu);
  const double operands = static_cast<double>(m + n) * static_cast<double>(k) * 0.53 / kBytesPerUs;
  return c.start + std::max(static_cast<double>(slice_chunks) * chunk, operands);
}

// The best cut of a product into this kind of tile, if it beats `best`.
void choose_slices(const TileCost& c, int64_t m, int64_t n, int64_t k, Mx4Tiles& best) {
  const int64_t chunks = mx4_chunks(k);
  const double tiles = static_cast<double>((m + c.bm - 1) / c.bm) * static_cast<double>((n + c.bn - 1) / c.bn);
  for (const int64_t wanted : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
    if (wanted > 1 && chunks < 2 * wanted) continue;  // slices of two chunks at least
    const int64_t slice_chunks = (chunks + wanted - 1) / wanted, s = (chunks + slice_chunks - 1) / slice_chunks;
    const double units = tiles * static_cast<double>(s);
    if (units > 0x3FFFFFFF) continue;
    double cost = tile_cost(c, m, n, k, units, slice_chunks);
    // the join: a launch, and the partial sums written and read
    if (s > 1)
      cost += 2.2 + 0.03 * static_cast<double>(s) +
              static_cast<double>(s) * static_cast<double>(m) * static_cast<double>(n) * 8 / 4e6;
    if (best.cost != 0 && cost >= best.cost) continue;
    best.cost = cost;
    best.bm = c.bm;
    best.bn = c.bn;
    best.slices = static_cast<uint32_t>(s);
    best.slice_chunks = slice_chunks;
  }
  best.ldp = (n + 3) / 4 * 4;
  best.bytes = best.slices > 1 ? static_cast<uint64_t>(best.slices) * static_cast<uint64_t>(m) *
                                     static_cast<uint64_t>(best.ldp) * sizeof(float)
                               : 0u;
}

}  // namespace

Mx4Tiles choose_mx4_tiles(int64_t m, int64_t n, int64_t k) {
  Mx4Tiles best{};
  for (const TileCost& c : kTileCosts) choose_slices(c, m, n, k, best);
  return best;
}

namespace {

// Tiles for two products in one launch, where both fit on the chip at once and that is
// predicted to take less than one after the other.
bool choose_pair(const Mx4Gemm (&g)[2], Mx4Tiles (&tiles)[2]) {
  double least = 0;
  for (const Mx4Gemm& one : g) least += choose_mx4_tiles(one.m, one.n, one.k).cost;
  bool pair = false;
  for (const TileCost& c : kTileCosts) {
    Mx4Tiles t[2]{};
    double units = 0;
    for (int i = 0; i < 2; ++i) {
      choose_slices(c, g[i].m, g[i].n, g[i].k, t[i]);
      units += static_cast<double>((g[i].m + c.bm - 1) / c.bm) * static_cast<double>((g[i].n + c.bn - 1) / c.bn) * t[i].slices;
    }
    const double together = std::max(t[0].cost, t[1].cost);
    // (not the largest tile, whose workgroups fill a CU: 3000 x 2500 x 2500 65 us with it, 60 apart)
    if (t[0].cost == 0 || t[1].cost == 0 || c.resident < 2 || units > 256.0 * c.resident || together >= least) continue;
    least = together;
    pair = true;
    tiles[0] = t[0];
    tiles[1] = t[1];
  }
  return pair;
}

// The kernel's arguments, if it can take the product.
bool tile_args(const Mx4Gemm& g, const Mx4Tiles& t, float* partials, TileArgs& a) {
  if (g.m < 1 || g.n < 1 || g.k < 1 || g.m > kMaxMx4Size || g.n > kMaxMx4Size || g.k > kMaxMx4Sum ||
      g.dtype > RNS8_MI355X_BF16 || reinterpret_cast<uintptr_t>(g.a) % 16 || reinterpret_cast<uintptr_t>(g.b) % 16 ||
      t.slices < 1 || t.slice_chunks < 1 || (t.slices > 1 && !partials))
    return false;
  const int64_t chunks = mx4_chunks(g.k);
  // (every slice has a chunk)
  if (t.slice_chunks * (t.slices - 1) >= chunks || t.slice_chunks * t.slices < chunks) return false;
  a.a = g.a;
  a.b = g.b;
  a.bias = g.bias;
  a.out = g.out;
  a.partials = t.slices > 1 ? partials : nullptr;
  a.ldo = g.ldo;
  a.ldp = t.ldp;
  a.m = static_cast<uint32_t>(g.m);
  a.n = static_cast<uint32_t>(g.n);
  a.groups_m = static_cast<uint32_t>(mx4_groups(g.m));
  a.groups_n = static_cast<uint32_t>(mx4_groups(g.n));
  a.chunks = static_cast<uint32_t>(chunks);
  a.stride = static_cast<uint32_t>(mx4_stride(g.k));
  a.dtype = g.dtype;
  a.slice_chunks = static_cast<uint32_t>(t.slice_chunks);
  return true;
}

// (no slices: the bias alone)
hipError_t launch_join(const Mx4Gemm& g, const float* partials, uint32_t slices, int64_t ldp, hipStream_t stream) {
  const JoinArgs j{partials, slices, g.m, g.n, ldp, g.ldo, g.bias, g.out, g.dtype};
  const int64_t blocks = std::min<int64_t>((g.m * (ldp / 4) + 255) / 256, 1 << 20);
  hipLaunchKernelGGL(mx4_join_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, j);
  return hipGetLastError();
}

// Products of one kind of tile in one launch, then the joins of those cut into slices.
hipError_t launch_tiles(const Mx4Gemm* g, const Mx4Tiles* t, float* const* partials, int count, const Mx4Sums& sums,
                        hipStream_t stream) {
  TwoProducts p{};
  p.sums = sums;
  uint32_t slices[2] = {};
  for (int i = 0; i < count; ++i) {
    if (t[i].bm != t[0].bm || t[i].bn != t[0].bn || !tile_args(g[i], t[i], partials[i], p.product[i])) return hipErrorInvalidValue;
    slices[i] = t[i].slices;
  }
  hipError_t e = hipErrorInvalidValue;
  if (t[0].bm == 256 && count == 1) e = launch_cfg<8, 8, 2, 1>(p, slices, count, stream);
  if (t[0].bm == 128) e = launch_cfg<4, 4, 2, 2>(p, slices, count, stream);
  if (t[0].bm == 64) e = launch_cfg<2, 4, 1, 4>(p, slices, count, stream);
  for (int i = 0; i < count && e == hipSuccess; ++i)
    if (slices[i] > 1) e = launch_join(g[i], partials[i], slices[i], t[i].ldp, stream);
  return e;
}

// Few rows read b once however many waves share it.
constexpr int64_t kMaxRowsChannels = int64_t{1} << 26;
bool rows_take(int64_t m, int64_t n) { return m <= kMx4Rows && n <= kMaxRowsChannels; }
bool tiles_take(const Mx4Gemm& g) { return g.m > 0 && g.n > 0 && g.k > 0 && !g.x && !rows_take(g.m, g.n); }

// Whether one launch takes both, and their tiles.
bool as_pair(const Mx4Gemm (&g)[2], Mx4Tiles (&tiles)[2]) {
  return tiles_take(g[0]) && tiles_take(g[1]) && choose_pair(g, tiles);
}

}  // namespace

bool linear_mx4_in_one_kernel(int64_t m, int64_t n) { return m <= kMx4FusedRows && n <= kMaxRowsChannels; }

uint64_t gemm_mx4_bytes(int64_t m, int64_t n, int64_t k) {
  return m == 0 || n == 0 || k == 0 || rows_take(m, n) ? 0u : choose_mx4_tiles(m, n, k).bytes;
}

hipError_t launch_gemm_mx4(const Mx4Gemm& g, void* workspace, hipStream_t stream) {
  if (g.m == 0 || g.n == 0) return hipSuccess;
  if (g.k == 0) return launch_join(g, nullptr, 0, (g.n + 3) / 4 * 4, stream);
  if (!tiles_take(g)) return launch_mx4_rows(g, stream);
  const Mx4Tiles t = choose_mx4_tiles(g.m, g.n, g.k);
  float* const partials = static_cast<float*>(workspace);
  return launch_tiles(&g, &t, &partials, 1, Mx4Sums{}, stream);
}

void gemm_mx4_pair_bytes(const Mx4Gemm (&g)[2], uint64_t (&bytes)[2]) {
  Mx4Tiles t[2];
  const bool pair = as_pair(g, t);
  for (int i = 0; i < 2; ++i) bytes[i] = pair ? t[i].bytes : gemm_mx4_bytes(g[i].m, g[i].n, g[i].k);
}

hipError_t launch_gemm_mx4_pair(const Mx4Gemm (&g)[2], void* const (&workspaces)[2], const Mx4Sums& sums, hipStream_t stream) {
  Mx4Tiles t[2];
  if (as_pair(g, t)) {
    // the longer sums first: as the last units of the grid they would start last
    const int first = t[1].slice_chunks > t[0].slice_chunks ? 1 : 0;
    const Mx4Gemm products[2] = {g[first], g[1 - first]};
    const Mx4Tiles tiles[2] = {t[first], t[1 - first]};
    float* const partials[2] = {static_cast<float*>(workspaces[first]), static_cast<float*>(workspaces[1 - first])};
    return launch_tiles(products, tiles, partials, 2, sums, stream);
  }
  hipError_t e = sums.out ? launch_sum_partials(sums, stream) : hipSuccess;
  for (int i = 0; i < 2 && e == hipSuccess; ++i) e = launch_gemm_mx4(g[i], workspaces[i], stream);
  return e;
}

}  // namespace rns8x
