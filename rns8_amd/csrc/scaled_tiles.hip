// Tile kernels of the scaled 8-bit product (gfx950).
//
//   out[i][j] = a_scale[i] b_scale[j] sum_k a[i][k] b(k, j) + bias[j]
//
// Bound by the matrix cores where the product is large. The structure is that
// of the plane GEMM (gemm.hip): a persistent grid over output tiles (and K
// slices), each XCD a contiguous share; K in steps of 64 through LDS rings
// filled by buffer-load DMA four steps ahead, also across tile boundaries; one
// counted wait and one barrier per step; v_mfma_i32_16x16x64_i8 with the next
// step's fragments read beside it. What differs:
//   * b may be stored n x k (weights): its stages then hold BN rows of 64
//     K-contiguous bytes and its fragments are single ds_read_b128. Stored k x n
//     (both gradients), its stages and transpose reads are the plane GEMM's.
//   * k ends anywhere: lanes whose 16-byte chunk of a lies past the slice's K
//     load zero (an offset past the buffer), so b's bytes there do not matter.
//   * The accumulators are the exact sums: the epilogue converts each once to
//     32 bits, applies both scales and the bias, and rounds once. Neighbouring
//     lane groups swap halves so that 16-bit outputs leave in 16-byte stores.
//   * Few tiles: K is cut into slices whose int32 sums go to a workspace; a
//     second kernel adds them in 64 bits and runs the epilogue. The result does
//     not depend on the cut.
//   * Both gradients of a linear layer run in one launch (TilePair).
// Measured (bf16 outputs, medians): 8192^3 408 us (2.7 POP/s, 0.66 of the cycles in
// MFMA), 4096^3 61 us (2.25 POP/s, 0.46 of them: one tile to a CU, nothing beside its
// start and epilogue), 1000 x 1101 x 903 9.5 us.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dma.hpp"
#include "int_ops.hpp"
#include "kernels.hpp"
#include "scaled_epilogue.hpp"
#include "scaled_gemm.hpp"
#include "tables.hpp"

namespace rns8x {
namespace {

typedef int v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i lds_v2i;

__device__ __forceinline__ lds_v2i* as_lds_v2i(const int8_t* p) { return (lds_v2i*)(const_cast<int8_t*>(p)); }

// kWaves waves (2 x WN) each own TM x TN blocks of 16 x 16 outputs: a tile of
// (32 TM) x (16 TN WN). a is staged in chunks of two steps (whole cache lines),
// three deep; b in steps, four deep.
template <int TM_, int TN_, int WN_, bool kInner_>
struct Cfg {
  static constexpr int TM = TM_, TN = TN_, WN = WN_;
  static constexpr bool kInner = kInner_;
  static constexpr int kWaves = 2 * WN, kThreads = 64 * kWaves;
  static constexpr int BM = 32 * TM, BN = 16 * TN * WN, BK = 64;
  static constexpr int kBufA = BM * 2 * BK, kBufB = BK * BN;
  static constexpr int kSlotsA = 3, kStagesB = 4;
  static constexpr int kLds = kSlotsA * kBufA + kStagesB * kBufB;
  static constexpr int kDmaA = kBufA / 2048 / kWaves, kDmaB = kBufB / 1024 / kWaves;  // 1 KB blocks per wave and step
  static constexpr int kGroupM = 1024 / BM;  // tile rows per L2 reuse group
  static constexpr int kChunksB = kInner ? BN / 16 : 4;           // 16-byte chunks per b stage row
  static constexpr int kRowsPerBlockB = kInner ? 1024 / BN : 16;  // stage rows per 1 KB block
  static_assert(kDmaA >= 1 && kDmaA <= 4 && kDmaB >= 1 && kDmaB <= 4, "DMA blocks");
  static_assert(1024 % BN == 0 && TM % 2 == 0 && TN % 4 == 0, "tile config");
  static_assert(kLds <= 160 * 1024, "LDS per workgroup");
};

// Stage rows are XOR-swizzled in 16-byte chunks, applied on the global side of
// the DMA. a: rows of 8 chunks, 16 rows of one chunk read at a time. b stored n
// x k: rows of 4 chunks, four rows to a bank row, so every fourth row turns. b
// stored k x n: as in gemm.hip.
__device__ __forceinline__ int swizzle_a(int row, int chunk) { return chunk ^ ((row ^ ((row >> 3) & 1)) & 7); }
template <typename C>
__device__ __forceinline__ int swizzle_b(int row, int chunk) {
  if constexpr (!C::kInner) {
    return chunk ^ ((row >> 2) & 3);
  } else {
    const int x = row & 7, b4 = (row >> 4) & 1;
    if constexpr (C::BN == 256)
      return chunk ^ ((((2 * x) & 15) | (x >> 2)) ^ b4);
    else if constexpr (C::BN == 128)
      return chunk ^ (x ^ b4);
    else
      return chunk ^ (((x >> 1) ^ b4) & 3);
  }
}

template <int kId, int kPer, int kReads>
__device__ __forceinline__ void sched_slots() {
  if constexpr (kReads > 0) {
    __builtin_amdgcn_sched_group_barrier(0x008, kPer, kId);  // MFMA
    __builtin_amdgcn_sched_group_barrier(0x100, 1, kId);     // DS read
    sched_slots<kId, kPer, kReads - 1>();
  }
}

struct TileArgs {
  const int8_t *a, *b;
  const float *a_scale, *b_scale, *bias;
  void* out;
  int32_t* partials;  // [slices][m][ldp], or NULL
  int64_t ldo, ldp;
  uint32_t m, n, lda, ldb;
  uint32_t k16;  // k rounded up to 16
  uint32_t k;
  uint32_t dtype;
  // units: slice-major, tiles in groups of kGroupM tile rows
  uint32_t units, tiles_m;
  DivU31 tiles, group, rows, tail;
  uint32_t k_slice;
  uint32_t pairs;  // chunks of two steps that every unit runs
};

__device__ __forceinline__ uint32_t div_u31(uint32_t n, DivU31 v) { return __umulhi(n << 1, v.mul) >> v.shift; }

// One product or, with b stored k x n, two of one tile: the first `blocks`
// workgroups are the first's. Two small ones share the chip, and of two large ones
// the second's tiles start as the first's end (with loads of their own: the LDS of a
// CU holds one workgroup of the largest tiles, so nothing of the second's is on its way
// before). Both gradients of a layer of 118 x 8
// x 35 (with their quantization) 15.0 us in two launches, 10.2 in one; of 1024^3
// 29.3 and 23.1; of 4096^3 172.8 and 170.4. (With b stored n x k the kernel takes
// the first's arguments without waiting for `blocks`, 0.5 us.)
struct TilePair {
  TileArgs product[2];
  uint32_t blocks;
};

template <typename C, int kMinBlocks>
__global__ __launch_bounds__(C::kThreads, kMinBlocks) void scaled_tiles_kernel(TilePair pair_args) {
  constexpr int TM = C::TM, TN = C::TN, BM = C::BM, BN = C::BN, BK = C::BK;
  __shared__ __attribute__((aligned(16))) int8_t lds[C::kLds];

  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave_m = wave / C::WN;
  const int wave_n = wave % C::WN;

  const bool second = C::kInner && blockIdx.x >= pair_args.blocks;
  const TileArgs& args = pair_args.product[second ? 1 : 0];
  const uint32_t grid = !C::kInner ? gridDim.x : second ? gridDim.x - pair_args.blocks : pair_args.blocks;
  const uint32_t block = second ? blockIdx.x - pair_args.blocks : blockIdx.x;
  uint32_t u_first, u_step, u_end;
  if ((grid & 7u) == 0u) {
    const uint32_t xcd = block & 7u;
    u_first = static_cast<uint32_t>((static_cast<uint64_t>(xcd) * args.units) / 8) + (block >> 3);
    u_end = static_cast<uint32_t>((static_cast<uint64_t>(xcd + 1) * args.units) / 8);
    u_step = grid >> 3;
  } else {
    u_first = block;
    u_end = args.units;
    u_step = grid;
  }
  u_first = __builtin_amdgcn_readfirstlane(u_first);
  u_end = __builtin_amdgcn_readfirstlane(u_end);
  if (u_first >= u_end) return;

  struct Unit {
    uint32_t slice, m0, n0, kbeg, kend;  // kend: rounded up to 16 where b is n x k
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
    U.kbeg = U.slice * args.k_slice;
    U.kend = min(C::kInner ? args.k : args.k16, U.kbeg + args.k_slice);
    return U;
  };

  // ---- global -> LDS by DMA: lane offsets fixed, resources move with K ------------
  const uint32_t lda = args.lda, ldb = args.ldb;
  uint32_t a_voff[2 * C::kDmaA];
  uint32_t b_voff[C::kDmaB];
  int32_t a_koff[2];  // this lane's K offset in a chunk, in even and in odd blocks
#pragma unroll
  for (int i = 0; i < 2 * C::kDmaA; ++i) {
    const int row = 8 * (wave * 2 * C::kDmaA + i) + (lane >> 3);
    a_voff[i] = static_cast<uint32_t>(row) * lda + static_cast<uint32_t>(16 * swizzle_a(row, lane & 7));
    if (i < 2) a_koff[i] = 16 * swizzle_a(row, lane & 7);
  }
#pragma unroll
  for (int i = 0; i < C::kDmaB; ++i) {
    const int row = C::kRowsPerBlockB * (wave * C::kDmaB + i) + lane / C::kChunksB;
    b_voff[i] = static_cast<uint32_t>(row) * ldb + static_cast<uint32_t>(16 * swizzle_b<C>(row, lane % C::kChunksB));
  }
  const uint32_t lds_a = lds_address(lds) + static_cast<uint32_t>(wave * 2 * C::kDmaA * 1024);
  const uint32_t lds_b = lds_address(lds) + static_cast<uint32_t>(C::kSlotsA * C::kBufA + wave * C::kDmaB * 1024);

  // The chunk whose DMA is issued next, two chunks ahead of the compute
  // position; past a unit's K and past the last unit everything loads zero.
  struct Cursor {
    const int8_t *a, *b;
    int32_t a_n;    // bytes of a from `a` to the end of the unit's last row
    int32_t k_rem;  // K left in the unit
    int32_t b_n;    // n x k: bytes of b from `b` on; k x n: from the unit's first column in a row to the row's end
    int32_t dec;    // 2 BK, or 0 past the last unit (the others stay 0)
  };
  auto cursor_of = [&](const Unit& U, bool live) {
    const uint32_t a_rows = min(static_cast<uint32_t>(BM), args.m - U.m0);
    Cursor c;
    c.a = args.a + static_cast<uint64_t>(U.m0) * lda + U.kbeg;
    c.a_n = live ? static_cast<int32_t>((a_rows - 1u) * lda + args.k16 - U.kbeg) : 0;
    c.k_rem = live ? static_cast<int32_t>(U.kend - U.kbeg) : 0;
    c.dec = live ? 2 * BK : 0;
    if constexpr (C::kInner) {
      c.b = args.b + static_cast<uint64_t>(U.kbeg) * ldb + U.n0;
      c.b_n = static_cast<int32_t>(((args.n + 15u) & ~15u) - U.n0);
    } else {
      const uint32_t b_rows = min(static_cast<uint32_t>(BN), args.n - U.n0);
      c.b = args.b + static_cast<uint64_t>(U.n0) * ldb + U.kbeg;
      c.b_n = live ? static_cast<int32_t>((b_rows - 1u) * ldb + args.k16 - U.kbeg) : 0;
    }
    return c;
  };
  Cursor cur = cursor_of(decode(u_first), true);
  // One value to a thread of the first unit's scales and biases, so that its
  // epilogue finds them in the L2. (Kept to the end: a use waits for the loads, and
  // for the DMA behind them.)
  float touched[3] = {0.0f, 0.0f, 0.0f};
  if (!args.partials) {
    const Unit U = decode(u_first);
    if (args.a_scale) touched[0] = args.a_scale[min(U.m0 + static_cast<uint32_t>(tid) % BM, args.m - 1)];
    if (args.b_scale) touched[1] = args.b_scale[min(U.n0 + static_cast<uint32_t>(tid) % BN, args.n - 1)];
    if (args.bias) touched[2] = args.bias[min(U.n0 + static_cast<uint32_t>(tid) % BN, args.n - 1)];
  }
  const uint64_t b_step = C::kInner ? static_cast<uint64_t>(BK) * ldb : BK;
  auto src_a = [&]() { return buffer_rsrc(cur.a, cur.a_n); };
  auto src_b = [&](int half) {
    if constexpr (C::kInner) {
      // the step's k rows; a's bytes past k meet zeros
      const int32_t rows = min(max(cur.k_rem - half * BK, 0), static_cast<int32_t>(BK));
      return buffer_rsrc(cur.b + (half ? b_step : 0u), rows ? (rows - 1) * static_cast<int32_t>(ldb) + cur.b_n : 0);
    } else {
      return buffer_rsrc(cur.b + (half ? b_step : 0u), max(cur.b_n - half * BK, 0));
    }
  };
  auto cursor_advance = [&]() {
    cur.a += 2 * BK;
    cur.b += 2 * b_step;
    cur.a_n = max(cur.a_n - cur.dec, 0);
    cur.k_rem = max(cur.k_rem - cur.dec, 0);
    if constexpr (!C::kInner) cur.b_n = max(cur.b_n - cur.dec, 0);
  };
  auto dma_a = [&](v4i src, uint32_t slot, int half, int i) {
    const int block = half * C::kDmaA + i;
    uint32_t off = a_voff[block];
    if constexpr (!C::kInner) off = a_koff[block & 1] < cur.k_rem ? off : 0x80000000u;
    dma16_block(__builtin_amdgcn_readfirstlane(lds_a + slot), block, off, src);
  };
  auto dma_b = [&](v4i src, uint32_t stage, int i) {
    dma16_block(__builtin_amdgcn_readfirstlane(lds_b + stage), i, b_voff[i], src);
  };

  // ---- fragments: 16 K-contiguous bytes of a row (a) or column (b) per lane -------
  const int frag_row = lane & 15;
  const int frag_k = lane >> 4;
  struct Frags {
    v4i a[TM];
    v4i b[TN];
  };
  auto read_a = [&](uint32_t slot, int half, int i) {
    const int r = wave_m * (16 * TM) + 16 * i + frag_row;
    return *reinterpret_cast<const v4i*>(lds + slot + r * (2 * BK) + swizzle_a(frag_row, 4 * half + frag_k) * 16);
  };
  auto read_b = [&](uint32_t stage, int j) {
    const int8_t* const sb = lds + C::kSlotsA * C::kBufA + stage;
    if constexpr (C::kInner) {
      const int chunk = wave_n * TN + j;
      const int k = 16 * frag_k + (frag_row >> 1);
      const int8_t* const at = sb + k * BN + swizzle_b<C>(k, chunk) * 16 + 8 * (frag_row & 1);
      const v2i lo = __builtin_amdgcn_ds_read_tr8_b64_v2i32(as_lds_v2i(at));
      const v2i hi = __builtin_amdgcn_ds_read_tr8_b64_v2i32(as_lds_v2i(at + 8 * BN));
      return v4i{lo[0], lo[1], hi[0], hi[1]};
    } else {
      const int row = wave_n * (16 * TN) + 16 * j + frag_row;
      return *reinterpret_cast<const v4i*>(sb + row * BK + swizzle_b<C>(frag_row, frag_k) * 16);
    }
  };

  v4i acc[TM][TN];
  auto mfma_half = [&](auto first, const Frags& f, int i0) __attribute__((always_inline)) {
#pragma unroll
    for (int ii = 0; ii < TM / 2; ++ii)
#pragma unroll
      for (int jj = 0; jj < TN; ++jj) {
        const int i = i0 + ii, j = (ii & 1) ? TN - 1 - jj : jj;
        const v4i start = {0, 0, 0, 0};
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.b[j], f.a[i], decltype(first)::value ? start : acc[i][j],
                                                          0, 0, 0);
      }
  };
  constexpr int kMfma = TM / 2 * TN;
  constexpr int kReadsB = C::kInner ? 2 : 1;  // LDS instructions per b fragment
  constexpr int kReads = TM / 2 + kReadsB * TN / 2;
  constexpr int kPerSlot = kMfma * 3 / 4 / kReads > 0 ? kMfma * 3 / 4 / kReads : 1;
  auto schedule_region = [&](auto id, int i0) __attribute__((always_inline)) {
    constexpr int kId = decltype(id)::value;
#pragma unroll
    for (int i = 0; i < TM / 2; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) asm volatile("" ::"a"(acc[i0 + i][j]));
    sched_slots<kId, kPerSlot, kReads>();
    if constexpr (kMfma > kPerSlot * kReads)
      __builtin_amdgcn_sched_group_barrier(0x008, kMfma - kPerSlot * kReads, kId);
    __builtin_amdgcn_sched_barrier(0);
  };

  // ---- epilogue: element e of acc[i][j] is row m0 + 16 (wave_m TM + i) + (lane &
  // 15), column n0 + 16 (wave_n TN + j) + 4 (lane >> 4) + e -----------------------
  auto epilogue = [&](const Unit& U) {
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");  // the reads below are asm: MFMA results settle first
    const int64_t row0 = static_cast<int64_t>(U.m0) + wave_m * (16 * TM) + frag_row;
    const int64_t col0 = static_cast<int64_t>(U.n0) + wave_n * (16 * TN);
    const int64_t m = args.m, n = args.n;
    if (args.partials) {
      int32_t* const base = args.partials + (static_cast<int64_t>(U.slice) * m + row0) * args.ldp + col0 + 4 * frag_k;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const Acc4 v = acc_read4(acc[i][j]);
          if (row0 + 16 * i < m && col0 + 16 * j + 4 * frag_k < args.ldp)
            *reinterpret_cast<v4i*>(base + 16 * i * args.ldp + 16 * j) =
                v4i{static_cast<int>(v.v[0]), static_cast<int>(v.v[1]), static_cast<int>(v.v[2]),
                    static_cast<int>(v.v[3])};
        }
      return;
    }
    float sa[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) sa[i] = args.a_scale && row0 + 16 * i < m ? args.a_scale[row0 + 16 * i] : 1.0f;
    auto value = [&](const Acc4& v, int i, const float (&sb)[4], const float (&bias)[4], float (&f)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = scaled_value(static_cast<int>(v.v[e]), sa[i], sb[e], bias[e]);
    };
    auto write = [&](auto type) {
      using T = decltype(type);
      T* const out = static_cast<T*>(args.out);
#pragma unroll
      for (int j = 0; j < TN; j += 2) {
        float sb[2][4], bias[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          load4_or(args.b_scale, col0 + 16 * (j + h) + 4 * frag_k, n, 1.0f, sb[h]);
          load4_or(args.bias, col0 + 16 * (j + h) + 4 * frag_k, n, 0.0f, bias[h]);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int64_t row = row0 + 16 * i;
          float f[2][4];
          value(acc_read4(acc[i][j]), i, sb[0], bias[0], f[0]);
          value(acc_read4(acc[i][j + 1]), i, sb[1], bias[1], f[1]);
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int64_t c = col0 + 16 * (j + h) + 4 * frag_k;
              if (row < m && c < n) store4(out + row * args.ldo + c, n - c, f[h]);
            }
          } else {
            // Two blocks' 8-byte pieces: after swapping odd with even lane
            // groups, groups 0 and 2 hold block j's columns 0-7 and 8-15 of
            // the row, groups 1 and 3 block j + 1's.
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
            const int64_t c = col0 + 16 * (j + (frag_k & 1)) + 8 * (frag_k >> 1);
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

  // ---- pipeline (the plane GEMM's: see there for the order of its hazards) ----------
  constexpr int kDmaStep = C::kDmaA + C::kDmaB;
  Frags f0, f1;
  uint32_t slot0 = 0, slot1 = C::kBufA, slot2 = 2 * C::kBufA;
  uint32_t stage0 = 0, stage2 = 2 * C::kBufB;
  const bool one_chunk = args.pairs == 1u;
  auto unit_cursor = [&](uint32_t u) { return cursor_of(decode(min(u, u_end - 1)), u < u_end); };
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const v4i sa = src_a();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const v4i sb = src_b(half);
#pragma unroll
      for (int i = 0; i < C::kDmaA; ++i) dma_a(sa, c * C::kBufA, half, i);
#pragma unroll
      for (int i = 0; i < C::kDmaB; ++i) dma_b(sb, (2 * c + half) * C::kBufB, i);
    }
    cursor_advance();
    if (c == 0 && one_chunk) cur = unit_cursor(u_first + u_step);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm(2 * kDmaStep));  // chunk 0 landed
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TM; ++i) f0.a[i] = read_a(0, 0, i);
#pragma unroll
  for (int j = 0; j < TN; ++j) f0.b[j] = read_b(0, j);
  __syncthreads();  // b stage 0 is read: position 4 may overwrite it
  auto step = [&](auto first, auto half_c, const Frags& f, Frags& fn) __attribute__((always_inline)) {
    constexpr int half = decltype(half_c)::value;
    constexpr int kRegionLen = TM / 2 > TN / 2 ? (TM / 2 > 4 ? TM / 2 : 4) : (TN / 2 > 4 ? TN / 2 : 4);
    const uint32_t next_slot = half ? slot1 : slot0;
    const uint32_t next_stage = half ? stage2 : stage0 + C::kBufB;
    const uint32_t dma_stage = stage0 + half * C::kBufB;
    const v4i sa = src_a(), sb = src_b(half);
#pragma unroll
    for (int t = 0; t < kRegionLen; ++t) {
      if (t < TM / 2) fn.a[t] = read_a(next_slot, half ^ 1, t);
      if (t < TN / 2) fn.b[t] = read_b(next_stage, t);
      if (t < C::kDmaA) dma_a(sa, slot2, half, t);
    }
    mfma_half(first, f, 0);
    schedule_region(std::integral_constant<int, 1>{}, 0);
#pragma unroll
    for (int t = 0; t < kRegionLen; ++t) {
      if (t < TM / 2) fn.a[TM / 2 + t] = read_a(next_slot, half ^ 1, TM / 2 + t);
      if (t < TN / 2) fn.b[TN / 2 + t] = read_b(next_stage, TN / 2 + t);
      if (t < C::kDmaB) dma_b(sb, dma_stage, t);
    }
    mfma_half(first, f, TM / 2);
    if constexpr (half == 1) cursor_advance();
    schedule_region(std::integral_constant<int, 2>{}, TM / 2);
#pragma unroll
    for (int i = 0; i < TM; ++i) asm volatile("" ::"v"(fn.a[i]));
#pragma unroll
    for (int j = 0; j < TN; ++j) asm volatile("" ::"v"(fn.b[j]));
    __builtin_amdgcn_s_waitcnt(wait_vm(half ? 2 * kDmaStep : kDmaStep + C::kDmaB));
    __syncthreads();
  };
  auto pair = [&](auto first) __attribute__((always_inline)) {
    step(first, std::integral_constant<int, 0>{}, f0, f1);
    step(std::false_type{}, std::integral_constant<int, 1>{}, f1, f0);
    const uint32_t s = slot0;
    slot0 = slot1;
    slot1 = slot2;
    slot2 = s;
    stage0 ^= 2 * C::kBufB;
    stage2 ^= 2 * C::kBufB;
  };
  for (uint32_t u = u_first; u < u_end; u += u_step) {
    const Unit U = decode(u);
    const Cursor next = unit_cursor(u + (one_chunk ? 2 * u_step : u_step));
    auto enter_next = [&](bool enter) {
      cur.a = enter ? next.a : cur.a;
      cur.b = enter ? next.b : cur.b;
      cur.a_n = enter ? next.a_n : cur.a_n;
      cur.k_rem = enter ? next.k_rem : cur.k_rem;
      cur.b_n = enter ? next.b_n : cur.b_n;
      cur.dec = enter ? next.dec : cur.dec;
    };
    uint32_t left = args.pairs;
    enter_next(left <= 2u);
    pair(std::true_type{});
    for (--left; left; --left) {
      enter_next(left == 2u);
      pair(std::false_type{});
    }
    epilogue(U);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm(0));  // no DMA outlives the workgroup's LDS
  asm volatile("" ::"v"(touched[0]), "v"(touched[1]), "v"(touched[2]));
}

// The slices' sums in 64 bits, then the epilogue: four columns to a thread.
struct JoinArgs {
  const int32_t* partials;
  uint32_t slices;
  int64_t m, n, ldp, ldo;
  const float *a_scale, *b_scale, *bias;
  void* out;
  uint32_t dtype;
};

struct JoinPair {
  JoinArgs product[2];
  uint32_t blocks;  // the first's
};

template <typename T>
__device__ __forceinline__ void join_slices(const JoinArgs& a, uint32_t block, uint32_t blocks) {
  const int64_t quads = a.ldp / 4;
  for (int64_t q = static_cast<int64_t>(block) * 256 + threadIdx.x; q < a.m * quads;
       q += static_cast<int64_t>(blocks) * 256) {
    const int64_t row = q / quads, c = 4 * (q - row * quads);
    if (c >= a.n) continue;
    int64_t sum[4] = {};
    const int32_t* const p = a.partials + row * a.ldp + c;
    for (uint32_t s = 0; s < a.slices; s += 8) {  // eight loads in flight
      v4i v[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        v[i] = *reinterpret_cast<const v4i*>(p + static_cast<int64_t>(min(s + i, a.slices - 1)) * a.m * a.ldp);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += s + i < a.slices ? v[i][e] : 0;
    }
    const float sa = a.a_scale ? a.a_scale[row] : 1.0f;
    float sb[4], bias[4], f[4];
    load4_or(a.b_scale, c, a.n, 1.0f, sb);
    load4_or(a.bias, c, a.n, 0.0f, bias);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = scaled_value(sum[e], sa, sb[e], bias[e]);
    store4(static_cast<T*>(a.out) + row * a.ldo + c, a.n - c, f);
  }
}

__global__ __launch_bounds__(256) void join_slices_kernel(JoinPair p) {
  const bool second = blockIdx.x >= p.blocks;
  const JoinArgs& a = p.product[second ? 1 : 0];
  const uint32_t block = second ? blockIdx.x - p.blocks : blockIdx.x;
  const uint32_t blocks = second ? gridDim.x - p.blocks : p.blocks;
  if (a.dtype == RNS8_MI355X_F32)
    join_slices<float>(a, block, blocks);
  else if (a.dtype == RNS8_MI355X_F16)
    join_slices<f16>(a, block, blocks);
  else
    join_slices<bf16>(a, block, blocks);
}

// The product's tiles and units; the workgroups it takes (0: too many units).
template <typename Cf, int kMinBlocks>
uint32_t split_units(TileArgs& a, uint32_t slices) {
  const uint32_t tiles_m = (a.m + Cf::BM - 1) / Cf::BM, tiles_n = (a.n + Cf::BN - 1) / Cf::BN;
  const uint64_t tiles = static_cast<uint64_t>(tiles_m) * tiles_n, units = tiles * slices;
  if (units == 0 || units > 0x7FFFFFFFull) return 0;
  a.units = static_cast<uint32_t>(units);
  a.tiles_m = tiles_m;
  a.tiles = make_div_u31(static_cast<uint32_t>(tiles));
  a.group = make_div_u31(static_cast<uint32_t>(Cf::kGroupM) * tiles_n);
  a.rows = make_div_u31(Cf::kGroupM);
  a.tail = make_div_u31(tiles_m - (tiles_m - 1) / Cf::kGroupM * Cf::kGroupM);
  return static_cast<uint32_t>(persistent_grid(units, static_cast<uint64_t>(device_cu_count()) * kMinBlocks));
}

template <int TM, int TN, int WN, int kMinBlocks, bool kInner>
hipError_t launch_cfg(TilePair p, const uint32_t* slices, int count, hipStream_t stream) {
  using Cf = Cfg<TM, TN, WN, kInner>;
  p.blocks = split_units<Cf, kMinBlocks>(p.product[0], slices[0]);
  const uint32_t more = count > 1 ? split_units<Cf, kMinBlocks>(p.product[1], slices[1]) : 0;
  if (p.blocks == 0 || (count > 1 && more == 0)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((scaled_tiles_kernel<Cf, kMinBlocks>), dim3(p.blocks + more), dim3(Cf::kThreads), 0, stream, p);
  return hipGetLastError();
}

template <bool kInner>
hipError_t launch_tile(const TilePair& p, const TileShape& s, const uint32_t* slices, int count, hipStream_t stream) {
  if (s.bm == 256 && s.bn == 256) return launch_cfg<8, 8, 2, 1, kInner>(p, slices, count, stream);
  if (s.bm == 256 && s.bn == 128) return launch_cfg<8, 4, 2, 1, kInner>(p, slices, count, stream);
  if (s.bm == 128 && s.bn == 256) return launch_cfg<4, 8, 2, 1, kInner>(p, slices, count, stream);
  if (s.bm == 128 && s.bn == 128) return launch_cfg<4, 4, 2, 2, kInner>(p, slices, count, stream);
  if (s.bm == 64 && s.bn == 64) return launch_cfg<2, 4, 1, 4, kInner>(p, slices, count, stream);
  return hipErrorInvalidValue;
}

}  // namespace

namespace {

// A tile's costs in us, fitted to launches of 19 shapes from 64 x 64 x 100000 to
// 4096 x 8192 x 8192 in both layouts (bf16 outputs, every tile and 1 to 32
// slices each): a start (launch, first loads, epilogue) and one chunk of 128 K
// on a CU that holds one workgroup, where few CUs do (`alone`) and where all do
// (`full`: clock and memory are shared), and per workgroup where it holds more
// (`shared`).
struct TileCost {
  uint32_t bm, bn, resident;
  double start, alone, full, shared;
};
constexpr TileCost kTileCosts[] = {{256, 256, 1, 10.8, 1.05, 1.60, 1.60},
                                   {256, 128, 1, 6.6, 0.67, 1.10, 1.10},
                                   {128, 256, 1, 6.6, 0.71, 1.15, 1.15},
                                   {128, 128, 2, 5.8, 0.42, 0.50, 0.61},
                                   {64, 64, 4, 3.6, 0.35, 0.35, 0.25}};

double tile_cost(const TileCost& c, int64_t m, int64_t n, int64_t k, double units, int64_t k_slice) {
  const double chunks = static_cast<double>(std::max<int64_t>(1, (k_slice + 127) / 128));
  const double per_cu = std::ceil(units / 256);
  double chunk = c.alone + (c.full - c.alone) * std::min(1.0, units / 256);
  if (per_cu > 1) chunk = std::max(chunk, c.shared * per_cu);
  const double operands = static_cast<double>(m + n) * static_cast<double>(k) / kBytesPerUs;
  return c.start + std::max(chunks * chunk, operands);
}

}  // namespace

namespace {

// The best cut of a product into this kind of tile, if it beats `best`.
void choose_slices(const TileCost& c, int64_t m, int64_t n, int64_t k, TileShape& best) {
  const int64_t need = std::max<int64_t>(1, (k + kExactK - 1) / kExactK);
  const double tiles = static_cast<double>((m + c.bm - 1) / c.bm) * static_cast<double>((n + c.bn - 1) / c.bn);
  for (const int64_t wanted : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
    int64_t s = std::max(wanted, need);
    if (s > 1 && k < 256 * s) continue;  // slices of two chunks at least
    int64_t k_slice = k;
    if (s > 1) {
      k_slice = ((k + s - 1) / s + 127) / 128 * 128;
      k_slice = std::min<int64_t>(k_slice, kExactK / 128 * 128);
      s = (k + k_slice - 1) / k_slice;
    }
    const double units = tiles * static_cast<double>(s);
    if (units > 0x7FFFFFFF) continue;
    double cost = tile_cost(c, m, n, k, units, k_slice);
    // the join: a launch, and the partial sums written and read
    if (s > 1)
      cost += 2.2 + 0.03 * static_cast<double>(s) +
              static_cast<double>(s) * static_cast<double>(m) * static_cast<double>(n) * 8 / 4e6;
    if (best.cost != 0 && cost >= best.cost) continue;
    best.cost = cost;
    best.bm = c.bm;
    best.bn = c.bn;
    best.slices = static_cast<uint32_t>(s);
    best.k_slice = k_slice;
  }
  best.ldp = (n + 3) / 4 * 4;
  best.bytes = best.slices > 1 ? static_cast<uint64_t>(best.slices) * static_cast<uint64_t>(m) *
                                     static_cast<uint64_t>(best.ldp) * sizeof(int32_t)
                               : 0u;
}

}  // namespace

TileShape choose_tile_shape(int64_t m, int64_t n, int64_t k) {
  TileShape best{};
  for (const TileCost& c : kTileCosts) choose_slices(c, m, n, k, best);
  return best;
}

// In one launch where that is predicted to take less than two: products that fit
// on the chip together take as long as the longer one, others save a start.
bool choose_pair_shapes(const int64_t (&m)[2], const int64_t (&n)[2], const int64_t (&k)[2], TileShape (&shapes)[2]) {
  for (int i = 0; i < 2; ++i) shapes[i] = choose_tile_shape(m[i], n[i], k[i]);
  double least = shapes[0].cost + shapes[1].cost;
  bool one = false;
  for (const TileCost& c : kTileCosts) {
    TileShape s[2]{};
    double units = 0;
    for (int i = 0; i < 2; ++i) {
      choose_slices(c, m[i], n[i], k[i], s[i]);
      units += static_cast<double>((m[i] + c.bm - 1) / c.bm) * static_cast<double>((n[i] + c.bn - 1) / c.bn) * s[i].slices;
    }
    if (s[0].cost == 0 || s[1].cost == 0) continue;
    const double together = units <= 256.0 * c.resident ? std::max(s[0].cost, s[1].cost) : s[0].cost + s[1].cost - c.start / 2;
    if (together >= least) continue;
    least = together;
    one = true;
    shapes[0] = s[0];
    shapes[1] = s[1];
  }
  return one;
}

namespace {

// The kernel's arguments, if it can take the product.
bool tile_args(const ScaledGemm& g, const TileShape& shape, int32_t* partials, TileArgs& a) {
  const int64_t limit = int64_t{1} << 23;
  if (g.m <= 0 || g.n <= 0 || g.k < 0 || g.lda % 16 || g.ldb % 16 || g.lda >= limit || g.ldb >= limit ||
      reinterpret_cast<uintptr_t>(g.a) % 16 || reinterpret_cast<uintptr_t>(g.b) % 16 || g.m > 0x7FFFFFFF ||
      g.n > 0x7FFFFFFF - 256 || g.k > 0x7FFFFFFF - 256 || g.dtype > RNS8_MI355X_BF16)
    return false;
  const int64_t k16 = (g.k + 15) / 16 * 16;
  if (g.lda < k16 || (g.inner ? g.ldb < (g.n + 15) / 16 * 16 : g.ldb < k16)) return false;
  if (shape.slices == 0 || shape.k_slice > kExactK || (shape.slices > 1 && (!partials || shape.k_slice % 128)))
    return false;
  a = TileArgs{};
  a.a = g.a;
  a.b = g.b;
  a.a_scale = g.a_scale;
  a.b_scale = g.b_scale;
  a.bias = g.bias;
  a.out = g.out;
  a.partials = shape.slices > 1 ? partials : nullptr;
  a.ldo = g.ldo;
  a.ldp = shape.ldp;
  a.m = static_cast<uint32_t>(g.m);
  a.n = static_cast<uint32_t>(g.n);
  a.lda = static_cast<uint32_t>(g.lda);
  a.ldb = static_cast<uint32_t>(g.ldb);
  a.k16 = static_cast<uint32_t>(k16);
  a.k = static_cast<uint32_t>(g.k);
  a.dtype = g.dtype;
  a.k_slice = static_cast<uint32_t>(shape.slices > 1 ? shape.k_slice : k16);
  a.pairs = static_cast<uint32_t>(std::max<int64_t>(1, (a.k_slice + 127) / 128));
  return true;
}

}  // namespace

hipError_t launch_scaled_tiles(const ScaledGemm* g, const TileShape* shapes, int32_t* const* partials, int count,
                               hipStream_t stream) {
  TilePair p{};
  JoinPair j{};
  uint32_t slices[2] = {}, join_blocks[2] = {};
  int joins = 0;
  for (int i = 0; i < count; ++i) {
    if (g[i].inner != g[0].inner || (i > 0 && !g[i].inner) || shapes[i].bm != shapes[0].bm || shapes[i].bn != shapes[0].bn ||
        !tile_args(g[i], shapes[i], partials[i], p.product[i]))
      return hipErrorInvalidValue;
    slices[i] = shapes[i].slices;
    if (slices[i] == 1) continue;
    j.product[joins] = {partials[i], slices[i], g[i].m, g[i].n, shapes[i].ldp, g[i].ldo, g[i].a_scale, g[i].b_scale,
                        g[i].bias, g[i].out, g[i].dtype};
    join_blocks[joins++] = static_cast<uint32_t>(std::min<int64_t>((g[i].m * (shapes[i].ldp / 4) + 255) / 256, 1 << 20));
  }
  const hipError_t e = g[0].inner ? launch_tile<true>(p, shapes[0], slices, count, stream)
                                  : launch_tile<false>(p, shapes[0], slices, count, stream);
  if (e != hipSuccess || joins == 0) return e;
  j.blocks = join_blocks[0];
  hipLaunchKernelGGL(join_slices_kernel, dim3(join_blocks[0] + join_blocks[1]), dim3(256), 0, stream, j);
  return hipGetLastError();
}

}  // namespace rns8x
