// One workgroup's tile of a 16-bit matrix product A B^T with operands in either storage order, fp32 accumulation on
// v_mfma_f32_16x16x32_{bf16,f16}: the main loop of kernels whose epilogue is not a stored matrix (fh_vocab_loss.hip).
//
// The data path is fh_gemm16.hip's (a ring of four LDS stages of 32 k that global_load_lds fills three stages ahead, XOR-swizzled chunks,
// fragment reads between the products in fixed program order, one barrier per stage) with either operand in either order:
//   rows:      element (r, k) at p[row(r) * ld + k]. A stage is [rows][32 k], 64 bytes a row; a fragment (8 k of one row per lane) is one
//              ds_read_b128. row(r) may come from a list.
//   columns:   element (r, k) at p[k * ld + r]. A stage is [32 k][rows], kept as in memory; a fragment is two transposing reads of 4 k each
//              (ds_read_b64_tr_b16).
#pragma once

#include <hip/hip_runtime.h>

#include <utility>

#include "fh_common.h"
#include "fh_mfma16.h"

namespace fh {
namespace tile {

using namespace mfma16;

__device__ const uint4 kZeros = {0, 0, 0, 0};

// depth: elements are zeros from k = depth on (read only where the operand's loads are declared to end unevenly). last: the greatest row
// that exists; rows behind it are read as it is (column order: chunks of 8 rows that would end behind it end at it), and their products
// belong to nobody.
struct Operand {
  const uint16_t* p;
  int64_t ld;
  const int32_t* rows;
  int last, depth;
};

template <int TX, bool COLUMNS>
struct Fragments {
  u32x4_t v[TX];
};
template <int TX>
struct Fragments<TX, true> {
  u32x2_t low[TX], high[TX];  // the first and the last 4 of the lane's 8 k
};
template <int TX, bool C>
__device__ __forceinline__ u32x4_t fragment(const Fragments<TX, C>& f, int i) {
  if constexpr (C)
    return u32x4_t{f.low[i][0], f.low[i][1], f.high[i][0], f.high[i][1]};
  else
    return f.v[i];
}
// Ties fragment registers to the lgkmcnt(0) wait before: the reads are inline asm, whose results the compiler takes as there at once.
template <int TX, bool C>
__device__ __forceinline__ void tie(Fragments<TX, C>& f) {
#pragma unroll
  for (int i = 0; i < TX; ++i) {
    if constexpr (C) {
      asm volatile("" : "+v"(f.low[i]));
      asm volatile("" : "+v"(f.high[i]));
    } else {
      asm volatile("" : "+v"(f.v[i]));
    }
  }
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// One operand's way: R rows of the tile by NW waves' loads, TX blocks of 16 rows read by each wave. UNEVEN: the depth may end inside a stage.
template <int R, int TX, bool COLUMNS, bool UNEVEN, int NW>
struct Feed {
  static constexpr int kBytes = R * kBK * 2;
  static constexpr int kLoads = kBytes / 1024 / NW;  // load instructions per wave and stage
  static constexpr int kChunks = R / 8;              // column order: 16-byte chunks of a row of k
  static_assert(kBytes / 1024 % NW == 0, "a stage's loads split evenly over the waves");
  static_assert(!COLUMNS || (kChunks >= 8 && kChunks <= 64), "rows in [64, 512]");

  const uint16_t* src[kLoads];
  int64_t step;        // elements from a stage to the next
  int first[kLoads];   // the lane's first k in a stage
  int depth;
  int off[COLUMNS ? TX : 1];  // where the lane reads, bytes within a stage

  // r0: the tile's first row; mine: the wave's first row in the tile
  __device__ __forceinline__ void init(const Operand& o, int r0, int mine, int wave, int lane) {
    depth = o.depth;
    if constexpr (COLUMNS) {
      step = kBK * o.ld;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int k = (wave * kLoads + j) * (64 / kChunks) + lane / kChunks;
        const int chunk = (lane % kChunks) ^ b_swizzle16<kChunks>(k);
        first[j] = k;
        src[j] = o.p + k * o.ld + min(r0 + chunk * 8, o.last - 7);
      }
      // lane r = q + 4 e of group g points at k 8 g + e, rows 4 q .. 4 q + 3 of a block; the second read is 4 k further on
      const int g = lane >> 4, q = lane & 3, e = (lane & 15) >> 2, k = 8 * g + e;
#pragma unroll
      for (int i = 0; i < TX; ++i) {
        const int row = mine + 16 * i + 4 * q;
        off[i] = k * (R * 2) + ((row >> 3) ^ b_swizzle16<kChunks>(k)) * 16 + (row & 7) * 2;
      }
    } else {
      step = kBK;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int in_tile = (wave * kLoads + j) * 16 + (lane >> 2), row = min(r0 + in_tile, o.last);
        const int chunk = (lane & 3) ^ a_swizzle(in_tile);
        first[j] = chunk * 8;
        src[j] = o.p + static_cast<int64_t>(o.rows != nullptr ? o.rows[row] : row) * o.ld + chunk * 8;
      }
      const int row = mine + (lane & 15);
      off[0] = row * 64 + (((lane >> 4) ^ a_swizzle(row)) * 16);
    }
  }
  // load instruction J of stage kt to this operand's part of a stage
  template <int J>
  __device__ __forceinline__ void load(int kt, unsigned char* to, int wave) const {
    const uint16_t* from = src[J] + kt * step;
    if constexpr (UNEVEN) from = first[J] < depth - kt * kBK ? from : reinterpret_cast<const uint16_t*>(&kZeros);
    global_to_lds16(from, (FH_LDS void*)(to + (wave * kLoads + J) * 1024));
  }
  // read instruction N of blocks I0, I0 + 1, .. of the stage part at `base`
  template <int N, int I0, int TF>
  __device__ __forceinline__ void read(uint32_t base, Fragments<TF, COLUMNS>& f) const {
    if constexpr (COLUMNS) {
      if constexpr (N % 2 == 0)
        f.low[N / 2] = lds_read_tr16_b64<0>(base + off[I0 + N / 2]);
      else
        f.high[N / 2] = lds_read_tr16_b64<4 * R * 2>(base + off[I0 + N / 2]);
    } else {
      f.v[N] = lds_read_b128<(I0 + N) * 1024>(base + off[0]);
    }
  }
};

// The BM x BN tile at (m0, n0) of A B^T over k < 32 KT, by WAVES_M x WAVES_N waves. A wave's part begins at row WM (wave / WAVES_N), column
// WN (wave % WAVES_N); its lane l holds rows 16 i + 4 (l / 16) + x and column 16 j + l % 16 of it in acc[i][j][x]. On return all of the
// workgroup's waves are past their last use of `lds` (kLds bytes, 1 KB aligned).
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, bool A_COLUMNS, bool B_COLUMNS, bool A_UNEVEN, bool B_UNEVEN>
struct Product {
  static constexpr int kWaves = WAVES_M * WAVES_N, kThreads = kWaves * 64;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, TM = WM / 16, TN = WN / 16;
  using FeedA = Feed<BM, TM, A_COLUMNS, A_UNEVEN, kWaves>;
  using FeedB = Feed<BN, TN, B_COLUMNS, B_UNEVEN, kWaves>;
  static constexpr int kStage = FeedA::kBytes + FeedB::kBytes, kLds = kStages * kStage;
  static constexpr int kLoads = FeedA::kLoads + FeedB::kLoads;
  // Small wave tiles hold two full sets of fragments and run a stage as one phase; large ones split it over halves of the B blocks.
  static constexpr bool kOne = (TM + 2 * TN) * 8 + TM * TN * 4 <= 160;
  static constexpr int TB = kOne ? TN : TN / 2;
  static constexpr int kReadsA = A_COLUMNS ? 2 * TM : TM, kReadsB = B_COLUMNS ? 2 * TB : TB;
  static constexpr int kProducts = TM * TB;  // of a phase
  // reads are spread over the first three quarters of a phase's products, loads over the first half
  static constexpr int kReadSpan = kProducts * 3 / 4 > 0 ? kProducts * 3 / 4 : 1, kLoadSpan = kProducts / 2 > 0 ? kProducts / 2 : 1;
  static_assert(TM >= 1 && TN >= 2 && TN % 2 == 0 && 2 * kLoads <= 63, "tile shape");
  using Acc = f32x4_t[TM][TN];
  using SetA = Fragments<TM, A_COLUMNS>;
  using SetB = Fragments<TB, B_COLUMNS>;

  __device__ __forceinline__ static int wave() { return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)); }
  __device__ __forceinline__ static int lane() { return threadIdx.x & 63; }
  __device__ __forceinline__ static int wave_row() { return wave() / WAVES_N * WM; }
  __device__ __forceinline__ static int wave_column() { return wave() % WAVES_N * WN; }

  __device__ __forceinline__ static void run(unsigned char* lds, const Operand& a, const Operand& b, int m0, int n0, int KT, Acc& acc) {
    const int wave = Product::wave(), lane = Product::lane();
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (KT <= 0) return;
    FeedA fa;
    FeedB fb;
    fa.init(a, m0, wave_row(), wave, lane);
    fb.init(b, n0, wave_column(), wave, lane);
    const uint32_t ring = lds_addr((const FH_LDS void*)lds);

    // stages past the end load the last one again (nobody reads them), so that every step issues as many loads and the waits count right
    auto load_one = [&]<int J>(int kt) {
      unsigned char* to = lds + (kt & (kStages - 1)) * kStage;
      if constexpr (J < FeedA::kLoads)
        fa.template load<J>(min(kt, KT - 1), to, wave);
      else
        fb.template load<J - FeedA::kLoads>(min(kt, KT - 1), to + FeedA::kBytes, wave);
    };
    auto load_stage = [&](int kt) {
      [&]<int... J>(std::integer_sequence<int, J...>) { (load_one.template operator()<J>(kt), ...); }(std::make_integer_sequence<int, kLoads>{});
    };
    // read N of a stage's first set: A's blocks, then B's [0, TB)
    auto read_set = [&]<int N>(uint32_t base, SetA& sa, SetB& sb) {
      if constexpr (N < kReadsA)
        fa.template read<N, 0, TM>(base, sa);
      else
        fb.template read<N - kReadsA, 0, TB>(base + FeedA::kBytes, sb);
    };
    // The products of B's blocks [J0, J0 + TB), between them (NEXT) the reads of the stage at `base` into (sa_n, sb_n) and the loads of
    // stage load_kt, or the reads of the same stage's B blocks [TB, 2 TB) into sb_n.
    auto phase = [&]<int J0, bool NEXT>(SetA& sa, SetB& sb, uint32_t base, SetA& sa_n, SetB& sb_n, int load_kt) {
      constexpr int reads = NEXT ? kReadsA + kReadsB : kReadsB;
      [&]<int... M_>(std::integer_sequence<int, M_...>) {
        (
            [&] {
              constexpr int i = M_ / TB, j = M_ % TB;
              mfma16x<T>(fragment(sa, i), fragment(sb, j), acc[i][J0 + j]);
              constexpr int r0 = mfma16::first(M_, reads, kReadSpan);
              [&]<int... R_>(std::integer_sequence<int, R_...>) {
                if constexpr (NEXT)
                  (read_set.template operator()<r0 + R_>(base, sa_n, sb_n), ...);
                else
                  (fb.template read<r0 + R_, TB, TB>(base + FeedA::kBytes, sb_n), ...);
              }(std::make_integer_sequence<int, share(M_, reads, kReadSpan)>{});
              if constexpr (NEXT) {
                constexpr int l0 = mfma16::first(M_, kLoads, kLoadSpan);
                [&]<int... L_>(std::integer_sequence<int, L_...>) {
                  (load_one.template operator()<l0 + L_>(load_kt), ...);
                }(std::make_integer_sequence<int, share(M_, kLoads, kLoadSpan)>{});
              }
              __builtin_amdgcn_sched_barrier(0);
            }(),
            ...);
      }(std::make_integer_sequence<int, kProducts>{});
    };
    auto barrier_next = [&] {
      wait_vmcnt<kLoads>();  // this wave's part of stage kt + 1 is there (stage kt + 2 may be on its way)
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    // Stage kt with its first set in (sa, sb). The slot that is filled after the barrier held stage kt - 1, whose reads every wave waited
    // for before it arrived there.
    auto stage = [&](int kt, SetA& sa, SetA& sa_n, SetB& sb, SetB& sb_n) {
      const uint32_t cur = ring + (kt & (kStages - 1)) * kStage, nxt = ring + ((kt + 1) & (kStages - 1)) * kStage;
      if constexpr (kOne) {
        barrier_next();
        wait_lds();
        tie(sa);
        tie(sb);
        phase.template operator()<0, true>(sa, sb, nxt, sa_n, sb_n, kt + kStages - 1);
      } else {
        wait_lds();
        tie(sa);
        tie(sb);
        phase.template operator()<0, false>(sa, sb, cur, sa_n, sb_n, 0);
        barrier_next();
        wait_lds();
        tie(sb_n);
        phase.template operator()<TN - TB, true>(sa, sb_n, nxt, sa_n, sb, kt + kStages - 1);
      }
    };

    SetA sa0, sa1;
    SetB sb0, sb1;
    load_stage(0);
    load_stage(1);
    load_stage(2);
    wait_vmcnt<2 * kLoads>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    [&]<int... N_>(std::integer_sequence<int, N_...>) {
      (read_set.template operator()<N_>(ring, sa0, sb0), ...);
    }(std::make_integer_sequence<int, kReadsA + kReadsB>{});
    int kt = 0;
    for (; kt + 1 < KT; kt += 2) {
      stage(kt, sa0, sa1, sb0, sb1);
      if constexpr (kOne)
        stage(kt + 1, sa1, sa0, sb1, sb0);
      else
        stage(kt + 1, sa1, sa0, sb0, sb1);
    }
    if (kt < KT) stage(kt, sa0, sa1, sb0, sb1);
    // the last stage's reads of the one behind it (unused) still write their registers
    wait_lds();
    tie(sa0);
    tie(sa1);
    tie(sb0);
    tie(sb1);
    wait_vmcnt<0>();  // and its loads the ring
    __syncthreads();
  }

  // The tile in 16-bit storage, whole 16-byte vectors of 8 columns: each wave hands its part over through its own room in `lds` and calls
  // put(row, column, vector) with rows and columns of the tile. value(i, x, j): what lane l stores for its acc[i][j][x].
  template <typename Value, typename Put>
  __device__ __forceinline__ static void store(unsigned char* lds, Value&& value, Put&& put) {
    static_assert(kWaves * WM * WN * 2 <= kLds, "the waves' parts fit in the ring");
    const int lane = Product::lane(), g = lane >> 4, r = lane & 15;
    uint16_t* mine = reinterpret_cast<uint16_t*>(lds + wave() * (WM * WN * 2));
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int j = 0; j < TN; ++j) mine[(i * 16 + 4 * g + x) * WN + j * 16 + r] = Io<T>::store(value(i, x, j));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // from lane to lane of one wave, whose accesses run in their order
    __builtin_amdgcn_wave_barrier();
    constexpr int lanes = WN / 8, rows = 64 / lanes;
#pragma unroll 4
    for (int at = 0; at < WM; at += rows) {
      const int row = at + lane / lanes, c = lane % lanes * 8;
      put(wave_row() + row, wave_column() + c, *reinterpret_cast<const u32x4_t*>(mine + row * WN + c));
    }
  }
};

// Workgroup `block` of `tiles_m` x `tiles_n` tiles -> its tile: consecutive tiles on one XCD (workgroups go round the 8 of them), in groups of
// 8 tiles of rows, so that the tiles at work together share their operands in its L2. false: there is no such tile.
__device__ __forceinline__ bool place(uint32_t block, int tiles_m, int tiles_n, int& tm, int& tn) {
  const uint32_t total = static_cast<uint32_t>(tiles_m) * tiles_n;
  if (block >= total) return false;
  const uint32_t xcd = block & 7, each = total >> 3, more = total & 7;
  const uint32_t id = xcd * each + min(xcd, more) + (block >> 3);
  const uint32_t group = id / (8u * tiles_n), first = group * 8, size = min(static_cast<uint32_t>(tiles_m) - first, 8u);
  const uint32_t in = id - group * 8u * tiles_n;
  tm = static_cast<int>(first + in % size);
  tn = static_cast<int>(in / size);
  return true;
}

}  // namespace tile
}  // namespace fh
