// One workgroup's tile of a 16-bit matrix product A B^T with operands in either storage order, fp32 accumulation on
// v_mfma_f32_16x16x32_{bf16,f16}: the main loop of kernels whose epilogue is not a stored matrix (fh_vocab_loss.hip).
//
// A stage is 64 k of both operands. global_load_lds fills a ring of stages (16 bytes a lane, no registers between), chunks XOR-swizzled so
// that the fragments' reads meet no bank twice; the reads and the loads stand between the products in fixed program order; one barrier
// per stage. Either operand comes in either order:
//   rows:      element (r, k) at p[row(r) * ld + k]. In LDS [rows][64 k], 128 bytes a row: a whole cache line per row and stage (with 64 bytes
//              each line went from L2 to the CU twice, at 64 bytes a clock all that it has for two such operands). A fragment (8 k
//              of one row per lane) is one ds_read_b128. row(r) may come from a list.
//   columns:   element (r, k) at p[k * ld + r]. In LDS [64 k][rows], as in memory; a fragment is two transposing reads of 4 k each
//              (ds_read_b64_tr_b16).
//
// Measured in fh_vocab_loss.hip's kernels (256 x 256 tiles of eight waves): 1,290 to 1,380 TFLOP/s in long products, at 64 products,
// 24 (rows) to 48 (columns) LDS reads and 8 loads per wave and stage, no bank conflicts; bound by the board's power. With every load
// from L2 instead (a stage read again and again) the same instructions took 3 to 8 % less. Not kept: stages of 32 k in a ring of four
// (8 to 10 % slower for two operands in rows), four waves of 128 x 128 (6 % slower, and their epilogues spill), reads in the first half or
// quarter of a phase, loads spread over all of it, raised wave priority (within 2 %, the noise).
#pragma once

#include <hip/hip_runtime.h>

#include <utility>

#include "fh_common.h"
#include "fh_mfma16.h"

namespace fh {
namespace tile {

using namespace mfma16;

constexpr int kDepth = 64;  // k of a stage: two steps of 32
constexpr int kStep = 32;

__device__ const uint4 kZeros = {0, 0, 0, 0};

// depth: elements are zeros from k = depth on (read only where the operand's loads are declared to end unevenly). last: the greatest row
// that exists; rows behind it are read as it is (column order: chunks of 8 rows that would end behind it end at it), and their products
// belong to nobody. ld is less than 2^22.
struct Operand {
  const uint16_t* p;
  int64_t ld;
  const int32_t* rows;  // Lie::kListed
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

// The swizzle of a row's 16-byte chunks (row order): two rows share the banks' 256 bytes, so rows 2 apart must differ.
__device__ __forceinline__ int row_swizzle(int row) { return (row >> 1) & 7; }

// How an operand lies: in rows, in rows that a list names, or in columns. UNEVEN: the depth may end inside a stage (one more comparison and
// select per load: 3 to 7 % of a long product).
enum class Lie { kRows, kListed, kColumns };

// One operand's way: R rows of the tile by NW waves' loads, TX blocks of 16 rows read by each wave.
template <int R, int TX, Lie LIE, bool UNEVEN, int NW>
struct Feed {
  static constexpr bool COLUMNS = LIE == Lie::kColumns;
  static constexpr int kBytes = R * kDepth * 2;
  static constexpr int kLoads = kBytes / 1024 / NW;  // load instructions per wave and stage
  static constexpr int kChunks = R / 8;              // column order: 16-byte chunks of a row of k
  static_assert(kBytes / 1024 % NW == 0, "a stage's loads split evenly over the waves");
  static_assert(!COLUMNS || (kChunks >= 8 && kChunks <= 64), "rows in [64, 512]");

  // The lane's place: 32 bits from an address that all lanes share, which a load takes as they are; 64 bits where rows come from a list.
  const unsigned char* base;
  const unsigned char* listed[kLoads];
  uint32_t place[kLoads];
  int64_t step;       // bytes from a stage to the next
  int first[kLoads];  // the lane's first k in a stage
  int depth;
  int off[COLUMNS ? TX : 2];  // where the lane reads, bytes within a stage: per block, or per step of 32 k

  // r0: the tile's first row; mine: the wave's first row in the tile
  __device__ __forceinline__ void init(const Operand& o, int r0, int mine, int wave, int lane) {
    depth = o.depth;
    const unsigned char* p = reinterpret_cast<const unsigned char*>(o.p);
    if constexpr (COLUMNS) {
      const int at = min(r0, o.last - 7);
      base = p + static_cast<int64_t>(at) * 2;
      step = kDepth * o.ld * 2;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int k = (wave * kLoads + j) * (64 / kChunks) + lane / kChunks;
        const int chunk = (lane % kChunks) ^ b_swizzle16<kChunks>(k);
        first[j] = k;
        place[j] = static_cast<uint32_t>(k) * static_cast<uint32_t>(o.ld * 2) + static_cast<uint32_t>(min(r0 + chunk * 8, o.last - 7) - at) * 2;
      }
      // lane r = q + 4 e of group g points at k 8 g + e, rows 4 q .. 4 q + 3 of a block; the second read is 4 k further on
      const int g = lane >> 4, q = lane & 3, e = (lane & 15) >> 2, k = 8 * g + e;
#pragma unroll
      for (int i = 0; i < TX; ++i) {
        const int row = mine + 16 * i + 4 * q;
        off[i] = k * (R * 2) + ((row >> 3) ^ b_swizzle16<kChunks>(k)) * 16 + (row & 7) * 2;
      }
    } else {
      const int at = min(r0, o.last);
      base = LIE == Lie::kListed ? p : p + static_cast<int64_t>(at) * o.ld * 2;
      step = kDepth * 2;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int in_tile = (wave * kLoads + j) * 8 + (lane >> 3), row = min(r0 + in_tile, o.last);
        const int chunk = (lane & 7) ^ row_swizzle(in_tile);
        first[j] = chunk * 8;
        if constexpr (LIE == Lie::kListed)
          listed[j] = p + o.rows[row] * o.ld * 2 + chunk * 16;
        else
          place[j] = static_cast<uint32_t>(row - at) * static_cast<uint32_t>(o.ld * 2) + chunk * 16;
      }
      const int row = mine + (lane & 15);
#pragma unroll
      for (int h = 0; h < 2; ++h) off[h] = row * (kDepth * 2) + (((lane >> 4) + 4 * h) ^ row_swizzle(row)) * 16;
    }
  }
  // load instruction J of stage kt to this operand's part of a stage
  template <int J>
  __device__ __forceinline__ void load(int kt, unsigned char* to, int wave) const {
    const unsigned char* from = LIE == Lie::kListed ? listed[J] + kt * step : base + kt * step + place[J];
    if constexpr (UNEVEN) from = first[J] < depth - kt * kDepth ? from : reinterpret_cast<const unsigned char*>(&kZeros);
    global_to_lds16(from, (FH_LDS void*)(to + (wave * kLoads + J) * 1024));
  }
  // read instruction N of blocks I0, I0 + 1, .. for step H of the stage part at `base`
  template <int N, int I0, int H, int TF>
  __device__ __forceinline__ void read(uint32_t base, Fragments<TF, COLUMNS>& f) const {
    if constexpr (COLUMNS) {
      if constexpr (N % 2 == 0)
        f.low[N / 2] = lds_read_tr16_b64<H * kStep * R * 2>(base + off[I0 + N / 2]);
      else
        f.high[N / 2] = lds_read_tr16_b64<(H * kStep + 4) * R * 2>(base + off[I0 + N / 2]);
    } else {
      f.v[N] = lds_read_b128<(I0 + N) * 16 * kDepth * 2>(base + off[H]);
    }
  }
};

// The BM x BN tile at (m0, n0) of A B^T over k < 64 KT, by WAVES_M x WAVES_N waves. A wave's part begins at row WM (wave / WAVES_N), column
// WN (wave % WAVES_N); its lane l holds row 16 i + l % 16, columns 16 j + 4 (l / 16) + x of it in acc[i][j][x] (the instruction's operands
// change places: four columns of a row in a lane are what every epilogue here wants). On return all of the workgroup's waves are
// past their last use of `lds` (kLds bytes, 1 KB aligned).
// A stage is two steps. Small wave tiles hold two full sets of fragments and take a step in one phase; large ones take it in two, over halves
// of the B blocks. While a phase's products run the next phase's fragments are read; in the stage's last one, after a barrier behind which
// the next stage is there and this one is read, the stage STAGES ahead is loaded into this one's place.
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, int STAGES, Lie LIE_A, Lie LIE_B, bool UNEVEN_A, bool UNEVEN_B>
struct Product {
  static constexpr int kWaves = WAVES_M * WAVES_N, kThreads = kWaves * 64;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, TM = WM / 16, TN = WN / 16;
  static constexpr bool A_COLUMNS = LIE_A == Lie::kColumns, B_COLUMNS = LIE_B == Lie::kColumns;
  using FeedA = Feed<BM, TM, LIE_A, UNEVEN_A, kWaves>;
  using FeedB = Feed<BN, TN, LIE_B, UNEVEN_B, kWaves>;
  static constexpr int kStage = FeedA::kBytes + FeedB::kBytes, kLds = STAGES * kStage;
  static constexpr int kLoads = FeedA::kLoads + FeedB::kLoads;
  static constexpr bool kOne = (TM + 2 * TN) * 8 + TM * TN * 4 <= 160;
  static constexpr int TB = kOne ? TN : TN / 2;
  static constexpr int kReadsA = A_COLUMNS ? 2 * TM : TM, kReadsB = B_COLUMNS ? 2 * TB : TB;
  static constexpr int kProducts = TM * TB;  // of a phase
  // reads are spread over the first three quarters of a phase's products, loads over the first half
  static constexpr int kReadSpan = kProducts * 3 / 4 > 0 ? kProducts * 3 / 4 : 1, kLoadSpan = kProducts / 2 > 0 ? kProducts / 2 : 1;
  static_assert(TM >= 1 && TN >= 2 && TN % 2 == 0 && STAGES >= 2 && (STAGES - 1) * kLoads <= 63, "tile shape");
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

    // stages past the end load the last one again (nobody reads them), so that every stage issues as many loads and the waits count right
    auto load_one = [&]<int J>(int kt, int slot) {
      unsigned char* to = lds + slot * kStage;
      if constexpr (J < FeedA::kLoads)
        fa.template load<J>(min(kt, KT - 1), to, wave);
      else
        fb.template load<J - FeedA::kLoads>(min(kt, KT - 1), to + FeedA::kBytes, wave);
    };
    auto load_stage = [&](int kt) {
      [&]<int... J>(std::integer_sequence<int, J...>) { (load_one.template operator()<J>(kt, kt), ...); }(std::make_integer_sequence<int, kLoads>{});
    };
    // read N of the first set of step H: A's blocks, then B's [0, TB)
    auto read_set = [&]<int N, int H>(uint32_t base, SetA& sa, SetB& sb) {
      if constexpr (N < kReadsA)
        fa.template read<N, 0, H>(base, sa);
      else
        fb.template read<N - kReadsA, 0, H>(base + FeedA::kBytes, sb);
    };
    // The products of B's blocks [J0, J0 + TB), between them (NEXT) the reads of the first set of step H of the stage at `base` into (sa_n, sb_n),
    // or those of the same step's B blocks [TB, 2 TB) into sb_n; LOAD: and the loads of stage load_kt into `slot`.
    auto phase = [&]<int J0, int H, bool NEXT, bool LOAD>(SetA& sa, SetB& sb, uint32_t base, SetA& sa_n, SetB& sb_n, int load_kt, int slot) {
      constexpr int reads = NEXT ? kReadsA + kReadsB : kReadsB;
      [&]<int... M_>(std::integer_sequence<int, M_...>) {
        (
            [&] {
              constexpr int i = M_ / TB, j = M_ % TB;
              mfma16x<T>(fragment(sb, j), fragment(sa, i), acc[i][J0 + j]);
              constexpr int r0 = mfma16::first(M_, reads, kReadSpan);
              [&]<int... R_>(std::integer_sequence<int, R_...>) {
                if constexpr (NEXT)
                  (read_set.template operator()<r0 + R_, H>(base, sa_n, sb_n), ...);
                else
                  (fb.template read<r0 + R_, TB, H>(base + FeedA::kBytes, sb_n), ...);
              }(std::make_integer_sequence<int, share(M_, reads, kReadSpan)>{});
              if constexpr (LOAD) {
                constexpr int l0 = mfma16::first(M_, kLoads, kLoadSpan);
                [&]<int... L_>(std::integer_sequence<int, L_...>) {
                  (load_one.template operator()<l0 + L_>(load_kt, slot), ...);
                }(std::make_integer_sequence<int, share(M_, kLoads, kLoadSpan)>{});
              }
              __builtin_amdgcn_sched_barrier(0);
            }(),
            ...);
      }(std::make_integer_sequence<int, kProducts>{});
    };
    auto ready = [&](SetA& sa, SetB& sb) {
      wait_lds();
      tie(sa);
      tie(sb);
    };
    // this wave's reads of the stage are done (wait_lds before it) and its part of the next one is there; behind the barrier, everybody's
    auto turn = [&] {
      wait_vmcnt<(STAGES - 2) * kLoads>();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };

    SetA sa0, sa1;
    SetB sb0, sb1;
    [&]<int... S_>(std::integer_sequence<int, S_...>) { (load_stage(S_), ...); }(std::make_integer_sequence<int, STAGES>{});
    wait_vmcnt<(STAGES - 1) * kLoads>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    [&]<int... N_>(std::integer_sequence<int, N_...>) {
      (read_set.template operator()<N_, 0>(ring, sa0, sb0), ...);
    }(std::make_integer_sequence<int, kReadsA + kReadsB>{});
    int slot = 0;
    for (int kt = 0; kt < KT; ++kt) {
      const int next = slot + 1 == STAGES ? 0 : slot + 1;
      const uint32_t cur = ring + slot * kStage, nxt = ring + next * kStage;
      if constexpr (kOne) {
        ready(sa0, sb0);
        phase.template operator()<0, 1, true, false>(sa0, sb0, cur, sa1, sb1, 0, 0);
        ready(sa1, sb1);
        turn();
        phase.template operator()<0, 0, true, true>(sa1, sb1, nxt, sa0, sb0, kt + STAGES, slot);
      } else {
        ready(sa0, sb0);
        phase.template operator()<0, 0, false, false>(sa0, sb0, cur, sa1, sb1, 0, 0);
        ready(sa0, sb1);
        phase.template operator()<TN - TB, 1, true, false>(sa0, sb1, cur, sa1, sb0, 0, 0);
        ready(sa1, sb0);
        phase.template operator()<0, 1, false, false>(sa1, sb0, cur, sa0, sb1, 0, 0);
        ready(sa1, sb1);
        turn();
        phase.template operator()<TN - TB, 0, true, true>(sa1, sb1, nxt, sa0, sb0, kt + STAGES, slot);
      }
      slot = next;
    }
    // the last stage's reads of the one behind it (unused) still write their registers
    wait_lds();
    tie(sa0);
    tie(sa1);
    tie(sb0);
    tie(sb1);
    wait_vmcnt<0>();  // and its loads the ring
    __syncthreads();
  }

  // acc in 16-bit storage as whole 16-byte vectors of 8 columns: each wave hands its part over through its own room in `lds` and calls
  // put(row, column, vector) with rows and columns of the tile. Chunks of a row are XORed with it: 16 rows' pieces meet in no bank.
  template <typename Put>
  __device__ __forceinline__ static void store(unsigned char* lds, const Acc& acc, Put&& put) {
    static_assert(kWaves * WM * WN * 2 <= kLds, "the waves' parts fit in the ring");
    constexpr int chunks = WN / 8, rows = 64 / chunks;
    const int lane = Product::lane(), g = lane >> 4, r = lane & 15;
    unsigned char* mine = lds + wave() * (WM * WN * 2);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int row = i * 16 + r, chunk = (2 * j + (g >> 1)) ^ (r & (chunks - 1));
        *reinterpret_cast<u32x2_t*>(mine + row * (WN * 2) + chunk * 16 + (g & 1) * 8) =
            u32x2_t{store2<T>(acc[i][j][0], acc[i][j][1]), store2<T>(acc[i][j][2], acc[i][j][3])};
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // from lane to lane of one wave, whose accesses run in their order
    __builtin_amdgcn_wave_barrier();
#pragma unroll 4
    for (int at = 0; at < WM; at += rows) {
      const int row = at + lane / chunks, c = lane % chunks;
      put(wave_row() + row, wave_column() + c * 8,
          *reinterpret_cast<const u32x4_t*>(mine + row * (WN * 2) + ((c ^ (row & 15 & (chunks - 1))) * 16)));
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
