// What the attention kernels over packed sequences and over a paged cache share: where a row of a tile comes from, LDS tiles that
// serve both row and transposed fragments, and the 32-row products on v_mfma_f32_32x32x16.
//
// Rows. The query rows of one key head are taken together: row r of a sequence is its token r / group, head
// kv_head * group + r % group, so the heads that share keys and values share every tile of them, and a lane (one row of a 32-row
// tile) carries its own last visible key.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "fh_common.h"
#include "fh_mfma16.h"

namespace fh {
namespace attn {

using namespace mfma16;

typedef short s16x4_t __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int64_t kMaxBlocks = 0xffffff;  // of 256 threads: a grid dimension holds fewer than 2^32 threads
constexpr float kLn2 = 0.69314718055994530942f;

// r / d for 0 <= r < 2^31 as (r * mul) >> shift: with 2^(l-1) < d <= 2^l, mul = ceil(2^(31+l) / d) exceeds the quotient by less
// than d / 2^(31+l), which times r stays below one step of 1/d.
struct Divider {
  uint32_t d, mul, shift;
};
inline Divider make_divider(uint32_t d) {
  uint32_t l = 0;
  while ((uint64_t{1} << l) < d) ++l;
  return {d, static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + d - 1) / d), 31 + l};
}
__device__ __forceinline__ int divide(int r, const Divider& v) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(r)) * v.mul) >> v.shift);
}

// cu_seqlens is device data: whatever it holds, a sequence's rows stay within the tensors' rows.
struct Span {
  int begin, end;
};
__device__ __forceinline__ Span sequence(const int32_t* cu, int b, int rows) {
  const int s = min(max(cu[b], 0), rows);
  return {s, min(max(cu[b + 1], s), rows)};
}

// Work slots. The tiles of `tile` rows (rows = tokens * per_token) of all sequences are numbered without knowing the lengths on the
// host: sequence b's begin at slot(b) = floor(cu[b] * per_token / tile) + b, which leaves room for its ceil(length / tile) tiles
// before slot(b + 1). Slots that no tile takes end at once. Every wave looks 64 sequences up at a time.
// Host: floor(rows * per_token / tile) + batch slots.
// Where cu_seqlens decreases, the sequence found may begin behind the slot: tile_in() takes such a tile for none.
__device__ __forceinline__ int find_sequence(const int32_t* cu, int batch, int rows, int per_token, int tile_shift, int slot,
                                             int& first_slot, Span& seq) {
  const int lane = threadIdx.x & 63;
  int found = 0, begin = 0, end = 0;
  for (int base = 0; base < batch; base += 64) {
    const int b = base + lane;
    bool before = false;
    int s = 0, e = 0;
    if (b < batch) {
      s = min(max(cu[b], 0), rows);
      e = min(max(cu[b + 1], s), rows);
      before = ((static_cast<int64_t>(s) * per_token) >> tile_shift) + b <= slot;
    }
    const int n = __popcll(__ballot(before));
    if (n > 0) {
      begin = __builtin_amdgcn_readlane(s, n - 1);
      end = __builtin_amdgcn_readlane(e, n - 1);
    }
    found += n;
    if (n < 64) break;
  }
  seq = {begin, end};
  first_slot = static_cast<int>((static_cast<int64_t>(begin) * per_token) >> tile_shift) + found - 1;
  return found - 1;
}

__device__ __forceinline__ bool tile_in(int first_row, int rows) {
  return static_cast<uint32_t>(first_row) < static_cast<uint32_t>(rows);
}

// The last sequence that begins at `token` or before it (the one that holds it, if any does), or -1.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int batch, int token) {
  int found = 0;
  for (int base = 0; base < batch; base += 64) {
    const int i = base + static_cast<int>(threadIdx.x & 63);
    const uint64_t m = __ballot(i < batch && cu[min(i, batch)] <= token);
    found += __popcll(m);
    if (m != ~uint64_t{0}) break;
  }
  return __builtin_amdgcn_readfirstlane(found - 1);
}

// LDS tiles: rows of DH 16-bit values, 16-byte chunks XORed with swz(row). 16 rows' equal chunks (a row fragment read: lane -> row
// l % 32, 16 bytes) fall on 16 different 16-byte columns of the 64 banks, and the 64-byte windows of 4 consecutive rows (a transposed
// read) on 4 different ones, so both kinds of read are free of conflicts.
template <int DH>
__device__ __forceinline__ int swz(int row) {
  if constexpr (DH == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
  return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}
template <int DH>
__device__ __forceinline__ int tile_at(int row, int chunk) {
  return row * (DH * 2) + ((chunk ^ swz<DH>(row)) << 4);
}

// Fragments of a tile in LDS. rows(): rows row0 .. row0 + 31 (lane l: row l % 32), slice s of 16 values (lane half: 8 of them).
// columns(): the transposed operand: lane l: column 32 dt + l % 32, the 8 rows row0 + 4 (l / 32) + {0..3, 8..11} of a 16-row slice,
// which is the order in which a 32x32 product's result holds its rows.
// A tile starts on a multiple of its row's length, so a slice or column tile is one XOR on the lane's byte address, and rows are
// offsets in the instruction (a reader per buffer: at()).
template <int DH>
struct TileReader {
  uint32_t row_at, col_at[2];
  __device__ __forceinline__ TileReader(const void* lds, int lane) {
    const uint32_t base = lds_addr((const FH_LDS void*)lds);
    const int l32 = lane & 31, hi = lane >> 5;
    row_at = base + l32 * (DH * 2) + ((swz<DH>(l32) ^ hi) << 4);
    const int g = lane >> 4, rr = lane & 15, qd = rr & 3, e = rr >> 2;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int row = 8 * part + 4 * (g >> 1) + e;
      col_at[part] = base + row * (DH * 2) + (qd & 1) * 8 + ((swz<DH>(row) ^ (2 * (g & 1) + (qd >> 1))) << 4);
    }
  }
  // the same fragments of the tile `bytes` further on (a multiple of the row's length)
  __device__ __forceinline__ TileReader at(int bytes) const {
    TileReader r = *this;
    r.row_at += bytes;
    r.col_at[0] += bytes;
    r.col_at[1] += bytes;
    return r;
  }
  __device__ __forceinline__ u32x4_t rows(int row0, int s) const {
    return *(reinterpret_cast<const FH_LDS u32x4_t*>(row_at ^ static_cast<uint32_t>(s << 5)) + row0 * (DH / 8));
  }
  __device__ __forceinline__ u32x4_t columns(int row0, int dt) const {
    const u32x2_t a = read(row0, dt, 0), b = read(row0, dt, 1);
    return u32x4_t{a[0], a[1], b[0], b[1]};
  }

 private:
  __device__ __forceinline__ u32x2_t read(int row0, int dt, int part) const {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                           reinterpret_cast<FH_LDS s16x4_t*>(col_at[part] ^ static_cast<uint32_t>(dt << 6)) +
                                           row0 * (DH / 4)));
  }
};

// The same for 16x16x32 products. rows(): rows row0 .. row0 + 15 (lane l: row l % 16), slice s of 32 values (8 in each 16-lane group).
// columns(): lane l: column 16 dt + l % 16, the rows 4 (l / 16) + {0..3, 16..19} of a 32-row tile: the order in which two results
// of 16 rows hold them.
template <int DH>
struct TileReader16 {
  uint32_t row_at, col_at;
  __device__ __forceinline__ TileReader16(const void* lds, int lane) {
    const uint32_t base = lds_addr((const FH_LDS void*)lds);
    const int l16 = lane & 15, g = lane >> 4, qd = lane & 3, e = (lane >> 2) & 3;
    row_at = base + l16 * (DH * 2) + ((swz<DH>(l16) ^ g) << 4);
    const int row = 4 * g + e;
    col_at = base + row * (DH * 2) + (qd & 1) * 8 + ((swz<DH>(row) ^ (qd >> 1)) << 4);
  }
  __device__ __forceinline__ u32x4_t rows(int row0, int s) const {
    return *(reinterpret_cast<const FH_LDS u32x4_t*>(row_at ^ static_cast<uint32_t>(s << 6)) + row0 * (DH / 8));
  }
  __device__ __forceinline__ u32x4_t columns(int bytes, int dt) const {  // of the tile `bytes` further on
    const uint32_t at = col_at ^ static_cast<uint32_t>(dt << 5);
    const u32x2_t a = read(at + bytes), b = read(at + bytes + 16 * DH * 2);
    return u32x4_t{a[0], a[1], b[0], b[1]};
  }

 private:
  __device__ __forceinline__ static u32x2_t read(uint32_t at) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<FH_LDS s16x4_t*>(at)));
  }
};

// Values that are not finite, in a block of keys that some rows of a workgroup's tile see and others do not. A product sums over the whole
// block, and 0 times NaN is NaN: so there they are replaced by zeros in LDS, and their places are noted, for the rows that do see them to
// be given them at the end.
template <typename T>
constexpr uint32_t kExponent = std::is_same_v<T, bf16_t> ? 0x7f80 : 0x7c00;  // not finite: all of these bits
// w: the chunks that this thread has written to rows row0, row0 + PASS .. of the tile in LDS; note(row, column, bits). 10 instructions per
// chunk, in such blocks only. (No loop in the rare part, and none that the compiler makes for atomics on one address: either gives the
// whole kernel 16 registers more, which cost the gradients with 64 dims a wave per SIMD, 53 us instead of 48.)
template <typename T, int DH, int PASS, int N, typename Note>
__device__ __forceinline__ void scrub(unsigned char* tile, int row0, int chunk, const u32x4_t (&w)[N], Note note) {
  constexpr uint32_t ONES = kExponent<T>, LOW = ONES & (0u - ONES);
  uint32_t carry = 0;  // into a value's sign bit: an exponent of ones
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) carry |= (w[n][j] & (ONES * 0x10001u)) + LOW * 0x10001u;
  if ((carry & 0x80008000u) == 0) return;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    u32x4_t x = w[n];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t bits = (x[j / 2] >> (16 * (j & 1))) & 0xffffu;
      if ((bits & ONES) == ONES) {
        note(row0 + n * PASS, chunk * 8 + j, bits);
        x[j / 2] &= j & 1 ? 0xffffu : 0xffff0000u;
      }
    }
    *reinterpret_cast<u32x4_t*>(tile + tile_at<DH>(row0 + n * PASS, chunk)) = x;
  }
}

// The first key of each column of values that holds +inf or NaN, and that holds -inf or NaN.
template <typename T, int DH>
struct NotFinite {
  int first[2][DH], any;
  __device__ __forceinline__ void clear(int tid) {  // by 2 DH threads or more
    if (tid < 2 * DH) first[tid / DH][tid % DH] = 0x7fffffff;
    if (tid == 0) any = 0;
  }
  __device__ __forceinline__ void note(int key, int d, uint32_t bits) {
    const bool nan = (bits & 0x7fffu) > kExponent<T>, negative = (bits & 0x8000u) != 0;
    if (nan || !negative) atomicMin(&first[0][d], key);
    if (nan || negative) atomicMin(&first[1][d], key);
    any = 1;
  }
  // what column d's sum gains for a row that sees the keys up to lim
  __device__ __forceinline__ float gain(int d, int lim) const {
    const float plus = lim >= first[0][d] ? __builtin_inff() : 0.0f, minus = lim >= first[1][d] ? __builtin_inff() : 0.0f;
    return plus - minus;
  }
};

// Two values rounded to nearest even in one instruction for either type, a NaN to a NaN. (store2 gives an f16 NaN one set of bits, by
// a branch per value: the forward of 7 sequences of 0 .. 200 tokens in f16 took 11.5 us with it instead of 7.5.)
template <typename T>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef std::conditional_t<std::is_same_v<T, bf16_t>, __bf16, _Float16> t;
  typedef t t2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, t2));
}

// max(m, a, b), one v_max3_f32; a NaN counts for nothing. (Not as inline assembly: a, b are products' results, and the compiler keeps the
// wait states that the matrix unit needs before they are read only for instructions that it knows.)
__device__ __forceinline__ float max3(float m, float a, float b) { return fmaxf(fmaxf(m, a), b); }

// max / sum of a lane's value and the other half's (same row of a 32x32 result, the other 16 of its values)
__device__ __forceinline__ void both_halves(float v, float& low, float& high) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  low = __uint_as_float(r[0]);
  high = __uint_as_float(r[1]);
}
__device__ __forceinline__ float half_max(float v) {
  float a, b;
  both_halves(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float half_sum(float v) {
  float a, b;
  both_halves(v, a, b);
  return a + b;
}

// over the 4 lanes l, l + 16, l + 32, l + 48
__device__ __forceinline__ float quarter_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return half_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarter_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return half_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

__device__ __forceinline__ void clear(f32x16_t& a) {
#pragma unroll
  for (int x = 0; x < 16; ++x) a[x] = 0.0f;
}

// f16's range for the operand of a product whose sums go on over many tiles: probabilities of long rows and derivatives of small ones
// lie below its smallest values, derivatives of large ones past its largest. A lane's sums (a column of the result, shared by the lane
// halves) are kept times a power of two, `up`, and its operands are multiplied by that before they are rounded. up falls, never rises:
// where the tile's largest operand would pass 2^15 it becomes what takes that to 2^10 .. 2^11, and the sums so far are scaled with it.
// So an operand is off by half a step of its own down to 2^-24 of the largest one so far, and by 2^-35 of that below. Nothing for
// bf16, which has fp32's range. Costs f16 gradients 7 to 9 % (2897 + 1034 + 165 tokens, 32 heads over 8 of 128: 456 us instead of 426).
template <typename T>
struct OperandRange {
  uint32_t up = (127u + 60) << 23;  // bits of an fp32 power of two
  template <int N>
  __device__ __forceinline__ void fit(f32x16_t& s, f32x16_t (&acc)[N]) {
    if constexpr (std::is_same_v<T, f16_t>) {
      float top = 0.0f;
#pragma unroll
      for (int x = 0; x < 16; x += 2) top = max3(top, __builtin_fabsf(s[x]), __builtin_fabsf(s[x + 1]));
      top = half_max(top);
      const bool past = top * __uint_as_float(up) > 32768.0f;
      if (__any(past)) {
        const uint32_t next = past ? (264u << 23) - (__float_as_uint(top) & 0x7f800000u) : up;  // 2^10 / 2^floor(log2 top)
        const float f = __uint_as_float(next) * inverse();
        up = next;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int x = 0; x < 16; ++x) acc[i][x] *= f;
      }
#pragma unroll
      for (int x = 0; x < 16; ++x) s[x] *= __uint_as_float(up);
    }
  }
  // the sums as they are
  template <int N>
  __device__ __forceinline__ void undo(f32x16_t (&acc)[N]) const {
    if constexpr (std::is_same_v<T, f16_t>) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) acc[i][x] *= inverse();
    }
  }

 private:
  __device__ __forceinline__ float inverse() const { return __uint_as_float((254u << 23) - up); }
};

// Slice hf (16 of its rows) of a 32x32 result rounded to T, as the operand of the next product.
template <typename T>
__device__ __forceinline__ u32x4_t pack_slice(const f32x16_t& p, int hf) {
  u32x4_t w;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = narrow2<T>(p[8 * hf + 2 * j], p[8 * hf + 2 * j + 1]);
  return w;
}

// Products with their fragments read ahead, in this order: an LDS read takes as long as four products, and the compiler by itself places
// each read one or two products before its use.
// acc = rows row0 .. row0 + 31 of the tile times the fragments f
template <typename T, int DH, int AHEAD = 4>
__device__ __forceinline__ void row_product(const TileReader<DH>& tile, int row0, const u32x4_t (&f)[DH / 16], f32x16_t& acc) {
  constexpr int N = DH / 16;
  u32x4_t r[N];
  clear(acc);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) r[i] = tile.rows(row0, i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    mfma32<T>(r[i], f[i], acc);
    if (i + AHEAD < N) r[i + AHEAD] = tile.rows(row0, i + AHEAD);
    __builtin_amdgcn_sched_barrier(0);
  }
}
// the first 16 rows' fragments of column_product, to be read before the values are ready
template <int DH>
__device__ __forceinline__ void read_columns(const TileReader<DH>& tile, int row0, u32x4_t (&first)[DH / 32]) {
#pragma unroll
  for (int dt = 0; dt < DH / 32; ++dt) first[dt] = tile.columns(row0, dt);
  __builtin_amdgcn_sched_barrier(0);
}
// acc += (rows row0 .. row0 + 31 of the tile)^T times p, a 32x32 result as two packed slices
template <typename T, int DH>
__device__ __forceinline__ void column_product(const TileReader<DH>& tile, int row0, const u32x4_t (&p)[2],
                                               const u32x4_t (&first)[DH / 32], f32x16_t (&acc)[DH / 32]) {
  u32x4_t second[DH / 32];
#pragma unroll
  for (int dt = 0; dt < DH / 32; ++dt) second[dt] = tile.columns(row0 + 16, dt);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int dt = 0; dt < DH / 32; ++dt) mfma32<T>(first[dt], p[0], acc[dt]);
#pragma unroll
  for (int dt = 0; dt < DH / 32; ++dt) mfma32<T>(second[dt], p[1], acc[dt]);
}

// Row x of lane half hi in a 32x32 result.
__device__ __forceinline__ constexpr int result_row(int x, int hi) { return 8 * (x / 4) + 4 * hi + x % 4; }

// Every load so far has arrived. Before a loop whose loads run ahead of their use: without it the compiler, which cannot tell the
// first iteration from the others, waits inside the loop for all loads in flight wherever it uses a value loaded before the loop.
__device__ __forceinline__ void settle() { wait_vmcnt<0>(); }

// LDS changes hands between the lanes of one wave: what they wrote before is there for the reads behind it, and what they read is read
// before the writes behind it. The wave's LDS accesses run in their order, so this costs no instruction; it keeps the compiler, which
// looks at one lane at a time, from moving them across.
__device__ __forceinline__ void hand_over() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A 16-byte chunk of 8 values at p when `there`, else zeros.
__device__ __forceinline__ u32x4_t load_chunk(const uint16_t* p, bool there) {
  u32x4_t v{0, 0, 0, 0};
  if (there) v = *reinterpret_cast<const u32x4_t*>(p);
  return v;
}

// A lane's transposed accumulators (DH / 32 tiles of [32 values of d][32 rows]) as one row of 16-bit values at `row`; dh values are
// kept (dh % 8 == 0, so 4-value pieces are whole).
template <typename T, int DH>
__device__ __forceinline__ void store_row(uint16_t* row, const f32x16_t (&acc)[DH / 32], float scale, int hi, int dh) {
#pragma unroll
  for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * dt + 8 * q + 4 * hi;
      if (d < dh) {
        u32x2_t w;
        w[0] = narrow2<T>(acc[dt][4 * q] * scale, acc[dt][4 * q + 1] * scale);
        w[1] = narrow2<T>(acc[dt][4 * q + 2] * scale, acc[dt][4 * q + 3] * scale);
        *reinterpret_cast<u32x2_t*>(row + d) = w;
      }
    }
}

}  // namespace attn
}  // namespace fh
