// Attention of packed query rows over keys and values that are packed rows themselves (kDense), or rows of a paged cache in 16 bits
// (kPaged) or e4m3 (kE4m3). For row r of a sequence with last visible key lim(r):
//   s_u = scale q . k_u (u <= lim),  m = max s,  l = sum exp(s - m),  out = sum exp(s - m) v / l,  lse = m + log l
// in one pass over blocks of 64 keys with a running m and l (fp32, base 2). A wave owns 32 rows; its workgroup's W waves share the
// blocks in LDS, two buffers, the next block on its way in registers while this one is used. Scores are formed transposed
// (K Q^T), so a lane holds one row's scores: maximum and sum stay in the lane but for one exchange of the halves, and the
// probabilities, rounded to the storage type, are in place as the operand of V^T P^T.
// Measured: 5003 + 2318 + 871 tokens, 32 heads over 8, 128 dims, causal, bf16: 297 to 307 us, 830 to 860 TFLOP/s of visible pairs (a
// library product of 8192^3: 1,249); f16 325. What bounds it at long sequences is that matrix and vector work, about as much of
// each, overlap little: of 657 k cycles per SIMD the matrix unit is busy for 252 k and the vector ALU for 279 k, and the two waves of a
// SIMD, of different workgroups, fall into no order in which one's products run beside the other's exponentials. Within a wave
// the code places a product between every few exponentials; both in separate stretches 310 us; a wait for the next block at the
// loop's start 318; 256 rows per workgroup 302; raised wave priority around the products 312-320. Eight sequences of 512, 16 heads of
// 64: 16.8 us, launch and the latencies of a workgroup's up to eight dependent blocks. Where tiles are few, two waves share 32 rows and
// split each block's keys.
// The accumulators are scaled again only when a row's maximum grows by more than 8 (base 2) over the one in use: sums and
// probabilities then stay within 2^8 of their usual range, which fp32 and the rounding to 16 bits do not notice.
// Masked scores are -inf by selection, never by addition, and rows of keys that are not there are zeros in LDS, so nothing that
// lies behind a sequence's end, on an unused part of a page or on a page number out of range reaches a result; and values that are not
// finite reach the rows that see them only (scrub()).
#pragma once

#include "fh_attention_tile.h"

namespace fh {
namespace attn {

enum KvSource : int { kDense = 0, kPaged = 1, kE4m3 = 2 };

constexpr int kBlock = 64;  // keys per block

struct RowsArgs {
  const uint16_t* q;
  uint16_t* out;
  float* lse;  // [tokens, heads] or null
  int64_t ldq, ldo;
  const int32_t* cu;
  int tokens, batch, heads, kv_heads, dh;
  Divider group;
  int causal;
  float scale;
  int slots;
  // splits > 1: part z of a longer sequence's keys goes to part_out [splits][tokens * heads][dh] (normalised) and part_lse (base 2)
  int splits, part_keys;
  float* part_out;
  float* part_lse;
  // keys and values
  const void* k;
  const void* v;
  int64_t ldk, ldv;  // kDense: elements between tokens
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  const int32_t* table;
  const int32_t* kv_lens;
  int64_t table_stride;
  int pages, page_shift;
};

// 8 e4m3 values times a power of two (the fp32 `scale`), as 8 values of T: exact in bf16; in f16 exact but below its smallest normal
// value, where the values of f16 rows that such a scale was made for do not lie; past T's largest value infinite, see below_infinity().
template <typename T>
__device__ __forceinline__ u32x4_t widen_e4m3(const u32x2_t& w, float scale) {
  u32x4_t o;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (std::is_same_v<T, bf16_t>) {
      o[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, false));
      o[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, true));
    } else {
      o[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], scale, false));
      o[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], scale, true));
    }
  }
  return o;
}
// The largest values of T (f16 63,488 and more, bf16 248 2^120) are nearest to 256 times their row's scale, which T cannot hold: widened,
// they become its largest value. kTopScale: the byte of the least scale with such values.
template <typename T>
constexpr uint32_t kTopScale = std::is_same_v<T, bf16_t> ? 127 + 120 : 127 + 8;
template <typename T>
__device__ __forceinline__ u32x4_t below_infinity(u32x4_t o) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t size = o[i] & 0x7fff7fffu;
    o[i] -= ((size & 0xffffu) == kExponent<T> ? 1u : 0u) + ((size >> 16) == kExponent<T> ? 0x10000u : 0u);
  }
  return o;
}

// One block of BK keys and values on its way from memory to LDS: thread t carries chunk t % CH of rows t / CH + n PASS. Of a paged
// cache, lane j holds the page of key j % BK, looked up one block ahead, and its scales; the threads that carry the row take them from
// that lane.
template <typename T, int DH, int SRC, int THREADS, int BK>
struct KvStage {
  static constexpr int CH = DH / 8, PASS = THREADS / CH, N = BK / PASS;
  static_assert(BK % PASS == 0 && BK <= 64, "whole passes, a lane per key");
  using Raw = std::conditional_t<SRC == kE4m3, u32x2_t, u32x4_t>;
  Raw k[N], v[N];
  int page;         // of this lane's key in the block that load() takes next; -1: none
  uint32_t scales;  // kE4m3: of this lane's key in the block on its way: the key's byte, the value's
  uint64_t there;   // kPaged, kE4m3: keys of that block that exist
  const uint16_t* kp;  // kDense: this thread's chunk of the block that load() takes next
  const uint16_t* vp;

  // before the first load(), with that block's kb
  __device__ __forceinline__ void start(const RowsArgs& a, int begin, const int32_t* table, int kv_head, int kb, int kend, int tid) {
    if constexpr (SRC == kDense) {
      const int64_t row = begin + kb + tid / CH, col = static_cast<int64_t>(kv_head) * a.dh + tid % CH * 8;
      kp = static_cast<const uint16_t*>(a.k) + row * a.ldk + col;
      vp = static_cast<const uint16_t*>(a.v) + row * a.ldv + col;
    } else {
      look_up(a, table, kb, kend, tid);
    }
  }

  __device__ __forceinline__ void look_up(const RowsArgs& a, const int32_t* table, int kb, int kend, int tid) {
    if constexpr (SRC != kDense) {
      const int key = kb + (tid & (BK - 1));
      page = key < kend ? table[key >> a.page_shift] : -1;
    }
  }

  // STEP: from this block to the next that this stage takes
  template <int STEP = BK>
  __device__ __forceinline__ void load(const RowsArgs& a, const int32_t* table, int kv_head, int kb, int kend, int tid) {
    const int chunk = tid % CH, row0 = tid / CH;
    const bool inside = chunk * 8 < a.dh;
    if constexpr (SRC == kDense) {
      if (kb + BK <= kend && a.dh == DH) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          k[n] = *reinterpret_cast<const u32x4_t*>(kp + n * PASS * a.ldk);
          v[n] = *reinterpret_cast<const u32x4_t*>(vp + n * PASS * a.ldv);
        }
      } else {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const bool ok = inside && kb + row0 + n * PASS < kend;
          k[n] = load_chunk(kp + n * PASS * a.ldk, ok);
          v[n] = load_chunk(vp + n * PASS * a.ldv, ok);
        }
      }
      kp += STEP * a.ldk;
      vp += STEP * a.ldv;
      return;
    }
    const int in_page = (1 << a.page_shift) - 1;
    auto cache_row = [&](int p, int key) {
      return ((static_cast<int64_t>(p) << a.page_shift) + (key & in_page)) * a.kv_heads + kv_head;
    };
    if constexpr (SRC != kDense) {
      if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages)) page = -1;
      there = __ballot(page >= 0);
      if constexpr (BK < 64) there |= ~uint64_t{0} << BK;
    }
    if constexpr (SRC == kE4m3) {
      scales = 0x7f7fu;
      if (page >= 0) {
        const int64_t row = cache_row(page, kb + (tid & (BK - 1)));
        scales = a.k_scale[row] | (static_cast<uint32_t>(a.v_scale[row]) << 8);
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int key = kb + row0 + n * PASS;
      if constexpr (SRC != kDense) {
        const int p = __shfl(page, row0 + n * PASS, 64);
        const bool ok = inside && p >= 0;
        const int64_t at = cache_row(p, key) * a.dh + chunk * 8;
        if constexpr (SRC == kPaged) {
          k[n] = load_chunk(static_cast<const uint16_t*>(a.k) + at, ok);
          v[n] = load_chunk(static_cast<const uint16_t*>(a.v) + at, ok);
        } else {
          k[n] = u32x2_t{0, 0};
          v[n] = u32x2_t{0, 0};
          if (ok) {
            k[n] = *reinterpret_cast<const u32x2_t*>(static_cast<const uint8_t*>(a.k) + at);
            v[n] = *reinterpret_cast<const u32x2_t*>(static_cast<const uint8_t*>(a.v) + at);
          }
        }
      }
    }
    look_up(a, table, kb + STEP, kend, tid);
  }

  __device__ __forceinline__ void store(unsigned char* kbuf, unsigned char* vbuf, int tid) const {
    const int chunk = tid % CH, row0 = tid / CH;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int at = tile_at<DH>(row0 + n * PASS, chunk);
      u32x4_t kw, vw;
      if constexpr (SRC == kE4m3) {
        const uint32_t sc = __shfl(scales, row0 + n * PASS, 64);
        kw = widen_e4m3<T>(k[n], __uint_as_float((sc & 0xffu) << 23));
        vw = widen_e4m3<T>(v[n], __uint_as_float((sc >> 8) << 23));
      } else {
        kw = k[n];
        vw = v[n];
      }
      *reinterpret_cast<u32x4_t*>(kbuf + at) = kw;
      *reinterpret_cast<u32x4_t*>(vbuf + at) = vw;
    }
    if constexpr (SRC == kE4m3) {
      // rare, so looked for once per key (per chunk, on the way: 64 sequences' step 149 us instead of 142); in a loop only where a
      // thread has more chunks than registers for them (the loop's own addresses spill in the 256-thread form)
      if (__any((scales & 0xffu) >= kTopScale<T> || (scales >> 8) >= kTopScale<T>)) {
#pragma unroll(N <= 4 ? N : 1)
        for (int n = 0; n < N; ++n) {
          const int at = tile_at<DH>(row0 + n * PASS, chunk);
          *reinterpret_cast<u32x4_t*>(kbuf + at) = below_infinity<T>(*reinterpret_cast<const u32x4_t*>(kbuf + at));
          *reinterpret_cast<u32x4_t*>(vbuf + at) = below_infinity<T>(*reinterpret_cast<const u32x4_t*>(vbuf + at));
        }
      }
    }
  }

  // after store(), before the next load()
  template <typename Note>
  __device__ __forceinline__ void scrub_values(unsigned char* vbuf, int tid, Note note) const {
    const int chunk = tid % CH, row0 = tid / CH;
    if constexpr (SRC == kE4m3) {
      u32x4_t w[N];
#pragma unroll
      for (int n = 0; n < N; ++n) w[n] = *reinterpret_cast<const u32x4_t*>(vbuf + tile_at<DH>(row0 + n * PASS, chunk));
      scrub<T, DH, PASS>(vbuf, row0, chunk, w, note);
    } else {
      scrub<T, DH, PASS>(vbuf, row0, chunk, v, note);
    }
  }
};

// A row's factor and log-sum-exp (base 2) where its sum is 0. No key seen: zeros, and -inf. Keys seen, every score of them -inf: 0 / 0, so
// NaN; as one of several parts zeros that weigh less than any finite score's, with kNoScore for the join to tell.
constexpr float kNoScore = -3.402823466e38f;
__device__ __forceinline__ void weigh_nothing(bool sees, bool whole, float& inv, float& lse2) {
  inv = sees && whole ? __builtin_nanf("") : 0.0f;
  lse2 = sees && !whole ? kNoScore : -__builtin_inff();
}

// The running softmax of a wave's 32 rows over blocks of NT 32-key tiles in LDS, and the accumulators of the output.
template <typename T, int DH>
struct RowState {
  float m = -__builtin_inff(), l = 0.0f;  // l: the lane half's share
  f32x16_t o[DH / 32];
  __device__ __forceinline__ RowState() {
#pragma unroll
    for (int dt = 0; dt < DH / 32; ++dt) clear(o[dt]);
  }

  // One 32-key tile. raise(): takes the running maximum up to the tile's, and returns the reference of its exponentials; mixed():
  // exponentials, their sum, and the probabilities as the operand of V^T P^T.
  // key: the tile's first; there: bit u of the tile's keys that exist
  __device__ __forceinline__ static void mask(f32x16_t& s, int key, int lim, uint32_t there, int hi) {
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const int u = result_row(x, hi);
      s[x] = key + u <= lim && ((there >> u) & 1) != 0 ? s[x] : -__builtin_inff();
    }
  }
  __device__ __forceinline__ float raise(const f32x16_t& s, float c) {
    float top = -__builtin_inff();
#pragma unroll
    for (int x = 0; x < 16; x += 2) top = max3(top, s[x], s[x + 1]);
    top = half_max(top) * c;
    if (__any(top > m + 8.0f)) {
      const float next = fmaxf(m, top);
      const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[dt][x] *= f;
    }
    return m == -__builtin_inff() ? 0.0f : m;
  }
  // weigh the tile s (reference `ref`) into p while the next tile's scores are formed from kt: a product, then the exponentials of as
  // many values as take its time, and so on in this order; fragments are read three products ahead. vf: the first half of the
  // values' fragments, read on the way.
  __device__ __forceinline__ void mixed(f32x16_t& s, float c, float ref, u32x4_t (&p)[2], const TileReader<DH>& kt, int row0,
                                        const u32x4_t (&qf)[DH / 16], f32x16_t& next, const TileReader<DH>& vt, int vrow,
                                        u32x4_t (&vf)[DH / 32]) {
    constexpr int N = DH / 16, PER = 16 / N, AHEAD = 3;
    u32x4_t kf[N];
    clear(next);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) kf[i] = kt.rows(row0, i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      mfma32<T>(kf[i], qf[i], next);
      if (i + AHEAD < N) kf[i + AHEAD] = kt.rows(row0, i + AHEAD);
      if (i >= N - DH / 32) vf[i - (N - DH / 32)] = vt.columns(vrow, i - (N - DH / 32));
#pragma unroll
      for (int x = PER * i; x < PER * (i + 1); ++x) {
        s[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x], c, -ref));
        l += s[x];
      }
#pragma unroll
      for (int x = PER * i; x < PER * (i + 1); x += 2) p[x / 8][x % 8 / 2] = narrow2<T>(s[x], s[x + 1]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // the sums of the wave whose `share` is 1 go into the other's, through room[.. * 64]
  __device__ __forceinline__ void join(float* room, int share) {
    if (share == 1) {
      room[0] = m;
      room[64] = l;
#pragma unroll
      for (int i = 0; i < DH / 2; ++i) room[(2 + i) * 64] = o[i / 16][i % 16];
    }
    __syncthreads();
    if (share == 1) return;
    const float other = room[0], top = fmaxf(m, other), ref = top == -__builtin_inff() ? 0.0f : top;
    const float f = __builtin_amdgcn_exp2f(m - ref), g = __builtin_amdgcn_exp2f(other - ref);
    m = top;
    l = l * f + room[64] * g;
#pragma unroll
    for (int i = 0; i < DH / 2; ++i) o[i / 16][i % 16] = o[i / 16][i % 16] * f + room[(2 + i) * 64] * g;
  }
  // sees(): whether the lane's row sees a key, asked of the whole wave where a row's sum is 0
  template <typename Sees>
  __device__ __forceinline__ void finish(float& inv, float& lse2, bool whole, Sees sees) {
    const float sum = half_sum(l);
    inv = 1.0f / sum;
    lse2 = m + __log2f(sum);
    if (__any(sum == 0.0f)) {
      const bool any = sees();
      if (sum == 0.0f) weigh_nothing(any, whole, inv, lse2);
    }
  }

  __device__ __forceinline__ void write_part(const RowsArgs& a, int64_t row, float inv, float lse2, int hi) const {
    if (hi == 0) a.part_lse[row] = lse2;
    float* p = a.part_out + row * a.dh;
#pragma unroll
    for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d = 32 * dt + 8 * q + 4 * hi;
        if (d < a.dh)
          *reinterpret_cast<float4*>(p + d) =
              make_float4(o[dt][4 * q] * inv, o[dt][4 * q + 1] * inv, o[dt][4 * q + 2] * inv, o[dt][4 * q + 3] * inv);
      }
  }
};

// The tile of rows that a workgroup takes and the keys that they see.
struct RowTile {
  Span seq;
  int rows;         // of the sequence and key head
  int tile0;        // the tile's first row
  int keys, first;  // keys of the sequence, and the place of its first row among them
  const int32_t* table;

  // false: no tile at this slot
  template <int SRC>
  __device__ __forceinline__ bool find(const RowsArgs& a, int slot, int shift) {
    const int group = static_cast<int>(a.group.d);
    int first_slot = 0;
    const int b = find_sequence(a.cu, a.batch, a.tokens, group, shift, slot, first_slot, seq);
    if (b < 0) return false;
    const int new_rows = seq.end - seq.begin;
    rows = new_rows * group;
    tile0 = (slot - first_slot) << shift;
    if (!tile_in(tile0, rows)) return false;
    keys = new_rows;
    first = 0;
    table = nullptr;
    if constexpr (SRC != kDense) {
      // a length past what the block table's row can hold is taken as that
      const int64_t cap = a.table_stride << a.page_shift;
      keys = max(a.kv_lens[b], 0);
      if (keys > cap) keys = static_cast<int>(cap);
      first = keys - new_rows;
      table = a.table + b * a.table_stride;
    }
    return true;
  }
  __device__ __forceinline__ int limit(const RowsArgs& a, int r) const {  // last visible key of row r
    return a.causal ? min(first + divide(min(r, rows - 1), a.group), keys - 1) : keys - 1;
  }
  // Whether any of the keys kbegin .. min(lim, kend - 1) exists; by a whole wave (lim is a lane's), 64 pages at a time.
  template <int SRC>
  __device__ __forceinline__ bool sees(const RowsArgs& a, int kbegin, int kend, int lim) const {
    if constexpr (SRC == kDense) return kbegin <= min(lim, kend - 1);
    const int pages = kbegin < kend ? ((kend - 1) >> a.page_shift) + 1 : 0;
    for (int base = kbegin >> a.page_shift; base < pages; base += 64) {
      const int i = base + static_cast<int>(threadIdx.x & 63);
      const uint64_t there = __ballot(i < pages && static_cast<uint32_t>(table[min(i, pages - 1)]) < static_cast<uint32_t>(a.pages));
      if (there != 0) return max((base + __builtin_ctzll(there)) << a.page_shift, kbegin) <= lim;  // the first one
    }
    return false;
  }
  // Parts: z takes keys z * part .. (z + 1) * part - 1, the last part all that follow. False: nothing for this part to write (a
  // sequence that the first part covers is written whole by it; the join goes by the same rule).
  __device__ __forceinline__ bool part(const RowsArgs& a, int z, int& kbegin, int& kend, bool& whole) const {
    whole = a.splits == 1 || keys <= a.part_keys;
    if (whole) return z == 0;
    kbegin = z * a.part_keys;
    if (z + 1 < a.splits) kend = min(kend, kbegin + a.part_keys);
    return kbegin < keys;
  }
};

// KSHARE 2: two waves share 32 rows, each taking one 32-key tile of every block; their sums are joined through LDS.
template <typename T, int DH, int SRC, int W, int KSHARE>
__global__ __launch_bounds__(W * 64, 2) void attention_rows_kernel(const RowsArgs a) {
  constexpr int BYTES = kBlock * DH * 2;  // one block of keys, or of values
  constexpr int ROWS = 32 * W / KSHARE;
  static_assert((ROWS & (ROWS - 1)) == 0, "rows per workgroup: a power of two");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4 * BYTES];
  __shared__ NotFinite<T, DH> bad;

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Neighbouring workgroups take neighbouring key heads of one slot: with the dispatch order over the 8 XCDs, an XCD sees few heads'
  // keys and values at a time. The last slots, a causal sequence's longest, go first.
  const int kv_head = static_cast<int>(blockIdx.x) % a.kv_heads;
  const int slot = a.slots - 1 - static_cast<int>(blockIdx.x) / a.kv_heads;
  RowTile tile;
  if (!tile.find<SRC>(a, slot, __builtin_ctz(ROWS))) return;
  int kbegin = 0, kend = tile.limit(a, tile.tile0 + ROWS - 1) + 1;
  bool whole;
  if (!tile.part(a, static_cast<int>(blockIdx.z), kbegin, kend, whole)) return;

  const int share = wave / (W / KSHARE);
  const int r0 = tile.tile0 + wave % (W / KSHARE) * 32, r = r0 + l32;
  const bool live = r < tile.rows;
  const int lim = tile.limit(a, r);
  const int lim_low = tile.limit(a, r0), lim_high = tile.limit(a, r0 + 31);  // rows are in order of their tokens
  const int token = divide(min(r, tile.rows - 1), a.group);
  const int group = static_cast<int>(a.group.d);
  const int head = kv_head * group + (min(r, tile.rows - 1) - token * group);
  const int64_t trow = tile.seq.begin + token;

  u32x4_t qf[DH / 16];
  {
    const uint16_t* qr = a.q + trow * a.ldq + static_cast<int64_t>(head) * a.dh;
#pragma unroll
    for (int s = 0; s < DH / 16; ++s) qf[s] = load_chunk(qr + 16 * s + 8 * hi, live && 16 * s + 8 * hi < a.dh);
  }

  const float c = a.scale * kLog2e;
  RowState<T, DH> state;
  KvStage<T, DH, SRC, W * 64, kBlock> stage;
  const TileReader<DH> tiles(lds, lane);
  uint64_t there = ~uint64_t{0}, there_next = ~uint64_t{0};
  // rows of the tile see the keys up to `common`; blocks with others are looked through for values that are not finite
  const int common = tile.limit(a, tile.tile0);
  const bool uneven = kbegin < kend && common != tile.limit(a, tile.tile0 + ROWS - 1);
  auto look = [&](unsigned char* values, int kb) {
    if (uneven && kb + kBlock - 1 > common)
      stage.scrub_values(values, tid, [&](int row, int d, uint32_t bits) { bad.note(kb + row, d, bits); });
  };
  if (kbegin < kend) {
    stage.start(a, tile.seq.begin, tile.table, kv_head, kbegin, kend, tid);
    stage.load(a, tile.table, kv_head, kbegin, kend, tid);
    if (uneven) {
      bad.clear(tid);
      __syncthreads();
    }
    stage.store(lds, lds + BYTES, tid);
    look(lds + BYTES, kbegin);
    if constexpr (SRC != kDense) there = stage.there;
  }
  settle();
  __syncthreads();
  if (kbegin + kBlock < kend) stage.load(a, tile.table, kv_head, kbegin + kBlock, kend, tid);
  f32x16_t s0, s1;
  row_product<T, DH>(tiles, 32 * share, qf, s0);
  int buf = 0;
  for (int kb = kbegin; kb < kend; kb += kBlock) {
    const bool more = kb + kBlock < kend, mine = kb <= lim_high;
    const bool edge = kb + kBlock - 1 > lim_low || there != ~uint64_t{0};
    const TileReader<DH> kt = tiles.at(buf * 2 * BYTES), vt = kt.at(BYTES);
    u32x4_t p[2], vf[DH / 32];
    if (KSHARE == 1 && mine) {
      if (edge) state.mask(s0, kb, lim, static_cast<uint32_t>(there), hi);
      const float ref = state.raise(s0, c);
      state.mixed(s0, c, ref, p, kt, 32, qf, s1, vt, 0, vf);
    }
    __syncthreads();  // every wave has read the other buffer's last values
    if (more) {
      unsigned char* next = lds + (buf ^ 1) * 2 * BYTES;
      stage.store(next, next + BYTES, tid);
      look(next + BYTES, kb + kBlock);
      if constexpr (SRC != kDense) there_next = stage.there;
      if (kb + 2 * kBlock < kend) stage.load(a, tile.table, kv_head, kb + 2 * kBlock, kend, tid);
    }
    if (KSHARE == 1 && mine) column_product<T, DH>(vt, 0, p, vf, state.o);
    __syncthreads();  // the next block is in LDS
    if (KSHARE == 2) {
      if (mine) {
        if (edge) state.mask(s0, kb + 32 * share, lim, static_cast<uint32_t>(there >> (32 * share)), hi);
        const float ref = state.raise(s0, c);
        state.mixed(s0, c, ref, p, tiles.at((buf ^ 1) * 2 * BYTES), 32 * share, qf, s1, vt, 32 * share, vf);
        column_product<T, DH>(vt, 32 * share, p, vf, state.o);
        s0 = s1;
      }
    } else if (mine) {
      if (edge) state.mask(s1, kb + 32, lim, static_cast<uint32_t>(there >> 32), hi);
      const float ref = state.raise(s1, c);
      // (after the last block: scores of nothing, unused)
      state.mixed(s1, c, ref, p, tiles.at((buf ^ 1) * 2 * BYTES), 0, qf, s0, vt, 32, vf);
      column_product<T, DH>(vt, 32, p, vf, state.o);
    }
    there = there_next;
    buf ^= 1;
  }

  if constexpr (KSHARE == 2) {
    __syncthreads();  // the last block is used
    state.join(reinterpret_cast<float*>(lds) + wave % (W / 2) * ((DH / 2 + 2) * 64) + lane, share);
    if (share == 1) return;
  }
  float inv, lse2;
  state.finish(inv, lse2, whole, [&] { return tile.template sees<SRC>(a, kbegin, kend, lim); });
  if (!live) return;
  if (uneven && bad.any != 0) {
#pragma unroll
    for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
      for (int x = 0; x < 16; ++x) state.o[dt][x] += bad.gain(32 * dt + result_row(x, hi), lim);
  }
  if (!whole) {
    state.write_part(a, (static_cast<int64_t>(blockIdx.z) * a.tokens + trow) * a.heads + head, inv, lse2, hi);
    return;
  }
  store_row<T, DH>(a.out + trow * a.ldo + static_cast<int64_t>(head) * a.dh, state.o, inv, hi, a.dh);
  if (a.lse != nullptr && hi == 0) a.lse[trow * a.heads + head] = lse2 * kLn2;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace attn
}  // namespace fh
