// Attention over packed sequences with grouped heads (fh_attention_packed_fwd) and its gradients (fh_attention_packed_grad).
// Forward: attention_rows_kernel of fh_attention_rows.h over dense keys and values.
//
// Gradients, with D = sum_d dout out, p = exp(scale q.k - lse), dp = dout.v, ds = p (dp - D):
//   dq = scale sum_u ds k_u,  dk = scale sum_r ds q_r,  dv = sum_r p dout_r,
// the sums over r running over the rows of every head of the group. Two kernels, each forming p and dp again from q, k, v and
// dout (7 products instead of the 5 that one kernel with atomic sums of dq would need), so that every sum has one owner and one
// order: results do not depend on scheduling, and no fp32 copy of dq is needed.
//   attention_dq_kernel:  32 rows per wave as in the forward; D is formed from its rows and kept for the second kernel.
//   attention_dkv_kernel: 32 keys per wave, keys and values in registers, blocks of 64 rows of q and dout in LDS.
// p and ds are rounded to the storage type as operands of the second products, in f16 times a power of two that keeps them in its range
// (OperandRange); everything else is fp32.
// Measured: 2897 + 1034 + 165 tokens, 32 heads over 8, 128 dims, causal, bf16: 425 to 433 us (traced: dq 164, dk and dv 248, the
// parts' sum 12), 455 TFLOP/s counted as 5 products, 637 as the 7 that are made; f16 456; 3300 tokens in 8 sequences, 16 heads of 64: 48.5 us.
// Bound by the waits of a tile's dependent steps (product, exponentials, product), which two waves per SIMD do not fill: the matrix
// unit is busy for 116 k of 379 k cycles per SIMD in dq and 190 k of 604 k in dk and dv, the vector ALU for 97 k and 177 k.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "fh_attention_rows.h"

namespace fh {
namespace {

using namespace attn;

struct GradArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* out;
  const uint16_t* dout;
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  const float* lse;
  float* delta;  // [tokens, heads]
  const int32_t* cu;
  int64_t ldq, ldk, ldv, ldo;
  int tokens, batch, heads, kv_heads, dh;
  Divider group;
  int causal;
  float scale;
  int slots;
  int tile_keys;  // keys of a workgroup of the second kernel
  int parts;      // of the rows of a key tile
  float* part;  // parts > 1: [parts][dv, dk][tokens][kv_heads * dh]
};

constexpr int kWholeBlocks = 32;  // key tiles of no more blocks of rows are not cut
constexpr int kLeastBlocks = 8;   // of a part

// KSHARE 2: two waves share 32 rows, each taking one 32-key tile of a block, and their sums are joined through LDS.
template <typename T, int DH, int W, int KSHARE>
__global__ __launch_bounds__(W * 64, 2) void attention_dq_kernel(const GradArgs a) {
  constexpr int BYTES = kBlock * DH * 2;
  constexpr int ROWS = 32 * W / KSHARE, SHIFT = __builtin_ctz(ROWS);
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4 * BYTES];
  // The first key with a value that is not finite, of those that scrub() zeroes, per 8 columns: every score of a row that sees it, so every
  // derivative, is not finite either.
  __shared__ int first_bad[DH / 8];

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kv_head = static_cast<int>(blockIdx.x) % a.kv_heads;
  const int slot = a.slots - 1 - static_cast<int>(blockIdx.x) / a.kv_heads;
  const int group = static_cast<int>(a.group.d);
  int first_slot = 0;
  Span seq;
  if (find_sequence(a.cu, a.batch, a.tokens, group, SHIFT, slot, first_slot, seq) < 0) return;
  const int keys = seq.end - seq.begin, rows = keys * group;
  const int tile0 = (slot - first_slot) * ROWS;
  if (!tile_in(tile0, rows)) return;
  auto limit = [&](int r) { return a.causal ? divide(min(r, rows - 1), a.group) : keys - 1; };
  const int kend = limit(tile0 + ROWS - 1) + 1;

  const int share = wave / (W / KSHARE);
  const int r0 = tile0 + wave % (W / KSHARE) * 32, r = r0 + l32;
  const bool live = r < rows;
  const int lim = limit(r), lim_low = limit(r0), lim_high = limit(r0 + 31);
  const int token = divide(min(r, rows - 1), a.group);
  const int head = kv_head * group + (min(r, rows - 1) - token * group);
  const int64_t trow = seq.begin + token;

  u32x4_t qf[DH / 16], gf[DH / 16];
  float delta = 0.0f;
  {
    const uint16_t* qr = a.q + trow * a.ldq + static_cast<int64_t>(head) * a.dh;
    const int64_t oat = trow * a.ldo + static_cast<int64_t>(head) * a.dh;
#pragma unroll
    for (int s = 0; s < DH / 16; ++s) {
      const int d = 16 * s + 8 * hi;
      const bool ok = live && d < a.dh;
      qf[s] = load_chunk(qr + d, ok);
      gf[s] = load_chunk(a.dout + oat + d, ok);
      const u32x4_t ov = load_chunk(a.out + oat + d, ok);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        delta = __builtin_fmaf(load_lo<T>(gf[s][j]), load_lo<T>(ov[j]), delta);
        delta = __builtin_fmaf(load_hi<T>(gf[s][j]), load_hi<T>(ov[j]), delta);
      }
    }
  }
  delta = half_sum(delta);
  const int64_t stat = trow * a.heads + head;
  const float lse2 = live ? a.lse[stat] * kLog2e : 0.0f;
  const float c = a.scale * kLog2e;

  f32x16_t acc[DH / 32];
#pragma unroll
  for (int dt = 0; dt < DH / 32; ++dt) clear(acc[dt]);

  OperandRange<T> range;

  // keys and values as the forward stages them
  RowsArgs kv{};
  kv.k = a.k;
  kv.v = a.v;
  kv.ldk = a.ldk;
  kv.ldv = a.ldv;
  kv.dh = a.dh;
  KvStage<T, DH, kDense, W * 64, kBlock> stage;
  const TileReader<DH> tiles(lds, lane);
  auto scores = [&](const TileReader<DH>& kt, const TileReader<DH>& vt, int t, f32x16_t& s, f32x16_t& dp) {  // q k, dout v: 32 keys
    clear(s);
    clear(dp);
#pragma unroll
    for (int i = 0; i < DH / 16; ++i) {
      mfma32<T>(kt.rows(32 * t, i), qf[i], s);
      mfma32<T>(vt.rows(32 * t, i), gf[i], dp);
    }
  };
  stage.start(kv, seq.begin, nullptr, kv_head, 0, kend, tid);
  stage.load(kv, nullptr, kv_head, 0, kend, tid);
  const int common = limit(tile0);
  const bool uneven = common != kend - 1;
  auto look = [&](unsigned char* keys_at, int kb) {
    if (uneven && kb + kBlock - 1 > common)
      scrub<T, DH, stage.PASS>(keys_at, tid / stage.CH, tid % stage.CH, stage.k,
                               [&](int row, int d, uint32_t) { atomicMin(&first_bad[d / 8], kb + row); });
  };
  if (uneven) {
    if (tid < DH / 8) first_bad[tid] = 0x7fffffff;
    __syncthreads();
  }
  stage.store(lds, lds + BYTES, tid);
  look(lds, 0);
  settle();
  __syncthreads();
  int buf = 0;
  for (int kb = 0; kb < kend; kb += kBlock) {
    const bool more = kb + kBlock < kend;
    if (more) stage.load(kv, nullptr, kv_head, kb + kBlock, kend, tid);
    if (kb <= lim_high) {
      const TileReader<DH> kt = tiles.at(buf * 2 * BYTES), vt = kt.at(BYTES);
      const bool edge = kb + kBlock - 1 > lim_low;
      if (lim_high < kBlock) {
        // Rows that see one block: D = sum p dp / sum p from the block itself, as a difference from the first key's dp. D from the
        // rounded output is off by a rounding of every out, which counts beside dp - D where a row sees few keys; and where it sees
        // one, dp - D has to vanish.
        float d0 = 0.0f, d = 0.0f, sum = 0.0f, unused;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x16_t s, dp;
          scores(kt, vt, t, s, dp);
          if (t == 0) both_halves(dp[0], d0, unused);
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const bool seen = 32 * t + result_row(x, hi) <= lim;
            const float p = seen ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[x], c, -lse2)) : 0.0f;
            sum += p;
            d = seen ? __builtin_fmaf(p, dp[x] - d0, d) : d;
          }
        }
        delta = d0 + half_sum(d) / half_sum(sum);
      }
#pragma unroll
      for (int i = 0; i < 2 / KSHARE; ++i) {
        const int t = KSHARE == 2 ? share : i;
        f32x16_t s, dp;
        scores(kt, vt, t, s, dp);
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x], c, -lse2));
          s[x] = p * (dp[x] - delta);
        }
        if (edge) {
#pragma unroll
          for (int x = 0; x < 16; ++x) s[x] = kb + 32 * t + result_row(x, hi) <= lim ? s[x] : 0.0f;
        }
        range.fit(s, acc);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const u32x4_t ds = pack_slice<T>(s, hf);
#pragma unroll
          for (int dt = 0; dt < DH / 32; ++dt) mfma32<T>(kt.columns(32 * t + 16 * hf, dt), ds, acc[dt]);
        }
      }
    }
    if (more) {
      unsigned char* next = lds + (buf ^ 1) * 2 * BYTES;
      stage.store(next, next + BYTES, tid);
      look(next, kb + kBlock);
    }
    __syncthreads();
    buf ^= 1;
  }
  range.undo(acc);
  if (uneven) {
    int first = first_bad[0];
#pragma unroll
    for (int i = 1; i < DH / 8; ++i) first = min(first, first_bad[i]);
    if (lim >= first) {
#pragma unroll
      for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
        for (int x = 0; x < 16; ++x) acc[dt][x] = __builtin_nanf("");
    }
  }
  if constexpr (KSHARE == 2) {
    float* room = reinterpret_cast<float*>(lds) + wave % (W / 2) * (DH / 2 * 64) + lane;
    if (share == 1) {
#pragma unroll
      for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
        for (int x = 0; x < 16; ++x) room[(dt * 16 + x) * 64] = acc[dt][x];
    }
    __syncthreads();
    if (share == 1) return;
#pragma unroll
    for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[dt][x] += room[(dt * 16 + x) * 64];
  }
  if (live && hi == 0) a.delta[stat] = delta;
  if (live) store_row<T, DH>(a.dq + trow * a.ldq + static_cast<int64_t>(head) * a.dh, acc, a.scale, hi, a.dh);
}

constexpr int kGradRows = 64;  // rows of q and dout per block

// The rows [begin, end) that part z of a key tile sums over, in whole blocks, and the tile's number of parts.
struct RowRange {
  int begin, end, parts;
};
__device__ __forceinline__ RowRange row_range(const GradArgs& a, int tile0, int rows, int z) {
  const int first = a.causal ? tile0 * static_cast<int>(a.group.d) / kGradRows : 0;  // rows that see key u: r >= u * group
  const int blocks = (rows + kGradRows - 1) / kGradRows - first;
  if (a.parts == 1 || blocks <= kWholeBlocks) return {first * kGradRows, z == 0 ? rows : 0, 1};
  const int per = max((blocks + a.parts - 1) / a.parts, kLeastBlocks);
  return {(first + z * per) * kGradRows, min(rows, (first + (z + 1) * per) * kGradRows), (blocks + per - 1) / per};
}

// 32 PAIRS keys per workgroup of 2 PAIRS waves: waves w and w + PAIRS own the same 32 keys (with 4 pairs on one SIMD); the first
// sums dv (two products: q k and p dout), the second dk (three: q k, dout v and ds q). Forming q k twice leaves each wave one
// accumulator, which is what lets two waves share a SIMD's registers. At the first size above (dk and dv alone): both sums in one wave
// of 400 registers 821 us; this form 255; p handed from the first wave to the second through LDS, four products and a barrier
// more, 304.
template <typename T, int DH, int PAIRS>
__global__ __launch_bounds__(PAIRS * 128, PAIRS == 2 ? 3 : 2) void attention_dkv_kernel(const GradArgs a) {
  constexpr int BYTES = kGradRows * DH * 2, KEYS = 32 * PAIRS, SHIFT = __builtin_ctz(KEYS);
  constexpr int CH = DH / 8, PASS = PAIRS * 128 / CH, N = kGradRows / PASS;
  static_assert(kGradRows % PASS == 0, "whole passes");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4 * BYTES];
  __shared__ __attribute__((aligned(16))) float stats[2][2][kGradRows];  // per buffer: lse (base 2), D
  // Rows with values that are not finite, of those that scrub() zeroes: the last of q per 8 columns (its scores are not finite), the
  // last in each column of dout (dv's; its D is not finite, which reaches dk by itself), and whether there is any.
  __shared__ int last_q[DH / 8], last_dout[DH], any_bad;

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool for_dk = wave >= PAIRS;
  const int kv_head = static_cast<int>(blockIdx.x) % a.kv_heads;
  // the parts of a tile side by side: a causal sequence's first keys, seen by most rows, go first with all their parts
  const int work = static_cast<int>(blockIdx.x) / a.kv_heads, slot = work / a.parts, z = work - slot * a.parts;
  const int group = static_cast<int>(a.group.d);
  int first_slot = 0;
  Span seq;
  if (find_sequence(a.cu, a.batch, a.tokens, 1, SHIFT, slot, first_slot, seq) < 0) return;
  const int keys = seq.end - seq.begin, rows = keys * group;
  const int tile0 = (slot - first_slot) * KEYS;
  if (!tile_in(tile0, keys)) return;
  const RowRange range = row_range(a, tile0, rows, z);
  if (z >= range.parts) return;

  const int k0 = tile0 + (wave & (PAIRS - 1)) * 32, key = k0 + l32;
  const bool live = key < keys;
  const int64_t krow = seq.begin + (live ? key : 0);
  const int64_t col = static_cast<int64_t>(kv_head) * a.dh;
  u32x4_t kf[DH / 16], vf[DH / 16];
#pragma unroll
  for (int s = 0; s < DH / 16; ++s) {
    const int d = 16 * s + 8 * hi;
    kf[s] = load_chunk(a.k + krow * a.ldk + col + d, live && d < a.dh);
    vf[s] = load_chunk(a.v + krow * a.ldv + col + d, live && d < a.dh);
  }
  const int my_first = a.causal ? key * group : 0;

  const int chunk = tid % CH, srow = tid / CH;
  const bool inside = chunk * 8 < a.dh;
  u32x4_t qs[N], gs[N];
  float stat = 0.0f;
  auto load = [&](int rb) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = rb + srow + n * PASS;
      const int token = divide(min(r, rows - 1), a.group);
      const int head = kv_head * group + (min(r, rows - 1) - token * group);
      const int64_t trow = seq.begin + token;
      const int64_t c0 = static_cast<int64_t>(head) * a.dh + chunk * 8;
      qs[n] = load_chunk(a.q + trow * a.ldq + c0, inside && r < rows);
      gs[n] = load_chunk(a.dout + trow * a.ldo + c0, inside && r < rows);
    }
    if (tid < 2 * kGradRows) {
      const int r = rb + (tid & (kGradRows - 1));
      stat = 0.0f;
      if (r < rows) {
        const int token = divide(r, a.group);
        const int64_t at = (seq.begin + token) * static_cast<int64_t>(a.heads) + kv_head * group + (r - token * group);
        stat = tid < kGradRows ? a.lse[at] * kLog2e : a.delta[at];
      }
    }
  };
  auto store = [&](int buf) {
    unsigned char* qb = lds + buf * 2 * BYTES;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int at = tile_at<DH>(srow + n * PASS, chunk);
      *reinterpret_cast<u32x4_t*>(qb + at) = qs[n];
      *reinterpret_cast<u32x4_t*>(qb + BYTES + at) = gs[n];
    }
    if (tid < 2 * kGradRows) stats[buf][tid / kGradRows][tid & (kGradRows - 1)] = stat;
  };

  f32x16_t acc[DH / 32];
#pragma unroll
  for (int dt = 0; dt < DH / 32; ++dt) clear(acc[dt]);
  OperandRange<T> operands;
  const float c = a.scale * kLog2e;
  const TileReader<DH> tiles(lds, lane);
  // blocks of rows that some keys of the tile are not seen by
  auto look = [&](int buf, int rb) {
    if (a.causal && rb < (tile0 + KEYS - 1) * group) {
      unsigned char* qb = lds + buf * 2 * BYTES;
      scrub<T, DH, PASS>(qb, srow, chunk, qs, [&](int row, int d, uint32_t) { atomicMax(&last_q[d / 8], rb + row), any_bad = 1; });
      scrub<T, DH, PASS>(qb + BYTES, srow, chunk, gs, [&](int row, int d, uint32_t) { atomicMax(&last_dout[d], rb + row), any_bad = 1; });
    }
  };
  if (range.begin < range.end) {
    load(range.begin);
    if (tid < DH) last_dout[tid] = -1;
    if (tid < DH / 8) last_q[tid] = -1;
    if (tid == 0) any_bad = 0;
    __syncthreads();
    store(0);
    look(0, range.begin);
  }
  settle();
  __syncthreads();
  int buf = 0;
  for (int rb = range.begin; rb < range.end; rb += kGradRows) {
    const bool more = rb + kGradRows < range.end;
    if (more) load(rb + kGradRows);
    const TileReader<DH> qt = tiles.at(buf * 2 * BYTES), gt = qt.at(BYTES);
#pragma unroll
    for (int t = 0; t < kGradRows / 32; ++t) {
      const int r0 = rb + 32 * t;
      // the wave's first key is seen from row k0 * group on
      if (a.causal && r0 + 32 <= k0 * group) continue;
      const bool edge = a.causal && r0 < (k0 + 31) * group;
      f32x16_t s;
      row_product<T, DH, 3>(qt, 32 * t, kf, s);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 ls = *reinterpret_cast<const float4*>(&stats[buf][0][32 * t + 8 * q + 4 * hi]);
        const float lv[4] = {ls.x, ls.y, ls.z, ls.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * q + j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * q + j], c, -lv[j]));
      }
      const TileReader<DH> operand = for_dk ? qt : gt;
      if (for_dk) {
        f32x16_t dp;
        row_product<T, DH, 3>(gt, 32 * t, vf, dp);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 dl = *reinterpret_cast<const float4*>(&stats[buf][1][32 * t + 8 * q + 4 * hi]);
          const float dd[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) s[4 * q + j] *= dp[4 * q + j] - dd[j];
        }
      }
      if (edge) {
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = r0 + result_row(x, hi) >= my_first ? s[x] : 0.0f;
      }
      operands.fit(s, acc);
      u32x4_t columns[DH / 32], p[2];
      read_columns<DH>(operand, 32 * t, columns);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) p[hf] = pack_slice<T>(s, hf);
      column_product<T, DH>(operand, 32 * t, p, columns, acc);
    }
    if (more) {
      store(buf ^ 1);
      look(buf ^ 1, rb + kGradRows);
    }
    __syncthreads();
    buf ^= 1;
  }
  operands.undo(acc);
  if (!live) return;
  if (range.begin < range.end && a.causal && any_bad != 0) {
    int last = last_q[0];
#pragma unroll
    for (int i = 1; i < DH / 8; ++i) last = max(last, last_q[i]);
#pragma unroll
    for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
      for (int x = 0; x < 16; ++x)
        if (my_first <= max(last, last_dout[32 * dt + result_row(x, hi)])) acc[dt][x] = __builtin_nanf("");
  }
  const float factor = for_dk ? a.scale : 1.0f;
  if (range.parts == 1) {
    store_row<T, DH>(for_dk ? a.dk + krow * a.ldk + col : a.dv + krow * a.ldv + col, acc, factor, hi, a.dh);
    return;
  }
  float* p = a.part + ((static_cast<int64_t>(z) * 2 + for_dk) * a.tokens + krow) * a.kv_heads * a.dh + col;
#pragma unroll
  for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * dt + 8 * q + 4 * hi;
      if (d < a.dh)
        *reinterpret_cast<float4*>(p + d) = make_float4(acc[dt][4 * q] * factor, acc[dt][4 * q + 1] * factor,
                                                        acc[dt][4 * q + 2] * factor, acc[dt][4 * q + 3] * factor);
    }
}

// dk and dv of the key tiles whose rows were cut into parts: the parts' sum, in their order. A wave takes 512 of a token's
// values, two chains of loads a lane: with one, two parts of 4096 tokens, 8 heads of 128 take 2.5 us longer, with four, eight parts of
// 1900 tokens, a head of 64, 2.7.
constexpr int kJoin = 2;

template <typename T>
__global__ __launch_bounds__(256) void attention_dkv_join_kernel(const GradArgs a) {
  const int width = a.kv_heads * a.dh, slices = (2 * width + kJoin * 256 - 1) / (kJoin * 256);
  const int64_t work = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int token = static_cast<int>(work / slices), slice = static_cast<int>(work - static_cast<int64_t>(token) * slices);
  if (token >= a.tokens) return;
  const int b = sequence_of(a.cu, a.batch, token);
  if (b < 0) return;
  const Span seq = sequence(a.cu, b, a.tokens);
  if (token < seq.begin || token >= seq.end) return;
  const int rows = (seq.end - seq.begin) * static_cast<int>(a.group.d);
  const int tile0 = (token - seq.begin) / a.tile_keys * a.tile_keys;
  const int parts = row_range(a, tile0, rows, 0).parts;
  if (parts == 1) return;
  const int64_t stride = static_cast<int64_t>(a.tokens) * width;
  float4 t[kJoin];
  const float* p[kJoin];
  int at[kJoin];
  bool there[kJoin], for_dk[kJoin];
#pragma unroll
  for (int j = 0; j < kJoin; ++j) {
    const int i = ((slice * kJoin + j) * 64 + static_cast<int>(threadIdx.x & 63)) * 4;  // dv's values, then dk's
    there[j] = i < 2 * width;
    for_dk[j] = i >= width;
    at[j] = there[j] ? i - for_dk[j] * width : 0;
    p[j] = a.part + (there[j] && for_dk[j] ? stride : 0) + static_cast<int64_t>(token) * width + at[j];
    t[j] = *reinterpret_cast<const float4*>(p[j]);
  }
#pragma unroll 2
  for (int z = 1; z < parts; ++z) {
#pragma unroll
    for (int j = 0; j < kJoin; ++j) {
      const float4 y = *reinterpret_cast<const float4*>(p[j] + z * 2 * stride);
      t[j].x += y.x;
      t[j].y += y.y;
      t[j].z += y.z;
      t[j].w += y.w;
    }
  }
#pragma unroll
  for (int j = 0; j < kJoin; ++j) {
    if (!there[j]) continue;
    u32x2_t w;
    w[0] = narrow2<T>(t[j].x, t[j].y);
    w[1] = narrow2<T>(t[j].z, t[j].w);
    uint16_t* out = for_dk[j] ? a.dk + token * a.ldk : a.dv + token * a.ldv;
    *reinterpret_cast<u32x2_t*>(out + at[j]) = w;
  }
}

// One wave per row that no sequence covers.
__global__ __launch_bounds__(256) void packed_clear_kernel(const int32_t* cu, int batch, uint4* x, int rows, int64_t chunks) {
  const int row = static_cast<int>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= rows || (row >= cu[0] && row < cu[batch])) return;
  for (int64_t i = threadIdx.x & 63; i < chunks; i += 64) x[row * chunks + i] = uint4{0, 0, 0, 0};
}

fh_status check_packed(const char* fn, const fh_packed_attention* g) {
  const std::string f(fn);
  if (g == nullptr) return fail(FH_INVALID_ARGUMENT, f + ": null descriptor");
  if (g->dtype != FH_BF16 && g->dtype != FH_F16) return fail(FH_UNIMPLEMENTED, f + ": needs bf16 or f16");
  if (g->dh < 8 || g->dh > 128 || g->dh % 8 != 0) return fail(FH_UNIMPLEMENTED, f + ": head dim must be a multiple of 8 up to 128");
  if (g->tokens < 0 || g->batch < 0) return fail(FH_INVALID_ARGUMENT, f + ": negative tokens or batch");
  if (g->heads < 1 || g->kv_heads < 1 || g->heads % g->kv_heads != 0)
    return fail(FH_INVALID_ARGUMENT, f + ": heads must be a multiple of kv_heads");
  if (g->causal != 0 && g->causal != 1) return fail(FH_INVALID_ARGUMENT, f + ": causal must be 0 or 1");
  if (!(g->scale > 0.0f) || !std::isfinite(g->scale)) return fail(FH_INVALID_ARGUMENT, f + ": scale must be positive and finite");
  if (g->heads > 65535 || g->tokens > 0x7fffffff || g->batch > 0x3fffffff ||
      (g->tokens + 256) * g->heads + g->batch * g->kv_heads > 0x7fffffff)
    return fail(FH_INVALID_ARGUMENT, f + ": more than 2^31 rows (tokens x heads)");
  if (g->tokens * g->heads / 128 + (g->batch + 1) * g->kv_heads > kMaxBlocks / 2)
    return fail(FH_INVALID_ARGUMENT, f + ": more rows than one launch takes");
  if (g->q_stride < g->heads * g->dh || g->out_stride < g->heads * g->dh || g->k_stride < g->kv_heads * g->dh ||
      g->v_stride < g->kv_heads * g->dh)
    return fail(FH_INVALID_ARGUMENT, f + ": a row stride is shorter than its row");
  if ((g->q_stride | g->k_stride | g->v_stride | g->out_stride) % 8 != 0)
    return fail(FH_INVALID_ARGUMENT, f + ": row strides must be multiples of 8 elements");
  return FH_OK;
}

// workgroups of `tile`-row tiles with per_token rows a token
int64_t slots_for(const fh_packed_attention& g, int64_t per_token, int64_t tile) { return g.tokens * per_token / tile + g.batch; }

int64_t delta_bytes(const fh_packed_attention& g) { return (g.tokens * g.heads * 4 + 15) / 16 * 16; }

// Two waves share 32 rows where tiles of 128 rows leave CUs with fewer waves than hide the steps of a block: fewer than two
// workgroups a CU in the forward (12 sequences of up to 1886 tokens, 4 heads over 2 of 64: 22.7 us instead of 34; one of 4000, 8 heads
// over 1 of 128: 74 instead of 95; 480 workgroups: 57 either way), one and a half for dq (8 heads of 128 over 2000 tokens: 139 instead
// of 164 in all; 416 workgroups: 50.3 instead of 48.5; 1048: 485 instead of 430).
int key_shares(const fh_packed_attention& g, bool gradients) {
  const int64_t tiles = (g.tokens * (g.heads / g.kv_heads) + 127) / 128 * g.kv_heads, cus = device_cu_count();
  return tiles < (gradients ? cus + cus / 2 : 2 * cus) ? 2 : 1;
}

// dk, dv. Keys per workgroup: 128, or 64 where that leaves fewer than two workgroups a CU and the head dim's registers allow the
// longer staging (3300 tokens in 8 sequences, 16 heads of 64: 48 us in all instead of 57).
int64_t grad_keys(const fh_packed_attention& g) {
  return g.dh <= 64 && (g.tokens + 127) / 128 * g.kv_heads < 2 * device_cu_count() ? 64 : 128;
}
// A key tile's rows are cut into parts where the tiles are few: a causal sequence's first keys are seen by all of its rows, so the
// longest tile would otherwise outlast the others by twice their mean. As many as fill the chip once (three workgroups of 64 keys a CU,
// or one of 128), and at least enough to even the tiles out. 32 heads over 8 of 64, 2800 tokens: 3 parts 137 us in all, 2 161; 8 heads
// over 1 of 64, 1900 tokens: 8 parts 102, 4 143; 8 heads over 2 of 128, 2000 tokens: 8 parts 138, 16 178 (a second round).
int64_t grad_parts(const fh_packed_attention& g) {
  const int64_t keys = grad_keys(g), tiles = (g.tokens + keys - 1) / keys * g.kv_heads, cus = device_cu_count();
  // rows of a sequence four times the mean length: the lengths themselves are on the device
  const int64_t longest = std::min(g.tokens, 4 * g.tokens / std::max<int64_t>(g.batch, 1));
  const int64_t blocks = longest * (g.heads / g.kv_heads) / kGradRows;
  if (tiles >= 2 * cus || blocks <= kWholeBlocks) return 1;
  return std::min<int64_t>(keys == 64 ? std::max<int64_t>(3 * cus / tiles, 3) : std::max<int64_t>(cus / tiles, 2), 8);
}

}  // namespace
}  // namespace fh

using namespace fh;

extern "C" fh_status fh_attention_packed_fwd(const fh_packed_attention* g, const void* q, const void* k, const void* v,
                                             const int32_t* cu_seqlens, void* out, float* lse, void* stream) {
  const char* fn = "fh_attention_packed_fwd";
  if (fh_status st = check_packed(fn, g); st != FH_OK) return st;
  if (g->tokens == 0 || g->batch == 0) return FH_OK;
  if (!q || !k || !v || !out || !cu_seqlens) return fail(FH_INVALID_ARGUMENT, std::string(fn) + ": null pointer");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(FH_INVALID_ARGUMENT, std::string(fn) + ": q, k, v and out must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(cu_seqlens) | reinterpret_cast<uintptr_t>(lse)) % 4 != 0)
    return fail(FH_INVALID_ARGUMENT, std::string(fn) + ": cu_seqlens and lse must be 4-byte aligned");
  RowsArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.ldq = g->q_stride;
  a.ldo = g->out_stride;
  a.cu = cu_seqlens;
  a.tokens = static_cast<int>(g->tokens);
  a.batch = static_cast<int>(g->batch);
  a.heads = static_cast<int>(g->heads);
  a.kv_heads = static_cast<int>(g->kv_heads);
  a.dh = static_cast<int>(g->dh);
  a.group = make_divider(static_cast<uint32_t>(g->heads / g->kv_heads));
  a.causal = g->causal;
  a.scale = g->scale;
  a.splits = 1;
  a.k = k;
  a.v = v;
  a.ldk = g->k_stride;
  a.ldv = g->v_stride;
  constexpr int W = 4;
  const int share = key_shares(*g, false);
  a.slots = static_cast<int>(slots_for(*g, a.group.d, 32 * W / share));
  const dim3 grid(static_cast<uint32_t>(a.slots) * static_cast<uint32_t>(a.kv_heads));
  auto launch = [&]<typename T, int DH>() {
    if (share == 2)
      hipLaunchKernelGGL((attention_rows_kernel<T, DH, kDense, W, 2>), grid, dim3(W * 64), 0, static_cast<hipStream_t>(stream), a);
    else
      hipLaunchKernelGGL((attention_rows_kernel<T, DH, kDense, W, 1>), grid, dim3(W * 64), 0, static_cast<hipStream_t>(stream), a);
  };
  if (g->dtype == FH_BF16) {
    if (g->dh <= 64) launch.template operator()<bf16_t, 64>(); else launch.template operator()<bf16_t, 128>();
  } else {
    if (g->dh <= 64) launch.template operator()<f16_t, 64>(); else launch.template operator()<f16_t, 128>();
  }
  return launch_status("attention_rows_kernel launch");
}

extern "C" int64_t fh_attention_packed_grad_workspace(const fh_packed_attention* g) {
  if (check_packed("fh_attention_packed_grad_workspace", g) != FH_OK) return -1;
  const int64_t parts = grad_parts(*g);
  return delta_bytes(*g) + (parts > 1 ? parts * 2 * g->tokens * g->kv_heads * g->dh * 4 : 0);
}

extern "C" fh_status fh_attention_packed_grad(const fh_packed_attention* g, const void* q, const void* k, const void* v,
                                              const int32_t* cu_seqlens, const void* out, const float* lse, const void* dout,
                                              void* dq, void* dk, void* dv, void* workspace, int64_t workspace_bytes,
                                              void* stream) {
  const std::string fn = "fh_attention_packed_grad";
  if (fh_status st = check_packed(fn.c_str(), g); st != FH_OK) return st;
  if (g->tokens == 0 || g->batch == 0) return FH_OK;
  if (!q || !k || !v || !cu_seqlens || !out || !lse || !dout || !dq || !dk || !dv || !workspace)
    return fail(FH_INVALID_ARGUMENT, fn + ": null pointer");
  for (const void* p : {q, k, v, out, dout, static_cast<const void*>(dq), static_cast<const void*>(dk),
                        static_cast<const void*>(dv), static_cast<const void*>(workspace)})
    if (!aligned16(p)) return fail(FH_INVALID_ARGUMENT, fn + ": tensors and the workspace must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(cu_seqlens) | reinterpret_cast<uintptr_t>(lse)) % 4 != 0)
    return fail(FH_INVALID_ARGUMENT, fn + ": cu_seqlens and lse must be 4-byte aligned");
  if (workspace_bytes < g->tokens * g->heads * 4) return fail(FH_INVALID_ARGUMENT, fn + ": workspace too small");
  GradArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<const uint16_t*>(out);
  a.dout = static_cast<const uint16_t*>(dout);
  a.dq = static_cast<uint16_t*>(dq);
  a.dk = static_cast<uint16_t*>(dk);
  a.dv = static_cast<uint16_t*>(dv);
  a.lse = lse;
  a.delta = static_cast<float*>(workspace);
  a.tile_keys = static_cast<int>(grad_keys(*g));
  a.parts = workspace_bytes < fh_attention_packed_grad_workspace(g) ? 1 : static_cast<int>(grad_parts(*g));
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + delta_bytes(*g));
  a.cu = cu_seqlens;
  a.ldq = g->q_stride;
  a.ldk = g->k_stride;
  a.ldv = g->v_stride;
  a.ldo = g->out_stride;
  a.tokens = static_cast<int>(g->tokens);
  a.batch = static_cast<int>(g->batch);
  a.heads = static_cast<int>(g->heads);
  a.kv_heads = static_cast<int>(g->kv_heads);
  a.dh = static_cast<int>(g->dh);
  a.group = make_divider(static_cast<uint32_t>(g->heads / g->kv_heads));
  a.causal = g->causal;
  a.scale = g->scale;
  hipStream_t s = static_cast<hipStream_t>(stream);
  constexpr int W = 4;
  auto launch = [&]<typename T, int DH>() {
    const int share = key_shares(*g, true);
    a.slots = static_cast<int>(slots_for(*g, a.group.d, 32 * W / share));
    const dim3 tiles(static_cast<uint32_t>(a.slots) * static_cast<uint32_t>(a.kv_heads));
    if (share == 2)
      hipLaunchKernelGGL((attention_dq_kernel<T, DH, W, 2>), tiles, dim3(W * 64), 0, s, a);
    else
      hipLaunchKernelGGL((attention_dq_kernel<T, DH, W, 1>), tiles, dim3(W * 64), 0, s, a);
    if (fh_status st = launch_status("attention_dq_kernel launch"); st != FH_OK) return st;
    a.slots = static_cast<int>(slots_for(*g, 1, a.tile_keys));
    const dim3 grid(static_cast<uint32_t>(a.slots) * static_cast<uint32_t>(a.kv_heads) * static_cast<uint32_t>(a.parts));
    if constexpr (DH == 64) {
      if (a.tile_keys == 64) hipLaunchKernelGGL((attention_dkv_kernel<T, DH, 2>), grid, dim3(256), 0, s, a);
    }
    if (a.tile_keys == 128) hipLaunchKernelGGL((attention_dkv_kernel<T, DH, 4>), grid, dim3(512), 0, s, a);
    if (fh_status st = launch_status("attention_dkv_kernel launch"); st != FH_OK || a.parts == 1) return st;
    const int64_t slices = (2 * g->kv_heads * g->dh + kJoin * 256 - 1) / (kJoin * 256);
    hipLaunchKernelGGL((attention_dkv_join_kernel<T>), dim3(static_cast<uint32_t>((g->tokens * slices + 3) / 4)), dim3(256), 0, s, a);
    return launch_status("attention_dkv_join_kernel launch");
  };
  if (g->dtype == FH_BF16)
    return g->dh <= 64 ? launch.template operator()<bf16_t, 64>() : launch.template operator()<bf16_t, 128>();
  return g->dh <= 64 ? launch.template operator()<f16_t, 64>() : launch.template operator()<f16_t, 128>();
}

extern "C" fh_status fh_packed_clear(const int32_t* cu_seqlens, int64_t batch, void* x, int64_t rows, int64_t row_bytes, void* stream) {
  const std::string fn = "fh_packed_clear";
  if (batch < 0 || batch > 0x3fffffff || rows < 0 || rows > 4 * kMaxBlocks || row_bytes < 0 || row_bytes % 16 != 0)
    return fail(FH_INVALID_ARGUMENT, fn + ": bad batch, rows or row_bytes");
  if (rows == 0 || row_bytes == 0) return FH_OK;
  if (!cu_seqlens || !x || !aligned16(x) || reinterpret_cast<uintptr_t>(cu_seqlens) % 4 != 0)
    return fail(FH_INVALID_ARGUMENT, fn + ": null or unaligned pointer");
  hipLaunchKernelGGL(packed_clear_kernel, dim3(static_cast<uint32_t>((rows + 3) / 4)), dim3(256), 0, static_cast<hipStream_t>(stream),
                     cu_seqlens, static_cast<int>(batch), static_cast<uint4*>(x), static_cast<int>(rows), row_bytes / 16);
  return launch_status("packed_clear_kernel launch");
}
