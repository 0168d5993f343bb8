// Attention of new tokens over a paged cache (fh_attention_paged), in two forms chosen by the rows that a key head has to serve at
// once (new tokens times the group's heads):
//   up to 32, decoding steps: attention_keys_kernel. Tiles of 16 rows, and the keys are shared out among the waves of the
//     workgroup. Nothing but the cache's bytes counts: every wave keeps one or two blocks of 32 keys and values on their way in
//     registers while it uses another from LDS of its own, so no wave ever waits for another. (With tiles of 32 rows, mostly empty, and one
//     block on its way, 64 sequences' step over an e4m3 cache of 550 MB took 165 us, bound by the waits for memory.)
//     Measured, 32 heads over 8, 128 dims: that step 142 us (3.9 TB/s), one new token over 32768 keys of 16 bits 35.5 us (26 and 5.3
//     for the join; 134 MB).
//   more, chunks: attention_rows_kernel of fh_attention_rows.h, whose waves share the keys and own 32 rows each. 2025 new tokens
//     of 7 sequences over up to 8,192 keys: 232 to 236 us, 580 TFLOP/s; in one part per sequence 456 us, the longest sequence's tiles alone.
// The form is the call's, by its longest sequence. 60 sequences' one token beside a chunk of 512 over 2,048 keys, contexts of 127 to 8,191:
// 180 us over an e4m3 cache (apart, in two calls, 73 + 59), 173 over 16 bits (124 + 54).
// Both cut long contexts into parts (keys z * part_keys ..) where the tiles alone would leave CUs idle; attention_join_kernel sums the
// parts, weighted by their log-sum-exps, in their order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "fh_attention_rows.h"
#include "fh_paged_cache.h"

namespace fh {
namespace {

using namespace attn;

constexpr int kWaves = 4;

// Keys [kbegin, kend) in blocks of 32, block i to wave i % kWaves; then the waves' sums are joined through LDS. Products are
// 16x16x32: scores transposed (a lane holds 8 keys of one row), probabilities in place as the operand of V^T P^T.
template <typename T, int DH, int SRC>
__global__ __launch_bounds__(kWaves * 64, 2) void attention_keys_kernel(const RowsArgs a) {
  constexpr int BK = 32, BYTES = BK * DH * 2, PITCH = DH + 4, ROWS = 16;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[kWaves * 2 * BYTES];
  __shared__ float stats[2][kWaves][ROWS];
  __shared__ NotFinite<T, DH> bad;
  static_assert(ROWS * PITCH * 4 <= 2 * BYTES, "a wave's room holds its fp32 sums");

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kv_head = static_cast<int>(blockIdx.x) % a.kv_heads;
  const int slot = static_cast<int>(blockIdx.x) / a.kv_heads;
  RowTile tile;
  if (!tile.find<SRC>(a, slot, 4)) return;
  int kbegin = 0, kend = tile.limit(a, tile.tile0 + ROWS - 1) + 1;
  bool whole;
  if (!tile.part(a, static_cast<int>(blockIdx.z), kbegin, kend, whole)) return;

  const int group = static_cast<int>(a.group.d);
  const int lim = tile.limit(a, tile.tile0 + l16), lim_low = tile.limit(a, tile.tile0);
  const bool uneven = lim_low != tile.limit(a, tile.tile0 + ROWS - 1);  // rows of several tokens
  if (uneven) {
    bad.clear(tid);
    __syncthreads();
  }

  unsigned char* mine = lds + wave * 2 * BYTES;
  // blocks on their way: 16 KB a wave either way (two of 128 16-bit values would spill)
  constexpr int DEPTH = SRC == kE4m3 || DH == 64 ? 2 : 1;
  constexpr int STEP = DEPTH * kWaves * BK;  // between a stage's blocks
  KvStage<T, DH, SRC, 64, BK> stages[DEPTH];
  const int kfirst = kbegin + wave * BK;
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) stages[i].start(a, tile.seq.begin, tile.table, kv_head, kfirst + i * kWaves * BK, kend, lane);
  u32x4_t qf[DH / 32];
  {
    const int r = min(tile.tile0 + l16, tile.rows - 1), token = divide(r, a.group), head = kv_head * group + r - token * group;
    const uint16_t* qr = a.q + (tile.seq.begin + token) * a.ldq + static_cast<int64_t>(head) * a.dh;
#pragma unroll
    for (int s = 0; s < DH / 32; ++s) qf[s] = load_chunk(qr + 32 * s + 8 * g, 32 * s + 8 * g < a.dh);
  }
  const float c = a.scale * kLog2e;
  float m = -__builtin_inff(), l = 0.0f;  // l: the lane's share
  f32x4_t o[DH / 16];
#pragma unroll
  for (int dt = 0; dt < DH / 16; ++dt) o[dt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const TileReader16<DH> tiles(mine, lane);

  auto use = [&](int kb, uint64_t there) {  // the block in LDS
    f32x4_t s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < DH / 32; ++i) mfma16x<T>(tiles.rows(16 * t, i), qf[i], s[t]);
    }
    if (kb + BK - 1 > lim_low || there != ~uint64_t{0}) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int u = 16 * t + 4 * g + x;
          s[t][x] = kb + u <= lim && ((there >> u) & 1) != 0 ? s[t][x] : -__builtin_inff();
        }
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int x = 0; x < 4; x += 2) top = max3(top, s[t][x], s[t][x + 1]);
    top = quarter_max(top) * c;
    if (__any(top > m + 8.0f)) {
      const float next = fmaxf(m, top);
      const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < DH / 16; ++dt)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[dt][x] *= f;
    }
    const float ms = m == -__builtin_inff() ? 0.0f : m;
    u32x4_t p;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[t][x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][x], c, -ms));
        l += s[t][x];
      }
      p[2 * t] = narrow2<T>(s[t][0], s[t][1]);
      p[2 * t + 1] = narrow2<T>(s[t][2], s[t][3]);
    }
#pragma unroll
    for (int dt = 0; dt < DH / 16; ++dt) mfma16x<T>(tiles.columns(BYTES, dt), p, o[dt]);
  };

  settle();
#pragma unroll
  for (int i = 0; i < DEPTH; ++i)
    if (kfirst + i * kWaves * BK < kend)
      stages[i].template load<STEP>(a, tile.table, kv_head, kfirst + i * kWaves * BK, kend, lane);
  for (int kb = kfirst; kb < kend; kb += STEP) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      const int at = kb + i * kWaves * BK;
      if (at < kend) {
        stages[i].store(mine, mine + BYTES, lane);
        if (uneven && at + BK - 1 > lim_low)
          stages[i].scrub_values(mine + BYTES, lane, [&](int row, int d, uint32_t bits) { bad.note(at + row, d, bits); });
        hand_over();
        const uint64_t there = stages[i].there;
        if (at + STEP < kend) stages[i].template load<STEP>(a, tile.table, kv_head, at + STEP, kend, lane);
        use(at, there);
        hand_over();
      }
    }
  }

  // every wave's maximum and sum per row, and its accumulators at the common scale
  const float sum = quarter_sum(l);
  if (g == 0) {
    stats[0][wave][l16] = m;
    stats[1][wave][l16] = sum;
  }
  __syncthreads();
  float top = stats[0][0][l16];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, stats[0][w][l16]);
  const float f = __builtin_amdgcn_exp2f(m - (top == -__builtin_inff() ? 0.0f : top));
  float* room = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int dt = 0; dt < DH / 16; ++dt)
    *reinterpret_cast<float4*>(room + l16 * PITCH + 16 * dt + 4 * g) =
        make_float4(o[dt][0] * f, o[dt][1] * f, o[dt][2] * f, o[dt][3] * f);
  __syncthreads();

  // 16 threads per row, DH / 16 values each
  const int row = tid >> 4, d = (tid & 15) * (DH / 16), r = tile.tile0 + row;
  float high = stats[0][0][row], total = 0.0f;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) high = fmaxf(high, stats[0][w][row]);
  const float ref = high == -__builtin_inff() ? 0.0f : high;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) total += stats[1][w][row] * __builtin_amdgcn_exp2f(stats[0][w][row] - ref);
  float inv = 1.0f / total, lse2 = ref + __log2f(total);
  if (__any(total == 0.0f)) {
    const bool sees = tile.template sees<SRC>(a, kbegin, kend, tile.limit(a, r));
    if (total == 0.0f) weigh_nothing(sees, whole, inv, lse2);
  }
  if (r >= tile.rows) return;
  const int token = divide(r, a.group);
  const int64_t trow = tile.seq.begin + token, head = kv_head * group + r - token * group;
  const int64_t part_row = (static_cast<int64_t>(blockIdx.z) * a.tokens + trow) * a.heads + head;
  if (!whole && (tid & 15) == 0) a.part_lse[part_row] = lse2;
#pragma unroll
  for (int i = 0; i < DH / 64; ++i) {  // 4 values at a time
    const int at = d + 4 * i;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(lds + w * 2 * BYTES) + row * PITCH + at);
      y.x += v.x;
      y.y += v.y;
      y.z += v.z;
      y.w += v.w;
    }
    if (uneven && bad.any != 0) {
      const int seen = tile.limit(a, r);
      y.x += bad.gain(at, seen);
      y.y += bad.gain(at + 1, seen);
      y.z += bad.gain(at + 2, seen);
      y.w += bad.gain(at + 3, seen);
    }
    if (at < a.dh) {
      if (!whole) {
        *reinterpret_cast<float4*>(a.part_out + part_row * a.dh + at) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
      } else {
        u32x2_t w;
        w[0] = narrow2<T>(y.x * inv, y.y * inv);
        w[1] = narrow2<T>(y.z * inv, y.w * inv);
        *reinterpret_cast<u32x2_t*>(a.out + trow * a.ldo + head * a.dh + at) = w;
      }
    }
  }
}

// The parts' weighted sum: out = sum_z w_z out_z / sum_z w_z, w_z = 2^(lse_z - max lse). Half a wave holds a row (4 values a lane, head
// dims up to 128); WAVES waves share a (token, head)'s parts, part z to half-wave z % (2 WAVES). 4 waves where the parts are many:
// 128 parts of 32 rows took 12.3 us with one wave each, 8 loads deep, and the join is all that runs then.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void attention_join_kernel(const RowsArgs a) {
  constexpr int PER = 4 / WAVES, HALVES = 2 * WAVES;
  __shared__ float4 sums[WAVES > 1 ? WAVES : 1][32];
  __shared__ float weights[WAVES > 1 ? WAVES : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * PER + (WAVES > 1 ? 0 : wave);
  const int64_t rows = static_cast<int64_t>(a.tokens) * a.heads;
  if (row >= rows) return;
  const int token = static_cast<int>(row / a.heads);
  const int b = sequence_of(a.cu, a.batch, token);
  if (b < 0) return;
  const Span seq = sequence(a.cu, b, a.tokens);
  if (token < seq.begin || token >= seq.end) return;  // rows outside the sequences stay as they are
  const int64_t cap = a.table_stride << a.page_shift;
  int keys = max(a.kv_lens[b], 0);
  if (keys > cap) keys = static_cast<int>(cap);
  if (keys <= a.part_keys) return;  // written whole
  const int parts = min((keys - 1) / a.part_keys + 1, a.splits);

  const int lane = threadIdx.x & 63, half = lane >> 5, d = (lane & 31) * 4;
  float top = -__builtin_inff();
  for (int z = lane; z < parts; z += 64) top = fmaxf(top, a.part_lse[z * rows + row]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float ref = top == -__builtin_inff() ? 0.0f : top;
  float sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const int z0 = (WAVES > 1 ? 2 * wave : 0) + half;
#pragma unroll 8
  for (int z = z0; z < parts; z += HALVES) {
    const float w = __builtin_amdgcn_exp2f(a.part_lse[z * rows + row] - ref);
    float4 p = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (d < a.dh) p = *reinterpret_cast<const float4*>(a.part_out + (z * rows + row) * a.dh + d);
    sum += w;
    acc[0] += w * p.x;
    acc[1] += w * p.y;
    acc[2] += w * p.z;
    acc[3] += w * p.w;
  }
  sum = half_sum(sum);
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = half_sum(acc[j]);
  if constexpr (WAVES > 1) {
    if (half == 0) sums[wave][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    if (lane == 0) weights[wave] = sum;
    __syncthreads();
    if (wave != 0) return;
    sum = 0.0f;
    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float4 y = sums[w][lane & 31];
      t.x += y.x;
      t.y += y.y;
      t.z += y.z;
      t.w += y.w;
      sum += weights[w];
    }
    acc[0] = t.x;
    acc[1] = t.y;
    acc[2] = t.z;
    acc[3] = t.w;
  }
  const float inv = sum == 0.0f ? 0.0f : top == kNoScore ? __builtin_nanf("") : 1.0f / sum;
  if (half == 0 && d < a.dh) {
    u32x2_t w;
    w[0] = narrow2<T>(acc[0] * inv, acc[1] * inv);
    w[1] = narrow2<T>(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<u32x2_t*>(a.out + token * a.ldo + (row - static_cast<int64_t>(token) * a.heads) * a.dh + d) = w;
  }
}

// How a call is cut: the form, the tiles' slots, and the parts of the keys.
struct Plan {
  bool by_keys;
  int shares;  // chunks: waves that share 32 rows
  int64_t slots, splits, part_keys;
};

Plan plan(const fh_paged_cache& c, int64_t tokens, int64_t heads, int64_t max_new, int64_t max_keys) {
  const int64_t group = heads / c.kv_heads, cus = device_cu_count();
  max_new = std::min(max_new, tokens);
  max_keys = std::min(max_keys, c.table_stride * c.page_size);
  Plan p{};
  p.by_keys = max_new * group <= 32;
  // chunks with few tiles, as in the forward over packed rows: two waves share 32 rows
  auto tiles_of = [&](int64_t rows) {
    p.slots = tokens * group / rows + c.batch;
    return std::max<int64_t>(1, c.kv_heads * std::min(p.slots, c.batch * ((max_new * group + rows - 1) / rows)));
  };
  p.shares = p.by_keys || tiles_of(32 * kWaves) >= 2 * cus ? 1 : 2;
  const int64_t tiles = tiles_of(p.by_keys ? 16 : 32 * kWaves / p.shares);
  // Tiles that the expected lengths make, and enough parts for 6 (by keys) or 3 rounds of the workgroups that fit the chip, so that
  // sequences of different lengths even out; no part shorter than 8 blocks. (Two rounds by keys: the 64 sequences above 156 us
  // instead of 139, the longest parts start last.)
  const int64_t want = ((p.by_keys ? 12 : 6) * cus + tiles - 1) / tiles;
  const int64_t least = p.by_keys ? 256 : 512;
  const int64_t parts = std::max<int64_t>(1, std::min({want, max_keys / least, int64_t{128}}));
  p.part_keys = std::max(least, ((max_keys + parts - 1) / parts + kBlock - 1) / kBlock * kBlock);
  p.splits = parts;
  return p;
}

fh_status check_call(const std::string& fn, const fh_paged_cache* c, int64_t tokens, int64_t heads, int64_t max_new, int64_t max_keys) {
  if (fh_status st = check_paged_cache(fn, c); st != FH_OK) return st;
  if (tokens < 0 || max_new < 0 || max_keys < 0) return fail(FH_INVALID_ARGUMENT, fn + ": negative tokens, max_new or max_keys");
  if (heads < 1 || heads % c->kv_heads != 0) return fail(FH_INVALID_ARGUMENT, fn + ": heads must be a multiple of kv_heads");
  if (heads > 65535 || tokens > 0x7fffffff || (tokens + 256) * heads + c->batch * c->kv_heads > 0x7fffffff)
    return fail(FH_INVALID_ARGUMENT, fn + ": more than 2^31 rows (tokens x heads)");
  return FH_OK;
}

}  // namespace
}  // namespace fh

using namespace fh;

extern "C" int64_t fh_attention_paged_workspace(const fh_paged_cache* c, int64_t tokens, int64_t heads, int64_t max_new,
                                                int64_t max_keys) {
  if (check_call("fh_attention_paged_workspace", c, tokens, heads, max_new, max_keys) != FH_OK) return -1;
  const int64_t splits = plan(*c, tokens, heads, max_new, max_keys).splits;
  return splits > 1 ? splits * tokens * heads * (c->dh + 1) * 4 : 0;
}

extern "C" fh_status fh_attention_paged(const fh_paged_cache* c, const void* q, int64_t q_stride, void* out, int64_t out_stride,
                                        int64_t tokens, int64_t heads, const int32_t* cu_seqlens, float scale, int64_t max_new,
                                        int64_t max_keys, void* workspace, int64_t workspace_bytes, void* stream) {
  const std::string fn = "fh_attention_paged";
  if (fh_status st = check_call(fn, c, tokens, heads, max_new, max_keys); st != FH_OK) return st;
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(FH_INVALID_ARGUMENT, fn + ": scale must be positive and finite");
  if (tokens == 0 || c->batch == 0) return FH_OK;
  if (!q || !out || !cu_seqlens) return fail(FH_INVALID_ARGUMENT, fn + ": null pointer");
  if (!aligned16(q) || !aligned16(out)) return fail(FH_INVALID_ARGUMENT, fn + ": q and out must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(cu_seqlens) % 4 != 0) return fail(FH_INVALID_ARGUMENT, fn + ": cu_seqlens must be 4-byte aligned");
  if (q_stride < heads * c->dh || out_stride < heads * c->dh || (q_stride | out_stride) % 8 != 0)
    return fail(FH_INVALID_ARGUMENT, fn + ": row strides must be multiples of 8 elements, no shorter than a row");
  RowsArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.ldq = q_stride;
  a.ldo = out_stride;
  a.cu = cu_seqlens;
  a.tokens = static_cast<int>(tokens);
  a.batch = static_cast<int>(c->batch);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(c->kv_heads);
  a.dh = static_cast<int>(c->dh);
  a.group = make_divider(static_cast<uint32_t>(heads / c->kv_heads));
  a.causal = 1;
  a.scale = scale;
  a.k = c->k;
  a.v = c->v;
  a.k_scale = c->k_scale;
  a.v_scale = c->v_scale;
  a.table = c->block_table;
  a.table_stride = c->table_stride;
  a.kv_lens = c->kv_lens;
  a.pages = static_cast<int>(c->pages);
  a.page_shift = page_shift(c->page_size);
  const Plan p = plan(*c, tokens, heads, max_new, max_keys);
  if (p.slots * c->kv_heads > kMaxBlocks || (p.splits > 1 && tokens * heads > kMaxBlocks))
    return fail(FH_INVALID_ARGUMENT, fn + ": more rows than one launch takes");
  a.splits = static_cast<int>(p.splits);
  a.part_keys = static_cast<int>(std::min<int64_t>(p.part_keys, 0x7fffffff));
  a.slots = static_cast<int>(p.slots);
  if (a.splits > 1) {
    if (workspace_bytes < fh_attention_paged_workspace(c, tokens, heads, max_new, max_keys))
      return fail(FH_INVALID_ARGUMENT, fn + ": workspace too small");
    if (workspace == nullptr || !aligned16(workspace)) return fail(FH_INVALID_ARGUMENT, fn + ": the workspace must be 16-byte aligned");
    a.part_out = static_cast<float*>(workspace);
    a.part_lse = a.part_out + a.splits * tokens * heads * c->dh;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<uint32_t>(a.slots) * static_cast<uint32_t>(a.kv_heads), 1, static_cast<uint32_t>(a.splits));
  auto launch = [&]<typename T, int DH>() {
    if (p.by_keys && c->cache_dtype == FH_E4M3)
      hipLaunchKernelGGL((attention_keys_kernel<T, DH, kE4m3>), grid, dim3(kWaves * 64), 0, s, a);
    else if (p.by_keys)
      hipLaunchKernelGGL((attention_keys_kernel<T, DH, kPaged>), grid, dim3(kWaves * 64), 0, s, a);
    else if (c->cache_dtype == FH_E4M3 && p.shares == 2)
      hipLaunchKernelGGL((attention_rows_kernel<T, DH, kE4m3, kWaves, 2>), grid, dim3(kWaves * 64), 0, s, a);
    else if (c->cache_dtype == FH_E4M3)
      hipLaunchKernelGGL((attention_rows_kernel<T, DH, kE4m3, kWaves, 1>), grid, dim3(kWaves * 64), 0, s, a);
    else if (p.shares == 2)
      hipLaunchKernelGGL((attention_rows_kernel<T, DH, kPaged, kWaves, 2>), grid, dim3(kWaves * 64), 0, s, a);
    else
      hipLaunchKernelGGL((attention_rows_kernel<T, DH, kPaged, kWaves, 1>), grid, dim3(kWaves * 64), 0, s, a);
    if (fh_status st = launch_status("fh_attention_paged launch"); st != FH_OK || a.splits == 1) return st;
    const int64_t rows = tokens * heads;
    if (a.splits > 8)
      hipLaunchKernelGGL((attention_join_kernel<T, 4>), dim3(static_cast<uint32_t>(rows)), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((attention_join_kernel<T, 1>), dim3(static_cast<uint32_t>((rows + 3) / 4)), dim3(256), 0, s, a);
    return launch_status("attention_join_kernel launch");
  };
  if (c->dtype == FH_BF16)
    return c->dh <= 64 ? launch.template operator()<bf16_t, 64>() : launch.template operator()<bf16_t, 128>();
  return c->dh <= 64 ? launch.template operator()<f16_t, 64>() : launch.template operator()<f16_t, 128>();
}
