// Attention of new tokens over a paged cache (fh_attention_paged), in two forms chosen by the rows that a key head has to serve at
// once (new tokens times the group's heads):
//   up to 32, decoding steps: attention_keys_kernel. One tile of 32 rows, and the keys are shared out among the waves of the
//     workgroup. Nothing but the cache's bytes counts: every wave keeps a block of 32 keys and values on its way in registers
//     while it uses the last one from LDS of its own, so no wave ever waits for another.
//   more, chunks: attention_rows_kernel of fh_attention_rows.h, whose waves share the keys and own 32 rows each.
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

// Keys [kbegin, kend) in blocks of 32, block i to wave i % kWaves; then the waves' sums are joined through LDS.
template <typename T, int DH, int SRC>
__global__ __launch_bounds__(kWaves * 64, 2) void attention_keys_kernel(const RowsArgs a) {
  constexpr int BK = 32, BYTES = BK * DH * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[kWaves * 2 * BYTES];
  __shared__ float stats[2][kWaves][32];
  static_assert(2 * BYTES == 32 * DH * 4, "a wave's room holds its fp32 sums");

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kv_head = static_cast<int>(blockIdx.x) % a.kv_heads;
  const int slot = static_cast<int>(blockIdx.x) / a.kv_heads;
  RowTile tile;
  if (!tile.find<SRC>(a, slot, 5)) return;
  int kbegin = 0, kend = tile.limit(a, tile.tile0 + 31) + 1;
  bool whole;
  if (!tile.part(a, static_cast<int>(blockIdx.z), kbegin, kend, whole)) return;

  const int r = tile.tile0 + l32;
  const bool live = r < tile.rows;
  const int lim = tile.limit(a, r), lim_low = tile.limit(a, tile.tile0);
  const int token = divide(min(r, tile.rows - 1), a.group);
  const int group = static_cast<int>(a.group.d);
  const int head = kv_head * group + (min(r, tile.rows - 1) - token * group);
  const int64_t trow = tile.seq.begin + token;

  unsigned char* mine = lds + wave * 2 * BYTES;
  KvStage<T, DH, SRC, 64, BK> stage;
  const int kfirst = kbegin + wave * BK;
  stage.start(a, tile.seq.begin, tile.table, kv_head, kfirst, kend, lane);
  u32x4_t qf[DH / 16];
  {
    const uint16_t* qr = a.q + trow * a.ldq + static_cast<int64_t>(head) * a.dh;
#pragma unroll
    for (int s = 0; s < DH / 16; ++s) qf[s] = load_chunk(qr + 16 * s + 8 * hi, live && 16 * s + 8 * hi < a.dh);
  }
  const float c = a.scale * kLog2e;
  RowState<T, DH> state;
  const TileReader<DH> tiles(mine, lane);
  constexpr int STEP = kWaves * BK;
  if (kfirst < kend) {
    settle();
    stage.template load<STEP>(a, tile.table, kv_head, kfirst, kend, lane);
    for (int kb = kfirst; kb < kend; kb += STEP) {
      stage.store(mine, mine + BYTES, lane);
      const uint64_t there = stage.there;
      if (kb + STEP < kend) stage.template load<STEP>(a, tile.table, kv_head, kb + STEP, kend, lane);
      state.template block<1>(tiles, tiles.at(BYTES), qf, c, kb, kb + BK - 1 > lim_low || there != ~uint64_t{0}, lim, there, hi);
    }
  }

  // every wave's maximum and sum, then its accumulators at the common scale: wave w sums the rows' d in [w DH / 4, (w + 1) DH / 4)
  const float sum = half_sum(state.l);
  if (hi == 0) {
    stats[0][wave][l32] = state.m;
    stats[1][wave][l32] = sum;
  }
  __syncthreads();
  float top = stats[0][0][l32], total = 0.0f;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, stats[0][w][l32]);
  const float ref = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) total += stats[1][w][l32] * __builtin_amdgcn_exp2f(stats[0][w][l32] - ref);
  const float f = __builtin_amdgcn_exp2f(state.m - ref);
  float* room = reinterpret_cast<float*>(mine);  // [DH][32]: the rows of the transposed result, a lane per row
#pragma unroll
  for (int dt = 0; dt < DH / 32; ++dt)
#pragma unroll
    for (int x = 0; x < 16; ++x) room[(32 * dt + result_row(x, hi)) * 32 + l32] = state.o[dt][x] * f;
  __syncthreads();
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int64_t part_row = (static_cast<int64_t>(blockIdx.z) * a.tokens + trow) * a.heads + head;
  if (live && !whole && wave == 0 && hi == 0)
    a.part_lse[part_row] = total == 0.0f ? -__builtin_inff() : ref + __log2f(total);
  const float* all = reinterpret_cast<const float*>(lds);
#pragma unroll
  for (int i = 0; i < DH / 32; ++i) {  // 4 values a lane and step
    const int d = wave * (DH / 4) + 8 * i + 4 * hi;
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) v += all[w * (DH * 32) + (d + j) * 32 + l32];
      y[j] = v * inv;
    }
    if (live && d < a.dh) {
      if (!whole) {
        *reinterpret_cast<float4*>(a.part_out + part_row * a.dh + d) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
        u32x2_t w;
        w[0] = store2<T>(y[0], y[1]);
        w[1] = store2<T>(y[2], y[3]);
        *reinterpret_cast<u32x2_t*>(a.out + trow * a.ldo + static_cast<int64_t>(head) * a.dh + d) = w;
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
  const int parts = min((keys + a.part_keys - 1) / a.part_keys, a.splits);

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
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  if (half == 0 && d < a.dh) {
    u32x2_t w;
    w[0] = store2<T>(acc[0] * inv, acc[1] * inv);
    w[1] = store2<T>(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<u32x2_t*>(a.out + token * a.ldo + (row - static_cast<int64_t>(token) * a.heads) * a.dh + d) = w;
  }
}

// How a call is cut: the form, the tiles' slots, and the parts of the keys.
struct Plan {
  bool by_keys;
  int64_t slots, splits, part_keys;
};

Plan plan(const fh_paged_cache& c, int64_t tokens, int64_t heads, int64_t max_new, int64_t max_keys) {
  const int64_t group = heads / c.kv_heads, cus = device_cu_count();
  max_new = std::min(max_new, tokens);
  max_keys = std::min(max_keys, c.table_stride * c.page_size);
  Plan p{};
  p.by_keys = max_new * group <= 32;
  const int64_t rows = p.by_keys ? 32 : 32 * kWaves;
  p.slots = tokens * group / rows + c.batch;
  // Tiles that the expected lengths make, and enough parts for 4 (by keys; 2 fit a CU) or 3 rounds of workgroups, so that sequences
  // of different lengths even out; no part shorter than 8 (4) blocks.
  const int64_t tiles = std::max<int64_t>(1, c.kv_heads * std::min(p.slots, c.batch * ((max_new * group + rows - 1) / rows)));
  const int64_t want = ((p.by_keys ? 4 : 6) * cus + tiles - 1) / tiles;
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
    else if (c->cache_dtype == FH_E4M3)
      hipLaunchKernelGGL((attention_rows_kernel<T, DH, kE4m3, kWaves>), grid, dim3(kWaves * 64), 0, s, a);
    else
      hipLaunchKernelGGL((attention_rows_kernel<T, DH, kPaged, kWaves>), grid, dim3(kWaves * 64), 0, s, a);
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
