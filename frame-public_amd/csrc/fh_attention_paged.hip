// Attention of new tokens over a paged cache (fh_attention_paged): attention_rows_kernel of fh_attention_rows.h over pages. Few rows
// over long contexts leave most CUs without a workgroup, so the keys are cut into parts that a second launch joins.
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

int64_t tiles_of(const fh_paged_cache& c, int64_t tokens, int64_t heads) {
  return (tokens * (heads / c.kv_heads) / (32 * kWaves) + c.batch) * c.kv_heads;
}

// Parts of the keys: enough for two workgroups per CU, none shorter than 4 blocks of the longest context.
int64_t plan_splits(const fh_paged_cache& c, int64_t tokens, int64_t heads, int64_t max_new, int64_t max_keys) {
  const int64_t group = heads / c.kv_heads;
  const int64_t tiles = std::min(tiles_of(c, tokens, heads), c.batch * c.kv_heads * ((max_new * group + 32 * kWaves - 1) / (32 * kWaves)));
  const int64_t want = (2 * device_cu_count() + tiles - 1) / std::max<int64_t>(tiles, 1);
  const int64_t blocks = (max_keys + kBlock - 1) / kBlock;
  return std::max<int64_t>(1, std::min({want, blocks / 4, int64_t{128}}));
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
  const int64_t splits = plan_splits(*c, tokens, heads, max_new, max_keys);
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
  a.splits = static_cast<int>(plan_splits(*c, tokens, heads, max_new, max_keys));
  if (a.splits > 1) {
    if (workspace_bytes < fh_attention_paged_workspace(c, tokens, heads, max_new, max_keys))
      return fail(FH_INVALID_ARGUMENT, fn + ": workspace too small");
    if (workspace == nullptr || !aligned16(workspace)) return fail(FH_INVALID_ARGUMENT, fn + ": the workspace must be 16-byte aligned");
    a.part_out = static_cast<float*>(workspace);
    a.part_lse = a.part_out + a.splits * tokens * heads * c->dh;
  }
  a.slots = static_cast<int>(tiles_of(*c, tokens, heads) / c->kv_heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<uint32_t>(a.slots) * static_cast<uint32_t>(a.kv_heads), 1, static_cast<uint32_t>(a.splits));
  auto launch = [&]<typename T, int DH>() {
    if (c->cache_dtype == FH_E4M3)
      hipLaunchKernelGGL((attention_rows_kernel<T, DH, kE4m3, kWaves>), grid, dim3(kWaves * 64), 0, s, a);
    else
      hipLaunchKernelGGL((attention_rows_kernel<T, DH, kPaged, kWaves>), grid, dim3(kWaves * 64), 0, s, a);
    if (fh_status st = launch_status("attention_rows_kernel launch"); st != FH_OK || a.splits == 1) return st;
    const int64_t rows = tokens * heads;
    hipLaunchKernelGGL((attention_join_kernel<T>), dim3(static_cast<uint32_t>((rows + 3) / 4)), dim3(256), 0, s, a);
    return launch_status("attention_join_kernel launch");
  };
  if (c->dtype == FH_BF16)
    return c->dh <= 64 ? launch.template operator()<bf16_t, 64>() : launch.template operator()<bf16_t, 128>();
  return c->dh <= 64 ? launch.template operator()<f16_t, 64>() : launch.template operator()<f16_t, 128>();
}
