// Host checks of a paged cache's descriptor, shared by the kernels that write, read and attend over it.
#pragma once

#include <cstdint>
#include <string>

#include "fh_common.h"

namespace fh {

inline int page_shift(int64_t page_size) {
  int s = 0;
  while ((int64_t{1} << s) < page_size) ++s;
  return s;
}

inline fh_status check_paged_cache(const std::string& fn, const fh_paged_cache* c) {
  if (c == nullptr) return fail(FH_INVALID_ARGUMENT, fn + ": null descriptor");
  if (c->dtype != FH_BF16 && c->dtype != FH_F16) return fail(FH_UNIMPLEMENTED, fn + ": needs bf16 or f16");
  if (c->cache_dtype != c->dtype && c->cache_dtype != FH_E4M3)
    return fail(FH_UNIMPLEMENTED, fn + ": the cache holds the tensors' type or e4m3");
  if (c->dh < 8 || c->dh > 128 || c->dh % 8 != 0) return fail(FH_UNIMPLEMENTED, fn + ": head dim must be a multiple of 8 up to 128");
  if (c->page_size < 1 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)) != 0)
    return fail(FH_UNIMPLEMENTED, fn + ": page size must be a power of two up to 65536");
  if (c->kv_heads < 1 || c->kv_heads > 65535 || c->batch < 0 || c->batch > 0x3fffffff || c->pages < 0 || c->pages > 0x7fffffff ||
      c->table_stride < 0 || c->table_stride > 0x7fff0000 / c->page_size)  // (positions and a few blocks more fit 32 bits)
    return fail(FH_INVALID_ARGUMENT, fn + ": bad kv_heads, batch, pages or table_stride");
  if (c->batch == 0) return FH_OK;
  if (c->kv_lens == nullptr || (c->table_stride > 0 && c->block_table == nullptr) || (c->pages > 0 && (!c->k || !c->v)))
    return fail(FH_INVALID_ARGUMENT, fn + ": null pointer in the descriptor");
  if (c->pages > 0 && c->cache_dtype == FH_E4M3 && (!c->k_scale || !c->v_scale))
    return fail(FH_INVALID_ARGUMENT, fn + ": an e4m3 cache needs k_scale and v_scale");
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 != 0)
    return fail(FH_INVALID_ARGUMENT, fn + ": the cache must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(c->kv_lens) | reinterpret_cast<uintptr_t>(c->block_table)) % 4 != 0)
    return fail(FH_INVALID_ARGUMENT, fn + ": block_table and kv_lens must be 4-byte aligned");
  return FH_OK;
}

}  // namespace fh
