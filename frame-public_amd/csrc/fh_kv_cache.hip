// The paged key/value cache: fh_kv_cache_write puts new tokens' rows at their positions, fh_kv_cache_read brings rows back.
// e4m3: a row (one token, one head) is stored as e4m3 values and one E8M0 byte, its scale: the least power of two p >= 2^-126 with
// max|row| <= 448 p, and 1 for a row of zeros. A power of two costs the 3-bit fraction nothing against any other scale and is
// undone exactly: the cached value e4m3 * p is a bf16 value, so attention needs no further rounding of it. Values that are not
// finite become NaN, and the maximum is taken over the others.
// Both directions move 16 bytes of the tensors' side per lane, a row in DH / 8 lanes (8 or 16, power of two, for the maximum's
// shuffles); they are bound by memory, and by the launch for a step's few rows. Measured, 8 heads of 128: 65,532 cached rows read
// as bf16 84 us (404 MB, 4.8 TB/s; a copy reaches 5.13), 8,192 rows written 14.3 us (50 MB, 3.5 TB/s); one row in flight per
// thread and a lookup per row: 154 and 16.7 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "fh_attention_rows.h"
#include "fh_paged_cache.h"

namespace fh {
namespace {

using namespace attn;

struct CacheArgs {
  void* k;  // the cache
  void* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  uint16_t* xk;  // the packed rows
  uint16_t* xv;
  int64_t ldk, ldv;
  const int32_t* cu;
  const int32_t* table;
  const int32_t* kv_lens;
  int64_t table_stride;
  int tokens, batch, kv_heads, dh, pages, page_shift;
};

// The cache row of packed row `token` (its slot), or -1: outside the sequences, past the block table, a page that does not exist.
// New tokens stand at the end of their sequence (WRITE), rows that are read at its beginning.
template <bool WRITE>
__device__ __forceinline__ int64_t slot_of(const CacheArgs& a, int token, bool& in_sequence) {
  // the first sequence that ends after the token
  int lo = 0, hi = a.batch;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid + 1] > token) hi = mid; else lo = mid + 1;
  }
  in_sequence = lo < a.batch && a.cu[lo] <= token;
  if (!in_sequence) return -1;
  const Span seq = sequence(a.cu, lo, a.tokens);
  const int64_t cap = a.table_stride << a.page_shift;
  int64_t len = max(a.kv_lens[lo], 0);
  if (len > cap) len = cap;
  const int64_t position = token - seq.begin + (WRITE ? len - (seq.end - seq.begin) : 0);
  if (position < 0 || position >= len) return -1;
  const int page = a.table[lo * a.table_stride + (position >> a.page_shift)];
  if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages)) return -1;
  return (static_cast<int64_t>(page) << a.page_shift) + (position & ((1 << a.page_shift) - 1));
}

// Exponent byte of the least power of two p with top <= 448 p: 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t scale_byte(float top) {
  const uint32_t u = __float_as_uint(top);
  if (u == 0) return 127;
  const int e = static_cast<int>(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(max(e, 1));
}

// 8 values of T over 2^(byte - 127), to e4m3 (nearest even; the quotients lie within its range)
template <typename T>
__device__ __forceinline__ u32x2_t narrow_e4m3(const float (&v)[8], uint32_t byte) {
  const float inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte); byte 1 .. 247
  u32x2_t w{0, 0};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = v[4 * i + j] * inv;
    int p = 0;
    p = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], p, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], p, true);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (!(__builtin_fabsf(v[4 * i + j]) < __builtin_inff())) p = (p & ~(0xff << (8 * j))) | (0x7f << (8 * j));
    w[i] = static_cast<uint32_t>(p);
  }
  return w;
}

// A workgroup takes `per` tokens: their cache rows are looked up once, a thread each, then their rows (token, head) move LANES lanes
// a row, keys and values by the same thread, kUnroll rows of both in flight.
constexpr int kUnroll = 4, kMostTokens = 32;

template <typename T, int LANES, bool E4M3, bool WRITE>
__global__ __launch_bounds__(256) void kv_cache_kernel(const CacheArgs a, int per, Divider by_heads) {
  __shared__ int64_t slots[kMostTokens];
  __shared__ int owned[kMostTokens];
  const int t0 = static_cast<int>(blockIdx.x) * per;
  const int count = min(per, a.tokens - t0);
  if (static_cast<int>(threadIdx.x) < count) {
    bool in_sequence;
    slots[threadIdx.x] = slot_of<WRITE>(a, t0 + static_cast<int>(threadIdx.x), in_sequence);
    owned[threadIdx.x] = in_sequence;
  }
  __syncthreads();
  constexpr int ROWS = 256 / LANES;
  const int chunk = threadIdx.x % LANES;
  const bool inside = chunk * 8 < a.dh;
  const int rows = count * a.kv_heads;
  for (int r0 = static_cast<int>(threadIdx.x) / LANES; r0 < (rows + ROWS - 1) / ROWS * ROWS; r0 += kUnroll * ROWS) {
    bool there[kUnroll], mine[kUnroll];
    int64_t at[kUnroll], crow[kUnroll], xk[kUnroll], xv[kUnroll];
    u32x4_t w[kUnroll][2];
    u32x2_t c[kUnroll][2];
    uint32_t byte[kUnroll][2];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int r = min(r0 + u * ROWS, rows - 1), t = divide(r, by_heads), head = r - t * a.kv_heads;
      const bool row = r0 + u * ROWS < rows;
      mine[u] = row && inside && owned[t];
      there[u] = row && inside && slots[t] >= 0;
      crow[u] = slots[t] * a.kv_heads + head;
      at[u] = crow[u] * a.dh + chunk * 8;
      const int64_t col = static_cast<int64_t>(head) * a.dh + chunk * 8;
      xk[u] = (t0 + t) * a.ldk + col;
      xv[u] = (t0 + t) * a.ldv + col;
      if constexpr (WRITE) {
        w[u][0] = load_chunk(a.xk + xk[u], there[u]);
        w[u][1] = load_chunk(a.xv + xv[u], there[u]);
      } else if constexpr (E4M3) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          c[u][i] = u32x2_t{0, 0};
          byte[u][i] = 127;
          if (there[u]) {
            c[u][i] = *reinterpret_cast<const u32x2_t*>(static_cast<const uint8_t*>(i ? a.v : a.k) + at[u]);
            byte[u][i] = (i ? a.v_scale : a.k_scale)[crow[u]];
          }
        }
      } else {
        w[u][0] = load_chunk(static_cast<const uint16_t*>(a.k) + at[u], there[u]);
        w[u][1] = load_chunk(static_cast<const uint16_t*>(a.v) + at[u], there[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (!WRITE) {
          // positions without a cached row read as zeros
          if constexpr (E4M3) {
            w[u][i] = widen_e4m3<T>(c[u][i], __uint_as_float(byte[u][i] << 23));
            if (byte[u][i] >= kTopScale<T>) w[u][i] = below_infinity<T>(w[u][i]);
          }
          if (mine[u]) *reinterpret_cast<u32x4_t*>(i ? a.xv + xv[u] : a.xk + xk[u]) = w[u][i];
        } else if constexpr (!E4M3) {
          if (there[u]) *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(i ? a.v : a.k) + at[u]) = w[u][i];
        } else {
          float v[8];
          unpack_vec<T>(uint4{w[u][i][0], w[u][i][1], w[u][i][2], w[u][i][3]}, v);
          float top = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float s = __builtin_fabsf(v[j]);
            if (s < __builtin_inff()) top = fmaxf(top, s);
          }
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
          const uint32_t scale = scale_byte(top);
          if (there[u]) {
            *reinterpret_cast<u32x2_t*>(static_cast<uint8_t*>(i ? a.v : a.k) + at[u]) = narrow_e4m3<T>(v, scale);
            if (chunk == 0) (i ? a.v_scale : a.k_scale)[crow[u]] = static_cast<uint8_t>(scale);
          }
        }
      }
  }
}

template <bool WRITE>
fh_status run(const std::string& fn, const fh_paged_cache* c, void* k, int64_t k_stride, void* v, int64_t v_stride, int64_t tokens,
              const int32_t* cu_seqlens, void* stream) {
  if (fh_status st = check_paged_cache(fn, c); st != FH_OK) return st;
  if (tokens < 0 || tokens > 0x7fffffff) return fail(FH_INVALID_ARGUMENT, fn + ": bad tokens");
  if (tokens == 0 || c->batch == 0) return FH_OK;
  if (!k || !v || !cu_seqlens) return fail(FH_INVALID_ARGUMENT, fn + ": null pointer");
  if (!aligned16(k) || !aligned16(v)) return fail(FH_INVALID_ARGUMENT, fn + ": k and v must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(cu_seqlens) % 4 != 0) return fail(FH_INVALID_ARGUMENT, fn + ": cu_seqlens must be 4-byte aligned");
  if (k_stride < c->kv_heads * c->dh || v_stride < c->kv_heads * c->dh || (k_stride | v_stride) % 8 != 0)
    return fail(FH_INVALID_ARGUMENT, fn + ": row strides must be multiples of 8 elements, no shorter than a row");
  CacheArgs a{};
  a.k = c->k;
  a.v = c->v;
  a.k_scale = c->k_scale;
  a.v_scale = c->v_scale;
  a.xk = static_cast<uint16_t*>(k);
  a.xv = static_cast<uint16_t*>(v);
  a.ldk = k_stride;
  a.ldv = v_stride;
  a.cu = cu_seqlens;
  a.table = c->block_table;
  a.kv_lens = c->kv_lens;
  a.table_stride = c->table_stride;
  a.tokens = static_cast<int>(tokens);
  a.batch = static_cast<int>(c->batch);
  a.kv_heads = static_cast<int>(c->kv_heads);
  a.dh = static_cast<int>(c->dh);
  a.pages = static_cast<int>(c->pages);
  a.page_shift = page_shift(c->page_size);
  auto launch = [&]<typename T, int LANES, bool E4M3>() {
    // a few tokens per workgroup once every CU has several of them
    const int64_t per = std::min<int64_t>(kMostTokens, std::max<int64_t>(1, tokens / (4 * device_cu_count())));
    const int64_t blocks = (tokens + per - 1) / per;
    if (blocks > kMaxBlocks) return fail(FH_INVALID_ARGUMENT, fn + ": too many rows");
    hipLaunchKernelGGL((kv_cache_kernel<T, LANES, E4M3, WRITE>), dim3(static_cast<uint32_t>(blocks)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), a, static_cast<int>(per), make_divider(static_cast<uint32_t>(c->kv_heads)));
    return launch_status("kv_cache_kernel launch");
  };
  auto typed = [&]<typename T>() {
    if (c->cache_dtype == FH_E4M3)
      return c->dh <= 64 ? launch.template operator()<T, 8, true>() : launch.template operator()<T, 16, true>();
    return c->dh <= 64 ? launch.template operator()<T, 8, false>() : launch.template operator()<T, 16, false>();
  };
  return c->dtype == FH_BF16 ? typed.template operator()<bf16_t>() : typed.template operator()<f16_t>();
}

}  // namespace
}  // namespace fh

using namespace fh;

extern "C" fh_status fh_kv_cache_write(const fh_paged_cache* cache, const void* k, int64_t k_stride, const void* v,
                                       int64_t v_stride, int64_t tokens, const int32_t* cu_seqlens, void* stream) {
  return run<true>("fh_kv_cache_write", cache, const_cast<void*>(k), k_stride, const_cast<void*>(v), v_stride, tokens, cu_seqlens,
                   stream);
}

extern "C" fh_status fh_kv_cache_read(const fh_paged_cache* cache, void* k, int64_t k_stride, void* v, int64_t v_stride,
                                      int64_t tokens, const int32_t* cu_seqlens, void* stream) {
  return run<false>("fh_kv_cache_read", cache, k, k_stride, v, v_stride, tokens, cu_seqlens, stream);
}
