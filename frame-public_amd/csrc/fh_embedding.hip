// Token embedding (fh_embedding_fwd) and the gradient of its table (fh_embedding_grad).
//
// Forward: out[t] = scale * table[ids[t]], a copy bound by memory: a wave per 4 KB of a row, 16 bytes per lane and access.
//
// Gradient: dtable[v] = base[v] + scale * sum_{t: ids[t] = v} dout[t]. The tokens are sorted by id (stable, so a sum's order is the
// tokens'), and the sorted list is cut into chunks of kChunk tokens whatever the ids are, so that frequent and rare ids are the same
// work: a wave sums the rows of a chunk id by id, ids that lie within a chunk are finished there, the rest leave fp32 parts that a
// join adds in their order. No atomics on floats: every sum has one order. Rows that no token names are zeros or base's, written
// by copies that the sort runs beside.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "fh_common.h"

namespace fh {
namespace {

typedef unsigned int u4_t __attribute__((ext_vector_type(4)));
// global memory takes 16-byte accesses at element alignment
typedef u4_t u4_any __attribute__((aligned(2)));

constexpr int kRowVectors = 4;  // 16-byte vectors of a row per lane (forward)
constexpr int kChunk = 16;      // sorted tokens that one wave sums

template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(typename Io<T>::storage));

// V consecutive elements at p, or the first n of them (rows shorter than a vector).
template <typename T, int V>
__device__ __forceinline__ void load_elems(const typename Io<T>::storage* p, int n, float (&v)[V]) {
  if (n >= V) {
    const u4_t w = *reinterpret_cast<const u4_any*>(p);
    unpack_vec<T>(uint4{w[0], w[1], w[2], w[3]}, v);
  } else {
#pragma unroll
    for (int x = 0; x < V; ++x) v[x] = x < n ? Io<T>::load(p[x]) : 0.0f;
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_elems(typename Io<T>::storage* p, int n, const float (&v)[V]) {
  if (n >= V) {
    const uint4 w = pack_vec<T>(v);
    *reinterpret_cast<u4_any*>(p) = u4_t{w.x, w.y, w.z, w.w};
  } else {
#pragma unroll
    for (int x = 0; x < V; ++x)
      if (x < n) p[x] = Io<T>::store(v[x]);
  }
}

struct EmbedArgs {
  const void* table;
  const void* in;  // dout
  const void* base;
  void* out;  // or dtable
  const int32_t* ids;
  int64_t ld;
  int tokens, vocab, dim;
  uint32_t blocks;  // of columns that one wave holds, in a row
  float scale;
  // gradient: the tokens sorted by id, and the parts of ids that cross chunks [chunks][2][dim]
  uint32_t* keys;
  uint32_t* order;
  float* part;
  int chunks;
};

template <typename T>
__global__ __launch_bounds__(256) void embedding_kernel(const EmbedArgs a) {
  using S = typename Io<T>::storage;
  constexpr int V = kVec<T>;
  const int lane = threadIdx.x & 63;
  const uint32_t work = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int token = static_cast<int>(work / a.blocks), block = static_cast<int>(work % a.blocks);
  if (token >= a.tokens) return;
  const int id = a.ids[token];
  const bool named = id >= 0 && id < a.vocab;
  const S* row = static_cast<const S*>(a.table) + static_cast<int64_t>(named ? id : 0) * a.dim;
  S* out = static_cast<S*>(a.out) + token * a.ld;
  float v[kRowVectors][V];
#pragma unroll
  for (int i = 0; i < kRowVectors; ++i) {
    const int c = ((block * kRowVectors + i) * 64 + lane) * V;
    if (c < a.dim && named) load_elems<T, V>(row + c, a.dim - c, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kRowVectors; ++i) {
    const int c = ((block * kRowVectors + i) * 64 + lane) * V;
    if (c >= a.dim) continue;
#pragma unroll
    for (int x = 0; x < V; ++x) v[i][x] = named ? v[i][x] * a.scale : 0.0f;
    store_elems<T, V>(out + c, a.dim - c, v[i]);
  }
}

// ---- sorting the tokens by id: least significant digits first, stable ----

constexpr int kSortThreads = 256, kSortItems = 8, kSortTile = kSortThreads * kSortItems, kSortWaves = kSortThreads / 64;
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;

struct SortArgs {
  const int32_t* ids;        // the first pass reads the ids; those outside the vocabulary sort behind all others, as `vocab`
  const uint32_t* keys_in;   // later ones what the pass before left
  const uint32_t* order_in;
  uint32_t* keys_out;
  uint32_t* order_out;
  uint32_t* counts;  // [bins][tiles], then where each begins
  int tokens, vocab, tiles, shift, bits;
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, int i) {
  if (a.keys_in != nullptr) return a.keys_in[i];
  const int id = a.ids[i];
  return static_cast<uint32_t>(id >= 0 && id < a.vocab ? id : a.vocab);
}

// Lanes of the wave that hold the same digit as this one (`there`: lanes that hold one at all).
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, uint64_t there) {
  uint64_t m = there;
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot((digit >> b) & 1);
    m &= (digit >> b) & 1 ? set : ~set;
  }
  return m;
}

// LDS changes hands between the lanes of one wave, whose accesses run in their order: the compiler is told not to move them across.
__device__ __forceinline__ void hand_over() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// SCATTER false: how many tokens of the tile have each digit. true: each token to its place.
template <bool SCATTER>
__global__ __launch_bounds__(kSortThreads) void sort_tile_kernel(const SortArgs a) {
  __shared__ uint32_t bins[kSortWaves][kMaxBins];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nbins = 1 << a.bits;
  for (int b = tid; b < kSortWaves * kMaxBins; b += kSortThreads) (&bins[0][0])[b] = 0;
  __syncthreads();
  const int first = static_cast<int>(blockIdx.x) * kSortTile + wave * (kSortTile / kSortWaves);
  uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int i = first + j * 64 + lane;
    key[j] = i < a.tokens ? sort_key(a, i) : 0;
  }
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const bool there = first + j * 64 + lane < a.tokens;
    const uint32_t digit = (key[j] >> a.shift) & (nbins - 1);
    const uint64_t same = same_digit(digit, a.bits, __ballot(there));
    const uint64_t below = same & ((1ull << lane) - 1);
    // the wave's lanes read a count before its first lane raises it, and the next item's behind that
    const uint32_t seen = bins[wave][digit];
    hand_over();
    if (there && below == 0) bins[wave][digit] = seen + __popcll(same);
    hand_over();
    rank[j] = seen + __popcll(below);
  }
  __syncthreads();
  for (int b = tid; b < nbins; b += kSortThreads) {
    uint32_t sum = 0;
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t n = bins[w][b];
      if (SCATTER) bins[w][b] = sum;
      sum += n;
    }
    if (!SCATTER) a.counts[b * a.tiles + blockIdx.x] = sum;
  }
  if constexpr (SCATTER) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      const int i = first + j * 64 + lane;
      if (i >= a.tokens) continue;
      const uint32_t digit = (key[j] >> a.shift) & (nbins - 1);
      const uint32_t to = a.counts[digit * a.tiles + blockIdx.x] + bins[wave][digit] + rank[j];
      a.keys_out[to] = key[j];
      a.order_out[to] = a.order_in != nullptr ? a.order_in[i] : static_cast<uint32_t>(i);
    }
  }
}

// counts -> where each digit of each tile begins, by one workgroup.
__global__ __launch_bounds__(1024) void sort_scan_kernel(uint32_t* counts, int n) {
  __shared__ uint32_t waves[16];
  __shared__ uint32_t carry;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) carry = 0;
  __syncthreads();
  for (int at = 0; at < n; at += 4096) {
    uint32_t v[4], sum = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = at + tid * 4 + x;
      v[x] = i < n ? counts[i] : 0;
      sum += v[x];
    }
    uint32_t scan = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t up = __shfl_up(scan, o, 64);
      if (lane >= o) scan += up;
    }
    if (lane == 63) waves[wave] = scan;
    __syncthreads();
    uint32_t before = carry;
    for (int w = 0; w < wave; ++w) before += waves[w];
    uint32_t run = before + scan - sum;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = at + tid * 4 + x;
      if (i < n) counts[i] = run;
      run += v[x];
    }
    __syncthreads();
    if (tid == 1023) carry = run;
    __syncthreads();
  }
}

// ---- dtable ----

// base, or zeros, in every row; the sums overwrite the named ones. In elements of one size or 16 bytes.
template <typename E>
__global__ __launch_bounds__(256) void embedding_base_kernel(const E* base, E* dtable, int64_t n) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) dtable[i] = base != nullptr ? base[i] : E{};
}

// dtable[id] columns c .. <- base + scale * sum
template <typename T>
__device__ __forceinline__ void finish_row(const EmbedArgs& a, uint32_t id, int c, float (&sum)[kVec<T>]) {
  using S = typename Io<T>::storage;
  constexpr int V = kVec<T>;
  const int64_t at = static_cast<int64_t>(id) * a.dim + c;
  float b[V];
#pragma unroll
  for (int x = 0; x < V; ++x) b[x] = 0.0f;
  if (a.base != nullptr) load_elems<T, V>(static_cast<const S*>(a.base) + at, a.dim - c, b);
#pragma unroll
  for (int x = 0; x < V; ++x) sum[x] = b[x] + a.scale * sum[x];
  store_elems<T, V>(static_cast<S*>(a.out) + at, a.dim - c, sum);
}

// A wave sums the rows of chunk `chunk` of the sorted tokens, 64 vectors of columns wide. An id's sum is finished if all of its tokens
// lie in the chunk; otherwise it is a part: [0] of an id that began in an earlier chunk, [1] of one that begins here.
template <typename T>
__global__ __launch_bounds__(256) void embedding_sum_kernel(const EmbedArgs a) {
  using S = typename Io<T>::storage;
  constexpr int V = kVec<T>;
  const int lane = threadIdx.x & 63;
  const uint32_t work = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int chunk = static_cast<int>(work / a.blocks);
  const int c = (static_cast<int>(work % a.blocks) * 64 + lane) * V;
  if (chunk >= a.chunks) return;
  const int first = chunk * kChunk, n = min(kChunk, a.tokens - first);
  // lane i: token i of the chunk; lane 16 the one behind the chunk, lane 17 the one before it
  const int at = lane == kChunk + 1 ? first - 1 : first + min(lane, kChunk);
  const uint32_t none = 0xffffffffu;
  const uint32_t mine = at >= 0 && at < a.tokens ? a.keys[at] : none;
  const uint32_t token = lane < n ? a.order[first + lane] : 0;
  const uint32_t before = __builtin_amdgcn_readlane(mine, kChunk + 1);
  float row[kChunk][V];
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    const uint32_t key = __builtin_amdgcn_readlane(mine, i);
    const int64_t t = __builtin_amdgcn_readlane(token, i);
    if (i < n && key < static_cast<uint32_t>(a.vocab) && c < a.dim)
      load_elems<T, V>(static_cast<const S*>(a.in) + t * a.ld + c, a.dim - c, row[i]);
  }
  float sum[V];
#pragma unroll
  for (int x = 0; x < V; ++x) sum[x] = 0.0f;
  bool began_here = __builtin_amdgcn_readlane(mine, 0) != before;
#pragma unroll
  for (int i = 0; i < kChunk; ++i) {
    const uint32_t key = __builtin_amdgcn_readlane(mine, i);
    if (i >= n || key >= static_cast<uint32_t>(a.vocab)) break;
#pragma unroll
    for (int x = 0; x < V; ++x) sum[x] += row[i][x];
    const bool ends = __builtin_amdgcn_readlane(mine, i + 1) != key;
    if (!ends && i + 1 < kChunk) continue;
    if (c < a.dim) {
      if (ends && began_here) {
        finish_row<T>(a, key, c, sum);
      } else {
        float* p = a.part + (static_cast<int64_t>(chunk) * 2 + (began_here ? 1 : 0)) * a.dim + c;
#pragma unroll
        for (int x = 0; x < V; ++x)
          if (c + x < a.dim) p[x] = sum[x];
      }
    }
#pragma unroll
    for (int x = 0; x < V; ++x) sum[x] = 0.0f;
    began_here = true;
  }
}

// The parts of an id that begins in chunk `chunk` and goes on behind it, in the chunks' order: each of the workgroup's four waves adds a
// run of them, the runs are added in LDS. Workgroups of other chunks end at once.
template <typename T>
__global__ __launch_bounds__(256) void embedding_join_kernel(const EmbedArgs a) {
  constexpr int V = kVec<T>;
  __shared__ float runs[4][64][V];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int chunk = static_cast<int>(blockIdx.x / a.blocks);
  const int c = static_cast<int>((blockIdx.x % a.blocks) * 64 + lane) * V;
  const int behind = (chunk + 1) * kChunk;  // the first token behind the chunk (there is one: the last chunk has no workgroup)
  const uint32_t key = a.keys[behind];
  if (key != a.keys[behind - 1] || key >= static_cast<uint32_t>(a.vocab)) return;
  const int first = chunk * kChunk;
  if (first > 0 && a.keys[first - 1] == key) return;  // began earlier
  int low = behind + 1, high = a.tokens;              // the first token with a greater id
  while (low < high) {
    const int mid = low + (high - low) / 2;
    if (a.keys[mid] > key) high = mid; else low = mid + 1;
  }
  const int parts = (low - 1) / kChunk - chunk + 1, each = (parts + 3) / 4;
  float sum[V];
#pragma unroll
  for (int x = 0; x < V; ++x) sum[x] = 0.0f;
  if (c < a.dim)
    for (int p = wave * each; p < min(parts, (wave + 1) * each); ++p) {
      const float* q = a.part + (static_cast<int64_t>(chunk + p) * 2 + (p == 0 ? 1 : 0)) * a.dim + c;
#pragma unroll
      for (int x = 0; x < V; ++x)
        if (c + x < a.dim) sum[x] += q[x];
    }
#pragma unroll
  for (int x = 0; x < V; ++x) runs[wave][lane][x] = sum[x];
  __syncthreads();
  if (wave != 0 || c >= a.dim) return;
#pragma unroll
  for (int x = 0; x < V; ++x) sum[x] = ((runs[0][lane][x] + runs[1][lane][x]) + runs[2][lane][x]) + runs[3][lane][x];
  finish_row<T>(a, key, c, sum);
}

constexpr int64_t kMaxGrid = 0x7fffffff;

fh_status check_embedding(const std::string& fn, const fh_token_embedding* g) {
  if (g == nullptr) return fail(FH_INVALID_ARGUMENT, fn + ": null geometry");
  if (!is_supported_float(g->dtype)) return fail(FH_UNIMPLEMENTED, fn + ": dtype must be f32, f16 or bf16");
  if (g->tokens < 0 || g->vocab < 1 || g->dim < 1) return fail(FH_INVALID_ARGUMENT, fn + ": bad tokens, vocab or dim");
  // the grids' and the sort's indexes are 32-bit
  if (g->vocab > 0x7ffffffe || g->dim > (1 << 20) || g->tokens > (1 << 28) || g->tokens * ((g->dim + 63) / 64) > kMaxGrid)
    return fail(FH_INVALID_ARGUMENT, fn + ": too large");
  if (g->row_stride < g->dim) return fail(FH_INVALID_ARGUMENT, fn + ": row_stride is less than dim");
  if (g->row_stride > (int64_t{1} << 40)) return fail(FH_INVALID_ARGUMENT, fn + ": too large");
  if (!std::isfinite(g->scale)) return fail(FH_INVALID_ARGUMENT, fn + ": scale must be finite");
  return FH_OK;
}

bool misaligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(bytes - 1)) != 0; }

// Workspace: keys and order twice (the passes of the sort go back and forth), the counts, the parts.
struct GradPlan {
  int64_t tiles, chunks, passes, bits;
  int64_t list, counts, part, bytes;  // bytes of one list, offsets
};
GradPlan grad_plan(const fh_token_embedding& g) {
  GradPlan p{};
  int64_t key_bits = 1;
  while ((int64_t{1} << key_bits) <= g.vocab) ++key_bits;  // keys are 0 .. vocab
  p.passes = (key_bits + kMaxBits - 1) / kMaxBits;
  p.bits = (key_bits + p.passes - 1) / p.passes;
  p.tiles = (g.tokens + kSortTile - 1) / kSortTile;
  p.chunks = (g.tokens + kChunk - 1) / kChunk;
  p.list = (g.tokens * 4 + 15) / 16 * 16;
  p.counts = 4 * p.list;
  p.part = p.counts + (p.tiles * kMaxBins * 4 + 15) / 16 * 16;
  p.bytes = p.part + p.chunks * 2 * g.dim * 4;
  return p;
}

}  // namespace
}  // namespace fh

using namespace fh;

extern "C" fh_status fh_embedding_fwd(const fh_token_embedding* g, const void* table, const int32_t* ids, void* out, void* stream) {
  const std::string fn = "fh_embedding_fwd";
  if (fh_status st = check_embedding(fn, g); st != FH_OK) return st;
  if (g->tokens == 0) return FH_OK;
  const int64_t esz = dtype_size(g->dtype);
  if (!table || !ids || !out) return fail(FH_INVALID_ARGUMENT, fn + ": null pointer");
  if (misaligned(table, esz) || misaligned(out, esz) || misaligned(ids, 4)) return fail(FH_INVALID_ARGUMENT, fn + ": unaligned pointer");
  EmbedArgs a{};
  a.table = table;
  a.out = out;
  a.ids = ids;
  a.ld = g->row_stride;
  a.tokens = static_cast<int>(g->tokens);
  a.vocab = static_cast<int>(g->vocab);
  a.dim = static_cast<int>(g->dim);
  a.scale = g->scale;
  const int64_t width = 64 * kRowVectors * 16 / esz;
  a.blocks = static_cast<uint32_t>((g->dim + width - 1) / width);
  const dim3 grid(static_cast<uint32_t>((g->tokens * a.blocks + 3) / 4));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (g->dtype == FH_F32) hipLaunchKernelGGL((embedding_kernel<float>), grid, dim3(256), 0, s, a);
  if (g->dtype == FH_F16) hipLaunchKernelGGL((embedding_kernel<f16_t>), grid, dim3(256), 0, s, a);
  if (g->dtype == FH_BF16) hipLaunchKernelGGL((embedding_kernel<bf16_t>), grid, dim3(256), 0, s, a);
  return launch_status("embedding_kernel launch");
}

extern "C" int64_t fh_embedding_grad_workspace(const fh_token_embedding* g) {
  if (check_embedding("fh_embedding_grad_workspace", g) != FH_OK) return -1;
  return grad_plan(*g).bytes;
}

extern "C" fh_status fh_embedding_grad(const fh_token_embedding* g, const void* dout, const int32_t* ids, const void* base,
                                       void* dtable, void* workspace, int64_t workspace_bytes, void* stream) {
  const std::string fn = "fh_embedding_grad";
  if (fh_status st = check_embedding(fn, g); st != FH_OK) return st;
  const int64_t esz = dtype_size(g->dtype);
  if (!dtable || (g->tokens > 0 && (!dout || !ids || !workspace))) return fail(FH_INVALID_ARGUMENT, fn + ": null pointer");
  if (misaligned(dtable, esz) || misaligned(base, esz) || misaligned(dout, esz) || misaligned(ids, 4))
    return fail(FH_INVALID_ARGUMENT, fn + ": unaligned pointer");
  if (misaligned(workspace, 16)) return fail(FH_INVALID_ARGUMENT, fn + ": the workspace must be 16-byte aligned");
  const GradPlan p = grad_plan(*g);
  if (workspace_bytes < p.bytes) return fail(FH_INVALID_ARGUMENT, fn + ": workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);

  if (base != dtable) {
    const int64_t bytes = g->vocab * g->dim * esz;
    const bool wide = bytes % 16 == 0 && !misaligned(base, 16) && !misaligned(dtable, 16);
    const int64_t n = wide ? bytes / 16 : bytes / esz;
    const dim3 grid(static_cast<uint32_t>(std::min<int64_t>((n + 255) / 256, 8 * device_cu_count())));
    if (wide)
      hipLaunchKernelGGL((embedding_base_kernel<uint4>), grid, dim3(256), 0, s, static_cast<const uint4*>(base), static_cast<uint4*>(dtable), n);
    else if (esz == 4)
      hipLaunchKernelGGL((embedding_base_kernel<uint32_t>), grid, dim3(256), 0, s, static_cast<const uint32_t*>(base), static_cast<uint32_t*>(dtable), n);
    else
      hipLaunchKernelGGL((embedding_base_kernel<uint16_t>), grid, dim3(256), 0, s, static_cast<const uint16_t*>(base), static_cast<uint16_t*>(dtable), n);
    if (fh_status st = launch_status("embedding_base_kernel launch"); st != FH_OK) return st;
  }
  if (g->tokens == 0) return FH_OK;

  char* ws = static_cast<char*>(workspace);
  auto list = [&](int i) { return reinterpret_cast<uint32_t*>(ws + i * p.list); };
  SortArgs sort{};
  sort.ids = ids;
  sort.counts = reinterpret_cast<uint32_t*>(ws + p.counts);
  sort.tokens = static_cast<int>(g->tokens);
  sort.vocab = static_cast<int>(g->vocab);
  sort.tiles = static_cast<int>(p.tiles);
  sort.bits = static_cast<int>(p.bits);
  for (int pass = 0; pass < p.passes; ++pass) {
    sort.shift = pass * sort.bits;
    sort.keys_out = list(2 * (pass & 1));
    sort.order_out = list(2 * (pass & 1) + 1);
    hipLaunchKernelGGL((sort_tile_kernel<false>), dim3(static_cast<uint32_t>(p.tiles)), dim3(kSortThreads), 0, s, sort);
    if (fh_status st = launch_status("sort_tile_kernel launch"); st != FH_OK) return st;
    hipLaunchKernelGGL(sort_scan_kernel, dim3(1), dim3(1024), 0, s, sort.counts, static_cast<int>(p.tiles << p.bits));
    if (fh_status st = launch_status("sort_scan_kernel launch"); st != FH_OK) return st;
    hipLaunchKernelGGL((sort_tile_kernel<true>), dim3(static_cast<uint32_t>(p.tiles)), dim3(kSortThreads), 0, s, sort);
    if (fh_status st = launch_status("sort_tile_kernel launch"); st != FH_OK) return st;
    sort.keys_in = sort.keys_out;
    sort.order_in = sort.order_out;
  }

  EmbedArgs a{};
  a.in = dout;
  a.base = base;
  a.out = dtable;
  a.ld = g->row_stride;
  a.tokens = static_cast<int>(g->tokens);
  a.vocab = static_cast<int>(g->vocab);
  a.dim = static_cast<int>(g->dim);
  a.scale = g->scale;
  a.keys = sort.keys_out;
  a.order = sort.order_out;
  a.part = reinterpret_cast<float*>(ws + p.part);
  a.chunks = static_cast<int>(p.chunks);
  const int64_t width = 64 * 16 / esz;
  a.blocks = static_cast<uint32_t>((g->dim + width - 1) / width);
  auto launch = [&]<typename T>() {
    hipLaunchKernelGGL((embedding_sum_kernel<T>), dim3(static_cast<uint32_t>((p.chunks * a.blocks + 3) / 4)), dim3(256), 0, s, a);
    if (fh_status st = launch_status("embedding_sum_kernel launch"); st != FH_OK || p.chunks == 1) return st;
    hipLaunchKernelGGL((embedding_join_kernel<T>), dim3(static_cast<uint32_t>((p.chunks - 1) * a.blocks)), dim3(256), 0, s, a);
    return launch_status("embedding_join_kernel launch");
  };
  if (g->dtype == FH_F32) return launch.template operator()<float>();
  return g->dtype == FH_F16 ? launch.template operator()<f16_t>() : launch.template operator()<bf16_t>();
}
