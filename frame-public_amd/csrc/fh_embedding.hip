// Token embedding (fh_embedding_fwd) and the gradient of its table (fh_embedding_grad).
//
// Forward: out[t] = scale * table[ids[t]], a copy bound by memory: a wave per 4 KB of a row, 16 bytes per lane and access.
//
// Gradient: dtable[v] = base[v] + scale * sum_{t: ids[t] = v} dout[t]. The tokens are sorted by id (stable, so a sum's order is the
// tokens'), and the sorted list is cut into chunks of 8 or 16 tokens whatever the ids are, so that the sums of frequent and rare ids are the
// same work: a wave sums the rows of a chunk id by id, ids that lie within a chunk are finished there, the rest leave fp32 parts that a
// join adds in their order, an id's by one workgroup per 64 vectors of columns (16 bytes each): the join's time grows with the most frequent id. No
// atomics on floats: every sum has one order. Rows that no token names are zeros or base's: all rows are
// written so beside the sort, in the launches that a few workgroups of it would leave the chip idle in, and the sums overwrite theirs.
// Few tokens need no sort: an id's first token looks for the others and sums them, in one launch.
//
// Measured: forward, 8,192 tokens of 131,072 x 4,096 bf16: 21.8 us, 5.1 TB/s; 64 tokens of 1,024: 6.7 (the call). Gradient: 32,768 tokens of
// 131,072 x 4,096 bf16: 283 to 306 us (sort and zeros 207, sums 57, join 16) for 0.24 GB that must be read and 1.07 written (194 at 6.3 and 6.9
// TB/s, the rates of reads and writes alone; named rows are written twice); 4,096 of 32,768 x 1,024 on a base 34 us (20, 8 and 6); 301 of 5,003 x
// 333 f32 7 us, about what any call takes. Tokens of a table of 32,768 x 1,024 bf16 in place, as frequent as words, half of them one id, all of them:
// 4,096 24, 41 and 56 us; 32,768 72, 135 and 201; 131,072 185, 431 and 699.
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

template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(typename Io<T>::storage));

// A vector of consecutive elements at p, or the first n of them (rows shorter than a vector) and zeros.
template <typename T>
__device__ __forceinline__ uint4 load_bits(const typename Io<T>::storage* p, int n) {
  if (n >= kVec<T>) {
    const u4_t w = *reinterpret_cast<const u4_any*>(p);
    return uint4{w[0], w[1], w[2], w[3]};
  }
  typename Io<T>::storage e[kVec<T>] = {};
#pragma unroll
  for (int x = 0; x < kVec<T>; ++x)
    if (x < n) e[x] = p[x];
  uint4 w;
  __builtin_memcpy(&w, e, 16);
  return w;
}
template <typename T, int V>
__device__ __forceinline__ void load_elems(const typename Io<T>::storage* p, int n, float (&v)[V]) {
  unpack_vec<T>(load_bits<T>(p, n), v);
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
  // gradient: the tokens sorted by id, and the parts of ids that cross chunks [chunks][2][part_ld], whole vectors
  uint32_t* keys;
  uint32_t* order;
  float* part;
  int chunks, part_ld;  // chunks of CHUNK tokens
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
// tokens that one workgroup sorts: 16,384 in 40 us, which base's writing hides; 32,768 in 140 (registers), where several workgroups take 55
constexpr int kSortAlone = 16 * 1024;
constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;

// What a launch of the sort writes beside it: base's values, or zeros, in a share of dtable. One store per thread, past the caches, which the
// sums want (131,072 x 4,096 bf16 and one token: 177 us; a loop over the table in as many threads as run at once 225, four stores per
// thread 218, through the caches 200 and 60 us more for the sums).
struct BaseArgs {
  const void* base;
  void* dtable;
  int64_t begin, end;  // in units of `size` bytes
  int size;            // 16, or the elements' own where something is not aligned to 16
};
template <typename E>
__device__ __forceinline__ void copy_base(const BaseArgs& a, int64_t at) {
  if (at < a.end) __builtin_nontemporal_store(a.base != nullptr ? static_cast<const E*>(a.base)[at] : E{}, static_cast<E*>(a.dtable) + at);
}
__device__ __forceinline__ void write_base(const BaseArgs& a, int group) {
  const int64_t at = a.begin + static_cast<int64_t>(group) * blockDim.x + threadIdx.x;
  if (a.size == 16) copy_base<u4_t>(a, at);
  else if (a.size == 4) copy_base<uint32_t>(a, at);
  else copy_base<uint16_t>(a, at);
}

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

// How many tokens of the tile have each digit (integers: the additions' order changes nothing).
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const SortArgs a, const BaseArgs base) {
  __shared__ uint32_t bins[kMaxBins];
  if (static_cast<int>(blockIdx.x) >= a.tiles) return write_base(base, static_cast<int>(blockIdx.x) - a.tiles);
  const int tid = threadIdx.x, nbins = 1 << a.bits, first = static_cast<int>(blockIdx.x) * kSortTile + tid;
  uint32_t key[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) key[j] = first + j * kSortThreads < a.tokens ? sort_key(a, first + j * kSortThreads) : 0;
  for (int b = tid; b < nbins; b += kSortThreads) bins[b] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j)
    if (first + j * kSortThreads < a.tokens) atomicAdd(&bins[(key[j] >> a.shift) & (nbins - 1)], 1u);
  __syncthreads();
  for (int b = tid; b < nbins; b += kSortThreads) a.counts[b * a.tiles + blockIdx.x] = bins[b];
}

// Each token of the tile to its place.
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(const SortArgs a, const BaseArgs base) {
  __shared__ uint32_t bins[kSortWaves][kMaxBins];
  if (static_cast<int>(blockIdx.x) >= a.tiles) return write_base(base, static_cast<int>(blockIdx.x) - a.tiles);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nbins = 1 << a.bits;
  const int first = static_cast<int>(blockIdx.x) * kSortTile + wave * (kSortTile / kSortWaves);
  uint32_t key[kSortItems], order[kSortItems], rank[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int i = first + j * 64 + lane;
    key[j] = i < a.tokens ? sort_key(a, i) : 0;
    order[j] = a.order_in != nullptr && i < a.tokens ? a.order_in[i] : static_cast<uint32_t>(i);
  }
  for (int b = tid; b < kSortWaves * kMaxBins; b += kSortThreads) (&bins[0][0])[b] = 0;
  __syncthreads();
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
    uint32_t at = a.counts[b * a.tiles + blockIdx.x];
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t n = bins[w][b];
      bins[w][b] = at;
      at += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    if (first + j * 64 + lane >= a.tokens) continue;
    const uint32_t to = bins[wave][(key[j] >> a.shift) & (nbins - 1)] + rank[j];
    a.keys_out[to] = key[j];
    a.order_out[to] = order[j];
  }
}

// counts -> where each digit of each tile begins, by one workgroup.
__global__ __launch_bounds__(1024) void sort_scan_kernel(uint32_t* counts, int n, const BaseArgs base) {
  __shared__ uint32_t waves[16];
  __shared__ uint32_t carry;
  if (blockIdx.x > 0) return write_base(base, static_cast<int>(blockIdx.x) - 1);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) carry = 0;
  __syncthreads();
  constexpr int EACH = 16;
  for (int at = 0; at < n; at += 1024 * EACH) {
    uint32_t v[EACH], sum = 0;
#pragma unroll
    for (int x = 0; x < EACH; ++x) v[x] = at + tid * EACH + x < n ? counts[at + tid * EACH + x] : 0;
#pragma unroll
    for (int x = 0; x < EACH; ++x) sum += v[x];
    uint32_t scan = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t lower = __shfl_up(scan, o, 64);
      if (lane >= o) scan += lower;
    }
    if (lane == 63) waves[wave] = scan;
    __syncthreads();
    uint32_t run = carry + scan - sum;
#pragma unroll
    for (int w = 0; w < 16; ++w)
      if (w < wave) run += waves[w];
#pragma unroll
    for (int x = 0; x < EACH; ++x) {
      if (at + tid * EACH + x < n) counts[at + tid * EACH + x] = run;
      run += v[x];
    }
    __syncthreads();
    if (tid == 1023) carry = run;
    __syncthreads();
  }
}

// The whole sort by one workgroup, ITEMS * 1024 tokens at most (fewer than 2^16: tokens and places in 16 bits), which go through LDS between the
// passes, keys first, then the tokens.
template <int ITEMS>
__global__ __launch_bounds__(1024) void sort_all_kernel(const SortArgs a, int passes, const BaseArgs base) {
  __shared__ uint32_t moved[ITEMS * 1024];
  __shared__ uint16_t bins[16][kMaxBins];
  __shared__ uint32_t sums[16];
  if (blockIdx.x > 0) return write_base(base, static_cast<int>(blockIdx.x) - 1);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nbins = 1 << a.bits, first = wave * ITEMS * 64 + lane;
  uint32_t key[ITEMS], state[ITEMS];  // state: the token, and above it its rank, then its place
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int i = first + j * 64;
    state[j] = i;
    key[j] = i < a.tokens ? sort_key(a, i) : 0;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * a.bits;
    for (int b = tid; b < 16 * kMaxBins / 2; b += 1024) reinterpret_cast<uint32_t*>(&bins[0][0])[b] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const bool there = first + j * 64 < a.tokens;
      const uint32_t digit = (key[j] >> shift) & (nbins - 1);
      const uint64_t same = same_digit(digit, a.bits, __ballot(there));
      const uint64_t below = same & ((1ull << lane) - 1);
      const uint32_t seen = bins[wave][digit];
      hand_over();
      if (there && below == 0) bins[wave][digit] = static_cast<uint16_t>(seen + __popcll(same));
      hand_over();
      state[j] = (state[j] & 0xffffu) | ((seen + __popcll(below)) << 16);
      __builtin_amdgcn_sched_barrier(0);  // one item's ballots at a time: the registers
    }
    __syncthreads();
    // where each wave's share of each digit begins
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) sum += tid < nbins ? bins[w][tid] : 0;
    uint32_t scan = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t lower = __shfl_up(scan, o, 64);
      if (lane >= o) scan += lower;
    }
    if (lane == 63) sums[wave] = scan;
    __syncthreads();
    uint32_t at = scan - sum;
#pragma unroll
    for (int w = 0; w < 16; ++w)
      if (w < wave) at += sums[w];
    if (tid < nbins) {
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        const uint32_t n = bins[w][tid];
        bins[w][tid] = static_cast<uint16_t>(at);
        at += n;
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      if (first + j * 64 >= a.tokens) continue;
      const uint32_t to = bins[wave][(key[j] >> shift) & (nbins - 1)] + (state[j] >> 16);
      state[j] = (state[j] & 0xffffu) | (to << 16);
      moved[to] = key[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) key[j] = first + j * 64 < a.tokens ? moved[first + j * 64] : 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (first + j * 64 < a.tokens) moved[state[j] >> 16] = state[j] & 0xffffu;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) state[j] = first + j * 64 < a.tokens ? moved[first + j * 64] : 0;
  }
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const int i = first + j * 64;
    if (i >= a.tokens) continue;
    a.keys_out[i] = key[j];
    a.order_out[i] = state[j] & 0xffffu;
  }
}

// ---- dtable ----

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

// Columns c .. of a chunk's part: of the id that begins in it and goes on, or of the one that began earlier.
template <int V>
__device__ __forceinline__ float4* part_at(const EmbedArgs& a, int chunk, bool begins, int c) {
  return reinterpret_cast<float4*>(a.part + (static_cast<int64_t>(chunk) * 2 + (begins ? 1 : 0)) * a.part_ld + c);
}

// A wave sums the rows of chunk `chunk` of the sorted tokens, 64 vectors of columns wide. An id's sum is finished if all of its tokens
// lie in the chunk; otherwise it is a part: [0] of an id that began in an earlier chunk, [1] of one that begins here.
template <typename T, int CHUNK>
__global__ __launch_bounds__(256) void embedding_sum_kernel(const EmbedArgs a) {
  using S = typename Io<T>::storage;
  constexpr int V = kVec<T>;
  const int lane = threadIdx.x & 63;
  const uint32_t work = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int chunk = static_cast<int>(work / a.blocks);
  const int c = (static_cast<int>(work % a.blocks) * 64 + lane) * V;
  if (chunk >= a.chunks) return;
  const int first = chunk * CHUNK, n = min(CHUNK, a.tokens - first);
  // lane i: token i of the chunk; lane CHUNK the one behind the chunk, the next the one before it
  const int at = lane == CHUNK + 1 ? first - 1 : first + min(lane, CHUNK);
  const uint32_t none = 0xffffffffu;
  const uint32_t mine = at >= 0 && at < a.tokens ? a.keys[at] : none;
  const uint32_t token = lane < n ? a.order[first + lane] : 0;
  const uint32_t before = __builtin_amdgcn_readlane(mine, CHUNK + 1);
  uint4 row[CHUNK];  // as it is stored
#pragma unroll
  for (int i = 0; i < CHUNK; ++i) {
    const uint32_t key = __builtin_amdgcn_readlane(mine, i);
    const int64_t t = __builtin_amdgcn_readlane(token, i);
    row[i] = i < n && key < static_cast<uint32_t>(a.vocab) && c < a.dim ? load_bits<T>(static_cast<const S*>(a.in) + t * a.ld + c, a.dim - c)
                                                                      : uint4{0, 0, 0, 0};
  }
  float sum[V];
#pragma unroll
  for (int x = 0; x < V; ++x) sum[x] = 0.0f;
  bool began_here = __builtin_amdgcn_readlane(mine, 0) != before;
#pragma unroll
  for (int i = 0; i < CHUNK; ++i) {
    const uint32_t key = __builtin_amdgcn_readlane(mine, i);
    if (i >= n || key >= static_cast<uint32_t>(a.vocab)) break;
    float v[V];
    unpack_vec<T>(row[i], v);
#pragma unroll
    for (int x = 0; x < V; ++x) sum[x] += v[x];
    const bool ends = __builtin_amdgcn_readlane(mine, i + 1) != key;
    if (!ends && i + 1 < CHUNK) continue;
    if (c < a.dim) {
      if (ends && began_here) {
        finish_row<T>(a, key, c, sum);
      } else {
        float4* p = part_at<V>(a, chunk, began_here, c);
#pragma unroll
        for (int x = 0; x < V / 4; ++x) p[x] = float4{sum[4 * x], sum[4 * x + 1], sum[4 * x + 2], sum[4 * x + 3]};
      }
    }
#pragma unroll
    for (int x = 0; x < V; ++x) sum[x] = 0.0f;
    began_here = true;
  }
}

// sum += parts first .. last - 1 of the id that begins in chunk `chunk`, in their order; the loads of eight at a time
template <typename T>
__device__ __forceinline__ void add_parts(const EmbedArgs& a, int chunk, int first, int last, int c, float (&sum)[kVec<T>]) {
  constexpr int V = kVec<T>, AHEAD = 8;
  for (int p = first; p < last; p += AHEAD) {
    float4 v[AHEAD][V / 4];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int at = min(p + i, last - 1);
#pragma unroll
      for (int x = 0; x < V / 4; ++x) v[i][x] = part_at<V>(a, chunk + at, at == 0, c)[x];
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (p + i >= last) break;
#pragma unroll
      for (int x = 0; x < V / 4; ++x) {
        sum[4 * x] += v[i][x].x;
        sum[4 * x + 1] += v[i][x].y;
        sum[4 * x + 2] += v[i][x].z;
        sum[4 * x + 3] += v[i][x].w;
      }
    }
  }
}

// The parts of ids that go on behind the chunk they begin in. Each of the workgroup's four waves looks at one chunk; few parts are added by
// the wave itself, many by the four waves together, each a run of them.
template <typename T, int CHUNK>
__global__ __launch_bounds__(256) void embedding_join_kernel(const EmbedArgs a) {
  constexpr int V = kVec<T>, FEW = 8;
  __shared__ float runs[4][64][V];
  __shared__ int many[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int group = static_cast<int>(blockIdx.x / a.blocks) * 4;
  const int c = static_cast<int>((blockIdx.x % a.blocks) * 64 + lane) * V;
  const int chunk = group + wave, behind = (chunk + 1) * CHUNK;  // the first token behind the chunk
  uint32_t key = 0;
  int parts = 0;
  if (behind < a.tokens) {
    key = a.keys[behind];
    const uint32_t last = a.keys[behind - 1], before = chunk > 0 ? a.keys[chunk * CHUNK - 1] : 0xffffffffu;
    if (key == last && key != before && key < static_cast<uint32_t>(a.vocab)) {
      int low = behind + 1, high = a.tokens;  // the first token with a greater id lies there: 64 looks at a time
      while (low < high) {
        const int step = (high - low + 63) / 64, at = low + lane * step;
        const int upto = __popcll(__ballot(at < high && a.keys[min(at, high - 1)] <= key));
        high = min(low + upto * step, high);
        low = upto == 0 ? high : low + (upto - 1) * step + 1;
      }
      parts = (low - 1) / CHUNK - chunk + 1;
    }
  }
  float sum[V];
#pragma unroll
  for (int x = 0; x < V; ++x) sum[x] = 0.0f;
  if (parts > 0 && parts <= FEW && c < a.dim) {
    add_parts<T>(a, chunk, 0, parts, c, sum);
    finish_row<T>(a, key, c, sum);
  }
  if (lane == 0) many[wave] = parts > FEW ? parts : 0;
  __syncthreads();
  for (int w = 0; w < 4; ++w) {
    const int all = many[w], each = (all + 3) / 4;
    if (all == 0) continue;
#pragma unroll
    for (int x = 0; x < V; ++x) sum[x] = 0.0f;
    if (c < a.dim) add_parts<T>(a, group + w, wave * each, min(all, (wave + 1) * each), c, sum);
#pragma unroll
    for (int x = 0; x < V; ++x) runs[wave][lane][x] = sum[x];
    __syncthreads();
    if (wave == w && c < a.dim) {
#pragma unroll
      for (int x = 0; x < V; ++x) sum[x] = ((runs[0][lane][x] + runs[1][lane][x]) + runs[2][lane][x]) + runs[3][lane][x];
      finish_row<T>(a, key, c, sum);
    }
    __syncthreads();
  }
}

// ---- few tokens: no sort ----

// Taken for up to 1,024 tokens whose workgroups are 4,096 at most and write at most 2^22 units (us, with this kernel and with the sort's three
// launches; bf16 unless said): 301 of 5,003 x 333 f32: 7.3, 15.4; 64 of 32,768 x 1,024: 14.8, 18 (on another base 24, 30; in place 6.8, 15);
// 512 of 131,072 x 4,096 in place: 12, 18 (1,000, 8,000 workgroups: 25, 18); 512 tokens of one id: 19, 22; 1,000: 34, 27, but 1,000 as
// frequent as words on a base 26, 32 and of 50,257 x 64 f32 7.4, 15. 2^26 units of 131,072 x 4,096: 228, 185 (every workgroup reads the ids).
constexpr int kFew = 1024, kFewGroups = 4096, kFewThreads = 256, kFewWaves = kFewThreads / 64;
constexpr int64_t kFewUnits = int64_t{1} << 22;

// One launch. The first `groups` workgroups: each looks for its token's id among all; the id's first token sums the rows of all of them, 64
// vectors of columns wide, many rows by four waves, each a run of them. The others write base or zeros, `row_units` units a row, in the
// rows that no token names. Tokens: EACH * kFewThreads at most.
template <typename T, int EACH>
__global__ __launch_bounds__(kFewThreads) void embedding_few_kernel(const EmbedArgs a, const BaseArgs base, uint32_t groups, uint32_t row_units) {
  using S = typename Io<T>::storage;
  constexpr int V = kVec<T>, AHEAD = 16;
  __shared__ float runs[kFewWaves][64][V];
  __shared__ uint16_t list[EACH * kFewThreads];
  __shared__ int counts[EACH * kFewWaves];
  __shared__ uint8_t named[kFewThreads];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int ids[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) ids[j] = j * kFewThreads + tid < a.tokens ? a.ids[j * kFewThreads + tid] : -1;
  if (blockIdx.x >= groups) {
    const int64_t at = base.begin + static_cast<int64_t>(blockIdx.x - groups) * kFewThreads, row = at / row_units;
    named[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < EACH; ++j)  // the workgroup's units lie in as many rows as it has threads at most
      if (ids[j] - row >= 0 && ids[j] - row < kFewThreads) named[ids[j] - row] = 1;
    __syncthreads();
    if (named[(static_cast<uint32_t>(at - row * row_units) + tid) / row_units]) return;
    return write_base(base, static_cast<int>(blockIdx.x - groups));
  }
  const int token = static_cast<int>(blockIdx.x / a.blocks);
  const int c = (static_cast<int>(blockIdx.x % a.blocks) * 64 + lane) * V;
  const int id = a.ids[token];
  if (id < 0 || id >= a.vocab) return;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const uint64_t all = __ballot(ids[j] == id);
    if (lane == 0) counts[j * kFewWaves + wave] = __popcll(all);
  }
  __syncthreads();
  int n = 0;  // tokens of the id
#pragma unroll
  for (int i = 0; i < EACH * kFewWaves; ++i) {
    const int j = i / kFewWaves;
    const uint64_t all = __ballot(ids[j] == id);
    if (i % kFewWaves == wave && ids[j] == id)
      list[n + __popcll(all & ((1ull << lane) - 1))] = static_cast<uint16_t>(j * kFewThreads + tid);
    n += __builtin_amdgcn_readfirstlane(counts[i]);
  }
  __syncthreads();
  if (list[0] != token) return;
  // the list's run that this wave sums
  const int each = n <= AHEAD ? n : (n + kFewWaves - 1) / kFewWaves, first = wave * each, last = min(n, first + each);
  float sum[V];
#pragma unroll
  for (int x = 0; x < V; ++x) sum[x] = 0.0f;
  for (int p = first; p < last; p += AHEAD) {
    const int mine = list[min(p + (lane & (AHEAD - 1)), last - 1)];
    uint4 row[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int64_t t = __builtin_amdgcn_readlane(mine, i);
      row[i] = p + i < last && c < a.dim ? load_bits<T>(static_cast<const S*>(a.in) + t * a.ld + c, a.dim - c) : uint4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      float v[V];
      unpack_vec<T>(row[i], v);
#pragma unroll
      for (int x = 0; x < V; ++x) sum[x] = p + i < last ? sum[x] + v[x] : sum[x];
    }
  }
  if (n > AHEAD) {
#pragma unroll
    for (int x = 0; x < V; ++x) runs[wave][lane][x] = sum[x];
    __syncthreads();
#pragma unroll
    for (int x = 0; x < V; ++x) {
      sum[x] = runs[0][lane][x];
      for (int w = 1; w < kFewWaves; ++w) sum[x] += runs[w][lane][x];
    }
  }
  if (wave == 0 && c < a.dim) finish_row<T>(a, id, c, sum);
}

constexpr int64_t kMaxUnits = int64_t{1} << 31;  // that one launch writes beside the sort

fh_status check_embedding(const std::string& fn, const fh_token_embedding* g) {
  if (g == nullptr) return fail(FH_INVALID_ARGUMENT, fn + ": null geometry");
  if (!is_supported_float(g->dtype)) return fail(FH_UNIMPLEMENTED, fn + ": dtype must be f32, f16 or bf16");
  if (g->tokens < 0 || g->vocab < 1 || g->dim < 1) return fail(FH_INVALID_ARGUMENT, fn + ": bad tokens, vocab or dim");
  // a launch has fewer than 2^32 threads: 2^26 waves (of 1,024 columns or more of a token; the gradient's have fewer)
  if (g->vocab > 0x7ffffffe || g->dim > (1 << 20) || g->tokens > (1 << 25) || g->tokens * ((g->dim + 1023) / 1024) >= (1 << 26) ||
      g->vocab * g->dim > (int64_t{1} << 38))
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
  int64_t part_ld, chunk;
};
GradPlan grad_plan(const fh_token_embedding& g) {
  GradPlan p{};
  int64_t key_bits = 1;
  while ((int64_t{1} << key_bits) <= g.vocab) ++key_bits;  // keys are 0 .. vocab
  p.passes = (key_bits + kMaxBits - 1) / kMaxBits;
  p.bits = (key_bits + p.passes - 1) / p.passes;
  p.tiles = (g.tokens + kSortTile - 1) / kSortTile;
  // as long chunks as give every CU 16 waves of 1 KB of a row (4,096 tokens of 1,024 bf16: 13.8 us for sums and join with 8, 17.7 with 16;
  // 32,768 of 4,096: 153 with 8, 137 with 16)
  const int64_t blocks = (g.dim * dtype_size(g.dtype) + 1023) / 1024;
  p.chunk = (g.tokens + 15) / 16 * blocks >= 16 * device_cu_count() ? 16 : 8;
  p.chunks = (g.tokens + p.chunk - 1) / p.chunk;
  p.list = (g.tokens * 4 + 15) / 16 * 16;
  p.counts = 4 * p.list;
  p.part = p.counts + (p.tiles * kMaxBins * 4 + 15) / 16 * 16;
  p.part_ld = (g.dim + 7) / 8 * 8;
  p.bytes = p.part + p.chunks * 2 * p.part_ld * 4;
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

  // base (or zeros), in equal shares beside the sort's launches (32,768 tokens of 131,072 x 4,096: 283 us in all, 302 beside the first alone)
  const int64_t bytes = g->vocab * g->dim * esz;
  BaseArgs share{};
  share.base = base;
  share.dtable = dtable;
  share.size = bytes % 16 == 0 && !misaligned(base, 16) && !misaligned(dtable, 16) ? 16 : static_cast<int>(esz);
  const int64_t units = base == dtable ? 0 : bytes / share.size;
  const bool alone = g->tokens <= kSortAlone;  // one workgroup sorts
  const int64_t sorts = alone ? 1 : 3 * p.passes, before = units / kMaxUnits, launches = before + sorts;
  int64_t launched = 0;
  // the next share, and how many workgroups of `threads` write it
  auto sharers = [&](int64_t threads) {
    share.begin = units * launched / launches;
    share.end = units * ++launched / launches;
    return static_cast<uint32_t>((share.end - share.begin + threads - 1) / threads);
  };

  EmbedArgs a{};
  a.in = dout;
  a.base = base;
  a.out = dtable;
  a.ids = ids;
  a.ld = g->row_stride;
  a.tokens = static_cast<int>(g->tokens);
  a.vocab = static_cast<int>(g->vocab);
  a.dim = static_cast<int>(g->dim);
  a.scale = g->scale;
  const int64_t width = 64 * 16 / esz;
  a.blocks = static_cast<uint32_t>((g->dim + width - 1) / width);

  if (g->tokens > 0 && g->tokens <= kFew && g->tokens * a.blocks <= kFewGroups) {
    // a row is a whole number of units here
    BaseArgs rest = share;
    rest.size = g->dim * esz % 16 == 0 && !misaligned(base, 16) && !misaligned(dtable, 16) ? 16 : static_cast<int>(esz);
    rest.end = base == dtable ? 0 : bytes / rest.size;
    auto launch = [&]<typename T, int EACH>() {
      const uint32_t row_units = static_cast<uint32_t>(g->dim * esz / rest.size), groups = static_cast<uint32_t>(g->tokens * a.blocks);
      const dim3 grid(groups + static_cast<uint32_t>((rest.end + kFewThreads - 1) / kFewThreads));
      hipLaunchKernelGGL((embedding_few_kernel<T, EACH>), grid, dim3(kFewThreads), 0, s, a, rest, groups, row_units);
      return launch_status("embedding_few_kernel launch");
    };
    auto by_tokens = [&]<typename T>() {
      return g->tokens <= kFew / 2 ? launch.template operator()<T, kFew / kFewThreads / 2>() : launch.template operator()<T, kFew / kFewThreads>();
    };
    if (rest.end <= kFewUnits) {
      if (g->dtype == FH_F32) return by_tokens.template operator()<float>();
      return g->dtype == FH_F16 ? by_tokens.template operator()<f16_t>() : by_tokens.template operator()<bf16_t>();
    }
  }

  char* ws = static_cast<char*>(workspace);
  auto list = [&](int i) { return reinterpret_cast<uint32_t*>(ws + i * p.list); };
  SortArgs sort{};
  sort.ids = ids;
  sort.tokens = static_cast<int>(g->tokens);
  sort.vocab = static_cast<int>(g->vocab);
  sort.bits = static_cast<int>(p.bits);
  for (int64_t i = 0; i < before; ++i) {  // what would be too many threads beside the sort is written before it
    hipLaunchKernelGGL(sort_count_kernel, dim3(sharers(kSortThreads)), dim3(kSortThreads), 0, s, sort, share);
    if (fh_status st = launch_status("sort_count_kernel launch"); st != FH_OK) return st;
  }
  if (g->tokens == 0) {
    const uint32_t groups = sharers(kSortThreads);
    if (groups == 0) return FH_OK;
    hipLaunchKernelGGL(sort_count_kernel, dim3(groups), dim3(kSortThreads), 0, s, sort, share);
    return launch_status("sort_count_kernel launch");
  }
  if (alone) {
    sort.keys_out = list(0);
    sort.order_out = list(1);
    const int passes = static_cast<int>(p.passes);
    const dim3 grid(1 + sharers(1024));
    if (g->tokens <= 1024)
      hipLaunchKernelGGL((sort_all_kernel<1>), grid, dim3(1024), 0, s, sort, passes, share);
    else if (g->tokens <= 4096)
      hipLaunchKernelGGL((sort_all_kernel<4>), grid, dim3(1024), 0, s, sort, passes, share);
    else
      hipLaunchKernelGGL((sort_all_kernel<16>), grid, dim3(1024), 0, s, sort, passes, share);
    if (fh_status st = launch_status("sort_all_kernel launch"); st != FH_OK) return st;
  } else {
    sort.counts = reinterpret_cast<uint32_t*>(ws + p.counts);
    sort.tiles = static_cast<int>(p.tiles);
    const uint32_t tiles = static_cast<uint32_t>(p.tiles);
    for (int pass = 0; pass < p.passes; ++pass) {
      sort.shift = pass * sort.bits;
      sort.keys_out = list(2 * (pass & 1));
      sort.order_out = list(2 * (pass & 1) + 1);
      uint32_t groups = sharers(kSortThreads);
      hipLaunchKernelGGL(sort_count_kernel, dim3(tiles + groups), dim3(kSortThreads), 0, s, sort, share);
      if (fh_status st = launch_status("sort_count_kernel launch"); st != FH_OK) return st;
      groups = sharers(1024);
      hipLaunchKernelGGL(sort_scan_kernel, dim3(1 + groups), dim3(1024), 0, s, sort.counts, static_cast<int>(p.tiles << p.bits), share);
      if (fh_status st = launch_status("sort_scan_kernel launch"); st != FH_OK) return st;
      groups = sharers(kSortThreads);
      hipLaunchKernelGGL(sort_scatter_kernel, dim3(tiles + groups), dim3(kSortThreads), 0, s, sort, share);
      if (fh_status st = launch_status("sort_scatter_kernel launch"); st != FH_OK) return st;
      sort.keys_in = sort.keys_out;
      sort.order_in = sort.order_out;
    }
  }

  a.keys = sort.keys_out;
  a.order = sort.order_out;
  a.part = reinterpret_cast<float*>(ws + p.part);
  a.chunks = static_cast<int>(p.chunks);
  a.part_ld = static_cast<int>(p.part_ld);
  auto launch = [&]<typename T, int CHUNK>() {
    hipLaunchKernelGGL((embedding_sum_kernel<T, CHUNK>), dim3(static_cast<uint32_t>((p.chunks * a.blocks + 3) / 4)), dim3(256), 0, s, a);
    if (fh_status st = launch_status("embedding_sum_kernel launch"); st != FH_OK || p.chunks == 1) return st;
    hipLaunchKernelGGL((embedding_join_kernel<T, CHUNK>), dim3(static_cast<uint32_t>((p.chunks + 3) / 4 * a.blocks)), dim3(256), 0, s, a);
    return launch_status("embedding_join_kernel launch");
  };
  auto by_chunk = [&]<typename T>() { return p.chunk == 16 ? launch.template operator()<T, 16>() : launch.template operator()<T, 8>(); };
  if (g->dtype == FH_F32) return by_chunk.template operator()<float>();
  return g->dtype == FH_F16 ? by_chunk.template operator()<f16_t>() : by_chunk.template operator()<bf16_t>();
}
