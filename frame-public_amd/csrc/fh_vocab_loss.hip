// Softmax cross entropy over a vocabulary without keeping the logits (fh_vocab_loss_fwd) and its gradients (fh_vocab_loss_grad).
//
// With z = x w^T, lse = log sum_v exp z and one target per row:
//   forward:   a tile of logits leaves per row the maximum and the sum of exponentials of all but the target's, which a second kernel joins over
//              the tiles of the vocabulary, in their order; with o = log of that sum, row_loss = log(1 + exp(o - z[target])): however small a
//              confident row's loss is, it keeps its bits, which lse - z[target] loses, and 1 + a small sum as well.
//   gradients: with g = exp(z - lse) - [v = target], dx = f g w and dw = f g^T x, f = dloss (/ count for the mean): a piece of
//              the vocabulary at a time, whose logits are formed again, whose g is kept in the storage type (f16: times 2^14, so that
//              probabilities down to 2^-28 keep their bits) and read by both products. f is left to the products' results.
// Rows without a target are taken out first: a list of the others stands for x's rows (forward), or they are copied together (gradients,
// where rows are also summed over, and what such rows hold must not reach the sums). Their number is on the device alone: grids are made
// for all rows, and workgroups without work end at once.
//
// Measured (bf16; two cards, which differ by 6 % under this load):
//   7,373 rows of 131,072 x 4,096:  loss 5.75 to 6.15 ms, 1,290 to 1,380 TFLOP/s (a plain product of these sizes by the vendor's library
//                                   5.48 ms). The matrix unit is busy for 75 % of the cycles at 1.75 GHz of 2.4: the board's power.
//   3,686 rows of the same:         gradients 9.33 to 10.2 ms, 1,160 to 1,270 TFLOP/s over three products; per piece of 16,384 columns
//                                   derivatives 411 us, dx 409, dw 399 (busy for 71, 71 and 67 % of the cycles).
//   4,096 rows of 32,768 x 1,024:   225 to 259 us and 730 to 805. Short products: 4 us of a tile's 31 are its beginning and end. Within the first
//                                   10 ms of such calls one card took 246, then 302, then 243 us for the logits: its power regulation.
//   333 rows of 5,003 x 1,000, f16: gradients 35 us: three dependent launches (traced, where none overlaps the next, 38: derivatives 13, products
//                                   20, dx' join 5). A derivative tile waits 0.8 us for each of its 16 stages: few tiles are on a CU to hide it.
//   1 row of 131,072 x 4,096:       180 us, 6.0 TB/s: the bytes of w (64 x 128 tiles, two stages ahead).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "fh_common.h"
#include "fh_tile_product.h"

namespace fh {
namespace {

using namespace tile;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// What g is multiplied by in the storage type.
template <typename T>
constexpr float kRaise = std::is_same_v<T, f16_t> ? 0x1p14f : 1.0f;

// Stages of a tile's ring: two of 64 KB for the largest, 32 KB each for the next; three for the small ones, whose stages are short.
template <int BM>
constexpr int kRing = BM >= 128 ? 2 : 3;

struct LossArgs {
  const uint16_t* x;
  const uint16_t* w;
  const int32_t* targets;
  int64_t ldx, ldw;
  int tokens, vocab, dim;
  int mean, loss_dtype;
  float* lse;
  float* row_loss;
  void* loss;
  const void* dloss;
  uint16_t* dx;
  uint16_t* dw;
  // workspace
  int* count;        // rows with a target
  int32_t* rows;     // which they are, in their order
  float* at_target;  // their target's logit
  int32_t* targets_c;  // and their targets
  float2* part;        // [column tiles][tokens]: from, sum of exp(z - from) over all but the target
  int tiles_n;
  // gradients: the rows with a target copied together, their log-sum-exps, a piece of g, fp32 sums of dx over the pieces
  uint16_t* xc;
  float* lse_c;
  uint16_t* g;
  int64_t ldg;
  float* dx_sum;  // [splits][tokens][dim]
  int first, last;  // columns of the piece
  int splits;       // of a piece's columns in dx' product
  int first_piece, last_piece;
};

// max and sum over the 4 lanes that share a row of a tile
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float row_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
// A maximum that exponents can be taken against: of a row of -infinity, 0.
__device__ __forceinline__ float origin(float m) { return m == -INFINITY ? 0.0f : m; }
// exp(z - from). The difference is formed first: of logits near their maximum it is exact, however large they are, and a row's largest counts as
// exactly 1. (z log2 e - from log2 e in one fused operation saves one of three per logit, and is off by the rounding of from log2 e: a
// probability too large for the row's log-sum-exp at a few hundred, infinite or zero from logits of 2^32 on.)
__device__ __forceinline__ float exp_from(float z, float from) { return __builtin_amdgcn_exp2f((z - from) * kLog2e); }
// {from, sum of exp(z - from)} of two sets of logits. An empty sum (logits of -infinity) is 0 and its from says nothing.
__device__ __forceinline__ float2 add_exponentials(const float2& a, const float2& b) {
  if (a.y == 0.0f) return b;
  if (b.y == 0.0f) return a;
  const float from = fmaxf(a.x, b.x);
  return float2{from, a.y * exp_from(a.x, from) + b.y * exp_from(b.x, from)};
}

// Runs f(i, j, x) for the lane's place in acc that is column `target` of row i of the wave's part (columns from `column` on). Few tiles hold the target
// of any of their rows, so the rows are asked first and the columns only where one answers.
template <typename P, typename F>
__device__ __forceinline__ void at_targets(const int (&target)[P::TM], int column, F&& f) {
#pragma unroll
  for (int i = 0; i < P::TM; ++i) {
    const int in = target[i] - column;
    if (__ballot(in >= 0 && in < P::WN) == 0) continue;
#pragma unroll
    for (int j = 0; j < P::TN; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (in == 16 * j + 4 * (P::lane() >> 4) + x) f(i, j, x);
  }
}

// ---- rows with a target ----

// The list of rows with a target, their number and targets; the others' outputs, or (gradients: lse_c) the log-sum-exps. Workgroup b takes
// the b'th run of `each` rows and counts the targets before it by itself: it reads them once more instead of waiting for the others
// (8,192 rows: 6 us; one workgroup that reads its rows once 13, and 20 with the log-sum-exps).
__global__ __launch_bounds__(1024) void loss_rows_kernel(const LossArgs a, int each) {
  __shared__ int waves[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int begin = static_cast<int>(blockIdx.x) * each, end = min(a.tokens, begin + each);
  auto counts = [&](int target) { return target >= 0 && target < a.vocab; };
  // the workgroup's sum of n, to all
  auto total = [&](int n) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    if (lane == 0) waves[wave] = n;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) sum += waves[w];
    __syncthreads();
    return sum;
  };
  int n = 0;
#pragma unroll 8
  for (int t = tid; t < begin; t += 1024) n += counts(a.targets[t]);
  int before = begin > 0 ? total(n) : 0;
  for (int at = begin; at < end; at += 1024) {
    const int t = at + tid;
    const int target = t < end ? a.targets[t] : -1;
    const bool mine = counts(target);
    const uint64_t mask = __ballot(mine);
    if (lane == 0) waves[wave] = __popcll(mask);
    __syncthreads();
    int to = before + __popcll(mask & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      if (w < wave) to += waves[w];
      before += waves[w];
    }
    __syncthreads();
    if (mine) {
      a.rows[to] = t;
      a.targets_c[to] = target;
      if (a.lse_c != nullptr) a.lse_c[to] = a.lse[t];
    } else if (t < end && a.lse_c == nullptr) {
      a.lse[t] = 0.0f;
      if (a.row_loss != nullptr) a.row_loss[t] = 0.0f;
    }
  }
  if (blockIdx.x + 1 == gridDim.x && tid == 0) *a.count = before;
}

// The same list for up to MOST rows, by every workgroup for itself in LDS, which saves a launch; returns the rows' number. The workgroup that
// is `first` also writes what loss_rows_kernel writes.
template <int MOST>
struct FewRows {
  int32_t rows[MOST], targets[MOST];
  int waves[16];
};
template <int THREADS, int MOST>
__device__ __forceinline__ int list_few_rows(const LossArgs& a, FewRows<MOST>& few, bool first) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int count = 0;
  for (int at = 0; at < a.tokens; at += THREADS) {
    const int t = at + static_cast<int>(threadIdx.x);
    const int target = t < a.tokens ? a.targets[t] : -1;
    const bool mine = target >= 0 && target < a.vocab;
    const uint64_t mask = __ballot(mine);
    if (lane == 0) few.waves[wave] = __popcll(mask);
    __syncthreads();
    int to = count + __popcll(mask & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) to += few.waves[w];
      count += few.waves[w];
    }
    if (mine) {
      few.rows[to] = t;
      few.targets[to] = target;
    }
    __syncthreads();
    if (!first) continue;
    if (mine) {
      a.rows[to] = t;
      a.targets_c[to] = target;
      if (a.lse_c != nullptr) a.lse_c[to] = a.lse[t];
    } else if (t < a.tokens && a.lse_c == nullptr) {
      a.lse[t] = 0.0f;
      if (a.row_loss != nullptr) a.row_loss[t] = 0.0f;
    }
  }
  if (first && threadIdx.x == 0) *a.count = count;
  return count;
}

// ---- forward ----

// FEW: up to kFewRows rows, which the workgroups list themselves (us, with a launch for the list before: 16 rows of 5,000 x 512 14 and 10, 333 of
// 50,261 x 1,000 42 and 40, 500 of 32,768 x 256 23.4 and 21.2; the same from 80 us on). Three of the smallest tiles and their lists still fit a CU.
constexpr int kFewRows = 512;
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, bool UNEVEN, bool FEW>
__global__ __launch_bounds__(WAVES_M* WAVES_N * 64) void loss_logits_kernel(const LossArgs a) {
  using P = Product<T, BM, BN, WAVES_M, WAVES_N, kRing<BM>, Lie::kListed, Lie::kRows, UNEVEN, UNEVEN>;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[P::kLds];
  __shared__ FewRows<FEW ? kFewRows : 1> few;
  int count;
  const int32_t *rows = a.rows, *targets = a.targets_c;
  if constexpr (FEW) {
    count = list_few_rows<P::kThreads>(a, few, blockIdx.x == 0);
    rows = few.rows;
    targets = few.targets;
  } else {
    count = *a.count;
  }
  int tm, tn;
  if (!place(blockIdx.x, (count + BM - 1) / BM, a.tiles_n, tm, tn)) return;
  const int m0 = tm * BM, n0 = tn * BN;
  typename P::Acc acc;
  P::run(lds, {a.x, a.ldx, rows, count - 1, a.dim}, {a.w, a.ldw, nullptr, a.vocab - 1, a.dim}, m0, n0, (a.dim + kDepth - 1) / kDepth, acc);
  float2(*joined)[BM] = reinterpret_cast<float2(*)[BM]>(lds);
  const int g = P::lane() >> 4, r = P::lane() & 15, row0 = P::wave_row() + r, column = n0 + P::wave_column();
  if (n0 + BN > a.vocab) {  // columns that do not exist are tokens of probability zero
#pragma unroll
    for (int i = 0; i < P::TM; ++i)
#pragma unroll
      for (int j = 0; j < P::TN; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (column + 16 * j + 4 * g + x >= a.vocab) acc[i][j][x] = -INFINITY;
  }
  int target[P::TM];
#pragma unroll
  for (int i = 0; i < P::TM; ++i) target[i] = m0 + row0 + 16 * i < count ? targets[m0 + row0 + 16 * i] : -1;
  at_targets<P>(target, column, [&](int i, int j, int x) {
    a.at_target[m0 + row0 + 16 * i] = acc[i][j][x];
    acc[i][j][x] = -INFINITY;  // the sums are the other tokens'
  });
#pragma unroll
  for (int i = 0; i < P::TM; ++i) {
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < P::TN; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) top = fmaxf(top, acc[i][j][x]);
    const float from = origin(row_max(top));
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < P::TN; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) sum += exp_from(acc[i][j][x], from);
    sum = row_sum(sum);
    if (g == 0) joined[P::wave() % WAVES_N][row0 + 16 * i] = float2{from, sum};
  }
  __syncthreads();
  for (int row = threadIdx.x; row < BM; row += P::kThreads) {
    if (m0 + row >= count) break;
    float2 both = joined[0][row];
    for (int w = 1; w < WAVES_N; ++w) both = add_exponentials(both, joined[w][row]);
    a.part[static_cast<int64_t>(tn) * a.tokens + m0 + row] = both;
  }
}

__device__ __forceinline__ void store_loss(const LossArgs& a, double sum, int count) {
  const float loss = static_cast<float>(a.mean && count > 0 ? sum / count : sum);
  if (a.loss_dtype == FH_F32) *static_cast<float*>(a.loss) = loss;
  if (a.loss_dtype == FH_BF16) *static_cast<uint16_t*>(a.loss) = Io<bf16_t>::store(loss);
  if (a.loss_dtype == FH_F16) *static_cast<uint16_t*>(a.loss) = Io<f16_t>::store(loss);
}

// ROWS rows per workgroup, THREADS / ROWS threads each a share of the tiles, eight of them at a time; the shares are joined in their
// order. ALL: the only workgroup, which forms the loss as well.
template <int ROWS, int THREADS, bool ALL>
__global__ __launch_bounds__(THREADS) void loss_join_kernel(const LossArgs a) {
  constexpr int SHARES = THREADS / ROWS, AHEAD = 8;
  __shared__ float2 shares[SHARES][ROWS];
  __shared__ float losses[ROWS];
  const int row = threadIdx.x % ROWS, share = threadIdx.x / ROWS, count = *a.count;
  const int m = static_cast<int>(blockIdx.x) * ROWS + row;
  const bool live = m < count;
  float2 sum{0.0f, 0.0f};
  if (live)
    for (int first = share; first < a.tiles_n; first += AHEAD * SHARES) {
      float2 p[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) p[i] = a.part[static_cast<int64_t>(min(first + i * SHARES, a.tiles_n - 1)) * a.tokens + m];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (first + i * SHARES < a.tiles_n) sum = add_exponentials(sum, p[i]);
    }
  shares[share][row] = sum;
#pragma unroll
  for (int o = SHARES / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (share < o) shares[share][row] = sum = add_exponentials(sum, shares[share + o][row]);
  }
  float loss = 0.0f;
  if (share == 0 && live) {
    // d: the others' log-sum-exp less the target's logit (a logit of +infinity has no distance). Neither result is below what it is added to, so
    // lse is not less than any logit: the others' sum, with their largest, is 1 at least.
    const float z = a.at_target[m], above = kLn2 * __builtin_amdgcn_logf(sum.y);
    const float d = z == INFINITY ? NAN : (sum.x - z) + above;
    const float more = log1pf(expf(-fabsf(d)));
    const bool none = sum.y == 0.0f && z == -INFINITY;  // no token has a probability
    const int t = a.rows[m];
    a.lse[t] = none ? -INFINITY : (d > 0.0f ? sum.x + above : z) + more;
    loss = fmaxf(d, 0.0f) + more;
    a.at_target[m] = loss;
    if (a.row_loss != nullptr) a.row_loss[t] = loss;
  }
  if constexpr (ALL) {
    if (share == 0) losses[row] = loss;
    __syncthreads();
    if (threadIdx.x == 0) {
      double all = 0.0;
      for (int r = 0; r < ROWS; ++r) all += losses[r];
      store_loss(a, all, count);
    }
  }
}

// The loss, by one workgroup: the rows' losses in one order, in double. (By the join's workgroup that is through last: 1,000 rows of 5,000 x 512
// 39 us in all, 22 with this launch: every workgroup has to write its caches back.)
__global__ __launch_bounds__(1024) void loss_sum_kernel(const LossArgs a) {
  __shared__ double shares[1024];
  const int tid = threadIdx.x, count = *a.count;
  double sum = 0.0;
  for (int m = tid; m < count; m += 1024) sum += a.at_target[m];
  shares[tid] = sum;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if (tid < o) shares[tid] += shares[tid + o];
    __syncthreads();
  }
  if (tid == 0) store_loss(a, shares[0], count);
}

// ---- gradients ----

// A wave per row: xc's row m is x's row rows[m]; rows behind the last, up to a multiple of 64, are zeros (dw sums over them); dx's rows
// without a target are zeros. FEW: up to kGatherFew rows, which the workgroups list themselves (1,024 rows of 5,000 x 512: 51 us in all,
// 57 for one row more and a launch for the list).
constexpr int kGatherFew = 1024;
__device__ __forceinline__ void gather_row(const LossArgs& a, const int32_t* rows, int count, int t) {
  const int lane = threadIdx.x & 63, end = (count + 63) / 64 * 64;
  const u32x4_t zeros{0, 0, 0, 0};
  if (t < end) {
    const uint16_t* from = t < count ? a.x + rows[t] * a.ldx : nullptr;
    for (int c = lane * 8; c < a.dim; c += 512)
      *reinterpret_cast<u32x4_t*>(a.xc + static_cast<int64_t>(t) * a.dim + c) = from != nullptr ? *reinterpret_cast<const u32x4_t*>(from + c) : zeros;
  }
  if (a.dx != nullptr && t < a.tokens && !(a.targets[t] >= 0 && a.targets[t] < a.vocab))
    for (int c = lane * 8; c < a.dim; c += 512) *reinterpret_cast<u32x4_t*>(a.dx + t * a.ldx + c) = zeros;
}
template <bool FEW>
__global__ __launch_bounds__(256) void loss_gather_kernel(const LossArgs a) {
  __shared__ FewRows<FEW ? kGatherFew : 1> few;
  const int t = static_cast<int>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if constexpr (FEW) {
    const int count = list_few_rows<256>(a, few, blockIdx.x == 0);
    gather_row(a, few.rows, count, t);
  } else {
    gather_row(a, a.rows, *a.count, t);
  }
}

__device__ __forceinline__ float loss_factor(const LossArgs& a) {
  const float d = a.loss_dtype == FH_F32    ? *static_cast<const float*>(a.dloss)
                  : a.loss_dtype == FH_BF16 ? Io<bf16_t>::load(*static_cast<const uint16_t*>(a.dloss))
                                            : Io<f16_t>::load(*static_cast<const uint16_t*>(a.dloss));
  return a.mean ? d / static_cast<float>(*a.count) : d;
}

template <typename P>
__device__ __forceinline__ void scale(typename P::Acc& acc, float f) {
#pragma unroll
  for (int i = 0; i < P::TM; ++i)
#pragma unroll
    for (int j = 0; j < P::TN; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[i][j][x] *= f;
}

// g of a piece: columns first .. last - 1 of the vocabulary, zeros behind them and in the tile's rows that no row with a target is.
// FEW: up to kFewRows rows, which the workgroups list themselves and read where they are; the first `gathers` workgroups do what
// loss_gather_kernel does.
// A launch less: both gradients of 16 rows of 5,000 x 512 19.4 us before, 16.7 now, of 333 of 5,003 x 1,000 40 and 35, of 512 of 2,048 x 2,048
// 39 and 34.
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, bool UNEVEN, bool FEW>
__global__ __launch_bounds__(WAVES_M* WAVES_N * 64) void loss_derivative_kernel(const LossArgs a, uint32_t gathers) {
  using P = Product<T, BM, BN, WAVES_M, WAVES_N, kRing<BM>, FEW ? Lie::kListed : Lie::kRows, Lie::kRows, UNEVEN, UNEVEN>;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[P::kLds];
  __shared__ FewRows<FEW ? kFewRows : 1> few;
  int count;
  if constexpr (FEW) {
    count = list_few_rows<P::kThreads>(a, few, blockIdx.x == 0);
    if (blockIdx.x < gathers) return gather_row(a, few.rows, count, static_cast<int>(blockIdx.x) * (P::kThreads / 64) + (threadIdx.x >> 6));
  } else {
    count = *a.count;
  }
  int tm, tn;
  if (!place(blockIdx.x - gathers, (count + BM - 1) / BM, static_cast<int>(a.ldg / BN), tm, tn)) return;
  const int m0 = tm * BM, n0 = tn * BN;
  typename P::Acc acc;
  P::run(lds, {FEW ? a.x : a.xc, FEW ? a.ldx : a.dim, FEW ? few.rows : nullptr, count - 1, a.dim},
         {a.w + a.first * a.ldw, a.ldw, nullptr, a.vocab - 1 - a.first, a.dim}, m0, n0, (a.dim + kDepth - 1) / kDepth, acc);
  const int row0 = m0 + P::wave_row() + (P::lane() & 15), column = a.first + n0 + P::wave_column();
  int target[P::TM];
#pragma unroll
  for (int i = 0; i < P::TM; ++i) {
    const int m = min(row0 + 16 * i, count - 1);
    const float lse = FEW ? a.lse[few.rows[m]] : a.lse_c[m];
    target[i] = FEW ? few.targets[m] : a.targets_c[m];
#pragma unroll
    for (int j = 0; j < P::TN; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[i][j][x] = __builtin_amdgcn_exp2f((acc[i][j][x] - lse) * kLog2e) * kRaise<T>;
  }
  at_targets<P>(target, column, [&](int i, int j, int x) { acc[i][j][x] -= kRaise<T>; });
  if (m0 + BM > count || a.first + n0 + BN > a.last) {
#pragma unroll
    for (int i = 0; i < P::TM; ++i)
#pragma unroll
      for (int j = 0; j < P::TN; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (row0 + 16 * i >= count || column + 16 * j + 4 * (P::lane() >> 4) + x >= a.last) acc[i][j][x] = 0.0f;
  }
  P::store(lds, acc, [&](int row, int c, const u32x4_t& v) {
    *reinterpret_cast<u32x4_t*>(a.g + static_cast<int64_t>(m0 + row) * a.ldg + n0 + c) = v;
  });
}

// A tile of dx: one split's share of a piece.
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, bool UNEVEN>
using DxProduct = Product<T, BM, BN, WAVES_M, WAVES_N, kRing<BM>, Lie::kRows, Lie::kColumns, false, UNEVEN>;
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, bool UNEVEN>
__device__ __forceinline__ void dx_tile(const LossArgs& a, unsigned char* lds, uint32_t block, int split) {
  using P = DxProduct<T, BM, BN, WAVES_M, WAVES_N, UNEVEN>;
  const int count = *a.count;
  int tm, tn;
  if (!place(block, (count + BM - 1) / BM, (a.dim + BN - 1) / BN, tm, tn)) return;
  // this split's share of the piece's stages
  const int stages = (a.last - a.first + kDepth - 1) / kDepth, share = (stages + a.splits - 1) / a.splits;
  const int k0 = split * share, KT = min(share, stages - k0);
  const int m0 = tm * BM, n0 = tn * BN, from = a.first + k0 * kDepth, depth = a.last - from;
  typename P::Acc acc;
  P::run(lds, {a.g + k0 * kDepth, a.ldg, nullptr, count - 1, depth}, {a.w + from * a.ldw, a.ldw, nullptr, a.dim - 1, depth}, m0, n0, KT, acc);
  const bool whole = a.splits == 1 && a.last_piece;
  if (!a.first_piece || !whole) {
    const int row0 = m0 + P::wave_row() + (P::lane() & 15), col0 = n0 + P::wave_column() + 4 * (P::lane() >> 4);
#pragma unroll
    for (int i = 0; i < P::TM; ++i) {
      if (row0 + 16 * i >= count) continue;
      f32x4_t* sum = reinterpret_cast<f32x4_t*>(a.dx_sum + (static_cast<int64_t>(split) * a.tokens + row0 + 16 * i) * a.dim + col0);
#pragma unroll
      for (int j = 0; j < P::TN; ++j) {
        if (col0 + 16 * j >= a.dim) continue;
        if (!a.first_piece) acc[i][j] += sum[4 * j];
        if (!whole) sum[4 * j] = acc[i][j];
      }
    }
  }
  if (!whole) return;
  scale<P>(acc, loss_factor(a) / kRaise<T>);
  P::store(lds, acc, [&](int row, int c, const u32x4_t& v) {
    if (m0 + row < count && n0 + c < a.dim) *reinterpret_cast<u32x4_t*>(a.dx + a.rows[m0 + row] * a.ldx + n0 + c) = v;
  });
}
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, bool UNEVEN>
__global__ __launch_bounds__(WAVES_M* WAVES_N * 64) void loss_dx_kernel(const LossArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[DxProduct<T, BM, BN, WAVES_M, WAVES_N, UNEVEN>::kLds];
  dx_tile<T, BM, BN, WAVES_M, WAVES_N, UNEVEN>(a, lds, blockIdx.x, static_cast<int>(blockIdx.y));
}

// dx from the splits' sums, in their order: 8 columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void loss_dx_join_kernel(const LossArgs a) {
  const int vectors = a.dim / 8;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int m = static_cast<int>(at / vectors), c = static_cast<int>(at % vectors) * 8;
  if (m >= *a.count) return;
  f32x4_t low{0.0f, 0.0f, 0.0f, 0.0f}, high = low;
  for (int s = 0; s < a.splits; ++s) {
    const f32x4_t* p = reinterpret_cast<const f32x4_t*>(a.dx_sum + (static_cast<int64_t>(s) * a.tokens + m) * a.dim + c);
    low += p[0];
    high += p[1];
  }
  const float f = loss_factor(a) / kRaise<T>;
  *reinterpret_cast<u32x4_t*>(a.dx + a.rows[m] * a.ldx + c) =
      u32x4_t{store2<T>(low[0] * f, low[1] * f), store2<T>(low[2] * f, low[3] * f), store2<T>(high[0] * f, high[1] * f),
              store2<T>(high[2] * f, high[3] * f)};
}

// A tile of dw.
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N>
using DwProduct = Product<T, BM, BN, WAVES_M, WAVES_N, kRing<BM>, Lie::kColumns, Lie::kColumns, false, false>;
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N>
__device__ __forceinline__ void dw_tile(const LossArgs& a, unsigned char* lds, uint32_t block) {
  using P = DwProduct<T, BM, BN, WAVES_M, WAVES_N>;
  const int count = *a.count;
  int tm, tn;
  if (!place(block, static_cast<int>((a.last - a.first + BM - 1) / BM), (a.dim + BN - 1) / BN, tm, tn)) return;
  const int m0 = tm * BM, n0 = tn * BN;
  typename P::Acc acc;
  P::run(lds, {a.g, a.ldg, nullptr, static_cast<int>(a.ldg) - 1, 0}, {a.xc, a.dim, nullptr, a.dim - 1, 0}, m0, n0, (count + kDepth - 1) / kDepth, acc);
  scale<P>(acc, count > 0 ? loss_factor(a) / kRaise<T> : 0.0f);
  P::store(lds, acc, [&](int row, int c, const u32x4_t& v) {
    const int64_t to = a.first + m0 + row;
    if (to < a.last && n0 + c < a.dim) *reinterpret_cast<u32x4_t*>(a.dw + to * a.ldw + n0 + c) = v;
  });
}
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N>
__global__ __launch_bounds__(WAVES_M* WAVES_N * 64) void loss_dw_kernel(const LossArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[DwProduct<T, BM, BN, WAVES_M, WAVES_N>::kLds];
  dw_tile<T, BM, BN, WAVES_M, WAVES_N>(a, lds, blockIdx.x);
}

// Both in one launch, where either is small: `dx_tiles` workgroups for each of dx' splits, then dw's.
template <typename T, bool UNEVEN>
__global__ __launch_bounds__(256) void loss_products_kernel(const LossArgs a, uint32_t dx_tiles) {
  using X = DxProduct<T, 64, 64, 2, 2, UNEVEN>;
  using W = DwProduct<T, 64, 64, 2, 2>;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[X::kLds > W::kLds ? X::kLds : W::kLds];
  const uint32_t of_dx = dx_tiles * static_cast<uint32_t>(a.splits);
  if (blockIdx.x < of_dx) dx_tile<T, 64, 64, 2, 2, UNEVEN>(a, lds, blockIdx.x % dx_tiles, static_cast<int>(blockIdx.x / dx_tiles));
  else dw_tile<T, 64, 64, 2, 2>(a, lds, blockIdx.x - of_dx);
}

// ---- host ----

constexpr int kLeastPiece = 256;
constexpr int64_t kPieceValues = int64_t{1} << 26;  // of g: 128 MB (3,686 rows of 131,072 columns: 9.64 ms; 256 MB 9.68, 512 MB 9.56)
constexpr int64_t kMostPieceValues = int64_t{1} << 28;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

fh_status check_loss(const std::string& fn, const fh_vocab_loss* g) {
  if (g == nullptr) return fail(FH_INVALID_ARGUMENT, fn + ": null geometry");
  if (g->dtype != FH_BF16 && g->dtype != FH_F16) return fail(FH_UNIMPLEMENTED, fn + ": dtype must be bf16 or f16");
  if (g->loss_dtype != FH_F32 && g->loss_dtype != g->dtype) return fail(FH_INVALID_ARGUMENT, fn + ": loss_dtype must be f32 or dtype");
  if (g->mean != 0 && g->mean != 1) return fail(FH_INVALID_ARGUMENT, fn + ": mean must be 0 or 1");
  if (g->tokens < 0 || g->vocab < 1 || g->dim < 8) return fail(FH_INVALID_ARGUMENT, fn + ": bad tokens, vocab or dim");
  if (g->dim % 8 != 0) return fail(FH_UNIMPLEMENTED, fn + ": dim must be a multiple of 8");
  // a launch has fewer than 2^32 threads: 2^22 of the largest tiles, of 512 threads (smaller ones are taken where these are few)
  auto tiles = [](int64_t m, int64_t n) { return up(m, 256) / 256 * (up(n, 256) / 256); };
  if (g->tokens > (1 << 24) || g->vocab > (1 << 24) || g->dim > (1 << 20) || tiles(g->tokens, std::max(g->vocab, g->dim)) > (1 << 22) ||
      tiles(g->vocab, g->dim) > (1 << 22))
    return fail(FH_INVALID_ARGUMENT, fn + ": too large");
  for (int64_t ld : {g->x_stride, g->w_stride})
    if (ld < g->dim || ld % 8 != 0 || ld >= (int64_t{1} << 22))
      return fail(FH_INVALID_ARGUMENT, fn + ": strides must be multiples of 8, at least dim and less than 2^22");
  return FH_OK;
}

// The tile of a product of m rows and n columns: the largest that gives (nearly) every CU a workgroup, as in fh_gemm16.hip (loss of 8,192
// rows of 131,072 x 512: 1,106 us in 256 x 256 tiles, 1,451 in 128 x 128; 400 rows of 131,072 x 1,024: 136 and 173; dw of 512 rows of
// 131,072 x 4,096, eight stages a tile: 6 % of the whole call slower in 128 x 128, 19 % in 64 x 128).
struct Shape {
  int m, n;
};
Shape tile_for(int64_t m, int64_t n) {
  const int64_t cus = device_cu_count();
  auto tiles = [&](int64_t bm, int64_t bn) { return up(m, bm) / bm * (up(n, bn) / bn); };
  if (m >= 256 && n >= 256 && tiles(256, 256) * 4 >= cus * 3) return {256, 256};
  if (m >= 128 && n >= 128 && tiles(128, 128) >= cus) return {128, 128};
  if (n >= 128 && tiles(64, 128) >= cus) return {64, 128};
  return {64, 64};
}
// launch<BM, BN, WAVES_M, WAVES_N>(workgroups) with tiles of shape t over m x n
template <typename F>
void by_tile(Shape t, int64_t m, int64_t n, F&& launch) {
  const dim3 grid(static_cast<uint32_t>(up(m, t.m) / t.m * (up(n, t.n) / t.n)));
  if (t.m == 256) launch.template operator()<256, 256, 4, 2>(grid);
  else if (t.m == 128) launch.template operator()<128, 128, 2, 4>(grid);
  else if (t.n == 128) launch.template operator()<64, 128, 2, 2>(grid);
  else launch.template operator()<64, 64, 2, 2>(grid);
}

// dx is small and its sums are long, a piece's columns: where tiles leave CUs idle, the columns are split among `splits` workgroups, whose
// sums a second launch joins. The cheapest by rounds of workgroups over the CUs, a tile's products over its share of the columns
// at the rates below, and a stage's worth of waiting at either end (4,096 rows of 32,768 x 1,024: dx 445 us in 128 x 128 tiles, 276 and 16
// for the join in four splits of 256 x 256; 333 of 5,003 x 1,000: 23, and 10 and 5).
struct DxPlan {
  Shape tile;
  int splits;
};
DxPlan dx_plan(int64_t tokens, int64_t dim, int64_t columns) {
  const int64_t cus = device_cu_count(), stages = up(columns, 64) / 64;
  DxPlan best{{64, 64}, 1};
  double least = 0.0;
  const struct {
    Shape t;
    int together;   // workgroups of a CU
    double stage;   // us of a stage with so many
  } kinds[] = {{{256, 256}, 1, 1.7}, {{128, 128}, 2, 1.25}, {{64, 128}, 2, 0.75}, {{64, 64}, 3, 0.6}};
  for (const auto& k : kinds)
    for (int splits = 1; splits <= 8; splits *= 2) {
      const int64_t tiles = up(tokens, k.t.m) / k.t.m * (up(dim, k.t.n) / k.t.n) * splits, share = (stages + splits - 1) / splits;
      const double rounds = static_cast<double>(up(tiles, cus * k.together) / (cus * k.together));
      const double us = rounds * (static_cast<double>(share) + 4.0) * k.stage + (splits > 1 ? 4.0 + splits * tokens * dim * 8 / 4e6 : 0.0);
      if (least == 0.0 || us < least) {
        least = us;
        best = {k.t, splits};
      }
    }
  return best;
}

// Where dx takes the smallest tiles and dw has few of them, 8 per CU, one launch does both in those tiles (both gradients, us, two launches
// before: 16 rows of 5,000 x 512 23.6 and 19.4, 333 of 5,003 x 1,000 43 and 40, 1,000 of 5,000 x 512 50.6 and 45.5, at the limit 512 of
// 8,192 x 1,024 59.6 and 59.3). Behind it dw's larger tiles gain.
constexpr int64_t kTogether = 8;

struct Room {
  int64_t bytes = 0;
  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += up(n, 256);
    return at;
  }
};
struct ForwardRoom {
  int64_t count, rows, targets, at_target, part, bytes;
  int64_t tiles_n;
};
ForwardRoom forward_room(const fh_vocab_loss& g) {
  Room r;
  ForwardRoom f{};
  f.count = r.take(4);
  f.rows = r.take(4 * g.tokens);
  f.targets = r.take(4 * g.tokens);
  f.at_target = r.take(4 * g.tokens);
  const int64_t columns = tile_for(g.tokens, g.vocab).n;
  f.tiles_n = up(g.vocab, columns) / columns;
  f.part = r.take(8 * g.tokens * f.tiles_n);
  f.bytes = r.bytes;
  return f;
}
struct GradRoom {
  int64_t count, rows, targets, lse, xc, dx_sum, g, bytes;
  int64_t g_rows;
};
// with a piece of `columns`, dx' product in `splits`
GradRoom grad_room(const fh_vocab_loss& g, int64_t columns, int splits) {
  Room r;
  GradRoom f{};
  f.g_rows = up(g.tokens, 256);
  f.count = r.take(4);
  f.rows = r.take(4 * g.tokens);
  f.targets = r.take(4 * g.tokens);
  f.lse = r.take(4 * g.tokens);
  f.xc = r.take(2 * f.g_rows * g.dim);
  f.dx_sum = r.take(columns < g.vocab || splits > 1 ? 4 * splits * g.tokens * g.dim : 0);
  f.g = r.take(2 * f.g_rows * columns);
  f.bytes = r.bytes;
  return f;
}
struct GradPlan {
  int64_t columns;  // of a piece
  DxPlan dx;
};
GradPlan best_plan(const fh_vocab_loss& g) {
  const int64_t all = up(g.vocab, kLeastPiece), rows = up(std::max<int64_t>(g.tokens, 1), 256);
  GradPlan p{};
  // at least as many columns as give every CU one of dw's largest tiles (8,192 rows of 131,072 x 512: 3.48 ms, 3.84 by kPieceValues alone)
  const int64_t round = up(up(device_cu_count() * 65536, g.dim) / g.dim, kLeastPiece);
  const int64_t columns = std::min(std::max(kPieceValues / rows, round), kMostPieceValues / rows) / kLeastPiece * kLeastPiece;
  p.columns = std::min(all, std::max<int64_t>(columns, kLeastPiece));
  p.dx = dx_plan(g.tokens, g.dim, std::min(p.columns, g.vocab));
  return p;
}
int64_t best_room(const fh_vocab_loss& g) {
  const GradPlan p = best_plan(g);
  return grad_room(g, p.columns, p.dx.splits).bytes;
}
// one piece in one split needs no room for sums
int64_t least_room(const fh_vocab_loss& g) {
  return std::min({grad_room(g, kLeastPiece, 1).bytes, grad_room(g, best_plan(g).columns, 1).bytes, best_room(g)});
}
// The best plan, or what `bytes` have room for: without splits, and then the widest piece that fits.
GradPlan plan_for(const fh_vocab_loss& g, int64_t bytes) {
  GradPlan p = best_plan(g);
  if (bytes >= grad_room(g, p.columns, p.dx.splits).bytes) return p;
  p.dx = {tile_for(g.tokens, g.dim), 1};
  if (bytes >= grad_room(g, p.columns, 1).bytes) return p;
  const GradRoom least = grad_room(g, kLeastPiece, 1);
  // room beside the sums between pieces, which a piece of the whole vocabulary would not need
  p.columns = std::min(p.columns, (bytes - least.g) / (2 * least.g_rows) / kLeastPiece * kLeastPiece);
  if (p.columns >= g.vocab) p.columns = up(g.vocab, kLeastPiece) - kLeastPiece;
  return p;
}

LossArgs loss_args(const fh_vocab_loss& g, const void* x, const void* w, const int32_t* targets) {
  LossArgs a{};
  a.x = static_cast<const uint16_t*>(x);
  a.w = static_cast<const uint16_t*>(w);
  a.targets = targets;
  a.ldx = g.x_stride;
  a.ldw = g.w_stride;
  a.tokens = static_cast<int>(g.tokens);
  a.vocab = static_cast<int>(g.vocab);
  a.dim = static_cast<int>(g.dim);
  a.mean = g.mean;
  a.loss_dtype = g.loss_dtype;
  return a;
}

fh_status list_rows(const LossArgs& a, hipStream_t stream) {
  // at most 64 workgroups: what they count again stays few times the rows
  const int each = static_cast<int>(std::max<int64_t>(up((a.tokens + 63) / 64, 1024), 1024));
  hipLaunchKernelGGL(loss_rows_kernel, dim3(static_cast<uint32_t>(std::max(1, (a.tokens + each - 1) / each))), dim3(1024), 0, stream, a, each);
  return launch_status("loss_rows_kernel launch");
}

template <typename F>
fh_status by_type(int32_t dtype, F&& f) {
  return dtype == FH_BF16 ? f.template operator()<bf16_t>() : f.template operator()<f16_t>();
}

}  // namespace
}  // namespace fh

using namespace fh;

extern "C" int64_t fh_vocab_loss_workspace(const fh_vocab_loss* g) {
  if (check_loss("fh_vocab_loss_workspace", g) != FH_OK) return -1;
  return forward_room(*g).bytes;
}

extern "C" fh_status fh_vocab_loss_fwd(const fh_vocab_loss* g, const void* x, const void* w, const int32_t* targets, void* loss,
                                       float* row_loss, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  const std::string fn = "fh_vocab_loss_fwd";
  if (fh_status st = check_loss(fn, g); st != FH_OK) return st;
  if (!loss || !workspace || (g->tokens > 0 && (!x || !w || !targets || !lse))) return fail(FH_INVALID_ARGUMENT, fn + ": null pointer");
  if (!aligned16(x) || !aligned16(w) || !aligned16(workspace))
    return fail(FH_INVALID_ARGUMENT, fn + ": x, w and the workspace must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(targets) | reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(row_loss)) % 4 != 0 ||
      reinterpret_cast<uintptr_t>(loss) % dtype_size(g->loss_dtype) != 0)
    return fail(FH_INVALID_ARGUMENT, fn + ": targets, loss, row_loss and lse must be aligned to their elements");
  const ForwardRoom room = forward_room(*g);
  if (workspace_bytes < room.bytes) return fail(FH_INVALID_ARGUMENT, fn + ": workspace too small");
  char* ws = static_cast<char*>(workspace);
  LossArgs a = loss_args(*g, x, w, targets);
  a.loss = loss;
  a.row_loss = row_loss;
  a.lse = lse;
  a.count = reinterpret_cast<int*>(ws + room.count);
  a.rows = reinterpret_cast<int32_t*>(ws + room.rows);
  a.at_target = reinterpret_cast<float*>(ws + room.at_target);
  a.part = reinterpret_cast<float2*>(ws + room.part);
  a.targets_c = reinterpret_cast<int32_t*>(ws + room.targets);
  a.tiles_n = static_cast<int>(room.tiles_n);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool few = g->tokens > 0 && g->tokens <= kFewRows;
  if (!few)
    if (fh_status st = list_rows(a, s); st != FH_OK) return st;
  if (g->tokens > 0) {
    const fh_status st = by_type(g->dtype, [&]<typename T>() {
      by_tile(tile_for(g->tokens, g->vocab), g->tokens, g->vocab, [&]<int BM, int BN, int WM, int WN>(dim3 grid) {
        auto go = [&]<bool UNEVEN, bool FEW>() {
          hipLaunchKernelGGL((loss_logits_kernel<T, BM, BN, WM, WN, UNEVEN, FEW>), grid, dim3(WM * WN * 64), 0, s, a);
        };
        const bool uneven = g->dim % kDepth != 0;
        if (few) return uneven ? go.template operator()<true, true>() : go.template operator()<false, true>();
        uneven ? go.template operator()<true, false>() : go.template operator()<false, false>();
      });
      return launch_status("loss_logits_kernel launch");
    });
    if (st != FH_OK) return st;
    // up to 16 rows by one workgroup, which sums them too (16 rows of 5,000 x 512: 14 us in all, 17 with the sum's launch); a few: a workgroup
    // each (one row of 1,024 tiles by 16 threads: 32 us)
    if (g->tokens <= 16) {
      hipLaunchKernelGGL((loss_join_kernel<16, 1024, true>), dim3(1), dim3(1024), 0, s, a);
      return launch_status("loss_join_kernel launch");
    }
    if (g->tokens <= 4 * device_cu_count())
      hipLaunchKernelGGL((loss_join_kernel<1, 256, false>), dim3(static_cast<uint32_t>(g->tokens)), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((loss_join_kernel<16, 256, false>), dim3(static_cast<uint32_t>((g->tokens + 15) / 16)), dim3(256), 0, s, a);
    if (fh_status st2 = launch_status("loss_join_kernel launch"); st2 != FH_OK) return st2;
  }
  hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, s, a);
  return launch_status("loss_sum_kernel launch");
}

extern "C" int64_t fh_vocab_loss_grad_workspace(const fh_vocab_loss* g) {
  if (check_loss("fh_vocab_loss_grad_workspace", g) != FH_OK) return -1;
  return best_room(*g);
}

extern "C" int64_t fh_vocab_loss_grad_least(const fh_vocab_loss* g) {
  if (check_loss("fh_vocab_loss_grad_least", g) != FH_OK) return -1;
  return least_room(*g);
}

extern "C" fh_status fh_vocab_loss_grad(const fh_vocab_loss* g, const void* x, const void* w, const int32_t* targets, const float* lse,
                                        const void* dloss, void* dx, void* dw, void* workspace, int64_t workspace_bytes, void* stream) {
  const std::string fn = "fh_vocab_loss_grad";
  if (fh_status st = check_loss(fn, g); st != FH_OK) return st;
  if (!dx && !dw) return FH_OK;
  if (g->tokens == 0 && !dw) return FH_OK;
  if (!workspace || !dloss || (g->tokens > 0 && (!x || !w || !targets || !lse))) return fail(FH_INVALID_ARGUMENT, fn + ": null pointer");
  for (const void* p : {x, w, static_cast<const void*>(dx), static_cast<const void*>(dw), static_cast<const void*>(workspace)})
    if (!aligned16(p)) return fail(FH_INVALID_ARGUMENT, fn + ": tensors and the workspace must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(targets) | reinterpret_cast<uintptr_t>(lse)) % 4 != 0 ||
      reinterpret_cast<uintptr_t>(dloss) % dtype_size(g->loss_dtype) != 0)
    return fail(FH_INVALID_ARGUMENT, fn + ": targets, lse and dloss must be aligned to their elements");
  if (workspace_bytes < least_room(*g)) return fail(FH_INVALID_ARGUMENT, fn + ": workspace too small");
  const GradPlan plan = plan_for(*g, workspace_bytes);
  const int64_t columns = plan.columns;
  const GradRoom room = grad_room(*g, columns, plan.dx.splits);
  char* ws = static_cast<char*>(workspace);
  LossArgs a = loss_args(*g, x, w, targets);
  a.lse = const_cast<float*>(lse);
  a.dloss = dloss;
  a.dx = static_cast<uint16_t*>(dx);
  a.dw = static_cast<uint16_t*>(dw);
  a.count = reinterpret_cast<int*>(ws + room.count);
  a.rows = reinterpret_cast<int32_t*>(ws + room.rows);
  a.targets_c = reinterpret_cast<int32_t*>(ws + room.targets);
  a.lse_c = reinterpret_cast<float*>(ws + room.lse);
  a.xc = reinterpret_cast<uint16_t*>(ws + room.xc);
  a.dx_sum = reinterpret_cast<float*>(ws + room.dx_sum);
  a.g = reinterpret_cast<uint16_t*>(ws + room.g);
  a.splits = plan.dx.splits;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint32_t gathers = static_cast<uint32_t>(up(g->tokens, 64) / 4);  // of four rows
  const bool few = g->tokens > 0 && g->tokens <= kGatherFew;
  const bool fewer = few && g->tokens <= kFewRows && tile_for(g->tokens, std::min(up(g->vocab, kLeastPiece), columns)).m == 64;
  if (!few)
    if (fh_status st = list_rows(a, s); st != FH_OK) return st;
  if (g->tokens > 0 && !fewer) {
    if (few)
      hipLaunchKernelGGL((loss_gather_kernel<true>), dim3(gathers), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((loss_gather_kernel<false>), dim3(gathers), dim3(256), 0, s, a);
    if (fh_status st = launch_status("loss_gather_kernel launch"); st != FH_OK) return st;
  }
  auto together = [&](const LossArgs& p) {
    return dx && dw && plan.dx.tile.m == 64 && plan.dx.tile.n == 64 &&
           up(p.last - p.first, 64) / 64 * (up(g->dim, 64) / 64) <= kTogether * device_cu_count();
  };
  return by_type(g->dtype, [&]<typename T>() {
    for (int64_t first = 0; first < g->vocab; first += columns) {
      a.first = static_cast<int>(first);
      a.last = static_cast<int>(std::min(g->vocab, first + columns));
      a.first_piece = first == 0;
      a.last_piece = a.last == g->vocab;
      a.ldg = up(a.last - a.first, kLeastPiece);
      if (g->tokens > 0) {
        by_tile(tile_for(g->tokens, a.ldg), g->tokens, a.ldg, [&]<int BM, int BN, int WM, int WN>(dim3 grid) {
          auto go = [&]<bool UNEVEN, bool FEW>() {
            if (FEW) grid.x += gathers;
            hipLaunchKernelGGL((loss_derivative_kernel<T, BM, BN, WM, WN, UNEVEN, FEW>), grid, dim3(WM * WN * 64), 0, s, a, FEW ? gathers : 0);
          };
          const bool uneven = g->dim % kDepth != 0;
          if constexpr (BM == 64) {
            if (fewer && first == 0) return uneven ? go.template operator()<true, true>() : go.template operator()<false, true>();
          }
          uneven ? go.template operator()<true, false>() : go.template operator()<false, false>();
        });
        if (fh_status st = launch_status("loss_derivative_kernel launch"); st != FH_OK) return st;
        if (together(a)) {
          const uint32_t dx_tiles = static_cast<uint32_t>(up(g->tokens, 64) / 64 * (up(g->dim, 64) / 64));
          const dim3 grid(dx_tiles * static_cast<uint32_t>(a.splits) + static_cast<uint32_t>(up(a.last - a.first, 64) / 64 * (up(g->dim, 64) / 64)));
          if ((a.last - a.first) % kDepth != 0)
            hipLaunchKernelGGL((loss_products_kernel<T, true>), grid, dim3(256), 0, s, a, dx_tiles);
          else
            hipLaunchKernelGGL((loss_products_kernel<T, false>), grid, dim3(256), 0, s, a, dx_tiles);
          if (fh_status st = launch_status("loss_products_kernel launch"); st != FH_OK) return st;
          continue;
        }
        if (dx)
          by_tile(plan.dx.tile, g->tokens, g->dim, [&]<int BM, int BN, int WM, int WN>(dim3 grid) {
            grid.y = static_cast<uint32_t>(a.splits);
            if ((a.last - a.first) % kDepth != 0)
              hipLaunchKernelGGL((loss_dx_kernel<T, BM, BN, WM, WN, true>), grid, dim3(WM * WN * 64), 0, s, a);
            else
              hipLaunchKernelGGL((loss_dx_kernel<T, BM, BN, WM, WN, false>), grid, dim3(WM * WN * 64), 0, s, a);
          });
        if (fh_status st = launch_status("loss_dx_kernel launch"); st != FH_OK) return st;
      }
      if (dw)
        by_tile(tile_for(a.last - a.first, g->dim), a.last - a.first, g->dim, [&]<int BM, int BN, int WM, int WN>(dim3 grid) {
          hipLaunchKernelGGL((loss_dw_kernel<T, BM, BN, WM, WN>), grid, dim3(WM * WN * 64), 0, s, a);
        });
      if (fh_status st = launch_status("loss_dw_kernel launch"); st != FH_OK) return st;
    }
    if (dx && a.splits > 1 && g->tokens > 0) {
      hipLaunchKernelGGL((loss_dx_join_kernel<T>), dim3(static_cast<uint32_t>((g->tokens * (g->dim / 8) + 255) / 256)), dim3(256), 0, s, a);
      return launch_status("loss_dx_join_kernel launch");
    }
    return FH_OK;
  });
}
