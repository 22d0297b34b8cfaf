// Softmax cross entropy of a linear layer's results, which are never kept:
//   z_i = W x_i + b,  lse_i = log(sum over v of exp(z_iv)),  loss_i = lse_i - z_i[t_i];
//   dz_iv = f_i (exp(z_iv - lse_i) - [v = t_i]),  dx = dz W,  dW = dz^T x,  db = sum over i of dz_i,
// where f_i is the upstream gradient of loss_i.
//
// Rows without a target take part in nothing, so the others are gathered first
// (rows_kernel, gather_kernel), and the products after that have as many rows as there
// are targets; what they cost goes by the targets and not by the batch.  How many there are
// stays on the device: launches are sized for all, and workgroups past the last row end.
//
// Forward: the products' workgroups reduce every 64 logits of a row to their maximum and
// the sum of exponentials beside it, and pick the target's, for whose 64 they also give the sum
// without it; lse_kernel joins these.
// Backward: the vocabulary goes in pieces.  A piece's logits are formed again, turned into
// dz on their way out, and multiplied into dx, a running FP32 sum over the pieces, and dW,
// whose rows the piece completes.  The logits' second product is what not keeping them
// costs: 8 operations a weight and row where 6 would do.
//
// Ahead: where all f_i will be the same number the gradients are formed with the loss, but
// for that number, in 6.  The rows go in chunks.  A chunk's logits leave their product as
// exponentials beside the maximum of their 64; once all of the chunk's rows have their lse,
// slope_kernel turns these into dz, which is multiplied into dx and a running FP32 sum of dW.
// FP32 sums are what stays for the backward, which scales and rounds them.
//
// 16384 x 4096 into 131072 words, bf16, ahead, 44.4 ms: the logits' product 15.0 (1.17 PFLOP/s; 14.0 without keeping
// the exponentials), dx 13.4, dW 14.6, slope_kernel 1.6, scale_kernel 0.66; forming the logits again it took 56.4.
// One row of it, the forward alone, 180 us: the weight at 6.0 TB/s.
//
// dz is rounded to the operands' type, as the products' operands have to be; that of batches of up to
// 128 rows comes in two parts of 16 bits, as if it were twice as many rows (a larger batch of which few
// rows have a target keeps one part).  In FP16 dz is held times a
// power of two that puts the largest |f_i| between 2^14 and 2^15: probabilities down to 2^-39 of
// the largest factor stay above zero then.  The results' last step divides by it, exactly.  The
// other types have the range without.
#include <algorithm>

#include "fh_plan.h"
#include "linear.h"

namespace fh {
namespace {

constexpr int kRowThreads = 1024;

struct RowsArgs {
  const int64_t* targets;
  int64_t ignore;
  int rows, vocab;
  int* live;          // how many rows have a target; backward: and twice as many
  int* index;         // [rows] which ones, in their order
  int* label;         // [rows] their targets; -1 for one that is out of range
  float* losses;      // forward: [rows] zeroed where there is no target, or null
  // backward
  const float* grad;  // of the loss, or of each row's
  int per_row, mean, scaled;
  const float2* lse;  // [rows] in the order of `index`: lse and 1 - p of the target
  float4* row;        // [rows] lse, the factor and p - 1
  float* scale;       // what undoes the factors' power of two
};

// Sum over the workgroup of a count for each thread, and of those before it.
__device__ __forceinline__ int before(bool mine, int& total, int (&area)[2][kRowThreads / 64], int& turn) {
  const uint64_t mask = __ballot(mine);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int* counts = area[turn];
  turn ^= 1;  // what the others may still read stays
  if (lane == 0) counts[wave] = __popcll(mask);
  __syncthreads();
  int sum = 0, mine_before = 0;
#pragma unroll
  for (int w = 0; w < kRowThreads / 64; ++w) {
    if (w == wave) mine_before = sum;
    sum += counts[w];
  }
  total = sum;
  return mine_before + lanes_below(mask);
}

// One workgroup: targets are few beside anything else here.
template <bool Backward>
__global__ __launch_bounds__(kRowThreads) void rows_kernel(RowsArgs a) {
  __shared__ int area[2][kRowThreads / 64];
  __shared__ float most[kRowThreads / 64];
  int turn = 0, done = 0, total;
  float power = 1.f, mean = 1.f;
  if constexpr (Backward) {
    // The largest finite factor's size, and how many factors there are.
    float largest = 0.f;
    int count = 0;
    for (int64_t r = threadIdx.x; r < a.rows; r += kRowThreads) {
      if (a.targets[r] == a.ignore) continue;
      ++count;
      const float g = __builtin_fabsf(a.grad[a.per_row ? r : 0]);
      if (g < __builtin_inff()) largest = __builtin_fmaxf(largest, g);
    }
    __shared__ int counts[kRowThreads / 64];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      largest = __builtin_fmaxf(largest, __shfl_xor(largest, d));
      count += __shfl_xor(count, d);
    }
    if ((threadIdx.x & 63) == 0) {
      most[threadIdx.x >> 6] = largest;
      counts[threadIdx.x >> 6] = count;
    }
    __syncthreads();
    count = 0;
    for (int w = 0; w < kRowThreads / 64; ++w) {
      largest = __builtin_fmaxf(largest, most[w]);
      count += counts[w];
    }
    mean = a.mean ? static_cast<float>(count) : 1.f;
    largest /= mean;
    if (a.scaled && largest > 0.f) {
      const int e = 14 - (static_cast<int>(__float_as_uint(largest) >> 23) - 127);
      power = __builtin_ldexpf(1.f, e < -112 ? -112 : e > 126 ? 126 : e);
    }
    if (threadIdx.x == 0) *a.scale = 1.f / power;
  }
  for (int64_t first = 0; first < a.rows; first += kRowThreads) {
    const int64_t r = first + threadIdx.x;
    const int64_t t = r < a.rows ? a.targets[r] : a.ignore;
    const bool mine = r < a.rows && t != a.ignore;
    const int at = done + before(mine, total, area, turn);
    done += total;
    if (mine) {
      const bool valid = t >= 0 && t < a.vocab;
      a.index[at] = static_cast<int>(r);
      a.label[at] = valid ? static_cast<int>(t) : -1;
      if constexpr (Backward) {
        const float f = valid ? a.grad[a.per_row ? r : 0] / mean * power : __builtin_nanf("");
        a.row[at] = make_float4(a.lse[at].x, f, -a.lse[at].y, 0.f);
      }
    } else if (!Backward && r < a.rows && a.losses != nullptr) {
      a.losses[r] = 0.f;
    }
  }
  if (threadIdx.x == 0) {
    a.live[0] = done;
    if (Backward) a.live[1] = 2 * done;
  }
}

struct GatherArgs {
  const void* src;    // [rows, cols], rows src_stride elements apart
  int64_t src_stride;
  const int* live;
  const int* index;
  void* out;          // [rows, ld], zero past cols
  void* twice;        // [2 rows, ld] each row twice, or null
  int64_t ld;
  int cols;
  // Rows of dx without a target are zeroed, unless it is null.
  const int64_t* targets;
  int64_t ignore, rows;
  void* dx;
};

template <typename T>
__device__ __forceinline__ void zero_row(const int64_t* targets, int64_t ignore, int64_t row, int cols, void* dx) {
  if (dx == nullptr || targets[row] != ignore) return;
  auto* to = static_cast<typename T::storage*>(dx) + row * cols;
  for (int c = (threadIdx.x & 63) * kVec<T>; c < cols; c += 64 * kVec<T>) store_row<T>(U32x4{0, 0, 0, 0}, to, c, cols);
}

// A wavefront to each row, and to each that has a target.
template <typename T>
__global__ __launch_bounds__(256) void gather_kernel(GatherArgs a) {
  using S = typename T::storage;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  zero_row<T>(a.targets, a.ignore, row, a.cols, a.dx);
  if (row >= *a.live) return;
  const S* from = static_cast<const S*>(a.src) + a.index[row] * a.src_stride;
  S* to = static_cast<S*>(a.out) + row * a.ld;
  for (int c = (threadIdx.x & 63) * kVec<T>; c < a.ld; c += 64 * kVec<T>) {
    const U32x4 w = load_row<T>(from, c, a.cols);
    __builtin_memcpy(to + c, &w, 16);
    if (a.twice != nullptr) {
      __builtin_memcpy(static_cast<S*>(a.twice) + 2 * row * a.ld + c, &w, 16);
      __builtin_memcpy(static_cast<S*>(a.twice) + (2 * row + 1) * a.ld + c, &w, 16);
    }
  }
}

struct SlopeArgs {
  void* dz;             // [rows, ld]: exponentials, and then the gradients
  int64_t ld;
  const float2* stats;  // [groups, stats_ld]
  int64_t stats_ld;
  const float2* lse;    // lse and 1 - p of the target
  const int *live, *label;
  int row0, rows;
  float* sums;          // [rows / 64, ld] column sums of each 64 rows, or null
};

// exp(z - lse) - [target] from exp(z - maximum of its 64): 64 vectors of 64 rows a workgroup, a
// wavefront to every fourth row.  The target's is what its logit gave, in FP32: 1 - p would show the
// exponential's rounding where p is close to one.  Column sums are of what is not rounded yet.  Bound by
// memory: 8192 rows of 131072 words, 4.3 GB, take 0.79 ms (5.4 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void slope_kernel(SlopeArgs a) {
  using S = typename T::storage;
  using Z = Saved<T>;
  constexpr int V = kVec<T>, kAhead = 4;
  __shared__ float area[4][V][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (static_cast<int>(blockIdx.x) * 64 + lane) * V;
  const int more = *a.live - a.row0, rows = more < a.rows ? more : a.rows;
  const float2* stats = a.stats + static_cast<int64_t>(c / 64) * a.stats_ld;
  const int start = static_cast<int>(blockIdx.y) * 64, last = start + 64 < rows ? start + 64 : rows;
  if (start >= rows) return;  // the whole workgroup
  float sums[V] = {};
  for (int first = start + wave; c < a.ld && first < last; first += 4 * kAhead) {
    U32x4 raw[kAhead];
    float top[kAhead];
    float2 lse[kAhead];
    int label[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int r = first + 4 * u < last ? first + 4 * u : first;
      __builtin_memcpy(&raw[u], static_cast<const S*>(a.dz) + r * a.ld + c, 16);
      top[u] = stats[r].x;
      lse[u] = a.lse[r];
      label[u] = a.label[r];
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (first + 4 * u >= last) break;
      float f[V];
      to_floats<Z>(raw[u], f);
      // A target out of range makes its row NaN.
      const float times = (label[u] < 0 ? __builtin_nanf("") : expf(top[u] - lse[u].x)) *
                          (T::code == BF16::code ? 1.f / kKept : 1.f);  // FP16 and FP32 keep their scales
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] *= times;
      const int at = label[u] - c;
      if (at >= 0 && at < V) {
        const float hit = -lse[u].y * (T::code == F16::code ? kKept : 1.f);
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = k == at ? hit : f[k];
      }
      const U32x4 w = from_floats<T>(f);
      __builtin_memcpy(static_cast<S*>(a.dz) + (first + 4 * u) * a.ld + c, &w, 16);
#pragma unroll
      for (int k = 0; k < V; ++k) sums[k] += f[k];
    }
  }
  if (a.sums == nullptr) return;
#pragma unroll
  for (int k = 0; k < V; ++k) area[wave][k][lane] = sums[k];
  __syncthreads();
  float* to = a.sums + static_cast<int64_t>(blockIdx.y) * a.ld + static_cast<int64_t>(blockIdx.x) * 64 * V;
  for (int i = threadIdx.x; i < 64 * V && static_cast<int>(blockIdx.x) * 64 * V + i < a.ld; i += 256)
    to[i] = ((area[0][i % V][i / V] + area[1][i % V][i / V]) + area[2][i % V][i / V]) + area[3][i % V][i / V];
}

// out[index[i]] = (sums[2 i] + sums[2 i + 1]) scale: rows in two parts.
template <typename T>
__global__ __launch_bounds__(256) void parts_kernel(const float* sums, const int* live, const int* index,
                                                    const float* scale, int cols, void* out) {
  constexpr int V = 8;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= *live) return;
  const float* from = sums + 2 * row * cols;
  auto* to = static_cast<typename T::storage*>(out) + static_cast<int64_t>(index[row]) * cols;
  for (int c = (threadIdx.x & 63) * V; c < cols; c += 64 * V) {
    float f[V], g[V];
    load_some(from + c, cols - c, f);
    load_some(from + cols + c, cols - c, g);
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = (f[k] + g[k]) * *scale;
    typename T::storage e[V];
    round_some<T>(f, e);
    store_some(e, to + c, cols - c);
  }
}

// out = sums times grad, over how many rows have a target for a mean (nothing where none has): a
// wavefront to a row, or to every gridDim.y-th 512 columns of it.  With an index the first `live`
// rows, row k into row index[k], beside zeros for those without a target.
struct ScaleArgs {
  const float* sums;
  const int *live, *index;
  const float* grad;
  int mean;
  float factor;
  int64_t rows;
  int cols;
  void* out;
  const int64_t* targets;
  int64_t ignore;
};
template <typename T>
__global__ __launch_bounds__(256) void scale_kernel(ScaleArgs a) {
  constexpr int V = 8;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const int live = *a.live;
  if (a.index != nullptr) {
    if (blockIdx.y == 0) zero_row<T>(a.targets, a.ignore, row, a.cols, a.out);
    if (row >= live) return;
  }
  const float times = live == 0 ? 0.f : *a.grad / (a.mean ? static_cast<float>(live) : 1.f);
  const float* from = a.sums + row * a.cols;
  auto* to = static_cast<typename T::storage*>(a.out) + (a.index != nullptr ? a.index[row] : row) * a.cols;
  for (int c = (blockIdx.y * 64 + (threadIdx.x & 63)) * V; c < a.cols; c += gridDim.y * 64 * V) {
    float f[V];
    load_some(from + c, a.cols - c, f);
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = f[k] * a.factor * times;
    typename T::storage e[V];
    if constexpr (T::code == F32::code) __builtin_memcpy(e, f, sizeof(e));
    else round_some<T>(f, e);
    store_some(e, to + c, a.cols - c);
  }
}

struct LseArgs {
  const float2* stats;  // [groups, ld]
  int64_t ld;
  int groups, rows;
  const int* live;
  int row0;
  const int* label;
  const int* index;
  const float *chosen, *rest;
  float2* lse;          // [rows] in the order of `index`: lse and 1 - p of the target
  float* losses;        // likewise, or by their rows
  int by_row;
};

// Joins two pairs of a maximum and a sum of exponentials beside it.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = __builtin_fmaxf(a.x, b.x), from = m == -__builtin_inff() ? 0.f : m;
  return make_float2(m, a.y * expf(a.x - from) + b.y * expf(b.x - from));
}

// Sixteen wavefronts, `across` rows (a power of two, up to 64) by 1024 / across groups.
__global__ __launch_bounds__(1024) void lse_kernel(LseArgs a, int across) {
  __shared__ float2 area[1024];
  const int live = *a.live - a.row0, rows = live < a.rows ? live : a.rows;
  const int row = static_cast<int>(blockIdx.x) * across + (threadIdx.x & (across - 1));
  if (static_cast<int>(blockIdx.x) * across >= rows) return;  // the whole workgroup
  float2 sum = make_float2(-__builtin_inff(), 0.f);  // of all but the target
  const int label = row < rows ? a.label[row] : -1;
  if (row < rows) {
    for (int g = threadIdx.x / across; g < a.groups; g += 1024 / across) {
      float2 part = a.stats[static_cast<int64_t>(g) * a.ld + row];
      if (label >= 0 && g == label / 64) part.y = a.rest[row];
      sum = join(sum, part);
    }
  }
  area[threadIdx.x] = sum;
  for (int d = 512; d >= across; d >>= 1) {
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < d) area[threadIdx.x] = sum = join(sum, area[threadIdx.x + d]);
  }
  if (static_cast<int>(threadIdx.x) < across && row < rows) {
    const float chosen = label >= 0 ? a.chosen[row] : -__builtin_inff();
    const float below = sum.x - chosen;  // how far the target is below the maximum
    const float all = sum.y + (label >= 0 ? expf(chosen - sum.x) : 0.f), log_all = logf(all);
    a.lse[row] = make_float2(sum.x + log_all, sum.y / all);
    // A loss close to zero keeps its digits as the logarithm of one more than the others' share.
    const float loss = below < 16.f ? log1pf(sum.y * expf(below)) : below + log_all;
    a.losses[a.by_row ? a.index[row] : row] = label >= 0 ? loss : __builtin_nanf("");
  }
}

// The sum of the losses, or their mean, by one workgroup in FP64.
__global__ __launch_bounds__(1024) void loss_kernel(const float* losses, const int* live, int mean, float* out) {
  __shared__ double area[1024];
  const int count = *live;
  double sum = 0.0;
  for (int i = threadIdx.x; i < count; i += 1024) sum += losses[i];
  area[threadIdx.x] = sum;
  for (int d = 512; d > 0; d >>= 1) {
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < d) area[threadIdx.x] = sum = sum + area[threadIdx.x + d];
  }
  if (threadIdx.x == 0) *out = static_cast<float>(mean ? sum / count : sum);
}

struct BiasArgs {
  const void* dz;      // [rows, ld]
  int64_t ld;
  int cols, rows;
  const int* live;
  int row0;
  float* partial;      // [gridDim.y, cols], or null where the sums are db already
  float* sums;         // [cols] of the chunks so far, or null where there is one
  const float* scale;  // what db is times, or null
  void* out;
  int out_f32;         // its type: FP32, or dz's
};

template <typename T>
__device__ __forceinline__ void put_bias(const BiasArgs& a, int c, float sum) {
  if (a.scale != nullptr) sum *= *a.scale;
  if (a.out_f32) static_cast<float*>(a.out)[c] = sum;
  else static_cast<typename T::storage*>(a.out)[c] = from_f32<T>(sum);
}

// Column sums of dz: 32 V columns and every gridDim.y-th 32 rows a workgroup, half a wavefront to a row.
template <typename T>
__global__ __launch_bounds__(1024) void bias_kernel(BiasArgs a) {
  using S = typename T::storage;
  constexpr int V = kVec<T>;
  __shared__ float area[32][V][32];
  const int lane = threadIdx.x & 31, half = threadIdx.x >> 5;
  const int first = static_cast<int>(blockIdx.x) * 32 * V, c = first + lane * V;
  const int more = *a.live - a.row0, rows = more < a.rows ? more : a.rows;
  float sums[V] = {};
#pragma unroll 4
  for (int row = blockIdx.y * 32 + half; row < rows; row += gridDim.y * 32) {
    float f[V];
    to_floats<T>(load_row<T>(static_cast<const S*>(a.dz) + row * a.ld, c, a.cols), f);
#pragma unroll
    for (int i = 0; i < V; ++i) sums[i] += f[i];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) area[half][i][lane] = sums[i];
  __syncthreads();
  const int mine = static_cast<int>(threadIdx.x), to = first + mine;
  if (mine >= 32 * V || to >= a.cols) return;
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < 32; ++w) sum += area[w][mine % V][mine / V];
  if (a.partial != nullptr) a.partial[static_cast<int64_t>(blockIdx.y) * a.cols + to] = sum;
  else put_bias<T>(a, to, sum);
}

// A chunk's `count` partial sums added to those of the chunks before it; db after the last one.
template <typename T>
__global__ __launch_bounds__(256) void join_bias_kernel(BiasArgs a, int count, bool first, bool last) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.cols) return;
  float sum = first ? 0.f : a.sums[c];
#pragma unroll 8
  for (int i = 0; i < count; ++i) sum += a.partial[static_cast<int64_t>(i) * a.cols + c];
  if (last) put_bias<T>(a, c, sum);
  else a.sums[c] = sum;
}

// Column sums of a chunk from those of each 64 rows, as far as rows are live, added to the chunks' before it.
__global__ __launch_bounds__(256) void join_rows_kernel(const float* parts, const int* live, int row0, int rows, int ld,
                                                        int cols, float* out) {
  const int c = blockIdx.x * 256 + threadIdx.x, more = *live - row0, count = ((more < rows ? more : rows) + 63) / 64;
  if (c >= cols) return;
  float sum = row0 == 0 ? 0.f : out[c];
#pragma unroll 8
  for (int i = 0; i < count; ++i) sum += parts[static_cast<int64_t>(i) * ld + c];
  out[c] = sum;
}

int element(int dtype) { return dtype == F32::code ? 4 : 2; }

char* bytes_on(const void* p, int64_t bytes) {
  return p != nullptr ? reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(p) + bytes) : nullptr;
}

dim3 blocks_of(int64_t items, int each) { return dim3(static_cast<uint32_t>((items + each - 1) / each)); }

// db of `cols` words from the dz of `chunks` chunks of up to `most` rows each, one after the other.
class BiasSums {
 public:
  BiasSums(bool wanted, int64_t chunks, int64_t most, int64_t cols, int dtype, Workspace& ws)
      : dtype_(dtype), down_(most <= 512 ? 1 : static_cast<int>(std::min<int64_t>(most / 256, 64))) {
    if (!wanted) return;
    if (chunks * down_ > 1) partial_ = ws.take<float>(down_ * cols);
    if (chunks > 1) sums_ = ws.take<float>(cols);
  }
  // Adds `rows` rows from row0 on, the last ones or not; `args` has the output.
  hipError_t add(BiasArgs args, const Laid& dz, int64_t row0, int64_t rows, bool last, hipStream_t stream) const {
    args.dz = dz.data;
    args.ld = dz.ld;
    args.row0 = static_cast<int>(row0);
    args.rows = static_cast<int>(rows);
    args.partial = partial_;
    args.sums = sums_;
    return with_type(dtype_, [&](auto t) {
      using T = decltype(t);
      const int64_t each = 32 * kVec<T>;
      const dim3 grid(static_cast<uint32_t>((args.cols + each - 1) / each), static_cast<uint32_t>(down_));
      bias_kernel<T><<<grid, dim3(1024), 0, stream>>>(args);
      if (partial_ != nullptr)
        join_bias_kernel<T><<<blocks_of(args.cols, 256), dim3(256), 0, stream>>>(args, down_, row0 == 0, last);
      return hipGetLastError();
    });
  }

 private:
  int dtype_, down_;
  float *partial_ = nullptr, *sums_ = nullptr;
};

// The rows with a target and x's rows of them.
struct Rows {
  int *live, *index, *label;
  Laid x, twice;  // and each row of x twice
};

hipError_t gather(const LossArgs& a, RowsArgs r, bool backward, bool twice, Workspace& ws, Rows& got, hipStream_t stream) {
  const int64_t v = a.dtype == F32::code ? 4 : 8, ld = (a.cols + v - 1) / v * v;
  r.targets = a.targets;
  r.ignore = a.ignore;
  r.rows = static_cast<int>(a.rows);
  r.vocab = static_cast<int>(a.vocab);
  r.live = got.live = a.places != nullptr ? a.places : ws.take<int>(2);
  r.index = got.index = a.places != nullptr ? a.places + 1 : ws.take<int>(a.rows);
  r.label = got.label = ws.take<int>(a.rows);
  GatherArgs g{a.x, a.x_stride, got.live, got.index, ws.take<char>(a.rows * ld * element(a.dtype)),
               twice ? ws.take<char>(2 * a.rows * ld * element(a.dtype)) : nullptr, ld, static_cast<int>(a.cols), a.targets, a.ignore, a.rows, backward ? a.dx : nullptr};
  got.x = {g.out, ld};
  got.twice = {g.twice, ld};
  if (ws.dry()) return hipSuccess;
  if (backward) rows_kernel<true><<<dim3(1), dim3(kRowThreads), 0, stream>>>(r);
  else rows_kernel<false><<<dim3(1), dim3(kRowThreads), 0, stream>>>(r);
  return with_type(a.dtype, [&](auto t) {
    gather_kernel<decltype(t)><<<blocks_of(a.rows, 4), dim3(256), 0, stream>>>(g);
    return hipGetLastError();
  });
}

// A product of the loss; a sum over few results may go in slices.
hipError_t multiply(LossProductArgs& p, const Laid& a, const Laid& b, int dtype, bool a_cols, bool b_cols, Finish finish,
                    Workspace& ws, hipStream_t stream) {
  p.a = a.data;
  p.lda = a.ld;
  p.b = b.data;
  p.ldb = b.ld;
  plan_product(p, dtype, a_cols, b_cols, finish);
  const int64_t groups = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.slices, units = compute_units();
  if (finish == Finish::kSum && !a_cols && p.side_n >= 128 && (p.slices > 1 || p.k > 64) && groups <= 4 * units) {
    // Rows without a target may leave compute units without a tile, and the sum go in more slices.
    p.loss.groups = static_cast<int>(groups);
    p.loss.units = static_cast<int>(units);
    p.partial = ws.take<float>(groups / p.tiles_n * p.side_m * p.n);
  } else if (p.slices > 1) {
    p.partial = ws.take<float>(static_cast<int64_t>(p.slices) * p.m * p.n);
  }
  return ws.dry() ? hipSuccess : launch_product(p, dtype, a_cols, b_cols, stream, finish, &p.loss);
}

// z = x W^T + b of `count` rows and `outs` of the vocabulary.
LossProductArgs logits(const LossArgs& a, const Rows& rows, int64_t row0, int64_t count, int64_t col0, int64_t outs) {
  LossProductArgs p{};
  p.m = static_cast<int>(count);
  p.n = static_cast<int>(outs);
  p.k = static_cast<int>(a.cols);
  p.bias = bytes_on(a.bias, col0 * element(a.bias_dtype));
  p.bias_f32 = a.bias_dtype == F32::code;
  p.loss.live = rows.live;
  p.loss.row0 = static_cast<int>(row0);
  p.loss.label = rows.label + row0;
  p.loss.col0 = static_cast<int>(col0);
  return p;
}

Laid rows_from(const Laid& a, int64_t row, int dtype) { return {bytes_on(a.data, row * a.ld * element(dtype)), a.ld}; }

// Rows of a workgroup that joins their statistics, a power of two.
int lse_rows(int64_t rows) {
  int across = 64;
  while (across > rows || (across > 4 && rows / across < compute_units())) across >>= 1;
  return across;
}

// Rows whose 16-bit gradients come in two parts.  Rounded to one part a result may be off by half a unit in the last
// place of the one term that makes most of it, and its own rounding: over hundreds of rows 1.4 times the latter alone
// in the root mean square, over a few up to twice.  65 to 128 rows take 1.09 to 1.21 times as long in two parts, 200
// 1.14 to 1.27.
constexpr int64_t kTwoParts = 128;
constexpr int64_t kStats = int64_t{1} << 25;  // maxima and sums at a time: 256 MB
// Bytes of exponentials or dz at a time.  Half as many take 1 ms more of 44.7 for 16384 x 4096 into 131072 words: dW's
// sum is read and written for each chunk.
constexpr int64_t kPiece = int64_t{1} << 31;

}  // namespace

hipError_t launch_cross_entropy(const LossArgs& a, void* workspace, int64_t* bytes, hipStream_t stream) {
  Workspace ws(workspace);
  const bool by_row = a.reduction == FH_REDUCE_NONE;
  RowsArgs r{};
  r.losses = by_row ? a.loss : nullptr;
  Rows rows;
  hipError_t err = gather(a, r, false, false, ws, rows, stream);
  Laid w;
  if (err == hipSuccess) err = lay_out(a.weight, a.w_stride, a.vocab, a.cols, a.dtype, ws, w, stream);
  const int64_t groups = (a.vocab + 63) / 64;
  const int64_t most = std::min<int64_t>(std::min<int64_t>(a.rows, most_product_rows(a.vocab)),
                                         std::max<int64_t>(256, kStats / groups / 256 * 256));
  auto* stats = ws.take<float2>(groups * most);
  auto* chosen = ws.take<float>(most);
  auto* rest = ws.take<float>(most);
  float* losses = by_row ? a.loss : ws.take<float>(a.rows);
  const int across = lse_rows(a.rows);
  if (err == hipSuccess) {
    err = in_slices(a.rows, most, [&](int64_t row0, int64_t count) {
      LossProductArgs p = logits(a, rows, row0, count, 0, a.vocab);
      p.loss.stats = stats;
      p.loss.stats_ld = most;
      p.loss.chosen = chosen;
      p.loss.rest = rest;
      const hipError_t e = multiply(p, rows_from(rows.x, row0, a.dtype), w, a.dtype, false, false, Finish::kStats, ws, stream);
      if (e != hipSuccess || ws.dry()) return e;
      const LseArgs l{stats, most, static_cast<int>(groups), static_cast<int>(count), rows.live, static_cast<int>(row0),
                      rows.label + row0, rows.index + row0, chosen, rest, static_cast<float2*>(a.lse) + row0, by_row ? losses : losses + row0, by_row};
      lse_kernel<<<blocks_of(count, across), dim3(1024), 0, stream>>>(l, across);
      return hipGetLastError();
    });
  }
  if (err == hipSuccess && !by_row && !ws.dry()) {
    loss_kernel<<<dim3(1), dim3(1024), 0, stream>>>(losses, rows.live, a.reduction == FH_REDUCE_MEAN, a.loss);
    err = hipGetLastError();
  }
  if (bytes != nullptr) *bytes = ws.used();
  return err;
}

hipError_t launch_cross_entropy_ahead(const LossArgs& a, void* workspace, int64_t* bytes, hipStream_t stream) {
  Workspace ws(workspace);
  Rows rows;
  hipError_t err = gather(a, RowsArgs{}, false, false, ws, rows, stream);
  Laid w;
  if (err == hipSuccess) err = lay_out(a.weight, a.w_stride, a.vocab, a.cols, a.dtype, ws, w, stream);
  if (err != hipSuccess) return err;
  const int64_t groups = (a.vocab + 63) / 64, ld = (a.vocab + 7) / 8 * 8;
  // Rows at a time: 2^18 at most, as slope_kernel's grid has a row for each 64.
  const int64_t most = std::min<int64_t>(
      std::min<int64_t>(std::min<int64_t>(a.rows, 1 << 18), most_product_rows(std::max(a.vocab, a.cols))),
      std::max<int64_t>(256, std::min<int64_t>(kStats / groups, kPiece / (ld * element(a.dtype))) / 256 * 256));
  auto* stats = ws.take<float2>(groups * most);
  auto* chosen = ws.take<float>(most);
  auto* rest = ws.take<float>(most);
  auto* lse = ws.take<float2>(most);
  auto* losses = ws.take<float>(a.rows);
  const Laid dz{ws.take<char>(most * ld * element(a.dtype)), ld};
  auto* db_parts = a.db_sums != nullptr ? ws.take<float>((most + 63) / 64 * ld) : nullptr;
  const int64_t before = ws.used();
  int64_t most_used = before;
  // Products follow one another on the stream, and share the space for what their slices add up to.
  const auto multiply_next = [&](LossProductArgs& p, const Laid& x, const Laid& y, bool a_cols, bool b_cols, Finish finish) {
    Workspace part(bytes_on(workspace, before));
    const hipError_t e = multiply(p, x, y, a.dtype, a_cols, b_cols, finish, part, stream);
    most_used = std::max(most_used, before + part.used());
    return e;
  };
  err = in_slices(a.rows, most, [&](int64_t row0, int64_t count) {
    const Laid x = rows_from(rows.x, row0, a.dtype);
    LossProductArgs p = logits(a, rows, row0, count, 0, a.vocab);
    p.loss.stats = stats;
    p.loss.stats_ld = most;
    p.loss.chosen = chosen;
    p.loss.rest = rest;
    p.loss.ld = ld;
    p.out = const_cast<void*>(dz.data);
    hipError_t e = multiply_next(p, x, w, false, false, Finish::kExp);
    if (e == hipSuccess && !ws.dry()) {
      const int across = lse_rows(count);
      const LseArgs l{stats, most, static_cast<int>(groups), static_cast<int>(count), rows.live, static_cast<int>(row0),
                      rows.label + row0, rows.index + row0, chosen, rest, lse, losses + row0, 0};
      lse_kernel<<<blocks_of(count, across), dim3(1024), 0, stream>>>(l, across);
      const SlopeArgs s{const_cast<void*>(dz.data), ld, stats, most, lse, rows.live, rows.label + row0,
                        static_cast<int>(row0), static_cast<int>(count), db_parts};
      e = with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        const dim3 grid(blocks_of(ld, 64 * kVec<T>).x, blocks_of(count, 64).x);
        slope_kernel<T><<<grid, dim3(256), 0, stream>>>(s);
        return hipGetLastError();
      });
      if (e == hipSuccess && db_parts != nullptr) {
        join_rows_kernel<<<blocks_of(a.vocab, 256), dim3(256), 0, stream>>>(
            db_parts, rows.live, static_cast<int>(row0), static_cast<int>(count), static_cast<int>(ld),
            static_cast<int>(a.vocab), a.db_sums);
        e = hipGetLastError();
      }
    }
    LossProductArgs s{};
    s.loss.live = rows.live;
    s.loss.row0 = static_cast<int>(row0);
    s.n = static_cast<int>(a.cols);
    if (e == hipSuccess && a.dx_sums != nullptr) {
      LossProductArgs q = s;
      q.m = static_cast<int>(count);
      q.k = static_cast<int>(a.vocab);
      q.loss.sums = a.dx_sums + row0 * a.cols;
      q.loss.first = 1;
      e = multiply_next(q, dz, w, false, true, Finish::kSum);
    }
    if (e == hipSuccess && a.dw_sums != nullptr) {
      LossProductArgs q = s;
      q.m = static_cast<int>(a.vocab);
      q.k = static_cast<int>(count);
      q.loss.sums = a.dw_sums;
      q.loss.first = row0 == 0;
      e = multiply_next(q, dz, x, true, true, Finish::kSum);
    }
    return e;
  });
  if (err == hipSuccess && !ws.dry()) {
    loss_kernel<<<dim3(1), dim3(1024), 0, stream>>>(losses, rows.live, a.reduction == FH_REDUCE_MEAN, a.loss);
    err = hipGetLastError();
  }
  if (bytes != nullptr) *bytes = most_used;
  return err;
}

hipError_t launch_cross_entropy_scale(const LossArgs& a, hipStream_t stream) {
  ScaleArgs s{};
  s.live = a.places;
  s.grad = a.grad;
  s.mean = a.reduction == FH_REDUCE_MEAN;
  s.factor = a.dtype == F16::code ? 1.f / kKept : 1.f;
  const auto scale = [&](int64_t rows, int64_t cols, const float* sums, const int* index, void* out, int dtype) {
    s.rows = rows;
    s.cols = static_cast<int>(cols);
    s.sums = sums;
    s.index = index;
    s.out = out;
    return with_type(dtype, [&](auto t) {
      const int64_t across = rows >= 4 * compute_units() ? 1 : std::min<int64_t>((cols + 511) / 512, 1024);
      scale_kernel<decltype(t)><<<dim3(blocks_of(rows, 4).x, static_cast<uint32_t>(across)), dim3(256), 0, stream>>>(s);
      return hipGetLastError();
    });
  };
  s.targets = a.targets;
  s.ignore = a.ignore;
  hipError_t err = hipSuccess;
  if (a.dx != nullptr) err = scale(a.rows, a.cols, a.dx_sums, a.places + 1, a.dx, a.dtype);
  if (err == hipSuccess && a.dweight != nullptr) err = scale(a.vocab, a.cols, a.dw_sums, nullptr, a.dweight, a.dtype);
  if (err == hipSuccess && a.dbias != nullptr) err = scale(1, a.vocab, a.db_sums, nullptr, a.dbias, a.bias_dtype);
  return err;
}

hipError_t launch_cross_entropy_backward(const LossArgs& a, void* workspace, int64_t* bytes, hipStream_t stream) {
  Workspace ws(workspace);
  // Few rows' gradients in two parts of 16 bits each, for as many rows more: the products are bound by reading the
  // weight and writing its gradient.
  const int parts = a.dtype != F32::code && a.rows <= kTwoParts ? 2 : 1;
  RowsArgs r{};
  r.grad = a.grad;
  r.per_row = a.reduction == FH_REDUCE_NONE;
  r.mean = a.reduction == FH_REDUCE_MEAN;
  r.scaled = a.dtype == F16::code;
  r.lse = static_cast<const float2*>(a.lse);
  r.row = ws.take<float4>(a.rows);
  r.scale = ws.take<float>(1);
  Rows rows;
  hipError_t err = gather(a, r, true, parts == 2 && a.dweight != nullptr, ws, rows, stream);
  Laid w;
  if (err == hipSuccess) err = lay_out(a.weight, a.w_stride, a.vocab, a.cols, a.dtype, ws, w, stream);
  if (err != hipSuccess) return err;
  const int es = element(a.dtype);
  // Pieces of the vocabulary, as even as whole tiles allow, for at most 65536 rows at a time.
  const int64_t most_rows = std::min<int64_t>(std::min<int64_t>(a.rows, 1 << 16), most_product_rows(a.cols));
  int64_t piece = std::min<int64_t>(std::min<int64_t>(a.vocab, std::max<int64_t>(1024, kPiece / (most_rows * es))),
                                    most_product_rows(std::max(a.cols, most_rows)));
  const int64_t pieces = (a.vocab + piece - 1) / piece;
  piece = std::min<int64_t>(a.vocab, ((a.vocab + pieces - 1) / pieces + 255) / 256 * 256);
  const int64_t ld = (piece + 7) / 8 * 8, chunks = (a.rows + most_rows - 1) / most_rows;
  const Laid dz{ws.take<char>(parts * most_rows * ld * es), ld};
  auto* dx_sums = a.dx != nullptr && (parts == 2 || piece < a.vocab) ? ws.take<float>(parts * a.rows * a.cols) : nullptr;
  auto* dw_sums = a.dweight != nullptr && chunks > 1 ? ws.take<float>(piece * a.cols) : nullptr;
  const BiasSums db(a.dbias != nullptr, chunks, parts * most_rows, piece, a.dtype, ws);
  // Products follow one another on the stream, and share the space for what their slices add up to.
  const int64_t before = ws.used();
  int64_t most_used = before;
  const auto shared = [&](auto call) {
    Workspace part(bytes_on(workspace, before));
    const hipError_t e = call(part);
    most_used = std::max(most_used, before + part.used());
    return e;
  };
  if (err == hipSuccess) {
    err = in_slices(a.vocab, piece, [&](int64_t col0, int64_t outs) {
      const Laid wp = rows_from(w, col0, a.dtype);
      BiasArgs db_args{};
      db_args.cols = static_cast<int>(outs);
      db_args.live = rows.live + (parts - 1);
      db_args.scale = r.scale;
      db_args.out = bytes_on(a.dbias, col0 * element(a.bias_dtype));
      db_args.out_f32 = a.bias_dtype == F32::code;
      return in_slices(a.rows, most_rows, [&](int64_t row0, int64_t count) {
        const Laid xp = rows_from(rows.x, row0, a.dtype);
        hipError_t e = shared([&](Workspace& part) {
          LossProductArgs p = logits(a, rows, row0, count, col0, outs);
          p.loss.row = r.row + row0;
          p.loss.parts = parts;
          p.loss.ld = (outs + 7) / 8 * 8;
          p.out = const_cast<void*>(dz.data);
          return multiply(p, xp, wp, a.dtype, false, false, Finish::kSlope, part, stream);
        });
        const Laid d{dz.data, (outs + 7) / 8 * 8};
        LossProductArgs s{};
        s.loss.live = rows.live + (parts - 1);  // two parts: twice the rows
        s.loss.row0 = static_cast<int>(row0);
        s.loss.scale = r.scale;
        if (e == hipSuccess && a.dx != nullptr) {
          e = shared([&](Workspace& part) {
            LossProductArgs p = s;
            p.m = static_cast<int>(parts * count);
            p.n = static_cast<int>(a.cols);
            p.k = static_cast<int>(outs);
            p.loss.sums = dx_sums != nullptr ? dx_sums + row0 * a.cols : nullptr;
            p.loss.first = col0 == 0;
            p.loss.last = parts == 1 && col0 + outs == a.vocab;
            p.loss.index = rows.index + row0;
            p.out = a.dx;
            return multiply(p, d, wp, a.dtype, false, true, Finish::kSum, part, stream);
          });
        }
        if (e == hipSuccess && a.dweight != nullptr) {
          e = shared([&](Workspace& part) {
            LossProductArgs p = s;
            p.m = static_cast<int>(outs);
            p.n = static_cast<int>(a.cols);
            p.k = static_cast<int>(parts * count);
            p.loss.sums = dw_sums;
            p.loss.first = row0 == 0;
            p.loss.last = row0 + count == a.rows;
            p.out = bytes_on(a.dweight, col0 * a.cols * es);
            return multiply(p, d, parts == 2 ? rows.twice : xp, a.dtype, true, true, Finish::kSum, part, stream);
          });
        }
        if (e == hipSuccess && a.dbias != nullptr && !ws.dry())
          e = db.add(db_args, d, row0, parts * count, row0 + count == a.rows, stream);
        return e;
      });
    });
  }
  if (err == hipSuccess && a.dx != nullptr && parts == 2 && !ws.dry()) {
    err = with_half_type(a.dtype, [&](auto t) {
      parts_kernel<decltype(t)><<<blocks_of(a.rows, 4), dim3(256), 0, stream>>>(
          dx_sums, rows.live, rows.index, r.scale, static_cast<int>(a.cols), a.dx);
      return hipGetLastError();
    });
  }
  if (bytes != nullptr) *bytes = most_used;
  return err;
}

}  // namespace fh
