// Rows of a table, scaled and copied into the residual streams, and the table's gradient:
//   y[i, s] = scale W[t_i],   dW[v] = scale (sum over i with t_i = v, in their order, over s of g[i, s]).
//
// Both move memory and nothing else.  The forward reads a row once for all streams.
//
// The gradient sorts the tokens (stably, by radix: up to 4096 in one workgroup's LDS, more in
// tiles through memory), so that a row's terms are neighbours.  The sorted places go in chunks, a
// wavefront to a chunk and a strip of columns, which adds up the runs of equal tokens.  A run that
// lies in one chunk is written at once; the parts of one that goes over several, FP32, are joined
// by another kernel in their order.  Rows whose token does not occur are zeros, written beside
// that.  Up to 2048 tokens are not sorted: each workgroup looks for its rows'.  Sums are FP32, in the
// tokens' order within a chunk and chunk by chunk, and rounded once; nothing depends on the order in
// which workgroups run.
//
// 16384 tokens of 4096 bf16 columns in four streams, 131072 words: forward 137 us (671 MB, 4.9 TB/s), the
// gradient's sums and zeros 320 (1.6 GB, 5.0 TB/s), the sort before it 22 and the joining after it 10.
#include <algorithm>

#include "fh_plan.h"
#include "fh_kernels.h"
#include "fh_vec.h"
#include "workspace.h"

namespace fh {
namespace {

// Four tokens a workgroup, a wavefront and Vectors vectors a lane to each; blockIdx.y strips of columns.
constexpr int kVectors = 2;
template <typename T>
__global__ __launch_bounds__(256) void embedding_kernel(EmbeddingArgs a) {
  using S = typename T::storage;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (i >= a.count) return;
  const int cols = static_cast<int>(a.cols);
  const int c = (static_cast<int>(blockIdx.y) * kVectors * 64 + (threadIdx.x & 63)) * kVec<T>;
  const int64_t token = a.tokens[i];
  // A token out of range, which only a wait for the device could report, gives NaN.
  const bool valid = token >= 0 && token < a.vocab;
  const S* from = static_cast<const S*>(a.weight) + (valid ? token : 0) * a.w_stride;
  U32x4 w[kVectors];
#pragma unroll
  for (int u = 0; u < kVectors; ++u) w[u] = load_row<T>(from, c + u * 64 * kVec<T>, cols);
  if (a.scale != 1.f || !valid) {
#pragma unroll
    for (int u = 0; u < kVectors; ++u) {
      float f[kVec<T>];
      to_floats<T>(w[u], f);
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) f[k] = valid ? f[k] * a.scale : __builtin_nanf("");
      w[u] = from_floats<T>(f);
    }
  }
  S* to = static_cast<S*>(a.out) + i * a.streams * a.cols;
  for (int s = 0; s < a.streams; ++s, to += a.cols) {
#pragma unroll
    for (int u = 0; u < kVectors; ++u) store_row<T>(w[u], to, c + u * 64 * kVec<T>, cols);
  }
}

// ---- sorting -------------------------------------------------------------------------

constexpr int kThreads = 1024, kWaves = kThreads / 64;

// A token's key: itself, or the first number past the vocabulary where it has no gradient.
__device__ __forceinline__ uint32_t key_of(const EmbeddingArgs& a, int64_t i) {
  const int64_t t = a.tokens[i];
  return static_cast<uint32_t>(t >= 0 && t < a.vocab && t != a.padding ? t : a.vocab);
}

// Exclusive sums of `Each` counts a thread, in the threads' order.
template <int Each>
__device__ __forceinline__ void scan(uint32_t (&v)[Each], uint32_t (&area)[kWaves]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t sum = 0;
#pragma unroll
  for (int e = 0; e < Each; ++e) {
    const uint32_t mine = v[e];
    v[e] = sum;
    sum += mine;
  }
  uint32_t upto = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t other = __shfl_up(upto, d);
    if (lane >= d) upto += other;
  }
  if (lane == 63) area[wave] = upto;
  __syncthreads();
  uint32_t base = upto - sum;
  for (int w = 0; w < wave; ++w) base += area[w];
#pragma unroll
  for (int e = 0; e < Each; ++e) v[e] += base;
}

// A tile's places in the order of Bits bits of its keys, equal ones as they were.  Wavefront
// w holds keys 64 P w .. 64 P (w + 1) - 1, 64 at a time.  Afterwards counts[digit][wave] is the
// place of that wavefront's first key with that digit.
template <int P, int Bits>
__device__ __forceinline__ void rank(const uint32_t (&key)[P], int shift, uint32_t (&place)[P],
                                     uint32_t (&counts)[kWaves << Bits], uint32_t (&area)[kWaves]) {
  constexpr int each = (kWaves << Bits) / kThreads;
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int e = 0; e < each; ++e) counts[e * kThreads + threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const uint32_t digit = key[i] >> shift & ((1u << Bits) - 1);
    uint64_t peers = ~uint64_t{0};
#pragma unroll
    for (int b = 0; b < Bits; ++b) {
      const bool set = digit >> b & 1;
      const uint64_t those = __ballot(set);
      peers &= set ? those : ~those;
    }
    uint32_t* count = counts + digit * kWaves + wave;
    const uint32_t before = *reinterpret_cast<volatile uint32_t*>(count);
    const int below = lanes_below(peers);
    place[i] = before + below;
    if (below == 0) *reinterpret_cast<volatile uint32_t*>(count) = before + __popcll(peers);
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  uint32_t v[each];
#pragma unroll
  for (int e = 0; e < each; ++e) v[e] = counts[threadIdx.x * each + e];
  scan<each>(v, area);
#pragma unroll
  for (int e = 0; e < each; ++e) counts[threadIdx.x * each + e] = v[e];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < P; ++i) place[i] += counts[(key[i] >> shift & ((1u << Bits) - 1)) * kWaves + wave];
}

// Up to 4096 tokens, in one workgroup: 13 us in three passes (2^18 words), where the four launches below take 20.
// (16384 took 44 so.)
constexpr int kMostAlone = 4 * kThreads;
__global__ __launch_bounds__(kThreads) void sort_tile_kernel(EmbeddingArgs a, int bits, uint32_t* keys, int* order) {
  constexpr int P = kMostAlone / kThreads, kBits = 6;
  __shared__ uint32_t counts[kWaves << kBits], area[kWaves], moved[P * kThreads];
  __shared__ uint16_t from[P * kThreads];
  const int first = (threadIdx.x >> 6) * 64 * P + (threadIdx.x & 63), count = static_cast<int>(a.count);
  uint32_t key[P], at[P], place[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    at[i] = first + 64 * i;
    key[i] = first + 64 * i < count ? key_of(a, first + 64 * i) : ~0u;  // past the last: they stay behind
  }
  for (int shift = 0; shift < bits; shift += kBits) {
    rank<P, kBits>(key, shift, place, counts, area);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      moved[place[i]] = key[i];
      from[place[i]] = static_cast<uint16_t>(at[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < P; ++i) {
      key[i] = moved[first + 64 * i];
      at[i] = from[first + 64 * i];
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (first + 64 * i >= count) continue;
    keys[first + 64 * i] = key[i];
    order[first + 64 * i] = static_cast<int>(at[i]);
  }
}

// Several tiles, a count and a move for each digit.  Tiles of 1024 keys while there are at most 64 of them, as each
// workgroup adds up the counts of all: 16384 tokens sort in 20 us, 131072, in 32 tiles of 4096, in 36 (in tiles
// of 16384, on eight compute units, 92), 600000, in tiles of 16384, in 95.  That addition goes by the square of the
// tiles: 2^22 tokens take 0.23 ms in two passes, 2^24 1.1, 2^26 8.8 and 2^27 27.
constexpr int kDigit = 9;  // bits of a pass

// keys null: the tokens themselves.
__device__ __forceinline__ uint32_t key_at(const EmbeddingArgs& a, const uint32_t* keys, int64_t i) {
  return keys != nullptr ? keys[i] : key_of(a, i);
}

// How often each digit occurs in each tile: table[tile][digit].
__global__ __launch_bounds__(kThreads) void count_kernel(EmbeddingArgs a, int tile, const uint32_t* keys, int shift,
                                                         uint32_t* table) {
  __shared__ uint32_t counts[1 << kDigit];
  for (int d = threadIdx.x; d < 1 << kDigit; d += kThreads) counts[d] = 0;
  __syncthreads();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * tile;
  for (int i = threadIdx.x; i < tile && first + i < a.count; i += kThreads)
    atomicAdd(counts + (key_at(a, keys, first + i) >> shift & ((1u << kDigit) - 1)), 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < 1 << kDigit; d += kThreads) table[(static_cast<int64_t>(blockIdx.x) << kDigit) + d] = counts[d];
}

// Moves a tile's 1024 P keys to their places in the whole.
template <int P>
__global__ __launch_bounds__(kThreads) void move_kernel(EmbeddingArgs a, const uint32_t* keys, const int* order,
                                                        int shift, const uint32_t* table, uint32_t* to_keys,
                                                        int* to_order) {
  constexpr int kDigits = 1 << kDigit;
  __shared__ uint32_t counts[kWaves << kDigit], area[kWaves], base[kDigits], other[kWaves];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (P * kThreads);
  const int at = (threadIdx.x >> 6) * 64 * P + (threadIdx.x & 63);
  // A digit's place: after the smaller digits of all tiles and this one of the tiles before.
  uint32_t all[1] = {0}, before = 0;
  if (threadIdx.x < kDigits) {
#pragma unroll 16
    for (uint32_t tile = 0; tile < gridDim.x; ++tile) {
      const uint32_t n = table[(static_cast<int64_t>(tile) << kDigit) + threadIdx.x];
      before += tile < blockIdx.x ? n : 0;
      all[0] += n;
    }
  }
  scan<1>(all, other);
  if (threadIdx.x < kDigits) base[threadIdx.x] = all[0] + before;
  uint32_t key[P], place[P];
#pragma unroll
  for (int i = 0; i < P; ++i) key[i] = first + at + 64 * i < a.count ? key_at(a, keys, first + at + 64 * i) : ~0u;
  rank<P, kDigit>(key, shift, place, counts, area);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int64_t from = first + at + 64 * i;
    if (from >= a.count) continue;
    const uint32_t digit = key[i] >> shift & (kDigits - 1);
    const uint32_t to = base[digit] + place[i] - counts[digit * kWaves];
    to_keys[to] = key[i];
    to_order[to] = order != nullptr ? order[from] : static_cast<int>(from);
  }
}

// ---- sums ----------------------------------------------------------------------------

struct SumArgs {
  EmbeddingArgs a;
  const uint32_t* keys;  // [count], sorted
  const int* order;      // [count]
  float* partial;        // [chunks, 2, cols]: of the run that goes on from the chunk before, and that goes on after
  int chunk, chunks, strips, summing;  // summing: workgroups that do not write zeros
};

template <typename T>
__device__ __forceinline__ void put(const SumArgs& p, float (&f)[kVec<T>], uint32_t key, int c) {
#pragma unroll
  for (int k = 0; k < kVec<T>; ++k) f[k] *= p.a.scale;
  store_row<T>(from_floats<T>(f), static_cast<typename T::storage*>(p.a.out) + key * p.a.cols, c,
               static_cast<int>(p.a.cols));
}

template <int V>
__device__ __forceinline__ void keep(const SumArgs& p, const float (&f)[V], int64_t chunk, int which, int c) {
  float* to = p.partial + (chunk * 2 + which) * p.a.cols;
  if (c + V <= p.a.cols) {
    __builtin_memcpy(to + c, f, sizeof(f));
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (c + k < p.a.cols) to[c + k] = f[k];
  }
}

// A row of the table whose token does not occur: 64 rows a workgroup.
template <typename T>
__device__ __forceinline__ void write_zeros(const SumArgs& p, int64_t first) {
  const int lane = threadIdx.x & 63, cols = static_cast<int>(p.a.cols);
  const int64_t row = first + lane;
  int64_t low = 0, high = p.a.count;
  while (low < high) {
    const int64_t mid = (low + high) / 2;
    if (p.keys[mid] < static_cast<uint32_t>(row)) low = mid + 1;
    else high = mid;
  }
  const bool here = row >= p.a.vocab || (low < p.a.count && p.keys[low] == static_cast<uint32_t>(row));
  for (uint64_t left = ~__ballot(here) >> (threadIdx.x >> 6) & 0x1111111111111111ull; left != 0; left &= left - 1) {
    auto* to = static_cast<typename T::storage*>(p.a.out) +
               (first + (threadIdx.x >> 6) + __ffsll(static_cast<unsigned long long>(left)) - 1) * p.a.cols;
    for (int c = lane * kVec<T>; c < cols; c += 64 * kVec<T>) store_row<T>(U32x4{0, 0, 0, 0}, to, c, cols);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void sum_kernel(SumArgs p) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, kAhead = 8;
  if (static_cast<int>(blockIdx.x) >= p.summing) {
    write_zeros<T>(p, (static_cast<int64_t>(blockIdx.x) - p.summing) * 64);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int unit = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x) * 4 + (threadIdx.x >> 6));
  const int64_t chunk = unit / p.strips;
  if (chunk >= p.chunks) return;
  const int c = (unit % p.strips * 64 + lane) * V, cols = static_cast<int>(p.a.cols);
  const int64_t first = chunk * p.chunk;
  const int count = static_cast<int>(p.a.count - first < p.chunk ? p.a.count - first : p.chunk);
  const uint32_t none = static_cast<uint32_t>(p.a.vocab);
  // The chunk's keys and rows, one a lane.
  const uint32_t my_key = lane < count ? p.keys[first + lane] : none;
  const int my_row = lane < count ? p.order[first + lane] : 0;
  const uint32_t before = first > 0 ? p.keys[first - 1] : none, after = first + count < p.a.count ? p.keys[first + count] : none;
  const int valid = __popcll(__ballot(my_key != none));  // those without a gradient come last
  if (valid == 0) return;
  uint32_t key = __builtin_amdgcn_readlane(my_key, 0);
  bool goes_on = key == before;
  float sum[V] = {};
  const int streams = p.a.streams, items = valid * streams;
  int place = 0, stream = 0;  // of the next load
  int at = 0, step = 0;       // of the next addition
  for (int i = 0; i < items; i += kAhead) {
    U32x4 raw[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i + u >= items) break;
      const int64_t row = static_cast<int64_t>(__builtin_amdgcn_readlane(my_row, place)) * streams + stream;
      raw[u] = load_row<T>(static_cast<const S*>(p.a.grad) + row * p.a.g_stride, c, cols);
      if (++stream == streams) {
        stream = 0;
        ++place;
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i + u >= items) break;
      if (step == 0) {
        const uint32_t next = __builtin_amdgcn_readlane(my_key, at);
        if (next != key) {
          if (goes_on) keep(p, sum, chunk, 0, c);
          else put<T>(p, sum, key, c);
          goes_on = false;
          key = next;
#pragma unroll
          for (int k = 0; k < V; ++k) sum[k] = 0.f;
        }
      }
      float f[V];
      to_floats<T>(raw[u], f);
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] += f[k];
      if (++step == streams) {
        step = 0;
        ++at;
      }
    }
  }
  if (goes_on) keep(p, sum, chunk, 0, c);
  else if (valid == count && after == key) keep(p, sum, chunk, 1, c);
  else put<T>(p, sum, key, c);
}

// The first place from `low` on whose key is above `key`, by a wavefront that asks 64 places at a time.
__device__ __forceinline__ int64_t end_of_run(const uint32_t* keys, int64_t low, int64_t high, uint32_t key) {
  while (low < high) {
    const int64_t step = (high - low + 63) / 64, at = low + (threadIdx.x & 63) * step;
    const int within = __popcll(__ballot(at < high && keys[at] <= key));  // of the places asked, in a row
    if (within == 0) return low;
    const int64_t last = low + (within - 1) * step;
    high = last + step < high ? last + step : high;
    low = last + 1;
  }
  return low;
}

// Runs over several chunks, by the chunk in which they begin: its part and those of the chunks after it, in
// order, an eighth of them a wavefront.
constexpr int kJoining = 8;
template <typename T>
__global__ __launch_bounds__(64 * kJoining) void join_runs_kernel(SumArgs p) {
  constexpr int V = kVec<T>, kAhead = 8;
  __shared__ float area[kJoining][V][64];
  const int64_t chunk = blockIdx.x / p.strips, first = chunk * p.chunk, end = first + p.chunk;
  if (end >= p.a.count) return;
  const uint32_t key = p.keys[end - 1];
  if (key >= static_cast<uint32_t>(p.a.vocab) || p.keys[end] != key || (first > 0 && p.keys[first - 1] == key)) return;
  const int64_t last = end_of_run(p.keys, end, p.a.count, key) - 1;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = (static_cast<int>(blockIdx.x) % p.strips * 64 + lane) * V, cols = static_cast<int>(p.a.cols);
  const int64_t parts = last / p.chunk - chunk + 1, to = parts * (wave + 1) / kJoining;
  float sum[V] = {};
  for (int64_t i = parts * wave / kJoining; i < to; i += kAhead) {
    float f[kAhead][V];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i + u >= to) break;
      const float* row = p.partial + ((chunk + i + u) * 2 + (i + u == 0 ? 1 : 0)) * p.a.cols;
      if (c + V <= cols) {
        __builtin_memcpy(f[u], row + c, sizeof(f[u]));
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) f[u][k] = c + k < cols ? row[c + k] : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i + u >= to) break;
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] += f[u][k];
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) area[wave][k][lane] = sum[k];
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    sum[k] = area[0][k][lane];
#pragma unroll
    for (int w = 1; w < kJoining; ++w) sum[k] += area[w][k][lane];
  }
  put<T>(p, sum, key, c);
}

// ---- few tokens ------------------------------------------------------------------------

constexpr int kFew = 2048, kRows = 64, kLong = 32;

// A wavefront's tokens in a block of rows: place and row of each, in their order.
struct Found {
  const uint32_t* list;
  int count;
};

// Adds the gradients of the tokens that are row `r`.
template <typename T>
__device__ __forceinline__ void add_found(const EmbeddingArgs& a, const Found& found, uint32_t r, int c,
                                          float (&sum)[kVec<T>]) {
  using S = typename T::storage;
  constexpr int V = kVec<T>, kAhead = 8;
  const int lane = threadIdx.x & 63, cols = static_cast<int>(a.cols);
  for (int base = 0; base < found.count; base += 64) {
    const uint32_t entry = base + lane < found.count ? found.list[base + lane] : ~0u;
    uint64_t left = __ballot(entry >> 16 == r);
    int stream = 0;
    while (left != 0) {
      U32x4 raw[kAhead];
      int loaded = 0;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (left == 0) break;
        const int at = __builtin_amdgcn_readlane(entry, __ffsll(static_cast<unsigned long long>(left)) - 1) & 0xFFFF;
        raw[u] = load_row<T>(static_cast<const S*>(a.grad) + (static_cast<int64_t>(at) * a.streams + stream) * a.g_stride,
                             c, cols);
        ++loaded;
        if (++stream == a.streams) {
          stream = 0;
          left &= left - 1;
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (u >= loaded) break;
        float f[V];
        to_floats<T>(raw[u], f);
#pragma unroll
        for (int k = 0; k < V; ++k) sum[k] += f[k];
      }
    }
  }
}

// By a workgroup's 256 threads, in lines of 128 bytes.
template <typename S>
__device__ __forceinline__ void fill_zeros(S* to, int64_t count) {
  constexpr int kLine = 128 / sizeof(S);
  const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(to) % 128 / sizeof(S));
  const int64_t begin = (kLine - off) % kLine < count ? (kLine - off) % kLine : count;
  const int64_t end = begin + (count - begin) / (16 / sizeof(S)) * (16 / sizeof(S));
  const int t = static_cast<int>(threadIdx.x);
  if (t < begin) to[t] = S{};
  for (int64_t i = begin + t * (16 / sizeof(S)); i < end; i += 256 * (16 / sizeof(S)))
    *reinterpret_cast<U32x4*>(to + i) = U32x4{0, 0, 0, 0};
  if (t < count - end) to[end + t] = S{};
}

// The gradient for up to 2048 tokens, in one launch where sorting takes two more: every workgroup looks
// through the tokens itself, adds up those of up to 64 rows, 2^shift apart, in a strip of columns, and
// writes the zeros of up to 64 rows in a row.  (The frequent words of a vocabulary in the order of their
// frequency are neighbours: sums of 64 rows in a row left most of the work to one workgroup, 90 us.  And
// zeros of single rows far apart are written in part lines: FP32 735 tokens into 127539 x 450 took 81 us,
// 164 into 25344 x 2195 71, now 49 and 44, filling as much memory alone 29 to 38.)  A wavefront to a row,
// all four to one that occurs often; each die takes neighbouring rows.
template <typename T>
__global__ __launch_bounds__(256) void few_kernel(EmbeddingArgs a, int strips, int shift) {
  constexpr int V = kVec<T>;
  __shared__ uint32_t list[4][kFew / 4], often[kRows], counts[4], there[2];
  __shared__ float area[4][V][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t die = blockIdx.x % 8, each = gridDim.x / 8, more = gridDim.x % 8;
  const uint32_t at = die * each + (die < more ? die : more) + blockIdx.x / 8;
  const uint32_t first = at / strips, apart = 1u << shift;
  const int c = (static_cast<int>(at % strips) * 64 + lane) * V, cols = static_cast<int>(a.cols);
  const int64_t zero = a.vocab * at / gridDim.x;
  const uint32_t zeros = static_cast<uint32_t>(a.vocab * (at + 1) / gridDim.x - zero);
  if (threadIdx.x < kRows) often[threadIdx.x] = 0;
  if (threadIdx.x < 2) there[threadIdx.x] = 0;
  __syncthreads();
  const int begin = static_cast<int>(a.count * wave / 4), end = static_cast<int>(a.count * (wave + 1) / 4);
  constexpr int kTurns = kFew / 4 / 64;
  uint32_t keys[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int place = begin + 64 * i + lane;
    keys[i] = place < end ? key_of(a, place) : static_cast<uint32_t>(a.vocab);
  }
  int count = 0;
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const uint32_t row = keys[i] >> shift;
    const bool mine = keys[i] < a.vocab && (keys[i] & (apart - 1)) == first;
    const uint64_t those = __ballot(mine);
    if (mine) {
      list[wave][count + lanes_below(those)] = row << 16 | static_cast<uint32_t>(begin + 64 * i + lane);
      atomicAdd(often + row, 1u);
    }
    count += __popcll(those);
    const uint32_t bit = keys[i] - static_cast<uint32_t>(zero);
    if (bit < zeros) atomicOr(there + (bit >> 5), 1u << (bit & 31));
  }
  if (lane == 0) counts[wave] = count;
  __syncthreads();
  using S = typename T::storage;
  const auto write = [&](int r, float (&sum)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) sum[k] *= a.scale;
    store_row<T>(from_floats<T>(sum), static_cast<S*>(a.out) + (first + (static_cast<int64_t>(r) << shift)) * a.cols,
                 c, cols);
  };
  const uint32_t times = often[lane];
  const uint64_t here = __ballot(times != 0), many = __ballot(times >= kLong);
  for (uint64_t left = here & ~many & 0x1111111111111111ull << wave; left != 0; left &= left - 1) {
    const int r = __ffsll(static_cast<unsigned long long>(left)) - 1;
    float sum[V] = {};
    for (int w = 0; w < 4; ++w) add_found<T>(a, {list[w], static_cast<int>(counts[w])}, r, c, sum);
    write(r, sum);
  }
  for (uint64_t left = many; left != 0; left &= left - 1) {
    const int r = __ffsll(static_cast<unsigned long long>(left)) - 1;
    float sum[V] = {};
    add_found<T>(a, {list[wave], count}, r, c, sum);
#pragma unroll
    for (int k = 0; k < V; ++k) area[wave][k][lane] = sum[k];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] = ((area[0][k][lane] + area[1][k][lane]) + area[2][k][lane]) + area[3][k][lane];
      write(r, sum);
    }
    __syncthreads();
  }
  // Runs of rows that do not occur.
  uint64_t left = ~(static_cast<uint64_t>(there[1]) << 32 | there[0]);
  if (zeros < 64) left &= (uint64_t{1} << zeros) - 1;
  while (left != 0) {
    const int r = __ffsll(static_cast<unsigned long long>(left)) - 1;
    const uint64_t rest = ~(left >> r);  // zero for 64 rows
    const int run = rest != 0 ? __ffsll(static_cast<unsigned long long>(rest)) - 1 : 64;
    fill_zeros(static_cast<S*>(a.out) + (zero + r) * a.cols, run * a.cols);
    left = run + r < 64 ? left & ~uint64_t{0} << (run + r) : 0;
  }
}

dim3 blocks_of(int64_t items, int64_t each) { return dim3(static_cast<uint32_t>((items + each - 1) / each)); }

// The keys in `keys` and `order` afterwards, through another pair.
hipError_t sort_tokens(const EmbeddingArgs& a, Workspace& ws, uint32_t*& keys, int*& order, hipStream_t stream) {
  keys = ws.take<uint32_t>(a.count);
  order = ws.take<int>(a.count);
  int bits = 1;
  while (a.vocab >> bits != 0) ++bits;  // of the vocabulary's size, the last key
  if (a.count <= kMostAlone) {
    if (ws.dry()) return hipSuccess;
    sort_tile_kernel<<<dim3(1), dim3(kThreads), 0, stream>>>(a, bits, keys, order);
    return hipGetLastError();
  }
  auto* other_keys = ws.take<uint32_t>(a.count);
  auto* other_order = ws.take<int>(a.count);
  const int each = a.count <= 64 * kThreads ? 1 : a.count <= 512 * kThreads ? 4 : 16;
  const int tile = each * kThreads;
  const dim3 tiles = blocks_of(a.count, tile), block(kThreads);
  auto* table = ws.take<uint32_t>(static_cast<int64_t>(tiles.x) << kDigit);
  if (ws.dry()) return hipSuccess;
  for (int shift = 0; shift < bits; shift += kDigit) {
    const uint32_t* from = shift > 0 ? keys : nullptr;
    const int* places = shift > 0 ? order : nullptr;
    count_kernel<<<tiles, block, 0, stream>>>(a, tile, from, shift, table);
    if (each == 1) move_kernel<1><<<tiles, block, 0, stream>>>(a, from, places, shift, table, other_keys, other_order);
    else if (each == 4) move_kernel<4><<<tiles, block, 0, stream>>>(a, from, places, shift, table, other_keys, other_order);
    else move_kernel<16><<<tiles, block, 0, stream>>>(a, from, places, shift, table, other_keys, other_order);
    std::swap(keys, other_keys);
    std::swap(order, other_order);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_embedding(const EmbeddingArgs& a, int dtype, hipStream_t stream) {
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const int64_t across = kVectors * 64 * kVec<T>;
    return in_slices(a.count, most_groups(256) * 4, [&](int64_t first, int64_t count) {
      EmbeddingArgs part = a;
      part.count = count;
      part.tokens = a.tokens + first;
      part.out = static_cast<typename T::storage*>(a.out) + first * a.streams * a.cols;
      const dim3 grid(static_cast<uint32_t>((count + 3) / 4), static_cast<uint32_t>((a.cols + across - 1) / across));
      embedding_kernel<T><<<grid, dim3(256), 0, stream>>>(part);
      return hipGetLastError();
    });
  });
}

hipError_t launch_embedding_backward(const EmbeddingArgs& a, int dtype, void* workspace, int64_t* bytes,
                                     hipStream_t stream) {
  const int64_t strip = 64 * (dtype == F32::code ? 4 : 8), strips = (a.cols + strip - 1) / strip;
  int shift = 0;
  while ((int64_t{kRows} << shift) < a.vocab) ++shift;
  // Two workgroups a compute unit, down to four rows in each: FP16 gradients of 1711 tokens of 2 x 1079 into 872 rows
  // take 15 us, with 64 rows in each 66.
  while ((int64_t{4} << shift) < a.vocab && (int64_t{1} << shift) * strips < 2 * compute_units()) ++shift;
  const int64_t few = std::min<int64_t>(int64_t{1} << shift, a.vocab) * strips;
  if (a.count <= kFew && few <= most_groups(256)) {
    if (bytes != nullptr) *bytes = 0;
    if (workspace == nullptr) return hipSuccess;
    return with_type(dtype, [&](auto t) {
      few_kernel<decltype(t)>
          <<<dim3(static_cast<uint32_t>(few)), dim3(256), 0, stream>>>(a, static_cast<int>(strips), shift);
      return hipGetLastError();
    });
  }
  Workspace ws(workspace);
  SumArgs p{};
  p.a = a;
  uint32_t* keys = nullptr;
  int* order = nullptr;
  hipError_t err = a.count > 0 ? sort_tokens(a, ws, keys, order, stream) : hipSuccess;
  if (err != hipSuccess) return err;
  p.keys = keys;
  p.order = order;
  p.strips = static_cast<int>(strips);
  // Chunks for about eight wavefronts a compute unit, of 16 to 64 places.
  p.chunk = 64;
  while (p.chunk > 16 && a.count / p.chunk * p.strips < 8 * compute_units()) p.chunk /= 2;
  p.chunks = static_cast<int>((a.count + p.chunk - 1) / p.chunk);
  p.partial = ws.take<float>(static_cast<int64_t>(p.chunks) * 2 * a.cols);
  if (bytes != nullptr) *bytes = ws.used();
  if (ws.dry()) return hipSuccess;
  const int64_t units = static_cast<int64_t>(p.chunks) * p.strips;
  p.summing = static_cast<int>((units + 3) / 4);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    sum_kernel<T><<<dim3(static_cast<uint32_t>(p.summing + (a.vocab + 63) / 64)), dim3(256), 0, stream>>>(p);
    if (p.chunks > 1) join_runs_kernel<T><<<dim3(static_cast<uint32_t>(units)), dim3(64 * kJoining), 0, stream>>>(p);
    return hipGetLastError();
  });
}

}  // namespace fh
