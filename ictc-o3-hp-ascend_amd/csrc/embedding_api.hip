// Rows of a table by index (an atom's species, the pair of species of an edge) times a scale, and the gradient
// of the table, gfx950.
//
//   y_i = s T[t_i]            dT[v] = s sum over {i : t_i = v} of dy_i, in the order of i
//
// A token outside the table (padding: -1) has a row of zeros and no gradient.
//
// The gradient sorts the tokens and sums runs of equal ones, so that no two workgroups add to one address: the sum's order
// is fixed, and rows with a tenth of all tokens cost what others cost.  Each workgroup has the same number of sorted
// tokens, split evenly over its groups of lanes; a group reads the gradient's rows in sorted order, writes the runs that lie
// within its share, and leaves its first and its last one in LDS, where runs over several groups are joined.
//
//   * Up to 255 rows (species, few pairs) of up to 64 columns, or with few tokens (see sorts_locally): a workgroup sorts its
//     own tokens, in LDS, and leaves a part for each row it meets; the second launch adds every row's parts up in order.
//     The sort then costs no launch and no traffic.
//   * Else: a radix sort of all tokens by 8 bits a pass (histogram, scan, scatter; stable).  Runs within a workgroup
//     are written at once.  One that goes on into the next workgroup's tokens leaves its part in that one's `head`,
//     or in `tail` of the one in which it begins; the last launch adds a row's parts up in order and writes zeros for
//     rows without tokens.
// Up to 32 tokens of a share and then up to 32 shares are added up in float32, the parts they leave in 64 bits.
//
// Bound by memory: dy and the table are read once, y and dT written once; the sort moves 8 to 16 bytes a token
// and pass.  500,001 tokens of 64 columns, 7,921 rows: lookup 22 us (5.9 TB/s), sort 29 (six launches of 3 to 10,
// bound by latency), sums 28 (4.6 TB/s), parts 7.  65,537 tokens of 512 columns, 50,000 rows: 36 us (7.4 TB/s; the
// table's rows repeat), sort 21, sums 34 to 39, parts 15.  105,634 tokens of 64 columns, 100 rows: lookup 7.2, sums 14,
// parts 10.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ictc_hip.h"

namespace ictc {
namespace {

constexpr int kEmbWave = 64;
constexpr int kEmbThreads = 256;
constexpr int kEmbWaves = kEmbThreads / kEmbWave;
constexpr int kRadix = 256;                  // digits of 8 bits
constexpr int kRounds = 4;                   // of a wave over its part of a tile (8: sorts of 500,001 and 65,537 tokens
                                             // 32 and 27 us against 29 and 21; 2: 31 and 18)
constexpr int kTile = kRounds * kEmbThreads;
constexpr int kLoads = 8;                    // rows on their way at a time
constexpr int kParts = 16;                   // parts of a row on their way at a time
constexpr int kShare = 32;                   // sorted tokens of a group of lanes at most
constexpr int kLeast = 8;                    // lanes of a group that sums them: at most 32 groups, which are joined one after
                                             // another (400,000 tokens of 4 columns, 200 rows 33 us, with one lane 66; of
                                             // 16 columns, 30 rows 28 against 26)
constexpr int kLong = 32;                    // parts of a row that one group adds up
constexpr int kFewRows = kRadix - 1;         // rows of tables whose tokens are sorted by the workgroup (and padding)
constexpr int kFewColumns = 64;
constexpr int64_t kFewValues = int64_t{1} << 21;      // of the gradient
constexpr int kMostLocal = 512;              // tokens of such a workgroup
constexpr int kRowGrid = 2048;               // workgroups that rows with parts are spread over
constexpr int kAhead = 4;                    // rows of a lookup's group of lanes at a time

typedef float ef4 __attribute__((ext_vector_type(4), aligned(4)));

// A thread's four columns of a row of `width`; the last ones may be fewer.
struct Quad {
  int at, count;

  __device__ __forceinline__ Quad(int first, int width) : at(first) {
    const int left = width - first;
    count = left < 0 ? 0 : left > 4 ? 4 : left;
  }

  __device__ __forceinline__ ef4 load(const float* row) const {
    ef4 t = {0.f, 0.f, 0.f, 0.f};
    if (count == 4) return *reinterpret_cast<const ef4*>(row + at);
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < count) t[j] = row[at + j];
    return t;
  }

  // Read once: past the caches.
  __device__ __forceinline__ ef4 stream(const float* row) const {
    ef4 t = {0.f, 0.f, 0.f, 0.f};
    if (count == 4) return __builtin_nontemporal_load(reinterpret_cast<const ef4*>(row + at));
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < count) t[j] = row[at + j];
    return t;
  }

  __device__ __forceinline__ void stream(float* row, const ef4& t) const {
    if (count == 4) {
      __builtin_nontemporal_store(t, reinterpret_cast<ef4*>(row + at));
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < count) row[at + j] = t[j];
    }
  }

  __device__ __forceinline__ void store(float* row, const ef4& t) const {
    if (count == 4) {
      *reinterpret_cast<ef4*>(row + at) = t;
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < count) row[at + j] = t[j];
    }
  }
};

// Threads of a row (a power of two, a wave at most); wider rows take several workgroups side by side (gridDim.y).
__host__ __device__ inline int row_threads(int width) {
  int threads = 1;
  while (threads < kEmbWave && 4 * threads < width) threads *= 2;
  return threads;
}

template <typename I>
__global__ void __launch_bounds__(kEmbThreads)
embedding_forward_kernel(const I* __restrict__ tokens, const float* __restrict__ table, float* __restrict__ out,
                         int64_t rows, int width, float scale, int64_t count, int threads) {
  const int groups = kEmbThreads / threads, group = threadIdx.x / threads;
  const Quad q((blockIdx.y * threads + (threadIdx.x & (threads - 1))) * 4, width);
  const int64_t step = static_cast<int64_t>(gridDim.x) * groups * kAhead;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * groups * kAhead + group; base < count; base += step) {
    int64_t t[kAhead];
    ef4 v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = base + k * groups;
      t[k] = i < count ? static_cast<int64_t>(tokens[i]) : -1;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const bool there = t[k] >= 0 && t[k] < rows;
      v[k] = there ? q.load(table + t[k] * width) : ef4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = base + k * groups;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[k][j] = t[k] >= 0 && t[k] < rows ? v[k][j] * scale : 0.f;
      if (i < count) q.stream(out + i * width, v[k]);
    }
  }
}

// A token as a sort key: those without a row come last.
__device__ __forceinline__ uint32_t key_of(int64_t t, int64_t rows) {
  return static_cast<uint32_t>(t >= 0 && t < rows ? t : rows);
}

// Digits of each tile, [digit][tile]; the first pass also clears the rows' spans.
template <typename I, bool FIRST>
__global__ void __launch_bounds__(kEmbThreads)
radix_count_kernel(const I* __restrict__ tokens, const uint32_t* __restrict__ keys, int64_t rows, int count, int shift,
                   uint32_t* __restrict__ counts, int2* __restrict__ spans) {
  __shared__ uint32_t bins[kRadix];
  bins[threadIdx.x] = 0;
  __syncthreads();
  const int first = blockIdx.x * kTile;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int i = first + k * kEmbThreads + threadIdx.x;
    if (i < count) atomicAdd(&bins[((FIRST ? key_of(tokens[i], rows) : keys[i]) >> shift) & (kRadix - 1)], 1u);
  }
  __syncthreads();
  counts[static_cast<int64_t>(threadIdx.x) * gridDim.x + blockIdx.x] = bins[threadIdx.x];
  if constexpr (FIRST)
    for (int64_t v = static_cast<int64_t>(blockIdx.x) * kEmbThreads + threadIdx.x; v < rows;
         v += static_cast<int64_t>(gridDim.x) * kEmbThreads)
      spans[v] = make_int2(0, 0);
}

// Sums before each entry over a workgroup's threads, and the whole sum.
__device__ __forceinline__ uint32_t scan(uint32_t x, uint32_t* lds, uint32_t& total) {
  const int lane = threadIdx.x & (kEmbWave - 1), wave = threadIdx.x / kEmbWave;
  uint32_t sum = x;
#pragma unroll
  for (int d = 1; d < kEmbWave; d *= 2) {
    const uint32_t o = __shfl_up(sum, d);
    if (lane >= d) sum += o;
  }
  __syncthreads();
  if (lane == kEmbWave - 1) lds[wave] = sum;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kEmbWaves; ++w) {
    if (w < wave) before += lds[w];
    total += lds[w];
  }
  return before + sum - x;
}

// Per digit: how many of it lie in the tiles before each, in place, and of all tiles.
__global__ void __launch_bounds__(kEmbThreads)
radix_scan_kernel(uint32_t* __restrict__ counts, uint32_t* __restrict__ totals, int tiles) {
  __shared__ uint32_t lds[kEmbWaves];
  uint32_t* row = counts + static_cast<int64_t>(blockIdx.x) * tiles;
  uint32_t before = 0;
  for (int first = 0; first < tiles; first += kEmbThreads) {
    const int k = first + threadIdx.x;
    uint32_t sum;
    const uint32_t own = scan(k < tiles ? row[k] : 0u, lds, sum);
    if (k < tiles) row[k] = before + own;
    before += sum;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

// Ranks of a wave's keys among its earlier ones with the same digit, 64 at a time: lanes of one digit find each other
// by eight votes, and the wave's counts so far (`counts`, raised on the way) give their rank.  Key k is there for
// lanes below `count` - 64 k.
template <int ROUNDS>
__device__ __forceinline__ void wave_ranks(const uint32_t (&key)[ROUNDS], int count, int shift, uint32_t* counts,
                                           uint32_t (&rank)[ROUNDS]) {
  const int lane = threadIdx.x & (kEmbWave - 1);
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const bool on = k * kEmbWave + lane < count;
    const uint32_t digit = (key[k] >> shift) & (kRadix - 1);
    uint64_t same = __ballot(on);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint64_t vote = __ballot((digit >> b) & 1u);
      same &= (digit >> b) & 1u ? vote : ~vote;
    }
    // (a wave's LDS operations are carried out in order: all lanes read the count before the first lane of each
    // digit raises it)
    const uint32_t before = counts[digit];
    const uint32_t below = __popcll(same & ((uint64_t{1} << lane) - 1));
    rank[k] = before + below;
    if (on && below == 0) counts[digit] = before + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// Keys and places to their positions by this digit, in order; a wave takes a quarter of the tile.
template <typename I, bool FIRST>
__global__ void __launch_bounds__(kEmbThreads)
radix_scatter_kernel(const I* __restrict__ tokens, const uint32_t* __restrict__ keys, const int32_t* __restrict__ places,
                     int64_t rows, int count, int shift, const uint32_t* __restrict__ counts,
                     const uint32_t* __restrict__ totals, uint32_t* __restrict__ out_keys,
                     int32_t* __restrict__ out_places) {
  __shared__ uint32_t ranks[kEmbWaves][kRadix];
  __shared__ uint32_t lds[kEmbWaves];
  const int lane = threadIdx.x & (kEmbWave - 1), wave = threadIdx.x / kEmbWave;
#pragma unroll
  for (int w = 0; w < kEmbWaves; ++w) ranks[w][threadIdx.x] = 0;
  __syncthreads();
  const int first = blockIdx.x * kTile + wave * (kTile / kEmbWaves);
  uint32_t key[kRounds], rank[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int i = first + k * kEmbWave + lane;
    key[k] = i < count ? (FIRST ? key_of(tokens[i], rows) : keys[i]) : 0u;
  }
  wave_ranks<kRounds>(key, count - first, shift, ranks[wave], rank);
  __syncthreads();
  uint32_t total;
  const uint32_t digit_start = scan(totals[threadIdx.x], lds, total);
  uint32_t at = digit_start + counts[static_cast<int64_t>(threadIdx.x) * gridDim.x + blockIdx.x];
#pragma unroll
  for (int w = 0; w < kEmbWaves; ++w) {
    const uint32_t own = ranks[w][threadIdx.x];
    ranks[w][threadIdx.x] = at;
    at += own;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int i = first + k * kEmbWave + lane;
    if (i < count) {
      const uint32_t to = ranks[wave][(key[k] >> shift) & (kRadix - 1)] + rank[k];
      out_keys[to] = key[k];
      out_places[to] = FIRST ? i : places[i];
    }
  }
}

// What a workgroup's groups of lanes leave to be joined: each one's first and last run.
struct Ends {
  ef4 sum[2][kEmbThreads];
  uint32_t key[2][kEmbThreads];      // of each group; equal: one run
};

// (Reading the gradient past the caches: 65,537 tokens of 512 columns 39 us against 53, 105,634 of 64 17 against 15.)
//
// Sums the runs of `size` sorted tokens, `share` of them to each group of lanes: key(i) and place(i) of the i-th,
// done(key, sum, from, to) for every run whole within them (from and to: its first and the end, in these tokens).
template <bool PAST, typename Key, typename At, typename Done>
__device__ __forceinline__ void sum_runs(int size, int share, int threads, const Quad& q, const float* __restrict__ grad,
                                         int64_t width, Ends& ends, Key&& key, At&& place, Done&& done) {
  const int groups = kEmbThreads / threads, group = threadIdx.x / threads, lane = threadIdx.x & (threads - 1);
  const int first = group * share < size ? group * share : size, end = size - first < share ? size : first + share;
  if (first < end) {
    const uint32_t head = key(first);
    uint32_t current = head;
    ef4 sum = {0.f, 0.f, 0.f, 0.f};
    int from = first;
    uint32_t next_key[kLoads];
    int64_t next[kLoads];
    const auto fetch = [&](int i) {       // (one batch of rows ahead)
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int at = i + j < end ? i + j : end - 1;
        next_key[j] = key(at);
        next[j] = place(at);
      }
    };
    fetch(first);
    for (int i = first; i < end; i += kLoads) {
      uint32_t k[kLoads];
      ef4 v[kLoads];
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        k[j] = next_key[j];
        v[j] = PAST ? q.stream(grad + next[j] * width) : q.load(grad + next[j] * width);
      }
      if (i + kLoads < end) fetch(i + kLoads);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        if (i + j >= end) break;
        if (k[j] != current) {
          if (from == first) ends.sum[0][threadIdx.x] = sum; else done(current, sum, from, i + j);
          current = k[j];
          from = i + j;
          sum = v[j];
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[c] += v[j][c];
        }
      }
    }
    ends.sum[from == first ? 0 : 1][threadIdx.x] = sum;
    if (lane == 0) ends.key[0][group] = head, ends.key[1][group] = current;
  }
  __syncthreads();
  // (one group of lanes: a run's end in one share and its head in the next are a step each)
  if (group) return;
  uint32_t current = 0;
  ef4 sum = {0.f, 0.f, 0.f, 0.f};
  bool begun = false;
  for (int g = 0; g < groups && g * share < size; ++g) {
    const uint32_t head = ends.key[0][g], last = ends.key[1][g];
    const ef4 v = ends.sum[0][g * threads + lane];
    if (begun && current == head) {
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[c] += v[c];
    } else {
      if (begun) done(current, sum, -1, g * share);
      current = head;
      sum = v;
    }
    begun = true;
    if (last != head) {
      done(current, sum, -1, -1);
      current = last;
      sum = ends.sum[1][g * threads + lane];
    }
  }
  if (begun) done(current, sum, -1, size);
}

// Parts of each row that a workgroup's tokens have, sorted here: parts [workgroups][rows][width], met [rows][workgroups].
template <typename I>
__global__ void __launch_bounds__(kEmbThreads)
embedding_local_kernel(const I* __restrict__ tokens, const float* __restrict__ grad, float* __restrict__ parts,
                       uint32_t* __restrict__ met, int rows, int width, int count, int size, int share, int threads) {
  constexpr int kLocalRounds = kMostLocal / kEmbThreads;
  __shared__ Ends ends;
  __shared__ uint32_t ranks[kEmbWaves][kRadix];
  __shared__ uint32_t lds[kEmbWaves];
  __shared__ uint16_t sorted_key[kMostLocal], sorted_place[kMostLocal];
  const int lane = threadIdx.x & (kEmbWave - 1), wave = threadIdx.x / kEmbWave;
  const int first = blockIdx.x * size, own = count - first < size ? count - first : size;
#pragma unroll
  for (int w = 0; w < kEmbWaves; ++w) ranks[w][threadIdx.x] = 0;
  __syncthreads();
  const int start = wave * (kLocalRounds * kEmbWave);
  uint32_t key[kLocalRounds], rank[kLocalRounds];
#pragma unroll
  for (int k = 0; k < kLocalRounds; ++k) {
    const int i = start + k * kEmbWave + lane;
    key[k] = i < own ? key_of(tokens[first + i], rows) : 0u;
  }
  wave_ranks<kLocalRounds>(key, own - start, 0, ranks[wave], rank);
  __syncthreads();
  uint32_t of_row = 0, total;
#pragma unroll
  for (int w = 0; w < kEmbWaves; ++w) of_row += ranks[w][threadIdx.x];
  uint32_t at = scan(of_row, lds, total);
#pragma unroll
  for (int w = 0; w < kEmbWaves; ++w) {
    const uint32_t mine = ranks[w][threadIdx.x];
    ranks[w][threadIdx.x] = at;
    at += mine;
  }
  if (static_cast<int>(threadIdx.x) < rows && blockIdx.y == 0)
    met[static_cast<int64_t>(threadIdx.x) * gridDim.x + blockIdx.x] = of_row;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kLocalRounds; ++k) {
    const int i = start + k * kEmbWave + lane;
    if (i < own) {
      const uint32_t to = ranks[wave][key[k]] + rank[k];
      sorted_key[to] = static_cast<uint16_t>(key[k]);
      sorted_place[to] = static_cast<uint16_t>(i);
    }
  }
  __syncthreads();
  const Quad q((blockIdx.y * threads + (threadIdx.x & (threads - 1))) * 4, width);
  sum_runs<false>(own, share, threads, q, grad, width, ends, [&](int i) { return static_cast<uint32_t>(sorted_key[i]); },
           [&](int i) { return static_cast<int64_t>(first + sorted_place[i]); },
           [&](uint32_t k, const ef4& sum, int, int) {
             if (static_cast<int>(k) < rows) q.store(parts + (static_cast<int64_t>(blockIdx.x) * rows + k) * width, sum);
           });
}

// Sums of the groups of lanes, in order, in the first one.
__device__ __forceinline__ void join_groups(double (&sum)[4], double (*lds)[4], int threads) {
  const int groups = kEmbThreads / threads, lane = threadIdx.x & (threads - 1);
#pragma unroll
  for (int j = 0; j < 4; ++j) lds[threadIdx.x][j] = sum[j];
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < threads)
    for (int g = 1; g < groups; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += lds[g * threads + lane][j];
}

__device__ __forceinline__ void add(double (&sum)[4], const ef4& v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) sum[j] += static_cast<double>(v[j]);
}

__device__ __forceinline__ ef4 scaled(const double (&sum)[4], float scale) {
  ef4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = static_cast<float>(sum[j] * static_cast<double>(scale));
  return v;
}

// A workgroup to a row: the parts of the workgroups that met it.
__global__ void __launch_bounds__(kEmbThreads)
embedding_local_join_kernel(const float* __restrict__ parts, const uint32_t* __restrict__ met, float* __restrict__ dtable,
                            int rows, int width, float scale, int workgroups, int threads) {
  __shared__ double lds[kEmbThreads][4];
  const int groups = kEmbThreads / threads, group = threadIdx.x / threads;
  const Quad q((blockIdx.y * threads + (threadIdx.x & (threads - 1))) * 4, width);
  const int64_t row = blockIdx.x;
  const int share = (workgroups + groups - 1) / groups;
  const int end = workgroups < (group + 1) * share ? workgroups : (group + 1) * share;
  const float* p = parts + row * width;
  double sum[4] = {};
  for (int w = group * share; w < end; w += kParts) {
    uint32_t there[kParts];
    ef4 v[kParts];
#pragma unroll
    for (int j = 0; j < kParts; ++j) there[j] = w + j < end ? met[row * workgroups + w + j] : 0u;
#pragma unroll
    for (int j = 0; j < kParts; ++j) {
      v[j] = ef4{0.f, 0.f, 0.f, 0.f};
      if (there[j]) v[j] = q.load(p + static_cast<int64_t>(w + j) * rows * width);
    }
#pragma unroll
    for (int j = 0; j < kParts; ++j) add(sum, v[j]);
  }
  join_groups(sum, lds, threads);
  if (group == 0) q.store(dtable + row * width, scaled(sum, scale));
}

// Sums of a workgroup's runs of all sorted tokens.  parts: [2][workgroups][width], heads and tails.
__global__ void __launch_bounds__(kEmbThreads)
embedding_chunk_kernel(const uint32_t* __restrict__ keys, const int32_t* __restrict__ places,
                       const float* __restrict__ grad, float* __restrict__ dtable, float* __restrict__ parts,
                       int2* __restrict__ spans, uint32_t rows, int width, float scale, int count, int size, int share,
                       int threads) {
  __shared__ Ends ends;
  const Quad q((blockIdx.y * threads + (threadIdx.x & (threads - 1))) * 4, width);
  const int first = blockIdx.x * size, own = count - first < size ? count - first : size;
  const uint32_t before = first ? keys[first - 1] : ~0u, after = first + own < count ? keys[first + own] : ~0u;
  // where rows begin and end
  if (blockIdx.y == 0)
    for (int i = first + threadIdx.x; i <= first + own; i += kEmbThreads) {
      if (i == first + own && i < count) break;            // (the next workgroup's)
      const uint32_t k = i < count ? keys[i] : ~0u, last = i ? keys[i - 1] : ~0u;
      if (k == last) continue;
      if (last < rows) spans[last].y = i;
      if (k < rows) spans[k].x = i;
    }
  sum_runs<true>(own, share, threads, q, grad, width, ends, [&](int i) { return keys[first + i]; },
           [&](int i) { return static_cast<int64_t>(places[first + i]); },
           [&](uint32_t k, const ef4& sum, int, int) {
             if (k >= rows) return;
             // (equal keys lie side by side: a run with the key before these tokens is the first one)
             float* to = k == before ? parts + static_cast<int64_t>(blockIdx.x) * width
                         : k == after ? parts + (static_cast<int64_t>(gridDim.x) + blockIdx.x) * width
                                      : dtable + static_cast<int64_t>(k) * width;
             ef4 v = sum;
             if (k != before && k != after) {
#pragma unroll
               for (int j = 0; j < 4; ++j) v[j] *= scale;
             }
             q.store(to, v);
           });
}

// Rows whose runs span workgroups from their parts, and zeros for rows without tokens.  A group of lanes to a row (and
// several rows to a group, one after the other), all of them to one of many parts; with few rows a workgroup to each.
__global__ void __launch_bounds__(kEmbThreads)
embedding_join_kernel(const float* __restrict__ parts, const int2* __restrict__ spans, float* __restrict__ dtable,
                      int64_t rows, int width, float scale, int size, int workgroups, int threads, int per) {
  __shared__ double lds[kEmbThreads][4];
  const int groups = kEmbThreads / threads, group = threadIdx.x / threads;
  const Quad q((blockIdx.y * threads + (threadIdx.x & (threads - 1))) * 4, width);
  const float* tails = parts + static_cast<int64_t>(workgroups) * width;
  const int most = per < groups ? 1 : kLong;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * per; base < rows; base += static_cast<int64_t>(gridDim.x) * per) {
    bool is_long = false;
    int2 span[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t row = base + k * groups + group;
      span[k] = k * groups + group < per && row < rows ? spans[row] : make_int2(0, -1);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t row = base + k * groups + group;
      if (span[k].y < 0) continue;
      const int from = span[k].x / size, to = span[k].y ? (span[k].y - 1) / size : 0;
      if (span[k].y == 0) {
        q.store(dtable + row * width, ef4{0.f, 0.f, 0.f, 0.f});
      } else if (to - from > most) {
        is_long = true;
      } else if (to > from) {
        double sum[4] = {};
        add(sum, q.load(tails + static_cast<int64_t>(from) * width));
        for (int c = from + 1; c <= to; ++c) add(sum, q.load(parts + static_cast<int64_t>(c) * width));
        q.store(dtable + row * width, scaled(sum, scale));
      }
    }
    if (!__syncthreads_or(is_long)) continue;
    for (int g = 0; g < per && base + g < rows; ++g) {
      const int2 span = spans[base + g];
      if (!span.y) continue;
      const int from = span.x / size, to = (span.y - 1) / size, of_row = to - from + 1;
      if (to - from <= most) continue;
      const int share = (of_row + groups - 1) / groups, stop = of_row < (group + 1) * share ? of_row : (group + 1) * share;
      double sum[4] = {};
      for (int p = group * share; p < stop; p += kLoads) {
        ef4 v[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          v[j] = ef4{0.f, 0.f, 0.f, 0.f};
          if (p + j < stop) v[j] = q.load((p + j ? parts : tails) + static_cast<int64_t>(from + p + j) * width);
        }
#pragma unroll
        for (int j = 0; j < kLoads; ++j) add(sum, v[j]);
      }
      join_groups(sum, lds, threads);
      if (group == 0) q.store(dtable + (base + g) * width, scaled(sum, scale));
      __syncthreads();
    }
  }
}

constexpr int64_t kMostTokens = (int64_t{1} << 31) - 2 * kTile;
constexpr int64_t kMostRows = (int64_t{1} << 31) - 2;
constexpr int kMostWidth = 1 << 20;
constexpr int kFill = 256;                   // workgroups that fill the chip

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// How the sorted tokens are split: `share` to a group of lanes, `size` to a workgroup.  Long shares leave fewer parts, short
// ones fill the chip when there are few tokens.
struct Split {
  int threads, columns, share, size, workgroups;

  Split(int width, int64_t count) {
    threads = row_threads(width) < kLeast ? kLeast : row_threads(width);
    columns = (width + 4 * threads - 1) / (4 * threads);
    const int groups = kEmbThreads / threads;
    share = kShare;
    while (share > kLoads && count / (static_cast<int64_t>(groups) * share) * columns < kFill) share /= 2;
    while (groups * share > kMostLocal) share /= 2;
    size = groups * share;
    workgroups = static_cast<int>((count + size - 1) / size);
  }
};

// Whether workgroups sort their own tokens.  The wider the rows, the fewer tokens a workgroup has, the more of them are of
// different rows and the more of the gradient's size its parts have (they are written and read again, and 255 rows of 256
// columns and more would take twice its size), against a sort of all tokens whose launches cost 8 us.  Of 100 rows,
// us here / with all sorted: 64 columns, 2,048 tokens 12 / 19, 65,536 21 / 24, 300,000 38 / 39; 128 columns 11 / 19,
// (20,000) 25 / 20, 29 / 28 and 94 / 48; 512 columns 12 / 19, (20,000) 32 / 29, 79 / 39 and 501 / 121; 10 and 255 rows
// of 512 columns, 300,000 tokens 472 / 126 and 499 / 123.
bool sorts_locally(int64_t rows, int width, int64_t count) {
  return rows <= kFewRows && (width <= kFewColumns || count * width <= kFewValues);
}

// Where everything lies in the workspace, in 4-byte units.
struct EmbeddingSpace {
  int64_t keys[2], places[2], counts, totals, spans, met, parts, size;
  int tiles;
  bool local;

  EmbeddingSpace(int64_t rows, int width, int64_t count, const Split& split) {
    tiles = static_cast<int>((count + kTile - 1) / kTile);
    local = sorts_locally(rows, width, count);
    int64_t at = 0;
    const auto take = [&](int64_t n) {
      const int64_t first = at;
      at += up(n, 64);
      return first;
    };
    for (int k = 0; k < 2; ++k) keys[k] = take(local ? 0 : count), places[k] = take(local ? 0 : count);
    counts = take(local ? 0 : static_cast<int64_t>(kRadix) * tiles);
    totals = take(local ? 0 : kRadix);
    spans = take(local ? 0 : 2 * rows);
    met = take(local ? rows * split.workgroups : 0);
    parts = take((local ? rows : 2) * static_cast<int64_t>(split.workgroups) * width);
    size = at;
  }
};

bool embedding_valid(int index_bytes, int64_t rows, int64_t width, int64_t count) {
  return (index_bytes == 4 || index_bytes == 8) && rows >= 1 && rows <= kMostRows && width >= 1 && width <= kMostWidth &&
         count >= 0 && count <= kMostTokens;
}

int embedding_launched() { return hipGetLastError() == hipSuccess ? ICTC_OK : ICTC_ERR_LAUNCH; }

// Workgroups for rows, `per` at a time: threads within 32 bits.
unsigned row_grid(int64_t rows, int64_t per, int columns) {
  const int64_t blocks = (rows + per - 1) / per, most = (int64_t{1} << 23) / columns;
  return static_cast<unsigned>(blocks < most ? blocks : most > 0 ? most : 1);
}

template <typename I>
int table_gradient(const I* tokens, const float* grad, float* dtable, int64_t rows, int width, float scale, int64_t count,
                   uint32_t* ws, hipStream_t stream) {
  const Split d(width, count);
  const EmbeddingSpace s(rows, width, count, d);
  const int n = static_cast<int>(count);
  float* parts = reinterpret_cast<float*>(ws + s.parts);
  if (s.local) {
    hipLaunchKernelGGL(embedding_local_kernel<I>, dim3(d.workgroups, d.columns), dim3(kEmbThreads), 0, stream, tokens,
                       grad, parts, ws + s.met, static_cast<int>(rows), width, n, d.size, d.share, d.threads);
    hipLaunchKernelGGL(embedding_local_join_kernel, dim3(static_cast<unsigned>(rows), d.columns), dim3(kEmbThreads), 0,
                       stream, parts, ws + s.met, dtable, static_cast<int>(rows), width, scale, d.workgroups, d.threads);
    return embedding_launched();
  }
  uint32_t* keys[2] = {ws + s.keys[0], ws + s.keys[1]};
  int32_t* places[2] = {reinterpret_cast<int32_t*>(ws + s.places[0]), reinterpret_cast<int32_t*>(ws + s.places[1])};
  int2* spans = reinterpret_cast<int2*>(ws + s.spans);
  int bits = 1;
  while (rows >> bits) ++bits;         // of the largest key, `rows`
  int now = 0;
  for (int shift = 0; shift < bits; shift += 8, now ^= 1) {
    const auto count_kernel = shift ? radix_count_kernel<I, false> : radix_count_kernel<I, true>;
    const auto scatter_kernel = shift ? radix_scatter_kernel<I, false> : radix_scatter_kernel<I, true>;
    hipLaunchKernelGGL(count_kernel, dim3(s.tiles), dim3(kEmbThreads), 0, stream, tokens, keys[now ^ 1], rows, n, shift,
                       ws + s.counts, spans);
    hipLaunchKernelGGL(radix_scan_kernel, dim3(kRadix), dim3(kEmbThreads), 0, stream, ws + s.counts, ws + s.totals,
                       s.tiles);
    hipLaunchKernelGGL(scatter_kernel, dim3(s.tiles), dim3(kEmbThreads), 0, stream, tokens, keys[now ^ 1],
                       places[now ^ 1], rows, n, shift, ws + s.counts, ws + s.totals, keys[now], places[now]);
    if (const int rc = embedding_launched()) return rc;
  }
  const int sorted = now ^ 1, most = kAhead * (kEmbThreads / d.threads);
  const int per = static_cast<int>(rows / kRowGrid < 1 ? 1 : rows / kRowGrid < most ? rows / kRowGrid : most);
  hipLaunchKernelGGL(embedding_chunk_kernel, dim3(d.workgroups, d.columns), dim3(kEmbThreads), 0, stream, keys[sorted],
                     places[sorted], grad, dtable, parts, spans, static_cast<uint32_t>(rows), width, scale, n, d.size,
                     d.share, d.threads);
  hipLaunchKernelGGL(embedding_join_kernel, dim3(row_grid(rows, per, d.columns), d.columns), dim3(kEmbThreads), 0, stream,
                     parts, spans, dtable, rows, width, scale, d.size, d.workgroups, d.threads, per);
  return embedding_launched();
}

}  // namespace
}  // namespace ictc

extern "C" {

int ictc_hip_embedding_forward(const void* tokens, int index_bytes, const float* table, float* out, int64_t rows,
                               int width, float scale, int64_t count, hipStream_t stream) {
  using namespace ictc;
  if (!embedding_valid(index_bytes, rows, width, count)) return ICTC_ERR_INVALID_ARGUMENT;
  if (count == 0) return ICTC_OK;
  if (!tokens || !table || !out) return ICTC_ERR_INVALID_ARGUMENT;
  const int threads = row_threads(width), columns = (width + 4 * threads - 1) / (4 * threads);
  const dim3 grid(row_grid(count, kAhead * (kEmbThreads / threads), columns), columns);
  if (index_bytes == 4)
    hipLaunchKernelGGL(embedding_forward_kernel<int32_t>, grid, dim3(kEmbThreads), 0, stream,
                       static_cast<const int32_t*>(tokens), table, out, rows, width, scale, count, threads);
  else
    hipLaunchKernelGGL(embedding_forward_kernel<int64_t>, grid, dim3(kEmbThreads), 0, stream,
                       static_cast<const int64_t*>(tokens), table, out, rows, width, scale, count, threads);
  return embedding_launched();
}

int64_t ictc_hip_embedding_workspace(int64_t rows, int width, int64_t count) {
  using namespace ictc;
  if (!embedding_valid(8, rows, width, count)) return -ICTC_ERR_INVALID_ARGUMENT;
  return EmbeddingSpace(rows, width, count, Split(width, count)).size;
}

int ictc_hip_embedding_table_grad(const void* tokens, int index_bytes, const float* grad, float* dtable, int64_t rows,
                                  int width, float scale, int64_t count, void* workspace, int64_t workspace_units,
                                  hipStream_t stream) {
  using namespace ictc;
  if (!embedding_valid(index_bytes, rows, width, count) || count == 0) return ICTC_ERR_INVALID_ARGUMENT;
  if (!tokens || !grad || !dtable || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
      workspace_units < ictc_hip_embedding_workspace(rows, width, count))
    return ICTC_ERR_INVALID_ARGUMENT;
  uint32_t* ws = static_cast<uint32_t*>(workspace);
  return index_bytes == 4 ? table_gradient(static_cast<const int32_t*>(tokens), grad, dtable, rows, width, scale, count,
                                           ws, stream)
                          : table_gradient(static_cast<const int64_t*>(tokens), grad, dtable, rows, width, scale, count,
                                           ws, stream);
}

}  // extern "C"
