// Rows of a table by index (an atom's species, the pair of species of an edge) times a scale, and the gradient
// of the table, gfx950.
//
//   y_i = s T[t_i]            dT[v] = s sum over {i : t_i = v} of dy_i, in the order of i
//
// A token outside the table (padding: -1) has a row of zeros and no gradient.
//
// The gradient sorts the tokens and sums runs of equal ones, so that no two workgroups add to one address: the sum's order
// is fixed, and rows with a tenth of all tokens cost what others cost.  The sort is a radix sort by 8 bits a
// pass (histogram, scan, scatter; stable).  The sorted tokens are cut into chunks of equal length; a group of lanes
// takes one, reads the gradient's rows in sorted order and writes every run that lies within it.  A run that
// goes on into the next chunk leaves its part in that chunk's `head`, or in `tail` of the chunk in which it
// begins; the last kernel adds a row's parts up in order (in 64 bits) and writes zeros for rows without tokens.
//
// Bound by memory: dy and the table are read once, y and dT written once; the sort moves 8 to 16 bytes a token
// and pass.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ictc_hip.h"

namespace ictc {
namespace {

constexpr int kEmbWave = 64;
constexpr int kEmbThreads = 256;
constexpr int kEmbWaves = kEmbThreads / kEmbWave;
constexpr int kRadix = 256;                  // digits of 8 bits
constexpr int kRounds = 8;                   // of a wave over its part of a tile
constexpr int kTile = kRounds * kEmbThreads;
constexpr int kChunk = 32;                   // sorted tokens of a group of lanes
constexpr int kLoads = 8;                    // rows on their way at a time
constexpr int kLong = 32;                    // parts of a row that one group adds up

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
  const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * groups + group; i < count; i += step) {
    const int64_t t = tokens[i];
    ef4 v = {0.f, 0.f, 0.f, 0.f};
    if (t >= 0 && t < rows) {
      v = q.load(table + t * width);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] *= scale;
    }
    q.store(out + i * width, v);
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

// Keys and places to their positions by this digit, in order.  A wave takes a quarter of the tile, 64 at a
// time: lanes of one digit find each other by eight votes, and the wave's counts so far give their rank.
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
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const bool on = first + k * kEmbWave + lane < count;
    const uint32_t digit = (key[k] >> shift) & (kRadix - 1);
    uint64_t same = __ballot(on);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint64_t vote = __ballot((digit >> b) & 1u);
      same &= (digit >> b) & 1u ? vote : ~vote;
    }
    // (a wave's LDS operations are carried out in order: the first lane of each digit reads the count before
    // it raises it, and the others have read it by then)
    const uint32_t before = ranks[wave][digit];
    const uint32_t below = __popcll(same & ((uint64_t{1} << lane) - 1));
    rank[k] = before + below;
    if (on && below == 0) ranks[wave][digit] = before + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
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

// Sums of a chunk's runs (see above).  parts: [2][chunks][width], heads and tails.
__global__ void __launch_bounds__(kEmbThreads)
embedding_chunk_kernel(const uint32_t* __restrict__ keys, const int32_t* __restrict__ places,
                       const float* __restrict__ grad, float* __restrict__ dtable, float* __restrict__ parts,
                       int2* __restrict__ spans, uint32_t rows, int width, float scale, int count, int chunks,
                       int threads) {
  const int groups = kEmbThreads / threads, group = threadIdx.x / threads, lane = threadIdx.x & (threads - 1);
  const int64_t chunk = static_cast<int64_t>(blockIdx.x) * groups + group;
  if (chunk >= chunks) return;
  const Quad q((blockIdx.y * threads + lane) * 4, width);
  const bool marks = blockIdx.y == 0 && lane == 0;
  const int first = static_cast<int>(chunk) * kChunk, end = count - first < kChunk ? count : first + kChunk;
  const uint32_t before = first ? keys[first - 1] : ~0u;
  uint32_t current = before;
  bool head = true;            // the run came from the chunk before
  ef4 sum = {0.f, 0.f, 0.f, 0.f};

  // The run of `current` ends at `at`, or goes on behind the chunk.
  const auto close = [&](int at, bool on) {
    if (current >= rows || (head && at == first)) return;       // (no row, or no run yet)
    float* to = head ? parts + chunk * width : on ? parts + (chunks + chunk) * width
                                                  : dtable + static_cast<int64_t>(current) * width;
    ef4 v = sum;
    if (!head && !on) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] *= scale;
    }
    q.store(to, v);
  };

  for (int i = first; i < end; i += kLoads) {
    uint32_t k[kLoads];
    ef4 v[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int at = i + j < end ? i + j : end - 1;
      k[j] = keys[at];
      v[j] = q.load(grad + static_cast<int64_t>(places[at]) * width);
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      if (i + j >= end) break;
      if (k[j] != current) {
        close(i + j, false);
        if (marks) {
          if (current < rows) spans[current].y = i + j;
          if (k[j] < rows) spans[k[j]].x = i + j;
        }
        current = k[j];
        head = false;
        sum = v[j];
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[c] += v[j][c];
      }
    }
  }
  const bool last = end == count;
  const bool on = !last && keys[end] == current;
  close(end, on);
  if (marks && last && current < rows) spans[current].y = count;
}

// Rows whose runs span chunks from their parts, and zeros for rows without tokens.
__global__ void __launch_bounds__(kEmbThreads)
embedding_join_kernel(const float* __restrict__ parts, const int2* __restrict__ spans, float* __restrict__ dtable,
                      int64_t rows, int width, float scale, int chunks, int threads) {
  __shared__ double sums[kEmbThreads][4];
  __shared__ int longs[kEmbThreads];
  const int groups = kEmbThreads / threads, group = threadIdx.x / threads, lane = threadIdx.x & (threads - 1);
  const Quad q((blockIdx.y * threads + lane) * 4, width);
  const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
  const float* tails = parts + static_cast<int64_t>(chunks) * width;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * groups; base < rows; base += step) {
    const int64_t row = base + group;
    bool is_long = false;
    if (row < rows) {
      const int2 span = spans[row];
      if (span.y == 0) {
        q.store(dtable + row * width, ef4{0.f, 0.f, 0.f, 0.f});
      } else {
        const int from = span.x / kChunk, to = (span.y - 1) / kChunk;
        is_long = to - from > kLong;
        if (to > from && !is_long) {
          const ef4 t = q.load(tails + static_cast<int64_t>(from) * width);
          double sum[4] = {t[0], t[1], t[2], t[3]};
          for (int c = from + 1; c <= to; ++c) {
            const ef4 h = q.load(parts + static_cast<int64_t>(c) * width);
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] += static_cast<double>(h[j]);
          }
          ef4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = static_cast<float>(sum[j] * scale);
          q.store(dtable + row * width, v);
        }
      }
    }
    if (lane == 0) longs[group] = is_long;
    __syncthreads();
    // rows of many parts: all groups add up their share, one row after the other
    for (int g = 0; g < groups; ++g) {
      if (!longs[g]) continue;
      const int2 span = spans[base + g];
      const int from = span.x / kChunk, to = (span.y - 1) / kChunk, parts_of = to - from + 1;
      const int share = (parts_of + groups - 1) / groups;
      double sum[4] = {};
      const int stop = parts_of < (group + 1) * share ? parts_of : (group + 1) * share;
#pragma unroll 4
      for (int p = group * share; p < stop; ++p) {
        const ef4 h = q.load((p ? parts : tails) + static_cast<int64_t>(from + p) * width);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += static_cast<double>(h[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[threadIdx.x][j] = sum[j];
      __syncthreads();
      if (group == 0) {
        for (int o = 1; o < groups; ++o)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[j] += sums[o * threads + lane][j];
        ef4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = static_cast<float>(sum[j] * scale);
        q.store(dtable + (base + g) * width, v);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

constexpr int64_t kMostTokens = (int64_t{1} << 31) - 2 * kTile;
constexpr int64_t kMostRows = (int64_t{1} << 31) - 2;
constexpr int kMostWidth = 1 << 20;

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Where everything lies in the workspace, in 4-byte units.
struct EmbeddingSpace {
  int64_t keys[2], places[2], counts, totals, spans, parts, size;
  int tiles, chunks;

  EmbeddingSpace(int64_t rows, int width, int64_t count) {
    tiles = static_cast<int>((count + kTile - 1) / kTile);
    chunks = static_cast<int>((count + kChunk - 1) / kChunk);
    int64_t at = 0;
    const auto take = [&](int64_t n) {
      const int64_t first = at;
      at += up(n, 64);
      return first;
    };
    for (int k = 0; k < 2; ++k) keys[k] = take(count), places[k] = take(count);
    counts = take(static_cast<int64_t>(kRadix) * tiles);
    totals = take(kRadix);
    spans = take(2 * rows);
    parts = take(2 * static_cast<int64_t>(chunks) * width);
    size = at;
  }
};

bool embedding_valid(int index_bytes, int64_t rows, int64_t width, int64_t count) {
  return (index_bytes == 4 || index_bytes == 8) && rows >= 1 && rows <= kMostRows && width >= 1 && width <= kMostWidth &&
         count >= 0 && count <= kMostTokens;
}

int embedding_launched() { return hipGetLastError() == hipSuccess ? ICTC_OK : ICTC_ERR_LAUNCH; }

// Rows to workgroups: enough to fill the chip several times over, threads within 32 bits.
unsigned row_grid(int64_t rows, int threads, int columns) {
  const int64_t groups = kEmbThreads / threads, blocks = (rows + groups - 1) / groups;
  const int64_t most = (int64_t{1} << 22) / columns;
  return static_cast<unsigned>(blocks < most ? blocks : most > 0 ? most : 1);
}

template <typename I>
int table_gradient(const I* tokens, const float* grad, float* dtable, int64_t rows, int width, float scale, int64_t count,
                   uint32_t* ws, hipStream_t stream) {
  const EmbeddingSpace s(rows, width, count);
  const int n = static_cast<int>(count);
  uint32_t* keys[2] = {ws + s.keys[0], ws + s.keys[1]};
  int32_t* places[2] = {reinterpret_cast<int32_t*>(ws + s.places[0]), reinterpret_cast<int32_t*>(ws + s.places[1])};
  int2* spans = reinterpret_cast<int2*>(ws + s.spans);
  float* parts = reinterpret_cast<float*>(ws + s.parts);
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
  const int sorted = now ^ 1, threads = row_threads(width), columns = (width + 4 * threads - 1) / (4 * threads);
  const int groups = kEmbThreads / threads;
  hipLaunchKernelGGL(embedding_chunk_kernel, dim3((s.chunks + groups - 1) / groups, columns), dim3(kEmbThreads), 0, stream,
                     keys[sorted], places[sorted], grad, dtable, parts, spans, static_cast<uint32_t>(rows), width, scale,
                     n, s.chunks, threads);
  hipLaunchKernelGGL(embedding_join_kernel, dim3(row_grid(rows, threads, columns), columns), dim3(kEmbThreads), 0, stream,
                     parts, spans, dtable, rows, width, scale, s.chunks, threads);
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
  const dim3 grid(row_grid(count, threads, columns), columns);
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
  return EmbeddingSpace(rows, width, count).size;
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
