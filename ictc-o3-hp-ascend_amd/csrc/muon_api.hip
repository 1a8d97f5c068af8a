// Orthogonalised updates of matrices: moving averages of gradients brought near an orthogonal matrix by
// Newton-Schulz products, many matrices at a time, gfx950.
//
//   M <- beta M + (1 - beta) g     U = beta M + (1 - beta) g  (or M)     X = U / (|U| + eps)
//   steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X           (on the shorter side, m <= n)
//   P <- (1 - lr wd) P - rate X
//
// Precision.  A singular value goes through p(s) = a s + b s^3 + c s^5 in every step, so small ones grow by a = 3.4
// each time and an error of X with them: products in bfloat16 would leave updates with 2 correct digits.  A product
// here is of about float32 accuracy on the float16 matrix cores: 2^11 x = hi + lo with hi = f16(2^11 x) and lo = f16(2^11 x - hi),
// 22 bits or an absolute 2^-36, whichever is larger (entries of X and A are near 1 and below), and
//   x y = 2^-22 (hi hi' + hi lo' + lo hi')  + (2^-22 x y, left out)
// in one float32 accumulator (sides of up to 32: float32 products).  Three products at 16 times the float32 instructions'
// rate.  Against 64 bits, errors of 14 kinds of matrices, rank-deficient ones among them, are 0.56 to 1.52 times those of
// a float32 iteration on the CPU (0.43 to 1.14 times with this card's library products): the bits that x has less than a
// float's 24 weigh less than the roundings of float32 sums, but they do weigh at sides of 200 and more.  What a power of
// two is chosen for grows at most 32-fold: |X| stays near 1 with coefficients for which the iteration is of use.  A
// matrix with |U| below eps, where X stays small, is kept times another power of two (2^e, see exponent_at), so that it
// has as many bits.  (The form that iterates A alone and multiplies X once has a third of the work for wide matrices, but
// doubles the error's growth: singular values below 1e-3 of the largest come out wrong, 1e-4 of the result at
// rank-deficient matrices.)
//
// Matrices with a shorter side of more than 128: all three products are of the form P Q^T with both operands' rows along
// the reduction (X X^T, A A^T, B (X^T)^T), so one kernel does them; X is kept in both orientations.  A and B are
// symmetric: only tiles on and above the diagonal are computed.  Every matrix of every tensor takes part in the same
// launches: `owner` says which matrix a workgroup's tile belongs to.  Sides are padded with zeros to whole tiles, which
// stay zero.  16 matrices of 1024 x 1024 and 8 of 1024 x 4096: average 106 us and normalise 169 (5.7 and 4.8 TB/s), then
// each step X X^T 204, B 111, B X 358 us, 850 TFLOP/s of float16 instructions over all (a large float16 product of the
// library 1,090).  By the counters B X reads 0.92 GB from memory (three times X^T and B: several XCDs take the same rows) and
// writes 0.40 (3.7 TB/s), takes 4.2 GB from the L2 (12 TB/s of 19) and keeps the matrix cores busy for 41 % of the cycles:
// none of them alone is the bound.
//
// Matrices with a shorter side of up to 128, of which most models have most: two launches a step, bound by latency.  A
// workgroup keeps 128 columns of X at a time: it multiplies them by B, and adds what they give to the next X X^T at
// once, from LDS; the other launch, one workgroup to a matrix, adds these parts up in order, and makes A A and B: 6.6
// and 4.6 us for the 29 matrices (64 rows or columns) of a C64 / lmax 2 model, 11.7 and 8.5 for the 47 (128) of a C128 /
// lmax 3 one.  (Done by the workgroup that is the last of its matrix to leave its part, it saves a launch, but what makes
// the parts of others visible within one costs more: a step of the C128 model's matrices 35 us against 23.)
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <new>
#include <vector>

#include "ictc_hip.h"

namespace ictc {
namespace {

constexpr int kMuThreads = 256;
constexpr int kMuWave = 64;
constexpr int kTensorsPerLaunch = 44;        // of the table in the kernel's arguments
constexpr int kPrep = 64;                    // side of a tile of the source
constexpr int kStep = 32;                    // reduction entries in LDS at a time
constexpr int64_t kMostBytes = int64_t{2} << 30;     // workspace that a call goes by, unless one matrix needs more

using half8 = _Float16 __attribute__((ext_vector_type(8)));
using half4 = _Float16 __attribute__((ext_vector_type(4)));
using f32x16 = float __attribute__((ext_vector_type(16)));
typedef float mf4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr float kScale = 2048.f, kUnscale = 1.f / kScale;      // of X and A as they are kept
constexpr int kMostExponent = 200;           // (2^-149 is the smallest number)

// One tensor's matrices, as the host describes them.
struct MuonTensor {
  const float* src;          // gradient, or the matrix itself
  float* momentum;           // null: src is the matrix
  float* out;                // parameter, or the result
  int64_t base;              // of the first matrix, in bytes of the workspace
  int32_t rows, cols, batches, first;          // first: index of the first matrix
  uint32_t prep, sym, apply, chunk;            // first tile (or chunk of columns) of each kind
  float rate;                // of the update, times the learning rate
};

struct MuonTable {
  MuonTensor tensor[kTensorsPerLaunch];
  int32_t count;
};

static_assert(sizeof(MuonTable) + 320 <= 4096, "kernel arguments are limited to 4 KB");
static_assert(kTensorsPerLaunch <= kMuWave, "a wave looks through the table");

// One matrix, in the workspace.  With a shorter side of up to 128: X^T [np][mp], two planes; B [mp][mp]; the parts of
// X X^T.  Else: X [mp][np], two planes; then X^T twice [np][mp], A and B [mp][mp].
struct MuonMatrix {
  const float* src;
  float* momentum;
  float* out;
  char* x;
  int32_t rows, cols, mp, np;
  uint32_t prep, prep_across;                  // tiles of the source
  uint32_t sym, apply;                         // tiles of products
  uint32_t chunk, chunks, chunk_parts;         // chunks of columns, of `chunk_parts` times kPart
  float rate;
  int32_t transposed;                          // more rows than columns
  uint32_t owner;                              // its index
};

// The first kind keeps planes of hi and lo parts; the second one 32 hi parts and their 32 lo parts side by side (kPair
// halves apart), so that a tile's load of 32 reduction entries takes whole lines of memory.
constexpr int kPair = 32;

__host__ __device__ constexpr int64_t paired_at(int64_t row, int64_t column, int64_t wide) {
  return (row * wide + column / kPair * kPair) * 2 + column % kPair;
}

struct MuonArgs {
  const MuonMatrix* matrices;
  const MuonMatrix* chunks;  // the matrix of each chunk of columns (a copy: one load less to wait for)
  const uint32_t *prep_owner, *sym_owner, *apply_owner;
  double* squares;           // of each tile of the source
  int32_t* exponents;        // of each matrix: X is kept times 2^e at first
  const float* clip;
  const float* lr_device;
  double weight_decay, eps;
  float beta, rest, lr;      // rest: 1 - beta
  float a, b, c;
  float b_kept, c_kept, unpoly;      // b and c for B as it is kept, from A and A A as they are; B's scale, inverse
  int32_t nesterov;
};

__device__ __forceinline__ bool skipped(const MuonArgs& a) { return a.clip && a.clip[1] != a.clip[1]; }

constexpr int64_t up_to(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

constexpr int kShort = 128;                  // shorter sides of matrices that are done in chunks of columns
constexpr int kPart = 128;                   // columns in LDS at a time
constexpr int kChunks = 24;                  // of a matrix, unless they get longer than kLongest parts
constexpr int kLongest = 4;
constexpr int kShortThreads = 512;

// Tiles and bytes of one matrix; sides padded to multiples of T, or for short ones to 32, 64 or 128 and kPart.
struct MuonSize {
  bool is_short;
  int64_t mp, np, prep, across, sym, apply, chunks, parts, bytes;
};

template <int T>
__host__ __device__ MuonSize muon_size(int64_t rows, int64_t cols) {
  MuonSize s;
  const int64_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  s.is_short = m <= kShort;
  if (s.is_short) {
    s.mp = m <= 32 ? 32 : m <= 64 ? 64 : 128, s.np = up_to(n, kPart);
    s.across = (cols + kPrep - 1) / kPrep;
    s.prep = (rows + kPrep - 1) / kPrep * s.across;
    const int64_t all = s.np / kPart, blocks = s.mp / 32;
    s.parts = (all + kChunks - 1) / kChunks;
    if (s.parts > kLongest) s.parts = kLongest;
    s.chunks = (all + s.parts - 1) / s.parts;
    s.sym = s.apply = 0;
    s.bytes = up_to(4 * s.np * s.mp + 4 * s.mp * s.mp + s.chunks * (blocks * (blocks + 1) / 2) * 4096, 256);
    return s;
  }
  s.mp = up_to(m, T), s.np = up_to(n, T);
  s.across = (rows > cols ? s.mp : s.np) / kPrep;
  s.prep = (s.mp / kPrep) * (s.np / kPrep);
  const int64_t i = s.mp / T, j = s.np / T;
  s.sym = i * (i + 1) / 2;
  s.apply = i * j;
  s.chunks = s.parts = 0;
  s.bytes = 12 * s.mp * s.np + 8 * s.mp * s.mp;
  return s;
}

// Where the descriptions and the owners of tiles lie.
struct MuonTables {
  char* workspace;
  MuonMatrix *matrices, *chunks;
  uint32_t *prep_owner, *sym_owner, *apply_owner;
};

template <int T>
__device__ __forceinline__ MuonMatrix matrix_of(const MuonTensor& t, const MuonSize& s, char* workspace, int b) {
  const int64_t values = static_cast<int64_t>(t.rows) * t.cols;
  MuonMatrix m;
  m.src = t.src + b * values;
  m.momentum = t.momentum ? t.momentum + b * values : nullptr;
  m.out = t.out + b * values;
  m.x = workspace + t.base + b * s.bytes;
  m.rows = t.rows, m.cols = t.cols, m.mp = static_cast<int32_t>(s.mp), m.np = static_cast<int32_t>(s.np);
  m.prep = t.prep + static_cast<uint32_t>(b * s.prep), m.prep_across = static_cast<uint32_t>(s.across);
  m.sym = t.sym + static_cast<uint32_t>(b * s.sym);
  m.apply = t.apply + static_cast<uint32_t>(b * s.apply);
  m.chunk = t.chunk + static_cast<uint32_t>(b * s.chunks), m.chunks = static_cast<uint32_t>(s.chunks);
  m.chunk_parts = static_cast<uint32_t>(s.parts);
  m.rate = t.rate;
  m.transposed = t.rows > t.cols;
  m.owner = t.first + static_cast<uint32_t>(b);
  return m;
}

// Descriptions of a tensor's matrices, and the owners of their tiles.
template <int T>
__device__ __forceinline__ void describe(const MuonTensor& t, const MuonTables& to) {
  const MuonSize s = muon_size<T>(t.rows, t.cols);
  for (int b = threadIdx.x; b < t.batches; b += kMuThreads) {
    const MuonMatrix m = matrix_of<T>(t, s, to.workspace, b);
    to.matrices[m.owner] = m;
  }
  for (int64_t k = threadIdx.x; k < t.batches * s.chunks; k += kMuThreads)
    to.chunks[t.chunk + k] = matrix_of<T>(t, s, to.workspace, static_cast<int>(k / s.chunks));
  const auto own = [&](uint32_t* owner, uint32_t first, int64_t each) {
    for (int64_t k = threadIdx.x; k < t.batches * each; k += kMuThreads)
      owner[first + k] = t.first + static_cast<uint32_t>(k / each);
  };
  if (!s.is_short) own(to.prep_owner, t.prep, s.prep);
  own(to.sym_owner, t.sym, s.sym);
  own(to.apply_owner, t.apply, s.apply);
}

// A tile of the source: its first row and column there, and what of it there is.
struct SourceTile {
  int r0, c0, rows, cols;

  __device__ __forceinline__ SourceTile(const MuonMatrix& m, uint32_t tile) {
    r0 = static_cast<int>(tile / m.prep_across) * kPrep;
    c0 = static_cast<int>(tile % m.prep_across) * kPrep;
    rows = m.rows - r0 < 0 ? 0 : m.rows - r0 > kPrep ? kPrep : m.rows - r0;
    cols = m.cols - c0 < 0 ? 0 : m.cols - c0 > kPrep ? kPrep : m.cols - c0;
  }
};

template <int THREADS = kMuThreads>
__device__ __forceinline__ double muon_block_sum(double x, double* part) {
#pragma unroll
  for (int d = kMuWave / 2; d; d >>= 1) x += __shfl_xor(x, d);
  if ((threadIdx.x & (kMuWave - 1)) == 0) part[threadIdx.x / kMuWave] = x;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / kMuWave; ++w) sum += part[w];
  return sum;
}

// The moving average and what is orthogonalised; each product and sum rounded for itself.
__device__ __forceinline__ float averaged(const MuonArgs& a, float m, float g) {
#pragma clang fp contract(off)
  return a.beta * m + a.rest * g;
}

// Global memory behind addresses that come out of memory, which the compiler cannot tell from LDS by itself.
template <typename V, typename T>
__device__ __forceinline__ V from_global(const T* p) {
  return *reinterpret_cast<const V __attribute__((address_space(1)))*>(reinterpret_cast<uintptr_t>(p));
}

template <typename V, typename T>
__device__ __forceinline__ void to_global(T* p, const V& v) {
  *reinterpret_cast<V __attribute__((address_space(1)))*>(reinterpret_cast<uintptr_t>(p)) = v;
}

// Four values of a row at any alignment, or the `count` that there are (zeros for the rest).
__device__ __forceinline__ mf4 load_quad(const float* p, int count) {
  mf4 v = {0.f, 0.f, 0.f, 0.f};
  if (count >= 4) return from_global<mf4>(p);
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < count) v[j] = from_global<float>(p + j);
  return v;
}

__device__ __forceinline__ void store_quad(float* p, int count, const mf4& v) {
  if (count >= 4) {
    to_global<mf4>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < count) to_global<float>(p + j, v[j]);
  }
}

constexpr int kQuadRows = kMuThreads / (kPrep / 4), kPasses = kPrep / kQuadRows;   // a tile's rows at a time, and times

// Moving averages, and the sum of squares (in 64 bits) of each tile of what is orthogonalised.  Bound by memory: 12
// bytes a value (momentum read and written, gradient read); all loads before the first store.  The last workgroups
// describe the table's tensors, one each, for the launches behind.
template <int T>
__global__ void __launch_bounds__(kMuThreads)
muon_average_kernel(const MuonTable table, const MuonArgs a, const MuonTables to, uint32_t first_tile, uint32_t tiles) {
  __shared__ double part[kMuThreads / kMuWave];
  if (blockIdx.x >= tiles) {
    describe<T>(table.tensor[blockIdx.x - tiles], to);
    return;
  }
  if (skipped(a)) return;
  // the tensor that the tile is of: the last one that begins at or before it
  const uint32_t tile = first_tile + blockIdx.x;
  const int lane = threadIdx.x & (kMuWave - 1);
  const int at = __builtin_amdgcn_readfirstlane(
      __popcll(__ballot(lane < table.count && table.tensor[lane < table.count ? lane : 0].prep <= tile)) - 1);
  const MuonTensor& tensor = table.tensor[at];
  const MuonSize size = muon_size<T>(tensor.rows, tensor.cols);
  const MuonMatrix m = matrix_of<T>(tensor, size, nullptr, static_cast<int>((tile - tensor.prep) / static_cast<uint32_t>(size.prep)));
  const SourceTile t(m, tile - m.prep);
  const float scale = a.clip ? a.clip[1] : 1.f;
  const int column = threadIdx.x % (kPrep / 4) * 4, count = t.cols - column, first = threadIdx.x / (kPrep / 4);
  const int64_t from = static_cast<int64_t>(t.r0 + first) * m.cols + t.c0 + column;
  mf4 u[kPasses], old[kPasses];
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    const int64_t at = from + static_cast<int64_t>(k * kQuadRows) * m.cols;
    const int there = first + k * kQuadRows < t.rows ? count : 0;
    u[k] = load_quad(m.src + at, there);
    if (m.momentum) old[k] = load_quad(m.momentum + at, there);
  }
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    if (m.momentum) {
      mf4 g = u[k];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        g[j] *= scale;
        old[k][j] = u[k][j] = averaged(a, old[k][j], g[j]);
        if (a.nesterov) u[k][j] = averaged(a, u[k][j], g[j]);
      }
      store_quad(m.momentum + from + static_cast<int64_t>(k * kQuadRows) * m.cols,
                 first + k * kQuadRows < t.rows ? count : 0, old[k]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += static_cast<double>(u[k][j]) * static_cast<double>(u[k][j]);
  }
  sum = muon_block_sum(sum, part);
  if (threadIdx.x == 0) a.squares[tile] = sum;
}

// (Both parts are of one float: left to itself the compiler may fold the product or sum behind it into one of two
// conversions to float16, and a tie that is none before it is rounded then gives another hi than lo is the rest of: an
// error of 2^-11 at one entry in 10^4.)
__device__ __forceinline__ void split(float x, _Float16& hi, _Float16& lo) {
  asm("" : "+v"(x));
  hi = static_cast<_Float16>(x);
  lo = static_cast<_Float16>(x - static_cast<float>(hi));
}

__device__ __forceinline__ float joined(_Float16 hi, _Float16 lo) {
  return static_cast<float>(hi) + static_cast<float>(lo);
}

// The same, or (SINGLE: sides of up to 32, whose products are float32 ones) the two halves of a float's bits, in the same
// places.
template <bool SINGLE>
__device__ __forceinline__ void split_for(float x, _Float16& hi, _Float16& lo) {
  if constexpr (SINGLE) {
    const uint32_t bits = __float_as_uint(x);
    hi = __builtin_bit_cast(_Float16, static_cast<uint16_t>(bits >> 16));
    lo = __builtin_bit_cast(_Float16, static_cast<uint16_t>(bits));
  } else {
    split(x, hi, lo);
  }
}

template <bool SINGLE>
__device__ __forceinline__ float joined_for(_Float16 hi, _Float16 lo) {
  if constexpr (SINGLE)
    return __uint_as_float(static_cast<uint32_t>(__builtin_bit_cast(uint16_t, hi)) << 16 | __builtin_bit_cast(uint16_t, lo));
  else
    return joined(hi, lo);
}

// The power of two that X is kept with before a step, from the one at first: |X| <= 2^-e, and a step multiplies it by at
// most |a| + |b| 4^-e + |c| 16^-e.
__device__ __forceinline__ int exponent_at(const MuonArgs& a, int e, int step) {
  for (; step && e; --step) {
    const float most = fabsf(a.a) + ldexpf(fabsf(a.b), -2 * e) + ldexpf(fabsf(a.c), -4 * e);
    e -= most > 1.f ? ilogbf(most) + 1 : 0;
    e = e < 0 ? 0 : e;
  }
  return e;
}

// What a matrix's values are multiplied by at first, as a float in [1, 2) and a power of two, which comes first: with
// both a value is at most 2^11 (|X| <= 1), so floats of any size stay in range, and the smallest lose no bits.
struct Scale {
  float mantissa;
  int exponent;

  __device__ __forceinline__ float of(float x) const { return ldexpf(x, exponent) * mantissa; }
};

// That scale from the matrix's tiles' squares (its power of two among it); every workgroup of the matrix calls it, and
// the one that is told to keeps the exponent.
template <int THREADS = kMuThreads>
__device__ __forceinline__ Scale first_scale(const MuonArgs& a, const MuonMatrix& m, uint32_t owner, bool keeps,
                                              double* part) {
  double sum = 0.0;
  // (the tiles that the source has, not those of its padding, which goes by the call's other matrices)
  const uint32_t across = (m.cols + kPrep - 1) / kPrep, tiles = (m.rows + kPrep - 1) / kPrep * across;
  for (uint32_t k = threadIdx.x; k < tiles; k += THREADS)
    sum += a.squares[m.prep + (across == m.prep_across ? k : k / across * m.prep_across + k % across)];
  const double norm = sqrt(muon_block_sum<THREADS>(sum, part)), share = norm / (norm + a.eps);
  const int e = share > 0.0 && share < 0.5 ? min(-ilogb(share) - 1, kMostExponent) : 0;
  if (threadIdx.x == 0 && keeps) a.exponents[owner] = e;
  const double scale = norm == 0.0 ? 1.0 : kScale / (norm + a.eps);      // (zeros stay zeros, however small eps is)
  const int power = ilogb(scale);
  return {static_cast<float>(ldexp(scale, -power)), power + e};
}

// Values of what is orthogonalised, from the source and (after muon_average_kernel) the moving average.
struct Source {
  mf4 g, m;

  __device__ __forceinline__ void load(const MuonArgs& a, const MuonMatrix& m_, int64_t at, int count) {
    if (!m_.momentum || a.nesterov) g = load_quad(m_.src + at, count);
    if (m_.momentum) m = load_quad(m_.momentum + at, count);
  }

  // Four of a column, as many of them as there are.
  __device__ __forceinline__ void load_down(const MuonArgs& a, const MuonMatrix& m_, int64_t at, int count) {
    g = m = mf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < count) {
        const int64_t from = at + static_cast<int64_t>(r) * m_.cols;
        if (!m_.momentum || a.nesterov) g[r] = from_global<float>(m_.src + from);
        if (m_.momentum) m[r] = from_global<float>(m_.momentum + from);
      }
  }

  __device__ __forceinline__ float value(const MuonArgs& a, const MuonMatrix& m_, int j, float scale, const Scale& first) const {
    return first.of(!m_.momentum ? g[j] : a.nesterov ? averaged(a, m[j], scale * g[j]) : m[j]);
  }
};

// X in both orientations from the source: tiles go through LDS.
__global__ void __launch_bounds__(kMuThreads) muon_normalise_kernel(const MuonArgs a) {
  __shared__ double part[kMuThreads / kMuWave];
  __shared__ float tile[kPrep][kPrep + 1];
  if (skipped(a)) return;
  const uint32_t owner = a.prep_owner[blockIdx.x];
  const MuonMatrix m = a.matrices[owner];
  const SourceTile t(m, blockIdx.x - m.prep);
  const int column = threadIdx.x % (kPrep / 4) * 4, first = threadIdx.x / (kPrep / 4);
  Source source[kPasses];
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    const int r = first + k * kQuadRows;
    source[k].load(a, m, static_cast<int64_t>(t.r0 + r) * m.cols + t.c0 + column, r < t.rows ? t.cols - column : 0);
  }
  const Scale inv = first_scale(a, m, owner, blockIdx.x == m.prep, part);
  const float scale = a.clip ? a.clip[1] : 1.f;
#pragma unroll
  for (int k = 0; k < kPasses; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) tile[first + k * kQuadRows][column + j] = source[k].value(a, m, j, scale, inv);
  __syncthreads();
  const int64_t values = static_cast<int64_t>(m.mp) * m.np;
  _Float16* const x = reinterpret_cast<_Float16*>(m.x);
#pragma unroll
  for (int side = 0; side < 2; ++side) {           // as it is, and transposed
    _Float16* to = x + ((side != 0) == (m.transposed != 0) ? 0 : 2 * values);
    const int64_t wide = (side != 0) == (m.transposed != 0) ? m.np : m.mp;
    const int first = side ? t.c0 : t.r0, along = side ? t.r0 : t.c0;
    for (int k = threadIdx.x; k < kPrep * kPrep / 8; k += kMuThreads) {
      const int r = k / (kPrep / 8), c = k % (kPrep / 8) * 8;
      half8 hi, lo;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        _Float16 h, l;
        split(side ? tile[c + j][r] : tile[r][c + j], h, l);
        hi[j] = h, lo[j] = l;
      }
      const int64_t at = paired_at(first + r, along + c, wide);
      to_global<half8>(to + at, hi);
      to_global<half8>(to + at + kPair, lo);
    }
  }
}

enum MuonPhase { kGram, kPoly, kApply, kLast, kFirst };

// The power of two that a product's results are multiplied by.
template <int PHASE>
__device__ __forceinline__ int shift_of(const MuonArgs& a, uint32_t owner, int step) {
  if constexpr (PHASE == kPoly || PHASE == kFirst) return 0;
  const int first = a.exponents[owner];
  if (!first) return 0;
  const int e = exponent_at(a, first, step);
  return PHASE == kGram ? -2 * e : PHASE == kApply ? exponent_at(a, first, step + 1) - e : -e;
}

// The last step's results: the matrix itself, or a parameter's update.
struct Update {
  float keep = 1.f, rate = 0.f;

  __device__ __forceinline__ Update() {}
  __device__ __forceinline__ Update(const MuonArgs& a, const MuonMatrix& m) {
    if (!m.momentum) return;
    const float lr = a.lr_device ? *a.lr_device : a.lr;
    keep = static_cast<float>(1.0 - static_cast<double>(lr) * a.weight_decay);
    rate = lr * m.rate;
  }

  // Consecutive results along a row of the result, from (row, column) on.
  template <int N>
  __device__ __forceinline__ void write(const MuonMatrix& m, int row, int column, const float (&v)[N]) const {
    if (row >= m.rows) return;
    float* const to = m.out + static_cast<int64_t>(row) * m.cols + column;
#pragma unroll
    for (int q = 0; q < N; q += 4) {
      const int count = m.cols - column - q;
      if (count <= 0) return;
      mf4 t = m.momentum ? load_quad(to + q, count) : mf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 4; ++r) t[r] = m.momentum ? keep * t[r] - rate * (v[q + r] * kUnscale) : v[q + r] * kUnscale;
      store_quad(to + q, count, t);
    }
  }
};

// 16 bytes a lane from global memory to consecutive places of LDS.
__device__ __forceinline__ void load_to_lds(const _Float16* from, _Float16* to) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint32_t __attribute__((address_space(1)))*>(
                                       reinterpret_cast<uintptr_t>(from)),
                                   reinterpret_cast<uint32_t __attribute__((address_space(3)))*>(
                                       static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to))),
                                   16, 0, 0);
}

// Workgroups go to the 8 XCDs in turn, and each has a cache of its own: 16 tiles in a row, which share rows of their
// operands, go to the same one (X X^T of 24 matrices of 1 to 4 million values 209 us, with 32 in a row 236 for the
// imbalance of long reductions, without 250).
constexpr uint32_t kXcds = 8, kUnit = 16;

__device__ __forceinline__ uint32_t tile_of(uint32_t block) {
  return (block / (kXcds * kUnit) * kXcds + block % kXcds) * kUnit + block / kXcds % kUnit;
}

int64_t tile_grid(int64_t tiles) { return up_to(tiles, kXcds * kUnit); }

// At most N of the wave's loads are still on their way, and then all waves go on: a barrier that leaves the others in
// flight (__syncthreads waits for all).
template <int N>
__device__ __forceinline__ void wait_for_loads() {
  if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  else if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  else if constexpr (N == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// All waves have their operands out of LDS.
__device__ __forceinline__ void wait_for_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Where an entry of a tile of results lies in LDS: rows of a column side by side, in groups of four that are turned with
// the column, so that neither 16 columns' groups nor 16 groups of 8 columns' single entries meet in a bank.
template <int T>
__device__ __forceinline__ int tile_at(int column, int row) {
  return column * T + (row ^ (((column ^ (column >> 3)) & (T < 64 ? T / 4 - 1 : 15)) * 4));
}

// One tile of P Q^T: T x T, four waves of (T/2) x (T/2).  Rows of 32 reduction entries (128 bytes with both parts) lie in
// LDS in eight groups of 16 bytes, whose order is turned with the row so that 16 rows' groups fill all banks; they come
// straight from global memory (a lane picks the group that belongs to its place), one step ahead of the products.
template <int T, int PHASE>
__global__ void __launch_bounds__(kMuThreads, 2) muon_product_kernel(const MuonArgs a, uint32_t tiles, int step) {
  constexpr int N = T / 64;                        // 32 x 32 products of a wave, each way
  __shared__ __align__(16) _Float16 lds[2][2][T * 2 * kStep];     // rows of P and of Q, hi and lo parts
  static_assert(sizeof(lds) >= sizeof(float) * T * T);
  float* const results = reinterpret_cast<float*>(lds);             // of the tile, behind the last step
  if (skipped(a)) return;
  constexpr bool kSym = PHASE == kGram || PHASE == kPoly;
  const uint32_t tile = tile_of(blockIdx.x);
  if (tile >= tiles) return;
  const uint32_t owner = (kSym ? a.sym_owner : a.apply_owner)[tile];
  const MuonMatrix m = a.matrices[owner];
  const int parity = step & 1;
  const uint32_t local = tile - (kSym ? m.sym : m.apply);
  int ti, tj;
  if constexpr (kSym) {
    tj = static_cast<int>((sqrtf(8.f * local + 1.f) - 1.f) * 0.5f);
    while (static_cast<uint32_t>(tj + 1) * (tj + 2) / 2 <= local) ++tj;
    while (static_cast<uint32_t>(tj) * (tj + 1) / 2 > local) --tj;
    ti = static_cast<int>(local) - tj * (tj + 1) / 2;
  } else {
    const uint32_t down = m.mp / T;
    ti = static_cast<int>(local % down), tj = static_cast<int>(local / down);
  }
  const int64_t values = static_cast<int64_t>(m.mp) * m.np;
  _Float16* const x = reinterpret_cast<_Float16*>(m.x);
  _Float16* const xt = x + 2 * values * (1 + parity);               // X^T now, and what it becomes
  _Float16* const xt_next = x + 2 * values * (2 - parity);
  _Float16* const gram = x + 6 * values;
  _Float16* const poly = gram + 2 * static_cast<int64_t>(m.mp) * m.mp;
  const _Float16* const p = PHASE == kGram ? x : PHASE == kPoly ? gram : poly;
  const _Float16* const q = PHASE == kGram ? x : PHASE == kPoly ? gram : xt;
  const int depth = PHASE == kGram ? m.np : m.mp;

  const int lane = threadIdx.x & (kMuWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kMuWave);
  const int wi = (wave & 1) * (T / 2), wj = (wave >> 1) * (T / 2);
  // (16 lanes read 16 rows at a time, from 64 banks: the groups of every other row are in the same ones)
  const auto turned = [](int row) { return (row >> 1) & 7; };
  const auto fetch = [&](int at, int buffer) {
    // a wave's load fills 8 rows, both parts of them; the tile has T / 8 of them for each operand
#pragma unroll
    for (int k = 0; k < T / 16; ++k) {
      const int piece = k * 4 + wave, which = piece / (T / 8), first = piece % (T / 8) * 8;
      const int row = first + lane / 8, group = (lane & 7) ^ turned(row);
      const _Float16* base = which ? q + static_cast<int64_t>(tj * T + row) * depth * 2
                                   : p + static_cast<int64_t>(ti * T + row) * depth * 2;
      load_to_lds(base + at * (2 * kStep) + group * 8, &lds[buffer][which][first * 2 * kStep]);
    }
  };
  // Two steps' rows are in LDS or on their way there.  A step's operands go to registers as a whole, so that its place
  // in LDS is free for the step after the next while its products run.
  constexpr int kLoads = T / 16;                   // of a wave and step
  f32x16 acc[N][N] = {};
  const int steps = depth / kStep;
  fetch(0, 0);
  if (steps > 1) fetch(1, 1);
  for (int s = 0; s < steps; ++s) {
    const int buffer = s & 1;
    if (s + 1 < steps) wait_for_loads<kLoads>(); else wait_for_loads<0>();
    half8 op[kStep / 16][4][N];
#pragma unroll
    for (int k = 0; k < kStep / 16; ++k)
#pragma unroll
      for (int which = 0; which < 4; ++which)
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int row = (which < 2 ? wi : wj) + n * 32 + (lane & 31), group = (which & 1) * 4 + k * 2 + lane / 32;
          op[k][which][n] = *reinterpret_cast<const half8*>(&lds[buffer][which / 2][row * 2 * kStep + (group ^ turned(row)) * 8]);
        }
    if (s + 2 < steps) {
      wait_for_lds();
      fetch(s + 2, buffer);
    }
#pragma unroll
    for (int k = 0; k < kStep / 16; ++k)
      // (hi lo', lo hi', hi hi': consecutive instructions go to different accumulators)
#pragma unroll
      for (int c = 0; c < 3; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j)
            acc[i][j] =
                __builtin_amdgcn_mfma_f32_32x32x16_f16(op[k][c == 1 ? 1 : 0][i], op[k][c == 0 ? 3 : 2][j], acc[i][j], 0, 0, 0);
  }
  __syncthreads();

  // Results leave through LDS, in whole lines.  A lane holds rows 8 (k / 4) + 4 (lane / 32) + k % 4 of column lane % 32 of
  // each 32 x 32 product.  Below the diagonal of a symmetric result stands the mirror image of what is above it, in blocks
  // of 64 within a tile as in whole tiles (hi lo' and lo hi' are added up in another order there): a matrix has the same
  // bits with both sizes of tiles, whatever else is in the call.
  const bool mirrors = kSym && T > 64 && ti == tj;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        const int row = wi + i * 32 + 2 * k + 4 * (lane / 32), column = wj + j * 32 + (lane & 31);
        mf4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = acc[i][j][k + r];
        if (!mirrors || wi <= wj) *reinterpret_cast<mf4*>(&results[tile_at<T>(column, row)]) = v;
        if (mirrors && wi < wj) {
#pragma unroll
          for (int r = 0; r < 4; ++r) results[tile_at<T>(row + r, column)] = v[r];
        }
      }
  __syncthreads();
  const int shift = shift_of<PHASE>(a, owner, step);
  const Update update = PHASE == kLast ? Update(a, m) : Update();
  // columns of the tile, 8 rows of one at a time: rows of what has its rows along the shorter side
  for (int unit = threadIdx.x; unit < T * T / 8; unit += kMuThreads) {
    const int column = unit / (T / 8), row = unit % (T / 8) * 8;
    const int64_t across = paired_at(tj * T + column, ti * T + row, m.mp);
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; q += 4) {
      const mf4 t = *reinterpret_cast<const mf4*>(&results[tile_at<T>(column, row + q)]);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[q + r] = t[r];
    }
    if constexpr (PHASE == kGram) {
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] *= kUnscale;
    } else {
      const _Float16* old = (PHASE == kPoly ? gram : xt) + across;
      const half8 hi = from_global<half8>(old), lo = from_global<half8>(old + kPair);
#pragma unroll
      for (int r = 0; r < 8; ++r)
        v[r] = PHASE == kPoly ? fmaf(a.b_kept, joined(hi[r], lo[r]), a.c_kept * v[r])
                              : fmaf(a.a, joined(hi[r], lo[r]), a.unpoly * v[r]);
    }
    if (PHASE != kPoly && shift) {
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] = ldexpf(v[r], shift);
    }
    uint32_t kept[8];
    if constexpr (PHASE == kLast) {
      if (m.transposed) update.write<8>(m, tj * T + column, ti * T + row, v);
#pragma unroll
      for (int r = 0; r < 8; ++r) kept[r] = __float_as_uint(v[r]);
    } else {
      _Float16* const mirror = (PHASE == kGram ? gram : PHASE == kPoly ? poly : xt_next) + across;
      half8 hi, lo;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        _Float16 h, l;
        split(v[r], h, l);
        hi[r] = h, lo[r] = l;
        kept[r] = __builtin_bit_cast(uint16_t, h) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, l)) << 16;
      }
      to_global<half8>(mirror, hi);
      to_global<half8>(mirror + kPair, lo);
    }
#pragma unroll
    for (int q = 0; q < 8; q += 4)
      *reinterpret_cast<mf4*>(&results[tile_at<T>(column, row + q)]) =
          mf4{__uint_as_float(kept[q]), __uint_as_float(kept[q + 1]), __uint_as_float(kept[q + 2]),
              __uint_as_float(kept[q + 3])};
  }
  if (kSym ? ti == tj : PHASE == kLast && m.transposed) return;      // (a tile on the diagonal holds its mirror image)
  __syncthreads();
  // rows of the tile, 8 columns of one at a time
  _Float16* const plain = PHASE == kGram ? gram : PHASE == kPoly ? poly : x;
  const int64_t wide = PHASE == kApply ? m.np : m.mp;
  for (int unit = threadIdx.x; unit < T * T / 8; unit += kMuThreads) {
    const int row = unit / (T / 8), column = unit % (T / 8) * 8;
    uint32_t kept[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) kept[r] = __float_as_uint(results[tile_at<T>(column + r, row)]);
    if constexpr (PHASE == kLast) {
      float v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] = __uint_as_float(kept[r]);
      update.write<8>(m, ti * T + row, tj * T + column, v);
    } else {
      half8 hi, lo;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        hi[r] = __builtin_bit_cast(_Float16, static_cast<uint16_t>(kept[r]));
        lo[r] = __builtin_bit_cast(_Float16, static_cast<uint16_t>(kept[r] >> 16));
      }
      _Float16* const to = plain + paired_at(ti * T + row, tj * T + column, wide);
      to_global<half8>(to, hi);
      to_global<half8>(to + kPair, lo);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// Matrices with a shorter side of up to 128
// ---------------------------------------------------------------------------------------------------------

// Where the group of 8 halves `group` of row `row` lies in LDS, rows of `groups` such groups: turned with the row, so
// that the groups that 16 lanes read fill all 64 banks.
__device__ __forceinline__ int turn_of(int row, int groups) { return row / (16 / groups) & (groups - 1); }

__device__ __forceinline__ int turned_at(int row, int group, int groups) {
  return (row * groups + (group ^ turn_of(row, groups))) * 8;
}

// Block `b` of the upper triangle, column by column.
__device__ __forceinline__ void upper_block(int b, int& i, int& j) {
  j = b >= 6 ? 3 : b >= 3 ? 2 : b >= 1 ? 1 : 0;
  i = b - j * (j + 1) / 2;
}

// (Two accumulators: a product waits for the one before it in the same accumulator twice as long as it takes to issue.)
// SINGLE: float32 products of float32 values, for sides of up to 32, where too few terms are added up for what is left
// out to cancel.  Errors of 64 x 8, 2 x 40 and 5 x 5 with columns of different size 5.3, 4.4 and 5.1e-7 of the result's
// norm; 6.1, 6.5 and 6.2 with values of two halves, more with the three products; 6.6, 6.1 and 5.7 with library products
// in float32.  These matrices' workgroups wait for the larger ones' either way.  (Which of 16 columns a lane's value is
// does not matter, as both operands have the same.)
template <bool SINGLE>
__device__ __forceinline__ void three_products(const half8& ah, const half8& al, const half8& bh, const half8& bl,
                                               f32x16& high, f32x16& low) {
  if constexpr (SINGLE) {
#pragma unroll
    for (int r = 0; r < 8; r += 2) {
      high = __builtin_amdgcn_mfma_f32_32x32x2f32(joined_for<true>(ah[r], al[r]), joined_for<true>(bh[r], bl[r]), high, 0, 0, 0);
      low = __builtin_amdgcn_mfma_f32_32x32x2f32(joined_for<true>(ah[r + 1], al[r + 1]),
                                                 joined_for<true>(bh[r + 1], bl[r + 1]), low, 0, 0, 0);
    }
    return;
  }
  low = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, low, 0, 0, 0);
  high = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, high, 0, 0, 0);
  low = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, low, 0, 0, 0);
}

// Where an entry of B lies: in the order in which a wave's lanes take it as an operand, 32 rows and 16 columns at a
// time, so that a load is one piece of memory.
template <int M>
__device__ __forceinline__ int operand_at(int row, int column) {
  return ((row / 32 * (M / 16) + column / 16) * 64 + column % 16 / 8 * 32 + row % 32) * 8 + column % 8;
}

// LDS of a chunk's workgroup: kPart columns of X, as their rows lie in X^T; the last step's results.
struct ShortLds {
  _Float16 xt[2][kPart * kShort];
  double part[kShortThreads / kMuWave];
};

using short4v = short __attribute__((ext_vector_type(4)));

// Eight entries along the columns of a row of X (a lane's operand for X X^T), from rows of X^T in LDS: the hardware turns
// blocks of 4 of its rows and 16 of its columns as it reads them, 16 lanes to a block.  row0: first of the wave's 32 rows
// of X; j0: first of 16 columns, of which a lane has those from 8 (lane / 32) on.
__device__ __forceinline__ half8 turned_operand(const _Float16* plane, int row0, int j0, int groups) {
  const int lane = threadIdx.x & (kMuWave - 1), of = lane & 15;
  const int row = row0 + (lane & 16) + (of & 3) * 4, j = j0 + lane / 32 * 8 + of / 4;
  half8 v;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const _Float16* const from = plane + turned_at(j + 4 * q, row / 8, groups) + row % 8;
    const short4v t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        reinterpret_cast<short4v __attribute__((address_space(3)))*>(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from))));
#pragma unroll
    for (int r = 0; r < 4; ++r) v[4 * q + r] = __builtin_bit_cast(_Float16, static_cast<uint16_t>(t[r]));
  }
  return v;
}

// The products of one chunk of columns, MB x 32 rows (see the top).  kFirst: the columns come from the source.
template <int PHASE, int MB>
__device__ __forceinline__ void short_chunk(const MuonArgs& a, const MuonMatrix& m, int step, ShortLds& lds) {
  constexpr int kWaves = kShortThreads / kMuWave;
  constexpr int M = 32 * MB, kGroups = M / 8, kBlocks = MB * (MB + 1) / 2, kMine = (kBlocks + kWaves - 1) / kWaves;
  constexpr int kTiles = MB == 4 ? 2 : 1;          // 32 x 32 products of a wave
  const int lane = threadIdx.x & (kMuWave - 1), half = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kMuWave);
  const int64_t plane = static_cast<int64_t>(m.np) * M;
  _Float16* const xt = reinterpret_cast<_Float16*>(m.x);
  const _Float16* const poly = xt + 2 * plane;
  const uint32_t chunk = blockIdx.x - m.chunk;
  const int first = static_cast<int>(chunk * m.chunk_parts), all = m.np / kPart;
  const int end = first + static_cast<int>(m.chunk_parts) < all ? first + static_cast<int>(m.chunk_parts) : all;
  const int row0 = wave % MB * 32, col0 = wave / MB * (32 * kTiles);        // of a wave's products
  const bool works = col0 < kPart;
  f32x16 gram[kMine] = {};

  for (int part = first; part < end; ++part) {
    _Float16* const columns = xt + static_cast<int64_t>(part) * kPart * M;
    if constexpr (PHASE == kFirst) {
      // four values of a column of X at a time: of a row of the source if it is transposed, else of four rows
      // (a loop, not straight code: instructions that run once have to be fetched, too)
      constexpr int kQuads = M * kPart / 4 / kShortThreads, kAtOnce = kQuads < 4 ? kQuads : 4;
      const float scale = a.clip ? a.clip[1] : 1.f;
      const Scale inv = first_scale<kShortThreads>(a, m, m.owner, chunk == 0 && part == first, lds.part);
#pragma unroll 1
      for (int base = 0; base < kQuads; base += kAtOnce) {
        Source source[kAtOnce];
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          const int k = (base + q) * kShortThreads + threadIdx.x;
          if (m.transposed) {
            const int row = k / (M / 4) + part * kPart, column = k % (M / 4) * 4;
            source[q].load(a, m, static_cast<int64_t>(row) * m.cols + column, row < m.rows ? m.cols - column : 0);
          } else {
            const int row = k / kPart * 4, column = k % kPart + part * kPart;
            source[q].load_down(a, m, static_cast<int64_t>(row) * m.cols + column, column < m.cols ? m.rows - row : 0);
          }
        }
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
          const int k = (base + q) * kShortThreads + threadIdx.x;
          half4 hi, lo;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            _Float16 h, l;
            split_for<MB == 1>(source[q].value(a, m, r, scale, inv), h, l);
            hi[r] = h, lo[r] = l;
          }
          const int i = m.transposed ? k % (M / 4) * 4 : k / kPart * 4, j = m.transposed ? k / (M / 4) : k % kPart;
          const int to = turned_at(j, i / 8, kGroups) + i % 8;
          *reinterpret_cast<half4*>(&lds.xt[0][to]) = hi;
          *reinterpret_cast<half4*>(&lds.xt[1][to]) = lo;
        }
      }
    } else {
      // a wave's load fills 64 groups of a plane
#pragma unroll
      for (int k = 0; k < 2 * kPart * kGroups / kShortThreads; ++k) {
        const int piece = k * kWaves + wave, p = piece / (kPart * kGroups / 64), group = piece % (kPart * kGroups / 64) * 64;
        const int j = (group + lane) / kGroups, turned = (group + lane) % kGroups ^ turn_of(j, kGroups);
        load_to_lds(columns + p * plane + (j * kGroups + turned) * 8, &lds.xt[p][group * 8]);
      }
      half8 b_op[2][M / 16];
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int k = 0; k < M / 16; ++k)
          b_op[p][k] = from_global<half8>(poly + p * M * M + operand_at<M>(row0, k * 16) + lane * 8);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      f32x16 acc[kTiles] = {};
      if (works) {
        f32x16 low[kTiles] = {};
#pragma unroll
        for (int k = 0; k < M / 16; ++k)
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const int from = turned_at(col0 + t * 32 + (lane & 31), k * 2 + half, kGroups);
            three_products<MB == 1>(b_op[0][k], b_op[1][k], *reinterpret_cast<const half8*>(&lds.xt[0][from]),
                           *reinterpret_cast<const half8*>(&lds.xt[1][from]), acc[t], low[t]);
          }
#pragma unroll
        for (int t = 0; t < kTiles; ++t) acc[t] += low[t];
      }
      const int shift = shift_of<PHASE>(a, m.owner, step);
      __syncthreads();         // all products have their operands: their places take the results
      if (works) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int k = 0; k < 16; k += 4) {
            const int row = row0 + 2 * k + 4 * half, j = col0 + t * 32 + (lane & 31);
            const int at = turned_at(j, row / 8, kGroups) + row % 8;
            half4 hi = *reinterpret_cast<const half4*>(&lds.xt[0][at]), lo = *reinterpret_cast<const half4*>(&lds.xt[1][at]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float v = fmaf(a.a, joined_for<MB == 1>(hi[r], lo[r]), a.unpoly * acc[t][k + r]);
              if (shift) v = ldexpf(v, shift);
              if constexpr (PHASE == kLast) {
                acc[t][k + r] = v;
              } else {
                _Float16 h, l;
                split_for<MB == 1>(v, h, l);
                hi[r] = h, lo[r] = l;
              }
            }
            if constexpr (PHASE != kLast) {
              *reinterpret_cast<half4*>(&lds.xt[0][at]) = hi;
              *reinterpret_cast<half4*>(&lds.xt[1][at]) = lo;
            }
          }
      }
      if constexpr (PHASE == kLast) {
        __syncthreads();
        float* const results = reinterpret_cast<float*>(lds.xt);
        static_assert(sizeof(lds.xt) >= sizeof(float) * kPart * M);
        if (works) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int k = 0; k < 16; k += 4)
              *reinterpret_cast<mf4*>(&results[tile_at<M>(col0 + t * 32 + (lane & 31), row0 + 2 * k + 4 * half)]) =
                  mf4{acc[t][k], acc[t][k + 1], acc[t][k + 2], acc[t][k + 3]};
        }
        __syncthreads();
        const Update update(a, m);
        for (int unit = threadIdx.x; unit < kPart * M / 8; unit += kShortThreads) {
          float v[8];
          const int j = m.transposed ? unit / (M / 8) : unit % (kPart / 8) * 8;
          const int i = m.transposed ? unit % (M / 8) * 8 : unit / (kPart / 8);
#pragma unroll
          for (int r = 0; r < 8; ++r) v[r] = results[m.transposed ? tile_at<M>(j, i + r) : tile_at<M>(j + r, i)];
          if (m.transposed) update.write<8>(m, part * kPart + j, i, v); else update.write<8>(m, i, part * kPart + j, v);
        }
      }
    }
    __syncthreads();
    if constexpr (PHASE != kLast) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int k = 0; k < kPart * kGroups / kShortThreads; ++k) {
          const int group = k * kShortThreads + threadIdx.x;
          to_global<half8>(columns + p * plane + group * 8,
                           *reinterpret_cast<const half8*>(&lds.xt[p][turned_at(group / kGroups, group % kGroups, kGroups)]));
        }
#pragma unroll
      for (int q = 0; q < kMine; ++q) {
        const int b = wave + kWaves * q;
        if (b >= kBlocks) continue;
        int bi, bj;
        upper_block(b, bi, bj);
        f32x16 low = {};
#pragma unroll 2
        for (int k = 0; k < kPart; k += 16)
          three_products<MB == 1>(turned_operand(lds.xt[0], bi * 32, k, kGroups), turned_operand(lds.xt[1], bi * 32, k, kGroups),
                         turned_operand(lds.xt[0], bj * 32, k, kGroups), turned_operand(lds.xt[1], bj * 32, k, kGroups),
                         gram[q], low);
        gram[q] += low;
      }
      if (part + 1 < end) __syncthreads();
    }
  }
  if constexpr (PHASE != kLast) {
    float* const parts = reinterpret_cast<float*>(xt + 2 * plane + 2 * M * M) + static_cast<int64_t>(chunk) * kBlocks * 1024;
#pragma unroll
    for (int q = 0; q < kMine; ++q) {
      const int b = wave + kWaves * q;
      if (b >= kBlocks) continue;
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        mf4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = gram[q][k + r] * kUnscale;
        to_global<mf4>(parts + b * 1024 + (k / 4 * 64 + lane) * 4, v);
      }
    }
  }
}

template <int PHASE>
__global__ void __launch_bounds__(kShortThreads) muon_chunk_kernel(const MuonArgs a, int step) {
  __shared__ __align__(16) ShortLds lds;
  if (skipped(a)) return;
  const MuonMatrix m = a.chunks[blockIdx.x];
  if (m.mp == 128) short_chunk<PHASE, 4>(a, m, step, lds);
  else if (m.mp == 64) short_chunk<PHASE, 2>(a, m, step, lds);
  else short_chunk<PHASE, 1>(a, m, step, lds);
}

constexpr int kPolyThreads = 512;

// A from its chunks' parts, in order, and B = b A + c A A: a workgroup to a matrix.
template <int MB>
__device__ __forceinline__ void short_poly(const MuonArgs& a, const MuonMatrix& m, uint32_t owner, int step,
                                           _Float16 (*lds)[kShort * kShort]) {
  constexpr int M = 32 * MB, kGroups = M / 8, kBlocks = MB * (MB + 1) / 2, kQuads = kBlocks * 256;
  constexpr int kMine = (kQuads + kPolyThreads - 1) / kPolyThreads;
  const int lane = threadIdx.x & (kMuWave - 1), half = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kMuWave);
  const int64_t plane = static_cast<int64_t>(m.np) * M;
  _Float16* const poly = reinterpret_cast<_Float16*>(m.x) + 2 * plane;
  const float* const parts = reinterpret_cast<const float*>(poly + 2 * M * M);
  const int shift = shift_of<kGram>(a, owner, step);
  mf4 sum[kMine] = {};
  constexpr int kAhead = MB == 4 ? 4 : 12;         // chunks whose parts are on their way at a time
  for (uint32_t first = 0; first < m.chunks; first += kAhead) {
    mf4 v[kAhead][kMine];
#pragma unroll
    for (int c = 0; c < kAhead; ++c)
#pragma unroll
      for (int q = 0; q < kMine; ++q) {
        const int quad = q * kPolyThreads + threadIdx.x;
        v[c][q] = mf4{0.f, 0.f, 0.f, 0.f};
        if (quad < kQuads && first + c < m.chunks)
          v[c][q] = from_global<mf4>(parts + (static_cast<int64_t>(first + c) * kQuads + quad) * 4);
      }
#pragma unroll
    for (int c = 0; c < kAhead; ++c)
#pragma unroll
      for (int q = 0; q < kMine; ++q)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[q][r] += v[c][q][r];
  }
#pragma unroll
  for (int q = 0; q < kMine; ++q) {
    const int quad = q * kPolyThreads + threadIdx.x;
    if (quad >= kQuads) continue;
    int bi, bj;
    upper_block(quad / 256, bi, bj);
    const int of = quad % 64, row = bi * 32 + quad % 256 / 64 * 8 + 4 * (of / 32), column = bj * 32 + (of & 31);
    half4 hi, lo;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      _Float16 h, l;
      split_for<MB == 1>(shift ? ldexpf(sum[q][r], shift) : sum[q][r], h, l);
      hi[r] = h, lo[r] = l;
      if (bi != bj) {
        const int to = turned_at(row + r, column / 8, kGroups) + column % 8;
        lds[0][to] = h, lds[1][to] = l;
      }
    }
    const int to = turned_at(column, row / 8, kGroups) + row % 8;
    *reinterpret_cast<half4*>(&lds[0][to]) = hi;
    *reinterpret_cast<half4*>(&lds[1][to]) = lo;
  }
  __syncthreads();
  // (a wave's blocks side by side)
  constexpr int kWaves = kPolyThreads / kMuWave, kEach = (kBlocks + kWaves - 1) / kWaves;
  f32x16 acc[kEach] = {}, low[kEach] = {};
#pragma unroll
  for (int k = 0; k < M / 16; ++k)
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const int b = wave + q * kWaves;
      if (b >= kBlocks) continue;
      int bi, bj;
      upper_block(b, bi, bj);
      const int i = turned_at(bi * 32 + (lane & 31), k * 2 + half, kGroups);
      const int j = turned_at(bj * 32 + (lane & 31), k * 2 + half, kGroups);
      three_products<MB == 1>(*reinterpret_cast<const half8*>(&lds[0][i]), *reinterpret_cast<const half8*>(&lds[1][i]),
                     *reinterpret_cast<const half8*>(&lds[0][j]), *reinterpret_cast<const half8*>(&lds[1][j]), acc[q], low[q]);
    }
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    const int b = wave + q * kWaves;
    if (b >= kBlocks) continue;
    int bi, bj;
    upper_block(b, bi, bj);
#pragma unroll
    for (int k = 0; k < 16; k += 4) {
      const int row = bi * 32 + 2 * k + 4 * half, column = bj * 32 + (lane & 31);
      const int from = turned_at(column, row / 8, kGroups) + row % 8;
      const half4 old_hi = *reinterpret_cast<const half4*>(&lds[0][from]);
      const half4 old_lo = *reinterpret_cast<const half4*>(&lds[1][from]);
      half4 hi, lo;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        _Float16 h, l;
        const float old = joined_for<MB == 1>(old_hi[r], old_lo[r]);
        split_for<MB == 1>(fmaf(a.b_kept, old, a.c_kept * (acc[q][k + r] + low[q][k + r])), h, l);
        hi[r] = h, lo[r] = l;
        if (bi != bj) {
          to_global<_Float16>(poly + operand_at<M>(row + r, column), h);
          to_global<_Float16>(poly + M * M + operand_at<M>(row + r, column), l);
        }
      }
      to_global<half4>(poly + operand_at<M>(column, row), hi);
      to_global<half4>(poly + M * M + operand_at<M>(column, row), lo);
    }
  }
}

__global__ void __launch_bounds__(kPolyThreads) muon_short_poly_kernel(const MuonArgs a, uint32_t first, int step) {
  __shared__ _Float16 lds[2][kShort * kShort];
  if (skipped(a)) return;
  const uint32_t owner = first + blockIdx.x;
  const MuonMatrix m = a.matrices[owner];
  if (m.mp == 128) short_poly<4>(a, m, owner, step, lds);
  else if (m.mp == 64) short_poly<2>(a, m, owner, step, lds);
  else short_poly<1>(a, m, owner, step, lds);
}

constexpr int64_t kMostSide = 1 << 20;
constexpr int64_t kMostMatrices = int64_t{1} << 23;
constexpr int64_t kFewTiles = 512;
constexpr int64_t kMostTiles = int64_t{1} << 23;      // of a launch: threads within 32 bits
constexpr int64_t kMostChunks = (int64_t{1} << 31) / (kShortThreads > kPolyThreads ? kShortThreads : kPolyThreads);

// A matrix of a call: of which tensor, and which of its matrices.
struct MuonPlace {
  int64_t tensor, matrix;
};

// A call's matrices up to `end` that take part in the same launches, and what they need.
struct MuonGroup {
  MuonPlace end;
  int64_t matrices, prep, sym, apply, chunks, bytes;

  void add(const MuonSize& s, int64_t batches) {
    matrices += batches, prep += batches * s.prep, sym += batches * s.sym, apply += batches * s.apply;
    chunks += batches * s.chunks, bytes += batches * s.bytes;
  }

  // Where the tables and the matrices lie in the workspace.
  int64_t at_prep() const { return up_to(matrices * static_cast<int64_t>(sizeof(MuonMatrix)), 256); }
  int64_t at_sym() const { return at_prep() + up_to(4 * prep, 256); }
  int64_t at_apply() const { return at_sym() + up_to(4 * sym, 256); }
  int64_t at_chunk() const { return at_apply() + up_to(4 * apply, 256); }
  int64_t at_squares() const { return at_chunk() + up_to(chunks * static_cast<int64_t>(sizeof(MuonMatrix)), 256); }
  int64_t at_exponents() const { return at_squares() + up_to(8 * prep, 256); }
  int64_t at_values() const { return at_exponents() + up_to(4 * matrices, 256); }
  int64_t size() const { return at_values() + bytes; }
};

// (Tensors that take no part are counted: the groups, and with them the workspace, go by the shapes alone.)  A stack
// of matrices is split where the group is full, so that no launch and no workspace grows with its length.
template <int T>
MuonGroup muon_group(const int64_t* rows, const int64_t* cols, const int64_t* batches, MuonPlace first, int64_t count) {
  MuonGroup g = {};
  MuonPlace at = first;
  while (at.tensor < count) {
    const int64_t k = at.tensor;
    if (rows[k] && cols[k] && at.matrix < batches[k]) {
      const MuonSize s = muon_size<T>(rows[k], cols[k]);
      int64_t fits = std::min({batches[k] - at.matrix, (kMostBytes - g.bytes) / s.bytes, (kMostTiles - g.prep) / s.prep,
                               kMostChunks - g.matrices});
      if (s.chunks) fits = std::min(fits, (kMostChunks - g.chunks) / s.chunks);
      if (!g.matrices) fits = std::max(fits, int64_t{1});
      if (fits <= 0) break;
      g.add(s, fits);
      at.matrix += fits;
      if (at.matrix < batches[k]) break;
    }
    ++at.tensor, at.matrix = 0;
  }
  g.end = at;
  return g;
}

bool muon_valid(const int64_t* rows, const int64_t* cols, const int64_t* batches, int64_t count) {
  if (count < 0 || count > 0x7fffffff || (count && (!rows || !cols || !batches))) return false;
  for (int64_t k = 0; k < count; ++k) {
    if (rows[k] < 0 || rows[k] > kMostSide || cols[k] < 0 || cols[k] > kMostSide || batches[k] < 0 ||
        batches[k] > kMostMatrices)
      return false;
    if (!rows[k] || !cols[k] || !batches[k]) continue;
    const MuonSize s = muon_size<128>(rows[k], cols[k]);
    if (s.prep > kMostTiles) return false;
  }
  return true;
}

bool muon_valid(const ictc_muon_desc* d, const float* lr_device) {
  if (!d) return false;
  for (const double c : d->coefficients)
    if (!isfinite(c)) return false;
  return d->beta >= 0.0 && d->beta < 1.0 && d->weight_decay >= 0.0 && d->eps > 0.0 && isfinite(d->eps) &&
         (lr_device || d->lr >= 0.f) && d->steps >= 1 && d->steps <= ICTC_MUON_MAX_STEPS &&
         (d->adjust == ICTC_MUON_SHAPE || d->adjust == ICTC_MUON_MATCH_RMS);
}

int muon_launched() { return hipGetLastError() == hipSuccess ? ICTC_OK : ICTC_ERR_LAUNCH; }

// Whether products go by tiles of 128 x 128 (and sides are padded to that): where these alone fill the chip twice.  They
// read half as much from LDS for a product as tiles of 64 x 64.
bool large_tiles(const int64_t* rows, const int64_t* cols, const int64_t* batches, int64_t count) {
  int64_t tiles = 0;
  for (int64_t k = 0; k < count; ++k)
    if (rows[k] && cols[k] && batches[k]) tiles += batches[k] * muon_size<128>(rows[k], cols[k]).apply;
  return tiles >= kFewTiles;
}

template <int T>
int64_t muon_workspace(const int64_t* rows, const int64_t* cols, const int64_t* batches, int64_t count) {
  int64_t most = 0;
  for (MuonPlace at = {}; at.tensor < count;) {
    const MuonGroup g = muon_group<T>(rows, cols, batches, at, count);
    if (g.size() > most) most = g.size();
    at = g.end;
  }
  return most;
}

int64_t muon_workspace(const int64_t* rows, const int64_t* cols, const int64_t* batches, int64_t count) {
  return large_tiles(rows, cols, batches, count) ? muon_workspace<128>(rows, cols, batches, count)
                                                 : muon_workspace<64>(rows, cols, batches, count);
}

template <int T>
int muon_run(const float* const* src, float* const* momentum, float* const* out, const int64_t* rows,
             const int64_t* cols, const int64_t* batches, int64_t count, const ictc_muon_desc* d, const float* clip,
             const float* lr_device, char* ws, int64_t ws_bytes, hipStream_t stream) {
  MuonArgs a;
  a.clip = clip, a.lr_device = lr_device;
  a.weight_decay = d->weight_decay, a.eps = d->eps;
  a.beta = static_cast<float>(d->beta), a.rest = static_cast<float>(1.0 - d->beta), a.lr = d->lr;
  a.a = static_cast<float>(d->coefficients[0]), a.b = static_cast<float>(d->coefficients[1]);
  a.c = static_cast<float>(d->coefficients[2]);
  // B as it is kept: below 2^15 for |X| up to 1.5
  const double most = 2.25 * fabs(d->coefficients[1]) + 5.0625 * fabs(d->coefficients[2]);
  const double poly = most > 16.0 ? ldexp(kScale, -ilogb(most / 16.0) - 1) : kScale;
  a.b_kept = static_cast<float>(d->coefficients[1] * poly / kScale);
  a.c_kept = static_cast<float>(d->coefficients[2] * poly / kScale / kScale);
  a.unpoly = static_cast<float>(1.0 / poly);
  a.nesterov = d->nesterov;
  for (MuonPlace from = {}; from.tensor < count;) {
    const MuonGroup g = muon_group<T>(rows, cols, batches, from, count);
    if (g.size() > ws_bytes) return ICTC_ERR_INVALID_ARGUMENT;
    MuonMatrix* const matrices = reinterpret_cast<MuonMatrix*>(ws);
    const auto owners = [&](int64_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
    uint32_t* const prep = owners(g.at_prep());
    uint32_t* const sym = owners(g.at_sym());
    uint32_t* const apply = owners(g.at_apply());
    MuonMatrix* const chunk = reinterpret_cast<MuonMatrix*>(ws + g.at_chunk());
    a.matrices = matrices, a.prep_owner = prep, a.sym_owner = sym, a.apply_owner = apply, a.chunks = chunk;
    const MuonTables tables{ws + g.at_values(), matrices, chunk, prep, sym, apply};
    a.squares = reinterpret_cast<double*>(ws + g.at_squares());
    a.exponents = reinterpret_cast<int32_t*>(ws + g.at_exponents());
    // those that take part, the ones with long shorter sides first
    MuonGroup at = {}, longs = {};
    MuonTable table;
    table.count = 0;
    int64_t sent = 0;        // tiles of the tables before
    const auto send = [&]() {
      if (!table.count) return static_cast<int>(ICTC_OK);
      hipLaunchKernelGGL(muon_average_kernel<T>, dim3(static_cast<unsigned>(at.prep - sent + table.count)), dim3(kMuThreads),
                         0, stream, table, a, tables, static_cast<uint32_t>(sent), static_cast<uint32_t>(at.prep - sent));
      table.count = 0, sent = at.prep;
      return muon_launched();
    };
    // (and of those the longest first: their tiles take longest)
    struct Piece {
      int64_t tensor, first, batches;
    };
    std::vector<Piece> order;
    for (MuonPlace p = from; p.tensor < count && p.tensor <= g.end.tensor; ++p.tensor, p.matrix = 0) {
      const int64_t t = p.tensor, stop = t < g.end.tensor ? batches[t] : g.end.matrix;
      if (src[t] && rows[t] && cols[t] && p.matrix < stop) order.push_back({t, p.matrix, stop - p.matrix});
    }
    const auto longer = [&](int64_t t) { return rows[t] > cols[t] ? rows[t] : cols[t]; };
    std::stable_sort(order.begin(), order.end(), [&](const Piece& x, const Piece& y) { return longer(x.tensor) > longer(y.tensor); });
    for (int shorts = 0; shorts < 2; ++shorts) {
      for (const Piece& piece : order) {
        const int64_t t = piece.tensor, before = piece.first * rows[t] * cols[t];
        const MuonSize s = muon_size<T>(rows[t], cols[t]);
        if (s.is_short != (shorts != 0)) continue;
        const double r = static_cast<double>(rows[t]), c = static_cast<double>(cols[t]);
        MuonTensor& e = table.tensor[table.count++];
        e.src = src[t] + before, e.momentum = momentum ? momentum[t] + before : nullptr, e.out = out[t] + before;
        e.base = at.bytes, e.rows = static_cast<int32_t>(rows[t]), e.cols = static_cast<int32_t>(cols[t]);
        e.batches = static_cast<int32_t>(piece.batches), e.first = static_cast<int32_t>(at.matrices);
        e.prep = static_cast<uint32_t>(at.prep), e.sym = static_cast<uint32_t>(at.sym);
        e.apply = static_cast<uint32_t>(at.apply), e.chunk = static_cast<uint32_t>(at.chunks);
        e.rate = static_cast<float>(d->adjust == ICTC_MUON_SHAPE ? sqrt(r > c ? r / c : 1.0) : 0.2 * sqrt(r > c ? r : c));
        at.add(s, piece.batches);
        if (table.count == kTensorsPerLaunch)
          if (const int rc = send()) return rc;
      }
      if (!shorts) longs = at;
    }
    if (const int rc = send()) return rc;
    from = g.end;
    if (!at.matrices) continue;
    const auto launch = [&](void (*kernel)(MuonArgs, int), int64_t grid, int step) {
      if (grid) hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(kShortThreads), 0, stream, a, step);
    };
    const auto product = [&](void (*kernel)(MuonArgs, uint32_t, int), int64_t tiles, int step) {
      if (tiles)
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tile_grid(tiles))), dim3(kMuThreads), 0, stream, a,
                           static_cast<uint32_t>(tiles), step);
    };
    if (longs.matrices)
      hipLaunchKernelGGL(muon_normalise_kernel, dim3(static_cast<unsigned>(longs.prep)), dim3(kMuThreads), 0, stream, a);
    launch(muon_chunk_kernel<kFirst>, at.chunks, 0);
    for (int step = 0; step < d->steps; ++step) {
      const bool last = step + 1 == d->steps;
      product(muon_product_kernel<T, kGram>, longs.sym, step);
      product(muon_product_kernel<T, kPoly>, longs.sym, step);
      product(last ? muon_product_kernel<T, kLast> : muon_product_kernel<T, kApply>, longs.apply, step);
      const uint32_t first = static_cast<uint32_t>(longs.matrices);
      if (at.matrices > longs.matrices)
        hipLaunchKernelGGL(muon_short_poly_kernel, dim3(static_cast<unsigned>(at.matrices - longs.matrices)),
                           dim3(kPolyThreads), 0, stream, a, first, step);
      launch(last ? muon_chunk_kernel<kLast> : muon_chunk_kernel<kApply>, at.chunks, step);
      if (const int rc = muon_launched()) return rc;
    }
  }
  return ICTC_OK;
}

// (No C++ exception leaves through the C interface.)
int muon_call(const float* const* src, float* const* momentum, float* const* out, const int64_t* rows,
              const int64_t* cols, const int64_t* batches, int64_t count, const ictc_muon_desc* d, const float* clip,
              const float* lr_device, void* ws, int64_t ws_bytes, hipStream_t stream) {
  const auto run = large_tiles(rows, cols, batches, count) ? muon_run<128> : muon_run<64>;
  try {
    return run(src, momentum, out, rows, cols, batches, count, d, clip, lr_device, static_cast<char*>(ws), ws_bytes,
               stream);
  } catch (const std::bad_alloc&) {
    return ICTC_ERR_LAUNCH;
  }
}

}  // namespace
}  // namespace ictc

extern "C" {

int64_t ictc_hip_muon_workspace(const int64_t* rows, const int64_t* cols, const int64_t* batches, int64_t count) {
  using namespace ictc;
  if (!muon_valid(rows, cols, batches, count)) return -ICTC_ERR_INVALID_ARGUMENT;
  return muon_workspace(rows, cols, batches, count);
}

int ictc_hip_orthogonalize(const float* const* in, float* const* out, const int64_t* rows, const int64_t* cols,
                           const int64_t* batches, int64_t count, const ictc_muon_desc* desc, void* workspace,
                           int64_t workspace_bytes, hipStream_t stream) {
  using namespace ictc;
  if (!muon_valid(rows, cols, batches, count) || !muon_valid(desc, nullptr)) return ICTC_ERR_INVALID_ARGUMENT;
  const int64_t need = muon_workspace(rows, cols, batches, count);
  if (need == 0) return ICTC_OK;
  if (!in || !out || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < need)
    return ICTC_ERR_INVALID_ARGUMENT;
  for (int64_t k = 0; k < count; ++k)
    if (rows[k] && cols[k] && batches[k] && (!in[k] || !out[k])) return ICTC_ERR_INVALID_ARGUMENT;
  return muon_call(in, nullptr, out, rows, cols, batches, count, desc, nullptr, nullptr, workspace, workspace_bytes,
                   stream);
}

int ictc_hip_muon_step(float* const* params, const float* const* grads, float* const* momentum, const int64_t* rows,
                       const int64_t* cols, const int64_t* batches, int64_t count, const ictc_muon_desc* desc,
                       const float* clip, const float* lr_device, void* workspace, int64_t workspace_bytes,
                       hipStream_t stream) {
  using namespace ictc;
  if (!muon_valid(rows, cols, batches, count) || !muon_valid(desc, lr_device)) return ICTC_ERR_INVALID_ARGUMENT;
  const int64_t need = muon_workspace(rows, cols, batches, count);
  if (need == 0) return ICTC_OK;
  if (!params || !grads || !momentum || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) ||
      workspace_bytes < need)
    return ICTC_ERR_INVALID_ARGUMENT;
  for (int64_t k = 0; k < count; ++k)
    if (rows[k] && cols[k] && batches[k] && grads[k] && (!params[k] || !momentum[k])) return ICTC_ERR_INVALID_ARGUMENT;
  return muon_call(grads, momentum, params, rows, cols, batches, count, desc, clip, lr_device, workspace,
                   workspace_bytes, stream);
}

}  // extern "C"
