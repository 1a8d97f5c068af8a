// The optimizer step of a model's training: the norm of all gradients, and one AdamW update of many
// tensors with moments in float32 or in 8 bits, gfx950.
//
//   g  <- c G                                  c: the clipping coefficient (1 without clipping)
//   m  <- b1 m + (1 - b1) g                    v <- b2 v + (1 - b2) g^2
//   p  <- (1 - lr wd) p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// Every tensor is a flat array; its moments lie in one flat state for all tensors, each tensor at the
// start of a block of 256 values.  The tensors' addresses travel in the kernel's arguments (kTensors to
// a launch), so a step copies nothing to the device beforehand and can be captured into a graph.
//
// 8-bit moments.  A block of 256 values has one byte f, the biased exponent of its largest magnitude
// (raised by one if that lies above 1.75 in its binade, so that rounding up never needs the next one).
// Relative to 2^(f - 127) a value is a small floating number: m has a sign, 4 exponent and 3 mantissa
// bits, v has 5 exponent and 3 mantissa bits; both go down to zero through subnormal steps.  Such a code
// is the top byte of a float32's exponent and mantissa once the value is scaled into the lowest 16 (or
// 32) binades of float32, so encoding is one ldexp, one addition of random bits below the kept ones and
// a shift, and decoding a shift and an ldexp.  Three choices keep the moving averages alive:
//   * the scale is a power of two, so a value that does not change is stored again exactly; with a scale
//     like the block's maximum every value would be rounded anew in every step;
//   * rounding is stochastic.  With b2 = 0.999 a step changes v by about 0.1 %, far below half a code
//     step (3 to 6 %): rounded to nearest, v would never move;
//   * a v above zero is never stored as zero: its root is divided by.
// A value that is not finite is stored as not-a-number (m 0x7f, v 0xff).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "ictc_hip.h"

namespace ictc {
namespace {

constexpr int kWaveSize = 64;
constexpr int kThreads = 256;
constexpr int kQuant = ICTC_MOMENT_BLOCK;        // values that share a scale: one wave, 4 a lane
constexpr int kWaves = kThreads / kWaveSize;
constexpr int kTensors = 184;                    // 21 bytes each, within the 4 KB of kernel arguments
constexpr int kMaskTensors = 16384;
constexpr float kFastEps = 1e-11f;               // times 2^-24 above the root of the smallest normal float
constexpr int64_t kStream = int64_t{1} << 24;     // values of a launch that no cache holds until their next use
constexpr int64_t kMostGroups = int64_t{1} << 23;  // workgroups of a launch that streams (threads within 32 bits)

// Blocks that a wave takes at a time.
constexpr int step_blocks(bool small, bool past) { return small && past ? 4 : 1; }

constexpr int kSkip = 4096;                      // 1 M values
constexpr int kMaxBlocks = 2048;                 // 8 workgroups for each of 256 CUs (a launch that does not stream)
constexpr int kNormTensors = 200;                // 20 bytes each
constexpr int kNormChunk = 4096;
constexpr int kNormBlocks = 2048;

// The tensors of one launch, in the order of the flat state without gaps (one without a gradient has a
// null address there).  Tensor i has the state's blocks [start[i], start[i + 1]), counted from the
// launch's first, and its last block holds tail[i] values (256: 0).
struct StepTable {
  float* param[kTensors];
  const float* grad[kTensors];
  uint32_t start[kTensors + 1];
  uint8_t tail[kTensors];
  int64_t state;     // the launch's first block
  int64_t row;       // the first tensor's row in progress
  int32_t count;     // (of the host's)
  uint32_t blocks;
};

// The tensors that take part in a step, one bit each.
struct RowMask {
  uint32_t bits[kMaskTensors / 32];
  int64_t first;
  int32_t count;
};

struct StepArgs {
  void* exp_avg;
  void* exp_avg_sq;
  uint8_t* exp_avg_top;
  uint8_t* exp_avg_sq_top;
  double* progress;
  const float* clip;
  const float* lr_device;
  double beta1, beta2, weight_decay;
  float lr, eps;
  uint32_t seed;
};

static_assert(sizeof(StepTable) + sizeof(StepArgs) + 16 <= 4096, "kernel arguments are limited to 4 KB");

__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0xBB67AE85u;
  x ^= x >> 15;
  x *= 0x6A09E667u;
  return x ^ (x >> 16);
}

template <int CTRL>
__device__ __forceinline__ uint32_t max_with(uint32_t x) {
  const uint32_t o = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xf, 0xf, false));
  return x > o ? x : o;
}

// Largest of a wave's unsigned values, in every lane (uniform): rotations by 8, 4, 2 and 1 within the
// rows of 16 lanes, then the four rows.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max_with<0x121>(max_with<0x122>(max_with<0x124>(max_with<0x128>(x))));
  const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
  const uint32_t c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
  const uint32_t ab = a > b ? a : b, cd = c > d ? c : d;
  return ab > cd ? ab : cd;
}

// The codes of 4 values, a byte each.  m is the hardware's 8-bit float with 4 exponent bits (the largest
// exponent's last code is its not-a-number), 2^8 the first power of two above it.
__device__ __forceinline__ void decode_signed(uint32_t codes, int top, float* m) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes), false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes), true);
  m[0] = ldexpf(lo[0], top - 135);
  m[1] = ldexpf(lo[1], top - 135);
  m[2] = ldexpf(hi[0], top - 135);
  m[3] = ldexpf(hi[1], top - 135);
}

// v: 5 exponent and 3 mantissa bits; 0xff is not a number (looked for in all four at once).
__device__ __forceinline__ void decode_unsigned(uint32_t codes, int top, float* v) {
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = ldexpf(__uint_as_float(((codes >> (8 * k)) & 0xFFu) << 20), top - 31);
  if (((codes & 0x7F7F7F7Fu) + 0x01010101u) & codes & 0x80808080u) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (((codes >> (8 * k)) & 0xFFu) == 0xFFu) v[k] = __uint_as_float(0x7FC00000u);
  }
}

__device__ __forceinline__ uint32_t max3(uint32_t a, uint32_t b, uint32_t c) {
  const uint32_t ab = a > b ? a : b;
  return ab > c ? ab : c;
}

constexpr uint32_t kInf = 0x7F800000u;

// Exponent byte of a block from its values' magnitudes as integers; not finite: those left out (uniform).
__device__ __forceinline__ int block_top(const float* x, bool& finite) {
  uint32_t b[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) b[k] = __float_as_uint(x[k]) & 0x7FFFFFFFu;
  uint32_t largest = wave_max(max3(max3(b[0], b[1], b[2]), b[3], 0u));
  finite = largest < kInf;
  if (!finite) {
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = b[k] < kInf ? b[k] : 0u;
    largest = wave_max(max3(max3(b[0], b[1], b[2]), b[3], 0u));
  }
  const int f = static_cast<int>((largest + 0x1FFFFFu) >> 23);
  return f < 1 ? 1 : f;
}

// Four codes from values, their block's exponent byte and 16 random bits each.
__device__ __forceinline__ uint32_t encode_signed(const float* m, int top, bool finite, const uint32_t* random) {
  uint32_t out = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t x = __float_as_uint(ldexpf(fabsf(m[k]), 15 - top));
    uint32_t code = (x + ((random[k] & 0xFFFFu) << 4)) >> 20;
    if (!finite && !(fabsf(m[k]) < INFINITY)) code = 0x7Fu;
    code |= (__float_as_uint(m[k]) >> 24) & 0x80u;
    out |= code << (8 * k);
  }
  return out;
}

__device__ __forceinline__ uint32_t encode_unsigned(const float* v, int top, bool finite, const uint32_t* random) {
  uint32_t out = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t b = __float_as_uint(v[k]), least = b < 1u ? b : 1u;    // above zero: at least code 1
    uint32_t code = (__float_as_uint(ldexpf(v[k], 31 - top)) + ((random[k] >> 16) << 4)) >> 20;
    code = code > least ? code : least;
    if (!finite && !(v[k] < INFINITY)) code = 0xFFu;
    out |= code << (8 * k);
  }
  return out;
}

// Index of the last entry that is at most `value` (start[0] is, the unused ones are the largest number):
// every lane compares its share and the ones are counted.
template <int MOST>
__device__ __forceinline__ int entry_of(const uint32_t* start, uint32_t value) {
  const int lane = threadIdx.x & (kWaveSize - 1);
  int n = 0;
#pragma unroll
  for (int k = 0; k < MOST; k += kWaveSize)
    n += __popcll(__ballot(k + lane < MOST && start[k + lane < MOST ? k + lane : 0] <= value));
  return __builtin_amdgcn_readfirstlane(n - 1);
}

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

template <typename T>
__device__ __forceinline__ T* uniform(T* p) {
  const uint64_t x = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<T*>((static_cast<uint64_t>(uniform(static_cast<uint32_t>(x >> 32))) << 32) |
                              uniform(static_cast<uint32_t>(x)));
}

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <bool STREAM>
__device__ __forceinline__ void load4(const float* p, float* v) {
  const f32x4* q = reinterpret_cast<const f32x4*>(p);
  const f32x4 x = STREAM ? __builtin_nontemporal_load(q) : *q;
  v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
}

template <bool STREAM>
__device__ __forceinline__ void store4(float* p, const float* v) {
  const f32x4 x = {v[0], v[1], v[2], v[3]};
  f32x4* q = reinterpret_cast<f32x4*>(p);
  if constexpr (STREAM) __builtin_nontemporal_store(x, q); else *q = x;
}

// What the blocks of one tensor share.
struct StepScalars {
  float coefficient, keep, rate, inv2, b1, b2, n1, n2, eps;
  uint32_t key;
};

// The moving averages, each product and sum rounded for itself: the same bits as float32 arithmetic gives
// elsewhere.  With products fused into the sums one in 2 million 8-bit codes would be rounded the other way.
__device__ __forceinline__ void moments(const StepScalars& c, const float* g, float* m, float* v) {
#pragma clang fp contract(off)
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float gk = c.coefficient * g[k];
    m[k] = c.b1 * m[k] + c.n1 * gk;
    v[k] = c.b2 * v[k] + c.n2 * (gk * gk);
  }
}

// A parameter behind its step, for the approximate reciprocal r: products and the last sum rounded in one given way.
// Left to the compiler, variants of the kernel fused different products into the sum, and the last bit of a
// parameter depended on how many blocks its wave took with it.
__device__ __forceinline__ float stepped(const StepScalars& c, float p, float m, float r) {
#pragma clang fp contract(off)
  const float down = c.rate * m * r;
  return __builtin_fmaf(c.keep, p, -down);
}

// The update of U whole blocks (or, with U = 1, of the first `left` of each lane's values): four values a
// lane and block, all loads before the first store.
template <bool SMALL, bool STREAM, int U, bool WHOLE>
__device__ __forceinline__ void update(const StepArgs& a, const StepScalars& c, float* param, const float* grad,
                                       int64_t block, int left) {
  const int lane = threadIdx.x & (kWaveSize - 1);
  const int64_t s = block * kQuant + lane * 4;
  uint8_t* const codes_m = static_cast<uint8_t*>(a.exp_avg) + s;
  uint8_t* const codes_v = static_cast<uint8_t*>(a.exp_avg_sq) + s;
  float* const values_m = static_cast<float*>(a.exp_avg) + s;
  float* const values_v = static_cast<float*>(a.exp_avg_sq) + s;
  float p[U][4] = {}, g[U][4] = {}, m[U][4], v[U][4];
  uint32_t cm[U], cv[U];
  int tm[U], tv[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if constexpr (WHOLE) {
      load4<STREAM>(param + u * kQuant, p[u]);
      load4<STREAM>(grad + u * kQuant, g[u]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < left) p[u][k] = param[k], g[u][k] = grad[k];
    }
    if constexpr (SMALL) {
      cm[u] = *reinterpret_cast<const uint32_t*>(codes_m + u * kQuant);
      cv[u] = *reinterpret_cast<const uint32_t*>(codes_v + u * kQuant);
      tm[u] = a.exp_avg_top[block + u], tv[u] = a.exp_avg_sq_top[block + u];
    } else {
      load4<STREAM>(values_m + u * kQuant, m[u]);
      load4<STREAM>(values_v + u * kQuant, v[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if constexpr (SMALL) {
      decode_signed(cm[u], tm[u], m[u]);
      decode_unsigned(cv[u], tv[u], v[u]);
    }
    moments(c, g[u], m[u], v[u]);
    if (SMALL && c.eps >= kFastEps) {
      // Roots and reciprocals to the last bit but one, without the steps for denormal roots (eps covers
      // them): with the exact ones instructions bound this variant (100 M values: 279 us against 250).
#pragma unroll
      for (int k = 0; k < 4; ++k)
        p[u][k] = stepped(c, p[u][k], m[u][k],
                          __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[u][k] * c.inv2) + c.eps));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        p[u][k] = c.keep * p[u][k] - c.rate * m[u][k] / (sqrtf(v[u][k] * c.inv2) + c.eps);
    }
    if constexpr (WHOLE) {
      store4<STREAM>(param + u * kQuant, p[u]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < left) param[k] = p[u][k];
    }
    if constexpr (SMALL) {
      bool fm, fv;
      tm[u] = block_top(m[u], fm), tv[u] = block_top(v[u], fv);
      uint32_t random[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) random[k] = mix(static_cast<uint32_t>(s) + u * kQuant + k + c.key);
      *reinterpret_cast<uint32_t*>(codes_m + u * kQuant) = encode_signed(m[u], tm[u], fm, random);
      *reinterpret_cast<uint32_t*>(codes_v + u * kQuant) = encode_unsigned(v[u], tv[u], fv, random);
      if (lane == 0) {
        a.exp_avg_top[block + u] = static_cast<uint8_t>(tm[u]);
        a.exp_avg_sq_top[block + u] = static_cast<uint8_t>(tv[u]);
      }
    } else {
      store4<STREAM>(values_m + u * kQuant, m[u]);
      store4<STREAM>(values_v + u * kQuant, v[u]);
    }
  }
}

// One wave to U consecutive blocks of 256 values; the launch's waves sweep over the blocks side by side,
// so a wave changes tensors often: the table and each tensor's scalars are in LDS.
//
// Bound by memory: 28 bytes a value (8-bit moments 16). 150 M values in 120 tensors: 694 us (6.0 TB/s) with
// float32 moments and 377 us (6.4 TB/s) with 8-bit ones, a copy of the same size runs at 5.3 to 5.9.  What
// that took, from 835 and 535 us with a contiguous range of blocks for each of 2,048 workgroups: lookups
// from LDS and waves side by side (the ranges met on the same memory channels), no reuse asked of the
// caches (`STREAM`, from kStream values on; below, the caches hold a model: 8 M values 37 us against
// 40), a workgroup for each piece of work instead of 2,048 that go on, and with 8-bit moments four blocks a
// wave at a time (292 us at 100 M against 254; with float32 moments one is the better: 448 against 469).
// The 8-bit variant was bound by its instructions at first (66 % of issue slots): hardware conversions of
// m, codes of four values handled together, and approximate roots took 40 % of them.
template <bool SMALL, bool STREAM>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const StepTable table, const StepArgs a) {
  constexpr int U = step_blocks(SMALL, STREAM);
  __shared__ float* params[kTensors];
  __shared__ const float* grads[kTensors];
  __shared__ uint32_t starts[kTensors + 1];
  __shared__ uint32_t tails[kTensors];
  __shared__ float rates[kTensors], inv2s[kTensors];
  __shared__ uint32_t keys[kTensors];
  const int thread = threadIdx.x, lane = thread & (kWaveSize - 1);
  StepScalars c;
  c.coefficient = a.clip ? a.clip[1] : 1.f;
  const float lr = a.lr_device ? *a.lr_device : a.lr;
  if (thread < table.count) {
    const double* row = a.progress + 3 * (table.row + thread);
    const double steps = row[0], power1 = row[1], power2 = row[2];
    params[thread] = table.param[thread];
    grads[thread] = table.grad[thread];
    tails[thread] = table.tail[thread];
    rates[thread] = lr / static_cast<float>(1.0 - power1 * a.beta1);
    inv2s[thread] = 1.f / static_cast<float>(1.0 - power2 * a.beta2);
    keys[thread] = mix(a.seed + static_cast<uint32_t>(static_cast<int64_t>(steps) + 1) * 0x9E3779B9u);
  }
  if (thread <= kTensors) starts[thread] = table.start[thread];
  __syncthreads();
  if (c.coefficient != c.coefficient) return;    // a norm that is not finite: nothing changes
  c.keep = static_cast<float>(1.0 - static_cast<double>(lr) * a.weight_decay);
  c.b1 = static_cast<float>(a.beta1), c.b2 = static_cast<float>(a.beta2);
  c.n1 = static_cast<float>(1.0 - a.beta1), c.n2 = static_cast<float>(1.0 - a.beta2);
  c.eps = a.eps;
  const uint32_t blocks = table.blocks, stride = gridDim.x * (kWaves * U);
  int last = 0;
  uint32_t start = 0, next = 0;
  float* param = nullptr;
  const float* grad = nullptr;
  bool wide = false;
  for (uint32_t first = (blockIdx.x * kWaves + uniform(static_cast<uint32_t>(thread / kWaveSize))) * U; first < blocks;
       first += stride) {
    const uint32_t end = blocks - first < U ? blocks : first + U;
    for (uint32_t b = first; b < end;) {
      if (b >= next) {
        const int i = entry_of<kTensors>(starts, b);
        start = uniform(starts[i]), next = uniform(starts[i + 1]);
        param = uniform(params[i]), grad = uniform(grads[i]), last = uniform(tails[i]);
        wide = ((reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
        c.rate = rates[i], c.inv2 = inv2s[i], c.key = keys[i];
      }
      const int64_t at = static_cast<int64_t>(b - start) * kQuant + lane * 4;
      const uint32_t whole = wide ? next - (last != 0) : 0u;     // blocks before it can be read four values at a time
      if (!grad) {
        b = next < end ? next : end;
      } else if (U > 1 && b + U <= whole && b + U <= end) {
        update<SMALL, STREAM, U, true>(a, c, param + at, grad + at, table.state + b, 4);
        b += U;
      } else if (b < whole) {
        update<SMALL, STREAM, 1, true>(a, c, param + at, grad + at, table.state + b, 4);
        ++b;
      } else {
        const int left = (b + 1 == next && last ? last : kQuant) - lane * 4;
        update<SMALL, STREAM, 1, false>(a, c, param + at, grad + at, table.state + b, left);
        ++b;
      }
    }
  }
}

// One more step for every tensor that took part.  A launch of its own: the update kernels read the steps
// in every workgroup, and a count of the workgroups that are done costs more (14 ns each, one address).
__global__ void __launch_bounds__(kThreads)
advance_kernel(const RowMask mask, double* __restrict__ progress, double beta1, double beta2,
               const float* __restrict__ clip) {
  if (clip && clip[1] != clip[1]) return;
  const int k = blockIdx.x * kThreads + threadIdx.x;
  if (k >= mask.count || !((mask.bits[k >> 5] >> (k & 31)) & 1u)) return;
  double* row = progress + 3 * (mask.first + k);
  row[0] += 1.0;
  row[1] *= beta1;
  row[2] *= beta2;
}

// Eight-bit moments as the values they stand for: 4 significant bits (m and v) and a power of two, exact in
// bfloat16.  Eight codes a thread, so that the stores are 16 bytes wide.  Bound by memory: 6 bytes a value.
__global__ void __launch_bounds__(kThreads)
moment_values_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ m_top, const uint8_t* __restrict__ v,
                     const uint8_t* __restrict__ v_top, uint16_t* __restrict__ m_out, uint16_t* __restrict__ v_out,
                     int64_t values) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads * 8;
  for (int64_t s = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * 8; s < values; s += stride) {
    const u32x2 cm = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(m + s));
    const u32x2 cv = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(v + s));
    const int tm = m_top[s / kQuant], tv = v_top[s / kQuant];
    float x[8], y[8];
    decode_signed(cm.x, tm, x);
    decode_signed(cm.y, tm, x + 4);
    decode_unsigned(cv.x, tv, y);
    decode_unsigned(cv.y, tv, y + 4);
    u32x4 om, ov;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      om[k] = (__float_as_uint(x[2 * k]) >> 16) | (__float_as_uint(x[2 * k + 1]) & 0xFFFF0000u);
      ov[k] = (__float_as_uint(y[2 * k]) >> 16) | (__float_as_uint(y[2 * k + 1]) & 0xFFFF0000u);
    }
    __builtin_nontemporal_store(om, reinterpret_cast<u32x4*>(m_out + s));
    __builtin_nontemporal_store(ov, reinterpret_cast<u32x4*>(v_out + s));
  }
}

struct NormTable {
  const float* grad[kNormTensors];
  int64_t elements[kNormTensors];
  uint32_t start[kNormTensors + 1];    // a tensor's first chunk of kNormChunk values
  int32_t count;     // (of the host's)
  uint32_t chunks;
};

__device__ __forceinline__ double block_sum(double x) {
  __shared__ double part[kWaves];
#pragma unroll
  for (int d = kWaveSize / 2; d; d >>= 1) x += __shfl_xor(x, d);
  if ((threadIdx.x & (kWaveSize - 1)) == 0) part[threadIdx.x / kWaveSize] = x;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) sum += part[w];
  return sum;
}

// Sums of squares in 64 bits (a float's square neither overflows nor vanishes there), one for each
// workgroup; a second launch adds them in order.  Bound by memory: 150 M values in 92 us (6.5 TB/s, past the caches;
// 150 us with the tables read from the kernel's arguments at every change of tensors), 1.5 M in 5 us.
template <bool STREAM>
__global__ void __launch_bounds__(kThreads) norm_partial_kernel(const NormTable table, double* __restrict__ partial) {
  __shared__ const float* grads[kNormTensors];
  __shared__ int64_t sizes[kNormTensors];
  __shared__ uint32_t starts[kNormTensors + 1];
  if (threadIdx.x < kNormTensors) {
    grads[threadIdx.x] = table.grad[threadIdx.x];
    sizes[threadIdx.x] = table.elements[threadIdx.x];
  }
  if (threadIdx.x <= kNormTensors) starts[threadIdx.x] = table.start[threadIdx.x];
  __syncthreads();
  double sum = 0.0;
  uint32_t start = 0, next = 0;
  const float* grad = nullptr;
  int64_t elements = 0;
  for (uint32_t chunk = blockIdx.x; chunk < table.chunks; chunk += gridDim.x) {
    if (chunk >= next) {
      const int i = entry_of<kNormTensors>(starts, chunk);
      start = uniform(starts[i]), next = uniform(starts[i + 1]);
      grad = uniform(grads[i]), elements = sizes[i];
    }
    const int64_t first = static_cast<int64_t>(chunk - start) * kNormChunk;
    if ((reinterpret_cast<uintptr_t>(grad) & 15) == 0 && first + kNormChunk <= elements) {
      float g[kNormChunk / kThreads];
#pragma unroll
      for (int k = 0; k < kNormChunk / (4 * kThreads); ++k)
        load4<STREAM>(grad + first + (k * kThreads + threadIdx.x) * 4, g + 4 * k);
#pragma unroll
      for (int k = 0; k < kNormChunk / kThreads; ++k) sum += static_cast<double>(g[k]) * static_cast<double>(g[k]);
    } else {
      const int64_t stop = first + kNormChunk < elements ? first + kNormChunk : elements;
      for (int64_t k = first + threadIdx.x; k < stop; k += kThreads) {
        const double x = grad[k];
        sum += x * x;
      }
    }
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kThreads)
norm_finish_kernel(const double* __restrict__ partial, int count, float max_norm, float* __restrict__ out) {
  double sum = 0.0;
  for (int k = threadIdx.x; k < count; k += kThreads) sum += partial[k];
  sum = block_sum(sum);
  if (threadIdx.x == 0) {
    const float norm = static_cast<float>(sqrt(sum)), ratio = max_norm / norm;     // of the norm that is returned
    out[0] = norm;
    const float coefficient = max_norm > 0.f && ratio < 1.f ? ratio : 1.f;
    out[1] = norm < INFINITY ? coefficient : __uint_as_float(0x7FC00000u);
  }
}

constexpr int64_t kMostElements = int64_t{1} << 38;     // of one tensor: 2^30 blocks
constexpr int64_t kMostUnits = int64_t{3} << 30;        // blocks or chunks of one launch, within 32 bits

// The end of the last tensor, and entries that no search finds.
void close_starts(uint32_t* start, int count, int most, int64_t end) {
  start[count] = static_cast<uint32_t>(end);
  for (int i = count + 1; i <= most; ++i) start[i] = ~0u;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int launched() { return hipGetLastError() == hipSuccess ? ICTC_OK : ICTC_ERR_LAUNCH; }

}  // namespace
}  // namespace ictc

extern "C" {

int64_t ictc_hip_gradient_norm_workspace(int64_t count) {
  using namespace ictc;
  if (count < 0) return -ICTC_ERR_INVALID_ARGUMENT;
  return (count == 0 ? 1 : ceil_div(count, kNormTensors)) * kNormBlocks;
}

int ictc_hip_gradient_norm(const float* const* grads, const int64_t* elements, int64_t count, float max_norm,
                           double* workspace, int64_t workspace_doubles, float* out, hipStream_t stream) {
  using namespace ictc;
  if (count < 0 || !out || !workspace || (count && (!grads || !elements)) ||
      workspace_doubles < ictc_hip_gradient_norm_workspace(count) || max_norm != max_norm)
    return ICTC_ERR_INVALID_ARGUMENT;
  for (int64_t k = 0; k < count; ++k)
    if (elements[k] < 0 || elements[k] > kMostElements || (elements[k] && !grads[k])) return ICTC_ERR_INVALID_ARGUMENT;
  int partials = 0;
  for (int64_t k = 0; k < count;) {
    NormTable table;
    table.count = 0;
    int64_t chunks = 0;
    for (; k < count && table.count < kNormTensors; ++k) {
      if (!elements[k]) continue;
      const int64_t more = ceil_div(elements[k], kNormChunk);
      if (chunks + more > kMostUnits) break;         // the next launch takes it
      table.grad[table.count] = grads[k];
      table.elements[table.count] = elements[k];
      table.start[table.count++] = static_cast<uint32_t>(chunks);
      chunks += more;
    }
    if (!table.count) continue;
    close_starts(table.start, table.count, kNormTensors, chunks);
    table.chunks = static_cast<uint32_t>(chunks);
    const int blocks = static_cast<int>(chunks < kNormBlocks ? chunks : kNormBlocks);
    if (partials + blocks > workspace_doubles) return ICTC_ERR_UNSUPPORTED;
    const auto kernel = chunks * kNormChunk >= kStream ? norm_partial_kernel<true> : norm_partial_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, stream, table, workspace + partials);
    if (const int rc = launched()) return rc;
    partials += blocks;
  }
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(kThreads), 0, stream, workspace, partials, max_norm, out);
  return launched();
}

int ictc_hip_adamw_step(float* const* params, const float* const* grads, const int64_t* elements, int64_t count,
                        const ictc_adamw_desc* desc, void* exp_avg, void* exp_avg_sq, uint8_t* exp_avg_top,
                        uint8_t* exp_avg_sq_top, double* progress, const float* clip, const float* lr_device,
                        hipStream_t stream) {
  using namespace ictc;
  if (count < 0 || !desc) return ICTC_ERR_INVALID_ARGUMENT;
  if (desc->moment_bits != 32 && desc->moment_bits != 8) return ICTC_ERR_UNSUPPORTED;
  if (!(desc->beta1 >= 0.0 && desc->beta1 < 1.0 && desc->beta2 >= 0.0 && desc->beta2 < 1.0 && desc->eps >= 0.f &&
        desc->weight_decay >= 0.0 && (lr_device || desc->lr >= 0.f)))
    return ICTC_ERR_INVALID_ARGUMENT;
  if (count == 0) return ICTC_OK;
  const bool small = desc->moment_bits == 8;
  if (!params || !grads || !elements || !progress || !exp_avg || !exp_avg_sq ||
      (small && (!exp_avg_top || !exp_avg_sq_top)))
    return ICTC_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(exp_avg) | reinterpret_cast<uintptr_t>(exp_avg_sq)) & (small ? 3 : 15))
    return ICTC_ERR_INVALID_ARGUMENT;
  for (int64_t k = 0; k < count; ++k)
    if (elements[k] < 0 || elements[k] > kMostElements || (elements[k] && grads[k] && !params[k]))
      return ICTC_ERR_INVALID_ARGUMENT;
  if (count > 0x7fffffff) return ICTC_ERR_INVALID_ARGUMENT;
  StepArgs args;
  args.exp_avg = exp_avg;
  args.exp_avg_sq = exp_avg_sq;
  args.exp_avg_top = exp_avg_top;
  args.exp_avg_sq_top = exp_avg_sq_top;
  args.progress = progress;
  args.clip = clip;
  args.lr_device = lr_device;
  args.beta1 = desc->beta1;
  args.beta2 = desc->beta2;
  args.weight_decay = desc->weight_decay;
  args.lr = desc->lr;
  args.eps = desc->eps;
  args.seed = desc->seed;
  int64_t state = 0;    // blocks of the tensors before k
  for (int64_t k = 0; k < count;) {
    if (!grads[k]) {    // a launch begins with a tensor that takes part
      state += ceil_div(elements[k++], kQuant);
      continue;
    }
    StepTable table;
    table.state = state;
    table.row = k;
    table.count = 0;
    int64_t blocks = 0;
    for (; k < count && table.count < kTensors; ++k) {
      const int64_t more = ceil_div(elements[k], kQuant);
      // a large tensor that takes no part ends the launch: its blocks would go by without work
      if (blocks + more > kMostUnits || (!grads[k] && more > kSkip)) break;
      table.param[table.count] = params[k];
      table.grad[table.count] = grads[k];
      table.tail[table.count] = static_cast<uint8_t>(elements[k] % kQuant);
      table.start[table.count++] = static_cast<uint32_t>(blocks);
      blocks += more;
    }
    state += blocks;
    if (!blocks) continue;
    close_starts(table.start, table.count, kTensors, blocks);
    table.blocks = static_cast<uint32_t>(blocks);
    const bool past = blocks * kQuant >= kStream;
    const int64_t groups = ceil_div(blocks, kWaves * step_blocks(small, past)), most = past ? kMostGroups : kMaxBlocks;
    const int grid = static_cast<int>(groups < most ? groups : most);
    const auto kernel = small ? past ? adamw_kernel<true, true> : adamw_kernel<true, false>
                              : past ? adamw_kernel<false, true> : adamw_kernel<false, false>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), 0, stream, table, args);
    if (const int rc = launched()) return rc;
  }
  for (int64_t first = 0; first < count; first += kMaskTensors) {
    RowMask mask = {};
    mask.first = first;
    mask.count = static_cast<int32_t>(count - first < kMaskTensors ? count - first : kMaskTensors);
    bool any = false;
    for (int k = 0; k < mask.count; ++k)
      if (grads[first + k]) mask.bits[k >> 5] |= 1u << (k & 31), any = true;
    if (!any) continue;
    hipLaunchKernelGGL(advance_kernel, dim3(static_cast<unsigned>(ceil_div(mask.count, kThreads))), dim3(kThreads), 0,
                       stream, mask, progress, desc->beta1, desc->beta2, clip);
    if (const int rc = launched()) return rc;
  }
  return ICTC_OK;
}

int ictc_hip_moment_values(const uint8_t* exp_avg, const uint8_t* exp_avg_top, const uint8_t* exp_avg_sq,
                           const uint8_t* exp_avg_sq_top, void* exp_avg_bf16, void* exp_avg_sq_bf16, int64_t values,
                           hipStream_t stream) {
  using namespace ictc;
  if (values < 0 || values % kQuant) return ICTC_ERR_INVALID_ARGUMENT;
  if (values == 0) return ICTC_OK;
  if (!exp_avg || !exp_avg_top || !exp_avg_sq || !exp_avg_sq_top || !exp_avg_bf16 || !exp_avg_sq_bf16 ||
      ((reinterpret_cast<uintptr_t>(exp_avg) | reinterpret_cast<uintptr_t>(exp_avg_sq)) & 7) ||
      ((reinterpret_cast<uintptr_t>(exp_avg_bf16) | reinterpret_cast<uintptr_t>(exp_avg_sq_bf16)) & 15))
    return ICTC_ERR_INVALID_ARGUMENT;
  const int64_t groups = ceil_div(values, 8 * kThreads);
  hipLaunchKernelGGL(moment_values_kernel, dim3(static_cast<unsigned>(groups < kMostGroups ? groups : kMostGroups)),
                     dim3(kThreads), 0, stream, exp_avg, exp_avg_top, exp_avg_sq, exp_avg_sq_top,
                     static_cast<uint16_t*>(exp_avg_bf16), static_cast<uint16_t*>(exp_avg_sq_bf16), values);
  return launched();
}

}  // extern "C"
