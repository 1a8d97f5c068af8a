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
constexpr int kChunk = kQuant * (kThreads / kWaveSize);
constexpr int kTensors = 96;                     // 40 bytes each, within the 4 KB of kernel arguments
constexpr int kMaxBlocks = 2048;                 // 8 workgroups for each of 256 CUs
constexpr int kNormTensors = 160;
constexpr int kNormChunk = 4096;
constexpr int kNormBlocks = 1024;

struct StepTensor {
  float* param;
  const float* grad;
  int64_t elements;
  int64_t state;     // first value in the flat state
  int32_t chunk;     // first chunk of this tensor in the launch
  int32_t row;       // its row in progress
};

struct StepTable {
  StepTensor t[kTensors];
  int32_t count;
  int32_t chunks;
  int32_t per_block;
};

struct StepArgs {
  void* exp_avg;
  void* exp_avg_sq;
  uint8_t* exp_avg_top;
  uint8_t* exp_avg_sq_top;
  double* progress;
  unsigned* ticket;
  const float* clip;
  const float* lr_device;
  double beta1, beta2, weight_decay;
  float lr, eps;
  uint32_t seed;
};

static_assert(sizeof(StepTable) + sizeof(StepArgs) <= 4096, "kernel arguments are limited to 4 KB");

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

// Exponent byte of a block from its largest finite magnitude.
__device__ __forceinline__ int block_top(uint32_t largest) {
  const int f = static_cast<int>((largest + 0x1FFFFFu) >> 23);
  return f < 1 ? 1 : f;
}

__device__ __forceinline__ uint32_t finite_magnitude(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0u;
}

// m: sign, 4 exponent bits, 3 mantissa bits; top code 0x7e, 0x7f not a number
__device__ __forceinline__ float decode_signed(uint32_t code, int top) {
  const uint32_t size = code & 0x7Fu;
  const float x = ldexpf(__uint_as_float(size << 20), top - 15);
  const float y = size == 0x7Fu ? __uint_as_float(0x7FC00000u) : x;
  return (code & 0x80u) ? -y : y;
}

__device__ __forceinline__ uint32_t encode_signed(float m, int top, uint32_t random16) {
  const float x = ldexpf(fabsf(m), 15 - top);
  const uint32_t code = (__float_as_uint(x) + (random16 << 4)) >> 20;
  const uint32_t size = fabsf(m) < INFINITY ? code : 0x7Fu;
  return size | ((__float_as_uint(m) >> 24) & 0x80u);
}

// v: 5 exponent bits, 3 mantissa bits; top code 0xfe, 0xff not a number
__device__ __forceinline__ float decode_unsigned(uint32_t code, int top) {
  const float x = ldexpf(__uint_as_float(code << 20), top - 31);
  return code == 0xFFu ? __uint_as_float(0x7FC00000u) : x;
}

__device__ __forceinline__ uint32_t encode_unsigned(float v, int top, uint32_t random16) {
  const float x = ldexpf(v, 31 - top);
  uint32_t code = (__float_as_uint(x) + (random16 << 4)) >> 20;
  code = code < 1u && v > 0.f ? 1u : code;
  return v < INFINITY ? code : 0xFFu;
}

template <bool SMALL>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const StepTable table, const StepArgs a) {
  const int lane = threadIdx.x & (kWaveSize - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
  const float coefficient = a.clip ? a.clip[1] : 1.f;
  const bool live = coefficient == coefficient;     // a norm that is not finite: nothing changes
  if (live) {
    int chunk = blockIdx.x * table.per_block;
    const int end = chunk + table.per_block < table.chunks ? chunk + table.per_block : table.chunks;
    int i = 0;
    for (int step = 64; step; step >>= 1)            // the last tensor that starts at or before the chunk
      if (i + step < table.count && table.t[i + step].chunk <= chunk) i += step;
    const float lr = a.lr_device ? *a.lr_device : a.lr;
    const float keep = static_cast<float>(1.0 - static_cast<double>(lr) * a.weight_decay);
    const float b1 = static_cast<float>(a.beta1), b2 = static_cast<float>(a.beta2);
    const float n1 = static_cast<float>(1.0 - a.beta1), n2 = static_cast<float>(1.0 - a.beta2);
    int loaded = -1;
    float rate = 0.f, inv2 = 0.f;
    uint32_t key = 0;
    bool wide = false;
    StepTensor t = table.t[i];
    for (; chunk < end; ++chunk) {
      while (i + 1 < table.count && table.t[i + 1].chunk <= chunk) ++i;
      if (i != loaded) {
        t = table.t[i];
        const double* row = a.progress + 3 * static_cast<int64_t>(t.row);
        rate = lr / static_cast<float>(1.0 - row[1] * a.beta1);
        inv2 = 1.f / static_cast<float>(1.0 - row[2] * a.beta2);
        if constexpr (SMALL)
          key = mix(a.seed + static_cast<uint32_t>(static_cast<int64_t>(row[0]) + 1) * 0x9E3779B9u);
        wide = ((reinterpret_cast<uintptr_t>(t.param) | reinterpret_cast<uintptr_t>(t.grad)) & 15) == 0;
        loaded = i;
      }
      const int64_t first = static_cast<int64_t>(chunk - t.chunk) * kChunk + wave * kQuant;
      if (first >= t.elements) continue;
      const int64_t at = first + lane * 4;
      float p[4] = {}, g[4] = {}, m[4], v[4];
      const bool whole = wide && first + kQuant <= t.elements;
      if (whole) {
        const float4 p4 = *reinterpret_cast<const float4*>(t.param + at);
        const float4 g4 = *reinterpret_cast<const float4*>(t.grad + at);
        p[0] = p4.x, p[1] = p4.y, p[2] = p4.z, p[3] = p4.w;
        g[0] = g4.x, g[1] = g4.y, g[2] = g4.z, g[3] = g4.w;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (at + k < t.elements) p[k] = t.param[at + k], g[k] = t.grad[at + k];
      }
      const int64_t s = t.state + at;
      [[maybe_unused]] const int64_t block = (t.state + first) / kQuant;
      if constexpr (SMALL) {
        const uint32_t cm = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.exp_avg) + s);
        const uint32_t cv = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.exp_avg_sq) + s);
        const int tm = a.exp_avg_top[block], tv = a.exp_avg_sq_top[block];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          m[k] = decode_signed((cm >> (8 * k)) & 0xFFu, tm);
          v[k] = decode_unsigned((cv >> (8 * k)) & 0xFFu, tv);
        }
      } else {
        const float4 m4 = *reinterpret_cast<const float4*>(static_cast<const float*>(a.exp_avg) + s);
        const float4 v4 = *reinterpret_cast<const float4*>(static_cast<const float*>(a.exp_avg_sq) + s);
        m[0] = m4.x, m[1] = m4.y, m[2] = m4.z, m[3] = m4.w;
        v[0] = v4.x, v[1] = v4.y, v[2] = v4.z, v[3] = v4.w;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float gk = coefficient * g[k];
        m[k] = b1 * m[k] + n1 * gk;
        v[k] = b2 * v[k] + n2 * (gk * gk);
        p[k] = keep * p[k] - rate * m[k] / (sqrtf(v[k] * inv2) + a.eps);
      }
      if (whole) {
        *reinterpret_cast<float4*>(t.param + at) = make_float4(p[0], p[1], p[2], p[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (at + k < t.elements) t.param[at + k] = p[k];
      }
      if constexpr (SMALL) {
        uint32_t lm = 0, lv = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t fm = finite_magnitude(m[k]), fv = finite_magnitude(v[k]);
          lm = lm > fm ? lm : fm;
          lv = lv > fv ? lv : fv;
        }
        const int tm = block_top(wave_max(lm)), tv = block_top(wave_max(lv));
        uint32_t cm = 0, cv = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t bits = mix(static_cast<uint32_t>(s) + k + key);
          cm |= encode_signed(m[k], tm, bits & 0xFFFFu) << (8 * k);
          cv |= encode_unsigned(v[k], tv, bits >> 16) << (8 * k);
        }
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.exp_avg) + s) = cm;
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.exp_avg_sq) + s) = cv;
        if (lane == 0) {
          a.exp_avg_top[block] = static_cast<uint8_t>(tm);
          a.exp_avg_sq_top[block] = static_cast<uint8_t>(tv);
        }
      } else {
        *reinterpret_cast<float4*>(static_cast<float*>(a.exp_avg) + s) = make_float4(m[0], m[1], m[2], m[3]);
        *reinterpret_cast<float4*>(static_cast<float*>(a.exp_avg_sq) + s) = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
  }
  // the workgroup that ends last advances the tensors' steps: every other one has read them by then
  __shared__ unsigned last;
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  if (live)
    for (int k = threadIdx.x; k < table.count; k += kThreads) {
      double* row = a.progress + 3 * static_cast<int64_t>(table.t[k].row);
      row[0] += 1.0;
      row[1] *= a.beta1;
      row[2] *= a.beta2;
    }
  if (threadIdx.x == 0) *a.ticket = 0u;
}

// Eight-bit moments as the values they stand for: 4 significant bits (m) and a power of two, exact in bfloat16.
__global__ void __launch_bounds__(kThreads)
moment_values_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ m_top, const uint8_t* __restrict__ v,
                     const uint8_t* __restrict__ v_top, uint16_t* __restrict__ m_out, uint16_t* __restrict__ v_out,
                     int64_t blocks) {
  const int lane = threadIdx.x & (kWaveSize - 1);
  const int64_t waves = static_cast<int64_t>(gridDim.x) * (kThreads / kWaveSize);
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * (kThreads / kWaveSize) + threadIdx.x / kWaveSize; b < blocks;
       b += waves) {
    const int64_t s = b * kQuant + lane * 4;
    const uint32_t cm = *reinterpret_cast<const uint32_t*>(m + s), cv = *reinterpret_cast<const uint32_t*>(v + s);
    const int tm = m_top[b], tv = v_top[b];
    ushort4 om, ov;
    uint16_t* pm = reinterpret_cast<uint16_t*>(&om);
    uint16_t* pv = reinterpret_cast<uint16_t*>(&ov);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      pm[k] = static_cast<uint16_t>(__float_as_uint(decode_signed((cm >> (8 * k)) & 0xFFu, tm)) >> 16);
      pv[k] = static_cast<uint16_t>(__float_as_uint(decode_unsigned((cv >> (8 * k)) & 0xFFu, tv)) >> 16);
    }
    *reinterpret_cast<ushort4*>(m_out + s) = om;
    *reinterpret_cast<ushort4*>(v_out + s) = ov;
  }
}

struct NormTensor {
  const float* grad;
  int64_t elements;
  int64_t chunk;
};

struct NormTable {
  NormTensor t[kNormTensors];
  int64_t chunks;
  int64_t per_block;
  int32_t count;
};

__device__ __forceinline__ double block_sum(double x) {
  __shared__ double part[kThreads / kWaveSize];
#pragma unroll
  for (int d = kWaveSize / 2; d; d >>= 1) x += __shfl_xor(x, d);
  if ((threadIdx.x & (kWaveSize - 1)) == 0) part[threadIdx.x / kWaveSize] = x;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / kWaveSize; ++w) sum += part[w];
  return sum;
}

// Sums of squares in 64 bits (a float's square neither overflows nor vanishes there), one for each
// workgroup; a second launch adds them in order.
__global__ void __launch_bounds__(kThreads) norm_partial_kernel(const NormTable table, double* __restrict__ partial) {
  int64_t chunk = blockIdx.x * table.per_block;
  const int64_t end = chunk + table.per_block < table.chunks ? chunk + table.per_block : table.chunks;
  int i = 0;
  for (int step = 128; step; step >>= 1)
    if (i + step < table.count && table.t[i + step].chunk <= chunk) i += step;
  double sum = 0.0;
  for (; chunk < end; ++chunk) {
    while (i + 1 < table.count && table.t[i + 1].chunk <= chunk) ++i;
    const NormTensor t = table.t[i];
    const int64_t first = (chunk - t.chunk) * kNormChunk;
    if ((reinterpret_cast<uintptr_t>(t.grad) & 15) == 0 && first + kNormChunk <= t.elements) {
#pragma unroll
      for (int k = 0; k < kNormChunk / (4 * kThreads); ++k) {
        const float4 g = *reinterpret_cast<const float4*>(t.grad + first + (k * kThreads + threadIdx.x) * 4);
        const double x = g.x, y = g.y, z = g.z, w = g.w;
        sum += x * x + y * y + z * z + w * w;
      }
    } else {
      const int64_t stop = first + kNormChunk < t.elements ? first + kNormChunk : t.elements;
      for (int64_t k = first + threadIdx.x; k < stop; k += kThreads) {
        const double x = t.grad[k];
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
    const double norm = sqrt(sum);
    const double ratio = static_cast<double>(max_norm) / norm;
    out[0] = static_cast<float>(norm);
    out[1] = !(norm < INFINITY) ? __uint_as_float(0x7FC00000u) : max_norm > 0.f && ratio < 1.0 ? static_cast<float>(ratio) : 1.f;
  }
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
    if (elements[k] < 0 || (elements[k] && !grads[k])) return ICTC_ERR_INVALID_ARGUMENT;
  int partials = 0;
  for (int64_t k = 0; k < count;) {
    NormTable table;
    table.count = 0;
    table.chunks = 0;
    for (; k < count && table.count < kNormTensors; ++k) {
      if (!elements[k]) continue;
      table.t[table.count++] = {grads[k], elements[k], table.chunks};
      table.chunks += ceil_div(elements[k], kNormChunk);
    }
    if (!table.count) continue;
    table.per_block = ceil_div(table.chunks, kNormBlocks);
    const int blocks = static_cast<int>(ceil_div(table.chunks, table.per_block));
    hipLaunchKernelGGL(norm_partial_kernel, dim3(blocks), dim3(kThreads), 0, stream, table, workspace + partials);
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
    if (elements[k] < 0 || elements[k] > (int64_t{1} << 40) || (elements[k] && grads[k] && !params[k]))
      return ICTC_ERR_INVALID_ARGUMENT;
  if (count > 0x7fffffff) return ICTC_ERR_INVALID_ARGUMENT;
  StepArgs args;
  args.exp_avg = exp_avg;
  args.exp_avg_sq = exp_avg_sq;
  args.exp_avg_top = exp_avg_top;
  args.exp_avg_sq_top = exp_avg_sq_top;
  args.progress = progress;
  args.ticket = reinterpret_cast<unsigned*>(progress + 3 * count);
  args.clip = clip;
  args.lr_device = lr_device;
  args.beta1 = desc->beta1;
  args.beta2 = desc->beta2;
  args.weight_decay = desc->weight_decay;
  args.lr = desc->lr;
  args.eps = desc->eps;
  args.seed = desc->seed;
  int64_t state = 0;
  for (int64_t k = 0; k < count;) {
    StepTable table;
    table.count = 0;
    int64_t chunks = 0;
    for (; k < count && table.count < kTensors; ++k) {
      const int64_t at = state;
      const int64_t more = ceil_div(elements[k], kChunk);
      state += ceil_div(elements[k], kQuant) * kQuant;
      if (!grads[k]) continue;                       // not part of this step
      if (chunks + more > 0x7fffffff - kMaxBlocks) { // the next launch takes it
        state = at;
        break;
      }
      table.t[table.count++] = {params[k], grads[k], elements[k], at, static_cast<int32_t>(chunks),
                                static_cast<int32_t>(k)};
      chunks += more;
    }
    if (!table.count) continue;
    table.chunks = static_cast<int32_t>(chunks);
    table.per_block = static_cast<int32_t>(chunks ? ceil_div(chunks, kMaxBlocks) : 1);
    const int blocks = static_cast<int>(chunks ? ceil_div(chunks, table.per_block) : 1);
    if (small)
      hipLaunchKernelGGL(adamw_kernel<true>, dim3(blocks), dim3(kThreads), 0, stream, table, args);
    else
      hipLaunchKernelGGL(adamw_kernel<false>, dim3(blocks), dim3(kThreads), 0, stream, table, args);
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
      ((reinterpret_cast<uintptr_t>(exp_avg) | reinterpret_cast<uintptr_t>(exp_avg_sq)) & 3) ||
      ((reinterpret_cast<uintptr_t>(exp_avg_bf16) | reinterpret_cast<uintptr_t>(exp_avg_sq_bf16)) & 7))
    return ICTC_ERR_INVALID_ARGUMENT;
  const int64_t blocks = values / kQuant;
  const int64_t groups = ceil_div(blocks, kThreads / kWaveSize);
  hipLaunchKernelGGL(moment_values_kernel, dim3(static_cast<unsigned>(groups < 4096 ? groups : 4096)), dim3(kThreads),
                     0, stream, exp_avg, exp_avg_top, exp_avg_sq, exp_avg_sq_top,
                     static_cast<uint16_t*>(exp_avg_bf16), static_cast<uint16_t*>(exp_avg_sq_bf16), blocks);
  return launched();
}

}  // extern "C"
