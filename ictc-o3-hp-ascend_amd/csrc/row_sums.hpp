// Sums over the threads that hold a row, and over workgroups' partial sums of columns: both norms' kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ictc {
namespace {

constexpr int kRowWave = 64;

template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}

template <int CTRL>
__device__ __forceinline__ double add_dpp(double x) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, 0xf, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, 0xf, 0xf, false);
  return x + __hiloint2double(hi, lo);
}

__device__ __forceinline__ float lane_value(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

__device__ __forceinline__ double lane_value(double x, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), lane),
                          __builtin_amdgcn_readlane(__double2loint(x), lane));
}

constexpr int kMaxWaves = 16;           // of a row
constexpr int kSums = 4;             // of a round at most

// Sums over a row's threads, in all of them and in a fixed order.
template <int S, int WIDE, typename T>
__device__ __forceinline__ void row_sums(T (&x)[S], int threads, double* lds, int& turn) {
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (WIDE || threads >= 2) x[s] = add_dpp<0xB1>(x[s]);         // quad_perm 1 0 3 2
    if (WIDE || threads >= 4) x[s] = add_dpp<0x4E>(x[s]);         // quad_perm 2 3 0 1
    if (WIDE || threads >= 8) x[s] = add_dpp<0x141>(x[s]);        // row_half_mirror
    if (WIDE || threads >= 16) x[s] = add_dpp<0x140>(x[s]);       // row_mirror
    if (WIDE || threads == 64)
      x[s] = (lane_value(x[s], 0) + lane_value(x[s], 16)) + (lane_value(x[s], 32) + lane_value(x[s], 48));
    else if (threads == 32)
      x[s] += __shfl_xor(x[s], 16);
  }
  if constexpr (WIDE) {
    // two slots in turn: a wave is at most one round ahead of another
    T* slot = reinterpret_cast<T*>(lds + turn * (kSums * kMaxWaves));
    turn ^= 1;
    const int waves = threads / kRowWave, wave = threadIdx.x / kRowWave;
    if ((threadIdx.x & (kRowWave - 1)) == 0) {
#pragma unroll
      for (int s = 0; s < S; ++s) slot[s * kMaxWaves + wave] = x[s];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S; ++s) {
      T sum = 0;
      for (int w = 0; w < waves; ++w) sum += slot[s * kMaxWaves + w];
      x[s] = sum;
    }
  }
}

// Column sums of the workgroups' partial gradients of two weights, in order: 16 columns a workgroup, and 32
// slices of the partials side by side, eight of whose loads are on their way at a time.
constexpr int kSlices = 32, kColumns = 16;

__global__ void __launch_bounds__(kSlices* kColumns)
norm_weight_kernel(const float* __restrict__ partial, float* __restrict__ dpost, float* __restrict__ dpre, int groups,
                   int columns) {
  __shared__ double part[kSlices][kColumns];
  const int at = threadIdx.x % kColumns, slice = threadIdx.x / kColumns;
  const int column = blockIdx.x * kColumns + at;          // of post's, then of pre's
  const int per = (groups + kSlices - 1) / kSlices;
  const int end = groups < (slice + 1) * per ? groups : (slice + 1) * per;
  double sum = 0.0;
  if (column < 2 * columns) {
    const float* p = partial + column;
    int g = slice * per;
    for (; g + 8 <= end; g += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = p[static_cast<int64_t>(g + k) * 2 * columns];
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += v[k];
    }
    for (; g < end; ++g) sum += p[static_cast<int64_t>(g) * 2 * columns];
  }
  part[slice][at] = sum;
  __syncthreads();
  if (slice || column >= 2 * columns) return;
  for (int s = 1; s < kSlices; ++s) sum += part[s][at];
  float* out = column < columns ? dpost : dpre;
  if (out) out[column < columns ? column : column - columns] = static_cast<float>(sum);
}

}  // namespace
}  // namespace ictc
