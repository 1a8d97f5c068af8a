// Layer norm of rows, alone or with SiLU behind it, with its gradients and the gradients of those, gfx950.
//
//   xc = x - mean(x)   r2 = 1 / (mean(xc^2) + eps)   rho = sqrt(r2)   xh = rho xc   z = w xh + b   y = f(z)
//
//   gradients, for a cotangent dy:  dz = f'(z) dy, e = w dz,
//     dx = J e,  J v = rho (v - mean(v) - xc r2 mean(v xc))  (symmetric)      dw = sum_n dz xh     db = sum_n dz
//
//   second order, for a cotangent u of dx:  t = J u, a = u - mean(u), c = e - mean(e), and with P, Q, R the means
//   of xc a, xc c and a c
//     dx'' = -rho^3 (xc (R - 3 r2 P Q) + Q a + P c) + J (w s),   s = w t dy f''(z)
//     ddy'' = w t f'(z)          dw'' = sum_n t dz + s xh          db'' = sum_n s
//   (the second term of dx'' is the way through f'(z); without an activation s = 0).
//
// Without an activation bound by memory: rows are read into registers once, all statistics are taken there and every
// result is written once.  With SiLU the instructions take longer: at 105,634 x 64 the vector units alone are busy for 11.5
// of 15.7, 16.5 of 20.8 and 23 of 32 us, at their highest clock.  Sums over a row, means and the projections of J are in
// 64 bits: what J leaves of a cotangent along xc is eps r2 of it, a difference of nearly equal numbers for a row of two
// values or with one large entry; xc itself is x - mean in 64 bits, exact where the mean is many times the spread.  The
// weights' gradients are added up in float32 over a thread's rows and a workgroup's, in 64 bits over workgroups
// (36,000,000 x 64: within 1e-6 of the largest).  A thread holds K groups of four columns, which are loaded as one vector at
// any float's alignment (a row of odd width ends in a part of one); a row's threads are a power of two of a wave's, so that
// rows of 64 columns share it, or 4 or 16 waves.  Forward, gradients with the weights', their sum over workgroups: 32,768
// x 512 23.8 us (5.6 TB/s), 38.5 (5.2), 3.9; 5,003 x 1,001 with SiLU (rows of 4 waves, 23 of 1,024 columns idle, a barrier
// to a sum) 13.2 (3.0 TB/s), 22.5 (2.7), 4.8; 105,634 x 64 with SiLU 15.2 (3.6), 20.7 (3.9), second derivatives 31.9 (4.2),
// 3.7.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ictc_hip.h"
#include "row_sums.hpp"

namespace ictc {
namespace {

constexpr int kLnThreads = 256;              // of a workgroup whose rows fit into a wave, or of a row
constexpr int kLnWideThreads = 1024;
constexpr int kLnGroups = 1024;              // workgroups that leave partial weight gradients
constexpr float kLog2E = 0x1.715476p+0f, kLog2ELow = 0x1.4ae0cp-26f, kLn2 = 0x1.62e43p-1f;

typedef float lf4 __attribute__((ext_vector_type(4), aligned(4)));

struct LayerNormArgs {
  const float *x, *weight, *bias, *dy, *u;
  float *y, *dx, *ddy;
  float* partial;             // per workgroup [2][width]: the weight's and the bias's gradients
  int64_t rows;
  int width;
  int threads;                // of a row
  int groups;                 // rows of a workgroup at a time
  float eps;
};

// Threads of a workgroup: rows within a wave (0) or in 4 (1) or 16 (2) waves of their own.
constexpr int ln_block(int wide) { return wide == 2 ? kLnWideThreads : kLnThreads; }

// Where a thread's columns are.
template <int K, int WIDE>
struct Columns {
  int group, thread, at[K], count[K];       // first column and number (0 to 4) of each group of four

  __device__ __forceinline__ explicit Columns(const LayerNormArgs& a) {
    group = WIDE ? 0 : threadIdx.x / a.threads;
    thread = WIDE ? threadIdx.x : threadIdx.x & (a.threads - 1);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      at[k] = (k * a.threads + thread) * 4;
      const int left = a.width - at[k];
      count[k] = left < 0 ? 0 : left > 4 ? 4 : left;
    }
  }

  // A row's values; zeros behind its end, and everywhere where there is no row.
  __device__ __forceinline__ void load(const float* row, bool on, float* v) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      lf4 t = {0.f, 0.f, 0.f, 0.f};
      if (on && row && count[k] == 4) {
        t = *reinterpret_cast<const lf4*>(row + at[k]);
      } else if (on && row) {
#pragma unroll
        for (int j = 0; j < 3; ++j)
          if (j < count[k]) t[j] = row[at[k] + j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * k + j] = t[j];
    }
  }

  template <bool PAST>
  __device__ __forceinline__ void store(float* row, bool on, const float* v) const {
    if (!on) return;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (count[k] == 4) {
        const lf4 t = {v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
        lf4* q = reinterpret_cast<lf4*>(row + at[k]);
        if constexpr (PAST) __builtin_nontemporal_store(t, q); else *q = t;
      } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
          if (j < count[k]) row[at[k] + j] = v[4 * k + j];
      }
    }
  }

  __device__ __forceinline__ bool valid(int i) const { return i % 4 < count[i / 4]; }
};

// sigmoid(z) and sigmoid(-z): q = e^-|z| as a power of two of a product in two parts (beyond 200 nothing changes), and a
// reciprocal with one step of Newton's.  Over 1.6 million z in [-80, 80] SiLU is within 3.8 units in the last place and its
// slope within 3.8 x 2^-24.  With expf and a division a third of all
// instructions is theirs (forward, 20,000 x 1,000: 43 us against 37).
__device__ __forceinline__ void sigmoids(float z, float& open, float& closed) {
  const float size = -fminf(fabsf(z), 200.f), high = size * kLog2E;
  const float low = fmaf(size, kLog2E, -high) + size * kLog2ELow;
  const float power = __builtin_amdgcn_exp2f(high), q = fmaf(power, low * kLn2, power), d = 1.f + q;
  const float near = __builtin_amdgcn_rcpf(d), inv = fmaf(fmaf(-d, near, 1.f), near, near);
  open = z < 0.f ? q * inv : inv;
  closed = z < 0.f ? inv : q * inv;
}

// A row's mean and r2 = 1 / (variance + eps).
template <int K, int WIDE>
__device__ __forceinline__ void statistics(const LayerNormArgs& a, const Columns<K, WIDE>& c, const float* x, double* lds,
                                           int& turn, double& mean, double& r2) {
  const double n = 1.0 / a.width;
  double sum[1] = {0.0};
#pragma unroll
  for (int i = 0; i < 4 * K; ++i) sum[0] += static_cast<double>(x[i]);
  row_sums<1, WIDE>(sum, a.threads, lds, turn);
  mean = sum[0] * n;
  sum[0] = 0.0;
#pragma unroll
  for (int i = 0; i < 4 * K; ++i) {
    const double d = c.valid(i) ? static_cast<double>(x[i]) - mean : 0.0;
    sum[0] += d * d;
  }
  row_sums<1, WIDE>(sum, a.threads, lds, turn);
  r2 = 1.0 / (sum[0] * n + static_cast<double>(a.eps));
}

template <int K, int WIDE, bool SILU>
__global__ void __launch_bounds__(ln_block(WIDE)) layer_norm_forward_kernel(const LayerNormArgs a) {
  __shared__ double lds[WIDE ? 2 * kSums * kMaxWaves : 1];
  int turn = 0;
  const Columns<K, WIDE> c(a);
  float w[4 * K], b[4 * K];
  c.load(a.weight, true, w);
  c.load(a.bias, true, b);
  const int64_t step = static_cast<int64_t>(gridDim.x) * a.groups;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * a.groups; base < a.rows; base += step) {
    const int64_t row = base + c.group;
    const bool on = row < a.rows;
    float x[4 * K];
    c.load(a.x + row * a.width, on, x);
    double mean, r2;
    statistics<K, WIDE>(a, c, x, lds, turn, mean, r2);
    const float rho = static_cast<float>(sqrt(r2));
#pragma unroll
    for (int i = 0; i < 4 * K; ++i) {
      const float z = fmaf(w[i], static_cast<float>(static_cast<double>(x[i]) - mean) * rho, b[i]);
      if constexpr (SILU) {
        float open, closed;
        sigmoids(z, open, closed);
        x[i] = z * open;
      } else {
        x[i] = z;
      }
    }
    c.template store<false>(a.y + row * a.width, on, x);
  }
}

// A workgroup's weight gradients: its threads' sums over their rows, added up over the rows side by side.
template <int K, int WIDE>
__device__ __forceinline__ void leave_partial(const LayerNormArgs& a, const Columns<K, WIDE>& c, const float* gw,
                                              const float* gb) {
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.width;
  if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < 4 * K; ++i)
      if (c.valid(i)) {
        out[c.at[i / 4] + i % 4] = gw[i];
        out[a.width + c.at[i / 4] + i % 4] = gb[i];
      }
  } else {
    __shared__ float sums[4 * K * kLnThreads];       // [groups][a row's threads][4 K]
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4 * K; ++i)       // columns in order within a group of rows
        sums[c.group * (4 * K * a.threads) + c.at[i / 4] + i % 4] = side ? gb[i] : gw[i];
      __syncthreads();
      for (int column = threadIdx.x; column < a.width; column += kLnThreads) {
        float sum = 0.f;
        for (int g = 0; g < a.groups; ++g) sum += sums[g * (4 * K * a.threads) + column];
        out[side * a.width + column] = sum;
      }
    }
  }
}

template <int K, int WIDE, bool SILU>
__global__ void __launch_bounds__(ln_block(WIDE)) layer_norm_backward_kernel(const LayerNormArgs a) {
  __shared__ double lds[WIDE ? 2 * kSums * kMaxWaves : 1];
  int turn = 0;
  const Columns<K, WIDE> c(a);
  const double n = 1.0 / a.width;
  float w[4 * K], b[4 * K], gw[4 * K] = {}, gb[4 * K] = {};
  c.load(a.weight, true, w);
  c.load(SILU ? a.bias : nullptr, true, b);
  const int64_t step = static_cast<int64_t>(gridDim.x) * a.groups;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * a.groups; base < a.rows; base += step) {
    const int64_t row = base + c.group;
    const bool on = row < a.rows;
    float x[4 * K], dz[4 * K];
    c.load(a.x + row * a.width, on, x);
    c.load(a.dy + row * a.width, on, dz);
    double mean, r2;
    statistics<K, WIDE>(a, c, x, lds, turn, mean, r2);
    const float rho = static_cast<float>(sqrt(r2));
    double sums[2] = {0.0, 0.0};      // of e and of e xc
#pragma unroll
    for (int i = 0; i < 4 * K; ++i) {
      const double xc = static_cast<double>(x[i]) - mean;
      const float xh = static_cast<float>(xc) * rho;
      if constexpr (SILU) {
        const float z = fmaf(w[i], xh, b[i]);
        float open, closed;
        sigmoids(z, open, closed);
        dz[i] *= open * fmaf(z, closed, 1.f);
      }
      gw[i] = fmaf(dz[i], xh, gw[i]);
      gb[i] += dz[i];
      const double e = static_cast<double>(w[i] * dz[i]);
      sums[0] += e;
      sums[1] += e * xc;
    }
    if (!a.dx) continue;
    row_sums<2, WIDE>(sums, a.threads, lds, turn);
    const double middle = sums[0] * n, along = sums[1] * n * r2;
#pragma unroll
    for (int i = 0; i < 4 * K; ++i) {
      const double e = static_cast<double>(w[i] * dz[i]), xc = static_cast<double>(x[i]) - mean;
      x[i] = rho * static_cast<float>(e - middle - xc * along);
    }
    c.template store<true>(a.dx + row * a.width, on, x);
  }
  if (a.partial) leave_partial<K, WIDE>(a, c, gw, gb);
}

template <int K, int WIDE, bool SILU>
__global__ void __launch_bounds__(ln_block(WIDE), K == 1 ? 4 : 1) layer_norm_second_kernel(const LayerNormArgs a) {
  __shared__ double lds[WIDE ? 2 * kSums * kMaxWaves : 1];
  int turn = 0;
  const Columns<K, WIDE> c(a);
  const double n = 1.0 / a.width;
  float w[4 * K], b[4 * K], gw[4 * K] = {}, gb[4 * K] = {};
  c.load(a.weight, true, w);
  c.load(SILU ? a.bias : nullptr, true, b);
  const int64_t step = static_cast<int64_t>(gridDim.x) * a.groups;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * a.groups; base < a.rows; base += step) {
    const int64_t row = base + c.group;
    const bool on = row < a.rows;
    float x[4 * K], dy[4 * K], u[4 * K], slope[SILU ? 4 * K : 1], bend[SILU ? 4 * K : 1];
    c.load(a.x + row * a.width, on, x);
    c.load(a.dy + row * a.width, on, dy);
    c.load(a.u + row * a.width, on, u);
    double mean, r2;
    statistics<K, WIDE>(a, c, x, lds, turn, mean, r2);
    const double root = sqrt(r2);
    const float rho = static_cast<float>(root);
    double head[2] = {0.0, 0.0}, pair[3] = {0.0, 0.0, 0.0};     // of u, e | u xc, e xc, u e
#pragma unroll
    for (int i = 0; i < 4 * K; ++i) {
      const double xc = static_cast<double>(x[i]) - mean;
      if constexpr (SILU) {
        const float z = fmaf(w[i], static_cast<float>(xc) * rho, b[i]);
        float open, closed;
        sigmoids(z, open, closed);
        slope[i] = open * fmaf(z, closed, 1.f);
        bend[i] = open * closed * fmaf(z, closed - open, 2.f) * dy[i];
      }
      const float dz = SILU ? slope[i] * dy[i] : dy[i];
      const double e = static_cast<double>(w[i] * dz), ui = static_cast<double>(u[i]);
      head[0] += ui;
      head[1] += e;
      pair[0] += ui * xc;
      pair[1] += e * xc;
      pair[2] += ui * e;
    }
    row_sums<2, WIDE>(head, a.threads, lds, turn);
    row_sums<3, WIDE>(pair, a.threads, lds, turn);
    const double mean_u = head[0] * n, mean_e = head[1] * n;
    const double P = pair[0] * n, Q = pair[1] * n, R = pair[2] * n - mean_u * mean_e;
    const double turned = R - 3.0 * r2 * P * Q, cube = root * r2;
    double back[2] = {0.0, 0.0};      // of w s and of w s xc
#pragma unroll
    for (int i = 0; i < 4 * K; ++i) {
      const double xc = static_cast<double>(x[i]) - mean;
      const double av = static_cast<double>(u[i]) - mean_u;
      const float t = rho * static_cast<float>(av - xc * (r2 * P));
      const float dz = SILU ? slope[i] * dy[i] : dy[i];
      const double cv = static_cast<double>(w[i] * dz) - mean_e;
      u[i] = static_cast<float>(-cube * (xc * turned + Q * av + P * cv));
      gw[i] = fmaf(t, dz, gw[i]);
      if constexpr (SILU) {
        const float s = w[i] * t * bend[i];
        gw[i] = fmaf(s, static_cast<float>(xc) * rho, gw[i]);
        gb[i] += s;
        bend[i] = w[i] * s;
        back[0] += static_cast<double>(bend[i]);
        back[1] += static_cast<double>(bend[i]) * xc;
        dy[i] = w[i] * t * slope[i];
      } else {
        dy[i] = w[i] * t;
      }
    }
    if (a.ddy) c.template store<true>(a.ddy + row * a.width, on, dy);
    if (!a.dx) continue;
    if constexpr (SILU) {
      row_sums<2, WIDE>(back, a.threads, lds, turn);
      const double middle = back[0] * n, along = back[1] * n * r2;
#pragma unroll
      for (int i = 0; i < 4 * K; ++i) {
        const double xc = static_cast<double>(x[i]) - mean;
        u[i] = fmaf(rho, static_cast<float>(static_cast<double>(bend[i]) - middle - xc * along), u[i]);
      }
    }
    c.template store<true>(a.dx + row * a.width, on, u);
  }
  if (a.partial) leave_partial<K, WIDE>(a, c, gw, gb);
}

struct LnShape {
  int threads, groups, wide, k;
  int64_t grid;
};

// A row within a wave up to 768 columns, 12 of a thread, then 4 or 16 waves with barriers.  Against 4 waves a row from 513
// columns on, 16,000 x 520 and x 768: forward 26 -> 16 and 24 -> 18 us, gradients 46 -> 29 and 46 -> 35, second 70 -> 45
// and 69 -> 49, with SiLU 97 -> 86 and 97 -> 83.  With 16 of a thread for 769 to 1,024 columns it is even: 5,003 x 1,001
// with SiLU 13.4 -> 13.3, 22.9 -> 24.2, 39 -> 49, without 12.1 -> 11.7, 19.8 -> 20.8, 29 -> 28.
LnShape ln_shape(int width, int64_t rows) {
  LnShape s;
  const int quads = (width + 3) / 4;
  s.wide = quads <= 3 * kRowWave ? 0 : quads <= 4 * kLnThreads ? 1 : 2;
  if (s.wide) {
    s.threads = ln_block(s.wide);
    s.groups = 1;
  } else {
    s.threads = 1;
    while (s.threads < quads && s.threads < kRowWave) s.threads *= 2;
    s.groups = kLnThreads / s.threads;
  }
  s.k = (quads + s.threads - 1) / s.threads;
  if (s.wide && s.k == 3) s.k = 4;
  s.grid = (rows + s.groups - 1) / s.groups;
  return s;
}

int64_t ln_groups(const LnShape& s) { return s.grid < kLnGroups ? s.grid : kLnGroups; }

using LnKernel = void (*)(LayerNormArgs);

template <int K, int WIDE, bool SILU>
LnKernel ln_kernel(int order) {
  return order == 0   ? layer_norm_forward_kernel<K, WIDE, SILU>
         : order == 1 ? layer_norm_backward_kernel<K, WIDE, SILU>
                      : layer_norm_second_kernel<K, WIDE, SILU>;
}

template <bool SILU>
LnKernel ln_kernel(int order, const LnShape& s) {
  if (s.wide == 0)
    return s.k == 1   ? ln_kernel<1, 0, SILU>(order)
           : s.k == 2 ? ln_kernel<2, 0, SILU>(order)
                      : ln_kernel<3, 0, SILU>(order);
  if (s.wide == 1)
    return s.k == 1 ? ln_kernel<1, 1, SILU>(order) : s.k == 2 ? ln_kernel<2, 1, SILU>(order) : ln_kernel<4, 1, SILU>(order);
  return ln_kernel<2, 2, SILU>(order);
}

bool ln_valid(int width, int activation, float eps, int64_t rows) {
  return rows >= 0 && rows <= (int64_t{1} << 40) && width >= 1 && width <= ICTC_LAYER_NORM_MAX_WIDTH && eps > 0.f &&
         eps < INFINITY && (activation == ICTC_ACTIVATION_NONE || activation == ICTC_ACTIVATION_SILU);
}

int ln_run(int order, LayerNormArgs a, int width, int activation, float eps, int64_t rows, float* dweight, float* dbias,
           hipStream_t stream) {
  const LnShape s = ln_shape(width, rows);
  a.rows = rows, a.width = width, a.eps = eps, a.threads = s.threads, a.groups = s.groups;
  const bool weights = dweight || dbias;
  if (!weights) a.partial = nullptr;
  const int64_t most = weights ? ln_groups(s) : (int64_t{1} << 31) / ln_block(s.wide);      // threads within 32 bits
  const int64_t grid = s.grid < most ? s.grid : most;
  if (grid) {
    const LnKernel kernel = activation == ICTC_ACTIVATION_SILU ? ln_kernel<true>(order, s) : ln_kernel<false>(order, s);
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(ln_block(s.wide)), 0, stream, a);
    if (hipGetLastError() != hipSuccess) return ICTC_ERR_LAUNCH;
  }
  if (weights) {
    hipLaunchKernelGGL(norm_weight_kernel, dim3((2 * width + kColumns - 1) / kColumns), dim3(kColumns * kSlices), 0,
                       stream, a.partial, dweight, dbias, static_cast<int>(grid), width);
    if (hipGetLastError() != hipSuccess) return ICTC_ERR_LAUNCH;
  }
  return ICTC_OK;
}

}  // namespace
}  // namespace ictc

extern "C" {

int64_t ictc_hip_layer_norm_workspace(int width, int64_t rows) {
  using namespace ictc;
  if (!ln_valid(width, ICTC_ACTIVATION_NONE, 1.f, rows)) return -ICTC_ERR_INVALID_ARGUMENT;
  const int64_t groups = ln_groups(ln_shape(width, rows));
  return (groups ? groups : 1) * 2 * width;
}

int ictc_hip_layer_norm_forward(const float* x, const float* weight, const float* bias, float* y, int width,
                                int activation, float eps, int64_t rows, hipStream_t stream) {
  using namespace ictc;
  if (!ln_valid(width, activation, eps, rows)) return ICTC_ERR_INVALID_ARGUMENT;
  if (rows == 0) return ICTC_OK;
  if (!x || !weight || !y) return ICTC_ERR_INVALID_ARGUMENT;
  LayerNormArgs a = {};
  a.x = x, a.weight = weight, a.bias = bias, a.y = y;
  return ln_run(0, a, width, activation, eps, rows, nullptr, nullptr, stream);
}

int ictc_hip_layer_norm_backward(const float* x, const float* weight, const float* bias, const float* grad_y, float* dx,
                                 float* dweight, float* dbias, float* workspace, int64_t workspace_floats, int width,
                                 int activation, float eps, int64_t rows, hipStream_t stream) {
  using namespace ictc;
  if (!ln_valid(width, activation, eps, rows)) return ICTC_ERR_INVALID_ARGUMENT;
  if ((dweight || dbias) && (!workspace || workspace_floats < ictc_hip_layer_norm_workspace(width, rows)))
    return ICTC_ERR_INVALID_ARGUMENT;
  if (!dx && !dweight && !dbias) return ICTC_OK;
  if (rows == 0 && !dweight && !dbias) return ICTC_OK;
  if (rows && (!x || !weight || !grad_y)) return ICTC_ERR_INVALID_ARGUMENT;
  LayerNormArgs a = {};
  a.x = x, a.weight = weight, a.bias = bias, a.dy = grad_y, a.dx = dx, a.partial = workspace;
  return ln_run(1, a, width, activation, eps, rows, dweight, dbias, stream);
}

int ictc_hip_layer_norm_second(const float* x, const float* weight, const float* bias, const float* grad_y,
                               const float* cot_x, float* dx, float* dgrad_y, float* dweight, float* dbias,
                               float* workspace, int64_t workspace_floats, int width, int activation, float eps,
                               int64_t rows, hipStream_t stream) {
  using namespace ictc;
  if (!ln_valid(width, activation, eps, rows)) return ICTC_ERR_INVALID_ARGUMENT;
  if ((dweight || dbias) && (!workspace || workspace_floats < ictc_hip_layer_norm_workspace(width, rows)))
    return ICTC_ERR_INVALID_ARGUMENT;
  if (!dx && !dgrad_y && !dweight && !dbias) return ICTC_OK;
  if (rows == 0 && !dweight && !dbias) return ICTC_OK;
  if (rows && (!x || !weight || !grad_y || !cot_x)) return ICTC_ERR_INVALID_ARGUMENT;
  LayerNormArgs a = {};
  a.x = x, a.weight = weight, a.bias = bias, a.dy = grad_y, a.u = cot_x, a.dx = dx, a.ddy = dgrad_y;
  a.partial = workspace;
  return ln_run(2, a, width, activation, eps, rows, dweight, dbias, stream);
}

}  // extern "C"
