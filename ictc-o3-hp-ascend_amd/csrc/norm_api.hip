// Norms of a residual block on equivariant node features, gfx950: the norm before a block, and the block's
// end in one pass (norm of its output, gate, residual sum, norm before the next block), each with its
// gradients and with the gradients of those (forces are gradients, and training on them asks for more).
//
// A row v holds degrees l = 0..L, per degree a [C, 2l+1] block.  With a_l = 1 / ((L+1) C (2l+1)),
//   q(v) = sum a_l v_lcm^2     rho(v) = (q + eps)^(-1/2)     N(v; w)_lcm = w_lc v_lcm rho(v)
// one statistic for the row: rotations mix only the components m of one l and c, on which neither q nor
// w depends, so N commutes with them; and every degree has the same share in q.
//
//   forward   h = x + k . b rho(b), k_lc = s sigmoid(g_lc) post_lc      y = N(h; pre)
//
//   VJP of V(v; e) = rho e - rho^3 a v <e, v>, the adjoint of N at cotangent e / w, is what both norms' gradients
//   are made of.  With cotangents dh, dy:
//     r = dh + V(h; pre dy)      dx = r      db = V(b; k r)
//     dg = s sigmoid' post rho_b <r, b>_lc   dpost = sum_n s sigmoid rho_b <r, b>_lc   dpre = sum_n rho_h <dy, h>_lc
//
//   second order, cotangents X, B, G of dx, db, dg.  For Phi = <B, V(v; e)>, S1 = <B, e>, S2 = <a B, v>, S3 = <e, v>:
//     dPhi/de = rho B - rho^3 S2 v
//     dPhi/dv = -rho^3 a v S1 + 3 rho^5 a v S2 S3 - rho^3 (a B S3 + e S2)
//   once at the block (v = b, e = k r), whose dPhi/de gives r's cotangent R = X + k dPhi/de + (G's part), and
//   once at the next norm (v = h, e = pre dy, R in B's place).  h's own cotangent H then goes back through the
//   forward pass in the same kernel: H to x, V(b; k H) to b, and so on (another pass over b and H otherwise,
//   and sums of two gradients of every operand: 100 us of 414 for 8,192 rows of C = 128, L = 3).
//
// All of it is bound by memory: a row is read into registers once, its sums are taken there, and its results
// are written once.  The gradients' sums and projections are in 64 bits: they take away the part of a
// cotangent along v (all but eps / (q + eps) of it for a row with one large entry), and the difference is
// as exact as the operands.  One thread holds one channel's (L+1)^2 components of every operand, so weights, gates and
// their gradients need no exchange between threads; its 1, 3, 5 and 7 components are loaded with vectors of
// that many words, which side by side fill whole lines.  A row's threads are a power of two of
// a wave's (for few channels, see shape_of) or up to 16 waves, whose sums meet in LDS.  (One degree to a wave, all of a
// row's in one workgroup: 325 us for the second derivatives of 8,192 rows of C = 128, L = 3; eight waves at each
// barrier.)
//
// Measured at C = 128, L = 3 (bytes as each kernel reads and writes them): forward of 32,768 rows 204 us, 5.6 TB/s;
// of 8,192 rows 48 us (6.0), gradients 81 us with weight gradients (5.4), second derivatives 158 us (4.6: two waves to
// a SIMD, and 1,900 instructions a wave and row).  The norm alone, 8,192 rows: gradients 43 us (4.7), second
// derivatives 67 (5.0).  With degrees to 3 registers spill in wider rows: gradients 3.6 to 4.7 TB/s and second
// derivatives 2.5 to 3.5 at 257 to 512 channels, 2.3 to 3.0 and 1.4 to 1.5 beyond.  These are the present code's; the
// pairs of times at single choices below are from when each was made, on the code of that time.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ictc_hip.h"
#include "row_sums.hpp"

namespace ictc {
namespace {

constexpr int kNormWave = 64;
constexpr int kNormThreads = 256;            // of a workgroup whose rows fit into a wave
constexpr int kNormMaxThreads = ICTC_NORM_MAX_CHANNELS;
constexpr int kNormGroups = 1024;            // workgroups that leave partial weight gradients

typedef float nf4 __attribute__((ext_vector_type(4), aligned(4)));

// Threads of a workgroup by where a row's threads are: 0 within a wave, else in up to 4, 8 or 16 waves of their own.
constexpr int most_threads(int wide) {
  return wide < 2 ? kNormThreads : wide == 2 ? 2 * kNormThreads : kNormMaxThreads;
}

struct NormArgs {
  const float *x, *block, *gate, *post, *pre, *h, *dh, *dy, *cx, *cb, *cg;
  float *out_h, *out_y, *dx, *db, *dg;
  float *gx, *gb, *gg, *gdh, *gdy;
  float* partial;             // per workgroup [2][L+1][C]: post's and pre's gradients
  int64_t rows;
  int64_t width_x;            // floats of a row of x, dx and cx
  int channels;
  int input_lmax;             // degrees of x that a row takes part with (at most L)
  int threads;                // of a row
  int groups;                 // rows of a workgroup at a time
  float scale, eps;
};

template <int N>
__device__ __forceinline__ void load_n(const float* p, float* v) {
  if constexpr (N == 1) {
    v[0] = *p;
  } else if constexpr (N == 3) {
    v[0] = p[0], v[1] = p[1], v[2] = p[2];      // (a vector type of three would take up four)
  } else {
    const nf4 t = *reinterpret_cast<const nf4*>(p);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    load_n<N - 4>(p + 4, v + 4);
  }
}

// The gradients' kernels store past the caches (8,192 rows of C = 128, L = 3: 77 us against 86, second
// derivatives 166 against 172; 2,048 rows: 24.0 against 24.3), the forward pass does not (51 us either way, 203
// against 207 for 32,768 rows), and no loads do (214, and 29 against 24 for the gradients of 2,048).
template <bool PAST, int N>
__device__ __forceinline__ void store_n(float* p, const float* v) {
  if constexpr (N == 1 || N == 3) {
#pragma unroll
    for (int m = 0; m < N; ++m) {
      if constexpr (PAST) __builtin_nontemporal_store(v[m], p + m); else p[m] = v[m];
    }
  } else {
    const nf4 t = {v[0], v[1], v[2], v[3]};
    nf4* q = reinterpret_cast<nf4*>(p);
    if constexpr (PAST) __builtin_nontemporal_store(t, q); else *q = t;
    store_n<PAST, N - 4>(p + 4, v + 4);
  }
}

// Where a thread's components of each degree are, in bytes from the workgroup's first row: 32 bits beside a
// uniform address.
template <int L>
struct Offsets {
  uint32_t at[L + 1];
};

template <int L>
__device__ __forceinline__ Offsets<L> offsets(int64_t width, int C, int c, int group) {
  Offsets<L> o;
#pragma unroll
  for (int l = 0; l <= L; ++l)
    o.at[l] = (static_cast<uint32_t>(group) * static_cast<uint32_t>(width) + C * l * l + c * (2 * l + 1)) * 4u;
  return o;
}

__device__ __forceinline__ const float* at_bytes(const float* p, uint32_t bytes) {
  return reinterpret_cast<const float*>(reinterpret_cast<const char*>(p) + bytes);
}

__device__ __forceinline__ float* at_bytes(float* p, uint32_t bytes) {
  return reinterpret_cast<float*>(reinterpret_cast<char*>(p) + bytes);
}

// A thread's components of the degrees up to `most`; the others are zero.
template <int L, int l = 0>
__device__ __forceinline__ void load_row(const float* rows, const Offsets<L>& o, int most, float* v) {
  if constexpr (l <= L) {
    if (l <= most) {
      load_n<2 * l + 1>(at_bytes(rows, o.at[l]), v + l * l);
    } else {
#pragma unroll
      for (int m = 0; m < 2 * l + 1; ++m) v[l * l + m] = 0.f;
    }
    load_row<L, l + 1>(rows, o, most, v);
  }
}

template <bool PAST, int L, int l = 0>
__device__ __forceinline__ void store_row(float* rows, const Offsets<L>& o, int most, const float* v) {
  if constexpr (l <= L) {
    if (l <= most) store_n<PAST, 2 * l + 1>(at_bytes(rows, o.at[l]), v + l * l);
    store_row<PAST, L, l + 1>(rows, o, most, v);
  }
}

template <int L>
__device__ __forceinline__ void clear_row(float* v) {
#pragma unroll
  for (int i = 0; i < (L + 1) * (L + 1); ++i) v[i] = 0.f;
}

constexpr int degree_of(int i) { return i < 1 ? 0 : i < 4 ? 1 : i < 9 ? 2 : 3; }

// The rows of a workgroup: which of them is this thread's, and the channel that it holds.
struct Place {
  int c, group;
  bool holds;
};

template <int WIDE>
__device__ __forceinline__ Place place(const NormArgs& a) {
  Place p;
  p.group = WIDE ? 0 : threadIdx.x / a.threads;
  p.c = WIDE ? threadIdx.x : threadIdx.x & (a.threads - 1);
  p.holds = p.c < a.channels;
  return p;
}

template <int L>
__device__ __forceinline__ void load_weight(const float* w, int C, const Place& t, float* out) {
#pragma unroll
  for (int l = 0; l <= L; ++l) out[l] = w && t.holds ? w[l * C + t.c] : 0.f;
}

template <int L, typename T>
__device__ __forceinline__ void shares(int C, T* a) {
#pragma unroll
  for (int l = 0; l <= L; ++l) a[l] = T(1) / static_cast<T>((L + 1) * (2 * l + 1) * C);
}

// One degree's sum of products of a thread's components.
template <int l>
__device__ __forceinline__ double product(const float* u, const float* v) {
  double s = 0.0;
#pragma unroll
  for (int m = 0; m < 2 * l + 1; ++m) s += static_cast<double>(u[l * l + m]) * static_cast<double>(v[l * l + m]);
  return s;
}

// f(Degree<0>{}), ..., f(Degree<L>{})
template <int l>
struct Degree {
  static constexpr int value = l;
};

template <int L, int l = 0, typename F>
__device__ __forceinline__ void degrees(F&& f) {
  if constexpr (l <= L) {
    f(Degree<l>{});
    degrees<L, l + 1>(f);
  }
}

// Values that are what they are from here on: the compiler neither carries them over in the 64-bit form it has
// of them nor moves the operations that make them behind a condition (all their operands would stay).
template <int N>
__device__ __forceinline__ void narrow(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i]));
}

// Sums over a thread's components of products, by degree.
template <int L>
__device__ __forceinline__ void products(const float* u, const float* v, double* out) {
#pragma unroll
  for (int l = 0; l <= L; ++l) out[l] = 0.0;
#pragma unroll
  for (int i = 0; i < (L + 1) * (L + 1); ++i)
    out[degree_of(i)] += static_cast<double>(u[i]) * static_cast<double>(v[i]);
}

// Gates of one row and what they leave, sigmoid(g) and sigmoid(-g), both to their last bits.
template <int L>
__device__ __forceinline__ void gates(const NormArgs& a, int64_t base, uint32_t own_gate, bool on, float* open,
                                      float* closed) {
#pragma unroll
  for (int l = 0; l <= L; ++l) {
    open[l] = 1.f, closed[l] = 0.f;
    if (a.gate && on) {
      const float g = *at_bytes(a.gate + (base * (L + 1) + l) * a.channels, own_gate);
      const float z = expf(-fabsf(g)), inv = 1.f / (1.f + z);
      open[l] = g < 0.f ? z * inv : inv;
      closed[l] = g < 0.f ? inv : z * inv;
    }
  }
}

template <int L, int WIDE, bool BLOCK, bool NEXT>
__global__ void __launch_bounds__(most_threads(WIDE)) norm_forward_kernel(const NormArgs a) {
  constexpr int D = (L + 1) * (L + 1);
  __shared__ double lds[WIDE ? 2 * kSums * kMaxWaves : 1];
  int turn = 0;
  const Place t = place<WIDE>(a);
  const int C = a.channels;
  const int64_t width = static_cast<int64_t>(C) * D;
  float post[L + 1], pre[L + 1], share[L + 1];
  load_weight<L>(BLOCK ? a.post : nullptr, C, t, post);
  load_weight<L>(NEXT ? a.pre : nullptr, C, t, pre);
  shares<L>(C, share);
  const Offsets<L> own = offsets<L>(width, C, t.c, t.group), own_x = offsets<L>(a.width_x, C, t.c, t.group);
  const uint32_t own_gate = (static_cast<uint32_t>(t.group) * (L + 1) * C + t.c) * 4u;
  const int64_t step = static_cast<int64_t>(gridDim.x) * a.groups;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * a.groups; base < a.rows; base += step) {
    const int64_t row = base + t.group;
    const bool on = t.holds && row < a.rows;
    float h[D], b[D];
    clear_row<L>(h);
    clear_row<L>(b);
    if (on) {
      if constexpr (BLOCK) load_row<L>(a.block + base * width, own, L, b);
      load_row<L>(a.x + base * a.width_x, own_x, a.input_lmax, h);
    }
    if constexpr (BLOCK) {
      float open[L + 1], closed[L + 1];
      gates<L>(a, base, own_gate, on, open, closed);
      float sums[1] = {0.f};
#pragma unroll
      for (int i = 0; i < D; ++i) sums[0] += share[degree_of(i)] * b[i] * b[i];
      row_sums<1, WIDE>(sums, a.threads, lds, turn);
      const float rho = 1.f / sqrtf(sums[0] + a.eps);
#pragma unroll
      for (int i = 0; i < D; ++i) h[i] += a.scale * open[degree_of(i)] * post[degree_of(i)] * rho * b[i];
      if (on) store_row<false, L>(a.out_h + base * width, own, L, h);
    }
    if constexpr (NEXT) {
      float sums[1] = {0.f};
#pragma unroll
      for (int i = 0; i < D; ++i) sums[0] += share[degree_of(i)] * h[i] * h[i];
      row_sums<1, WIDE>(sums, a.threads, lds, turn);
      const float rho = 1.f / sqrtf(sums[0] + a.eps);
#pragma unroll
      for (int i = 0; i < D; ++i) h[i] *= pre[degree_of(i)] * rho;
      if (on) store_row<false, L>(a.out_y + base * width, own, L, h);
    }
  }
}

// A workgroup's weight gradients: each thread's over its rows, then over the workgroup's row groups, in order.
template <int L, int WIDE>
__device__ __forceinline__ void write_partial(const NormArgs& a, const Place& t, const float* post, const float* pre,
                                              double* lds) {
  float* stage = reinterpret_cast<float*>(lds);
  const int C = a.channels;
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * (L + 1) * C;
#pragma unroll
  for (int l = 0; l <= L; ++l)
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const float mine = w ? pre[l] : post[l];
      if constexpr (WIDE) {
        if (t.holds) out[(w * (L + 1) + l) * C + t.c] = mine;
      } else {
        __syncthreads();
        stage[threadIdx.x] = mine;
        __syncthreads();
        if (t.group == 0 && t.holds) {
          float sum = 0.f;
          for (int g = 0; g < a.groups; ++g) sum += stage[g * a.threads + t.c];
          out[(w * (L + 1) + l) * C + t.c] = sum;
        }
      }
    }
}

template <int L, int WIDE, bool BLOCK, bool NEXT>
__global__ void __launch_bounds__(most_threads(WIDE)) norm_backward_kernel(const NormArgs a) {
  constexpr int D = (L + 1) * (L + 1);
  __shared__ double lds[WIDE ? 2 * kSums * kMaxWaves : kNormThreads / 2];
  int turn = 0;
  const Place t = place<WIDE>(a);
  const int C = a.channels;
  const int64_t width = static_cast<int64_t>(C) * D;
  float post[L + 1], pre[L + 1], dpost[L + 1] = {}, dpre[L + 1] = {};
  double share[L + 1];
  load_weight<L>(BLOCK ? a.post : nullptr, C, t, post);
  load_weight<L>(NEXT ? a.pre : nullptr, C, t, pre);
  shares<L>(C, share);
  const Offsets<L> own = offsets<L>(width, C, t.c, t.group), own_x = offsets<L>(a.width_x, C, t.c, t.group);
  const uint32_t own_gate = (static_cast<uint32_t>(t.group) * (L + 1) * C + t.c) * 4u;
  const int64_t step = static_cast<int64_t>(gridDim.x) * a.groups;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * a.groups; base < a.rows; base += step) {
    const int64_t row = base + t.group;
    const bool on = t.holds && row < a.rows;
    float h[D], b[D], r[D], dy[D];
    clear_row<L>(h);
    clear_row<L>(b);
    clear_row<L>(r);
    clear_row<L>(dy);
    if (on) {
      if constexpr (NEXT) {
        load_row<L>(a.h + base * width, own, L, h);
        load_row<L>(a.dy + base * width, own, L, dy);
      }
      if constexpr (BLOCK) load_row<L>(a.block + base * width, own, L, b);
      if (a.dh) load_row<L>(a.dh + base * width, own, L, r);
    }
    double hh[L + 1], yh[L + 1], bb[L + 1];
    products<L>(h, h, hh);
    products<L>(dy, h, yh);
    products<L>(b, b, bb);
    double sums[3] = {};      // q(h), <pre dy, h>, q(b)
#pragma unroll
    for (int l = 0; l <= L; ++l) {
      sums[0] += share[l] * hh[l];
      sums[1] += pre[l] * yh[l];
      sums[2] += share[l] * bb[l];
    }
    narrow(h), narrow(b), narrow(dy);
    row_sums<3, WIDE>(sums, a.threads, lds, turn);
    if constexpr (NEXT) {
      const double rho = 1.0 / sqrt(sums[0] + a.eps), pull = rho * rho * rho * sums[1];
#pragma unroll
      for (int i = 0; i < D; ++i) {
        const int l = degree_of(i);
        r[i] = static_cast<float>(r[i] + pre[l] * rho * dy[i] - share[l] * pull * h[i]);
      }
#pragma unroll
      for (int l = 0; l <= L; ++l) dpre[l] += static_cast<float>(rho * yh[l]);
    }
    narrow(r);
    if (on && a.dx) {
      store_row<true, L>(a.dx + base * a.width_x, own_x, a.input_lmax, r);
      float* out = a.dx + row * a.width_x;
      for (int64_t i = width + t.c; i < a.width_x; i += C) out[i] = 0.f;     // degrees of x beyond the block's
    }
    if constexpr (BLOCK) {
      float open[L + 1], closed[L + 1];
      gates<L>(a, base, own_gate, on, open, closed);
      double e[L + 1], k[L + 1], dot[1] = {0.0};
      products<L>(r, b, e);
#pragma unroll
      for (int l = 0; l <= L; ++l) {
        k[l] = a.scale * open[l] * post[l];
        dot[0] += k[l] * e[l];
      }
      narrow(r), narrow(b);
      row_sums<1, WIDE>(dot, a.threads, lds, turn);
      const double rho = 1.0 / sqrt(sums[2] + a.eps), pull = rho * rho * rho * dot[0];
#pragma unroll
      for (int i = 0; i < D; ++i) {
        const int l = degree_of(i);
        r[i] = static_cast<float>(rho * k[l] * r[i] - share[l] * pull * b[i]);
      }
      narrow(r);
      if (on && a.db) store_row<true, L>(a.db + base * width, own, L, r);
#pragma unroll
      for (int l = 0; l <= L; ++l) {
        const float along = a.scale * static_cast<float>(rho * e[l]) * open[l];
        dpost[l] += along;
        if (on && a.dg) *at_bytes(a.dg + (base * (L + 1) + l) * C, own_gate) = along * closed[l] * post[l];
      }
    }
  }
  if (a.partial) write_partial<L, WIDE>(a, t, dpost, dpre, lds);
}

// Two operands of every thread, put away in LDS (in place of others, where they are taken back).
template <int N>
__device__ __forceinline__ void put_away(float* stash, const float (&u)[N], const float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    stash[i * blockDim.x] = u[i];
    stash[(N + i) * blockDim.x] = v[i];
  }
  asm volatile("" ::: "memory");
}

template <int N>
__device__ __forceinline__ void take_back(const float* stash, float (&u)[N], float (&v)[N]) {
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) {
    u[i] = stash[i * blockDim.x];
    v[i] = stash[(N + i) * blockDim.x];
  }
}

// Where two of the second derivatives' operands wait in LDS: with all degrees to 3 a thread has 112 values, which with
// what goes beside them do not fit into 256 registers (132 bytes of scratch memory a thread without the LDS, 12 with
// it: 212 us for 8,192 rows of C = 128 against 172; one wave to a SIMD and 512 registers: 209).  With degrees to 2 they
// fit (109 us against 112 for 16,384 rows of C = 64), and rows that share a wave gain nothing (127 us against 130 at
// C = 32).  Rows of more than 256 threads do without it and spill (132 bytes a thread up to 512 threads, 616 beyond,
// where a thread has 128 registers): 40 to 64 KB of LDS would hold the operands of 320 to 512 threads; not built.
constexpr bool stashes(int lmax, int wide, bool block, bool next) { return lmax == 3 && wide == 1 && block && next; }

template <int L, int WIDE, bool BLOCK, bool NEXT>
__global__ void __launch_bounds__(most_threads(WIDE)) __attribute__((amdgpu_waves_per_eu(WIDE == 1 && L == 3 ? 2 : 1)))
norm_second_kernel(const NormArgs a) {
  constexpr int D = (L + 1) * (L + 1);
  __shared__ double lds[WIDE ? 2 * kSums * kMaxWaves : kNormThreads / 2];
  constexpr bool STASH = stashes(L, WIDE, BLOCK, NEXT);
  extern __shared__ float kept[];
  [[maybe_unused]] float* const stash = kept + threadIdx.x;
  int turn = 0;
  const Place t = place<WIDE>(a);
  const int C = a.channels;
  const int64_t width = static_cast<int64_t>(C) * D;
  float post[L + 1], pre[L + 1], gpost[L + 1] = {}, gpre[L + 1] = {};
  double share[L + 1];
  load_weight<L>(BLOCK ? a.post : nullptr, C, t, post);
  load_weight<L>(NEXT ? a.pre : nullptr, C, t, pre);
  shares<L>(C, share);
  const Offsets<L> own = offsets<L>(width, C, t.c, t.group), own_x = offsets<L>(a.width_x, C, t.c, t.group);
  const uint32_t own_gate = (static_cast<uint32_t>(t.group) * (L + 1) * C + t.c) * 4u;
  const int64_t step = static_cast<int64_t>(gridDim.x) * a.groups;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * a.groups; base < a.rows; base += step) {
    const int64_t row = base + t.group;
    const bool on = t.holds && row < a.rows;
    float h[D], b[D], r[D], dy[D], cb[D], R[D];
    clear_row<L>(h);
    clear_row<L>(b);
    clear_row<L>(r);
    clear_row<L>(dy);
    clear_row<L>(cb);
    clear_row<L>(R);
    if (on) {
      if constexpr (NEXT) {
        load_row<L>(a.h + base * width, own, L, h);
        load_row<L>(a.dy + base * width, own, L, dy);
      }
      if constexpr (BLOCK) {
        load_row<L>(a.block + base * width, own, L, b);
        if (a.cb) load_row<L>(a.cb + base * width, own, L, cb);
        if (a.dh) load_row<L>(a.dh + base * width, own, L, r);
      }
      if (a.cx) load_row<L>(a.cx + base * a.width_x, own_x, a.input_lmax, R);
    }
    double sums[4] = {};      // q(h), <pre dy, h>, q(b), <a B, b>
    degrees<L>([&](auto d) {
      constexpr int l = decltype(d)::value;
      if constexpr (NEXT) {
        sums[0] += share[l] * product<l>(h, h);
        sums[1] += pre[l] * product<l>(dy, h);
      }
      if constexpr (BLOCK) {
        sums[2] += share[l] * product<l>(b, b);
        sums[3] += share[l] * product<l>(cb, b);
      }
    });
    narrow(h), narrow(b), narrow(dy), narrow(cb);
    row_sums<4, WIDE>(sums, a.threads, lds, turn);
    const double rho_h = 1.0 / sqrt(sums[0] + a.eps), cube_h = rho_h * rho_h * rho_h;
    const double rho = 1.0 / sqrt(sums[2] + a.eps);
    [[maybe_unused]] float open[L + 1], closed[L + 1], gg[L + 1];
    if constexpr (BLOCK) {
      if constexpr (NEXT) {
        const double pull = cube_h * sums[1];
        degrees<L>([&](auto d) {
          constexpr int l = decltype(d)::value;
          const double up = pre[l] * rho_h, down = share[l] * pull;
#pragma unroll
          for (int i = l * l; i < (l + 1) * (l + 1); ++i) r[i] = static_cast<float>(r[i] + up * dy[i] - down * h[i]);
        });
        narrow(r), narrow(h), narrow(dy);
        if constexpr (STASH) put_away(stash, h, dy);
      }
      float cg[L + 1];
      gates<L>(a, base, own_gate, on, open, closed);
      double e[L + 1], f[L + 1];
      double dots[2] = {};     // S1 and G's part of dPhi/dv's first factor together, S3
      const double s2 = sums[3], cube = rho * rho * rho;
      degrees<L>([&](auto d) {
        constexpr int l = decltype(d)::value;
        cg[l] = a.cg && on ? *at_bytes(a.cg + (base * (L + 1) + l) * C, own_gate) : 0.f;
        e[l] = product<l>(r, b);
        f[l] = product<l>(r, cb);
        const double k = a.scale * open[l] * post[l], slope = a.scale * open[l] * closed[l] * post[l];
        dots[0] += k * f[l] + cg[l] * slope * e[l];      // (slope: the gate's derivative of k)
        dots[1] += k * e[l];
      });
      narrow(r), narrow(b), narrow(cb);
      row_sums<2, WIDE>(dots, a.threads, lds, turn);
      const double along = -cube * dots[0] + 3.0 * cube * rho * rho * s2 * dots[1], away = cube * dots[1];
      degrees<L>([&](auto d) {
        constexpr int l = decltype(d)::value;
        const double k = a.scale * open[l] * post[l], slope = a.scale * open[l] * closed[l] * post[l];
        const double through = rho * cg[l] * slope - cube * s2 * k;
        const float ck = static_cast<float>(rho * f[l] - cube * s2 * e[l]);     // k's cotangent
        const float pass = static_cast<float>(rho * e[l] * cg[l]);              // G's product
        gpost[l] += a.scale * open[l] * (ck + closed[l] * pass);
        gg[l] = static_cast<float>(slope) * (ck + (closed[l] - open[l]) * pass);
        const double ab = share[l] * along, ac = share[l] * away, up = k * rho;
#pragma unroll
        for (int i = l * l; i < (l + 1) * (l + 1); ++i) {
          R[i] = static_cast<float>(R[i] + up * cb[i] + through * b[i]);
          r[i] = static_cast<float>(ab * b[i] - ac * cb[i] + through * r[i]);      // b's gradient from here on
        }
      });
      narrow(R), narrow(r);
      if (on && a.gdh) store_row<true, L>(a.gdh + base * width, own, L, R);
    }
    if constexpr (NEXT) {
      if constexpr (STASH) {
        take_back(stash, h, dy);
        put_away(stash, b, r);
      }
      double dots[2] = {};    // <R, pre dy>, <a R, h>
      degrees<L>([&](auto d) {
        constexpr int l = decltype(d)::value;
        dots[0] += pre[l] * product<l>(R, dy);
        dots[1] += share[l] * product<l>(R, h);
      });
      narrow(R), narrow(h), narrow(dy);
      row_sums<2, WIDE>(dots, a.threads, lds, turn);
      const double along = -cube_h * dots[0] + 3.0 * cube_h * rho_h * rho_h * dots[1] * sums[1];
      const double pull = cube_h * dots[1], turned = cube_h * sums[1];
      degrees<L>([&](auto d) {
        constexpr int l = decltype(d)::value;
        const double ah = share[l] * along, ar = share[l] * turned, ay = pull * pre[l];
        double sum = 0.0;
#pragma unroll
        for (int i = l * l; i < (l + 1) * (l + 1); ++i) {
          const double ce = rho_h * R[i] - pull * h[i];                // the cotangent of e = pre dy
          sum += ce * dy[i];
          h[i] = static_cast<float>(ah * h[i] - ar * R[i] - ay * dy[i]);           // H from here on
          R[i] = static_cast<float>(pre[l] * ce);
        }
        gpre[l] += static_cast<float>(sum);
      });
      narrow(R), narrow(h);
      if (on && a.gdy) store_row<true, L>(a.gdy + base * width, own, L, R);
      if (on && a.gx) {
        store_row<true, L>(a.gx + base * a.width_x, own_x, a.input_lmax, h);
        float* out = a.gx + row * a.width_x;
        for (int64_t i = width + t.c; i < a.width_x; i += C) out[i] = 0.f;         // degrees of x beyond the block's
      }
    }
    if constexpr (BLOCK) {
      if constexpr (NEXT) {
        if constexpr (STASH) take_back(stash, b, r);
        double e[L + 1], dot[1] = {0.0};
        degrees<L>([&](auto d) {
          constexpr int l = decltype(d)::value;
          e[l] = product<l>(h, b);
          dot[0] += static_cast<double>(a.scale * open[l] * post[l]) * e[l];
        });
        narrow(h), narrow(b);
        row_sums<1, WIDE>(dot, a.threads, lds, turn);
        const double pull = rho * rho * rho * dot[0];
        degrees<L>([&](auto d) {
          constexpr int l = decltype(d)::value;
          const double up = rho * static_cast<double>(a.scale * open[l] * post[l]), down = share[l] * pull;
#pragma unroll
          for (int i = l * l; i < (l + 1) * (l + 1); ++i) r[i] = static_cast<float>(r[i] + up * h[i] - down * b[i]);
          const float pass = a.scale * static_cast<float>(rho * e[l]) * open[l];
          gpost[l] += pass;
          gg[l] += pass * closed[l] * post[l];
        });
      }
      narrow(r), narrow(gg);
      if (on && a.gb) store_row<true, L>(a.gb + base * width, own, L, r);
#pragma unroll
      for (int l = 0; l <= L; ++l)
        if (on && a.gg) *at_bytes(a.gg + (base * (L + 1) + l) * C, own_gate) = gg[l];
    }
  }
  if (a.partial) write_partial<L, WIDE>(a, t, gpost, gpre, lds);
}

struct NormShape {
  int threads, groups, block;
  int64_t grid;
  int wide;                   // see most_threads
};

// Rows of up to 64 channels share a wave, but for those of more than 32 with every degree to 3, which have one of their
// own: the second derivatives then keep two operands in LDS (16,384 rows of 64 channels: 160 us against 206, their
// gradients 74 against 82; with degrees to 2 98 against 96).
NormShape shape_of(int channels, int lmax, int64_t rows) {
  NormShape s;
  const bool shared = channels <= (lmax == 3 ? kNormWave / 2 : kNormWave);
  s.wide = shared ? 0 : channels <= most_threads(1) ? 1 : channels <= most_threads(2) ? 2 : 3;
  if (s.wide) {
    s.threads = (channels + kNormWave - 1) / kNormWave * kNormWave;
    s.groups = 1;
    s.block = s.threads;
  } else {
    s.threads = 1;
    while (s.threads < channels) s.threads *= 2;
    s.block = kNormThreads;
    s.groups = kNormThreads / s.threads;
  }
  s.grid = (rows + s.groups - 1) / s.groups;
  return s;
}

// Workgroups that leave partial weight gradients: more of them fill the chip, fewer leave less to add up.  Those of one
// wave are twice as many (second derivatives of 2,048 rows of 64 channels: 29 us against 33 with 1,024; gradients
// 21.4 against 20.9); second derivatives fit fewer large ones at a time (256 threads: 92 us with 512, 104 with 1,024).
int64_t partial_groups(const NormShape& s, int order) {
  int64_t most = kNormGroups;
  if (s.block == kNormWave) most *= 2;
  if (order == 2 && s.block >= kNormThreads) most /= 2;
  return s.grid < most ? s.grid : most;
}

using NormKernel = void (*)(NormArgs);

template <int L, int WIDE, bool BLOCK, bool NEXT>
NormKernel kernel_of(int order) {
  return order == 0   ? norm_forward_kernel<L, WIDE, BLOCK, NEXT>
         : order == 1 ? norm_backward_kernel<L, WIDE, BLOCK, NEXT>
                      : norm_second_kernel<L, WIDE, BLOCK, NEXT>;
}

template <int L, int WIDE>
NormKernel kernel_of(int order, bool block, bool next) {
  return !block ? kernel_of<L, WIDE, false, true>(order)
                : next ? kernel_of<L, WIDE, true, true>(order) : kernel_of<L, WIDE, true, false>(order);
}

template <int L>
NormKernel kernel_of(int order, int wide, bool block, bool next) {
  return wide == 0   ? kernel_of<L, 0>(order, block, next)
         : wide == 1 ? kernel_of<L, 1>(order, block, next)
         : wide == 2 ? kernel_of<L, 2>(order, block, next) : kernel_of<L, 3>(order, block, next);
}

bool valid(const ictc_norm_desc* d, int64_t rows) {
  return d && rows >= 0 && d->channels >= 1 && d->channels <= ICTC_NORM_MAX_CHANNELS && d->lmax >= 0 && d->lmax <= 3 &&
         d->input_lmax >= 0 && d->input_lmax <= 127 && d->eps > 0.f && rows <= (int64_t{1} << 40);
}

int run(int order, const ictc_norm_desc* d, NormArgs a, int64_t rows, bool block, bool next, float* dpost, float* dpre,
        hipStream_t stream) {
  const NormShape s = shape_of(d->channels, d->lmax, rows);
  a.rows = rows;
  a.channels = d->channels;
  a.width_x = static_cast<int64_t>(d->channels) * (d->input_lmax + 1) * (d->input_lmax + 1);
  a.input_lmax = d->input_lmax < d->lmax ? d->input_lmax : d->lmax;
  a.threads = s.threads;
  a.groups = s.groups;
  a.scale = d->residual_scale;
  a.eps = d->eps;
  const bool weights = dpost || dpre;
  if (!weights) a.partial = nullptr;
  const int64_t most = weights ? partial_groups(s, order) : (int64_t{1} << 31) / s.block;      // threads within 32 bits
  const int64_t grid = s.grid < most ? s.grid : most;
  const NormKernel kernel = d->lmax == 0   ? kernel_of<0>(order, s.wide, block, next)
                            : d->lmax == 1 ? kernel_of<1>(order, s.wide, block, next)
                            : d->lmax == 2 ? kernel_of<2>(order, s.wide, block, next)
                                           : kernel_of<3>(order, s.wide, block, next);
  if (grid) {
    const int columns = (d->lmax + 1) * (d->lmax + 1);
    const size_t lds = order == 2 && stashes(d->lmax, s.wide, block, next) ? 2 * sizeof(float) * columns * s.block : 0;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(s.block), lds, stream, a);
    if (hipGetLastError() != hipSuccess) return ICTC_ERR_LAUNCH;
  }
  if (weights) {
    const int columns = d->channels * (d->lmax + 1);
    hipLaunchKernelGGL(norm_weight_kernel, dim3((2 * columns + kColumns - 1) / kColumns), dim3(kColumns * kSlices), 0,
                       stream, a.partial, dpost, dpre, static_cast<int>(grid), columns);
    if (hipGetLastError() != hipSuccess) return ICTC_ERR_LAUNCH;
  }
  return ICTC_OK;
}

}  // namespace
}  // namespace ictc

extern "C" {

int64_t ictc_hip_norm_workspace(const ictc_norm_desc* desc, int64_t rows) {
  using namespace ictc;
  if (!valid(desc, rows)) return -ICTC_ERR_INVALID_ARGUMENT;
  const int64_t groups = partial_groups(shape_of(desc->channels, desc->lmax, rows), 1);
  return (groups ? groups : 1) * 2 * desc->channels * (desc->lmax + 1);
}

int ictc_hip_norm_forward(const ictc_norm_desc* desc, const float* x, const float* block, const float* gate,
                          const float* post, const float* pre, float* h, float* y, int64_t rows, hipStream_t stream) {
  using namespace ictc;
  if (!valid(desc, rows) || (!block && (gate || post || h || !pre || desc->input_lmax != desc->lmax)) ||
      (block && !post))
    return ICTC_ERR_INVALID_ARGUMENT;
  if (rows == 0) return ICTC_OK;
  if (!x || (block && !h) || (!pre != !y)) return ICTC_ERR_INVALID_ARGUMENT;
  NormArgs a = {};
  a.x = x, a.block = block, a.gate = gate, a.post = post, a.pre = pre, a.out_h = h, a.out_y = y;
  return run(0, desc, a, rows, block != nullptr, pre != nullptr, nullptr, nullptr, stream);
}

int ictc_hip_norm_backward(const ictc_norm_desc* desc, const float* h, const float* block, const float* gate,
                           const float* post, const float* pre, const float* grad_h, const float* grad_y, float* dx,
                           float* dblock, float* dgate, float* dpost, float* dpre, float* workspace,
                           int64_t workspace_floats, int64_t rows, hipStream_t stream) {
  using namespace ictc;
  if (!valid(desc, rows) ||
      (!block && (gate || post || grad_h || dblock || dpost || !pre || desc->input_lmax != desc->lmax)) ||
      (block && !post) || (dgate && !gate) || (dpre && !pre) || (!pre && grad_y))
    return ICTC_ERR_INVALID_ARGUMENT;
  if ((dpost || dpre) && (!workspace || workspace_floats < ictc_hip_norm_workspace(desc, rows)))
    return ICTC_ERR_INVALID_ARGUMENT;
  if (rows == 0 && !dpost && !dpre) return ICTC_OK;
  const bool next = pre && grad_y;
  if (rows && ((next && !h) || (!grad_y && !grad_h) || (!block && !grad_y))) return ICTC_ERR_INVALID_ARGUMENT;
  NormArgs a = {};
  a.h = h, a.block = block, a.gate = gate, a.post = post, a.pre = pre, a.dh = grad_h, a.dy = grad_y;
  a.dx = dx, a.db = dblock, a.dg = dgate, a.partial = workspace;
  return run(1, desc, a, rows, block != nullptr, next, dpost, dpre, stream);
}

int ictc_hip_norm_second(const ictc_norm_desc* desc, const float* h, const float* block, const float* gate,
                         const float* post, const float* pre, const float* grad_h, const float* grad_y,
                         const float* cot_x, const float* cot_block, const float* cot_gate, float* dx, float* dblock,
                         float* dgate, float* dgrad_h, float* dgrad_y, float* dpost, float* dpre, float* workspace,
                         int64_t workspace_floats, int64_t rows, hipStream_t stream) {
  using namespace ictc;
  const bool next = pre && grad_y;
  if (!valid(desc, rows) ||
      (!block && (gate || post || grad_h || cot_block || cot_gate || dblock || dgate || dgrad_h || dpost || !next ||
                  desc->input_lmax != desc->lmax)) ||
      (block && !post) || ((dgate || cot_gate) && !gate) || (dpre && !next) || ((dx || dgrad_y) && !next) ||
      (!pre && grad_y) || (!grad_y && !grad_h))
    return ICTC_ERR_INVALID_ARGUMENT;
  if ((dpost || dpre) && (!workspace || workspace_floats < ictc_hip_norm_workspace(desc, rows)))
    return ICTC_ERR_INVALID_ARGUMENT;
  if (rows == 0 && !dpost && !dpre) return ICTC_OK;
  if (rows && next && !h) return ICTC_ERR_INVALID_ARGUMENT;
  NormArgs a = {};
  a.h = h, a.block = block, a.gate = gate, a.post = post, a.pre = pre, a.dh = grad_h, a.dy = grad_y;
  a.cx = cot_x, a.cb = cot_block, a.cg = cot_gate;
  a.gx = dx, a.gb = dblock, a.gg = dgate, a.gdh = dgrad_h, a.gdy = dgrad_y, a.partial = workspace;
  return run(2, desc, a, rows, block != nullptr, next, dpost, dpre, stream);
}

}  // extern "C"
