// Root-mean-square norm with the residual's addition in front, an 8-bit
// output with a scale per row, and the gradients.
//
//   h = x + residual;  rstd = 1 / sqrt(mean(h^2) + epsilon);  y = gamma h rstd
//
// h is taken in float, before it is rounded for `sum`; sums of squares are
// float.  A row belongs to one wave or one workgroup, which keeps it in
// registers: one read of every input and one write of every output.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_util.h"
#include "tfma_internal.h"

namespace tfma {
namespace {

constexpr int kPack = 8;  // elements per lane and step
constexpr float kE4M3Max = 448.f;

template <typename S>
struct __attribute__((packed, aligned(1))) Pack {
  S v[kPack];
};

// kPack elements from column c of a row of n (global memory takes vector
// accesses at any alignment, so odd widths need no other path); zeros past
// the row.
template <class Tr>
__device__ inline void load_pack(const void* base, int64_t at, int c, int n, float (&out)[kPack]) {
  using S = typename Tr::S;
  const S* p = static_cast<const S*>(base) + at + c;
  if (c + kPack <= n) {
    const Pack<S> w = *reinterpret_cast<const Pack<S>*>(p);
#pragma unroll
    for (int j = 0; j < kPack; ++j) out[j] = Tr::ld(w.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kPack; ++j) out[j] = c + j < n ? Tr::ld(p[j]) : 0.f;
  }
}

template <class Tr>
__device__ inline void store_pack(void* base, int64_t at, int c, int n, const float (&in)[kPack]) {
  using S = typename Tr::S;
  S* p = static_cast<S*>(base) + at + c;
  if (c + kPack <= n) {
    Pack<S> w;
#pragma unroll
    for (int j = 0; j < kPack; ++j) w.v[j] = Tr::st(in[j]);
    *reinterpret_cast<Pack<S>*>(p) = w;
  } else {
#pragma unroll
    for (int j = 0; j < kPack; ++j)
      if (c + j < n) p[j] = Tr::st(in[j]);
  }
}

// Eight e4m3 values (round to nearest even; the inputs are within +-448).
__device__ inline void store_e4m3(void* base, int64_t at, int c, int n, const float (&in)[kPack]) {
  int w[2] = {0, 0};
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    w[q] = __builtin_amdgcn_cvt_pk_fp8_f32(in[4 * q], in[4 * q + 1], w[q], false);
    w[q] = __builtin_amdgcn_cvt_pk_fp8_f32(in[4 * q + 2], in[4 * q + 3], w[q], true);
  }
  uint8_t* p = static_cast<uint8_t*>(base) + at + c;
  Pack<uint8_t> b;
  __builtin_memcpy(&b, w, sizeof(b));
  if (c + kPack <= n) {
    *reinterpret_cast<Pack<uint8_t>*>(p) = b;
  } else {
#pragma unroll
    for (int j = 0; j < kPack; ++j)
      if (c + j < n) p[j] = b.v[j];
  }
}

// Squares are summed of values scaled by this power of two (about 1 / sqrt(n)):
// the sum overflows only where the mean does.
__device__ inline float square_scale(int n) { return ldexpf(1.f, -((32 - __clz(n)) / 2)); }
__device__ inline float rstd_of(float ss, float s, int n, float epsilon) {
  return 1.f / sqrtf(ss / (static_cast<float>(n) * s * s) + epsilon);
}

struct Sum {
  __device__ static float join(float a, float b) { return a + b; }
};
// Keeps a NaN, which a plain maximum drops.
struct Max {
  __device__ static float join(float a, float b) { return (a > b || a != a) ? a : b; }
};

// Joins v over the kThreads threads of a row; every thread gets the result.
// lds: one float per wave, free for reuse after the next barrier.
template <class J, int kThreads>
__device__ inline float join_row(float v, float* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = J::join(v, __shfl_xor(v, o));
  if constexpr (kThreads > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[wave] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) v = J::join(v, lds[w]);
  }
  return v;
}

// kThreads threads per row, which keep kPacks packs each: rows of up to
// kThreads * kPacks * 8 elements.  Rows of one wave sit four to a workgroup.
// Bound by HBM: 16384 x 2048 bf16 with the residual's addition 46.7 us, 5.75
// TB/s of compulsory bytes (a copy reaches 6.07); few rows by the launch (8 x
// 2048 3.7 us).  y is computed from the unrounded h and rounded once, by its
// store; in 8 bits it is divided by its row's scale in float first.
template <class Tr, int kThreads, int kPacks>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads) void norm_kernel(RmsNormArgs a) {
  __shared__ float lds[kThreads / 64];
  constexpr int kRows = kThreads < 256 ? 256 / kThreads : 1;
  const int64_t row = group_of_many(a.across) * kRows + threadIdx.x / kThreads;
  if (row >= a.rows) return;  // whole waves, and whole workgroups of one row
  const int tid = threadIdx.x % kThreads;
  const int n = static_cast<int>(a.c);
  const int64_t at = row * a.c;
  float h[kPacks][kPack];
  const float sc = square_scale(n);
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    const int c = (i * kThreads + tid) * kPack;
    load_pack<Tr>(a.x, at, c, n, h[i]);
  }
  if (a.residual) {
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      const int c = (i * kThreads + tid) * kPack;
      float r[kPack];
      load_pack<Tr>(a.residual, at, c, n, r);
#pragma unroll
      for (int j = 0; j < kPack; ++j) h[i][j] += r[j];
      store_pack<Tr>(a.sum, at, c, n, h[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kPacks; ++i)
#pragma unroll
    for (int j = 0; j < kPack; ++j) ss = fmaf(h[i][j] * sc, h[i][j] * sc, ss);
  ss = join_row<Sum, kThreads>(ss, lds);
  const float rstd = rstd_of(ss, sc, n, a.epsilon);
  if (a.rstd && tid == 0) a.rstd[row] = rstd;
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    const int c = (i * kThreads + tid) * kPack;
    float g[kPack];
    load_pack<TF32>(a.gamma, 0, c, n, g);
#pragma unroll
    for (int j = 0; j < kPack; ++j) {
      h[i][j] = h[i][j] * rstd * g[j];
      if (a.scale) top = Max::join(fabsf(h[i][j]), top);
    }
    if (!a.scale) store_pack<Tr>(a.y, at, c, n, h[i]);
  }
  if (!a.scale) return;
  top = join_row<Max, kThreads>(top, lds);
  const float scale = top / kE4M3Max;
  if (tid == 0) a.scale[row] = scale;
#pragma unroll
  for (int i = 0; i < kPacks; ++i) {
    const int c = (i * kThreads + tid) * kPack;
    float q[kPack];
#pragma unroll
    for (int j = 0; j < kPack; ++j) {
      // A row of zeros has scale 0 and zeros in it; the quotient may pass
      // the largest value by the division's rounding.
      const float v = scale == 0.f ? 0.f : h[i][j] / scale;
      q[j] = v > kE4M3Max ? kE4M3Max : (v < -kE4M3Max ? -kE4M3Max : v);
    }
    store_e4m3(a.y, at, c, n, q);
  }
}

// Rows of any length: the row is read again for each use.
template <class Tr>
__global__ __launch_bounds__(1024) void norm_long_kernel(RmsNormArgs a) {
  constexpr int kThreads = 1024;
  __shared__ float lds[kThreads / 64];
  const int64_t row = group_of_many(a.across);
  if (row >= a.rows) return;
  const int64_t at = row * a.c;
  const int n = static_cast<int>(a.c);
  const int tid = threadIdx.x;
  auto load_h = [&](int c, float (&h)[kPack]) {
    load_pack<Tr>(a.x, at, c, n, h);
    if (a.residual) {
      float r[kPack];
      load_pack<Tr>(a.residual, at, c, n, r);
#pragma unroll
      for (int j = 0; j < kPack; ++j) h[j] += r[j];
    }
  };
  const float sc = square_scale(n);
  float ss = 0.f;
  for (int c = tid * kPack; c < n; c += kThreads * kPack) {
    float h[kPack];
    load_h(c, h);
#pragma unroll
    for (int j = 0; j < kPack; ++j) ss = fmaf(h[j] * sc, h[j] * sc, ss);
  }
  ss = join_row<Sum, kThreads>(ss, lds);
  const float rstd = rstd_of(ss, sc, n, a.epsilon);
  if (a.rstd && tid == 0) a.rstd[row] = rstd;
  float scale = 0.f;
  if (a.scale) {
    float top = 0.f;
    for (int c = tid * kPack; c < n; c += kThreads * kPack) {
      float h[kPack], g[kPack];
      load_h(c, h);
      load_pack<TF32>(a.gamma, 0, c, n, g);
#pragma unroll
      for (int j = 0; j < kPack; ++j) top = Max::join(fabsf(h[j] * rstd * g[j]), top);
    }
    top = join_row<Max, kThreads>(top, lds);
    scale = top / kE4M3Max;
    if (tid == 0) a.scale[row] = scale;
  }
  // `sum` and `y` may be the inputs' own memory: nothing is read here that
  // this thread has not read before it writes.
  for (int c = tid * kPack; c < n; c += kThreads * kPack) {
    float h[kPack], g[kPack];
    load_h(c, h);
    load_pack<TF32>(a.gamma, 0, c, n, g);
    if (a.residual) store_pack<Tr>(a.sum, at, c, n, h);
#pragma unroll
    for (int j = 0; j < kPack; ++j) {
      h[j] = h[j] * rstd * g[j];
      if (a.scale) {
        const float v = scale == 0.f ? 0.f : h[j] / scale;
        h[j] = v > kE4M3Max ? kE4M3Max : (v < -kE4M3Max ? -kE4M3Max : v);
      }
    }
    if (a.scale)
      store_e4m3(a.y, at, c, n, h);
    else
      store_pack<Tr>(a.y, at, c, n, h);
  }
}

template <class Tr, int kThreads, int kPacks>
hipError_t launch_norm(RmsNormArgs a, hipStream_t stream) {
  constexpr int kRows = kThreads < 256 ? 256 / kThreads : 1;
  const int64_t groups = (a.rows + kRows - 1) / kRows;
  if (groups > kMostGroups) return hipErrorInvalidConfiguration;
  const dim3 grid = many_groups(groups);
  a.across = grid.x;
  TFMA_LAUNCH("tfma_rms_norm", (norm_kernel<Tr, kThreads, kPacks>), grid, dim3(kRows * kThreads), 0,
              stream, a);
  return hipGetLastError();
}

// One pack a thread as far as a workgroup goes: more waves, each with less to
// wait for (16384 x 2048 bf16 47.5 us; one wave of four packs a row 55.4; 4096 x
// 8192 48.7 against 53.4 for 256 threads of four).  Rows of up to 1024 take one
// wave and no barrier (30000 x 1000 bf16 48.8 us against 63.2 for 256 threads).
template <class Tr>
hipError_t norm_by_width(RmsNormArgs a, hipStream_t stream) {
  if (a.c <= 64 * 8) return launch_norm<Tr, 64, 1>(a, stream);
  if (a.c <= 64 * 16) return launch_norm<Tr, 64, 2>(a, stream);
  if (a.c <= 256 * 8) return launch_norm<Tr, 256, 1>(a, stream);
  if (a.c <= 512 * 8) return launch_norm<Tr, 512, 1>(a, stream);
  if (a.c <= 1024 * 8) return launch_norm<Tr, 1024, 1>(a, stream);
  if (a.c <= 1024 * 16) return launch_norm<Tr, 1024, 2>(a, stream);
  if (a.rows > kMostGroups) return hipErrorInvalidConfiguration;
  const dim3 grid = many_groups(a.rows);
  a.across = grid.x;
  TFMA_LAUNCH("tfma_rms_norm_long", norm_long_kernel<Tr>, grid, dim3(1024), 0, stream, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Gradients.  With xhat = h rstd and g = gamma dy,
//   dh = rstd (g - xhat mean(g xhat)) + dsum;  dgamma = sum over rows dy xhat.
// A workgroup takes a run of rows; each thread keeps the gamma gradients of
// its own columns and leaves them in `partial` [workgroups, c], which a
// second kernel adds in order.
// ---------------------------------------------------------------------------

// A pack as it is stored: the row's values wait for the row's sum in half the
// registers that floats would take.
template <class Tr>
__device__ inline void load_raw(const void* base, int64_t at, int c, int n,
                                Pack<typename Tr::S>& out) {
  using S = typename Tr::S;
  const S* p = static_cast<const S*>(base) + at + c;
  if (c + kPack <= n) {
    out = *reinterpret_cast<const Pack<S>*>(p);
  } else {
#pragma unroll
    for (int j = 0; j < kPack; ++j) out.v[j] = c + j < n ? p[j] : S(0);
  }
}

// Registers hold the row: kThreads threads with kPacks packs each; rows of
// one wave run four to a workgroup, which joins its four sums of gamma's
// gradient in LDS.
// Bound by HBM: 16384 x 2048 bf16 with a gradient of the sum 60.8 us over
// operands that come from memory (4.4 TB/s of compulsory bytes; 4.8 us of
// it are the second kernel), 48.2 where the caches hold part of them.
template <class Tr, int kThreads, int kPacks>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads) void norm_grad_kernel(
    RmsNormGradArgs a, int64_t rows_per) {
  using S = typename Tr::S;
  constexpr int kRows = kThreads < 256 ? 256 / kThreads : 1;
  constexpr int kWidth = kThreads * kPacks * kPack;
  __shared__ float lds[kThreads / 64];
  __shared__ float join[kRows > 1 ? kWidth : 1];
  const int slot = threadIdx.x / kThreads, tid = threadIdx.x % kThreads;
  const int n = static_cast<int>(a.c);
  const int64_t r0 = int64_t(blockIdx.x) * rows_per;
  const int64_t r1 = r0 + rows_per < a.rows ? r0 + rows_per : a.rows;
  float g[kPacks][kPack], acc[kPacks][kPack] = {};
#pragma unroll
  for (int i = 0; i < kPacks; ++i) load_pack<TF32>(a.gamma, 0, (i * kThreads + tid) * kPack, n, g[i]);
  for (int64_t row = r0 + slot; row < r1; row += kRows) {
    const int64_t at = row * a.c;
    Pack<S> dy[kPacks], h[kPacks], ds[kPacks] = {};
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      const int c = (i * kThreads + tid) * kPack;
      load_raw<Tr>(a.dy, at, c, n, dy[i]);
      load_raw<Tr>(a.h, at, c, n, h[i]);
    }
    if (a.dsum) {
#pragma unroll
      for (int i = 0; i < kPacks; ++i) load_raw<Tr>(a.dsum, at, (i * kThreads + tid) * kPack, n, ds[i]);
    }
    const float rstd = a.rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < kPacks; ++i)
#pragma unroll
      for (int j = 0; j < kPack; ++j)
        dot = fmaf(Tr::ld(dy[i].v[j]) * g[i][j], Tr::ld(h[i].v[j]) * rstd, dot);
    dot = join_row<Sum, kThreads>(dot, lds) / static_cast<float>(n);
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      float d[kPack];
#pragma unroll
      for (int j = 0; j < kPack; ++j) {
        const float xhat = Tr::ld(h[i].v[j]) * rstd, t = Tr::ld(dy[i].v[j]);
        d[j] = fmaf(rstd, fmaf(-xhat, dot, t * g[i][j]), Tr::ld(ds[i].v[j]));
        acc[i][j] = fmaf(t, xhat, acc[i][j]);
      }
      store_pack<Tr>(a.dx, at, (i * kThreads + tid) * kPack, n, d);
    }
  }
  float* partial = a.partial + int64_t(blockIdx.x) * a.c;
  if constexpr (kRows > 1) {
    for (int w = 0; w < kRows; ++w) {
      if (slot == w) {
#pragma unroll
        for (int i = 0; i < kPacks; ++i)
#pragma unroll
          for (int j = 0; j < kPack; ++j) {
            float* q = join + (i * kThreads + tid) * kPack + j;
            *q = w == 0 ? acc[i][j] : *q + acc[i][j];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < n; c += kRows * kThreads) partial[c] = join[c];
  } else {
#pragma unroll
    for (int i = 0; i < kPacks; ++i)
      store_pack<TF32>(partial, 0, (i * kThreads + tid) * kPack, n, acc[i]);
  }
}

// Rows of any length: the row is read twice and the sums are kept in
// `partial` itself.
template <class Tr>
__global__ __launch_bounds__(1024) void norm_grad_long_kernel(RmsNormGradArgs a, int64_t rows_per) {
  constexpr int kThreads = 1024;
  __shared__ float lds[kThreads / 64];
  const int tid = threadIdx.x;
  const int n = static_cast<int>(a.c);
  const int64_t r0 = int64_t(blockIdx.x) * rows_per;
  const int64_t r1 = r0 + rows_per < a.rows ? r0 + rows_per : a.rows;
  float* partial = a.partial + int64_t(blockIdx.x) * a.c;
  for (int64_t row = r0; row < r1; ++row) {
    const int64_t at = row * a.c;
    const float rstd = a.rstd[row];
    float dot = 0.f;
    for (int c = tid * kPack; c < n; c += kThreads * kPack) {
      float dy[kPack], h[kPack], g[kPack];
      load_pack<Tr>(a.dy, at, c, n, dy);
      load_pack<Tr>(a.h, at, c, n, h);
      load_pack<TF32>(a.gamma, 0, c, n, g);
#pragma unroll
      for (int j = 0; j < kPack; ++j) dot = fmaf(dy[j] * g[j], h[j] * rstd, dot);
    }
    dot = join_row<Sum, kThreads>(dot, lds) / static_cast<float>(n);
    for (int c = tid * kPack; c < n; c += kThreads * kPack) {
      float dy[kPack], h[kPack], g[kPack], d[kPack] = {}, p[kPack] = {};
      load_pack<Tr>(a.dy, at, c, n, dy);
      load_pack<Tr>(a.h, at, c, n, h);
      load_pack<TF32>(a.gamma, 0, c, n, g);
      if (a.dsum) load_pack<Tr>(a.dsum, at, c, n, d);
      if (row > r0) load_pack<TF32>(partial, 0, c, n, p);
#pragma unroll
      for (int j = 0; j < kPack; ++j) {
        const float xhat = h[j] * rstd;
        d[j] = fmaf(rstd, fmaf(-xhat, dot, dy[j] * g[j]), d[j]);
        p[j] = fmaf(dy[j], xhat, p[j]);
      }
      store_pack<Tr>(a.dx, at, c, n, d);
      store_pack<TF32>(partial, 0, c, n, p);
    }
  }
}

// Sums `partial` over its groups: a workgroup has 64 columns, its sixteen
// waves take groups in turn.
__global__ __launch_bounds__(1024) void gamma_sums_kernel(uint32_t across, int64_t groups, int64_t c,
                                                          const float* partial, float* out) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i = group_of_many(across) * 64 + lane;
  float s = 0.f;
  if (i < c) {
#pragma unroll 8
    for (int64_t g = wave; g < groups; g += 16) s += partial[g * c + i];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || i >= c) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += sums[w][lane];
  out[i] = s;
}

// Workgroups of the gradient: two per CU, four rows at a time for rows of
// one wave.  Up to sixteen such rows stay with one workgroup, whose sums are
// the result: no second launch.
int64_t grad_groups(int64_t rows, int64_t c) {
  const int64_t at_once = c <= 64 * 32 ? 4 : 1;
  if (rows > 0 && rows <= 4 * at_once) return 1;
  const int64_t want = (rows + at_once - 1) / at_once;
  return want < 512 ? want : 512;
}

template <class Tr, int kThreads, int kPacks>
hipError_t launch_norm_grad(const RmsNormGradArgs& a, int64_t groups, int64_t rows_per,
                            hipStream_t stream) {
  TFMA_LAUNCH("tfma_rms_norm_grad", (norm_grad_kernel<Tr, kThreads, kPacks>),
              dim3(static_cast<uint32_t>(groups)), dim3(kThreads < 256 ? 256 : kThreads), 0, stream,
              a, rows_per);
  return hipGetLastError();
}

// One wave a row as far as its registers go, which leaves no barrier between a
// row's loads and its sums (16384 x 2048 bf16 48.2 us, with 256 threads a row
// 54.7; 30000 x 1000 57.2 and 134); past that 256 threads (8192 x 4096 bf16
// 49.0 us, one wave 58.8; 4096 x 8192 50.7, with 1024 threads 51.6).
template <class Tr>
hipError_t norm_grad_by_width(const RmsNormGradArgs& a, int64_t groups, int64_t rows_per,
                              hipStream_t stream) {
  if (a.c <= 64 * 8) return launch_norm_grad<Tr, 64, 1>(a, groups, rows_per, stream);
  if (a.c <= 64 * 16) return launch_norm_grad<Tr, 64, 2>(a, groups, rows_per, stream);
  if (a.c <= 64 * 32) return launch_norm_grad<Tr, 64, 4>(a, groups, rows_per, stream);
  if (a.c <= 256 * 16) return launch_norm_grad<Tr, 256, 2>(a, groups, rows_per, stream);
  if (a.c <= 256 * 32) return launch_norm_grad<Tr, 256, 4>(a, groups, rows_per, stream);
  if (a.c <= 1024 * 16) return launch_norm_grad<Tr, 1024, 2>(a, groups, rows_per, stream);
  TFMA_LAUNCH("tfma_rms_norm_grad_long", norm_grad_long_kernel<Tr>,
              dim3(static_cast<uint32_t>(groups)), dim3(1024), 0, stream, a, rows_per);
  return hipGetLastError();
}

template <class Tr>
hipError_t norm_grad(const RmsNormGradArgs& a, hipStream_t stream) {
  int64_t groups = grad_groups(a.rows, a.c);
  if (groups > 0) {
    const int64_t rows_per = (a.rows + groups - 1) / groups;
    groups = (a.rows + rows_per - 1) / rows_per;
    RmsNormGradArgs b = a;
    if (groups == 1) b.partial = a.dgamma;
    const hipError_t e = norm_grad_by_width<Tr>(b, groups, rows_per, stream);
    if (e != hipSuccess || groups == 1) return e;
  }
  const dim3 grid = many_groups((a.c + 63) / 64);
  TFMA_LAUNCH("tfma_rms_norm_dgamma", gamma_sums_kernel, grid, dim3(1024), 0, stream, grid.x, groups,
              a.c, a.partial, a.dgamma);
  return hipGetLastError();
}

}  // namespace

hipError_t LaunchRmsNorm(DType t, const RmsNormArgs& a, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  switch (t) {
    case DType::kF32: return norm_by_width<TF32>(a, stream);
    case DType::kF16: return norm_by_width<TF16>(a, stream);
    default: return norm_by_width<TBF16>(a, stream);
  }
}

size_t RmsNormGradWorkspaceBytes(int64_t rows, int64_t c) {
  const int64_t groups = grad_groups(rows, c);
  return groups <= 1 ? 0 : static_cast<size_t>(groups) * static_cast<size_t>(c) * sizeof(float);
}

hipError_t LaunchRmsNormGrad(DType t, const RmsNormGradArgs& a, hipStream_t stream) {
  switch (t) {
    case DType::kF32: return norm_grad<TF32>(a, stream);
    case DType::kF16: return norm_grad<TF16>(a, stream);
    default: return norm_grad<TBF16>(a, stream);
  }
}

}  // namespace tfma
