// Distillation from a teacher's top logits, with the gradient of the
// student's logits.
//
//   p = softmax(teacher / T) over the row's entries, q = softmax(logits / T)
//   loss = w T^2 sum_j p_j (log p_j - log q[id_j])
//        = w T sum_j p_j (t_j - t* - (s[id_j] - s*) - T (ln S_t - ln S_s))
//   dloss / dlogits_i = w T (q_i - sum of the p_j with id_j = i)
//
// where * is a row's largest logit and S its sum of exp((logit - *) / T).  The
// second form is the one computed: the largest logit is subtracted first, so
// that no term is as large as the logits are, whose common offset would cost
// the loss its digits and whose finite masks (the type's lowest value) would
// overflow when they are scaled.
//
// An entry whose id is outside [0, v) or whose logit is -inf is absent; a row
// without entries has loss 0 and gradient 0.  One read of the logits and one
// write of the gradient: a workgroup keeps its row in registers between the
// maximum, the sum and the gradient.  Softmax statistics are float; the
// gradient is rounded once, by its store.
#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "device_util.h"
#include "tfma_internal.h"

namespace tfma {
namespace {

constexpr int kPack = 8;
constexpr float kLog2E = 1.4426950408889634f;

template <typename S>
struct __attribute__((packed, aligned(1))) Pack {
  S v[kPack];
};
// A pack in whole registers.
template <typename S>
struct Words {
  uint32_t w[kPack * sizeof(S) / 4];
};
template <typename S>
__device__ inline Words<S> load_words(const S* p) {
  const Pack<S> t = *reinterpret_cast<const Pack<S>*>(p);
  Words<S> w;
  __builtin_memcpy(&w, &t, sizeof(w));
  return w;
}
template <class Tr>
__device__ inline float element(const Words<typename Tr::S>& p, int j) {
  using S = typename Tr::S;
  if constexpr (sizeof(S) == 4) return __builtin_bit_cast(float, p.w[j]);
  return Tr::ld(static_cast<S>(j % 2 ? p.w[j / 2] >> 16 : p.w[j / 2] & 0xffffu));
}

// Joins over the workgroup; every thread gets the result.  lds: one float per
// wave.
template <int kThreads>
__device__ inline float max_block(float v, float* lds) {
  // A maximum that keeps NaN is not needed: a NaN comes back in the sum.
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) v = fmaxf(v, lds[w]);
  return v;
}

template <int kThreads>
__device__ inline float sum_block(float v, float* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) v += lds[w];
  return v;
}

// The teacher's side of a row in LDS: for each entry its id (-1: absent), its
// logit less the row's largest, and its probability.
struct Entries {
  int32_t* id;
  float* below;
  float* p;
};

// The factor of an exponent, finite for the smallest temperatures too (the
// largest logit's exponent is 0 times it).
__device__ inline float per_temperature(float c, float temperature) {
  return fminf(c / temperature, FLT_MAX);
}

// Fills `e` and `log_sum`, the logarithm of the entries' sum of exponentials,
// and returns whether the row has an entry.
template <class Tr, int kThreads>
__device__ inline bool load_entries(const DistillArgs& a, int64_t row, const Entries& e, float* lds,
                                    float& log_sum) {
  const float inv_t = per_temperature(1.f, a.temperature);
  float top = -INFINITY;
  bool nan = false;
  for (int j = threadIdx.x; j < a.k; j += kThreads) {
    const int64_t at = row * a.k + j;
    const int64_t i = a.ids64 ? static_cast<const int64_t*>(a.ids)[at]
                              : static_cast<const int32_t*>(a.ids)[at];
    float t = -INFINITY;
    if (i >= 0 && i < a.v)
      t = a.teacher_f32 ? static_cast<const float*>(a.teacher)[at]
                        : Tr::ld(static_cast<const typename Tr::S*>(a.teacher)[at]);
    e.id[j] = t != -INFINITY ? static_cast<int32_t>(i) : -1;
    e.below[j] = t;
    nan |= t != t;
    top = fmaxf(top, t);
  }
  top = max_block<kThreads>(nan ? INFINITY : top, lds);  // inf - inf is NaN again
  float sum = 0.f;
  for (int j = threadIdx.x; j < a.k; j += kThreads) {
    const float below = e.below[j] - top;
    const float p = e.id[j] >= 0 ? expf(below * inv_t) : 0.f;
    e.below[j] = below;
    e.p[j] = p;
    sum += p;
  }
  sum = sum_block<kThreads>(sum, lds);
  log_sum = logf(sum);
  for (int j = threadIdx.x; j < a.k; j += kThreads) e.p[j] /= sum;
  return top != -INFINITY;  // this thread's own entries are read next, or after a barrier
}

// T times the sum over the entries of p (log p - log q); x: the row's logits,
// top the largest of them, log_ratio the entries' logarithm less the logits'.
template <class Tr, int kThreads>
__device__ inline float divergence(const DistillArgs& a, const typename Tr::S* x, const Entries& e,
                                   float top, float log_ratio, float* lds) {
  const float shift = a.temperature * log_ratio;
  float term = 0.f;
  for (int j = threadIdx.x; j < a.k; j += kThreads)
    if (e.id[j] >= 0 && e.p[j] != 0.f)
      term += e.p[j] * (e.below[j] - (Tr::ld(x[e.id[j]]) - top) - shift);
  return sum_block<kThreads>(term, lds);
}

// exp((x - top) / T) with c = log2(e) / T: exactly 1 for the largest.  A row
// whose maximum is -inf gives NaN.
__device__ inline float soft(float x, float c, float top) {
  return __builtin_amdgcn_exp2f((x - top) * c);
}

// The gradient at the entries' places, over the q that the workgroup has
// stored there: equal ids take the sum of their p, in order, at the first of
// them.  `own` holds the entries' q.
template <class Tr, int kThreads>
__device__ inline void place_entries(const DistillArgs& a, typename Tr::S* back, const Entries& e,
                                     const float* own, float factor) {
  for (int j = threadIdx.x; j < a.k; j += kThreads) {
    const int32_t id = e.id[j];
    if (id < 0) continue;
    float mass = 0.f;
    bool first = true;
    for (int i = 0; i < a.k; ++i) {
      if (e.id[i] != id) continue;
      first &= i >= j;
      mass += e.p[i];
    }
    if (first) back[id] = Tr::st(factor * (own[j] - mass));
  }
}

// One row per workgroup.  kPacks packs of the row wait in registers as they
// are stored (rows of up to kThreads * kPacks * 8); kPacks = 0: the row is
// read again for each use.  The up to seven elements after the last whole pack
// belong to the first threads, one each.
// Bound by HBM where there are rows enough (4096 x 50304 bf16 with its gradient
// 184 us, 4.5 TB/s of compulsory bytes; each workgroup reads, then computes
// two exponentials an element, then writes, so that reads and writes overlap
// only between the rows that share a CU), else by one row's latency (61 x 50303
// f32 without the gradient 8.3 us).
template <class Tr, int kThreads, int kPacks>
__global__ __launch_bounds__(kThreads) void distill_kernel(DistillArgs a) {
  using S = typename Tr::S;
  __shared__ float lds[kThreads / 64];
  extern __shared__ float dyn[];
  const Entries e = {reinterpret_cast<int32_t*>(dyn), dyn + a.k, dyn + 2 * a.k};
  float* own = dyn + 3 * a.k;
  const int tid = threadIdx.x;
  const int64_t row = group_of_many(a.across);
  if (row >= a.rows) return;
  const S* x = static_cast<const S*>(a.logits) + row * a.v;
  const int v = static_cast<int>(a.v), whole = v & ~(kPack - 1);
  constexpr int kHeld = kPacks > 0 ? kPacks : 1;
  // The row's loads are on their way while the teacher's entries are read.
  Words<S> held[kHeld];
  if constexpr (kPacks > 0) {
    const uint32_t hidden = sizeof(S) == 4 ? 0xff800000u : 0x10001u * static_cast<uint16_t>(Tr::st(-INFINITY));
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
      const int c = (i * kThreads + tid) * kPack;
#pragma unroll
      for (uint32_t& w : held[i].w) w = hidden;
      if (c < whole) held[i] = load_words<S>(x + c);
    }
  }
  float rest = whole + tid < v ? Tr::ld(x[whole + tid]) : -INFINITY;
  auto each = [&](auto&& f) {
    if constexpr (kPacks > 0) {
#pragma unroll
      for (int i = 0; i < kPacks; ++i) {
        f((i * kThreads + tid) * kPack, held[i]);
        // Else the floats of one use would be kept for the next.
#pragma unroll
        for (uint32_t& w : held[i].w) asm volatile("" : "+v"(w));
      }
    } else {
#pragma unroll 4
      for (int c = tid * kPack; c < whole; c += kThreads * kPack) {
        Words<S> w = load_words<S>(x + c);
        f(c, w);
      }
    }
  };
  float log_entries;
  const bool some = load_entries<Tr, kThreads>(a, row, e, lds, log_entries);
  S* back = a.backprop ? static_cast<S*>(a.backprop) + row * a.v : nullptr;
  if (!some) {
    if (tid == 0) a.loss[row] = 0.f;
    if (back)
      for (int i = tid; i < v; i += kThreads) back[i] = Tr::st(0.f);
    return;
  }
  float top = rest;
  each([&](int, const Words<S>& w) {
#pragma unroll
    for (int j = 0; j < kPack; ++j) top = fmaxf(top, element<Tr>(w, j));
  });
  top = max_block<kThreads>(top, lds);
  const float c2 = per_temperature(kLog2E, a.temperature);
  float sum = soft(rest, c2, top);
  // Float rows in registers keep their exponentials in place of the logits, which
  // the gradient then only scales (2000 x 50304 f32 182 us, 198 with them computed
  // again).
  constexpr bool kKeep = kPacks > 0 && sizeof(S) == 4;
  each([&](int, Words<S>& w) {
#pragma unroll
    for (int j = 0; j < kPack; ++j) {
      const float q = soft(element<Tr>(w, j), c2, top);
      sum += q;
      if constexpr (kKeep) w.w[j] = f32_bits(q);
    }
  });
  sum = sum_block<kThreads>(sum, lds);
  const float weight = a.weights ? a.weights[row] : 1.f;
  const float kl = divergence<Tr, kThreads>(a, x, e, top, log_entries - logf(sum), lds);
  if (tid == 0) a.loss[row] = weight * a.temperature * kl;
  if (!back) return;

  // The gradient may take the logits' own memory: what the entries need of
  // them is read before the first store.
  const float inv_sum = 1.f / sum, factor = weight * a.temperature;
  for (int j = tid; j < a.k; j += kThreads)
    own[j] = e.id[j] >= 0 ? soft(Tr::ld(x[e.id[j]]), c2, top) * inv_sum : 0.f;
  __syncthreads();
  const float scale = factor * inv_sum;
  each([&](int c, const Words<S>& w) {
    if (c >= whole) return;
    Pack<S> o;
#pragma unroll
    for (int j = 0; j < kPack; ++j) {
      const float q = element<Tr>(w, j);
      o.v[j] = Tr::st(scale * (kKeep ? q : soft(q, c2, top)));
    }
    *reinterpret_cast<Pack<S>*>(back + c) = o;
  });
  if (whole + tid < v) back[whole + tid] = Tr::st(scale * soft(rest, c2, top));
  __syncthreads();  // the stores above come before those below
  place_entries<Tr, kThreads>(a, back, e, own, factor);
}

template <class Tr, int kThreads, int kPacks>
hipError_t launch(DistillArgs a, hipStream_t stream) {
  if (a.rows > kMostGroups) return hipErrorInvalidConfiguration;
  const dim3 grid = many_groups(a.rows);
  a.across = grid.x;
  TFMA_LAUNCH("tfma_distill", (distill_kernel<Tr, kThreads, kPacks>), grid, dim3(kThreads),
              4 * a.k * sizeof(float), stream, a);
  return hipGetLastError();
}

template <class Tr>
hipError_t by_width(const DistillArgs& a, hipStream_t stream) {
  constexpr int kStep = kPack * 256;
  // Few threads with many packs, so that several rows share a CU, some of which
  // load while others store.  Short rows take one wave each.  With the gradient,
  // us (in brackets the neighbour's): 16000 x 2000 bf16 54 (256 threads 73);
  // 8000 x 4000 bf16 46.7 (one wave 51.4); 4000 x 8000 bf16 42.5 (512 threads
  // 46.4), f32 70 (128 threads 74).
  if (a.v <= kStep) return launch<Tr, 64, 4>(a, stream);
  if (a.v <= 2 * kStep) return launch<Tr, 128, 4>(a, stream);
  if (a.v <= 4 * kStep) return launch<Tr, 256, 4>(a, stream);
  if constexpr (sizeof(typename Tr::S) == 2) {
    // 2000 x 16000 bf16 37.4 (512 threads 40.2), 1000 x 32000 34.1 (512 threads
    // 38.6), 4096 x 50304 183 (512 threads 198, 1024 304).
    if (a.v <= 8 * kStep) return launch<Tr, 256, 8>(a, stream);
    if (a.v <= 16 * kStep) return launch<Tr, 256, 16>(a, stream);
    if (a.v <= 28 * kStep) return launch<Tr, 256, 28>(a, stream);
  } else {
    // 2000 x 16000 f32 64.9 (256 threads 67.0), 1000 x 32000 63.0 (1024 threads
    // 71.8), 2000 x 50304 184 (512 threads 184).
    if (a.v <= 8 * kStep) return launch<Tr, 512, 4>(a, stream);
    if (a.v <= 16 * kStep) return launch<Tr, 512, 8>(a, stream);
    if (a.v <= 28 * kStep) return launch<Tr, 1024, 7>(a, stream);
  }
  return launch<Tr, 1024, 0>(a, stream);
}

}  // namespace

hipError_t LaunchDistill(DType t, const DistillArgs& a, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  switch (t) {
    case DType::kF32: return by_width<TF32>(a, stream);
    case DType::kF16: return by_width<TF16>(a, stream);
    default: return by_width<TBF16>(a, stream);
  }
}

}  // namespace tfma
