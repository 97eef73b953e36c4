// Matrix product with bias, activation and residual in its epilogue, and the
// products of its gradient, on the matrix cores (MFMA).
//
//   C[m, n] = act(sum_k A[m, k] B[k, n] * row_scale[m] * col_scale[n] + bias[n]) + residual[m, n]
//
// Each operand is stored either with k contiguous (A [M, K], B [N, K]) or
// with k as the row (A [K, M], B [K, N]): the forward product of TensorFlow's
// [K, N] weights reads B by rows of k, the gradient of the weights both.  A
// tile keeps its operand's own order in LDS; 16-bit tiles whose rows are k
// are transposed on their way to the registers (ds_read_b64_tr_b16).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_util.h"
#include "tfma_internal.h"

namespace tfma {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// 16 bytes at any address that holds whole elements (global memory takes
// vector accesses at any alignment).
struct __attribute__((packed, aligned(1))) Bytes16 {
  uint32_t w[4];
};

// Operand types.  A step of the product takes 128 bytes of k, in kParts parts;
// a wave's fragment of 16 rows of a part is one Frag per lane: lane l holds
// row l % 16 and, of part h, the k of the 16-byte chunk 4 h + l / 16 (e4m3:
// those of chunks l / 16 and 4 + l / 16).  Which k a matrix instruction calls
// which does not matter as long as both operands agree.
struct OpF16 {
  using S = uint16_t;
  using Frag = i32x4;
  static constexpr int kParts = 2;
  __device__ static void mma(const Frag& a, const Frag& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                               __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
struct OpBF16 {
  using S = uint16_t;
  using Frag = i32x4;
  static constexpr int kParts = 2;
  __device__ static void mma(const Frag& a, const Frag& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
struct OpF32 {
  using S = float;
  using Frag = i32x4;
  static constexpr int kParts = 2;
  __device__ static void mma(const Frag& a, const Frag& b, f32x4& c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
  }
};
// e4m3.  The matrix unit adds 8-bit products with fewer bits than a float has
// (measured: sums are off by up to 2^-13 of their largest product, with this
// instruction and with the narrower one of half its rate), so the results are
// half or bfloat16, whose own rounding is coarser.
struct OpFP8 {
  using S = uint8_t;
  using Frag = i32x8;
  static constexpr int kParts = 1;
  __device__ static void mma(const Frag& a, const Frag& b, f32x4& c) {
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
  }
};

constexpr int kRowBytes = 128;  // k bytes of a step

// ---------------------------------------------------------------------------
// Activations and their derivatives.
// ---------------------------------------------------------------------------
constexpr float kSqrt2OverPi = 0.7978845608028654f;

// 1 / (1 + e^-x).  For results of 16 bits through 2^y, whose argument's
// rounding grows with |x| to 30 units in float's last place where the result
// is still a normal number; for float results with the exact exponential.
template <bool kExact>
__device__ inline float sigmoid(float x) {
  if constexpr (kExact) return 1.f / (1.f + expf(-x));
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
}

// The normal distribution at z; e: exp(-z^2 / 2).  For results of 16 bits the
// tail beyond |z| is e times a polynomial in 1 / (1 + 0.32 |z|) without a
// constant term, fitted here to the scaled complementary error function for
// the least relative error (4.4e-7 over all z, next to 4.9e-4 of half's own
// rounding); erfcf makes 8192 x 2048 x 8192 bf16 289 us instead of 255.
template <bool kExact>
__device__ inline float normal_cdf(float z, float& e) {
  if constexpr (kExact) {
    e = expf(-0.5f * z * z);
    return 0.5f * erfcf(-0.7071067811865476f * z);
  }
  e = __builtin_amdgcn_exp2f(-0.7213475204444817f * z * z);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.32f, fabsf(z), 1.f));
  float p = 0.03451938390762332f;
  p = fmaf(p, t, -0.12242638526675143f);
  p = fmaf(p, t, 0.10610846685020263f);
  p = fmaf(p, t, 0.015594329802750986f);
  p = fmaf(p, t, 0.09737186472710228f);
  p = fmaf(p, t, 0.11343927545482123f);
  p = fmaf(p, t, 0.12773338312825433f);
  p = fmaf(p, t, 0.12765989817705162f);
  const float tail = p * t * e;
  return z < 0.f ? tail : 1.f - tail;
}

// One branch on the activation for kN values.
template <bool kExact, int kN>
__device__ inline void activate(float (&z)[kN], int act) {
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int j = 0; j < kN; ++j) z[j] = z[j] < 0.f ? 0.f : z[j];
      break;
    case kActGeluApproximate:
      // 0.5 (1 + tanh u) = sigmoid(2 u)
#pragma unroll
      for (int j = 0; j < kN; ++j)
        z[j] *= sigmoid<kExact>(2.f * kSqrt2OverPi * z[j] * fmaf(0.044715f * z[j], z[j], 1.f));
      break;
    case kActGeluExact:
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        float e;
        z[j] *= normal_cdf<kExact>(z[j], e);
      }
      break;
    case kActSilu:
#pragma unroll
      for (int j = 0; j < kN; ++j) z[j] *= sigmoid<kExact>(z[j]);
      break;
  }
}

template <bool kExact>
__device__ inline float activate_grad(float z, int act) {
  switch (act) {
    case kActRelu: return z > 0.f ? 1.f : 0.f;
    case kActGeluApproximate: {
      // d/dz [z s(v)] = s + s (1 - s) z v' with v = a z + b z^3.  s is 0 or 1
      // long before the square is held, so that no factor overflows beside
      // the 0.
      constexpr float kA = 2.f * kSqrt2OverPi, kB = kA * 0.044715f;
      const float z2 = fminf(z * z, 0x1p60f);
      const float s = sigmoid<kExact>(z * fmaf(kB, z2, kA));
      return fmaf(fmaf(-s, s, s) * z, fmaf(3.f * kB, z2, kA), s);
    }
    case kActGeluExact: {
      float e;
      const float cdf = normal_cdf<kExact>(z, e);
      return cdf + z * 0.3989422804014327f * e;
    }
    case kActSilu: {
      const float s = sigmoid<kExact>(z);
      return s * (1.f + z * (1.f - s));
    }
  }
  return 1.f;
}

// ---------------------------------------------------------------------------
// The product for operands with rows of more than 4 MiB, whose tiles' offsets
// pass 31 bits: tiles go to LDS through registers.  A workgroup of four waves
// computes a 128 x 128 tile of C, each wave 64 x 64 as 4 x 4 fragments of 16 x
// 16.  The weights' rows are the matrix instruction's first operand, so a lane
// ends with four consecutive n of one m.  (For other sizes the kernel below
// takes half the time: 8192 x 2048 x 8192 bf16 580 us here, 263 there.)
// ---------------------------------------------------------------------------
constexpr int kTile = 128;
constexpr int kThreads = 256;

// Bank spread: the 16-byte chunk c of tile row r is kept at chunk c ^ swz(r).
// Rows of k chunks: eight consecutive rows read the same chunk at once.
// Rows that are k, 16 bit: the transposing read takes 32 bytes of four
// consecutive k.  32 bit: the four lane groups read rows four apart.
template <class Op, bool kKRows>
__device__ inline int swz(int row) {
  if constexpr (kKRows) return row & 7;
  if constexpr (sizeof(typename Op::S) == 2) return (row & 3) << 1;
  return ((row >> 2) & 3) << 2;
}

// Guarded load of 16 bytes of row `row`, from column `col`: zeros outside
// [rows, cols].
template <typename S>
__device__ inline Bytes16 load_chunk(const S* __restrict__ p, int64_t ld, int64_t rows,
                                     int64_t cols, int64_t row, int64_t col) {
  constexpr int kN = 16 / static_cast<int>(sizeof(S));
  Bytes16 v = {{0, 0, 0, 0}};
  if (row >= rows || col >= cols) return v;
  const S* q = p + row * ld + col;
  if (col + kN <= cols) return *reinterpret_cast<const Bytes16*>(q);
  S e[kN] = {};
  for (int j = 0; j < kN - 1; ++j)
    if (col + j < cols) e[j] = q[j];
  __builtin_memcpy(&v, e, 16);
  return v;
}

// One operand's tile: 128 rows of 128 bytes (k contiguous), or 128 bytes'
// worth of k rows of 128 columns.
template <class Op, bool kKC>
struct Tile {
  using S = typename Op::S;
  static constexpr int kE = sizeof(S);
  static constexpr int kBK = kRowBytes / kE;
  static constexpr int kPitch = kKC ? kRowBytes : kTile * kE;
  static constexpr int kChunksPerRow = kPitch / 16;
  static constexpr int kBytes = kTile * kRowBytes;
  static constexpr int kPerThread = kBytes / 16 / kThreads;

  // rc: the tile's first row / column of C; k: first k.
  __device__ static void load(const S* p, int64_t ld, int64_t n, int64_t kdim, int64_t rc,
                              int64_t k, Bytes16 (&r)[kPerThread]) {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int id = i * kThreads + threadIdx.x;
      const int row = id / kChunksPerRow, col = id % kChunksPerRow * (16 / kE);
      r[i] = kKC ? load_chunk(p, ld, n, kdim, rc + row, k + col)
                 : load_chunk(p, ld, kdim, n, k + row, rc + col);
    }
  }
  __device__ static void store(char* lds, const Bytes16 (&r)[kPerThread]) {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int id = i * kThreads + threadIdx.x;
      const int row = id / kChunksPerRow, c = id % kChunksPerRow;
      i32x4 w;
      __builtin_memcpy(&w, &r[i], 16);
      *reinterpret_cast<i32x4*>(lds + row * kPitch + ((c ^ swz<Op, kKC>(row)) << 4)) = w;
    }
  }
  // The fragment of tile rows / columns [at, at + 16).
  __device__ static void fragment(const char* lds, int at, i32x4 (&f)[2]) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (kKC) {
        const int row = at + r;
        f[h] = *reinterpret_cast<const i32x4*>(lds + row * kPitch +
                                               (((4 * h + g) ^ swz<Op, true>(row)) << 4));
      } else if constexpr (kE == 2) {
        // Lane s of 16 reads four columns of row s / 4; after the
        // transpose lane i holds four k of column i.
        s16x4 t[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int row = 32 * h + 8 * g + 4 * q + (r >> 2);
          const int byte = (at + (r & 3) * 4) * 2;
          const int off = row * kPitch + (((byte >> 4) ^ swz<Op, false>(row)) << 4) + (byte & 15);
          t[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(lds + off));
        }
        f[h] = __builtin_bit_cast(i32x4, __builtin_shufflevector(t[0], t[1], 0, 1, 2, 3, 4, 5, 6, 7));
      } else {
        float t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 16 * h + 4 * g + j;
          const int byte = (at + r) * 4;
          const int off = row * kPitch + (((byte >> 4) ^ swz<Op, false>(row)) << 4) + (byte & 15);
          t[j] = *reinterpret_cast<const float*>(lds + off);
        }
        __builtin_memcpy(&f[h], t, 16);
      }
    }
  }
};

// kN consecutive n of row m, from the sums.  Bias, activation and residual take
// the float sum; y and, beside it, the value before the activation are each
// rounded once, by their stores.
template <class Tr, int kN>
__device__ inline void epilogue(const LinearEpilogue& e, int64_t m, int64_t n, int64_t cols,
                                float (&z)[kN]) {
  using S = typename Tr::S;
  struct __attribute__((packed, aligned(1))) Vec { S v[kN]; };
  const int64_t at = m * cols + n;
  // Whole vectors: global memory takes them at any alignment.
  if (cols - n >= kN) {
    if (e.row_scale) {
      struct __attribute__((packed, aligned(1))) Floats { float v[kN]; };
      const Floats cs = *reinterpret_cast<const Floats*>(e.col_scale + n);
      const float rs = e.row_scale[m];
#pragma unroll
      for (int j = 0; j < kN; ++j) z[j] *= rs * cs.v[j];
    }
    if (e.bias) {
      const Vec b = *reinterpret_cast<const Vec*>(static_cast<const S*>(e.bias) + n);
#pragma unroll
      for (int j = 0; j < kN; ++j) z[j] += Tr::ld(b.v[j]);
    }
    Vec o;
    if (e.pre) {
#pragma unroll
      for (int j = 0; j < kN; ++j) o.v[j] = Tr::st(z[j]);
      *reinterpret_cast<Vec*>(static_cast<S*>(e.pre) + at) = o;
    }
    activate<sizeof(S) == 4, kN>(z, e.act);
    if (e.residual) {
      const Vec r = *reinterpret_cast<const Vec*>(static_cast<const S*>(e.residual) + at);
#pragma unroll
      for (int j = 0; j < kN; ++j) z[j] += Tr::ld(r.v[j]);
    }
#pragma unroll
    for (int j = 0; j < kN; ++j) o.v[j] = Tr::st(z[j]);
    *reinterpret_cast<Vec*>(static_cast<S*>(e.y) + at) = o;
    return;
  }
  const int have = static_cast<int>(cols - n);
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    if (j >= have) break;
    if (e.row_scale) z[j] *= e.row_scale[m] * e.col_scale[n + j];
    if (e.bias) z[j] += Tr::ld(static_cast<const S*>(e.bias)[n + j]);
    if (e.pre) static_cast<S*>(e.pre)[at + j] = Tr::st(z[j]);
  }
  activate<sizeof(S) == 4, kN>(z, e.act);
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    if (j >= have) break;
    if (e.residual) z[j] += Tr::ld(static_cast<const S*>(e.residual)[at + j]);
    static_cast<S*>(e.y)[at + j] = Tr::st(z[j]);
  }
}

// The epilogue of a wave's kFM x kFN fragments: kRows rows of them at a time
// cross LDS, so that a lane has eight consecutive n and a row of the wave is
// stored whole.  region: the wave's own, kRows * 16 rows of kFN * 16 floats;
// the 16-byte chunk c of row r is kept at c ^ (r % 16).
template <class Tr, int kRows, int kFM, int kFN>
__device__ inline void store_wave(const LinearEpilogue& e, int64_t rows, int64_t cols, int64_t m0,
                                  int64_t n0, const f32x4 (&acc)[kFM][kFN], float* region) {
  constexpr int kPitch = kFN * 16, kMask = kFN * 4 - 1 < 15 ? kFN * 4 - 1 : 15;
  const int lane = threadIdx.x & 63;
  // One copy of the epilogue's code: the loop is not unrolled, and each turn
  // takes its fragments by a branch.
#pragma unroll 1
  for (int turn = 0; turn < kFM / kRows; ++turn) {
#pragma unroll
    for (int t = 0; t < kFM / kRows; ++t) {
      if (t != turn) continue;
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int j = 0; j < kFN; ++j)
          *reinterpret_cast<f32x4*>(region + (i * 16 + (lane & 15)) * kPitch +
                                    ((j * 4 + (lane >> 4)) ^ (lane & kMask)) * 4) =
              acc[t * kRows + i][j];
    }
    // The wave's own writes, read by other lanes of it.
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    constexpr int kLanes = kFN * 2;  // lanes per row
#pragma unroll 2
    for (int r = lane / kLanes; r < kRows * 16; r += 64 / kLanes) {
      const int c = lane % kLanes;
      const int64_t m = m0 + turn * kRows * 16 + r;
      float z[8];
      const float* p = region + r * kPitch;
      *reinterpret_cast<f32x4*>(z) = *reinterpret_cast<const f32x4*>(p + ((2 * c) ^ (r & kMask)) * 4);
      *reinterpret_cast<f32x4*>(z + 4) =
          *reinterpret_cast<const f32x4*>(p + ((2 * c + 1) ^ (r & kMask)) * 4);
      if (m < rows && n0 + c * 8 < cols) epilogue<Tr, 8>(e, m, n0 + c * 8, cols, z);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

template <class Op, class Tr, bool kAKC, bool kBKC>
__global__ __launch_bounds__(kThreads) void linear_kernel(GemmShape s, const void* a_, const void* b_,
                                                          LinearEpilogue ep) {
  using TA = Tile<Op, kAKC>;
  using TB = Tile<Op, kBKC>;
  using S = typename Op::S;
  __shared__ __attribute__((aligned(16))) char lds[TA::kBytes + TB::kBytes];
  const S* a = static_cast<const S*>(a_);
  const S* b = static_cast<const S*>(b_);
  const int64_t tiles_n = (s.n + kTile - 1) / kTile;
  const int64_t m0 = blockIdx.x / tiles_n * kTile, n0 = blockIdx.x % tiles_n * kTile;
  const int wave = threadIdx.x >> 6;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  f32x4 acc[4][4] = {};
  Bytes16 ra[TA::kPerThread], rb[TB::kPerThread];
  if (s.k > 0) {
    TA::load(a, s.lda, s.m, s.k, m0, 0, ra);
    TB::load(b, s.ldb, s.n, s.k, n0, 0, rb);
  }
  for (int64_t k = 0; k < s.k; k += TA::kBK) {
    __syncthreads();
    TA::store(lds, ra);
    TB::store(lds + TA::kBytes, rb);
    __syncthreads();
    if (k + TA::kBK < s.k) {
      TA::load(a, s.lda, s.m, s.k, m0, k + TA::kBK, ra);
      TB::load(b, s.ldb, s.n, s.k, n0, k + TA::kBK, rb);
    }
    i32x4 fa[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) TA::fragment(lds, wm + i * 16, fa[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      i32x4 fb[2];
      TB::fragment(lds + TA::kBytes, wn + j * 16, fb);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) Op::mma(fb[h], fa[i][h], acc[i][j]);
    }
  }
  __syncthreads();  // the tiles' LDS is free
  static_assert(4 * 32 * 64 * 4 <= TA::kBytes + TB::kBytes, "two rows of fragments per wave");
  store_wave<Tr, 2>(ep, s.m, s.n, m0 + wm, n0 + wn, acc,
                    reinterpret_cast<float*>(lds) + wave * 32 * 64);
}

// ---------------------------------------------------------------------------
// The product for operands whose rows are whole 16-byte vectors: tiles go from
// memory to LDS without registers (buffer loads with the LDS bit), the next
// step's while this one is multiplied.
//
// Measured, us, operands from memory (in brackets the library's plain product
// of the same size, warm): 8192 x 2048 x 8192 bf16 with bias, approximate GELU
// and the value before it kept 263 (224; 222 here without them), its gradient's
// two products 205 each, 4096 x 8192 x 2048 e4m3 71, 2048^3 f32 139, 16 x 2048 x
// 50304 bf16 45 (4.6 TB/s).  Large bf16 products are bound by the card's power
// with the matrix units half to two thirds busy, and by the epilogue's stores,
// which a wave's next loads wait behind; loads alone take 124 of 218 us (8192 x
// 8192 x 2048), all but the LDS reads 194.  64-byte steps (twice the requests,
// 238 against 218), more steps in flight (no change) and four waves of 128 x 128
// (250) were slower.
// ---------------------------------------------------------------------------
using Lds = __attribute__((address_space(3))) char;

// One operand's tile of kT rows (columns) of C and one step of k, loaded by
// kWaves waves.  The resource's base moves with k; what lies outside the
// matrix is outside the resource or is given an offset that is, and arrives as
// zeros.
template <class Op, bool kKC, int kT, int kWaves, bool kTurned>
struct DirectTile {
  using S = typename Op::S;
  using Frag = typename Op::Frag;
  static constexpr int kE = sizeof(S);
  static constexpr int kRow = kRowBytes;
  static constexpr int kBK = kRow / kE;
  static constexpr int kPitch = kKC ? kRow : kT * kE;
  static constexpr int kChunksPerRow = kPitch / 16;
  static constexpr int kBytes = kT * kRow;
  static constexpr int kLoads = kBytes / 1024 / kWaves;  // per wave; 64 lanes of 16 bytes
  static_assert(kLoads * 1024 * kWaves == kBytes, "whole loads");

  // Bank spread: the 16-byte chunk c of tile row r is kept at chunk
  // c ^ swizzle(r).  k contiguous: eight consecutive rows read the same chunk
  // at once.  Rows of k, 16 bit: the transposing read takes 32 bytes of four
  // consecutive k, 8 k apart for the next 16 lanes.  32 bit: the four groups
  // of 16 lanes read rows four apart.  (No conflicts in the main loop:
  // SQ_LDS_BANK_CONFLICT counts the epilogue's only.)
  __device__ static int swizzle(int row) {
    if constexpr (kKC) return row & 7;
    if constexpr (kE == 2) return (((row & 3) | ((row >> 1) & 4)) << 1) & (kChunksPerRow - 1);
    return (((row >> 2) & 3) << 2) & (kChunksPerRow - 1);
  }

  const char* base;
  int64_t step;  // bytes from one step of k to the next
  int64_t left;  // bytes from base to the end of the matrix
  int64_t kleft;  // k from base on
  int turn, turns, issued;  // kTurned: the step base is at, of how many, and how many were given
  int kvalid;  // of them in the step that `next` gave
  // Load i of a wave takes 1024 / kPitch rows, kRowsPerLoad below load i - 1's;
  // where that keeps the swizzle, one offset and column serve all.
  static constexpr int kRowsPerLoad = kWaves * 64 / kChunksPerRow;
  static constexpr bool kSame = kRowsPerLoad % 16 == 0;
  static constexpr int kOffs = kSame ? 1 : kLoads;
  uint32_t off[kOffs];
  int col[kOffs];  // kKC: the load's first k of the step
  uint32_t down;  // bytes between loads

  // rc: the tile's first row / column of C, of n; k in [k0, k1).
  // kTurned: the steps begin with step `first` of `steps` and go round.
  __device__ void init(const void* p, int64_t ld, int64_t n, int64_t kdim, int64_t rc, int64_t k0,
                       int64_t k1, int wave, int steps, int first) {
    const int lane = threadIdx.x & 63;
    const int64_t start = (kKC ? rc * ld + k0 : k0 * ld + rc) * kE;
    base = static_cast<const char*>(p) + start;
    step = (kKC ? kBK : kBK * ld) * kE;
    left = (kKC ? n : k1) * ld * kE - start;
    kleft = k1 - k0;
    if constexpr (kTurned) {
      turn = first;
      turns = steps;
      issued = 0;
      move(first);
    }
    down = static_cast<uint32_t>(kRowsPerLoad * ld * kE);
#pragma unroll
    for (int i = 0; i < kOffs; ++i) {
      const int at = (i * kWaves + wave) * 64 + lane;
      const int row = at / kChunksPerRow, c = (at % kChunksPerRow) ^ swizzle(row);
      col[i] = c * (16 / kE);
      off[i] = static_cast<uint32_t>(row * ld * kE + c * 16);
      if (!kKC && rc + col[i] >= n) off[i] = kOutside;
    }
  }
  __device__ void move(int steps) {
    base += steps * step;
    left -= steps * step;
    kleft -= steps * kBK;
  }
  // An offset past every resource, with any load's way down added.
  static constexpr uint32_t kOutside = 0x80000000u;

  // The resource of the next step; then base moves on.
  __device__ i32x4 next() {
    const int64_t most = 0x7fffffff;
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    const int64_t in = kleft > 0 && (!kTurned || issued < turns) ? left : 0;
    const i32x4 r = {static_cast<int>(at), static_cast<int>(at >> 32 & 0xffff),
                     static_cast<int>(in < most ? in : most), 0x00020000};
    kvalid = kleft < kBK ? static_cast<int>(kleft) : kBK;
    if constexpr (kTurned) {
      ++issued;
      const bool round = ++turn == turns;
      move(round ? 1 - turns : 1);
      if (round) turn = 0;
    } else {
      move(1);
    }
    return r;
  }
  // Load i of the step.  It is written out because the compiler, which does
  // not know which bytes of LDS it writes, would wait for it before every LDS
  // read; the kernel waits for it itself.  The no-ops stand for the five wait
  // states between a vector instruction that writes a scalar register (of r)
  // and a buffer load that reads it, and the one after m0 is written: the
  // compiler does not look into the text.  lds: byte address of the tile.
  __device__ void load(const i32x4& r, uint32_t lds, int wave, int i) {
    const int q = kSame ? 0 : i;
    const uint32_t first = kKC && col[q] >= kvalid ? kOutside : off[q];
    const uint32_t o = kSame ? first + i * down : first;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved, and clobbered
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :: "s"(lds + (i * kWaves + wave) * 1024), "v"(o), "s"(r)
                 : "m0", "memory");
#pragma clang diagnostic pop
  }
  // The fragment of 16 tile rows / columns from `at` on, of part h.
  __device__ static Frag fragment(const Lds* lds, int at, int h) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    if constexpr (kKC) {
      using Word = const __attribute__((address_space(3))) i32x4;
      const int row = at + r;
      const Lds* p = lds + row * kPitch;
      const i32x4 lo = *reinterpret_cast<Word*>(p + (((4 * h + g) ^ swizzle(row)) << 4));
      if constexpr (Op::kParts == 2) {
        return lo;
      } else {
        const i32x4 hi = *reinterpret_cast<Word*>(p + (((g + 4) ^ swizzle(row)) << 4));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    } else if constexpr (kE == 2) {
      // Lane s of 16 reads four columns of row s / 4; after the transpose
      // lane i holds four k of column i.
      s16x4 t[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int row = 32 * h + 8 * g + 4 * q + (r >> 2);
        const int byte = (at + (r & 3) * 4) * 2;
        const int off = row * kPitch + (((byte >> 4) ^ swizzle(row)) << 4) + (byte & 15);
        t[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(lds + off));
      }
      return __builtin_bit_cast(i32x4, __builtin_shufflevector(t[0], t[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      i32x4 t;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 16 * h + 4 * g + j;
        const int byte = (at + r) * 4;
        t[j] = *reinterpret_cast<const __attribute__((address_space(3))) int*>(
            lds + row * kPitch + (((byte >> 4) ^ swizzle(row)) << 4) + (byte & 15));
      }
      return t;
    }
  }
};

// The tiles of C and the split of k: item i of tiles_m * tiles_n * splits.
struct Items {
  int tiles_m, tiles_n, splits;
  int steps;  // of one split
  int64_t count() const { return int64_t(tiles_m) * tiles_n * splits; }
};

// Tiles in the order that workgroups take them: workgroup b runs on XCD b % 8,
// so each XCD gets a run of items of its own, and within the run tiles go down
// eight rows of C before the next column, which keeps the operands of 32
// concurrent tiles in the XCD's L2.
__device__ inline void item_of(uint32_t b, const Items& it, int& tm, int& tn, int& split) {
  const uint32_t tiles = it.tiles_m * it.tiles_n, n = tiles * it.splits, q = n / 8, r = n % 8;
  const uint32_t x = b % 8;
  const uint32_t at = x * q + (x < r ? x : r) + b / 8;
  split = at / tiles;
  const uint32_t t = at - split * tiles;
  const uint32_t band = t / (8 * it.tiles_n), in = t - band * 8 * it.tiles_n;
  const uint32_t rows = it.tiles_m - band * 8 < 8 ? it.tiles_m - band * 8 : 8;
  tm = band * 8 + in % rows;
  tn = in / rows;
}

// A configuration of the direct kernel: kTM x kTN of C per workgroup of
// kWavesM x kWavesN waves, and kSlots steps of k in LDS beside the epilogue's
// region.
// kTurned: with one row of tiles, where no two workgroups read the same B,
// each XCD begins an eighth of k after the one before, so that they do not all
// read the same columns of rows that lie a power of two apart (16 x 2048 x
// 50304 bf16 from memory: 52 us without, 45 with; with shared tiles 266 against
// 281 for 8192 x 2048 x 8192).
template <int kTM_, int kTN_, int kWavesM_, int kWavesN_, int kSlots_, int kRegionRows_,
          bool kTurned_ = false>
struct Config {
  static constexpr bool kTurned = kTurned_;
  // A tile's longest rows end below DirectTile::kOutside, which no sum of an
  // offset and the way down from it then passes by 2^32 either.
  static_assert((kTM_ > kTN_ ? kTM_ : kTN_) * kLinear8MaxK <= int64_t(1) << 31,
                "offsets in 31 bits");
  static constexpr int kTM = kTM_, kTN = kTN_, kWavesM = kWavesM_, kWavesN = kWavesN_,
                       kSlots = kSlots_, kWaves = kWavesM * kWavesN;
  static constexpr int kFM = kTM / kWavesM / 16, kFN = kTN / kWavesN / 16;  // fragments of a wave
  static constexpr int kRegionRows = kRegionRows_;  // fragment rows that cross LDS at once
  static_assert(kFM % kRegionRows == 0, "whole regions");
  static constexpr int kRegion = kRegionRows * 16 * kFN * 16;  // floats per wave
  static constexpr int lds() {
    return kSlots * (kTM + kTN) * kRowBytes + kWaves * kRegion * 4;
  }
};

// A persistent workgroup: items blockIdx.x, blockIdx.x + gridDim.x, ...; the
// first loads of the next item are on their way during the epilogue.
// partial: with more than one split, the sums [splits, m, n] go there in
// float and join_kernel finishes.
template <class Op, class Tr, bool kAKC, bool kBKC, class Cf>
__global__ __launch_bounds__(Cf::kWaves * 64) void direct_kernel(GemmShape s, Items items,
                                                                const void* a, const void* b,
                                                                LinearEpilogue ep, float* partial) {
  using TA = DirectTile<Op, kAKC, Cf::kTM, Cf::kWaves, Cf::kTurned>;
  using TB = DirectTile<Op, kBKC, Cf::kTN, Cf::kWaves, Cf::kTurned>;
  using Frag = typename Op::Frag;
  constexpr int kStage = TA::kBytes + TB::kBytes, kSlots = Cf::kSlots;
  constexpr int kFM = Cf::kFM, kFN = Cf::kFN;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  Lds* lds = (Lds*)smem;
  const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / Cf::kWavesN * (kFM * 16), wn = wave % Cf::kWavesN * (kFN * 16);
  float* region = reinterpret_cast<float*>(smem + kSlots * kStage) + wave * Cf::kRegion;

  // A ring of kSlots steps in LDS.  While one part's fragments are multiplied
  // the next part's are read.  Before a step's last part is multiplied - f32,
  // whose instructions take longest: after its first row - the waves meet: the
  // step's room is free, and the loads that fill it again run kSlots steps
  // ahead.  (2048^3 f32 142.5 us without that row, 138.5 with; 8192 x 2048 x
  // 8192 bf16 262 without one, 265 with.)  Steps past the end load zeros, so
  // every wait counts the same.
  TA ta;
  TB tb;
  uint32_t fill = 0, use = 0;  // byte offsets of the steps to fill and to read next
  auto advance = [](uint32_t& at) { at = at + kStage == kSlots * kStage ? 0 : at + kStage; };
  constexpr int kLoads = TA::kLoads + TB::kLoads, kParts = Op::kParts;
  constexpr int kInFlight = (kSlots - 2) * kLoads;
  static_assert(kInFlight < 64, "vmcnt has six bits");
  auto load_one = [&](const i32x4& ra, const i32x4& rb, int i) {
    if (i < TA::kLoads)
      ta.load(ra, at + fill, wave, i);
    else
      tb.load(rb, at + fill + TA::kBytes, wave, i - TA::kLoads);
  };
  auto load = [&]() {
    const i32x4 ra = ta.next(), rb = tb.next();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_one(ra, rb, i);
    advance(fill);
  };
  // Points the tiles at an item and starts its first loads.
  int tm, tn, split;
  auto start = [&](uint32_t item) {
    item_of(item, items, tm, tn, split);
    const int64_t k0 = int64_t(split) * items.steps * TA::kBK;
    const int64_t k1 = k0 + int64_t(items.steps) * TA::kBK < s.k ? k0 + int64_t(items.steps) * TA::kBK : s.k;
    const int first = items.tiles_m == 1 ? static_cast<int>(blockIdx.x % 8) * items.steps / 8 : 0;
    ta.init(a, s.lda, s.m, s.k, int64_t(tm) * Cf::kTM, k0, k1, wave, items.steps, first);
    tb.init(b, s.ldb, s.n, s.k, int64_t(tn) * Cf::kTN, k0, k1, wave, items.steps, first);
#pragma unroll
    for (int i = 0; i < kSlots - 1; ++i) load();
  };
  // A's fragments are read again as soon as their row of products is issued;
  // B's serve every row and have a second set (4096 x 8192 x 2048 e4m3 71.7 us
  // without one, 70.9 with; its fragments of the largest tile leave no registers
  // for one and are read in the last row).
  constexpr int kSets = Op::kParts == 2 || kFM <= 4 ? 2 : 1;
  Frag fa[kFM], fb[kSets][kFN];
  auto read_a = [&](int h, int i) { fa[i] = TA::fragment(lds + use, wm + i * 16, h); };
  auto read_b = [&](int p, int h, int j) {
    fb[p][j] = TB::fragment(lds + use + TA::kBytes, wn + j * 16, h);
  };
  constexpr int kMeet = sizeof(typename Op::S) == 4 ? 1 : 0;
  const uint32_t count = items.tiles_m * items.tiles_n * items.splits;
  uint32_t item = blockIdx.x;
  start(item);
  for (;;) {
    f32x4 acc[kFM][kFN] = {};
    // One part: the matrix instructions with the next reads and loads between
    // them, so that a queue that is full does not hold them up.
    auto body = [&](int p, int h) {
      const bool last = h == kParts - 1;
      i32x4 ra, rb;
      const int then = last ? 0 : h + 1;  // the part that is read
      const int from = last ? kMeet : 0;  // the first row with reads behind it
#pragma unroll
      for (int i = 0; i < kFM; ++i) {
        if (last && i == kMeet) {
          // The next step has arrived, and every wave has read this one.
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kInFlight) : "memory");
          advance(use);
          ra = ta.next();
          rb = tb.next();
#pragma unroll
          for (int q = 0; q < kMeet; ++q) read_a(then, q);
        }
#pragma unroll
        for (int j = 0; j < kFN; ++j) {
          Op::mma(fb[p % kSets][j], fa[i], acc[i][j]);
          if (kSets == 1 && i == kFM - 1) read_b(0, then, j);
        }
        if (i >= from) {
          const int at_row = i - from;
          read_a(then, i);
          if (kSets == 2) {
            constexpr int kSpread = kFM / 2;
#pragma unroll
            for (int q = at_row * kFN / kSpread; q < (at_row + 1) * kFN / kSpread && q < kFN; ++q)
              read_b(1 - p, then, q);
          }
          if (last) {
            constexpr int kRows = kFM - kMeet;
#pragma unroll
            for (int q = at_row * kLoads / kRows; q < (at_row + 1) * kLoads / kRows; ++q)
              load_one(ra, rb, q);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (last) advance(fill);
    };
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kInFlight) : "memory");
    load();
#pragma unroll
    for (int j = 0; j < kFN; ++j) read_b(0, 0, j);
#pragma unroll
    for (int i = 0; i < kFM; ++i) read_a(0, i);
    for (int t = 0; t < items.steps; t += 2 / kParts) {
      body(0, 0);
      body(1, kParts - 1);
    }
    // The loads past the end write zeros to the ring: they are waited for, by
    // every wave, before the next item's.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    fill = use = 0;
    const int64_t m0 = int64_t(tm) * Cf::kTM + wm, n0 = int64_t(tn) * Cf::kTN + wn;
    const int this_split = split;
    item += gridDim.x;
    const bool more = item < count;
    if (more) start(item);
    if (items.splits == 1) {
      store_wave<Tr, Cf::kRegionRows>(ep, s.m, s.n, m0, n0, acc, region);
    } else {
      float* out = partial + this_split * s.m * s.n;
#pragma unroll
      for (int i = 0; i < kFM; ++i) {
        const int64_t m = m0 + i * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < kFN; ++j) {
          const int64_t n = n0 + j * 16 + (lane >> 4) * 4;
          if (m >= s.m || n >= s.n) continue;
          struct __attribute__((packed, aligned(4))) Four { f32x4 v; };
          if (n + 4 <= s.n)
            reinterpret_cast<Four*>(out + m * s.n + n)->v = acc[i][j];
          else
            for (int q = 0; n + q < s.n; ++q) out[m * s.n + n + q] = acc[i][j][q];
        }
      }
    }
    if (!more) return;
  }
}

// Adds the splits' sums, which are float, in order and finishes them.  About 3 us
// for little data.
template <class Tr>
__global__ __launch_bounds__(256) void join_kernel(uint32_t across, int64_t m, int64_t n,
                                                   int splits, const float* partial,
                                                   LinearEpilogue e) {
  const int64_t per_row = (n + 7) / 8;
  const int64_t i = group_of_many(across) * 256 + threadIdx.x;
  if (i >= m * per_row) return;
  const int64_t row = i / per_row, col = i % per_row * 8;
  const float* p = partial + row * n + col;
  float z[8] = {};
  if (col + 8 <= n) {
    struct __attribute__((packed, aligned(4))) Eight { float v[8]; };
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const Eight w = *reinterpret_cast<const Eight*>(p + s * m * n);
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] += w.v[j];
    }
  } else {
    for (int s = 0; s < splits; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < n) z[j] += p[s * m * n + j];
  }
  epilogue<Tr, 8>(e, row, col, n, z);
}

template <class Tr>
hipError_t launch_join(const GemmShape& s, int splits, const void* workspace, const LinearEpilogue& e,
                       hipStream_t stream) {
  const int64_t groups = (s.m * ((s.n + 7) / 8) + 255) / 256;
  const dim3 grid = many_groups(groups);
  TFMA_LAUNCH("tfma_linear_join", join_kernel<Tr>, grid, dim3(256), 0, stream, grid.x, s.m, s.n,
              splits, static_cast<const float*>(workspace), e);
  return hipGetLastError();
}

// Whether rows of `ld` elements at p can go straight to LDS: every row starts
// on a 16-byte boundary, and a tile's offsets fit 31 bits.
bool direct_ok(const void* p, int64_t ld, int esize) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * esize % 16 == 0 &&
         ld * esize <= (int64_t(1) << 22);
}

template <class Op, class Tr, bool kAKC, bool kBKC, class Cf>
hipError_t launch_direct(const GemmShape& s, const void* a, const void* b, const LinearEpilogue& e,
                         void* workspace, int splits, hipStream_t stream) {
  constexpr int kLds = Cf::lds();
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
  constexpr int kBK = kRowBytes / static_cast<int>(sizeof(typename Op::S));
  const int64_t tiles_m = (s.m + Cf::kTM - 1) / Cf::kTM, tiles_n = (s.n + Cf::kTN - 1) / Cf::kTN;
  if (tiles_m * tiles_n * splits >= (int64_t(1) << 31)) return hipErrorInvalidConfiguration;
  const int64_t steps = (s.k + kBK - 1) / kBK;
  constexpr int kMult = 2 / Op::kParts;  // steps of a turn of the main loop
  const int64_t per = ((steps + splits - 1) / splits + kMult - 1) / kMult * kMult;
  const Items items = {static_cast<int>(tiles_m), static_cast<int>(tiles_n), splits,
                       static_cast<int>(per)};
  const int64_t at_once = DeviceCUs() * int64_t(160 * 1024 / kLds);
  const int64_t grid = items.count() < at_once ? items.count() : at_once;
  TFMA_LAUNCH("tfma_linear_direct", (direct_kernel<Op, Tr, kAKC, kBKC, Cf>),
              dim3(static_cast<uint32_t>(grid)), dim3(Cf::kWaves * 64), kLds, stream, s, items, a, b,
              e, static_cast<float*>(workspace));
  if (const hipError_t err = hipGetLastError(); err != hipSuccess || splits == 1) return err;
  return launch_join<Tr>(s, splits, workspace, e, stream);
}

// ---------------------------------------------------------------------------
// Products of at most 16 kMT rows, bound by the read of B or, for little of
// it, by the latency of a launch and of one read after the other: B goes
// straight to the registers, once, in whole pieces of 128 to 256 bytes, and the
// sixteen waves of a workgroup, which has 16 kNJ columns of C, share k and join
// in LDS.  Any sizes and alignments.
//
// B [n, k]: a lane reads 16 bytes of k of row l % 16 of a fragment.
// B [k, n], 16 bit: a lane reads kNJ n of each of 8 k and transposes the 8 x
// kNJ block by byte permutes; fragment j of the wave then has n = (l % 16) kNJ
// + j, and a lane ends with kNJ consecutive n.  32 bit: element j of the
// lane's 16 bytes is fragment j's already.
// ---------------------------------------------------------------------------
template <typename S, int kN>
__device__ inline void load_row(const S* __restrict__ p, int64_t ld, int64_t rows, int64_t cols,
                                int64_t row, int64_t col, uint32_t (&out)[kN * sizeof(S) / 4]) {
  struct __attribute__((packed, aligned(1))) Vec { uint32_t w[kN * sizeof(S) / 4]; };
  Vec v = {};
  if (row < rows && col < cols) {
    const S* q = p + row * ld + col;
    if (col + kN <= cols) {
      v = *reinterpret_cast<const Vec*>(q);
    } else {
      S e[kN] = {};
      for (int j = 0; j < kN - 1; ++j)
        if (col + j < cols) e[j] = q[j];
      __builtin_memcpy(&v, e, sizeof(v));
    }
  }
  __builtin_memcpy(out, &v, sizeof(v));
}

template <class Op, class Tr, bool kBKC, int kMT, int kNJ, int kWaves>
__global__ __launch_bounds__(kWaves * 64) void few_rows_kernel(
    GemmShape s, uint32_t across, int splits, int steps, const void* a_, const void* b_,
    LinearEpilogue ep, float* partial) {
  using S = typename Op::S;
  using Frag = typename Op::Frag;
  constexpr int kE = sizeof(S), kChunk = 16 / kE, kCols = 16 * kNJ;
  constexpr int kParts = kBKC ? Op::kParts : 1;
  constexpr int kRows = kBKC ? 0 : (kE == 2 ? 8 : 4);  // k of a lane and step, B [k, n]
  constexpr int kBK = kBKC ? kRowBytes / kE : 4 * kRows;
  constexpr int kQuads = sizeof(Frag) / 16;  // 16-byte chunks of a fragment
  constexpr int kPitch = kCols + 4;
  __shared__ __attribute__((aligned(16))) float sums[kWaves * 16 * kMT * kPitch];
  const S* a = static_cast<const S*>(a_);
  const S* b = static_cast<const S*>(b_);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const uint32_t group = static_cast<uint32_t>(group_of_many(across));
  const int tile = group / splits, split = group % splits;
  const int64_t n0 = int64_t(tile) * kCols;
  if (n0 >= s.n) return;
  f32x4 acc[kMT][kNJ] = {};
  const int64_t k_end = int64_t(split + 1) * steps * kBK < s.k ? int64_t(split + 1) * steps * kBK : s.k;
  for (int64_t k = (int64_t(split) * steps + wave) * kBK; k < k_end; k += kWaves * kBK) {
    Frag fx[kParts][kMT];
    uint32_t w[kBKC ? kParts * kNJ : kRows][kBKC ? sizeof(Frag) / 4 : kNJ * kE / 4];
    if constexpr (kBKC) {
#pragma unroll
      for (int h = 0; h < kParts; ++h)
#pragma unroll
        for (int j = 0; j < kNJ; ++j)
#pragma unroll
          for (int q = 0; q < kQuads; ++q) {
            uint32_t t[4];
            load_row<S, kChunk>(b, s.ldb, s.n, k_end, n0 + j * 16 + r, k + (4 * (h + q) + g) * kChunk,
                                t);
            __builtin_memcpy(w[h * kNJ + j] + 4 * q, t, 16);
          }
    } else {
#pragma unroll
      for (int t = 0; t < kRows; ++t)
        load_row<S, kNJ>(b, s.ldb, k_end, s.n, k + g * kRows + t, n0 + r * kNJ, w[t]);
    }
#pragma unroll
    for (int h = 0; h < kParts; ++h)
#pragma unroll
      for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
          uint32_t t[4];
          load_row<S, kChunk>(a, s.lda, s.m, k_end, i * 16 + r, k + (4 * (h + q) + g) * kChunk, t);
          __builtin_memcpy(reinterpret_cast<char*>(&fx[h][i]) + 16 * q, t, 16);
        }
    if constexpr (kBKC) {
#pragma unroll
      for (int h = 0; h < kParts; ++h)
#pragma unroll
        for (int j = 0; j < kNJ; ++j) {
          Frag fw;
          __builtin_memcpy(&fw, w[h * kNJ + j], sizeof(Frag));
#pragma unroll
          for (int i = 0; i < kMT; ++i) Op::mma(fw, fx[h][i], acc[i][j]);
        }
    } else {
#pragma unroll
      for (int j = 0; j < kNJ; ++j) {
        i32x4 fw;
        if constexpr (kE == 2) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            fw[q] = __builtin_amdgcn_perm(w[2 * q + 1][j / 2], w[2 * q][j / 2],
                                          j % 2 ? 0x07060302u : 0x05040100u);
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t) fw[t] = static_cast<int>(w[t][j]);
        }
#pragma unroll
        for (int i = 0; i < kMT; ++i) Op::mma(fw, fx[0][i], acc[i][j]);
      }
    }
  }
  float* mine = sums + wave * 16 * kMT * kPitch;
#pragma unroll
  for (int i = 0; i < kMT; ++i) {
    float* row = mine + (i * 16 + r) * kPitch;
    if constexpr (kBKC) {
#pragma unroll
      for (int j = 0; j < kNJ; ++j)
        *reinterpret_cast<f32x4*>(row + j * 16 + g * 4) = acc[i][j];
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int j = 0; j < kNJ; j += 4) {
          const f32x4 v = {acc[i][j][q], acc[i][j + 1][q], acc[i][j + 2][q], acc[i][j + 3][q]};
          *reinterpret_cast<f32x4*>(row + (g * 4 + q) * kNJ + j) = v;
        }
    }
  }
  __syncthreads();
  // Eight n of one row a thread: the waves' sums in order.
  for (int t = threadIdx.x; t < 16 * kMT * (kCols / 8); t += kWaves * 64) {
    const int m = t / (kCols / 8), c = t % (kCols / 8) * 8;
    if (m >= s.m || n0 + c >= s.n) continue;
    float z[8] = {};
    for (int v = 0; v < kWaves; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] += sums[(v * 16 * kMT + m) * kPitch + c + j];
    if (splits == 1) {
      epilogue<Tr, 8>(ep, m, n0 + c, s.n, z);
    } else {
      float* out = partial + (int64_t(split) * s.m + m) * s.n + n0 + c;
      for (int j = 0; j < 8 && n0 + c + j < s.n; ++j) out[j] = z[j];
    }
  }
}

// Which products few_rows_kernel takes: those of up to kFewRows rows whose
// operands cannot go straight to LDS; and those that it finishes in one launch
// of few turns per wave where the tiles of the other kernel need a split and a
// join.  Measured, this kernel / tiles, us:
//   B [k, n] bf16, up to 32 rows: 16 x 2048 x 8192 9.4 / 11.7, 32 x 2048 x 8192
//   11.1 / 12.3, 16 x 4096 x 8192 16.5 / 18.1; 16 x 4096 x 4096, with half the
//   workgroups, 14.9 / 12.2; f32 16 x 2048 x 2048 16.5 / 13.6;
//   B [n, k] bf16, up to 16 rows: 16 x 1024 x 1024 5.9 / 8.9, 16 x 4096 x 4096
//   10.6 / 11.9, 16 x 4096 x 8192, whose read the loads to LDS carry better,
//   21.6 / 15.4 (f32 16 x 4096 x 4096 20.3 / 25.7); 32 x 2048 x 8192 15.5 / 11.9;
//   B [n, k] e4m3, whose turn takes 2048 k and whose reads of A count, one
//   round of workgroups and less than a turn: 1 x 512 x 4096 5.3 / 6.4, 1 x 1536 x
//   1536 8.0 / 10.0, 4 x 1024 x 4096 7.1 / 8.3, 16 x 256 x 2048 4.7 / 5.4, 16 x
//   512 x 4096 6.4 / 6.4; past that 1 x 512 x 8192 7.7 / 6.5, 4 x 2048 x 2048 10.2
//   / 8.7, 16 x 1024 x 1024 8.8 / 8.2, 1 x 2048 x 8192 17.8 / 9.9, 16 x 4096 x 8192
//   47.6 / 13.3.
constexpr int kFewRows = 32;
constexpr int kFewWaves = 16;

// k of a step, and steps of a wave without a split.
int few_step(bool b_kc, int esize) { return b_kc ? kRowBytes / esize : (esize == 2 ? 32 : 16); }

bool few_rows(const GemmShape& s, bool direct, int esize) {
  if (!s.a_kc || s.m > kFewRows) return false;
  if (!direct) return true;
  if (esize == 1) return s.m <= 16 && s.n <= 4096 && s.k <= (s.m <= 4 ? 1536 : 512);
  const int64_t bytes = s.k * s.n * esize, turn = int64_t(kFewWaves) * few_step(s.b_kc, esize);
  const int64_t turns = (s.k + turn - 1) / turn;
  if (s.b_kc) return s.m <= 16 && s.k <= 4096 && bytes <= (int64_t(esize == 4 ? 72 : 48) << 20);
  return bytes <= (int64_t(72) << 20) && (turns <= 4 || (turns <= 8 && s.n >= 8192));
}

// Workgroups share k until about 256 of them are at work, where each wave has
// at least eight steps (1 x 2048 x 8192 bf16: 9.7 us in one launch; in two
// splits 8.6 and a join of 3.0).
int few_rows_splits(int64_t tiles, int64_t steps, int waves) {
  const int64_t want = (256 + tiles - 1) / tiles, most = steps / (8 * waves);
  const int64_t s = want < most ? want : most;
  return static_cast<int>(s < 1 ? 1 : (s > 16 ? 16 : s));
}

// Columns of a workgroup (nj * 16; enough of them to fill the chip at two where
// B is [n, k]) and splits of a product of few rows.
struct FewPlan {
  int nj;
  int splits;
};
FewPlan plan_few(bool b_kc, const GemmShape& s, int esize) {
  FewPlan p;
  p.nj = b_kc ? (s.n >= 32 * 512 ? 2 : 1) : 4;
  const int bk = few_step(b_kc, esize);
  p.splits = few_rows_splits((s.n + 16 * p.nj - 1) / (16 * p.nj), (s.k + bk - 1) / bk, kFewWaves);
  return p;
}

template <class Op, class Tr, bool kBKC, int kNJ>
hipError_t launch_few(const GemmShape& s, const void* a, const void* b, const LinearEpilogue& e,
                      void* workspace, int splits, hipStream_t stream) {
  const int bk = few_step(kBKC, sizeof(typename Op::S));
  const int64_t tiles = (s.n + 16 * kNJ - 1) / (16 * kNJ), all = (s.k + bk - 1) / bk;
  const int steps = static_cast<int>((all + splits - 1) / splits);
  const dim3 grid = many_groups(tiles * splits), block(kFewWaves * 64);
  float* partial = static_cast<float*>(workspace);
  constexpr bool kWide = sizeof(typename Op::S) > 1;  // e4m3 operands never need 32 rows
  if (!kWide || s.m <= 16)
    TFMA_LAUNCH("tfma_linear_few", (few_rows_kernel<Op, Tr, kBKC, 1, kNJ, kFewWaves>), grid, block, 0,
                stream, s, grid.x, splits, steps, a, b, e, partial);
  else if constexpr (kWide)
    TFMA_LAUNCH("tfma_linear_few", (few_rows_kernel<Op, Tr, kBKC, 2, kNJ, kFewWaves>), grid, block, 0,
                stream, s, grid.x, splits, steps, a, b, e, partial);
  if (const hipError_t err = hipGetLastError(); err != hipSuccess || splits == 1) return err;
  return launch_join<Tr>(s, splits, workspace, e, stream);
}

// The configurations, from the largest tile to the smallest.
using Direct256x256 = Config<256, 256, 2, 4, 2, 1>;
using Direct256x128 = Config<256, 128, 4, 2, 2, 2>;
using Direct128x128 = Config<128, 128, 2, 4, 3, 2>;
using Direct64x128 = Config<64, 128, 2, 4, 3, 1, true>;
enum DirectTag { k256x256, k256x128, k128x128, k64x128, kConfigs };

// A product's way: a configuration and a split of k, by the least of
//   rounds of workgroups x (start and epilogue + steps x time of a step) + join
// with times in us fitted on MI355X, one workgroup on every CU (a step is 128
// bytes of k).  Large tiles take the fewest bytes per product, small ones fill
// the chip.  Measured bf16, m x k x n, by tile 256x256 / 256x128 / 128x128 /
// 64x128: 4096 x 4096 x 4096 119 / 143 / 169 / 237 us, 2048 x 2048 x 2048
// 49 / 36 / 24 / 32, 1024 x 512 x 1024 20 / 13 / 9 / 7.5.  A join costs its
// launch and two passes over the sums.
struct Plan {
  int tag;
  int splits;
};

Plan plan_direct(DType t, bool e4m3, const GemmShape& s) {
  static constexpr int kTM[kConfigs] = {256, 256, 128, 64}, kTN[kConfigs] = {256, 128, 128, 128};
  struct Times {
    double fixed[kConfigs], step[kConfigs];
  };
  static constexpr Times k16 = {{12., 11., 7., 5.}, {1.67, 0.98, 0.53, 0.38}};
  static constexpr Times k32 = {{36., 14., 10., 6.}, {7.15, 3.83, 2.0, 1.1}};
  static constexpr Times k8 = {{20., 11., 7., 5.}, {2.0, 0.95, 0.53, 0.36}};
  const Times& times = e4m3 ? k8 : (t == DType::kF32 ? k32 : k16);
  const int esize = e4m3 ? 1 : DTypeBytes(t);
  const int64_t steps = (s.k * esize + kRowBytes - 1) / kRowBytes;
  const int64_t cus = DeviceCUs();
  Plan best = {k64x128, 1};
  double least = -1.;
  const int forced = TuneValue(kTuneLinearTile), forced_splits = TuneValue(kTuneLinearSplits);
  for (int c = 0; c < kConfigs; ++c) {
    if (forced >= 0 && forced < kConfigs && c != forced) continue;
    const int64_t tiles = ((s.m + kTM[c] - 1) / kTM[c]) * ((s.n + kTN[c] - 1) / kTN[c]);
    for (int splits = 1; splits <= 32; splits *= 2) {
      if (splits > 1 && (steps < 4 * splits || tiles * splits > 2 * cus)) break;
      const int64_t rounds = (tiles * splits + cus - 1) / cus, per = (steps + splits - 1) / splits;
      double time = rounds * (times.fixed[c] + per * times.step[c]);
      if (splits > 1) time += 4. + double(s.m) * s.n * splits * 8e-6 / 4.;
      if (least < 0. || time < least) {
        least = time;
        best = {c, splits};
      }
    }
  }
  if (forced_splits > 0 && forced_splits <= 32) best.splits = forced_splits;
  return best;
}

// Copies an operand of `rows` rows of `cols` elements to rows of `ld` (whole
// 16-byte vectors), with zeros after the row's own.  A wave copies 64 vectors
// of a row, so that no read waits for another (1021 x 1111 and 1999 x 1111 f16
// 7.4 us, of which a launch is about four; with the copies the product takes 28
// us, through registers without them 59).
struct PadArgs {
  const void* from[2];
  void* to[2];
  int64_t rows[2], cols[2], ld[2];
  uint32_t groups0, groups;  // workgroups of the first operand, and of both
  uint32_t across;  // the launch's, of many_groups
};
__host__ __device__ inline uint32_t pad_pieces(int64_t ld, int esize) {
  return static_cast<uint32_t>((ld * esize + 1023) / 1024);
}
template <typename S>
__global__ __launch_bounds__(256) void pad_kernel(PadArgs p) {
  constexpr int kN = 16 / static_cast<int>(sizeof(S));
  const uint32_t group = static_cast<uint32_t>(group_of_many(p.across));
  if (group >= p.groups) return;
  const int which = group < p.groups0 ? 0 : 1;
  const uint32_t piece = (group - (which ? p.groups0 : 0)) * 4 + (threadIdx.x >> 6);
  const uint32_t per_row = pad_pieces(p.ld[which], sizeof(S));
  const int64_t row = piece / per_row;
  const int64_t c = (int64_t(piece % per_row) * 64 + (threadIdx.x & 63)) * kN;
  if (row >= p.rows[which] || c >= p.ld[which]) return;
  const S* from = static_cast<const S*>(p.from[which]);
  const Bytes16 v = load_chunk(from, p.cols[which], p.rows[which], p.cols[which], row, c);
  i32x4 w;
  __builtin_memcpy(&w, &v, 16);
  *reinterpret_cast<i32x4*>(static_cast<S*>(p.to[which]) + row * p.ld[which] + c) = w;
}

int64_t padded(int64_t n, int esize) { return (n * esize + 15) / 16 * 16 / esize; }

// Operands that cannot go straight to LDS as they are are copied first, to
// rows of whole vectors at the front of the workspace.
struct Padding {
  bool a, b;
  int64_t rows_a, rows_b;
  size_t bytes_a, bytes_b;
  GemmShape shape;  // with the copies' rows
  bool direct;  // the shape then goes straight to LDS
};
Padding plan_padding(const GemmShape& s, int esize, const void* a, const void* b) {
  Padding p = {};
  p.shape = s;
  const auto one = [&](const void* at, bool kc, int64_t n, int64_t& ld, int64_t& rows, size_t& bytes) {
    rows = kc ? n : s.k;
    if (direct_ok(at, ld, esize)) return false;
    ld = padded(kc ? s.k : n, esize);
    bytes = (static_cast<size_t>(rows) * ld * esize + 255) & ~size_t(255);
    return true;
  };
  p.a = one(a, s.a_kc, s.m, p.shape.lda, p.rows_a, p.bytes_a);
  p.b = one(b, s.b_kc, s.n, p.shape.ldb, p.rows_b, p.bytes_b);
  p.direct = direct_ok(nullptr, p.shape.lda, esize) && direct_ok(nullptr, p.shape.ldb, esize);
  return p;
}

template <typename S>
hipError_t launch_pad(const GemmShape& s, const Padding& p, const void*& a, const void*& b,
                      char*& workspace, hipStream_t stream) {
  PadArgs args = {};
  int n = 0;
  const auto one = [&](const void*& from, int64_t rows, int64_t cols, int64_t ld, size_t bytes) {
    args.from[n] = from;
    args.to[n] = workspace;
    args.rows[n] = rows;
    args.cols[n] = cols;
    args.ld[n] = ld;
    from = workspace;
    workspace += bytes;
    ++n;
  };
  if (p.a) one(a, p.rows_a, s.a_kc ? s.k : s.m, p.shape.lda, p.bytes_a);
  if (p.b) one(b, p.rows_b, s.b_kc ? s.k : s.n, p.shape.ldb, p.bytes_b);
  constexpr int kE = sizeof(S);
  const int64_t groups0 = (args.rows[0] * pad_pieces(args.ld[0], kE) + 3) / 4;
  const int64_t groups = groups0 + (args.rows[1] * pad_pieces(args.ld[1], kE) + 3) / 4;
  if (groups == 0) return hipSuccess;
  if (groups >= (int64_t(1) << 30)) return hipErrorInvalidConfiguration;
  args.groups0 = static_cast<uint32_t>(groups0);
  args.groups = static_cast<uint32_t>(groups);
  const dim3 grid = many_groups(groups);
  args.across = grid.x;
  TFMA_LAUNCH("tfma_linear_pad", pad_kernel<S>, grid, dim3(256), 0, stream, args);
  return hipGetLastError();
}

// The caller's workspace; what does not fit is an error, not an overrun (the
// overrides may change between the query and the call).
struct Workspace {
  char* at;
  size_t bytes;
};
size_t sums_bytes(const GemmShape& s, int splits) {
  return splits > 1 ? static_cast<size_t>(splits) * s.m * s.n * sizeof(float) : 0;
}

template <class Op, class Tr, bool kAKC, bool kBKC>
hipError_t launch(const GemmShape& s, DType t, const void* a, const void* b, const LinearEpilogue& e,
                  Workspace ws, hipStream_t stream) {
  constexpr int kE = sizeof(typename Op::S);
  const bool direct = kE == 1 || (direct_ok(a, s.lda, kE) && direct_ok(b, s.ldb, kE));
  if constexpr (kAKC) {
    if (few_rows(s, direct, kE)) {
      const FewPlan p = plan_few(kBKC, s, kE);
      if (sums_bytes(s, p.splits) > ws.bytes) return hipErrorInvalidValue;
      if constexpr (kBKC) {
        if constexpr (kE > 1)  // e4m3: one round of workgroups
          if (p.nj == 2) return launch_few<Op, Tr, true, 2>(s, a, b, e, ws.at, p.splits, stream);
        return launch_few<Op, Tr, true, 1>(s, a, b, e, ws.at, p.splits, stream);
      } else {
        return launch_few<Op, Tr, false, 4>(s, a, b, e, ws.at, p.splits, stream);
      }
    }
  }
  const auto run = [&](const GemmShape& q) {
    const Plan p = plan_direct(t, kE == 1, q);
    if (sums_bytes(q, p.splits) > ws.bytes) return hipErrorInvalidValue;
    switch (p.tag) {
      case k256x256:
        return launch_direct<Op, Tr, kAKC, kBKC, Direct256x256>(q, a, b, e, ws.at, p.splits, stream);
      case k256x128:
        return launch_direct<Op, Tr, kAKC, kBKC, Direct256x128>(q, a, b, e, ws.at, p.splits, stream);
      case k128x128:
        return launch_direct<Op, Tr, kAKC, kBKC, Direct128x128>(q, a, b, e, ws.at, p.splits, stream);
      default:
        return launch_direct<Op, Tr, kAKC, kBKC, Direct64x128>(q, a, b, e, ws.at, p.splits, stream);
    }
  };
  if constexpr (kE == 1) {
    return run(s);
  } else {
    if (direct) return run(s);
    const Padding pad = plan_padding(s, kE, a, b);
    if (pad.direct) {
      const size_t copies = pad.bytes_a + pad.bytes_b;
      if (copies > ws.bytes) return hipErrorInvalidValue;
      ws.bytes -= copies;
      if (const hipError_t err = launch_pad<typename Op::S>(s, pad, a, b, ws.at, stream);
          err != hipSuccess)
        return err;
      return run(pad.shape);
    }
    // Rows of more than 4 MiB.
    const int64_t tiles = ((s.m + kTile - 1) / kTile) * ((s.n + kTile - 1) / kTile);
    if (tiles * kThreads > UINT32_MAX) return hipErrorInvalidConfiguration;
    TFMA_LAUNCH("tfma_linear", (linear_kernel<Op, Tr, kAKC, kBKC>),
                dim3(static_cast<uint32_t>(tiles)), dim3(kThreads), 0, stream, s, a, b, e);
    return hipGetLastError();
  }
}

template <class Op, class Tr>
hipError_t launch_layout(const GemmShape& s, DType t, const void* a, const void* b,
                         const LinearEpilogue& e, Workspace ws, hipStream_t stream) {
  if (s.a_kc && s.b_kc) return launch<Op, Tr, true, true>(s, t, a, b, e, ws, stream);
  if (s.a_kc) return launch<Op, Tr, true, false>(s, t, a, b, e, ws, stream);
  return launch<Op, Tr, false, false>(s, t, a, b, e, ws, stream);
}

// ---------------------------------------------------------------------------
// dz = dy act'(z), and the sums of its columns.  A thread owns eight
// columns; a workgroup's four waves take rows in turn and join their sums in
// LDS; the workgroups of one column strip leave their sums in `partial` [row
// groups, n], which a second kernel adds in order.  Up to 64 rows stay with one
// workgroup a strip, whose sums are the result.
// Bound by HBM, with the slope's arithmetic beside it.  Where the workgroups
// fill the chip a wave takes one row at a time, in registers for eight waves a
// SIMD, and z, which the forward pass wrote long ago, leaves the caches to dz:
// 8192 x 8192 bf16 83 us (4.9 TB/s) against 94 with four rows at a time.
// Where they do not, four rows at a time hide the loads' latency.
// dz is rounded to the tensors' type, which the products that follow take; the
// bias' sums are of the unrounded values.
// ---------------------------------------------------------------------------
constexpr int kDzCols = 64 * 8;

// kStream: the lines need not stay in the caches.
template <class V, bool kStream, typename S>
__device__ inline V load_eight(const S* p) {
  if constexpr (!kStream) return *reinterpret_cast<const V*>(p);
  typedef uint32_t Words __attribute__((ext_vector_type(sizeof(V) / 4), aligned(sizeof(S))));
  const Words w = __builtin_nontemporal_load(reinterpret_cast<const Words*>(p));
  V v;
  __builtin_memcpy(&v, &w, sizeof(v));
  return v;
}

template <class Tr, int kAtOnce>
__global__ __launch_bounds__(256) void dz_kernel(int64_t m, int64_t n, int act, int64_t rows_per,
                                                 const void* dy_, const void* z_, void* dz_,
                                                 int64_t ldz, float* partial, void* db) {
  using S = typename Tr::S;
  constexpr bool kStream = kAtOnce == 1;
  const S* dy = static_cast<const S*>(dy_);
  const S* z = static_cast<const S*>(z_);
  S* dz = static_cast<S*>(dz_);
  __shared__ float sums[4][kDzCols];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = int64_t(blockIdx.x) * kDzCols + lane * 8;
  const int64_t r0 = int64_t(blockIdx.y) * rows_per;
  const int64_t r1 = r0 + rows_per < m ? r0 + rows_per : m;
  const int have = n - c >= 8 ? 8 : (n > c ? static_cast<int>(n - c) : 0);
  float acc[8] = {};
  struct __attribute__((packed, aligned(1))) Eight { S v[8]; };
  if (have > 0) {
    for (int64_t r = r0 + wave; r < r1; r += 4 * kAtOnce) {
      Eight d[kAtOnce] = {}, zz[kAtOnce] = {};
      const int rows = r1 - r > 4 * (kAtOnce - 1) ? kAtOnce : static_cast<int>((r1 - r + 3) / 4);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (u >= rows) break;
        const int64_t at = (r + 4 * u) * n + c;
        if (have == 8) {
          d[u] = *reinterpret_cast<const Eight*>(dy + at);
          if (z) zz[u] = load_eight<Eight, kStream>(z + at);
        } else {
#pragma unroll
          for (int j = 0; j < 7; ++j) {
            if (j >= have) break;
            d[u].v[j] = dy[at + j];
            if (z) zz[u].v[j] = z[at + j];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (u >= rows) break;
        Eight o;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float v = Tr::ld(d[u].v[j]);
          if (z) v *= activate_grad<sizeof(S) == 4>(Tr::ld(zz[u].v[j]), act);
          acc[j] += v;
          o.v[j] = j < have ? Tr::st(v) : S(0);
        }
        // Zeros after the row's own columns, as far as dz's rows go.
        if (dz) {
          S* to = dz + (r + 4 * u) * ldz + c;
          if (c + 8 <= ldz) {
            *reinterpret_cast<Eight*>(to) = o;
          } else {
#pragma unroll
            for (int j = 0; j < 7; ++j)
              if (c + j < ldz) to[j] = o.v[j];
          }
        }
      }
    }
  }
  if (!db) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[wave][lane * 8 + j] = acc[j];
  __syncthreads();
  for (int i = threadIdx.x; i < kDzCols; i += 256) {
    const int64_t col = int64_t(blockIdx.x) * kDzCols + i;
    if (col >= n) continue;
    const float sum = (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
    if (gridDim.y == 1)
      static_cast<S*>(db)[col] = Tr::st(sum);
    else
      partial[int64_t(blockIdx.y) * n + col] = sum;
  }
}

// A workgroup adds 64 columns, its sixteen waves taking groups in turn.
template <class Tr>
__global__ __launch_bounds__(1024) void column_sums_kernel(int64_t groups, int64_t n,
                                                           const float* partial, void* out) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = int64_t(blockIdx.x) * 64 + lane;
  float s = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int64_t g = wave; g < groups; g += 16) s += partial[g * n + c];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= n) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += sums[w][lane];
  static_cast<typename Tr::S*>(out)[c] = Tr::st(s);
}

int64_t dz_groups(int64_t m, int64_t n) {
  const int64_t strips = n > 0 ? (n + kDzCols - 1) / kDzCols : 1;
  const int64_t want = (2048 + strips - 1) / strips;
  const int64_t most = m <= 64 ? 1 : (m + 15) / 16;
  return want < most ? want : (most > 0 ? most : 1);
}

template <class Tr>
hipError_t launch_dz(int64_t m, int64_t n, int act, const void* dy, const void* z, void* dz,
                     int64_t ldz, float* partial, void* db, hipStream_t stream) {
  const int64_t groups = dz_groups(m, n);
  const int64_t rows_per = (m + groups - 1) / groups;
  const int64_t strips = (n + kDzCols - 1) / kDzCols;
  if (m > 0) {
    const dim3 grid(static_cast<uint32_t>(strips), static_cast<uint32_t>(groups));
    if (strips * groups >= 4 * DeviceCUs())
      TFMA_LAUNCH("tfma_linear_dz", (dz_kernel<Tr, 1>), grid, dim3(256), 0, stream, m, n, act,
                  rows_per, dy, z, dz, ldz, partial, db);
    else
      TFMA_LAUNCH("tfma_linear_dz", (dz_kernel<Tr, 4>), grid, dim3(256), 0, stream, m, n, act,
                  rows_per, dy, z, dz, ldz, partial, db);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  if (!db || (m > 0 && groups == 1)) return hipSuccess;
  TFMA_LAUNCH("tfma_linear_db", column_sums_kernel<Tr>, dim3(static_cast<uint32_t>((n + 63) / 64)),
              dim3(1024), 0, stream, m > 0 ? groups : int64_t(0), n, partial, db);
  return hipGetLastError();
}

}  // namespace

size_t LinearWorkspaceBytes(DType t, bool e4m3, const GemmShape& s, const void* a, const void* b) {
  if (s.m == 0 || s.n == 0) return 0;
  const int esize = e4m3 ? 1 : DTypeBytes(t);
  const bool direct = e4m3 || (direct_ok(a, s.lda, esize) && direct_ok(b, s.ldb, esize));
  if (few_rows(s, direct, esize)) return sums_bytes(s, plan_few(s.b_kc, s, esize).splits);
  if (direct) return sums_bytes(s, plan_direct(t, e4m3, s).splits);
  const Padding p = plan_padding(s, esize, a, b);
  return p.direct ? p.bytes_a + p.bytes_b + sums_bytes(s, plan_direct(t, false, p.shape).splits) : 0;
}

hipError_t LaunchLinear(DType t, const GemmShape& s, const void* a, const void* b,
                        const LinearEpilogue& e, void* workspace, size_t workspace_bytes,
                        hipStream_t stream) {
  if (s.m == 0 || s.n == 0) return hipSuccess;
  const Workspace ws = {static_cast<char*>(workspace), workspace ? workspace_bytes : 0};
  switch (t) {
    case DType::kF32: return launch_layout<OpF32, TF32>(s, t, a, b, e, ws, stream);
    case DType::kF16: return launch_layout<OpF16, TF16>(s, t, a, b, e, ws, stream);
    default: return launch_layout<OpBF16, TBF16>(s, t, a, b, e, ws, stream);
  }
}

hipError_t LaunchLinear8(DType t, const GemmShape& s, const void* a, const void* b,
                         const LinearEpilogue& e, void* workspace, size_t workspace_bytes,
                        hipStream_t stream) {
  if (s.m == 0 || s.n == 0) return hipSuccess;
  const Workspace ws = {static_cast<char*>(workspace), workspace ? workspace_bytes : 0};
  return t == DType::kF16 ? launch<OpFP8, TF16, true, true>(s, t, a, b, e, ws, stream)
                          : launch<OpFP8, TBF16, true, true>(s, t, a, b, e, ws, stream);
}

bool LinearDirectOk(DType t, const void* p, int64_t ld) { return direct_ok(p, ld, DTypeBytes(t)); }
int64_t LinearPadded(DType t, int64_t n) { return padded(n, DTypeBytes(t)); }

size_t LinearDzPartialBytes(int64_t m, int64_t n) {
  return static_cast<size_t>(dz_groups(m, n)) * static_cast<size_t>(n) * sizeof(float);
}

hipError_t LaunchLinearDz(DType t, int64_t m, int64_t n, int act, const void* dy, const void* z,
                          void* dz, int64_t ldz, float* partial, void* db, hipStream_t stream) {
  if (n == 0) return hipSuccess;
  switch (t) {
    case DType::kF32: return launch_dz<TF32>(m, n, act, dy, z, dz, ldz, partial, db, stream);
    case DType::kF16: return launch_dz<TF16>(m, n, act, dy, z, dz, ldz, partial, db, stream);
    default: return launch_dz<TBF16>(m, n, act, dy, z, dz, ldz, partial, db, stream);
  }
}

}  // namespace tfma
