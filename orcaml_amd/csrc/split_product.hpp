// fp32 products on the bf16 matrix instructions.
//
// An fp32 value is the sum of three bf16 values: h is its upper half (8 significant bits,
// truncated, so a large finite value never rounds to infinity), m is x - h (exact) rounded to
// the nearest bf16, l is what is left (exact: at most 8 bits).  A product of two such sums
// has nine terms; the six of order 1, 2^-8 and 2^-16 (hh, hm + mh, hl + mm + lh) are taken and
// the other three left out: each is below 2^-23 of the product and centred on zero, so less
// than the rounding of an fp32 sum.  The instructions add in fp32.  Six bf16 products take
// 6 / 16 of the time of one on the fp32 instructions (157 against 2516 TFLOP/s).  (Publicly
// described, e.g. Henry, Tang and Heinecke 2019, "Leveraging the bfloat16 Artificial
// Intelligence Datatype For Higher-Precision Computations".)
// A value of an 8-bit checkpoint is one bf16 value, so a product with it has three terms.
//
// Operands are read in fp32 (or 8 bits) and taken apart on their way into LDS: no extra
// pass over memory and no copy of them.  LDS holds, for each of the three planes, 16-byte
// units of 8 consecutive k of one row, [k / 8][row], which is what a lane of the 32x32x16
// instruction takes.  The rows of one k / 8 are followed by padding, 8 units for all k / 8
// together, so that the stores of a k-fast operand (neighbouring lanes hold neighbouring
// k / 8) fall into different banks.
//
// Infinities and NaN: inf - inf in the split, and inf times an m or l of zero, make NaN where
// fp32 has an infinity.  So a block that ends with a value that is not finite multiplies its tile again
// on the fp32 instructions, from the same LDS layout (h + m + l is x; an infinity or NaN is
// kept in h alone).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "act8.hpp"
#include "activation.hpp"
#include "slab.hpp"

namespace orca_hip {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float acc32 __attribute__((ext_vector_type(16)));  // a lane's part of a 32 x 32 block
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// An operand: `rows` rows (the M or N side) of k values.
struct ProductOperand {
  const void* p;
  int64_t ld;             // elements between rows (k-fast) or between k values (k-slow)
  int rows;
  const uint8_t* scales;  // 8-bit: step bytes [rows / 32][lds]
  int64_t lds;
  // LoadSlopeFast, LoadSlopeSlow: the operand is p * act'(z), z of p's shape, in fp32 or as a checkpoint
  int act;
  const float* z;
  int64_t ldz;
  Act8 z8;
};

__device__ __forceinline__ uint32_t upper_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
__device__ __forceinline__ uint32_t round_pair(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{a, b}, bf16x2));
}
__device__ __forceinline__ float low_half(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high_half(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// A unit of 8 values on its way to LDS, a piece of work of five or six instructions at a time (what the
// matrix unit hides behind one of its own): pieces 2 j and 2 j + 1 split pair j, piece 8 stores the
// three planes (`plane` units apart).  SAFE: infinities and NaN stay in h, with m = l = 0.
template <bool SAFE>
struct SplitUnit {
  static constexpr int PIECES = 9;
  u32x4 h, m, l;
  float ra, rb;
  __device__ __forceinline__ void piece(int k, const float (&v)[8], u32x4* dst, int plane) {
    if (k == 8) {
      dst[0] = h;
      dst[plane] = m;
      dst[2 * plane] = l;
      return;
    }
    const int j = k / 2;
    const float a = v[2 * j], b = v[2 * j + 1];
    if (k % 2 == 0) {
      if (SAFE) {
        h[j] = upper_halves(a != a ? 0x7fc00000u : __float_as_uint(a), b != b ? 0x7fc00000u : __float_as_uint(b));
        ra = __builtin_isfinite(a) ? a - low_half(h[j]) : 0.0f;
        rb = __builtin_isfinite(b) ? b - high_half(h[j]) : 0.0f;
      } else {
        h[j] = upper_halves(__float_as_uint(a), __float_as_uint(b));
        ra = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u);
        rb = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
      }
    } else {
      m[j] = round_pair(ra, rb);
      l[j] = round_pair(ra - low_half(m[j]), rb - high_half(m[j]));
    }
  }
};

constexpr int unit_pitch(int rows, int kh) { return rows + 8 / kh; }

// Loaders: a stage is BK k values of ROWS rows, one unit of 8 k values of one row per thread.  Rows past
// the operand's last are the last one again (what they give is never stored); k values past the range are
// zero (tail).  piece(k) for k in 0 .. 8 takes the loaded unit to LDS.  The product comes out 1 / SCALE
// times too large, unless SAFE.

// k is contiguous: a unit is 32 bytes, at any alignment of its floats.
template <int ROWS, int BK, int THREADS>
struct LoadKFast {
  static constexpr float SCALE = 1.0f;
  static constexpr int PLANES = 3, KH = BK / 8, PITCH = unit_pitch(ROWS, KH), UNITS = PLANES * KH * PITCH;
  static_assert(ROWS * KH == THREADS, "a unit per thread");
  const float* p;
  float v[8];

  __device__ __forceinline__ void init(const ProductOperand& op, int row0, int64_t k0) {
    const int u = threadIdx.x;
    p = static_cast<const float*>(op.p) + (int64_t)min(row0 + u / KH, op.rows - 1) * op.ld + k0 + u % KH * 8;
  }
  __device__ __forceinline__ void load() {
    const floatx4 a = *reinterpret_cast<const floatx4_u*>(p), b = *reinterpret_cast<const floatx4_u*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
    p += BK;
  }
  __device__ __forceinline__ void load_tail(int left) {
    const int k = threadIdx.x % KH * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < left ? p[j] : 0.0f;
  }
  template <bool SAFE>
  __device__ __forceinline__ void piece(int k, SplitUnit<SAFE>& u, u32x4* s) const {
    u.piece(k, v, s + threadIdx.x % KH * PITCH + threadIdx.x / KH, KH * PITCH);
  }
};

// Rows are contiguous and k values lie op.ld apart: a wave reads 64 neighbouring rows of one k
// at a time, and the 8 that a thread collects are a unit, so the transpose costs nothing.
template <int ROWS, int BK, int THREADS>
struct LoadKSlow {
  static constexpr float SCALE = 1.0f;
  static constexpr int PLANES = 3, KH = BK / 8, PITCH = unit_pitch(ROWS, KH), UNITS = PLANES * KH * PITCH;
  static_assert(ROWS * KH == THREADS && ROWS % 64 == 0, "a unit per thread, whole waves per k");
  const char* base;  // uniform: the first of this wave's 8 k values
  int64_t ld;        // bytes
  uint32_t col;      // bytes
  float v[8];

  static __device__ __forceinline__ int kh() { return __builtin_amdgcn_readfirstlane(threadIdx.x / ROWS); }
  __device__ __forceinline__ void init(const ProductOperand& op, int row0, int64_t k0) {
    ld = op.ld * 4;
    base = static_cast<const char*>(op.p) + (k0 + kh() * 8) * ld;
    col = (uint32_t)min(row0 + (int)threadIdx.x % ROWS, op.rows - 1) * 4u;
  }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = *reinterpret_cast<const float*>(base + j * ld + col);
    base += BK * ld;
  }
  __device__ __forceinline__ void load_tail(int left) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = kh() * 8 + j < left ? *reinterpret_cast<const float*>(base + j * ld + col) : 0.0f;
  }
  template <bool SAFE>
  __device__ __forceinline__ void piece(int k, SplitUnit<SAFE>& u, u32x4* s) const {
    u.piece(k, v, s + threadIdx.x / ROWS * PITCH + threadIdx.x % ROWS, KH * PITCH);
  }
};

// A checkpoint read the same way: k values are its rows.  One plane, no split.
template <int ROWS, int BK, int THREADS>
struct LoadCodes {
  static constexpr float SCALE = 1.0f / 64;
  static constexpr int PLANES = 1, KH = BK / 8, PITCH = unit_pitch(ROWS, KH), UNITS = PLANES * KH * PITCH;
  static_assert(ROWS * KH == THREADS && ROWS % 64 == 0, "a unit per thread, whole waves per k");
  const char* base;     // uniform
  int64_t ld;
  uint32_t col;
  const uint8_t* step;  // of this thread's 8 k values
  int v[8];
  u32x2 b;

  static __device__ __forceinline__ int kh() { return __builtin_amdgcn_readfirstlane(threadIdx.x / ROWS); }
  __device__ __forceinline__ void init(const ProductOperand& op, int row0, int64_t k0) {
    ld = op.ld;
    base = static_cast<const char*>(op.p) + (k0 + kh() * 8) * ld;
    col = (uint32_t)min(row0 + (int)threadIdx.x % ROWS, op.rows - 1);
    // k0 and kh() * 8 are multiples of 8, a group's bytes fill its row to a multiple of 16
    step = op.scales + (int64_t)(col / kAct8Group) * op.lds + k0 + kh() * 8;
  }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = *reinterpret_cast<const int8_t*>(base + j * ld + col);
    b = *reinterpret_cast<const u32x2*>(step);
    step += BK;
    base += BK * ld;
  }
  __device__ __forceinline__ void load_tail(int left) {
    left -= kh() * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? *reinterpret_cast<const int8_t*>(base + j * ld + col) : 0;
    // the step bytes of rows past the last are whatever they are: 0 instead
    b = u32x2{0, 0};
    if (left > 0) {
      b = *reinterpret_cast<const u32x2*>(step);
      if (left < 8) {
        const uint64_t keep = (1ull << (8 * left)) - 1;
        b[0] &= (uint32_t)keep;
        b[1] &= (uint32_t)(keep >> 32);
      }
    }
  }
  template <bool SAFE>
  __device__ __forceinline__ void piece(int k, SplitUnit<SAFE>& u, u32x4* s) const {
    // The step byte as an exponent is 64 times the step, and an infinity for a group that is not finite:
    // its codes are zero, so its values NaN.  Where that overflows the product is not finite either, and
    // the block multiplies again with SAFE.
    auto value = [&](int j) {
      const uint32_t w = b[j / 4];
      if (SAFE) return __float_as_uint((float)v[j] * act8_step((w >> (8 * (j % 4))) & 255u));
      const uint32_t e = (j % 4 < 3 ? w << (23 - 8 * (j % 4)) : w >> 1) & 0x7f800000u;
      return __float_as_uint((float)v[j] * __uint_as_float(max(e, 7u << 23)));  // act8_step's least
    };
    if (k == 8)
      s[threadIdx.x / ROWS * PITCH + threadIdx.x % ROWS] = u.h;
    else if (k % 2 == 0)
      u.ra = __uint_as_float(value(k));
    else
      u.h[k / 2] = upper_halves(__float_as_uint(u.ra), value(k));
  }
};

// dz = dy * act'(z) on its way into a product, for backwards too small to make it in a launch of its own.  The
// slopes of a unit are taken with its first piece.
struct SlopeUnit {
  float v[8];
  uint32_t z[8];  // fp32 bits, or a code in the lowest byte and its step byte above
};
__device__ __forceinline__ float slope_code(uint32_t z) { return (float)(int8_t)z * act8_step(z >> 8); }

// k (dy's columns) is contiguous.  8 columns from a multiple of 8 on lie in one group of a checkpoint.
template <int ROWS, int BK, int THREADS>
struct LoadSlopeFast {
  static constexpr float SCALE = 1.0f;
  static constexpr int PLANES = 3, KH = BK / 8, PITCH = unit_pitch(ROWS, KH), UNITS = PLANES * KH * PITCH;
  static_assert(ROWS * KH == THREADS, "a unit per thread");
  const float* p;
  const float* z;
  const int8_t* codes;
  const uint8_t* scales;
  int64_t lds;
  int64_t k;
  int act;
  SlopeUnit u;

  __device__ __forceinline__ void init(const ProductOperand& op, int row0, int64_t k0) {
    const int64_t row = min(row0 + (int)threadIdx.x / KH, op.rows - 1);
    k = k0 + threadIdx.x % KH * 8;
    act = op.act;
    p = static_cast<const float*>(op.p) + row * op.ld + k;
    z = op.z + row * op.ldz + k;
    codes = op.z8.codes ? op.z8.codes + row * op.z8.cols + k : nullptr;
    scales = op.z8.scales + row;
    lds = op.z8.ld;
  }
  __device__ __forceinline__ void load() { fetch<false>(BK); }
  __device__ __forceinline__ void load_tail(int left) { fetch<true>(left); }
  template <bool TAIL>
  __device__ __forceinline__ void fetch(int left) {
    left -= threadIdx.x % KH * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) u.v[j] = !TAIL || j < left ? p[j] : 0.0f;
    if (act != ORCA_HIP_ACT_NONE && codes) {
      const uint32_t step = !TAIL || left > 0 ? scales[k / (int64_t)kAct8Group * lds] : 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) u.z[j] = !TAIL || j < left ? (uint8_t)codes[j] | step << 8 : 0u;
      codes += BK;
    } else if (act != ORCA_HIP_ACT_NONE) {
#pragma unroll
      for (int j = 0; j < 8; ++j) u.z[j] = !TAIL || j < left ? __float_as_uint(z[j]) : 0u;
      z += BK;
    }
    p += BK;
    k += BK;
  }
  template <bool SAFE>
  __device__ __forceinline__ void piece(int i, SplitUnit<SAFE>& unit, u32x4* s) {
    if (i == 0 && act != ORCA_HIP_ACT_NONE) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = codes ? slope_code(u.z[j]) : __uint_as_float(u.z[j]);
      activation_slopes<8>(act, f, u.v);
    }
    unit.piece(i, u.v, s + threadIdx.x % KH * PITCH + threadIdx.x / KH, KH * PITCH);
  }
};

// k values are dy's rows.
template <int ROWS, int BK, int THREADS>
struct LoadSlopeSlow {
  static constexpr float SCALE = 1.0f;
  static constexpr int PLANES = 3, KH = BK / 8, PITCH = unit_pitch(ROWS, KH), UNITS = PLANES * KH * PITCH;
  static_assert(ROWS * KH == THREADS && ROWS % 64 == 0, "a unit per thread, whole waves per k");
  const float* p;
  const float* z;
  const int8_t* codes;
  const uint8_t* scales;
  int64_t ld, ldz, ldc;
  int act;
  SlopeUnit u;

  __device__ __forceinline__ void init(const ProductOperand& op, int row0, int64_t k0) {
    const int64_t col = min(row0 + (int)threadIdx.x % ROWS, op.rows - 1), k = k0 + threadIdx.x / ROWS * 8;
    act = op.act;
    ld = op.ld;
    ldz = op.ldz;
    ldc = op.z8.cols;
    p = static_cast<const float*>(op.p) + k * ld + col;
    z = op.z + k * ldz + col;
    codes = op.z8.codes ? op.z8.codes + k * ldc + col : nullptr;
    scales = op.z8.scales + col / (int64_t)kAct8Group * op.z8.ld + k;
  }
  __device__ __forceinline__ void load() { fetch<false>(BK); }
  __device__ __forceinline__ void load_tail(int left) { fetch<true>(left); }
  template <bool TAIL>
  __device__ __forceinline__ void fetch(int left) {
    left -= threadIdx.x / ROWS * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) u.v[j] = !TAIL || j < left ? p[j * ld] : 0.0f;
    if (act != ORCA_HIP_ACT_NONE && codes) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        u.z[j] = !TAIL || j < left ? (uint8_t)codes[j * ldc] | (uint32_t)scales[j] << 8 : 0u;
      codes += BK * ldc;
      scales += BK;
    } else if (act != ORCA_HIP_ACT_NONE) {
#pragma unroll
      for (int j = 0; j < 8; ++j) u.z[j] = !TAIL || j < left ? __float_as_uint(z[j * ldz]) : 0u;
      z += BK * ldz;
    }
    p += BK * ld;
  }
  template <bool SAFE>
  __device__ __forceinline__ void piece(int i, SplitUnit<SAFE>& unit, u32x4* s) {
    if (i == 0 && act != ORCA_HIP_ACT_NONE) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = codes ? slope_code(u.z[j]) : __uint_as_float(u.z[j]);
      activation_slopes<8>(act, f, u.v);
    }
    unit.piece(i, u.v, s + threadIdx.x / ROWS * PITCH + threadIdx.x % ROWS, KH * PITCH);
  }
};

// BM x BN tiles by WM x WN waves, stages of BK k values, OCC blocks per CU.
template <int BM_, int BN_, int WM_, int WN_, int BK_, int OCC_>
struct ProductTile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = BK_, OCC = OCC_;
  static constexpr int THREADS = WM * WN * 64, FM = BM / WM / 32, FN = BN / WN / 32;
};

// A unit of work: FN blocks of a wave, 16 k values.  The first operand of the instruction is B, so a lane
// holds row lane % 32 of A's and, in element r, column (r / 4) * 8 + (lane / 32) * 4 + r % 4 of B's
// 32: four neighbouring columns of C in four registers.
// After matrix instruction g (of FN * terms), work(g) adds other work, which runs while the matrix unit is
// busy: about five vector instructions hide behind one of its 32 cycles.  Nothing moves across:
// the compiler left to itself puts all other work before the first of them.
template <class LA>
constexpr int terms() {
  return LA::PLANES == 3 ? 6 : 3;
}
template <int FN, class LA, class LB, bool FP32, class Work>
__device__ __forceinline__ void product_unit(const u32x4 (&a)[LA::PLANES], const u32x4 (&b)[FN][LB::PLANES],
                                             acc32 (&acc)[FN], Work work) {
  if constexpr (FP32) {
    auto whole = [](const u32x4* f, int planes, int e) {
      float x = 0.0f;
      for (int p = 0; p < planes; ++p) x = x + (e % 2 ? high_half(f[p][e / 2]) : low_half(f[p][e / 2]));
      return x;
    };
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(whole(b[j], LB::PLANES, e), whole(a, LA::PLANES, e), acc[j], 0,
                                                      0, 0);
  } else {
    // the smallest terms first
    constexpr int PA[6] = {0, 2, 1, 0, 1, 0}, PB[6] = {2, 0, 1, 1, 0, 0}, PB1[3] = {2, 1, 0};
#pragma unroll
    for (int t = 0; t < terms<LA>(); ++t) {
      const int pa = LA::PLANES == 3 ? PA[t] : 0, pb = LA::PLANES == 3 ? PB[t] : PB1[t];
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b[j][pb]),
                                                         __builtin_bit_cast(bf16x8, a[pa]), acc[j], 0, 0, 0);
        work(t * FN + j);
      }
    }
  }
}

// Unit u's parts of a stage: row block u % FM of k step u / FM, and the k step's FN column blocks.
template <class T, class LA>
__device__ __forceinline__ void read_a(const u32x4* __restrict__ s, int ra, int u, u32x4 (&a)[LA::PLANES]) {
  const int kh = 2 * (u / T::FM) + ((threadIdx.x & 63) >> 5);
#pragma unroll
  for (int p = 0; p < LA::PLANES; ++p) a[p] = s[(p * (T::BK / 8) + kh) * LA::PITCH + ra + 32 * (u % T::FM)];
}
template <class T, class LB>
__device__ __forceinline__ void read_b(const u32x4* __restrict__ s, int rb, int step, u32x4 (&b)[T::FN][LB::PLANES]) {
  const int kh = 2 * step + ((threadIdx.x & 63) >> 5);
#pragma unroll
  for (int p = LB::PLANES - 1; p >= 0; --p)
#pragma unroll
    for (int j = 0; j < T::FN; ++j) b[j][p] = s[(p * (T::BK / 8) + kh) * LB::PITCH + rb + 32 * j];
}

// A whole stage, its fragments read one unit ahead.
template <class T, class LA, class LB, bool FP32, class Work>
__device__ __forceinline__ void product_stage(const u32x4* __restrict__ sa, const u32x4* __restrict__ sb, int ra,
                                              int rb, acc32 (&acc)[T::FM][T::FN], Work work) {
  constexpr int UNITS = T::BK / 16 * T::FM;
  u32x4 a[2][LA::PLANES], b[2][T::FN][LB::PLANES];
  read_a<T, LA>(sa, ra, 0, a[0]);
  read_b<T, LB>(sb, rb, 0, b[0]);
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    if (u + 1 < UNITS) {
      if (u % T::FM == T::FM - 1) read_b<T, LB>(sb, rb, u / T::FM + 1, b[(u / T::FM + 1) & 1]);
      read_a<T, LA>(sa, ra, u + 1, a[(u + 1) & 1]);
    }
    product_unit<T::FN, LA, LB, FP32>(a[u & 1], b[u / T::FM & 1], acc[u % T::FM],
                                      [&](int g) { work(u * T::FN * terms<LA>() + g); });
  }
}

// acc += the tile's product over k in [k0, k1).  Two LDS buffers, one barrier a stage.  While stage t is
// multiplied, t + 1 goes from registers to the other buffer, each operand as soon as it may, and its
// registers take the loads of t + 2, which so have most of a stage to arrive.
template <class T, class LA, class LB, bool FP32>
__device__ __forceinline__ void product_loop(const ProductOperand& A, const ProductOperand& B, int m0, int n0,
                                             int64_t k0, int64_t k1, u32x4* __restrict__ smem,
                                             acc32 (&acc)[T::FM][T::FN]) {
  constexpr int STAGE = LA::UNITS + LB::UNITS, PIECES = SplitUnit<FP32>::PIECES;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int ra = wave / T::WN * (T::FM * 32) + (lane & 31), rb = wave % T::WN * (T::FN * 32) + (lane & 31);
  LA la;
  LB lb;
  la.init(A, m0, k0);
  lb.init(B, n0, k0);
  SplitUnit<FP32> ua, ub;
  const int full = (int)((k1 - k0) / T::BK), left = (int)((k1 - k0) % T::BK), n = full + (left > 0);
  auto load = [&](int t) {
    if (t < full) {
      la.load();
      lb.load();
    } else if (t < n) {
      la.load_tail(left);
      lb.load_tail(left);
    }
  };
  auto piece = [&](int k, u32x4* __restrict__ s) {  // A's, then B's
    if (k < PIECES)
      la.piece(k, ua, s);
    else
      lb.piece(k - PIECES, ub, s + LA::UNITS);
  };
  auto store = [&](int t) {
#pragma unroll
    for (int k = 0; k < 2 * PIECES; ++k) piece(k, smem + (t & 1) * STAGE);
  };
  if (n == 0) return;
  load(0);
  store(0);
  load(1);
  __syncthreads();
  int t = 0;
  if constexpr (!FP32) {
    // A stage whose next two are full ones: without a branch, its other work among its matrix
    // instructions, a piece each from a sixth of them on
    constexpr int GROUPS = T::BK / 16 * T::FM * T::FN * terms<LA>(), FIRST = GROUPS / 6;
    constexpr int EVERY = (GROUPS - FIRST) / (2 * PIECES) > 1 ? (GROUPS - FIRST) / (2 * PIECES) : 1;
    for (; t + 2 < full; ++t) {
      const u32x4* rd = smem + (t & 1) * STAGE;
      u32x4* wr = smem + ((t + 1) & 1) * STAGE;
      product_stage<T, LA, LB, false>(rd, rd + LA::UNITS, ra, rb, acc, [&](int g) {
#pragma unroll
        for (int k = 0; k < 2 * PIECES; ++k)
          if (min(FIRST + k * EVERY, GROUPS - 1) == g) {
            piece(k, wr);
            if (k == PIECES - 1) la.load();
            if (k == 2 * PIECES - 1) lb.load();
          }
        __builtin_amdgcn_sched_barrier(0);
      });
      __syncthreads();
    }
  }
  for (; t < n; ++t) {
    if (t + 1 < n) store(t + 1);
    load(t + 2);
    const u32x4* s = smem + (t & 1) * STAGE;
    product_stage<T, LA, LB, FP32>(s, s + LA::UNITS, ra, rb, acc, [](int) {});
    __syncthreads();
  }
}

// The product, again on the fp32 instructions if it holds what is not finite.
template <class T, class LA, class LB>
__device__ __forceinline__ void product(const ProductOperand& A, const ProductOperand& B, int m0, int n0, int64_t k0,
                                        int64_t k1, u32x4* __restrict__ smem, acc32 (&acc)[T::FM][T::FN]) {
  auto run = [&](auto fp32) {
#pragma unroll
    for (int i = 0; i < T::FM; ++i)
#pragma unroll
      for (int j = 0; j < T::FN; ++j) acc[i][j] = acc32{};
    product_loop<T, LA, LB, decltype(fp32)::value>(A, B, m0, n0, k0, k1, smem, acc);
  };
  run(std::false_type());
  bool off = false;
#pragma unroll
  for (int i = 0; i < T::FM; ++i)
#pragma unroll
    for (int j = 0; j < T::FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        off |= !(fabsf(acc[i][j][r]) < __builtin_inff());
        if (LA::SCALE != 1.0f) acc[i][j][r] = acc[i][j][r] * LA::SCALE;
      }
  if (__syncthreads_or(off)) run(std::true_type());
}

}  // namespace
}  // namespace orca_hip
