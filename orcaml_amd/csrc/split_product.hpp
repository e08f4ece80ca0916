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
// instruction takes.  The rows of one k / 8 are followed by two units of padding, so that
// the stores of a k-fast operand (neighbouring lanes hold neighbouring k / 8) fall into
// different banks.
//
// Infinities and NaN: inf - inf in the split, and inf times an m or l of zero, make NaN where
// fp32 has an infinity.  So a block that ends with a NaN anywhere multiplies its tile again
// on the fp32 instructions, from the same LDS layout (h + m + l is x; an infinity or NaN is
// kept in h alone).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "act8.hpp"
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
};

__device__ __forceinline__ uint32_t upper_halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
__device__ __forceinline__ uint32_t round_pair(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{a, b}, bf16x2));
}
__device__ __forceinline__ float low_half(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high_half(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// The three planes of a pair of values.  SAFE: infinities and NaN stay in h, with m = l = 0.
template <bool SAFE>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& h, uint32_t& m, uint32_t& l) {
  if (SAFE) {
    const bool fa = __builtin_isfinite(a), fb = __builtin_isfinite(b);
    const uint32_t ua = a != a ? 0x7fc00000u : __float_as_uint(a), ub = b != b ? 0x7fc00000u : __float_as_uint(b);
    h = upper_halves(ua, ub);
    const float ra = fa ? a - low_half(h) : 0.0f, rb = fb ? b - high_half(h) : 0.0f;
    m = round_pair(ra, rb);
    l = round_pair(ra - low_half(m), rb - high_half(m));
    return;
  }
  h = upper_halves(__float_as_uint(a), __float_as_uint(b));
  const float ra = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u);
  const float rb = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
  m = round_pair(ra, rb);
  l = round_pair(ra - low_half(m), rb - high_half(m));
}

// 8 values to the unit at `dst` of each plane (`plane` units apart).
template <bool SAFE>
__device__ __forceinline__ void store_split(const float (&v)[8], u32x4* dst, int plane) {
  u32x4 h, m, l;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t a, b, c;
    split_pair<SAFE>(v[2 * j], v[2 * j + 1], a, b, c);
    h[j] = a;
    m[j] = b;
    l[j] = c;
  }
  dst[0] = h;
  dst[plane] = m;
  dst[2 * plane] = l;
}

constexpr int unit_pitch(int rows) { return rows + 2; }

// Loaders: a stage is BK k values of ROWS rows, taken as units of 8 k values of one row,
// UN units per thread.  Rows past the operand's last are the last one again (what they give
// is never stored); k values past the range are zero (tail).

// k is contiguous: a unit is 32 bytes, at any alignment of its floats.
template <int ROWS, int BK, int THREADS>
struct LoadKFast {
  static constexpr int PLANES = 3, KH = BK / 8, UN = ROWS * KH / THREADS, PITCH = unit_pitch(ROWS);
  static constexpr int UNITS = PLANES * KH * PITCH;
  static_assert(ROWS * KH % THREADS == 0, "whole units per thread");
  const float* p[UN];
  float v[UN][8];

  __device__ __forceinline__ void init(const ProductOperand& op, int row0, int64_t k0) {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int u = threadIdx.x + i * THREADS;
      p[i] = static_cast<const float*>(op.p) + (int64_t)min(row0 + u / KH, op.rows - 1) * op.ld + k0 + u % KH * 8;
    }
  }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const floatx4 a = *reinterpret_cast<const floatx4_u*>(p[i]), b = *reinterpret_cast<const floatx4_u*>(p[i] + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[i][j] = a[j];
        v[i][4 + j] = b[j];
      }
      p[i] += BK;
    }
  }
  __device__ __forceinline__ void load_tail(int left) {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int k = (threadIdx.x + i * THREADS) % KH * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = k + j < left ? p[i][j] : 0.0f;
    }
  }
  template <bool SAFE>
  __device__ __forceinline__ void store(u32x4* s) const {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int u = threadIdx.x + i * THREADS;
      store_split<SAFE>(v[i], s + u % KH * PITCH + u / KH, KH * PITCH);
    }
  }
};

// Rows are contiguous and k values lie op.ld apart: a wave reads 64 neighbouring rows of one k
// at a time, and the 8 that a thread collects are a unit, so the transpose costs nothing.
template <int ROWS, int BK, int THREADS>
struct LoadKSlow {
  static constexpr int PLANES = 3, KH = BK / 8, UN = ROWS * KH / THREADS, PITCH = unit_pitch(ROWS);
  static constexpr int UNITS = PLANES * KH * PITCH;
  static_assert(ROWS * KH % THREADS == 0 && ROWS % 64 == 0, "whole units per thread, whole waves per k");
  const float* base;  // uniform
  int64_t ld;
  uint32_t col[UN];
  float v[UN][8];

  static __device__ __forceinline__ int kh(int i) {
    return __builtin_amdgcn_readfirstlane((threadIdx.x + i * THREADS) / ROWS);
  }
  __device__ __forceinline__ void init(const ProductOperand& op, int row0, int64_t k0) {
    ld = op.ld;
    base = static_cast<const float*>(op.p) + k0 * ld;
#pragma unroll
    for (int i = 0; i < UN; ++i) col[i] = (uint32_t)min(row0 + (int)(threadIdx.x + i * THREADS) % ROWS, op.rows - 1);
  }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const float* q = base + kh(i) * 8 * ld;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = (q + j * ld)[col[i]];
    }
    base += BK * ld;
  }
  __device__ __forceinline__ void load_tail(int left) {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const float* q = base + kh(i) * 8 * ld;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = kh(i) * 8 + j < left ? (q + j * ld)[col[i]] : 0.0f;
    }
  }
  template <bool SAFE>
  __device__ __forceinline__ void store(u32x4* s) const {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int u = threadIdx.x + i * THREADS;
      store_split<SAFE>(v[i], s + u / ROWS * PITCH + u % ROWS, KH * PITCH);
    }
  }
};

// A checkpoint read the same way: k values are its rows.  One plane, no split.
template <int ROWS, int BK, int THREADS>
struct LoadCodes {
  static constexpr int PLANES = 1, KH = BK / 8, UN = ROWS * KH / THREADS, PITCH = unit_pitch(ROWS);
  static constexpr int UNITS = PLANES * KH * PITCH;
  static_assert(ROWS * KH % THREADS == 0 && ROWS % 64 == 0, "whole units per thread, whole waves per k");
  const int8_t* base;  // uniform
  int64_t ld;
  uint32_t col[UN];
  const uint8_t* step[UN];  // of this thread's 8 k values
  int v[UN][8];
  u32x2 b[UN];

  static __device__ __forceinline__ int kh(int i) {
    return __builtin_amdgcn_readfirstlane((threadIdx.x + i * THREADS) / ROWS);
  }
  __device__ __forceinline__ void init(const ProductOperand& op, int row0, int64_t k0) {
    ld = op.ld;
    base = static_cast<const int8_t*>(op.p) + k0 * ld;
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      col[i] = (uint32_t)min(row0 + (int)(threadIdx.x + i * THREADS) % ROWS, op.rows - 1);
      // k0 and kh(i) * 8 are multiples of 8, a group's bytes fill its row to a multiple of 16
      step[i] = op.scales + (int64_t)(col[i] / kAct8Group) * op.lds + k0 + kh(i) * 8;
    }
  }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int8_t* q = base + kh(i) * 8 * ld;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = (q + j * ld)[col[i]];
      b[i] = *reinterpret_cast<const u32x2*>(step[i]);
      step[i] += BK;
    }
    base += BK * ld;
  }
  __device__ __forceinline__ void load_tail(int left) {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int8_t* q = base + kh(i) * 8 * ld;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = kh(i) * 8 + j < left ? (q + j * ld)[col[i]] : 0;
      // the step bytes of rows past the last are whatever they are: 0 instead
      b[i] = u32x2{0, 0};
      if (kh(i) * 8 < left) {
        b[i] = *reinterpret_cast<const u32x2*>(step[i]);
        const int have = min(left - kh(i) * 8, 8);
        if (have < 8) {
          const uint64_t keep = (1ull << (8 * have)) - 1;
          b[i][0] &= (uint32_t)keep;
          b[i][1] &= (uint32_t)(keep >> 32);
        }
      }
    }
  }
  template <bool SAFE>
  __device__ __forceinline__ void store(u32x4* s) const {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int u = threadIdx.x + i * THREADS;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = (float)v[i][j] * act8_step((b[i][j / 4] >> (8 * (j % 4))) & 255u);
      u32x4 h;
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = upper_halves(__float_as_uint(f[2 * j]), __float_as_uint(f[2 * j + 1]));
      s[u / ROWS * PITCH + u % ROWS] = h;
    }
  }
};

// BM x BN tiles by WM x WN waves, stages of BK k values, OCC blocks per CU.
template <int BM_, int BN_, int WM_, int WN_, int BK_, int OCC_>
struct ProductTile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = BK_, OCC = OCC_;
  static constexpr int THREADS = WM * WN * 64, FM = BM / WM / 32, FN = BN / WN / 32;
};

// The stage in `sa`, `sb` onto a wave's blocks.  The first operand of the instruction is B, so
// a lane holds row lane % 32 of A's and, in element r, column (r / 4) * 8 + (lane / 32) * 4 + r % 4
// of B's 32: four neighbouring columns of C in four registers.
template <class T, class LA, class LB, bool FP32>
__device__ __forceinline__ void product_stage(const u32x4* __restrict__ sa, const u32x4* __restrict__ sb, int ra,
                                              int rb, acc32 (&acc)[T::FM][T::FN]) {
  constexpr int KH = T::BK / 8;
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int s = 0; s < T::BK / 16; ++s) {
    const int kh = 2 * s + half;
    u32x4 b[T::FN][LB::PLANES];
#pragma unroll
    for (int j = 0; j < T::FN; ++j)
#pragma unroll
      for (int p = 0; p < LB::PLANES; ++p) b[j][p] = sb[(p * KH + kh) * LB::PITCH + rb + 32 * j];
#pragma unroll
    for (int i = 0; i < T::FM; ++i) {
      u32x4 a[LA::PLANES];
#pragma unroll
      for (int p = 0; p < LA::PLANES; ++p) a[p] = sa[(p * KH + kh) * LA::PITCH + ra + 32 * i];
      if constexpr (FP32) {
        auto whole = [](const u32x4* f, int planes, int e) {
          float x = 0.0f;
          for (int p = 0; p < planes; ++p) x = x + (e % 2 ? high_half(f[p][e / 2]) : low_half(f[p][e / 2]));
          return x;
        };
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int j = 0; j < T::FN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(whole(b[j], LB::PLANES, e), whole(a, LA::PLANES, e),
                                                             acc[i][j], 0, 0, 0);
      } else {
        // the smallest terms first
        auto term = [&](int pa, int pb) {
#pragma unroll
          for (int j = 0; j < T::FN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b[j][pb]),
                                                                __builtin_bit_cast(bf16x8, a[pa]), acc[i][j], 0, 0, 0);
        };
        if constexpr (LA::PLANES == 3) {
          term(0, 2);
          term(2, 0);
          term(1, 1);
          term(0, 1);
          term(1, 0);
          term(0, 0);
        } else {
          term(0, 2);
          term(0, 1);
          term(0, 0);
        }
      }
    }
  }
}

// acc = the tile's product over k in [k0, k1).  Two LDS buffers, one barrier a stage: the next
// stage's loads are in flight while this one is multiplied.
template <class T, class LA, class LB, bool FP32>
__device__ __forceinline__ void product_loop(const ProductOperand& A, const ProductOperand& B, int m0, int n0,
                                             int64_t k0, int64_t k1, u32x4* __restrict__ smem,
                                             acc32 (&acc)[T::FM][T::FN]) {
  constexpr int STAGE = LA::UNITS + LB::UNITS;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int ra = wave / T::WN * (T::FM * 32) + (lane & 31), rb = wave % T::WN * (T::FN * 32) + (lane & 31);
#pragma unroll
  for (int i = 0; i < T::FM; ++i)
#pragma unroll
    for (int j = 0; j < T::FN; ++j) acc[i][j] = acc32{};
  LA la;
  LB lb;
  la.init(A, m0, k0);
  lb.init(B, n0, k0);
  const int full = (int)((k1 - k0) / T::BK), left = (int)((k1 - k0) % T::BK), n = full + (left > 0);
  auto load = [&](int t) {
    if (t < full) {
      la.load();
      lb.load();
    } else {
      la.load_tail(left);
      lb.load_tail(left);
    }
  };
  auto store = [&](int t) {
    u32x4* s = smem + (t & 1) * STAGE;
    la.template store<FP32>(s);
    lb.template store<FP32>(s + LA::UNITS);
  };
  if (n == 0) return;
  load(0);
  store(0);
  __syncthreads();
  for (int t = 0; t < n; ++t) {
    if (t + 1 < n) load(t + 1);
    const u32x4* s = smem + (t & 1) * STAGE;
    product_stage<T, LA, LB, FP32>(s, s + LA::UNITS, ra, rb, acc);
    if (t + 1 < n) store(t + 1);
    __syncthreads();
  }
}

// The product, again on the fp32 instructions if it holds a NaN.
template <class T, class LA, class LB>
__device__ __forceinline__ void product(const ProductOperand& A, const ProductOperand& B, int m0, int n0, int64_t k0,
                                        int64_t k1, u32x4* __restrict__ smem, acc32 (&acc)[T::FM][T::FN]) {
  product_loop<T, LA, LB, false>(A, B, m0, n0, k0, k1, smem, acc);
  bool nan = false;
#pragma unroll
  for (int i = 0; i < T::FM; ++i)
#pragma unroll
    for (int j = 0; j < T::FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) nan |= acc[i][j][r] != acc[i][j][r];
  if (__syncthreads_or(nan)) product_loop<T, LA, LB, true>(A, B, m0, n0, k0, k1, smem, acc);
}

}  // namespace
}  // namespace orca_hip
