// 8-bit activation checkpoints: the format (include/orca_hip.h) and its arithmetic.
//
// 32 values along a row share the step 2^(b - 133), b the step byte.  With t the bits of the
// group's largest magnitude, (t + 0x10000) >> 23 is the biased exponent of t, one more where
// the mantissa is at least 127.5 / 64: the least b for which every value rounds to a code
// within 127.  So each is off by at most half a step, and none is clipped but where the step would pass
// the largest, 2^121 (magnitudes above 127.5 * 2^121).  The bits of
// magnitudes order as the magnitudes do, infinities and NaN above every number: one integer
// maximum finds all three.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace orca_hip {

constexpr size_t kAct8Group = 32;

// Bounds on the sizes and leading dimensions of the calls that take checkpoints: byte offsets stay below
// 2^63, column indexes in bytes below 2^32, and a launch of a block of 256 threads for 16 rows or columns below
// the runtime's 2^32 threads.
constexpr int kMaxSizeBits = 27, kMaxLdBits = 34;

struct Act8Layout {
  size_t groups;   // groups of 32 columns
  size_t ld;       // rows of a group's row of step bytes: a multiple of 16, so that 8 rows' bytes are one load
  size_t scales;   // offset of the step bytes
  size_t bytes;
};
inline Act8Layout act8_layout(size_t rows, size_t cols) {
  Act8Layout l;
  l.groups = (cols + kAct8Group - 1) / kAct8Group;
  l.ld = (rows + 15) / 16 * 16;
  l.scales = (rows * cols + 15) / 16 * 16;
  l.bytes = l.scales + l.groups * l.ld;
  return l;
}

// A checkpoint on the device (codes null: none).
struct Act8 {
  int8_t* codes = nullptr;
  uint8_t* scales = nullptr;
  int64_t cols = 0;  // codes per row
  int64_t ld = 0;    // Act8Layout::ld
};
inline Act8 act8_at(void* packed, size_t rows, size_t cols) {
  const Act8Layout l = act8_layout(rows, cols);
  Act8 a;
  if (packed) {
    a.codes = static_cast<int8_t*>(packed);
    a.scales = static_cast<uint8_t*>(packed) + l.scales;
    a.cols = (int64_t)cols;
    a.ld = (int64_t)l.ld;
  }
  return a;
}

namespace {

constexpr uint32_t kAct8NotFinite = 255;

__device__ __forceinline__ uint32_t act8_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// The step byte of a group whose largest magnitude has the bits `top`.
__device__ __forceinline__ uint32_t act8_byte(uint32_t top) {
  if (top >= 0x7f800000u) return kAct8NotFinite;
  return min(max((top + 0x10000u) >> 23, 7u), 254u);
}
// Code of v in a group with step byte b.  The product with the power of two is exact.
__device__ __forceinline__ int act8_code(float v, uint32_t b) {
  if (b == kAct8NotFinite) return 0;
  const float c = rintf(v * __uint_as_float((260u - b) << 23));
  return (int)fminf(fmaxf(c, -127.0f), 127.0f);
}
// The step of byte b (NaN for 255); a code times the step is a bf16 value.  Bytes below 7 are
// not written by this library; they read as 7, so that no step is subnormal.
__device__ __forceinline__ float act8_step(uint32_t b) {
  return __uint_as_float(b == kAct8NotFinite ? 0x7fc00000u : (max(b, 7u) - 6u) << 23);
}

}  // namespace
}  // namespace orca_hip
