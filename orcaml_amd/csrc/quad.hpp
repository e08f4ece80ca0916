// Four neighbouring columns of a row-major matrix, as one thread takes them: 16 bytes in fp32, 4 of a
// checkpoint, at any alignment.  At the end of a row fewer than four exist; loads are then moved back into
// the row, and once a thread has all its loads on their way, `settle` shifts the values into place.  (Loads
// behind a branch of some lanes wait for one another: the other lanes' branch writes the registers that
// they are to arrive in.)
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "act8.hpp"
#include "slab.hpp"

namespace orca_hip {
namespace {

struct Quad {
  int64_t c;      // the first column
  int64_t at;     // where the load starts
  int64_t group;  // of a checkpoint
  int shift;
  int have;       // how many of the four exist
  int n;          // columns of the matrix, at most 4
  bool whole;     // all of the wave's quads exist
};
__device__ __forceinline__ Quad quad_of(int64_t c, int64_t cols) {
  Quad q;
  q.c = c;
  q.at = max((int64_t)0, min(c, cols - 4));
  q.group = min(c, cols - 1) / (int64_t)kAct8Group;
  q.shift = (int)min((int64_t)3, c - q.at);
  q.have = (int)max((int64_t)0, min((int64_t)4, cols - c));
  q.n = (int)min((int64_t)4, cols);
  q.whole = __all(q.have == 4);
  return q;
}

__device__ __forceinline__ floatx4 load_quad(const float* row, const Quad& q) {
  if (q.n == 4) return *reinterpret_cast<const floatx4_u*>(row + q.at);
  return floatx4{row[0], row[min(1, q.n - 1)], row[min(2, q.n - 1)], 0.0f};
}
// What lies past the row's end is some value of the row.
__device__ __forceinline__ void settle(const Quad& q, floatx4& v) {
  if (!q.whole && q.n == 4) v = shift_down(v, q.shift);
}
__device__ __forceinline__ void store_quad(float* row, const Quad& q, floatx4 v) {
  float* p = row + q.c;
  if (q.have == 4) {
    *reinterpret_cast<floatx4_u*>(p) = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < q.have) p[j] = v[j];
}

typedef uint32_t word_u __attribute__((aligned(1)));
__device__ __forceinline__ uint32_t load_codes(const int8_t* row, const Quad& q) {
  if (q.n == 4) return *reinterpret_cast<const word_u*>(row + q.at);
  return (uint8_t)row[0] | (uint32_t)(uint8_t)row[min(1, q.n - 1)] << 8 | (uint32_t)(uint8_t)row[min(2, q.n - 1)] << 16;
}
__device__ __forceinline__ floatx4 settle_codes(const Quad& q, uint32_t w, uint32_t byte) {
  if (!q.whole && q.n == 4) w >>= 8 * q.shift;
  const float step = act8_step(byte);
  return floatx4{(float)(int8_t)w * step, (float)(int8_t)(w >> 8) * step, (float)(int8_t)(w >> 16) * step,
                 (float)(int8_t)(w >> 24) * step};
}
__device__ __forceinline__ void store_codes(int8_t* row, const Quad& q, floatx4 v, uint32_t b) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) w |= ((uint32_t)act8_code(v[j], b) & 255u) << (8 * j);
  int8_t* p = row + q.c;
  if (q.have == 4) {
    *reinterpret_cast<word_u*>(p) = w;
    return;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < q.have) p[j] = (int8_t)(w >> (8 * j));
}
// The bits of the largest magnitude among a quad's columns, and the step byte of the group of eight lanes.
__device__ __forceinline__ uint32_t quad_byte(floatx4 v, const Quad& q) {
  uint32_t t = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) t = max(t, j < q.have ? act8_magnitude(v[j]) : 0u);
#pragma unroll
  for (int d = 1; d < 8; d *= 2) t = max(t, (uint32_t)__shfl_xor((int)t, d));
  return act8_byte(t);
}

}  // namespace
}  // namespace orca_hip
