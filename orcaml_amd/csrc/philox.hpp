// The random numbers of a dropout: Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011).  A number depends on the seed, the call's offset and the value's place
// alone, so the backward draws the forward's again and no mask is kept, and no launch shape changes a result.
// A counter (col / 4, row, offset) gives the words of four neighbouring columns, which one thread holds.
//
// Cost: ten rounds of two 32 x 32 -> 64 bit products, which run at a quarter of the vector units' rate: 320 cycles
// of a SIMD for a wave's 256 values, and about 80 for the rest.  A CU's share of HBM (21 GB/s) brings the 8 bytes
// that a value's dropout moves no faster than 2.6 values a ns, and its four SIMDs draw 6.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace orca_hip {

// A dropout on the device.  A value is kept if its word is above `above`: the words that drop it are
// 0 .. rint(p 2^32) - 1, so the share kept is exact in the scale.
struct Dropout {
  int on = 0;
  uint32_t above = 0;
  float scale = 1.0f;  // 2^32 over the number of words that keep a value; 0 where none does
  uint32_t key[2] = {0, 0}, offset[2] = {0, 0};
};
inline Dropout dropout_of(double p, uint64_t seed, uint64_t offset) {
  Dropout d;
  const double words = 4294967296.0, border = std::nearbyint(p * words);
  d.on = border >= 1.0;
  if (!d.on) return d;
  d.above = (uint32_t)(border - 1.0);
  d.scale = border < words ? (float)(words / (words - border)) : 0.0f;
  d.key[0] = (uint32_t)seed;
  d.key[1] = (uint32_t)(seed >> 32);
  d.offset[0] = (uint32_t)offset;
  d.offset[1] = (uint32_t)(offset >> 32);
  return d;
}

namespace {

struct Words {
  uint32_t v[4];
};
// a ^ b ^ c in one instruction (its truth table).
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}
__device__ __forceinline__ Words philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = xor3((uint32_t)(b >> 32), c1, k0);
    c2 = xor3((uint32_t)(a >> 32), c3, k1);
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}
// The words of columns 4 quad .. 4 quad + 3 of a row (both below 2^27).
__device__ __forceinline__ Words dropout_words(const Dropout& d, int64_t row, int64_t quad) {
  return philox((uint32_t)quad, (uint32_t)row, d.offset[0], d.offset[1], d.key[0], d.key[1]);
}
__device__ __forceinline__ bool dropout_keeps(const Dropout& d, const Words& w, int j) { return w.v[j] > d.above; }

}  // namespace
}  // namespace orca_hip
