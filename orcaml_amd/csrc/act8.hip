// Packing activations into 8-bit checkpoints and back (format and arithmetic: act8.hpp).
// Both are one pass over memory.
#include <algorithm>
#include <string>

#include "act8.hpp"
#include "runtime.hpp"
#include "slab.hpp"

namespace orca_hip {
namespace {

// A thread takes four neighbouring columns of four rows that lie four apart (their loads are in flight
// together), eight lanes a group of 32 columns; a block 16 rows of 256 columns.
__global__ void __launch_bounds__(256) act8_pack_kernel(const float* __restrict__ x, int64_t ldx, int64_t rows,
                                                        int64_t cols, Act8 out) {
  typedef uint32_t word_u __attribute__((aligned(1)));
  const int64_t r0 = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 6);
  const int64_t c = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * 256 + (threadIdx.x & 63) * 4;
  const int have = (int)max((int64_t)0, min((int64_t)4, cols - c));
  floatx4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float* p = x + min(r0 + 4 * i, rows - 1) * ldx + c;
    v[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    if (have == 4) {
      v[i] = *reinterpret_cast<const floatx4_u*>(p);
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < have) v[i][j] = p[j];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = r0 + 4 * i;
    uint32_t top = max(max(act8_magnitude(v[i][0]), act8_magnitude(v[i][1])),
                       max(act8_magnitude(v[i][2]), act8_magnitude(v[i][3])));
#pragma unroll
    for (int d = 1; d < 8; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    const uint32_t b = act8_byte(top);
    if (row >= rows || have == 0) continue;
    int8_t* p = out.codes + row * cols + c;
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w |= ((uint32_t)act8_code(v[i][j], b) & 255u) << (8 * j);
    if (have == 4) {
      *reinterpret_cast<word_u*>(p) = w;
    } else {
      for (int j = 0; j < have; ++j) p[j] = (int8_t)(w >> (8 * j));
    }
    if ((threadIdx.x & 7) == 0) out.scales[c / 32 * out.ld + row] = (uint8_t)b;
  }
}

// A thread takes four neighbouring columns of four rows that lie four apart, so that a wave has their loads
// in flight together.
template <bool HALF>
__global__ void __launch_bounds__(256) act8_unpack_kernel(Act8 in, int64_t rows, int64_t cols, void* __restrict__ out,
                                                          int64_t ldo) {
  typedef uint32_t word_u __attribute__((aligned(1)));
  const int64_t r0 = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 6);
  const int64_t c = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * 256 + (threadIdx.x & 63) * 4;
  if (c >= cols) return;
  const int have = (int)min((int64_t)4, cols - c);
  uint32_t w[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = min(r0 + 4 * i, rows - 1);
    const int8_t* p = in.codes + row * cols + c;
    b[i] = in.scales[c / 32 * in.ld + row];
    w[i] = 0;
    if (have == 4) {
      w[i] = *reinterpret_cast<const word_u*>(p);
    } else {
      for (int j = 0; j < have; ++j) w[i] |= (uint32_t)(uint8_t)p[j] << (8 * j);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = r0 + 4 * i;
    if (row >= rows) break;
    const float step = act8_step(b[i]);
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __float_as_uint((float)(int8_t)(w[i] >> (8 * j)) * step);
    if (HALF) {  // exact
      uint16_t* o = static_cast<uint16_t*>(out) + row * ldo + c;
      if (have == 4) {
        typedef uint32_t pair_u __attribute__((ext_vector_type(2), aligned(2)));
        *reinterpret_cast<pair_u*>(o) = pair_u{v[0] >> 16 | (v[1] & 0xffff0000u), v[2] >> 16 | (v[3] & 0xffff0000u)};
      } else {
        for (int j = 0; j < have; ++j) o[j] = (uint16_t)(v[j] >> 16);
      }
    } else {
      float* o = static_cast<float*>(out) + row * ldo + c;
      if (have == 4) {
        *reinterpret_cast<floatx4_u*>(o) = floatx4{__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]),
                                                   __uint_as_float(v[3])};
      } else {
        for (int j = 0; j < have; ++j) o[j] = __uint_as_float(v[j]);
      }
    }
  }
}

dim3 act8_grid(size_t rows, size_t cols) {
  const size_t gx = (rows + 15) / 16, gy = (cols + 255) / 256, y = std::min<size_t>(gy, 32768);
  return dim3((unsigned)gx, (unsigned)y, (unsigned)((gy + y - 1) / y));
}

void act8_check(const char* op, size_t rows, size_t cols, size_t ld) {
  for (size_t v : {rows, cols})
    if (v >> kMaxSizeBits) fail_shape(op, "sizes below 2^" + std::to_string(kMaxSizeBits), std::to_string(v));
  if (ld > size_t(1) << kMaxLdBits)
    fail_shape(op, "a leading dimension of at most 2^" + std::to_string(kMaxLdBits), std::to_string(ld));
  if (ld < cols) fail_shape(op, "a leading dimension of at least " + std::to_string(cols), std::to_string(ld));
}

void act8_apart(const char* op, const void* out, size_t out_bytes, const void* in, size_t in_bytes) {
  const auto a = reinterpret_cast<uintptr_t>(out), b = reinterpret_cast<uintptr_t>(in);
  if (out_bytes && in_bytes && a < b + in_bytes && b < a + out_bytes)
    fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": the output overlaps the input");
}

}  // namespace

void act8_aligned(const void* packed, const char* what) {
  if (reinterpret_cast<uintptr_t>(packed) % 16)
    fail(ORCA_HIP_ERR_INTERNAL, std::string(what) + ": a checkpoint must be 16-byte aligned");
}

}  // namespace orca_hip

using namespace orca_hip;

extern "C" {

int orca_hip_act8_size(size_t rows, size_t cols, size_t* bytes, size_t* scales_offset) {
  return guard([&] {
    if (!bytes) fail(ORCA_HIP_ERR_INTERNAL, "act8_size: null output pointer");
    act8_check("act8_size", rows, cols, cols);
    const Act8Layout l = act8_layout(rows, cols);
    *bytes = l.bytes;
    if (scales_offset) *scales_offset = l.scales;
  });
}

int orca_hip_act8_pack(orca_hip_ctx* ctx, const float* x, size_t rows, size_t cols, size_t ldx, void* packed) {
  return guard([&] {
    act8_check("act8_pack", rows, cols, ldx);
    if (rows && cols && (!x || !packed)) fail(ORCA_HIP_ERR_INTERNAL, "act8_pack: null operand");
    act8_aligned(packed, "act8_pack");
    act8_apart("act8_pack", packed, act8_layout(rows, cols).bytes, x, matrix_bytes(rows, cols, ldx));
    bind(ctx);
    if (!rows || !cols) return;
    check_extent(ctx, x, matrix_bytes(rows, cols, ldx), "act8_pack (x)");
    check_extent(ctx, packed, act8_layout(rows, cols).bytes, "act8_pack (checkpoint)");
    const dim3 grid = act8_grid(rows, cols);
    ProfScope prof(ctx, "act8_pack", 0.0, 4.0 * rows * cols + (double)act8_layout(rows, cols).bytes);
    hipLaunchKernelGGL(act8_pack_kernel, grid, dim3(256), 0, ctx->stream, x, (int64_t)ldx, (int64_t)rows, (int64_t)cols,
                       act8_at(packed, rows, cols));
    ORCA_HIP_CHECK(hipGetLastError());
  });
}

int orca_hip_act8_unpack(orca_hip_ctx* ctx, const void* packed, size_t rows, size_t cols, int dtype, void* out,
                         size_t ldo) {
  return guard([&] {
    if (dtype != ORCA_HIP_F32 && dtype != ORCA_HIP_BF16) fail_dtype("act8_unpack", dtype);
    act8_check("act8_unpack", rows, cols, ldo);
    if (rows && cols && (!out || !packed)) fail(ORCA_HIP_ERR_INTERNAL, "act8_unpack: null operand");
    act8_aligned(packed, "act8_unpack");
    const size_t width = dtype == ORCA_HIP_F32 ? 4 : 2, out_bytes = matrix_bytes(rows, cols, ldo) / 4 * width;
    act8_apart("act8_unpack", out, out_bytes, packed, act8_layout(rows, cols).bytes);
    bind(ctx);
    if (!rows || !cols) return;
    check_extent(ctx, out, out_bytes, "act8_unpack (out)");
    check_extent(ctx, packed, act8_layout(rows, cols).bytes, "act8_unpack (checkpoint)");
    const dim3 grid = act8_grid(rows, cols);
    const Act8 in = act8_at(const_cast<void*>(packed), rows, cols);
    ProfScope prof(ctx, "act8_unpack", 0.0, (double)width * rows * cols + (double)act8_layout(rows, cols).bytes);
    if (dtype == ORCA_HIP_F32)
      hipLaunchKernelGGL(act8_unpack_kernel<false>, grid, dim3(256), 0, ctx->stream, in, (int64_t)rows, (int64_t)cols,
                         out, (int64_t)ldo);
    else
      hipLaunchKernelGGL(act8_unpack_kernel<true>, grid, dim3(256), 0, ctx->stream, in, (int64_t)rows, (int64_t)cols,
                         out, (int64_t)ldo);
    ORCA_HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
