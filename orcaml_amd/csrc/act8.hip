// Packing activations into 8-bit checkpoints and back (format and arithmetic: act8.hpp).
// Both are one pass over memory.
#include <string>

#include "act8.hpp"
#include "runtime.hpp"
#include "slab.hpp"

namespace orca_hip {
namespace {

// A thread takes four neighbouring columns of a row, eight lanes a group of 32 (DPP-free
// shuffles among them find its largest magnitude); a block 4 rows of 256 columns.
__global__ void __launch_bounds__(256) act8_pack_kernel(const float* __restrict__ x, int64_t ldx, int64_t rows,
                                                        int64_t cols, Act8 out) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t c = (int64_t)blockIdx.y * 256 + (threadIdx.x & 63) * 4;
  if (row >= rows) return;  // a whole wave
  const int have = (int)max((int64_t)0, min((int64_t)4, cols - c));
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (have == 4) {
    const floatx4 q = *reinterpret_cast<const floatx4_u*>(x + row * ldx + c);
    for (int j = 0; j < 4; ++j) v[j] = q[j];
  } else {
    for (int j = 0; j < 4; ++j)
      if (j < have) v[j] = x[row * ldx + c + j];
  }
  uint32_t top = max(max(act8_magnitude(v[0]), act8_magnitude(v[1])), max(act8_magnitude(v[2]), act8_magnitude(v[3])));
  for (int d = 1; d < 8; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  const uint32_t b = act8_byte(top);
  int8_t* p = out.codes + row * cols + c;
  uint32_t w = 0;
  for (int j = 0; j < 4; ++j) w |= ((uint32_t)act8_code(v[j], b) & 255u) << (8 * j);
  if (have == 4) {
    typedef uint32_t word_u __attribute__((aligned(1)));
    *reinterpret_cast<word_u*>(p) = w;
  } else {
    for (int j = 0; j < 4; ++j)
      if (j < have) p[j] = (int8_t)(w >> (8 * j));
  }
  if ((threadIdx.x & 7) == 0 && c < cols) out.scales[c / 32 * out.ld + row] = (uint8_t)b;
}

template <bool HALF>
__global__ void __launch_bounds__(256) act8_unpack_kernel(Act8 in, int64_t rows, int64_t cols, void* __restrict__ out,
                                                          int64_t ldo) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t c = (int64_t)blockIdx.y * 256 + (threadIdx.x & 63) * 4;
  if (row >= rows || c >= cols) return;
  const int have = (int)min((int64_t)4, cols - c);
  const float step = act8_step(in.scales[c / 32 * in.ld + row]);
  const int8_t* p = in.codes + row * cols + c;
  for (int j = 0; j < 4; ++j) {
    if (j >= have) break;
    const float v = (float)p[j] * step;
    if (HALF)
      static_cast<uint16_t*>(out)[row * ldo + c + j] = (uint16_t)(__float_as_uint(v) >> 16);  // exact
    else
      static_cast<float*>(out)[row * ldo + c + j] = v;
  }
}

void act8_apart(const char* op, const void* out, size_t out_bytes, const void* in, size_t in_bytes) {
  const auto a = reinterpret_cast<uintptr_t>(out), b = reinterpret_cast<uintptr_t>(in);
  if (out_bytes && in_bytes && a < b + in_bytes && b < a + out_bytes)
    fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": the output overlaps the input");
}

dim3 act8_grid(size_t rows, size_t cols, const char* op) {
  const size_t gx = (rows + 3) / 4, gy = (cols + 255) / 256;
  if (gx > 0x7fffffffu || gy > 65535) fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": matrix too large");
  return dim3((unsigned)gx, (unsigned)gy);
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
    if (cols && rows > (SIZE_MAX >> 8) / cols) fail(ORCA_HIP_ERR_SHAPE, "Shape mismatch during act8_size: size overflow");
    const Act8Layout l = act8_layout(rows, cols);
    *bytes = l.bytes;
    if (scales_offset) *scales_offset = l.scales;
  });
}

int orca_hip_act8_pack(orca_hip_ctx* ctx, const float* x, size_t rows, size_t cols, size_t ldx, void* packed) {
  return guard([&] {
    if (ldx < cols) fail_shape("act8_pack", "a leading dimension of at least " + std::to_string(cols), std::to_string(ldx));
    if (rows && cols && (!x || !packed)) fail(ORCA_HIP_ERR_INTERNAL, "act8_pack: null operand");
    act8_aligned(packed, "act8_pack");
    act8_apart("act8_pack", packed, act8_layout(rows, cols).bytes, x, matrix_bytes(rows, cols, ldx));
    bind(ctx);
    if (!rows || !cols) return;
    check_extent(ctx, x, matrix_bytes(rows, cols, ldx), "act8_pack (x)");
    check_extent(ctx, packed, act8_layout(rows, cols).bytes, "act8_pack (checkpoint)");
    const dim3 grid = act8_grid(rows, cols, "act8_pack");
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
    if (ldo < cols) fail_shape("act8_unpack", "a leading dimension of at least " + std::to_string(cols), std::to_string(ldo));
    if (rows && cols && (!out || !packed)) fail(ORCA_HIP_ERR_INTERNAL, "act8_unpack: null operand");
    act8_aligned(packed, "act8_unpack");
    const size_t width = dtype == ORCA_HIP_F32 ? 4 : 2, out_bytes = matrix_bytes(rows, cols, ldo) / 4 * width;
    act8_apart("act8_unpack", out, out_bytes, packed, act8_layout(rows, cols).bytes);
    bind(ctx);
    if (!rows || !cols) return;
    check_extent(ctx, out, out_bytes, "act8_unpack (out)");
    check_extent(ctx, packed, act8_layout(rows, cols).bytes, "act8_unpack (checkpoint)");
    const dim3 grid = act8_grid(rows, cols, "act8_unpack");
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
