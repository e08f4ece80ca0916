// Dropout by itself (orca_hip_dropout); inside the joint of two blocks it is part of norm.hip's kernels.
#include <algorithm>
#include <string>

#include "operand.hpp"
#include "philox.hpp"
#include "quad.hpp"
#include "runtime.hpp"

namespace orca_hip {
namespace {

constexpr int kDropRows = 4;  // rows of a thread, so that it has as many loads in flight

// A thread takes four neighbouring columns of kDropRows rows; `across` threads of a block lie along a row, the
// others below each other.  y may be x: a thread reads what it writes first.
__global__ void __launch_bounds__(256) dropout_kernel(const float* x, int64_t ldx, int64_t rows, int64_t cols, float* y,
                                                      int64_t ldy, int across_bits, Dropout d) {
  const int64_t down = 256 >> across_bits;
  const int64_t quad = ((((int64_t)blockIdx.z * gridDim.y + blockIdx.y) << across_bits) +
                        (threadIdx.x & ((1 << across_bits) - 1)));
  const int64_t r0 = (int64_t)blockIdx.x * down * kDropRows + (threadIdx.x >> across_bits);
  const Quad q = quad_of(quad * 4, cols);
  floatx4 v[kDropRows];
#pragma unroll
  for (int i = 0; i < kDropRows; ++i) v[i] = load_quad(x + min(r0 + i * down, rows - 1) * ldx, q);
#pragma unroll
  for (int i = 0; i < kDropRows; ++i) {
    const int64_t row = r0 + i * down;
    settle(q, v[i]);
    if (d.on) {
      const Words w = dropout_words(d, row, quad);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = dropout_keeps(d, w, j) ? v[i][j] * d.scale : 0.0f;
    }
    if (row < rows) store_quad(y + row * ldy, q, v[i]);
  }
}

}  // namespace
}  // namespace orca_hip

using namespace orca_hip;

extern "C" {

int orca_hip_dropout(orca_hip_ctx* ctx, size_t rows, size_t cols, const float* x, size_t ldx, double p, uint64_t seed,
                     uint64_t offset, float* y, size_t ldy) {
  return guard([&] {
    const char* op = "dropout";
    check_sizes(op, {rows, cols});
    check_ld("dropout (x)", ldx, cols);
    check_ld("dropout (y)", ldy, cols);
    if (!(p >= 0.0 && p <= 1.0)) fail(ORCA_HIP_ERR_INTERNAL, "dropout: p must be from 0 to 1");
    if (rows && cols && (!x || !y)) fail(ORCA_HIP_ERR_INTERNAL, "dropout: null operand");
    const Span xs = matrix_span(x, rows, cols, ldx), ys = matrix_span(y, rows, cols, ldy);
    if (x != y || ldx != ldy) check_apart(op, ys, xs);
    bind(ctx);
    if (!rows || !cols) return;
    check_extent(ctx, x, xs.bytes(), "dropout (x)");
    check_extent(ctx, y, ys.bytes(), "dropout (y)");
    const size_t quads = (cols + 3) / 4;
    int bits = 0;
    while (bits < 6 && (size_t(1) << bits) < quads) ++bits;
    const size_t across = (quads + (size_t(1) << bits) - 1) >> bits, gy = std::min<size_t>(across, 32768),
                 down = (size_t(256) >> bits) * kDropRows;
    const dim3 grid((unsigned)((rows + down - 1) / down), (unsigned)gy, (unsigned)((across + gy - 1) / gy));
    ProfScope prof(ctx, op, (double)rows * cols, 8.0 * rows * cols);
    hipLaunchKernelGGL(dropout_kernel, grid, dim3(256), 0, ctx->stream, x, (int64_t)ldx, (int64_t)rows, (int64_t)cols,
                       y, (int64_t)ldy, bits, dropout_of(p, seed, offset));
    ORCA_HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
