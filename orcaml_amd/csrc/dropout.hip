// Dropout by itself (orca_hip_dropout); inside the joint of two blocks it is part of norm.hip's kernels.
#include <algorithm>
#include <string>

#include "operand.hpp"
#include "philox.hpp"
#include "quad.hpp"
#include "runtime.hpp"

namespace orca_hip {
namespace {

// A thread takes four neighbouring columns; `across` = 2^across_bits threads of a block lie along a row, the others
// below each other.  y may be x: a thread reads what it writes first.
//
// Bound by HBM: 42 to 45 us at 8192 x 4096 by the box (6.3 to 6.0 TB/s), 6.6 at 1024 x 4096.  One quad a thread, blocks
// of up to 4 KiB of a row and non-temporal stores (four rows a thread with ordinary stores, its first form, took 67 and
// 8.4).  FAR: non-temporal loads too: 44.7 us for 46.0 at 8192 x 4096, whose operands pass the 256 MiB of the
// memory-side cache, but 22.8 for 22.2 at half of that and 7.8 for 6.6 at an eighth, which it may hold from the operator
// before.
template <bool FAR>
__global__ void __launch_bounds__(256) dropout_kernel(const float* x, int64_t ldx, int64_t rows, int64_t cols, float* y,
                                                      int64_t ldy, int across_bits, Dropout d) {
  const int64_t quad = ((((int64_t)blockIdx.z * gridDim.y + blockIdx.y) << across_bits) +
                        (threadIdx.x & ((1 << across_bits) - 1)));
  const int64_t down = 256 >> across_bits;
  const Quad q = quad_of(quad * 4, cols);
  for (int64_t r0 = (int64_t)blockIdx.x * down; r0 < rows; r0 += (int64_t)gridDim.x * down) {
    const int64_t row = r0 + (threadIdx.x >> across_bits);
    const float* from = x + min(row, rows - 1) * ldx;
    floatx4 v = FAR && q.n == 4 ? (floatx4)__builtin_nontemporal_load(reinterpret_cast<const floatx4_u*>(from + q.at))
                                : load_quad(from, q);
    settle(q, v);
    if (d.on) {
      const Words w = dropout_words(d, row, quad);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = dropout_keeps(d, w, j) ? v[j] * d.scale : 0.0f;
    }
    if (row >= rows) continue;
    if (q.have == 4)
      __builtin_nontemporal_store((floatx4_u)v, reinterpret_cast<floatx4_u*>(y + row * ldy + q.c));
    else
      store_quad(y + row * ldy, q, v);
  }
}

constexpr size_t kMaxBlocks = size_t(1) << 23;  // in the first dimension, whose threads the runtime counts in 32 bits
constexpr double kCacheBytes = 256.0 * (1 << 20);  // of the memory-side cache

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
    while (bits < 8 && (size_t(1) << bits) < quads) ++bits;
    const size_t across = (quads + (size_t(1) << bits) - 1) >> bits, gy = std::min<size_t>(across, 32768),
                 down = size_t(256) >> bits;
    const dim3 grid((unsigned)std::min((rows + down - 1) / down, kMaxBlocks), (unsigned)gy, (unsigned)((across + gy - 1) / gy));
    ProfScope prof(ctx, op, (double)rows * cols, 8.0 * rows * cols);
    hipLaunchKernelGGL(8.0 * rows * cols >= kCacheBytes ? dropout_kernel<true> : dropout_kernel<false>, grid, dim3(256), 0,
                       ctx->stream, x, (int64_t)ldx, (int64_t)rows, (int64_t)cols, y, (int64_t)ldy, bits,
                       dropout_of(p, seed, offset));
    ORCA_HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
