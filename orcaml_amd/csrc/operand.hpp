// Checks of matrix operands given by pointer, sizes and leading dimension, and a call's workspace: shared by the
// buffer-level entry points beyond the trait's.
#pragma once

#include <cstddef>
#include <cstdint>
#include <memory>
#include <string>

#include "act8.hpp"
#include "runtime.hpp"

namespace orca_hip {

// Fails unless a checkpoint's address is a multiple of 16 (act8.hip).
void act8_aligned(const void* packed, const char* what);

namespace {

inline void check_ld(const char* what, size_t ld, size_t cols) {
  if (ld > size_t(1) << kMaxLdBits)
    fail_shape(what, "a leading dimension of at most 2^" + std::to_string(kMaxLdBits), std::to_string(ld));
  if (ld < cols) fail_shape(what, "a leading dimension of at least " + std::to_string(cols), std::to_string(ld));
}
inline void check_sizes(const char* op, std::initializer_list<size_t> sizes) {
  for (size_t v : sizes)
    if (v >> kMaxSizeBits) fail_shape(op, "sizes below 2^" + std::to_string(kMaxSizeBits), std::to_string(v));
}
// An operand's rows of `width` bytes, `ld` bytes apart (one row: a contiguous buffer).
struct Span {
  const void* p;
  size_t rows, width, ld;
  size_t bytes() const { return rows && width ? (rows - 1) * ld + width : 0; }
};
inline Span matrix_span(const void* p, size_t rows, size_t cols, size_t ld) { return Span{p, rows, 4 * cols, 4 * ld}; }
inline Span buffer_span(const void* p, size_t bytes) { return Span{p, 1, bytes, bytes}; }
// A result must not lie in what the call reads, or in another result.  Columns of one matrix beside each
// other (the same ld) are apart.
inline void check_apart(const char* op, const Span& out, const Span& in) {
  const auto a = reinterpret_cast<uintptr_t>(out.p), b = reinterpret_cast<uintptr_t>(in.p);
  if (!out.p || !in.p || !out.bytes() || !in.bytes() || a >= b + in.bytes() || b >= a + out.bytes()) return;
  if (out.ld == in.ld && out.ld) {
    const size_t d = (a < b ? b - a : out.ld - (a - b) % out.ld) % out.ld;  // from out's columns to in's
    if (d >= out.width && out.ld - d >= in.width) return;
  }
  fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": an output overlaps another operand");
}
// Elements of a matrix, and of a checkpoint's storage; of sizes that the calls refuse, a number that no storage has.
inline size_t element_count(size_t rows, size_t cols) {
  return rows >> kMaxSizeBits || cols >> kMaxSizeBits ? SIZE_MAX : rows * cols;
}
inline size_t packed_count(size_t rows, size_t cols) {
  return element_count(rows, cols) == SIZE_MAX ? SIZE_MAX : (act8_layout(rows, cols).bytes + 3) / 4;
}
// A workspace goes back to the context's allocator when the call returns: a captured graph would write
// it at every replay, whoever has it then.
inline std::unique_ptr<Scratch> workspace(orca_hip_ctx* ctx, size_t bytes, const char* op) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  ORCA_HIP_CHECK(hipStreamIsCapturing(ctx->stream, &status));
  if (status != hipStreamCaptureStatusNone)
    fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": needs a workspace, which a captured graph cannot keep");
  return std::make_unique<Scratch>(ctx, bytes);
}

}  // namespace
}  // namespace orca_hip
