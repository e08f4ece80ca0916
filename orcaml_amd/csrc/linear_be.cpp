// The fused Linear and the 8-bit checkpoints on storages (orca_hip_be_linear_act and its
// neighbours): the buffer-level calls under the backend's lock, with contiguous operands.
#include "act8.hpp"
#include "runtime.hpp"

using namespace orca_hip;

namespace {

// Elements of a matrix, and of a checkpoint's storage; of sizes that the calls refuse, a number that no storage has.
size_t count(size_t rows, size_t cols) {
  return rows >> kMaxSizeBits || cols >> kMaxSizeBits ? SIZE_MAX : rows * cols;
}
size_t packed_count(size_t rows, size_t cols) {
  return count(rows, cols) == SIZE_MAX ? SIZE_MAX : (act8_layout(rows, cols).bytes + 3) / 4;
}

}  // namespace

extern "C" {

int orca_hip_be_act8_pack(orca_hip_backend* be, orca_hip_storage* x, size_t rows, size_t cols,
                          orca_hip_storage** out) {
  return be_run(be, {{x, count(rows, cols), "act8_pack"}}, {{packed_count(rows, cols), out}},
                [&](orca_hip_ctx* ctx, float* const* i, float* const* o) {
                  return orca_hip_act8_pack(ctx, i[0], rows, cols, cols, o[0]);
                });
}

int orca_hip_be_act8_unpack(orca_hip_backend* be, orca_hip_storage* packed, size_t rows, size_t cols,
                            orca_hip_storage** out) {
  return be_run(be, {{packed, packed_count(rows, cols), "act8_unpack"}}, {{count(rows, cols), out}},
                [&](orca_hip_ctx* ctx, float* const* i, float* const* o) {
                  return orca_hip_act8_unpack(ctx, i[0], rows, cols, ORCA_HIP_F32, o[0], cols);
                });
}

int orca_hip_be_linear_act(orca_hip_backend* be, orca_hip_storage* x, orca_hip_storage* w, orca_hip_storage* bias,
                           orca_hip_storage* residual, size_t M, size_t N, size_t K, int act, orca_hip_storage** y,
                           orca_hip_storage** z, orca_hip_storage** z8, orca_hip_storage** y8) {
  const size_t mn = count(M, N), packed = packed_count(M, N);
  return be_run(be,
                {{x, count(M, K), "linear_act (x)"},
                 {w, count(K, N), "linear_act (weight)"},
                 {bias, N, "linear_act (bias)", true},
                 {residual, mn, "linear_act (residual)", true}},
                {{mn, y}, {mn, z, true}, {packed, z8, true}, {packed, y8, true}},
                [&](orca_hip_ctx* ctx, float* const* i, float* const* o) {
                  orca_hip_linear_epilogue e{};
                  e.act = act;
                  e.bias = i[2];
                  e.residual = i[3];
                  e.ldr = N;
                  e.pre = o[1];
                  e.ldpre = N;
                  e.pre8 = o[2];
                  e.y8 = o[3];
                  return orca_hip_linear_act(ctx, M, N, K, i[0], K, i[1], N, o[0], N, &e);
                });
}

int orca_hip_be_linear_act_backward(orca_hip_backend* be, orca_hip_storage* dy, orca_hip_storage* w, size_t M,
                                    size_t N, size_t K, int act, orca_hip_storage* z, orca_hip_storage* z8,
                                    orca_hip_storage* x, orca_hip_storage* x8, orca_hip_storage* dx_add,
                                    orca_hip_storage** dx, orca_hip_storage** dw, orca_hip_storage** db) {
  const size_t mn = count(M, N), mk = count(M, K), kn = count(K, N);
  return be_run(be,
                {{dy, mn, "linear_act_backward (dy)"},
                 {w, kn, "linear_act_backward (weight)"},
                 {z, mn, "linear_act_backward (z)", true},
                 {z8, packed_count(M, N), "linear_act_backward (z8)", true},
                 {x, mk, "linear_act_backward (x)", true},
                 {x8, packed_count(M, K), "linear_act_backward (x8)", true},
                 {dx_add, mk, "linear_act_backward (dx_add)", true}},
                {{mk, dx, true}, {kn, dw, true}, {N, db, true}},
                [&](orca_hip_ctx* ctx, float* const* i, float* const* o) {
                  orca_hip_linear_saved s{};
                  s.act = act;
                  s.z = i[2];
                  s.ldz = N;
                  s.z8 = i[3];
                  s.x = i[4];
                  s.ldx = K;
                  s.x8 = i[5];
                  s.dx_add = i[6];
                  s.ldadd = K;
                  return orca_hip_linear_act_backward(ctx, M, N, K, i[0], N, i[1], N, &s, o[0], K, o[1], N, o[2]);
                });
}

}  // extern "C"
