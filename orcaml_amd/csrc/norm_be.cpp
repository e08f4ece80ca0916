// Norms, dropout and the joint of two residual blocks on storages (orca_hip_be_norm and its neighbours): the
// buffer-level calls under the backend's lock, with contiguous operands.
#include "act8.hpp"
#include "operand.hpp"
#include "runtime.hpp"

using namespace orca_hip;

namespace {

int null_block(const char* op) {
  return guard([&] { fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": null parameters"); });
}

// The buffer-level parameters; the pointers come with the operands.
orca_hip_residual_block block_of(const orca_hip_be_residual_block& b, const float* post_weight, const float* post_bias,
                                 const float* next_weight, const float* next_bias, const float* gate, size_t cols) {
  orca_hip_residual_block r{};
  r.post = {b.post, b.post_eps, post_weight, post_bias};
  r.next = {b.next, b.next_eps, next_weight, next_bias};
  r.gate = gate;
  r.groups = b.groups;
  r.ldgate = cols;
  r.residual_scale = b.residual_scale;
  r.block_scale = b.block_scale;
  r.p = b.p;
  r.seed = b.seed;
  r.offset = b.offset;
  return r;
}

}  // namespace

extern "C" {

int orca_hip_be_norm(orca_hip_backend* be, orca_hip_storage* x, size_t rows, size_t cols, int kind, float eps,
                     orca_hip_storage* weight, orca_hip_storage* bias, orca_hip_storage** y, orca_hip_storage** y8) {
  const size_t mn = element_count(rows, cols);
  return be_run(be, {{x, mn, "norm (x)"}, {weight, cols, "norm (weight)", true}, {bias, cols, "norm (bias)", true}},
                {{mn, y}, {packed_count(rows, cols), y8, true}},
                [&](orca_hip_ctx* ctx, float* const* i, float* const* o) {
                  const orca_hip_norm_params n{kind, eps, i[1], i[2]};
                  return orca_hip_norm(ctx, rows, cols, i[0], cols, &n, o[0], cols, o[1]);
                });
}

int orca_hip_be_norm_backward(orca_hip_backend* be, orca_hip_storage* dy, orca_hip_storage* x, size_t rows, size_t cols,
                              int kind, float eps, orca_hip_storage* weight, orca_hip_storage* dx_add,
                              orca_hip_storage** dx, orca_hip_storage** dweight, orca_hip_storage** dbias) {
  const size_t mn = element_count(rows, cols);
  return be_run(be,
                {{dy, mn, "norm_backward (dy)"},
                 {x, mn, "norm_backward (x)"},
                 {weight, cols, "norm_backward (weight)", true},
                 {dx_add, mn, "norm_backward (dx_add)", true}},
                {{mn, dx, true}, {cols, dweight, true}, {cols, dbias, true}},
                [&](orca_hip_ctx* ctx, float* const* i, float* const* o) {
                  const orca_hip_norm_params n{kind, eps, i[2], nullptr};
                  return orca_hip_norm_backward(ctx, rows, cols, i[0], cols, i[1], cols, &n, i[3], cols, o[0], cols,
                                                o[1], o[2]);
                });
}

int orca_hip_be_dropout(orca_hip_backend* be, orca_hip_storage* x, size_t rows, size_t cols, double p, uint64_t seed,
                        uint64_t offset, orca_hip_storage** y) {
  const size_t mn = element_count(rows, cols);
  return be_run(be, {{x, mn, "dropout"}}, {{mn, y}}, [&](orca_hip_ctx* ctx, float* const* i, float* const* o) {
    return orca_hip_dropout(ctx, rows, cols, i[0], cols, p, seed, offset, o[0], cols);
  });
}

int orca_hip_be_residual_norm(orca_hip_backend* be, orca_hip_storage* x, orca_hip_storage* f, size_t rows, size_t cols,
                              const orca_hip_be_residual_block* block, orca_hip_storage** y, orca_hip_storage** u,
                              orca_hip_storage** u8) {
  if (!block) return null_block("residual_norm");
  const size_t mn = element_count(rows, cols);
  const orca_hip_be_residual_block& b = *block;
  return be_run(be,
                {{x, mn, "residual_norm (x)"},
                 {f, mn, "residual_norm (f)"},
                 {b.post_weight, cols, "residual_norm (post weight)", true},
                 {b.post_bias, cols, "residual_norm (post bias)", true},
                 {b.next_weight, cols, "residual_norm (next weight)", true},
                 {b.next_bias, cols, "residual_norm (next bias)", true},
                 {b.gate, element_count(b.groups, cols), "residual_norm (gate)", true}},
                {{mn, y}, {mn, u, true}, {packed_count(rows, cols), u8, true}},
                [&](orca_hip_ctx* ctx, float* const* i, float* const* o) {
                  const orca_hip_residual_block p = block_of(b, i[2], i[3], i[4], i[5], i[6], cols);
                  return orca_hip_residual_norm(ctx, rows, cols, i[0], cols, i[1], cols, &p, o[0], cols, o[1], cols,
                                                o[2]);
                });
}

int orca_hip_be_residual_norm_backward(orca_hip_backend* be, orca_hip_storage* dy, orca_hip_storage* du,
                                       orca_hip_storage* f, orca_hip_storage* y, size_t rows, size_t cols,
                                       const orca_hip_be_residual_block* block, orca_hip_storage** dx,
                                       orca_hip_storage** df, orca_hip_storage** dgate, orca_hip_storage** dpost_weight,
                                       orca_hip_storage** dpost_bias, orca_hip_storage** dnext_weight,
                                       orca_hip_storage** dnext_bias) {
  if (!block) return null_block("residual_norm_backward");
  const size_t mn = element_count(rows, cols);
  const orca_hip_be_residual_block& b = *block;
  const size_t gn = element_count(b.groups, cols);
  return be_run(be,
                {{dy, mn, "residual_norm_backward (dy)", true},
                 {du, mn, "residual_norm_backward (du)", true},
                 {f, mn, "residual_norm_backward (f)", true},
                 {y, mn, "residual_norm_backward (y)", true},
                 {b.post_weight, cols, "residual_norm_backward (post weight)", true},
                 {b.post_bias, cols, "residual_norm_backward (post bias)", true},
                 {b.next_weight, cols, "residual_norm_backward (next weight)", true},
                 {b.next_bias, cols, "residual_norm_backward (next bias)", true},
                 {b.gate, gn, "residual_norm_backward (gate)", true}},
                {{mn, dx, true},
                 {mn, df, true},
                 {gn, dgate, true},
                 {cols, dpost_weight, true},
                 {cols, dpost_bias, true},
                 {cols, dnext_weight, true},
                 {cols, dnext_bias, true}},
                [&](orca_hip_ctx* ctx, float* const* i, float* const* o) {
                  const orca_hip_residual_block p = block_of(b, i[4], i[5], i[6], i[7], i[8], cols);
                  orca_hip_residual_grads g{};
                  g.dx = o[0];
                  g.df = o[1];
                  g.dgate = o[2];
                  g.lddx = g.lddf = g.lddgate = cols;
                  g.dpost_weight = o[3];
                  g.dpost_bias = o[4];
                  g.dnext_weight = o[5];
                  g.dnext_bias = o[6];
                  return orca_hip_residual_norm_backward(ctx, rows, cols, i[0], cols, i[1], cols, i[2], cols, i[3], cols,
                                                         &p, &g);
                });
}

}  // extern "C"
