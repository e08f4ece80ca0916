// A Linear with its activation and residual in the product's epilogue, and its backward
// (orca_hip_linear_act, orca_hip_linear_act_backward).  The products run on the bf16 matrix
// instructions at fp32 precision (split_product.hpp).
#include <algorithm>
#include <memory>
#include <string>

#include "act8.hpp"
#include "activation.hpp"
#include "runtime.hpp"
#include "split_product.hpp"

namespace orca_hip {

void act8_aligned(const void* packed, const char* what);

namespace {

// What becomes of a product: z = acc + bias, y = act(z) + residual.  The residual may be y itself.
struct LinearOut {
  int act = ORCA_HIP_ACT_NONE;
  const float* bias = nullptr;
  const float* residual = nullptr;
  int64_t ldr = 0;
  float* pre = nullptr;
  int64_t ldpre = 0;
  float* y = nullptr;
  int64_t ldy = 0;
  Act8 pre8, y8;
};

struct ProductArgs {
  ProductOperand A, B;
  int64_t M, N, K;
  int tiles_m, tiles_n, splits;
  int64_t chunk;  // k values per split, a multiple of every stage's
  float* ws;      // splits > 1: [split][M][N]
  LinearOut out;
};

// Four neighbouring columns of one row; `have` of them exist.
__device__ __forceinline__ floatx4 load_quad(const float* p, int have) {
  if (have == 4) return *reinterpret_cast<const floatx4_u*>(p);
  floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < have) v[j] = p[j];
  return v;
}
__device__ __forceinline__ void store_quad(float* p, int have, floatx4 v) {
  if (have == 4) {
    *reinterpret_cast<floatx4_u*>(p) = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < have) p[j] = v[j];
}
__device__ __forceinline__ void store_codes(int8_t* p, int have, floatx4 v, uint32_t b) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) w |= ((uint32_t)act8_code(v[j], b) & 255u) << (8 * j);
  if (have == 4) {
    typedef uint32_t word_u __attribute__((aligned(1)));
    *reinterpret_cast<word_u*>(p) = w;
    return;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < have) p[j] = (int8_t)(w >> (8 * j));
}
__device__ __forceinline__ uint32_t quad_top(floatx4 v, int have) {
  uint32_t t = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) t = max(t, j < have ? act8_magnitude(v[j]) : 0u);
  return t;
}
__device__ __forceinline__ floatx4 activate(int act, floatx4 z) {
  floatx4 y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = activation(act, z[j]);
  return y;
}

// A lane's part of a 32 x 32 block: row m, columns n + 8 q .. + 3 for q = 0 .. 3 (n past the half
// wave's four).  The other half wave holds the row's other 16 columns.
__device__ __forceinline__ void block_out(const LinearOut& o, const acc32& acc, int64_t m, int64_t n, int64_t M,
                                          int64_t N) {
  const bool row = m < M;
  uint32_t ztop = 0, ytop = 0;
  floatx4 z[4], y[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int64_t c = n + 8 * q;
    const int have = row ? (int)max((int64_t)0, min((int64_t)4, N - c)) : 0;
    z[q] = floatx4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
    if (o.bias) z[q] = z[q] + load_quad(o.bias + c, have);
    y[q] = activate(o.act, z[q]);
    if (o.residual) y[q] = y[q] + load_quad(o.residual + m * o.ldr + c, have);
    ztop = max(ztop, quad_top(z[q], have));
    ytop = max(ytop, quad_top(y[q], have));
  }
  uint32_t zb = 0, yb = 0;
  if (o.pre8.codes) zb = act8_byte(max(ztop, (uint32_t)__shfl_xor((int)ztop, 32)));
  if (o.y8.codes) yb = act8_byte(max(ytop, (uint32_t)__shfl_xor((int)ytop, 32)));
  if (!row) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int64_t c = n + 8 * q;
    const int have = (int)max((int64_t)0, min((int64_t)4, N - c));
    if (o.pre) store_quad(o.pre + m * o.ldpre + c, have, z[q]);
    store_quad(o.y + m * o.ldy + c, have, y[q]);
    if (o.pre8.codes) store_codes(o.pre8.codes + m * o.pre8.cols + c, have, z[q], zb);
    if (o.y8.codes) store_codes(o.y8.codes + m * o.y8.cols + c, have, y[q], yb);
  }
  if (n % 32 == 0 && n < N) {
    if (o.pre8.codes) o.pre8.scales[n / 32 * o.pre8.ld + m] = (uint8_t)zb;
    if (o.y8.codes) o.y8.scales[n / 32 * o.y8.ld + m] = (uint8_t)yb;
  }
}

template <class T, template <int, int, int> class LoadA, template <int, int, int> class LoadB>
__global__ void __launch_bounds__(T::THREADS, T::OCC* T::THREADS / 256) split_product_kernel(ProductArgs p) {
  using LA = LoadA<T::BM, T::BK, T::THREADS>;
  using LB = LoadB<T::BN, T::BK, T::THREADS>;
  __shared__ u32x4 smem[2 * (LA::UNITS + LB::UNITS)];
  // Consecutive blocks go to the 8 XCDs in turn: each XCD takes a run of tiles, eight tile rows
  // by column, so that its blocks share the operand panels in its L2.
  const int nb = gridDim.x, x = blockIdx.x % 8, lin = x * (nb / 8) + min(x, nb % 8) + blockIdx.x / 8;
  const int tiles = p.tiles_m * p.tiles_n, split = lin / tiles, tile = lin % tiles;
  const int width = 8 * p.tiles_n, first = tile / width * 8, rows = min(8, p.tiles_m - first);
  const int m0 = (first + tile % width % rows) * T::BM, n0 = tile % width / rows * T::BN;
  acc32 acc[T::FM][T::FN];
  product<T, LA, LB>(p.A, p.B, m0, n0, split * p.chunk, min(p.K, (split + 1) * p.chunk), smem, acc);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t m = m0 + wave / T::WN * (T::FM * 32) + (lane & 31);
  const int64_t n = n0 + wave % T::WN * (T::FN * 32) + (lane >> 5) * 4;
#pragma unroll
  for (int i = 0; i < T::FM; ++i)
#pragma unroll
    for (int j = 0; j < T::FN; ++j) {
      if (p.splits == 1) {
        block_out(p.out, acc[i][j], m + 32 * i, n + 32 * j, p.M, p.N);
        continue;
      }
      if (m + 32 * i >= p.M) continue;
      float* w = p.ws + ((int64_t)split * p.M + m + 32 * i) * p.N;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t c = n + 32 * j + 8 * q;
        store_quad(w + c, (int)max((int64_t)0, min((int64_t)4, p.N - c)),
                   floatx4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]});
      }
    }
}

// The splits' partial products, added in split order, and the epilogue.  A lane takes four columns,
// eight lanes a checkpoint's group of 32.
__global__ void __launch_bounds__(256) split_product_finish_kernel(ProductArgs p) {
  const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t c = (int64_t)blockIdx.y * 256 + (threadIdx.x & 63) * 4;
  if (m >= p.M) return;  // a whole wave
  const LinearOut& o = p.out;
  const int have = (int)max((int64_t)0, min((int64_t)4, p.N - c));
  floatx4 z = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < p.splits; ++s) z = z + load_quad(p.ws + ((int64_t)s * p.M + m) * p.N + c, have);
  if (o.bias) z = z + load_quad(o.bias + c, have);
  floatx4 y = activate(o.act, z);
  if (o.residual) y = y + load_quad(o.residual + m * o.ldr + c, have);
  auto group = [](uint32_t top) {
    for (int d = 1; d < 8; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    return act8_byte(top);
  };
  uint32_t zb = 0, yb = 0;
  if (o.pre8.codes) zb = group(quad_top(z, have));
  if (o.y8.codes) yb = group(quad_top(y, have));
  if (o.pre) store_quad(o.pre + m * o.ldpre + c, have, z);
  store_quad(o.y + m * o.ldy + c, have, y);
  const bool lead = (threadIdx.x & 7) == 0 && c < p.N;
  if (o.pre8.codes) {
    store_codes(o.pre8.codes + m * o.pre8.cols + c, have, z, zb);
    if (lead) o.pre8.scales[c / 32 * o.pre8.ld + m] = (uint8_t)zb;
  }
  if (o.y8.codes) {
    store_codes(o.y8.codes + m * o.y8.cols + c, have, y, yb);
    if (lead) o.y8.scales[c / 32 * o.y8.ld + m] = (uint8_t)yb;
  }
}

// dz = dy * act'(z) (z in fp32, or its checkpoint) and, per block of 64 rows, the column sums of dz.
// A thread takes four columns of 16 rows.
constexpr int kSlopeRows = 64;
__global__ void __launch_bounds__(256) slope_kernel(const float* __restrict__ dy, int64_t lddy, int act,
                                                    const float* __restrict__ z, int64_t ldz, Act8 z8,
                                                    float* __restrict__ dz, float* __restrict__ partial, int64_t M,
                                                    int64_t N) {
  __shared__ floatx4 sums[4][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t c = (int64_t)blockIdx.y * 256 + lane * 4, r0 = (int64_t)blockIdx.x * kSlopeRows + wave * 16;
  const int have = (int)max((int64_t)0, min((int64_t)4, N - c));
  floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int r = 0; r < 16; ++r) {
    const int64_t m = r0 + r;
    if (m >= M || have == 0) break;
    floatx4 g = load_quad(dy + m * lddy + c, have);
    if (act != ORCA_HIP_ACT_NONE) {
      floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (z8.codes) {
        const float step = act8_step(z8.scales[c / 32 * z8.ld + m]);
        for (int j = 0; j < 4; ++j)
          if (j < have) v[j] = (float)z8.codes[m * z8.cols + c + j] * step;
      } else {
        v = load_quad(z + m * ldz + c, have);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = g[j] * activation_slope(act, v[j]);
      store_quad(dz + m * N + c, have, g);
    }
    sum = sum + g;
  }
  if (!partial) return;
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave == 0)
    store_quad(partial + (int64_t)blockIdx.x * N + c, have, sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane]);
}

// db[n] = the sum of the blocks' column sums: 8 runs of blocks, each in order, then the runs in order.
__global__ void __launch_bounds__(256) slope_finish_kernel(const float* __restrict__ partial, int64_t blocks, int64_t N,
                                                           float* __restrict__ db) {
  __shared__ float sums[8][32];
  const int64_t n = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int run = threadIdx.x >> 5;
  const int64_t per = (blocks + 7) / 8, end = min(blocks, (run + 1) * per);
  float s = 0.0f;
  if (n < N)
    for (int64_t b = run * per; b < end; ++b) s = s + partial[b * N + n];
  sums[run][threadIdx.x & 31] = s;
  __syncthreads();
  if (run == 0 && n < N) {
    for (int i = 1; i < 8; ++i) s = s + sums[i][threadIdx.x];
    db[n] = s;
  }
}


dim3 quad_grid(int64_t rows, int64_t per, int64_t cols, const char* op) {
  const int64_t gx = (rows + per - 1) / per, gy = (cols + 255) / 256;
  if (gx > 0x7fffffff || gy > 65535) fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": matrix too large");
  return dim3((unsigned)gx, (unsigned)gy);
}

enum class Load { kFast, kSlow, kCodes };

using Tile128 = ProductTile<128, 128, 2, 2, 16, 2>;

template <class T>
void launch_tile(orca_hip_ctx* ctx, Load a, Load b, unsigned grid, const ProductArgs& p) {
  const dim3 threads(T::THREADS);
  if (a == Load::kFast && b == Load::kSlow)
    hipLaunchKernelGGL((split_product_kernel<T, LoadKFast, LoadKSlow>), dim3(grid), threads, 0, ctx->stream, p);
  else if (a == Load::kFast && b == Load::kFast)
    hipLaunchKernelGGL((split_product_kernel<T, LoadKFast, LoadKFast>), dim3(grid), threads, 0, ctx->stream, p);
  else if (a == Load::kSlow)
    hipLaunchKernelGGL((split_product_kernel<T, LoadKSlow, LoadKSlow>), dim3(grid), threads, 0, ctx->stream, p);
  else
    hipLaunchKernelGGL((split_product_kernel<T, LoadCodes, LoadKSlow>), dim3(grid), threads, 0, ctx->stream, p);
  ORCA_HIP_CHECK(hipGetLastError());
}

// out = the product of A [M][K] and B [N][K] with its epilogue.
void product(orca_hip_ctx* ctx, const char* name, Load la, const ProductOperand& A, Load lb, const ProductOperand& B,
             int64_t M, int64_t N, int64_t K, const LinearOut& out) {
  ProductArgs p{};
  p.A = A;
  p.B = B;
  p.M = M;
  p.N = N;
  p.K = K;
  p.out = out;
  const int64_t tm = (M + 127) / 128, tn = (N + 127) / 128;
  if (tm > 0x7fffffff / tn / 64) fail(ORCA_HIP_ERR_INTERNAL, std::string(name) + ": matrix too large");
  p.tiles_m = (int)tm;
  p.tiles_n = (int)tn;
  // too few tiles for the CUs: k in even runs of at least 64 values
  int64_t splits = std::max<int64_t>(1, std::min<int64_t>({2 * ctx->num_cus / (tm * tn), K / 64, 64}));
  p.chunk = std::max<int64_t>(64, ((K + splits - 1) / splits + 63) / 64 * 64);
  p.splits = (int)std::max<int64_t>(1, (K + p.chunk - 1) / p.chunk);
  std::unique_ptr<Scratch> ws;
  if (p.splits > 1) {
    ws.reset(new Scratch(ctx, sizeof(float) * (size_t)p.splits * M * N));
    p.ws = ws->as<float>();
  }
  std::string pname;
  if (ctx->prof.enabled)
    pname = std::string(name) + " " + std::to_string(M) + "x" + std::to_string(N) + "x" + std::to_string(K);
  ProfScope prof(ctx, pname.c_str(), 2.0 * M * N * K, 4.0 * ((double)M * K + (double)K * N + (double)M * N));
  launch_tile<Tile128>(ctx, la, lb, (unsigned)(tm * tn * p.splits), p);
  if (p.splits > 1) {
    hipLaunchKernelGGL(split_product_finish_kernel, quad_grid(M, 4, N, name), dim3(256), 0, ctx->stream, p);
    ORCA_HIP_CHECK(hipGetLastError());
  }
}

void check_ld(const char* what, size_t ld, size_t cols) {
  if (ld < cols) fail_shape(what, "a leading dimension of at least " + std::to_string(cols), std::to_string(ld));
}
void check_sizes(const char* op, size_t M, size_t N, size_t K) {
  for (size_t v : {M, N, K})
    if (v > 0x7fffff00u) fail_shape(op, "sizes below 2^31", std::to_string(v));
}
// A result must not lie in what the call still reads (or in another result).
void check_apart(const char* op, const void* out, size_t out_bytes, const void* in, size_t in_bytes) {
  const auto a = reinterpret_cast<uintptr_t>(out), b = reinterpret_cast<uintptr_t>(in);
  if (out && in && out_bytes && in_bytes && a < b + in_bytes && b < a + out_bytes)
    fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": an output overlaps another operand");
}
struct Span {
  const void* p;
  size_t bytes;
};
void check_act(const char* op, int act) {
  if (act < ORCA_HIP_ACT_NONE || act > ORCA_HIP_ACT_SILU)
    fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": unknown activation " + std::to_string(act));
}

}  // namespace
}  // namespace orca_hip

using namespace orca_hip;

extern "C" {

int orca_hip_linear_act(orca_hip_ctx* ctx, size_t M, size_t N, size_t K, const float* X, size_t ldx, const float* W,
                        size_t ldw, float* Y, size_t ldy, const orca_hip_linear_epilogue* epi) {
  return guard([&] {
    const char* op = "linear_act";
    check_sizes(op, M, N, K);
    check_ld("linear_act (x)", ldx, K);
    check_ld("linear_act (weight)", ldw, N);
    check_ld("linear_act (y)", ldy, N);
    const orca_hip_linear_epilogue none{};
    const orca_hip_linear_epilogue& e = epi ? *epi : none;
    check_act(op, e.act);
    if (e.residual) check_ld("linear_act (residual)", e.ldr, N);
    if (e.pre) check_ld("linear_act (pre)", e.ldpre, N);
    if (M && N && (!Y || (K && (!X || !W)))) fail(ORCA_HIP_ERR_INTERNAL, "linear_act: null operand");
    const size_t p8 = act8_layout(M, N).bytes;
    const Span x{X, matrix_bytes(M, K, ldx)}, w{W, matrix_bytes(K, N, ldw)}, b{e.bias, N * sizeof(float)},
        r{e.residual, matrix_bytes(M, N, e.ldr)}, y{Y, matrix_bytes(M, N, ldy)}, pre{e.pre, matrix_bytes(M, N, e.ldpre)},
        z8{e.pre8, p8}, y8{e.y8, p8};
    const Span outs[4] = {y, pre, z8, y8};
    for (int i = 0; i < 4; ++i) {
      for (const Span& s : {x, w, b}) check_apart(op, outs[i].p, outs[i].bytes, s.p, s.bytes);
      // y over its own residual, element by element, is in order
      if (!(i == 0 && e.residual == Y && e.ldr == ldy)) check_apart(op, outs[i].p, outs[i].bytes, r.p, r.bytes);
      for (int j = 0; j < i; ++j) check_apart(op, outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes);
    }
    act8_aligned(e.pre8, "linear_act (pre8)");
    act8_aligned(e.y8, "linear_act (y8)");
    bind(ctx);
    if (!M || !N) return;
    check_extent(ctx, x.p, x.bytes, "linear_act (x)");
    check_extent(ctx, w.p, w.bytes, "linear_act (weight)");
    check_extent(ctx, b.p, b.bytes, "linear_act (bias)");
    check_extent(ctx, r.p, r.bytes, "linear_act (residual)");
    check_extent(ctx, y.p, y.bytes, "linear_act (y)");
    check_extent(ctx, pre.p, pre.bytes, "linear_act (pre)");
    check_extent(ctx, z8.p, z8.bytes, "linear_act (pre8)");
    check_extent(ctx, y8.p, y8.bytes, "linear_act (y8)");
    LinearOut o;
    o.act = e.act;
    o.bias = e.bias;
    o.residual = e.residual;
    o.ldr = (int64_t)e.ldr;
    o.pre = e.pre;
    o.ldpre = (int64_t)e.ldpre;
    o.y = Y;
    o.ldy = (int64_t)ldy;
    o.pre8 = act8_at(e.pre8, M, N);
    o.y8 = act8_at(e.y8, M, N);
    product(ctx, op, Load::kFast, ProductOperand{X, (int64_t)ldx, (int)M, nullptr, 0}, Load::kSlow,
            ProductOperand{W, (int64_t)ldw, (int)N, nullptr, 0}, (int64_t)M, (int64_t)N, (int64_t)K, o);
  });
}

int orca_hip_linear_act_backward(orca_hip_ctx* ctx, size_t M, size_t N, size_t K, const float* dY, size_t lddy,
                                 const float* W, size_t ldw, const orca_hip_linear_saved* saved, float* dX,
                                 size_t lddx, float* dW, size_t lddw, float* db) {
  return guard([&] {
    const char* op = "linear_act_backward";
    check_sizes(op, M, N, K);
    const orca_hip_linear_saved none{};
    const orca_hip_linear_saved& s = saved ? *saved : none;
    check_act(op, s.act);
    const bool slope = s.act != ORCA_HIP_ACT_NONE;
    check_ld("linear_act_backward (dy)", lddy, N);
    if (dX) check_ld("linear_act_backward (weight)", ldw, N);
    if (dX) check_ld("linear_act_backward (dx)", lddx, K);
    if (dX && s.dx_add) check_ld("linear_act_backward (dx_add)", s.ldadd, K);
    if (dW) check_ld("linear_act_backward (dw)", lddw, N);
    if (slope && s.z) check_ld("linear_act_backward (z)", s.ldz, N);
    if (dW && s.x) check_ld("linear_act_backward (x)", s.ldx, K);
    if (slope && M && N && !s.z == !s.z8)
      fail(ORCA_HIP_ERR_INTERNAL, "linear_act_backward: one of z and z8 is needed");
    if (dW && M && N && K && !s.x == !s.x8)
      fail(ORCA_HIP_ERR_INTERNAL, "linear_act_backward: one of x and x8 is needed for dw");
    if (M && N && !dY) fail(ORCA_HIP_ERR_INTERNAL, "linear_act_backward: null dy");
    if (dX && M && N && K && !W) fail(ORCA_HIP_ERR_INTERNAL, "linear_act_backward: null weight");
    const Span dy{dY, matrix_bytes(M, N, lddy)}, w{dX ? W : nullptr, matrix_bytes(K, N, ldw)},
        z{slope ? s.z : nullptr, matrix_bytes(M, N, s.ldz)}, z8{slope ? s.z8 : nullptr, act8_layout(M, N).bytes},
        x{dW ? s.x : nullptr, matrix_bytes(M, K, s.ldx)}, x8{dW ? s.x8 : nullptr, act8_layout(M, K).bytes},
        add{dX ? s.dx_add : nullptr, matrix_bytes(M, K, s.ldadd)}, dx{dX, matrix_bytes(M, K, lddx)},
        dw{dW, matrix_bytes(K, N, lddw)}, dbs{db, N * sizeof(float)};
    const Span outs[3] = {dx, dw, dbs};
    for (int i = 0; i < 3; ++i) {
      for (const Span& in : {dy, w, z, z8, x, x8}) check_apart(op, outs[i].p, outs[i].bytes, in.p, in.bytes);
      // dx over dx_add, element by element, is in order (a gradient added up in place)
      if (!(i == 0 && s.dx_add == dX && s.ldadd == lddx)) check_apart(op, outs[i].p, outs[i].bytes, add.p, add.bytes);
      for (int j = 0; j < i; ++j) check_apart(op, outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes);
    }
    act8_aligned(z8.p, "linear_act_backward (z8)");
    act8_aligned(x8.p, "linear_act_backward (x8)");
    bind(ctx);
    check_extent(ctx, dy.p, dy.bytes, "linear_act_backward (dy)");
    check_extent(ctx, w.p, w.bytes, "linear_act_backward (weight)");
    check_extent(ctx, z.p, z.bytes, "linear_act_backward (z)");
    check_extent(ctx, z8.p, z8.bytes, "linear_act_backward (z8)");
    check_extent(ctx, x.p, x.bytes, "linear_act_backward (x)");
    check_extent(ctx, x8.p, x8.bytes, "linear_act_backward (x8)");
    check_extent(ctx, add.p, add.bytes, "linear_act_backward (dx_add)");
    check_extent(ctx, dx.p, dx.bytes, "linear_act_backward (dx)");
    check_extent(ctx, dw.p, dw.bytes, "linear_act_backward (dw)");
    check_extent(ctx, db, dbs.bytes, "linear_act_backward (db)");
    const bool want_dx = dX && M && K, want_dw = dW && K && N, want_db = db && N;
    const float* dz = dY;
    int64_t lddz = (int64_t)lddy;
    std::unique_ptr<Scratch> dzs, partial;
    const int64_t blocks = ((int64_t)M + kSlopeRows - 1) / kSlopeRows;
    if (N && (want_db || (slope && (want_dx || want_dw)))) {
      if (slope && M) {
        dzs.reset(new Scratch(ctx, sizeof(float) * M * N));
        dz = dzs->as<float>();
        lddz = (int64_t)N;
      }
      if (want_db && M) partial.reset(new Scratch(ctx, sizeof(float) * (size_t)blocks * N));
      ProfScope prof(ctx, "linear_act_slope", 0.0, (slope ? 12.0 : 4.0) * M * N);
      if (M) {
        hipLaunchKernelGGL(slope_kernel, quad_grid((int64_t)M, kSlopeRows, (int64_t)N, op), dim3(256), 0, ctx->stream,
                           dY, (int64_t)lddy, s.act, static_cast<const float*>(z.p), (int64_t)s.ldz,
                           act8_at(const_cast<void*>(z8.p), M, N), dzs ? dzs->as<float>() : nullptr,
                           partial ? partial->as<float>() : nullptr, (int64_t)M, (int64_t)N);
        ORCA_HIP_CHECK(hipGetLastError());
      }
      if (want_db) {
        hipLaunchKernelGGL(slope_finish_kernel, dim3((unsigned)((N + 31) / 32)), dim3(256), 0, ctx->stream,
                           partial ? partial->as<float>() : nullptr, M ? blocks : 0, (int64_t)N, db);
        ORCA_HIP_CHECK(hipGetLastError());
      }
    }
    if (want_dx) {
      LinearOut o;
      o.residual = s.dx_add;
      o.ldr = (int64_t)s.ldadd;
      o.y = dX;
      o.ldy = (int64_t)lddx;
      product(ctx, "linear_act_dx", Load::kFast, ProductOperand{dz, lddz, (int)M, nullptr, 0}, Load::kFast,
              ProductOperand{W, (int64_t)ldw, (int)K, nullptr, 0}, (int64_t)M, (int64_t)K, (int64_t)N, o);
    }
    if (want_dw) {
      LinearOut o;
      o.y = dW;
      o.ldy = (int64_t)lddw;
      ProductOperand a{s.x, (int64_t)s.ldx, (int)K, nullptr, 0};
      if (s.x8) {
        const Act8 q = act8_at(const_cast<void*>(s.x8), M, K);
        a = ProductOperand{q.codes, q.cols, (int)K, q.scales, q.ld};
      }
      product(ctx, "linear_act_dw", s.x8 ? Load::kCodes : Load::kSlow, a, Load::kSlow,
              ProductOperand{dz, lddz, (int)N, nullptr, 0}, (int64_t)K, (int64_t)N, (int64_t)M, o);
    }
  });
}

}  // extern "C"
