// A Linear with its activation and residual in the product's epilogue, and its backward
// (orca_hip_linear_act, orca_hip_linear_act_backward).  The products run on the bf16 matrix
// instructions at fp32 precision (split_product.hpp).
#include <algorithm>
#include <memory>
#include <string>

#include "act8.hpp"
#include "activation.hpp"
#include "operand.hpp"
#include "quad.hpp"
#include "runtime.hpp"
#include "split_product.hpp"

namespace orca_hip {
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

// The epilogue of a quad of row m (`row`: the row exists).  Eight neighbouring lanes hold a checkpoint's
// group of 32 columns.
__device__ __forceinline__ void quad_out(const LinearOut& o, floatx4 z, floatx4 bias, floatx4 residual, int64_t m,
                                         const Quad& q, bool row) {
  if (o.bias) {
    settle(q, bias);
    z = z + bias;
  }
  floatx4 y;
  activations<4>(o.act, z, y);
  if (o.residual) {
    settle(q, residual);
    y = y + residual;
  }
  uint32_t zb = 0, yb = 0;
  if (o.pre8.codes) zb = quad_byte(z, q);
  if (o.y8.codes) yb = quad_byte(y, q);
  if (!row || q.have == 0) return;
  if (o.pre) store_quad(o.pre + m * o.ldpre, q, z);
  store_quad(o.y + m * o.ldy, q, y);
  if (o.pre8.codes) {
    store_codes(o.pre8.codes + m * o.pre8.cols, q, z, zb);
    if (q.c % 32 == 0) o.pre8.scales[q.group * o.pre8.ld + m] = (uint8_t)zb;
  }
  if (o.y8.codes) {
    store_codes(o.y8.codes + m * o.y8.cols, q, y, yb);
    if (q.c % 32 == 0) o.y8.scales[q.group * o.y8.ld + m] = (uint8_t)yb;
  }
}
__device__ __forceinline__ floatx4 bias_quad(const LinearOut& o, const Quad& q) {
  return o.bias ? load_quad(o.bias, q) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
}
__device__ __forceinline__ floatx4 residual_quad(const LinearOut& o, int64_t m, const Quad& q) {
  return o.residual ? load_quad(o.residual + m * o.ldr, q) : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
}

template <class T, template <int, int, int> class LoadA, template <int, int, int> class LoadB>
constexpr int tile_units() {
  return 2 * (LoadA<T::BM, T::BK, T::THREADS>::UNITS + LoadB<T::BN, T::BK, T::THREADS>::UNITS);
}

// Block `block` of `blocks` of one product.
template <class T, template <int, int, int> class LoadA, template <int, int, int> class LoadB>
__device__ __forceinline__ void tile_product(const ProductArgs& p, int block, int blocks, u32x4* __restrict__ smem) {
  using LA = LoadA<T::BM, T::BK, T::THREADS>;
  using LB = LoadB<T::BN, T::BK, T::THREADS>;
  // Consecutive blocks go to the 8 XCDs in turn: each XCD takes a run of tiles, eight tile rows
  // by column, so that its blocks share the operand panels in its L2.
  const int x = block % 8, lin = x * (blocks / 8) + min(x, blocks % 8) + block / 8;
  const int tiles = p.tiles_m * p.tiles_n, split = lin / tiles, tile = lin % tiles;
  const int width = 8 * p.tiles_n, first = tile / width * 8, rows = min(8, p.tiles_m - first);
  const int m0 = (first + tile % width % rows) * T::BM, n0 = tile % width / rows * T::BN;
  acc32 acc[T::FM][T::FN];
  product<T, LA, LB>(p.A, p.B, m0, n0, split * p.chunk, min(p.K, (split + 1) * p.chunk), smem, acc);
  // The tile leaves through LDS, a 32 x 32 block of each wave at a time: a lane's four rows of four
  // columns lie along the rows then (whole lines to and from memory, and a checkpoint's group in eight
  // lanes), and the epilogue is one piece of code instead of one per block.
  constexpr int PITCH = 36;
  static_assert(T::THREADS / 64 * 32 * PITCH / 4 <= tile_units<T, LoadA, LoadB>(), "the waves' blocks fit the stages");
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  float* stage = reinterpret_cast<float*>(smem) + wave * 32 * PITCH;
#pragma unroll 1
  for (int b = 0; b < T::FM * T::FN; ++b) {
#pragma unroll
    for (int i = 0; i < T::FM * T::FN; ++i)
      if (i == b) {
        const acc32& v = acc[i / T::FN][i % T::FN];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<floatx4*>(stage + (lane & 31) * PITCH + 8 * q + (lane >> 5) * 4) =
              floatx4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
      }
    const int64_t m = m0 + wave / T::WN * (T::FM * 32) + b / T::FN * 32 + lane / 8;
    const Quad quad = quad_of(n0 + wave % T::WN * (T::FN * 32) + b % T::FN * 32 + lane % 8 * 4, p.N);
    floatx4 bias = {0.0f, 0.0f, 0.0f, 0.0f}, res[4];
    if (p.splits == 1) {
      bias = bias_quad(p.out, quad);
#pragma unroll
      for (int q = 0; q < 4; ++q) res[q] = residual_quad(p.out, min(m + 8 * q, p.M - 1), quad);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t r = m + 8 * q;
      const floatx4 z = *reinterpret_cast<const floatx4*>(stage + (lane / 8 + 8 * q) * PITCH + lane % 8 * 4);
      if (p.splits == 1)
        quad_out(p.out, z, bias, res[q], r, quad, r < p.M);
      else if (r < p.M)
        store_quad(p.ws + ((int64_t)split * p.M + r) * p.N, quad, z);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

template <class T>
__global__ void __launch_bounds__(T::THREADS, T::OCC* T::THREADS / 256) linear_act_kernel(ProductArgs p) {
  __shared__ u32x4 smem[tile_units<T, LoadKFast, LoadKSlow>()];
  tile_product<T, LoadKFast, LoadKSlow>(p, blockIdx.x, gridDim.x, smem);
}

// A quad of row m of a slope operand's z, as it is loaded and as it is used.
struct SlopeQuad {
  floatx4 z;
  uint32_t codes, byte;
};
__device__ __forceinline__ void load_slope(const ProductOperand& o, int64_t m, const Quad& q, SlopeQuad& s) {
  if (o.act == ORCA_HIP_ACT_NONE) return;
  if (o.z8.codes) {
    s.codes = load_codes(o.z8.codes + m * o.z8.cols, q);
    s.byte = o.z8.scales[q.group * o.z8.ld + m];
  } else {
    s.z = load_quad(o.z + m * o.ldz, q);
  }
}
__device__ __forceinline__ void apply_slope(const ProductOperand& o, const Quad& q, SlopeQuad& s, floatx4& g) {
  if (o.act == ORCA_HIP_ACT_NONE) return;
  if (o.z8.codes)
    s.z = settle_codes(q, s.codes, s.byte);
  else
    settle(q, s.z);
  activation_slopes<4>(o.act, s.z, g);
}

// The backward's two products and the last step of the bias gradient, each a run of blocks.
struct BackwardArgs {
  ProductArgs dx, dw;
  int dx_blocks, dw_blocks;  // the rest: db
  const float* partial;      // [partials][N]
  int64_t partials, N;
  float* db;
  ProductOperand dz;         // dz inside the products: dy and z
  int64_t M;
};

// db[n] = the sum of the slope kernel's column sums: RUNS runs of blocks, each in order, eight loads at a time, then
// the runs in order.
template <int RUNS>
__device__ __forceinline__ void finish_bias(const BackwardArgs& p, int block, float* __restrict__ sums) {
  const int64_t n = (int64_t)block * 32 + (threadIdx.x & 31);
  const int run = threadIdx.x >> 5;
  const int64_t per = (p.partials + RUNS - 1) / RUNS, end = min(p.partials, (run + 1) * per);
  const float* column = p.partial + min(n, p.N - 1);
  float s = 0.0f;
  for (int64_t b = run * per; b < end; b += 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = column[min(b + i, end - 1) * p.N];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (b + i < end) s = s + v[i];
  }
  sums[threadIdx.x] = s;
  __syncthreads();
  if (run == 0 && n < p.N) {
    for (int i = 1; i < RUNS; ++i) s = s + sums[32 * i + threadIdx.x];
    p.db[n] = s;
  }
}

#include "row_product.hpp"

// The same with dX on tiles of 64 and dW for a few rows.
template <class T, int MR>
__global__ void __launch_bounds__(256, T::OCC) row_backward_kernel(BackwardArgs p) {
  static_assert(T::THREADS == 256, "row_dw's block");
  __shared__ u32x4 smem[tile_units<T, LoadKFast, LoadKFast>()];
  const int block = blockIdx.x;
  if (block < p.dx_blocks)
    tile_product<T, LoadKFast, LoadKFast>(p.dx, block, p.dx_blocks, smem);
  else
    row_dw<MR, false>(p.dw, block - p.dx_blocks, reinterpret_cast<float*>(smem));
}

// Column sums of dz = dy * act'(z), 16 columns a block: 16 threads for each, every sixteenth row, eight rows'
// loads at a time, and the threads' sums in order.
constexpr int kSumCols = 16;
__device__ __forceinline__ void slope_sums(const ProductOperand& o, int64_t M, int64_t N, int block,
                                           float* __restrict__ db, float* __restrict__ sums) {
  const int col = threadIdx.x % kSumCols, run = threadIdx.x / kSumCols;
  const int64_t n = min((int64_t)block * kSumCols + col, N - 1);
  const float* dy = static_cast<const float*>(o.p) + n;
  float s = 0.0f;
  for (int64_t m0 = run; m0 < M; m0 += 128) {
    float g[8], z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t m = min(m0 + 16 * i, M - 1);
      g[i] = dy[m * o.ld];
      z[i] = 0.0f;
      if (o.act == ORCA_HIP_ACT_NONE) continue;
      z[i] = o.z8.codes ? (float)o.z8.codes[m * o.z8.cols + n] * act8_step(o.z8.scales[n / 32 * o.z8.ld + m])
                        : o.z[m * o.ldz + n];
    }
    activation_slopes<8>(o.act, z, g);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (m0 + 16 * i < M) s = s + g[i];
  }
  sums[threadIdx.x] = s;
  __syncthreads();
  if (run == 0 && block * (int64_t)kSumCols + col < N) {
    for (int i = 1; i < 16; ++i) s = s + sums[i * kSumCols + col];
    db[n] = s;
  }
}

// A small backward in one launch: dz is made inside the products (every tile of a row or column panel makes
// it again) and the bias gradient beside them.  MR: dW for a few rows, else (0) on tiles.
template <class T, template <int, int, int> class LoadX, int MR>
__global__ void __launch_bounds__(256, 2) small_backward_kernel(BackwardArgs p) {
  static_assert(T::THREADS == 256, "row_dw's block");
  __shared__ u32x4 smem[tile_units<T, LoadKFast, LoadKFast>()];
  const int block = blockIdx.x;
  if (block < p.dx_blocks) {
    tile_product<T, LoadSlopeFast, LoadKFast>(p.dx, block, p.dx_blocks, smem);
  } else if (block < p.dx_blocks + p.dw_blocks) {
    if constexpr (MR > 0)
      row_dw<MR, true>(p.dw, block - p.dx_blocks, reinterpret_cast<float*>(smem));
    else
      tile_product<T, LoadX, LoadSlopeSlow>(p.dw, block - p.dx_blocks, p.dw_blocks, smem);
  } else {
    slope_sums(p.dz, p.M, p.N, block - p.dx_blocks - p.dw_blocks, p.db, reinterpret_cast<float*>(smem));
  }
}

template <class T, template <int, int, int> class LoadX>
__global__ void __launch_bounds__(T::THREADS, T::OCC* T::THREADS / 256) linear_act_backward_kernel(BackwardArgs p) {
  __shared__ u32x4 smem[tile_units<T, LoadKFast, LoadKFast>()];  // the larger of the two products'
  const int block = blockIdx.x;
  if (block < p.dx_blocks)
    tile_product<T, LoadKFast, LoadKFast>(p.dx, block, p.dx_blocks, smem);
  else if (block < p.dx_blocks + p.dw_blocks)
    tile_product<T, LoadX, LoadKSlow>(p.dw, block - p.dx_blocks, p.dw_blocks, smem);
  else
    finish_bias<T::THREADS / 32>(p, block - p.dx_blocks - p.dw_blocks, reinterpret_cast<float*>(smem));
}

// The splits' partial products of up to two products, added in split order, and the epilogue.  A
// lane takes four columns, eight lanes a checkpoint's group of 32; a block 4 rows of 256 columns.
struct FinishArgs {
  ProductArgs p[2];
  int64_t blocks[2];
};
__global__ void __launch_bounds__(256) split_finish_kernel(FinishArgs a) {
  int64_t block = blockIdx.x;
  const bool second = block >= a.blocks[0];
  if (second) block -= a.blocks[0];
  const ProductArgs& p = a.p[second];
  const int64_t groups = (p.N + 255) / 256;
  const int64_t m = block / groups * 4 + (threadIdx.x >> 6);
  if (m >= p.M) return;  // a whole wave
  const Quad q = quad_of(block % groups * 256 + (threadIdx.x & 63) * 4, p.N);
  const floatx4 bias = bias_quad(p.out, q), residual = residual_quad(p.out, m, q);
  floatx4 z = {0.0f, 0.0f, 0.0f, 0.0f};
  const float* w = p.ws + m * p.N;
  const int64_t step = p.M * p.N;
  int s = 0;
  auto add = [&](auto count) {  // that many loads ahead of their additions
    constexpr int C = decltype(count)::value;
    floatx4 v[C];
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = load_quad(w + (s + i) * step, q);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      settle(q, v[i]);
      z = z + v[i];
    }
    s += C;
  };
  while (s + 8 <= p.splits) add(std::integral_constant<int, 8>());
  if (s + 4 <= p.splits) add(std::integral_constant<int, 4>());
  while (s < p.splits) add(std::integral_constant<int, 1>());
  quad_out(p.out, z, bias, residual, m, q, true);
}

// dz = dy * act'(z) (z in fp32, or its checkpoint) and, per block of 4 R rows, the column sums of dz.
// A thread takes four columns of R rows (R0, or for 0 `run`, a multiple of 4), four rows' loads at a time.  (R 4 without
// a loop: 256 x 1024 with GELU 1 us less.)
template <int R0>
__global__ void __launch_bounds__(256) slope_kernel(ProductOperand o, float* __restrict__ dz,
                                                    float* __restrict__ partial, int64_t M, int64_t N, int run) {
  const int R = R0 ? R0 : run;
  __shared__ floatx4 sums[4][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t r0 = ((int64_t)blockIdx.x * 4 + wave) * R;
  const int64_t c0 = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * 256;
  if (c0 >= N) return;  // the whole block
  const Quad q = quad_of(c0 + lane * 4, N);
  const float* dy = static_cast<const float*>(o.p);
  floatx4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int r = 0; r < R && r0 + r < M; r += 4) {
    const int rows = (int)min((int64_t)4, M - r0 - r);
    floatx4 g[4];
    SlopeQuad v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t m = r0 + r + min(i, rows - 1);
      g[i] = load_quad(dy + m * o.ld, q);
      load_slope(o, m, q, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i >= rows) break;
      settle(q, g[i]);
      apply_slope(o, q, v[i], g[i]);
      if (o.act != ORCA_HIP_ACT_NONE) store_quad(dz + (r0 + r + i) * N, q, g[i]);
      sum = sum + g[i];
    }
  }
  if (!partial) return;
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave == 0)
    store_quad(partial + (int64_t)blockIdx.x * N, q, sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane]);
}

// 256: eight waves of 128 x 64, the least LDS traffic for a matrix instruction; at 8192 x 4096 x 4096 228 TFLOP/s
// (of fp32 work; 128: 201, 64: 154).  128 and 64 for products with too few tiles of 256.
using Tile256 = ProductTile<256, 256, 2, 4, 16, 1>;
using Tile128 = ProductTile<128, 128, 2, 4, 32, 1>;
using Tile64 = ProductTile<64, 64, 2, 2, 32, 3>;

constexpr int64_t kMaxThreads = 0x7fffffff;  // of a launch

struct Plan {
  int tile = 0;       // 0: nothing to do
  int64_t blocks = 0;
  size_t ws = 0;      // floats of partial products
};

// Microseconds of products on tiles with their k ranges split, on an otherwise idle GPU of 256 CUs: fitted
// to 7700 products of 1 .. 8192 x 16 .. 4096 x 16 .. 4096, each timed with every tile and split (8 %
// rms near the best ones; the choice by it takes 1.7 % longer than the best of these tiles and splits, 11 % in one case of
// twenty).  The fp32 tiles of orca_hip_gemm are no part of it; below 1e9 multiply-adds they are quicker, up to twice.
// A launch; then the CU with the most blocks, `together` of them at a time: a stage's chain of
// waits, or its throughput; with splits the second launch, which reads and writes them.
struct TileCost {
  int tile, bk, together;
  double launch, chain, block, stage, each, finish, bytes_per_us;
};
constexpr TileCost kTileCosts[2][3] = {
    {{64, 32, 3, 5.5, 0.584, 0.0, 0.432, 0.97, 3.2, 6.0e6},
     {128, 32, 1, 5.5, 1.159, 2.65, 1.159, 2.65, 1.6, 2.9e6},
     {256, 16, 1, 8.0, 1.783, 7.44, 1.783, 7.44, 0.0, 3.5e6}},
    // the row operand is a checkpoint: half the matrix instructions
    {{64, 32, 3, 5.0, 0.495, 0.97, 0.305, 1.43, 3.5, 8.0e6},
     {128, 32, 1, 5.4, 0.765, 2.93, 0.819, 1.42, 2.2, 3.2e6},
     {256, 16, 1, 9.7, 1.031, 8.29, 1.031, 8.29, 0.0, 4.3e6}}};

// One way to cut a product.
struct Cut {
  int64_t tm, tn, splits, chunk, blocks;
  double chain, work, finish;  // us of a block alone, of a block among others, of the second launch
  double launch;
  int together;
};
constexpr int kMaxCuts = 13;
int cuts_of(orca_hip_ctx* ctx, const ProductArgs& p, bool codes, int tile, double slopes, Cut (&out)[kMaxCuts]) {
  const TileCost& c = kTileCosts[codes][tile];
  const int64_t tm = (p.M + c.tile - 1) / c.tile, tn = (p.N + c.tile - 1) / c.tile;
  int n = 0;
  const int64_t most = kMaxThreads / 512;  // threads of the largest tiles' blocks
  if (tm > most / tn) return 0;
  for (int64_t want : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 64, 128, 256}) {
    if (ctx->linear_splits) {  // that many, as far as k goes
      if (want > 1) break;
      want = ctx->linear_splits;
    } else if (want > 1 && (p.K < 48 * want || tm * tn * want > 8 * ctx->num_cus)) {
      break;
    }
    // even runs of a multiple of every stage's k values
    const int64_t chunk = std::max<int64_t>(64, ((p.K + want - 1) / want + 63) / 64 * 64);
    const int64_t splits = std::max<int64_t>(1, (p.K + chunk - 1) / chunk);
    if ((want > 1 && splits == 1 && n) || tm * tn > most / splits) continue;
    const double stages = (double)((std::min(chunk, p.K) + c.bk - 1) / c.bk);
    const double finish =
        splits > 1 ? c.finish + 4.0 * (double)(splits + 1) * (double)p.M * (double)p.N / c.bytes_per_us : 0.0;
    out[n++] = Cut{tm, tn, splits, chunk, tm * tn * splits, stages * (c.chain + slopes) + c.block,
                   stages * (c.stage + slopes / 2) + c.each, finish, c.launch, c.together};
  }
  return n;
}
Plan take(ProductArgs& p, int tile, const Cut& c) {
  p.tiles_m = (int)c.tm;
  p.tiles_n = (int)c.tn;
  p.splits = (int)c.splits;
  p.chunk = c.chunk;
  return Plan{kTileCosts[0][tile].tile, c.blocks, c.splits > 1 ? (size_t)c.splits * p.M * p.N : 0};
}

// The tile and the cuts of a product, or of two that share a launch (on one tile; `only`: that of this size).
// `slopes`: what a stage takes longer because dz is made in it.  Returns the microseconds expected.
double plan_products(orca_hip_ctx* ctx, ProductArgs* a, Plan* qa, ProductArgs* b, Plan* qb, bool b_codes,
                     const char* op, int only = 0, double slopes = 0.0) {
  if (ctx->linear_tile) only = ctx->linear_tile;
  double best = 0.0;
  int best_tile = -1;
  Cut best_a{}, best_b{};
  for (int tile = 0; tile < 3; ++tile) {
    if (only && kTileCosts[0][tile].tile != only) continue;
    Cut ca[kMaxCuts] = {}, cb[kMaxCuts] = {};
    const int na = a ? cuts_of(ctx, *a, false, tile, slopes, ca) : 1;
    const int nb = b ? cuts_of(ctx, *b, b_codes, tile, slopes, cb) : 1;
    for (int i = 0; i < na; ++i)
      for (int j = 0; j < nb; ++j) {
        const Cut &x = ca[i], &y = cb[j];
        const int64_t blocks = x.blocks + y.blocks, per_cu = (blocks + ctx->num_cus - 1) / ctx->num_cus;
        const int together = std::max(x.together, y.together);
        // each CU's blocks are of both kinds, in proportion
        const double work = ((double)x.blocks * x.work + (double)y.blocks * y.work) / (double)blocks;
        const double us = std::max(x.launch, y.launch) + x.finish + y.finish +
                          std::max((double)((per_cu + together - 1) / together) * std::max(x.chain, y.chain),
                                   (double)per_cu * work);
        if (best_tile >= 0 && us >= best) continue;
        best = us;
        best_tile = tile;
        best_a = x;
        best_b = y;
      }
  }
  if (best_tile < 0) fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": matrix too large");
  if (a) *qa = take(*a, best_tile, best_a);
  if (b) *qb = take(*b, best_tile, best_b);
  return best;
}

// Forward of a few rows: blocks of 16 columns, or of a checkpoint's groups of 32, and of more where that gives more
// blocks than CUs.  k is split, so that the blocks cover the CUs, from three steps of a block's loads on
// (4096 x 512 weights, two steps: 7.1 us in one launch and 8.3 in two; 10000 x 1000: 13.2 split).
Plan plan_rows(orca_hip_ctx* ctx, ProductArgs& p, int& groups) {
  Plan q;
  groups = p.out.pre8.codes || p.out.y8.codes ? 2 : 1;
  while (groups < kRowWaves && p.N > (int64_t)groups * kRowCols * ctx->num_cus) groups *= 2;
  const int64_t tn = (p.N + groups * kRowCols - 1) / (groups * kRowCols);
  const int64_t step = kRowWaves / groups * 16 * row_loads(p.M), steps = (p.K + step - 1) / step;
  const int64_t splits =
      steps < 3 ? 1 : std::max<int64_t>(1, std::min<int64_t>({ctx->num_cus / tn, p.K / step, 32}));
  p.chunk = std::max<int64_t>(1, (p.K + splits - 1) / splits);
  p.splits = (int)std::max<int64_t>(1, (p.K + p.chunk - 1) / p.chunk);
  p.tiles_m = 1;
  p.tiles_n = (int)tn;
  q.blocks = tn * p.splits;
  if (p.splits > 1) q.ws = (size_t)p.splits * p.M * p.N;
  return q;
}

void launch_rows(orca_hip_ctx* ctx, const ProductArgs& p, unsigned blocks, int groups) {
  const auto kernel = p.M == 1   ? row_forward_kernel<1>
                      : p.M == 2 ? row_forward_kernel<2>
                      : p.M <= 4 ? row_forward_kernel<4>
                                 : row_forward_kernel<8>;
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kRowWaves * 64), 0, ctx->stream, p, groups);
}

int64_t finish_blocks(const ProductArgs& p, const Plan& q) {
  return q.ws ? (p.M + 3) / 4 * ((p.N + 255) / 256) : 0;
}
void launch_finish(orca_hip_ctx* ctx, const ProductArgs& a, const Plan& qa, const ProductArgs& b, const Plan& qb,
                   const char* op) {
  FinishArgs f{{a, b}, {finish_blocks(a, qa), finish_blocks(b, qb)}};
  const int64_t grid = f.blocks[0] + f.blocks[1];
  if (!grid) return;
  if (grid > kMaxThreads / 256) fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": matrix too large");
  hipLaunchKernelGGL(split_finish_kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, f);
  ORCA_HIP_CHECK(hipGetLastError());
}

template <class T>
void launch_backward(orca_hip_ctx* ctx, bool codes, unsigned grid, const BackwardArgs& b) {
  if (codes)
    hipLaunchKernelGGL((linear_act_backward_kernel<T, LoadCodes>), dim3(grid), dim3(T::THREADS), 0, ctx->stream, b);
  else
    hipLaunchKernelGGL((linear_act_backward_kernel<T, LoadKSlow>), dim3(grid), dim3(T::THREADS), 0, ctx->stream, b);
  ORCA_HIP_CHECK(hipGetLastError());
}
void launch_backward(orca_hip_ctx* ctx, int tile, bool codes, unsigned grid, const BackwardArgs& b) {
  if (tile == 256)
    launch_backward<Tile256>(ctx, codes, grid, b);
  else if (tile == 128)
    launch_backward<Tile128>(ctx, codes, grid, b);
  else  // also where only the bias gradient is left to finish
    launch_backward<Tile64>(ctx, codes, grid, b);
}

// Up to where dz is made inside the products instead of in a launch before them, in rows and rows x in x out:
// the bias gradient beside them walks down the rows, and every tile takes its panel's slopes again.
// Measured on 55 layers: 11.2 against 14.7 us at 173 x 146 x 124 without an activation; with GELU equal around
// 3e7 (96 x 1605 x 341: 19.7 and 17.7 us, 64 x 784 x 128: 9.9 and 12.6).
constexpr size_t kInsideRows = 512;
constexpr double kInsideWork = 2.5e7, kInsideWorkPlain = 3e8;
// Below that the model decides: a stage of 32 k values takes 0.42 us longer with ReLU's slopes in it (40 x 30 x 1800
// unsplit: 60 us, 40 with a launch for the slopes), 0.69 with another activation's, 0.26 more from a
// checkpoint; the launch that makes them apart takes this long.
constexpr double kSlopeLaunch = 4.0;

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
    check_sizes(op, {M, N, K});
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
    const Span x = matrix_span(X, M, K, ldx), w = matrix_span(W, K, N, ldw), b = buffer_span(e.bias, 4 * N),
               r = matrix_span(e.residual, M, N, e.ldr), y = matrix_span(Y, M, N, ldy),
               pre = matrix_span(e.pre, M, N, e.ldpre), z8 = buffer_span(e.pre8, p8), y8 = buffer_span(e.y8, p8);
    const Span outs[4] = {y, pre, z8, y8};
    for (int i = 0; i < 4; ++i) {
      for (const Span& s : {x, w, b}) check_apart(op, outs[i], s);
      // y over its own residual, element by element, is in order
      if (!(i == 0 && e.residual == Y && e.ldr == ldy)) check_apart(op, outs[i], r);
      for (int j = 0; j < i; ++j) check_apart(op, outs[i], outs[j]);
    }
    act8_aligned(e.pre8, "linear_act (pre8)");
    act8_aligned(e.y8, "linear_act (y8)");
    bind(ctx);
    if (!M || !N) return;
    check_extent(ctx, x.p, x.bytes(), "linear_act (x)");
    check_extent(ctx, w.p, w.bytes(), "linear_act (weight)");
    check_extent(ctx, b.p, b.bytes(), "linear_act (bias)");
    check_extent(ctx, r.p, r.bytes(), "linear_act (residual)");
    check_extent(ctx, y.p, y.bytes(), "linear_act (y)");
    check_extent(ctx, pre.p, pre.bytes(), "linear_act (pre)");
    check_extent(ctx, z8.p, z8.bytes(), "linear_act (pre8)");
    check_extent(ctx, y8.p, y8.bytes(), "linear_act (y8)");
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
    ProductArgs p{};
    p.A = ProductOperand{X, (int64_t)ldx, (int)M, nullptr, 0};
    p.B = ProductOperand{W, (int64_t)ldw, (int)N, nullptr, 0};
    p.M = (int64_t)M;
    p.N = (int64_t)N;
    p.K = (int64_t)K;
    p.out = o;
    const bool few = M <= kRowsForward && !ctx->linear_tile;
    Plan q;
    int groups = 1;
    if (few)
      q = plan_rows(ctx, p, groups);
    else
      plan_products(ctx, &p, &q, nullptr, nullptr, false, op);
    std::unique_ptr<Scratch> ws;
    if (q.ws) {
      ws = workspace(ctx, sizeof(float) * q.ws, op);
      p.ws = ws->as<float>();
    }
    std::string pname;
    if (ctx->prof.enabled)
      pname = std::string(op) + (few ? "_rows" : "_t" + std::to_string(q.tile)) + " " + std::to_string(M) + "x" +
              std::to_string(N) + "x" + std::to_string(K);
    ProfScope prof(ctx, pname.c_str(), 2.0 * M * N * K, 4.0 * ((double)M * K + (double)K * N + (double)M * N));
    const dim3 grid((unsigned)q.blocks);
    if (few)
      launch_rows(ctx, p, (unsigned)q.blocks, groups);
    else if (q.tile == 256)
      hipLaunchKernelGGL(linear_act_kernel<Tile256>, grid, dim3(Tile256::THREADS), 0, ctx->stream, p);
    else if (q.tile == 128)
      hipLaunchKernelGGL(linear_act_kernel<Tile128>, grid, dim3(Tile128::THREADS), 0, ctx->stream, p);
    else
      hipLaunchKernelGGL(linear_act_kernel<Tile64>, grid, dim3(Tile64::THREADS), 0, ctx->stream, p);
    ORCA_HIP_CHECK(hipGetLastError());
    launch_finish(ctx, p, q, p, Plan(), op);
  });
}

int orca_hip_linear_act_backward(orca_hip_ctx* ctx, size_t M, size_t N, size_t K, const float* dY, size_t lddy,
                                 const float* W, size_t ldw, const orca_hip_linear_saved* saved, float* dX,
                                 size_t lddx, float* dW, size_t lddw, float* db) {
  return guard([&] {
    const char* op = "linear_act_backward";
    check_sizes(op, {M, N, K});
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
    const Span dy = matrix_span(dY, M, N, lddy), w = matrix_span(dX ? W : nullptr, K, N, ldw),
               z = matrix_span(slope ? s.z : nullptr, M, N, s.ldz),
               z8 = buffer_span(slope ? s.z8 : nullptr, act8_layout(M, N).bytes),
               x = matrix_span(dW ? s.x : nullptr, M, K, s.ldx),
               x8 = buffer_span(dW ? s.x8 : nullptr, act8_layout(M, K).bytes),
               add = matrix_span(dX ? s.dx_add : nullptr, M, K, s.ldadd), dx = matrix_span(dX, M, K, lddx),
               dw = matrix_span(dW, K, N, lddw), dbs = buffer_span(db, 4 * N);
    const Span outs[3] = {dx, dw, dbs};
    for (int i = 0; i < 3; ++i) {
      for (const Span& in : {dy, w, z, z8, x, x8}) check_apart(op, outs[i], in);
      // dx over dx_add, element by element, is in order (a gradient added up in place)
      if (!(i == 0 && s.dx_add == dX && s.ldadd == lddx)) check_apart(op, outs[i], add);
      for (int j = 0; j < i; ++j) check_apart(op, outs[i], outs[j]);
    }
    act8_aligned(z8.p, "linear_act_backward (z8)");
    act8_aligned(x8.p, "linear_act_backward (x8)");
    bind(ctx);
    check_extent(ctx, dy.p, dy.bytes(), "linear_act_backward (dy)");
    check_extent(ctx, w.p, w.bytes(), "linear_act_backward (weight)");
    check_extent(ctx, z.p, z.bytes(), "linear_act_backward (z)");
    check_extent(ctx, z8.p, z8.bytes(), "linear_act_backward (z8)");
    check_extent(ctx, x.p, x.bytes(), "linear_act_backward (x)");
    check_extent(ctx, x8.p, x8.bytes(), "linear_act_backward (x8)");
    check_extent(ctx, add.p, add.bytes(), "linear_act_backward (dx_add)");
    check_extent(ctx, dx.p, dx.bytes(), "linear_act_backward (dx)");
    check_extent(ctx, dw.p, dw.bytes(), "linear_act_backward (dw)");
    check_extent(ctx, db, dbs.bytes(), "linear_act_backward (db)");
    const float* dz = dY;
    int64_t lddz = (int64_t)lddy;
    std::unique_ptr<Scratch> dzs, partial;
    ProductOperand dyz{dY, (int64_t)lddy, (int)M, nullptr, 0};  // dy and what makes it dz
    dyz.act = s.act;
    dyz.z = static_cast<const float*>(z.p);
    dyz.ldz = (int64_t)s.ldz;
    dyz.z8 = act8_at(const_cast<void*>(z8.p), M, N);
    const bool want_dx = dX && M && K, want_dw = dW && K && N, want_db = db && N;
    // dW as outer products; the slopes of 16 rows there cost a thread more (4 us with GELU) than the tiles' padding
    auto few_rows = [&](bool in) {
      return M && !ctx->linear_tile && M <= (size_t)kRowsDw && want_dw && !(in && slope && M > 4);
    };
    // slopes inside the products: a launch less, but every tile takes its panel's slopes again
    bool inside = M && N && !ctx->linear_tile && M <= kInsideRows &&
                  (double)M * N * K <= (slope ? kInsideWork : kInsideWorkPlain);
    double slopes = 0.0;
    if (inside && slope) {
      slopes = (s.act == ORCA_HIP_ACT_RELU ? 0.42 : 0.69) + (s.z8 ? 0.26 : 0.0);
      auto expected = [&](bool in) {
        ProductArgs x{}, w{};
        x.M = w.K = (int64_t)M;
        x.N = w.M = (int64_t)K;
        x.K = w.N = (int64_t)N;
        Plan qx, qw;
        const bool on_tiles = want_dw && !few_rows(in);
        return !want_dx && !on_tiles ? kTileCosts[0][0].launch
                                     : plan_products(ctx, want_dx ? &x : nullptr, &qx, on_tiles ? &w : nullptr, &qw,
                                                     s.x8 != nullptr, op, Tile64::BM, in ? slopes : 0.0);
      };
      inside = expected(true) <= expected(false) + kSlopeLaunch;
    }
    const bool few = few_rows(inside);
    // 64 rows a block, 16 where that leaves CUs without one; more where the column sums would get long to add up
    const int64_t panels = ((int64_t)N + 255) / 256;
    int64_t rows = ((int64_t)M + 63) / 64 * panels >= ctx->num_cus ? 64 : 16;
    rows = std::max(rows, ((int64_t)M / 2048 + 15) / 16 * 16);
    const int64_t blocks = ((int64_t)M + rows - 1) / rows;
    const bool direct = blocks == 1 && !inside;  // a block's column sums are db
    if (N && !inside && (want_db || (slope && (want_dx || want_dw)))) {
      if (slope && M) {
        dzs = workspace(ctx, sizeof(float) * M * N, op);
        dz = dzs->as<float>();
        lddz = (int64_t)N;
      }
      if (want_db && M && !direct) partial = workspace(ctx, sizeof(float) * (size_t)blocks * N, op);
      if (M) {
        ProfScope prof(ctx, "linear_act_slope", 0.0, (slope ? 12.0 : 4.0) * M * N);
        const int64_t gy = std::min<int64_t>(panels, 32768);
        const dim3 sgrid((unsigned)blocks, (unsigned)gy, (unsigned)((panels + gy - 1) / gy));
        hipLaunchKernelGGL(rows == 16 ? slope_kernel<4> : slope_kernel<0>, sgrid, dim3(256), 0, ctx->stream, dyz,
                           dzs ? dzs->as<float>() : nullptr,
                           want_db && direct ? db : partial ? partial->as<float>() : nullptr, (int64_t)M, (int64_t)N,
                           (int)(rows / 4));
        ORCA_HIP_CHECK(hipGetLastError());
      }
    }
    BackwardArgs b{};
    b.N = (int64_t)N;
    const ProductOperand dzo = inside ? dyz : ProductOperand{dz, lddz, (int)M, nullptr, 0};
    b.dz = dyz;
    b.M = (int64_t)M;
    if (want_db && !direct) {
      b.db = db;
      b.partial = partial ? partial->as<float>() : nullptr;
      b.partials = M ? blocks : 0;
    }
    Plan qx, qw;
    if (want_dx) {
      b.dx.A = dzo;
      b.dx.B = ProductOperand{W, (int64_t)ldw, (int)K, nullptr, 0};
      b.dx.M = (int64_t)M;
      b.dx.N = (int64_t)K;
      b.dx.K = (int64_t)N;
      b.dx.out.residual = s.dx_add;
      b.dx.out.ldr = (int64_t)s.ldadd;
      b.dx.out.y = dX;
      b.dx.out.ldy = (int64_t)lddx;
    }
    if (want_dw) {
      b.dw.A = ProductOperand{s.x, (int64_t)s.ldx, (int)K, nullptr, 0};
      if (s.x8) {
        const Act8 q = act8_at(const_cast<void*>(s.x8), M, K);
        b.dw.A = ProductOperand{q.codes, q.cols, (int)K, q.scales, q.ld};
      }
      b.dw.B = dzo;
      b.dw.B.rows = (int)N;
      b.dw.M = (int64_t)K;
      b.dw.N = (int64_t)N;
      b.dw.K = (int64_t)M;
      b.dw.out.y = dW;
      b.dw.out.ldy = (int64_t)lddw;
    }
    if (want_dx || (want_dw && !few))
      plan_products(ctx, want_dx ? &b.dx : nullptr, &qx, want_dw && !few ? &b.dw : nullptr, &qw, s.x8 != nullptr, op,
                    few || inside ? Tile64::BM : 0, inside ? slopes : 0.0);
    if (few) qw.blocks = ((int64_t)K + kRowDw - 1) / kRowDw * (((int64_t)N + 255) / 256);
    std::unique_ptr<Scratch> ws;
    if (qx.ws + qw.ws) {
      ws = workspace(ctx, sizeof(float) * (qx.ws + qw.ws), op);
      b.dx.ws = ws->as<float>();
      b.dw.ws = ws->as<float>() + qx.ws;
    }
    const int64_t sums = inside ? kSumCols : 32;
    const int64_t grid = qx.blocks + qw.blocks + (b.db ? ((int64_t)N + sums - 1) / sums : 0);
    if (grid > kMaxThreads / 512) fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": matrix too large");
    if (!grid) return;
    std::string pname;
    if (ctx->prof.enabled)
      pname = std::string(op) + (inside ? "_inside" : "") +
              (few ? "_rows" : "_t" + std::to_string(std::max(qx.tile, qw.tile))) + " " + std::to_string(M) + "x" +
              std::to_string(N) + "x" + std::to_string(K);
    ProfScope prof(ctx, pname.c_str(), 2.0 * M * N * K * (want_dx + want_dw),
                   4.0 * ((double)M * N + (want_dx + want_dw) * ((double)M * K + (double)K * N)));
    b.dx_blocks = (int)qx.blocks;
    b.dw_blocks = (int)qw.blocks;
    if (inside) {
      const auto kernel = few && M <= 4   ? small_backward_kernel<Tile64, LoadKSlow, 4>
                          : few           ? small_backward_kernel<Tile64, LoadKSlow, 16>
                          : s.x8          ? small_backward_kernel<Tile64, LoadCodes, 0>
                                          : small_backward_kernel<Tile64, LoadKSlow, 0>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, b);
      ORCA_HIP_CHECK(hipGetLastError());
    } else if (few) {
      hipLaunchKernelGGL((M <= 4 ? row_backward_kernel<Tile64, 4> : row_backward_kernel<Tile64, 16>),
                         dim3((unsigned)grid), dim3(256), 0, ctx->stream, b);
      ORCA_HIP_CHECK(hipGetLastError());
    } else {
      launch_backward(ctx, std::max(qx.tile, qw.tile), s.x8 != nullptr, (unsigned)grid, b);
    }
    launch_finish(ctx, b.dx, qx, b.dw, qw, op);
  });
}

}  // extern "C"
