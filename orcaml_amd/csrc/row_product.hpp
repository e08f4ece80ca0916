// The fused Linear's products for batches of a few rows (part of linear_act.hip, which defines
// the epilogue).  They move the weight, or its gradient, once and do little with it, so what bounds them
// is memory, and a tile of the matrix instructions would be mostly padding.  They run on the vector units
// in fp32, MR rows at a time (rows past M count as zeros).

// Forward of at most 4 rows: a block takes 16 columns, so that the blocks of a wide layer cover the CUs and
// each finishes its outputs itself; a wave reads 16 k values of those columns with one load, and
// the block's 16 waves walk down k together, eight such loads each in flight.
constexpr int kRowCols = 16, kRowWaves = 16, kRowLoads = 8;
constexpr size_t kRowMaxCols = size_t(1) << 24;  // 2^30 threads
template <int MR>
__global__ void __launch_bounds__(kRowWaves * 64) row_forward_kernel(ProductArgs p) {
  __shared__ floatx4 sums[kRowWaves][MR][4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  // neighbouring columns on one XCD: two blocks read the halves of a line
  const int nb = gridDim.x, x8 = blockIdx.x % 8, block = x8 * (nb / 8) + min(x8, nb % 8) + blockIdx.x / 8;
  const int64_t split = block / p.tiles_n;
  const Quad quad = quad_of((int64_t)(block % p.tiles_n) * kRowCols + lane % 4 * 4, p.N);
  const int64_t kb = split * p.chunk, ke = min(p.K, kb + p.chunk);
  const float* x = static_cast<const float*>(p.A.p);
  const float* w = static_cast<const float*>(p.B.p);
  floatx4 acc[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) acc[m] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t k0 = kb + wave * 16; k0 < ke; k0 += kRowLoads * kRowWaves * 16) {
    floatx4 q[kRowLoads];
    float v[kRowLoads][MR];
#pragma unroll
    for (int i = 0; i < kRowLoads; ++i) {
      const int64_t k = min(k0 + i * (kRowWaves * 16) + lane / 4, ke - 1);
      q[i] = load_quad(w + k * p.B.ld, quad);
#pragma unroll
      for (int m = 0; m < MR; ++m) v[i][m] = x[min((int64_t)m, p.M - 1) * p.A.ld + k];
    }
#pragma unroll
    for (int i = 0; i < kRowLoads; ++i) {
      const bool in = k0 + i * (kRowWaves * 16) + lane / 4 < ke;
      settle(quad, q[i]);
#pragma unroll
      for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[m][j] = in ? fmaf(v[i][m], q[i][j], acc[m][j]) : acc[m][j];
    }
  }
  // over the wave's 16 k values, then over the waves in order
#pragma unroll
  for (int m = 0; m < MR; ++m) {
#pragma unroll
    for (int d = 4; d < 64; d *= 2)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[m][j] = acc[m][j] + __shfl_xor(acc[m][j], d);
    if (lane < 4) sums[wave][m][lane] = acc[m];
  }
  __syncthreads();
  const int64_t m = tid / 4;
  if (m >= min((int64_t)MR, p.M)) return;
  floatx4 z = sums[0][m][lane % 4];
  for (int i = 1; i < kRowWaves; ++i) z = z + sums[i][m][lane % 4];
  if (p.splits == 1)
    quad_out(p.out, z, bias_quad(p.out, quad), residual_quad(p.out, m, quad), m, quad, true);
  else
    store_quad(p.ws + (split * p.M + m) * p.N, quad, z);
}

// Block (64 rows of dW, 256 columns) of dW = x^T dz for batches of at most 16 rows, x in fp32 or as a
// checkpoint, dz in memory or (SLOPE) made here from dy and z: a lane holds its four columns of dz and
// writes one row of dW after the other.  67 MB of dW in 13 us (1 to 4 rows) and 18 us (16; the tiles 23),
// 5 us where the launch is all.
constexpr int kRowsDw = 16, kRowDw = 64;
template <int MR, bool SLOPE>
__device__ __forceinline__ void row_dw(const ProductArgs& p, int block, float* __restrict__ smem) {
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t tiles = (p.N + 255) / 256, k0 = block / tiles * kRowDw;
  const Quad quad = quad_of(block % tiles * 256 + lane * 4, p.N);
  const float* dz = static_cast<const float*>(p.B.p);
  // x's 64 columns, transposed
  for (int i = tid; i < kRowDw * MR; i += 256) {
    const int64_t k = k0 + i % kRowDw;
    const int m = i / kRowDw;
    float v = 0.0f;
    if (m < p.K && k < p.M)
      v = p.A.scales ? (float)static_cast<const int8_t*>(p.A.p)[m * p.A.ld + k] *
                           act8_step(p.A.scales[k / (int64_t)kAct8Group * p.A.lds + m])
                     : static_cast<const float*>(p.A.p)[m * p.A.ld + k];
    smem[i % kRowDw * MR + m] = v;
  }
  floatx4 g[MR];
  SlopeQuad z[SLOPE ? MR : 1];
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    const int64_t row = min((int64_t)m, p.K - 1);
    g[m] = load_quad(dz + row * p.B.ld, quad);
    if constexpr (SLOPE) load_slope(p.B, row, quad, z[m]);
  }
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    settle(quad, g[m]);
    if constexpr (SLOPE) apply_slope(p.B, quad, z[m], g[m]);
    if (m >= p.K) g[m] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  __syncthreads();
  for (int i = wave * (kRowDw / 4); i < (wave + 1) * (kRowDw / 4); ++i) {
    if (k0 + i >= p.M) break;
    floatx4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int q = 0; q < MR / 4; ++q) {
      const floatx4 x = *reinterpret_cast<const floatx4*>(smem + i * MR + 4 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = fmaf(x[e], g[4 * q + e][j], s[j]);
    }
    store_quad(p.out.y + (k0 + i) * p.out.ldy, quad, s);
  }
}
