// The fused Linear's products for batches of a few rows (part of linear_act.hip, which defines
// the epilogue).  They move the weight, or its gradient, once and do little with it, so what bounds them
// is memory, and a tile of the matrix instructions would be mostly padding.  They run on the vector units
// in fp32, MR rows at a time (rows past M count as zeros).

// Forward of at most 8 rows: a block's 16 waves take C groups of 16 columns, so that the blocks of a layer cover
// the CUs once and each finishes its outputs itself; a wave reads 16 k values of its columns with one load, and
// the 16 / C waves of a group walk down k together, row_loads such loads each in flight (fewer where the
// rows' sums take the registers).  4096 x 4096 weights (67 MB): 15.0 us for a row, 16.1 for four, 18.1 for eight,
// against 22.6 to 23 on the tiles; 1024 x 1024: 5.9, 7.6 and 7.7 against 9.5 to 10.6.  Sixteen rows took
// as long as the tiles or longer.  Blocks of 16 columns in every case: 37 us at 2 rows, 60 x 30000, now 5.9.
constexpr int kRowCols = 16, kRowWaves = 16;
constexpr size_t kRowsForward = 8;
constexpr int row_loads(int64_t rows) { return rows <= 4 ? 8 : 4; }
template <int MR>
__global__ void __launch_bounds__(kRowWaves * 64) row_forward_kernel(ProductArgs p, int C) {
  constexpr int LOADS = row_loads(MR);
  __shared__ __attribute__((aligned(16))) float sums[kRowWaves][MR][4][4];  // a quad each
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, down = kRowWaves / C;
  // neighbouring columns on one XCD: two blocks read the halves of a line
  const int nb = gridDim.x, x8 = blockIdx.x % 8, block = x8 * (nb / 8) + min(x8, nb % 8) + blockIdx.x / 8;
  const int64_t split = block / p.tiles_n, n0 = (int64_t)(block % p.tiles_n) * C * kRowCols;
  const int64_t kb = split * p.chunk, ke = min(p.K, kb + p.chunk);
  const float* x = static_cast<const float*>(p.A.p);
  const float* w = static_cast<const float*>(p.B.p);
  const Quad quad = quad_of(n0 + wave % C * kRowCols + lane % 4 * 4, p.N);
  floatx4 acc[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) acc[m] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t k0 = kb + wave / C * 16; k0 < ke; k0 += LOADS * down * 16) {
    floatx4 q[LOADS];
    float v[LOADS][MR];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int64_t k = min(k0 + i * (down * 16) + lane / 4, ke - 1);
      q[i] = load_quad(w + k * p.B.ld, quad);
#pragma unroll
      for (int m = 0; m < MR; ++m) v[i][m] = x[min((int64_t)m, p.M - 1) * p.A.ld + k];
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const bool in = k0 + i * (down * 16) + lane / 4 < ke;
      settle(quad, q[i]);
#pragma unroll
      for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[m][j] = in ? fmaf(v[i][m], q[i][j], acc[m][j]) : acc[m][j];
    }
  }
  // Over the wave's 16 k values, in halves: at each step a lane gives away half of its values and adds its
  // partner's to the others (15 exchanges for four rows instead of 64).
  constexpr int V = MR * 4, LEFT = V > 16 ? V / 16 : 1, COPIES = V < 16 ? 16 / V : 1;
  float v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = acc[i / 4][i % 4];
#pragma unroll
  for (int step = 0; step < 4; ++step) {
    const int d = 32 >> step, half = (V >> step) / 2;
    const bool up = lane & d;
    if (half == 0) v[0] = v[0] + __shfl_xor(v[0], d);
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float send = up ? v[i] : v[half + i], keep = up ? v[half + i] : v[i];
      v[i] = keep + __shfl_xor(send, d);
    }
  }
  if (lane / 4 % COPIES == 0)
#pragma unroll
    for (int i = 0; i < LEFT; ++i) {
      const int at = lane / 4 / COPIES * LEFT + i;  // 4 * row + column of the quad
      sums[wave][at / 4][lane % 4][at % 4] = v[i];
    }
  // then over the group's waves in order
  __syncthreads();
  // a row's 4 C quads lie in neighbouring lanes
  const int64_t m = tid / (4 * C);
  if (m >= min((int64_t)MR, p.M)) return;
  const int group = tid % (4 * C) / 4;
  auto part = [&](int i) { return *reinterpret_cast<const floatx4*>(sums[group + C * i][m][tid % 4]); };
  floatx4 z = part(0);
  for (int i = 1; i < down; ++i) z = z + part(i);
  const Quad out = quad_of(n0 + tid % (4 * C) * 4, p.N);
  if (p.splits == 1)
    quad_out(p.out, z, bias_quad(p.out, out), residual_quad(p.out, m, out), m, out, true);
  else
    store_quad(p.ws + (split * p.M + m) * p.N, out, z);
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
