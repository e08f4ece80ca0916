// Norms of rows and the joint of two residual blocks, with their backward passes (orca_hip_norm,
// orca_hip_residual_norm and their _backward).
//
// The formulas, for a row v of n values: unit(v) = (v - mean) r with r = 1 / sqrt(mean((v - mean)^2) + eps), or v r
// with r = 1 / sqrt(mean(v^2) + eps).  norm(v) = unit(v) w + b.  Its backward, with e = dv w:
// r (e - mean(e) - unit mean(e unit)), without mean(e) for the mean square; dw = sum dv unit, db = sum dv.
// The joint: y = s x + t gate drop(post(f)), u = next(y).  Its backward: g = dy + next's of du, dx = s g,
// dv = t gate keep g, df = post's of dv, dgate = sum over the gate row's rows of t keep g post(f).
//
// The backward takes the statistics again from the rows that it reads anyway, and draws the dropout's numbers
// again: nothing is kept between the passes.  Means and sums are fp32: a variance is taken around the row's mean,
// corrected by what that mean was off by (sum of the differences), so that a large common part of a row costs no
// digits.  Sums over rows run per block in row order, then over the blocks' partial sums in a second launch: no
// atomics, the same bits every time.
//
// Bound by HBM where there are many rows: 8192 x 4096 (134 MB an operand), rms without biases: norm backward 99 us
// (5.4 TB/s), joint forward 98 us (5.5), joint backward 159 us (5.1; 25 MB of partial sums and a launch of 8 us on
// top), where a copy of 1 GiB runs at 5.0.  Few rows take the latency of a row's chain of sums: 777 x 1501 backward
// 24 us, of which the partial sums take 5.  Registers decide the rest: see norm_backward_kernel.
#include <algorithm>
#include <cmath>
#include <memory>
#include <string>

#include "act8.hpp"
#include "ce_row.hpp"
#include "operand.hpp"
#include "philox.hpp"
#include "quad.hpp"
#include "runtime.hpp"
#include "slab.hpp"

namespace orca_hip {
namespace {

struct Norm {
  int kind = ORCA_HIP_NORM_NONE;
  float eps = 0.0f;
  const float* w = nullptr;  // null: ones
  const float* b = nullptr;  // null: zeros
};

struct NormForward {
  int64_t rows, cols;
  const float* x;
  int64_t ldx;
  const float* f;  // the block's output (a norm alone has none: y is x then, and not written)
  int64_t ldf;
  float* y;
  int64_t ldy;
  float* u;
  int64_t ldu;
  Act8 u8;
  Norm post, next;
  const float* gate;
  int64_t ldgate, gate_rows;  // rows of f for each of the gate's
  float rs, bs;
  Dropout drop;
};

// Sums over the rows that a backward gives.
enum { kSumGate, kSumPostW, kSumPostB, kSumNextW, kSumNextB, kSums };

struct NormBackward {
  int64_t rows, cols;
  const float* dy;  // may be null
  int64_t lddy;
  const float* du;  // null: nothing through u
  int64_t lddu;
  const float* f;
  int64_t ldf;
  const float* y;
  int64_t ldy;
  Norm post, next;
  const float* gate;
  int64_t ldgate, gate_rows;
  float rs, bs;
  Dropout drop;
  float* dx;
  int64_t lddx;
  float* df;
  int64_t lddf;
  float* dgate;
  int64_t lddgate;
  // The rows are in groups (one, but where each row of the gate has its own sum), and those in per_group pieces of
  // every per_group-th row each, so that the blocks work on neighbouring rows at a time: norm backward of 8192 x 4096 in
  // 99 us, in 107 with successive rows to a block.  Unit i is piece i % per_group of group i / per_group.
  int group_rows, groups, per_group;
  bool gate_each;     // the gate's gradient row by row, without a sum
  bool gate_grouped;  // its sums are those of the groups
  float* sum[kSums];  // where a sum goes: the result itself (one block), or a block's first partial sum
  int64_t sum_step;   // from one block's to the next one's
  float* stats;       // [rows][kRowStats] (norm_stats_kernel)
};

// ---------------------------------------------------------------- rows
// A row is held by NW waves.  One barrier a sum: successive ones take turns in LDS.
template <int NW>
struct Team {
  float* lds;  // 2 x NW x 4 floats
  int turn = 0;
  template <int N>
  __device__ __forceinline__ void sum(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if constexpr (NW > 1) {
      float* p = lds + turn * (NW * 4);
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i * NW + (threadIdx.x >> 6)] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] = p[i * NW];
#pragma unroll
        for (int k = 1; k < NW; ++k) v[i] += p[i * NW + k];
      }
    }
  }
};

// unit = ((v - mean) - rest) r, off = -rest r
struct Stats {
  float mean, off, r;
  __device__ __forceinline__ float unit(float v) const { return fmaf(v - mean, r, off); }
};
// From the first mean and the sums of the differences to it and of their squares.
// `share` is 1 / the number of values: a product with it costs a rounding more than a division, which takes ten
// instructions a thread.
__device__ __forceinline__ Stats stats_of(const Norm& n, float mean, float sum, float squares, float share) {
  const float rest = n.kind == ORCA_HIP_NORM_LAYER ? sum * share : 0.0f;
  float var = fmaf(-rest, rest, squares * share);
  var = var < 0.0f ? 0.0f : var;  // a NaN stays one
  const float r = 1.0f / sqrtf(var + n.eps);
  return Stats{mean, -rest * r, r};
}

// v where bit n of `kept` is set, else 0.
__device__ __forceinline__ float kept_or_zero(uint32_t kept, int n, float v) {
  return __int_as_float(__float_as_int(v) & __builtin_amdgcn_sbfe((int)kept, n, 1));
}
__device__ __forceinline__ floatx4 splat(float v) { return floatx4{v, v, v, v}; }
__device__ __forceinline__ floatx4 load4(const float* row, int64_t c, int64_t cols) {
  if (c + 4 <= cols) return *reinterpret_cast<const floatx4_u*>(row + c);
  floatx4 v = splat(0.0f);
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (c + j < cols) v[j] = row[c + j];
  return v;
}
__device__ __forceinline__ void store4(float* row, int64_t c, int64_t cols, floatx4 v) {
  if (c + 4 <= cols) {
    *reinterpret_cast<floatx4_u*>(row + c) = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (c + j < cols) row[c + j] = v[j];
}
__device__ __forceinline__ floatx4 weight4(const float* w, int64_t c, int64_t cols, float none) {
  return w ? load4(w, c, cols) : splat(none);
}

// ---------------------------------------------------------------- rows of any length
constexpr int kStream = 256;  // threads of a block, 4 columns each at a time

// Sums along a row: quad(c, t) adds what the row's columns c .. c + 3 give.  A thread adds up runs of 64 quads and those
// to each other: of a row of n values a term goes through 256 + n / 65536 additions of a thread's, not through n / 256
// (the squares of a row of 2^24 values all alike: the deviation is off by up to 3e-6, and was by 7e-5).
constexpr int64_t kRun = 64 * kStream * 4;
template <int N, class F>
__device__ __forceinline__ void row_sums(int64_t cols, Team<4>& team, float (&t)[N], F quad) {
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = 0.0f;
  int c = threadIdx.x * 4, end = (int)min(cols, kRun);
  for (; c < end; c += kStream * 4) quad(c, t);
  while (end < cols) {
    end = (int)min(cols, end + kRun);
    float run[N] = {};
    for (; c < end; c += kStream * 4) quad(c, run);
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] += run[i];
  }
  team.sum(t);
}

__device__ __forceinline__ Stats stream_stats(const Norm& n, const float* row, int64_t cols, Team<4>& team) {
  float mean = 0.0f;
  const float share = 1.0f / (float)cols;
  if (n.kind == ORCA_HIP_NORM_LAYER) {
    float t[1];
    row_sums(cols, team, t, [&](int64_t c, float (&t)[1]) {
      const floatx4 v = load4(row, c, cols);
      t[0] += (v.x + v.y) + (v.z + v.w);
    });
    mean = t[0] * share;
  }
  float t[2];
  row_sums(cols, team, t, [&](int64_t c, float (&t)[2]) {
    const floatx4 v = load4(row, c, cols);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float d = c + j < cols ? v[j] - mean : 0.0f;
      t[0] += d;
      t[1] = fmaf(d, d, t[1]);
    }
  });
  return stats_of(n, mean, t[0], t[1], share);
}

template <bool JOINT>
__global__ void __launch_bounds__(kStream) norm_stream_kernel(NormForward a) {
  __shared__ float lds[2 * 4 * 4];
  Team<4> team{lds};
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float* y = a.x + row * a.ldx;
    if (JOINT) {
      const float *x = y, *f = a.f + row * a.ldf, *gate = a.gate ? a.gate + row / a.gate_rows * a.ldgate : nullptr;
      float* out = a.y + row * a.ldy;
      Stats s{0.0f, 0.0f, 1.0f};
      if (a.post.kind != ORCA_HIP_NORM_NONE) s = stream_stats(a.post, f, a.cols, team);
      for (int64_t c = threadIdx.x * 4; c < a.cols; c += kStream * 4) {
        floatx4 v = load4(f, c, a.cols);
        if (a.post.kind != ORCA_HIP_NORM_NONE) {
          const floatx4 w = weight4(a.post.w, c, a.cols, 1.0f), b = weight4(a.post.b, c, a.cols, 0.0f);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = fmaf(s.unit(v[j]), w[j], b[j]);
        }
        const floatx4 g = weight4(gate, c, a.cols, 1.0f), xv = load4(x, c, a.cols);
        Words words{};
        if (a.drop.on) words = dropout_words(a.drop, row, c / 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float t = v[j] * (g[j] * (a.bs * a.drop.scale));
          v[j] = fmaf(a.rs, xv[j], !a.drop.on || dropout_keeps(a.drop, words, j) ? t : 0.0f);
        }
        store4(out, c, a.cols, v);
      }
      y = out;  // a thread reads back what it wrote itself
    }
    if (a.next.kind == ORCA_HIP_NORM_NONE) continue;
    const Stats s = stream_stats(a.next, y, a.cols, team);
    float* u = a.u + row * a.ldu;
    for (int64_t c0 = 0; c0 < a.cols; c0 += kStream * 4) {
      const int64_t c = c0 + threadIdx.x * 4;
      floatx4 v = splat(0.0f);
      if (c < a.cols) {
        v = load4(y, c, a.cols);
        const floatx4 w = weight4(a.next.w, c, a.cols, 1.0f), b = weight4(a.next.b, c, a.cols, 0.0f);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = fmaf(s.unit(v[j]), w[j], b[j]);
        store4(u, c, a.cols, v);
      }
      if (a.u8.codes) {
        const Quad q = quad_of(c, a.cols);
        const uint32_t byte = quad_byte(v, q);
        if (q.have > 0) {
          store_codes(a.u8.codes + row * a.u8.cols, q, v, byte);
          if ((threadIdx.x & 7) == 0) a.u8.scales[q.group * a.u8.ld + row] = (uint8_t)byte;
        }
      }
    }
  }
}

// What a backward needs to know of each row: Stats, mean(e) and mean(e unit) of the next norm, then of the post norm.
constexpr int kRowStats = 10;
__global__ void __launch_bounds__(kStream) norm_stats_kernel(NormBackward a, bool block) {
  __shared__ float lds[2 * 4 * 4];
  Team<4> team{lds};
  const float share = 1.0f / (float)a.cols;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float *y = a.y + row * a.ldy, *du = a.du + row * a.lddu, *dy = a.dy + row * a.lddy;
    Stats sy{0.0f, 0.0f, 0.0f};
    float c1 = 0.0f, c2 = 0.0f;
    if (a.du) {
      sy = stream_stats(a.next, y, a.cols, team);
      float t[2];
      row_sums(a.cols, team, t, [&](int64_t c, float (&t)[2]) {
        const floatx4 v = load4(y, c, a.cols), d = load4(du, c, a.cols), w = weight4(a.next.w, c, a.cols, 1.0f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (c + j >= a.cols) break;
          const float e = d[j] * w[j];
          t[0] += e;
          t[1] = fmaf(e, sy.unit(v[j]), t[1]);
        }
      });
      c1 = a.next.kind == ORCA_HIP_NORM_LAYER ? t[0] * share : 0.0f;
      c2 = t[1] * share;
    }
    Stats sf{0.0f, 0.0f, 0.0f};
    float p1 = 0.0f, p2 = 0.0f;
    if (block && a.post.kind != ORCA_HIP_NORM_NONE) {
      const float *f = a.f + row * a.ldf, *gate = a.gate ? a.gate + row / a.gate_rows * a.ldgate : nullptr;
      sf = stream_stats(a.post, f, a.cols, team);
      float t[2];
      row_sums(a.cols, team, t, [&](int64_t c, float (&t)[2]) {
        floatx4 g = splat(0.0f);
        if (a.dy) g = load4(dy, c, a.cols);
        if (a.du) {
          const floatx4 v = load4(y, c, a.cols), d = load4(du, c, a.cols), w = weight4(a.next.w, c, a.cols, 1.0f);
#pragma unroll
          for (int j = 0; j < 4; ++j) g[j] += sy.r * (fmaf(-sy.unit(v[j]), c2, d[j] * w[j]) - c1);
        }
        const floatx4 v = load4(f, c, a.cols), w = weight4(a.post.w, c, a.cols, 1.0f);
        const floatx4 gt = weight4(gate, c, a.cols, 1.0f);
        Words words{};
        if (a.drop.on) words = dropout_words(a.drop, row, c / 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (c + j >= a.cols) break;
          const bool kept = !a.drop.on || dropout_keeps(a.drop, words, j);
          const float e = kept ? g[j] * (a.bs * a.drop.scale) * gt[j] * w[j] : 0.0f;
          t[0] += e;
          t[1] = fmaf(e, sf.unit(v[j]), t[1]);
        }
      });
      p1 = a.post.kind == ORCA_HIP_NORM_LAYER ? t[0] * share : 0.0f;
      p2 = t[1] * share;
    }
    if (threadIdx.x == 0) {
      float* s = a.stats + row * kRowStats;
      const float v[kRowStats] = {sy.mean, sy.off, sy.r, c1, c2, sf.mean, sf.off, sf.r, p1, p2};
#pragma unroll
      for (int i = 0; i < kRowStats; ++i) s[i] = v[i];
    }
  }
}

// The gradients, a block for 1024 columns (a strip) and a piece of rows, from the rows' statistics.  The strips of a piece
// follow each other.
__global__ void __launch_bounds__(kStream) norm_strip_kernel(NormBackward a, bool block) {
  const unsigned strips = (unsigned)((a.cols + kStream * 4 - 1) / (kStream * 4));
  const unsigned strip = blockIdx.x % strips, first = blockIdx.x / strips, blocks = gridDim.x / strips;
  const int64_t c = ((int64_t)strip * kStream + threadIdx.x) * 4;
  if (c >= a.cols) return;
  const floatx4 zero = splat(0.0f);
  const floatx4 wn = weight4(a.next.w, c, a.cols, 1.0f), wp = weight4(a.post.w, c, a.cols, 1.0f);
  const floatx4 bp = weight4(a.post.b, c, a.cols, 0.0f);
  const bool post = a.post.kind != ORCA_HIP_NORM_NONE;
  floatx4 sum[kSums] = {zero, zero, zero, zero, zero};
  for (int unit = first; unit < a.groups * a.per_group; unit += blocks) {
    const int group = unit / a.per_group, r0 = group * a.group_rows;
    for (int64_t row = r0 + unit % a.per_group; row < r0 + a.group_rows; row += a.per_group) {
      float s[kRowStats] = {};
      if (a.stats) {
#pragma unroll
        for (int i = 0; i < kRowStats; ++i) s[i] = a.stats[row * kRowStats + i];
      }
      floatx4 g = zero;
      if (a.dy) g = load4(a.dy + row * a.lddy, c, a.cols);
      if (a.du) {
        const floatx4 v = load4(a.y + row * a.ldy, c, a.cols), d = load4(a.du + row * a.lddu, c, a.cols);
        const Stats sy{s[0], s[1], s[2]};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float unit = sy.unit(v[j]);
          g[j] += sy.r * (fmaf(-unit, s[4], d[j] * wn[j]) - s[3]);
          sum[kSumNextW][j] = fmaf(d[j], unit, sum[kSumNextW][j]);
          sum[kSumNextB][j] += d[j];
        }
      }
      if (a.dx) store4(a.dx + row * a.lddx, c, a.cols, floatx4{g.x * a.rs, g.y * a.rs, g.z * a.rs, g.w * a.rs});
      if (!block) continue;
      floatx4 v = zero, unit = zero, dv, each;
      if (a.f) v = load4(a.f + row * a.ldf, c, a.cols);
      if (post) {
        const Stats sf{s[5], s[6], s[7]};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          unit[j] = sf.unit(v[j]);
          v[j] = fmaf(unit[j], wp[j], bp[j]);
        }
      }
      const floatx4 gate = weight4(a.gate ? a.gate + row / a.gate_rows * a.ldgate : nullptr, c, a.cols, 1.0f);
      Words words{};
      if (a.drop.on) words = dropout_words(a.drop, row, c / 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool kept = !a.drop.on || dropout_keeps(a.drop, words, j);
        dv[j] = kept ? g[j] * (a.bs * a.drop.scale) : 0.0f;
        each[j] = kept ? dv[j] * v[j] : 0.0f;
        sum[kSumGate][j] += each[j];
        dv[j] *= gate[j];
        sum[kSumPostB][j] += dv[j];
        if (post) {
          sum[kSumPostW][j] = fmaf(dv[j], unit[j], sum[kSumPostW][j]);
          dv[j] = s[7] * (fmaf(-unit[j], s[9], dv[j] * wp[j]) - s[8]);
        }
      }
      if (a.gate_each) store4(a.dgate + row * a.lddgate, c, a.cols, each);
      if (a.df) store4(a.df + row * a.lddf, c, a.cols, dv);
    }
    if (a.gate_grouped && a.per_group == 1 && a.dgate) {
      store4(a.dgate + (int64_t)group * a.lddgate, c, a.cols, sum[kSumGate]);
      sum[kSumGate] = zero;
    }
  }
#pragma unroll
  for (int i = 0; i < kSums; ++i)
    if (a.sum[i]) store4(a.sum[i] + first * a.sum_step, c, a.cols, sum[i]);
}

// ---------------------------------------------------------------- rows in registers
// A row of up to T x Q x 4 values held by T = 64 NW threads, Q quads of neighbouring columns each, quads T apart.
// One wave (NW = 1): blocks of four waves with a row each, and no barrier.
template <int NW>
constexpr int kRowThreads = NW == 1 ? 256 : 64 * NW;

template <int NW, int Q>
struct RowCols {
  static constexpr int T = 64 * NW;
  int cols, c0;
  bool full, ragged;  // every thread has all its columns; quads are cut off at the end
  uint32_t at[Q];     // where a quad's load starts, in bytes (32 bits and a uniform row: no 64-bit address a lane)
  __device__ __forceinline__ explicit RowCols(int64_t n)
      : cols((int)n), c0((int)(threadIdx.x % T) * 4), full((int)n == T * Q * 4), ragged((n & 3) != 0) {
    // Loads are moved back into the row at its end, so that none waits behind a branch; settle() then shifts the
    // values into place, with zeros for what does not exist.
#pragma unroll
    for (int i = 0; i < Q; ++i) at[i] = 4u * (uint32_t)min(c(i), cols - 4);
  }
  __device__ __forceinline__ int c(int i) const { return c0 + i * T * 4; }
  // How many of a quad's columns exist (or a number beyond 0 .. 4).  Opaque: the compiler would else keep the
  // comparisons of a whole row, two scalar registers each, and spill them.
  __device__ __forceinline__ int have(int i) const {
    int h = cols - c(i);
    asm volatile("" : "+v"(h));
    return h;
  }
  __device__ __forceinline__ floatx4 load(const float* row, int i) const {
    return *reinterpret_cast<const floatx4_u*>(reinterpret_cast<const char*>(row) + at[i]);
  }
  __device__ __forceinline__ void settle(floatx4& v, int i) const {
    if (full) return;
    const int h = have(i);
    if (ragged) v = shift_down(v, h > 0 && h < 4 ? 4 - h : 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < h ? v[j] : 0.0f;
  }
  // Zeros for what does not exist.
  __device__ __forceinline__ void mask(floatx4& v, int i) const {
    if (full) return;
    const int h = have(i);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < h ? v[j] : 0.0f;
  }
  __device__ __forceinline__ void load_row(const float* row, floatx4 (&v)[Q]) const {
#pragma unroll
    for (int i = 0; i < Q; ++i) v[i] = load(row, i);
  }
  __device__ __forceinline__ void settle_row(floatx4 (&v)[Q]) const {
#pragma unroll
    for (int i = 0; i < Q; ++i) settle(v[i], i);
  }
  // A weight's values in the row's columns (`none` where there is no weight), to be settled.
  __device__ __forceinline__ void load_weight(const float* w, float none, floatx4 (&v)[Q]) const {
    if (w) {
      load_row(w, v);
      return;
    }
#pragma unroll
    for (int i = 0; i < Q; ++i) v[i] = splat(none);
  }
  __device__ __forceinline__ void store(float* row, int i, floatx4 v) const {
    float* p = reinterpret_cast<float*>(reinterpret_cast<char*>(row) + 4u * (uint32_t)c(i));
    const int h = have(i);
    if (h >= 4) {
      __builtin_nontemporal_store((floatx4_u)v, reinterpret_cast<floatx4_u*>(p));
      return;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < h) p[j] = v[j];
  }
  // A quad's codes of an 8-bit checkpoint; eight neighbouring threads share a step.
  __device__ __forceinline__ void store_codes(const Act8& out, int64_t row, int i, floatx4 v) const {
    mask(v, i);
    uint32_t top = max(max(act8_magnitude(v.x), act8_magnitude(v.y)), max(act8_magnitude(v.z), act8_magnitude(v.w)));
#pragma unroll
    for (int d = 1; d < 8; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    const uint32_t byte = act8_byte(top);
    const int h = have(i);
    if (h <= 0) return;
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w |= ((uint32_t)act8_code(v[j], byte) & 255u) << (8 * j);
    int8_t* p = out.codes + row * out.cols + (uint32_t)c(i);
    if (h >= 4) {
      *reinterpret_cast<word_u*>(p) = w;
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < h) p[j] = (int8_t)(w >> (8 * j));
    }
    if ((threadIdx.x & 7) == 0) out.scales[((uint32_t)c(i) >> 5) * out.ld + row] = (uint8_t)byte;
  }
  // Bit 4 i + j: the dropout keeps column c(i) + j.
  __device__ __forceinline__ uint32_t kept(const Dropout& d, int64_t row) const {
    static_assert(Q <= 8, "a word has 32 bits");
    if (!d.on) return 0xffffffffu;
    uint32_t bits = 0;
    Dropout o = d;
    if (NW >= 8) asm volatile("" : "+s"(o.key[0]), "+s"(o.key[1]));  // or all rounds' keys stay in registers
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const Words w = dropout_words(o, row, c(i) >> 2);
#pragma unroll
      for (int j = 0; j < 4; ++j) bits |= (uint32_t)dropout_keeps(o, w, j) << (4 * i + j);
    }
    return bits;
  }
};

template <int NW, int Q>
__device__ __forceinline__ Stats row_stats(const Norm& n, const floatx4 (&v)[Q], const RowCols<NW, Q>& rc,
                                           Team<NW>& team) {
  const float share = 1.0f / (float)rc.cols;
  float mean = 0.0f, t[2] = {0.0f, 0.0f};
  if (n.kind == ORCA_HIP_NORM_LAYER) {
    float m[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < Q; ++i) m[0] += (v[i].x + v[i].y) + (v[i].z + v[i].w);
    team.sum(m);
    mean = m[0] * share;
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      floatx4 d = v[i] - mean;
      rc.mask(d, i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t[0] += d[j];
        t[1] = fmaf(d[j], d[j], t[1]);
      }
    }
    team.sum(t);
  } else {
    float q[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < Q; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) q[0] = fmaf(v[i][j], v[i][j], q[0]);
    team.sum(q);
    t[1] = q[0];
  }
  return stats_of(n, mean, t[0], t[1], share);
}

// The forward.  A team takes every step-th row and has the loads of its next row in flight while it works on one:
// the weights stay in registers, since a load behind those would have to wait for them.
template <int NW, int Q, bool JOINT>
__global__ void __launch_bounds__(kRowThreads<NW>) norm_rows_kernel(NormForward a) {
  constexpr int TEAMS = kRowThreads<NW> / (64 * NW);
  __shared__ float lds[2 * NW * 4];
  Team<NW> team{lds};
  const RowCols<NW, Q> rc(a.cols);
  const bool gates = JOINT && a.gate && a.gate_rows != a.rows;  // a gate for each row
  int64_t row = (int64_t)blockIdx.x * TEAMS + (TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
  const int64_t step = (int64_t)gridDim.x * TEAMS;
  if (row >= a.rows) return;
  floatx4 wp[Q], bp[Q], wn[Q], bn[Q], gate[Q];
  floatx4 x1[Q], f1[Q];
  // the weights first, one after the other (with all loads under way together the same: joint 777 x 1501 10.4 us)
  const auto load_weight = [&](const float* w, float none, floatx4 (&v)[Q]) {
    rc.load_weight(w, none, v);
    if (w) rc.settle_row(v);
  };
  load_weight(a.next.w, 1.0f, wn);
  load_weight(a.next.b, 0.0f, bn);
  if (JOINT) {
    load_weight(a.post.w, 1.0f, wp);
    load_weight(a.post.b, 0.0f, bp);
    load_weight(gates ? nullptr : a.gate, 1.0f, gate);
  }
  rc.load_row(a.x + row * a.ldx, x1);
  if (JOINT) rc.load_row(a.f + row * a.ldf, f1);
  while (true) {
    floatx4 v[Q], f[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      v[i] = x1[i];
      if (JOINT) f[i] = f1[i];
    }
    if (gates) rc.load_row(a.gate + (uint32_t)row / (uint32_t)a.gate_rows * a.ldgate, gate);
    const int64_t after = row + step;
    if (after < a.rows) {
      rc.load_row(a.x + after * a.ldx, x1);
      if (JOINT) rc.load_row(a.f + after * a.ldf, f1);
    }
    rc.settle_row(v);
    if (JOINT) {
      const uint32_t kept = rc.kept(a.drop, row);
      rc.settle_row(f);
      if (a.post.kind != ORCA_HIP_NORM_NONE) {
        const Stats s = row_stats<NW, Q>(a.post, f, rc, team);
#pragma unroll
        for (int i = 0; i < Q; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) f[i][j] = fmaf(s.unit(f[i][j]), wp[i][j], bp[i][j]);
      }
      const float k = a.bs * a.drop.scale;
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        floatx4 g = gate[i];
        if (gates) rc.settle(g, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float t = f[i][j] * (g[j] * k);
          v[i][j] = fmaf(a.rs, v[i][j], kept_or_zero(kept, 4 * i + j, t));
        }
        rc.store(a.y + row * a.ldy, i, v[i]);
        rc.mask(v[i], i);  // a bias may have stood behind the row
      }
    }
    if (a.next.kind != ORCA_HIP_NORM_NONE) {
      const Stats s = row_stats<NW, Q>(a.next, v, rc, team);
#pragma unroll
      for (int i = 0; i < Q; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = fmaf(s.unit(v[i][j]), wn[i][j], bn[i][j]);
        rc.store(a.u + row * a.ldu, i, v[i]);
        if (a.u8.codes) rc.store_codes(a.u8, row, i, v[i]);
      }
    }
    if (after >= a.rows) return;
    row = after;
  }
}

// The whole backward of the rows of a block's pieces: NEXT: a gradient through u; BLOCK: the gradients of the
// block; POST: its output is normed; BIAS: a norm has a bias, or its gradient is wanted.
//
// Two stages a row, each with the other one's loads in flight: the next norm (y, du), then the block (dy, f).  The
// weights are in LDS: loads of theirs would wait for those of the rows, and registers go into the sums.
//
// Two blocks a CU are worth about as much as loads ahead: with both norms and biases, eight waves of a row keep to 128
// registers without (8192 x 4096: layer norms 166 us, 180 with loads ahead and one block; rms norms, gate and dropout
// 185 and 177), and four waves, which do for the others, to 256 (159 us without biases; 178 where more left one block).
//
// Spills (the compiler's report): every kernel with BLOCK keeps 34 to 108 scalar registers in lanes of vector ones and
// takes them back inside the row loop (<4, 4, 1, 1, 1, 0>, the large joint's: 97).  <8, 2, 1, 1, 1, 1> spills nine vector
// registers to memory, <8, 4, 1, 1, 1, 1> two.
template <int NW, int Q, bool NEXT, bool BLOCK, bool POST, bool BIAS>
__global__ void __launch_bounds__(kRowThreads<NW>, NW == 8 && Q == 2 ? 4 : NW == 4 && Q == 4 ? 2 : 1)
norm_backward_kernel(NormBackward a) {
  constexpr bool PIPE = !(NEXT && BLOCK && POST && NW == 8);
  constexpr int T = 64 * NW, TEAMS = kRowThreads<NW> / T;
  constexpr int WN = 0, WP = NEXT, BP = WP + POST, GATE = BP + (POST && BIAS), VECTORS = GATE + BLOCK;
  __shared__ float lds[2 * NW * 4];
  __shared__ floatx4 weights[VECTORS * Q * T];
  __shared__ floatx4 sums_lds[TEAMS > 1 ? TEAMS * T * Q : 1];
  Team<NW> team{lds};
  const RowCols<NW, Q> rc(a.cols);
  const int tm = TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0, t = threadIdx.x % T;
  const float share = 1.0f / (float)a.cols, k = a.bs * a.drop.scale;
  const bool gates = BLOCK && a.gate && a.gate_rows != a.rows;  // a gate for each row
  const int units = a.groups * a.per_group, step = a.per_group * TEAMS;
  floatx4 v[Q], d[Q], g[Q], f[Q];
  // The loads of a row's stages.
  const auto load_next = [&](int64_t row) {
    rc.load_row(a.y + row * a.ldy, v);
    rc.load_row(a.du + row * a.lddu, d);
  };
  const auto load_block = [&](int64_t row) {
    if (a.dy) rc.load_row(a.dy + row * a.lddy, g);
    if (BLOCK && a.f) rc.load_row(a.f + row * a.ldf, f);
  };
  // The first row of a unit, with its loads under way.
  int group, r1;
  int64_t row;
  const auto start = [&](int unit) {
    group = unit / a.per_group;
    r1 = (group + 1) * a.group_rows;
    row = group * a.group_rows + unit % a.per_group * TEAMS + tm;
    if (!PIPE || row >= r1) return;
    if (NEXT) load_next(row);
    load_block(row);
  };
  start(blockIdx.x);
  {
    floatx4 w[VECTORS][Q];
    if (NEXT) rc.load_weight(a.next.w, 1.0f, w[WN]);
    if (POST) rc.load_weight(a.post.w, 1.0f, w[WP]);
    if (POST && BIAS) rc.load_weight(a.post.b, 0.0f, w[BP]);
    if (BLOCK) rc.load_weight(gates ? nullptr : a.gate, 1.0f, w[GATE]);
    // a thread reads only what it wrote (all teams write the same)
#pragma unroll
    for (int n = 0; n < VECTORS; ++n) {
      rc.settle_row(w[n]);
#pragma unroll
      for (int i = 0; i < Q; ++i) weights[(n * Q + i) * T + t] = w[n][i];
    }
  }
  const auto weight = [&](int n, int i) { return weights[(n * Q + i) * T + t]; };
  floatx4 sum[kSums][Q];
#pragma unroll
  for (int n = 0; n < kSums; ++n)
#pragma unroll
    for (int i = 0; i < Q; ++i) sum[n][i] = splat(0.0f);
  // the block's teams' sums, added up, to `out`
  const auto flush = [&](floatx4 (&v)[Q], float* out) {
    if constexpr (TEAMS > 1) {
#pragma unroll
      for (int i = 0; i < Q; ++i) sums_lds[(tm * Q + i) * T + t] = v[i];
      __syncthreads();
      if (tm == 0) {
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          floatx4 s = v[i];
#pragma unroll
          for (int m = 1; m < TEAMS; ++m) s += sums_lds[(m * Q + i) * T + t];
          rc.store(out, i, s);
        }
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int i = 0; i < Q; ++i) rc.store(out, i, v[i]);
    }
  };
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
    if (unit != (int)blockIdx.x) start(unit);
    for (; row < r1; row += step) {
      const bool more = row + step < r1;
      if (!PIPE) {
        load_next(row);
        load_block(row);
      }
      const uint32_t kept = BLOCK ? rc.kept(a.drop, row) : 0;
      Stats s{0.0f, 0.0f, 0.0f};
      float c1 = 0.0f, c2 = 0.0f;
      if (NEXT) {
        rc.settle_row(v);
        rc.settle_row(d);
        s = row_stats<NW, Q>(a.next, v, rc, team);
        float e[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          const floatx4 wn = weight(WN, i);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[i][j] = s.unit(v[i][j]);
            sum[kSumNextW][i][j] = fmaf(d[i][j], v[i][j], sum[kSumNextW][i][j]);
            if (BIAS) sum[kSumNextB][i][j] += d[i][j];
            d[i][j] *= wn[j];
            e[0] += d[i][j];
            e[1] = fmaf(d[i][j], v[i][j], e[1]);
          }
        }
        team.sum(e);
        c1 = a.next.kind == ORCA_HIP_NORM_LAYER ? e[0] * share : 0.0f;
        c2 = e[1] * share;
      }
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        if (a.dy)
          rc.settle(g[i], i);
        else
          g[i] = splat(0.0f);
        if (NEXT) {
#pragma unroll
          for (int j = 0; j < 4; ++j) g[i][j] = fmaf(s.r, fmaf(-v[i][j], c2, d[i][j]) - c1, g[i][j]);
        }
        if (a.dx) rc.store(a.dx + row * a.lddx, i, g[i] * a.rs);
      }
      if (PIPE && NEXT && more) load_next(row + step);
      if (!BLOCK) {
        if (more) load_block(row + step);
        continue;
      }
      if (a.f)
        rc.settle_row(f);
      else
#pragma unroll
        for (int i = 0; i < Q; ++i) f[i] = splat(0.0f);
      if (POST) s = row_stats<NW, Q>(a.post, f, rc, team);
      float e[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        floatx4 each, wp, bp, gate;
        if (POST) wp = weight(WP, i);
        if (POST && BIAS) bp = weight(BP, i);
        if (gates) {
          gate = rc.load(a.gate + (a.gate_rows == 1 ? row : group) * a.ldgate, i);
          rc.settle(gate, i);
        } else {
          gate = weight(GATE, i);
        }
        rc.mask(g[i], i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (POST) f[i][j] = s.unit(f[i][j]);
          const float out = POST ? BIAS ? fmaf(f[i][j], wp[j], bp[j]) : f[i][j] * wp[j] : f[i][j];
          float dv = kept_or_zero(kept, 4 * i + j, g[i][j] * k);
          each[j] = kept_or_zero(kept, 4 * i + j, dv * out);
          sum[kSumGate][i][j] += each[j];
          dv *= gate[j];
          if (POST) {
            sum[kSumPostW][i][j] = fmaf(dv, f[i][j], sum[kSumPostW][i][j]);
            if (BIAS) sum[kSumPostB][i][j] += dv;
            dv *= wp[j];
            e[0] += dv;
            e[1] = fmaf(dv, f[i][j], e[1]);
          }
          g[i][j] = dv;
        }
        if (a.gate_each) rc.store(a.dgate + row * a.lddgate, i, each);
      }
      if (POST) {
        team.sum(e);
        c1 = a.post.kind == ORCA_HIP_NORM_LAYER ? e[0] * share : 0.0f;
        c2 = e[1] * share;
#pragma unroll
        for (int i = 0; i < Q; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) g[i][j] = s.r * (fmaf(-f[i][j], c2, g[i][j]) - c1);
      }
      if (a.df) {
#pragma unroll
        for (int i = 0; i < Q; ++i) rc.store(a.df + row * a.lddf, i, g[i]);
      }
      if (PIPE && more) load_block(row + step);
    }
    if (BLOCK && a.gate_grouped && a.per_group == 1 && a.dgate) {
      flush(sum[kSumGate], a.dgate + (int64_t)group * a.lddgate);
#pragma unroll
      for (int i = 0; i < Q; ++i) sum[kSumGate][i] = splat(0.0f);
    }
  }
#pragma unroll
  for (int n = 0; n < kSums; ++n)
    if (a.sum[n]) flush(sum[n], a.sum[n] + blockIdx.x * a.sum_step);
}

// ---------------------------------------------------------------- the blocks' partial sums
struct NormFinish {
  int64_t cols, blocks, step;  // of the partial sums; `step` floats from one block's to the next one's
  int count;                   // sums over all blocks
  const float* from[kSums];
  float* to[kSums];
  const float* gate_from;  // and over each group's blocks
  float* dgate;
  int64_t lddgate, groups, per_group;
};
// A block adds up 32 columns: a thread four columns of every 64th partial sum, eight of them in flight, then the
// eight threads of a wave and the eight waves that have the same columns.
__global__ void __launch_bounds__(512) norm_finish_kernel(NormFinish a) {
  __shared__ floatx4 lds[8][8];
  const int q = threadIdx.x & 7, k = threadIdx.x >> 3, wave = threadIdx.x >> 6;
  const int64_t c = ((int64_t)blockIdx.x * 8 + q) * 4, at = max((int64_t)0, min(c, a.cols - 4));
  for (int64_t i = blockIdx.y; i < a.count + a.groups; i += gridDim.y) {
    const int64_t group = i - a.count;
    const float* from = group < 0 ? a.from[i] : a.gate_from + group * a.per_group * a.step;
    float* to = group < 0 ? a.to[i] : a.dgate + group * a.lddgate;
    const int64_t blocks = group < 0 ? a.blocks : a.per_group;
    floatx4 t = splat(0.0f);
    for (int64_t b0 = k; b0 < blocks; b0 += 64 * 8) {
      floatx4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float* p = from + min(b0 + 64 * u, blocks - 1) * a.step;
        v[u] = a.cols < 4 ? load4(p, c, a.cols) : *reinterpret_cast<const floatx4_u*>(p + at);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (b0 + 64 * u >= blocks) v[u] = splat(0.0f);
      t += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    if (a.cols >= 4) t = shift_down(t, (int)min((int64_t)3, c - at));  // what lies behind the row is not stored
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int d = 8; d < 64; d *= 2) t[j] += __shfl_xor(t[j], d);
    if ((threadIdx.x & 63) < 8) lds[wave][q] = t;
    __syncthreads();
    if (threadIdx.x < 8 && c < a.cols) {
#pragma unroll
      for (int w = 1; w < 8; ++w) t += lds[w][q];
      store4(to, c, a.cols, t);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- host
void check_norm(const char* op, const orca_hip_norm_params& n, bool none) {
  if (n.kind < (none ? ORCA_HIP_NORM_NONE : ORCA_HIP_NORM_LAYER) || n.kind > ORCA_HIP_NORM_RMS)
    fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": unknown norm " + std::to_string(n.kind));
  if (n.kind != ORCA_HIP_NORM_NONE && !(n.eps >= 0.0f && n.eps < INFINITY))
    fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": eps must be a finite number from 0 on");
}
Norm norm_of(const orca_hip_norm_params& n) {
  Norm r;
  r.kind = n.kind;
  if (n.kind == ORCA_HIP_NORM_NONE) return r;
  r.eps = n.eps;
  r.w = n.weight;
  r.b = n.bias;
  return r;
}
void check_block(const char* op, const char* gate, size_t rows, size_t cols, const orca_hip_residual_block& b) {
  check_norm(op, b.post, true);
  check_norm(op, b.next, true);
  if (!(b.p >= 0.0 && b.p <= 1.0))
    fail(ORCA_HIP_ERR_INTERNAL, std::string(op) + ": a dropout's p must be from 0 to 1");
  if (!b.gate) return;
  if (!b.groups || b.groups >> kMaxSizeBits || rows % b.groups)
    fail_shape(op, "a number of gate rows that divides " + std::to_string(rows), std::to_string(b.groups));
  check_ld(gate, b.ldgate, cols);
}
Span vector_span(const float* p, size_t cols) { return buffer_span(p, 4 * cols); }

// The operands of a call with what they are, for the checks that each call makes.
struct Operand {
  Span span;
  const char* what;
};
void check_operands(orca_hip_ctx* ctx, const char* op, std::initializer_list<Operand> operands) {
  for (const Operand& o : operands) {
    if (!o.span.p || !o.span.bytes()) continue;
    size_t have = 0;
    const auto where = ctx->alloc.locate(o.span.p, &have);
    if (where == CachingAllocator::Where::kUnknown ||
        (where == CachingAllocator::Where::kLive && o.span.bytes() <= have))
      continue;
    check_extent(ctx, o.span.p, o.span.bytes(), (std::string(op) + " (" + o.what + ")").c_str());  // fails
  }
}

constexpr unsigned kMaxBlocks = 1u << 20;  // of 256 threads and more; the kernels step over the rest

// Rows of up to 8192 values stay in registers; longer ones, and rows shorter than a quad, are gone over in passes.
constexpr int64_t kMaxRegisterRow = 8192;
// Calls f with the waves of a row and the quads of a thread, as template arguments.  Rows of 2049 to 4096 values: four
// waves, or eight (`many`) where four would have no registers left (kept quads and sums of both norms).
template <class F>
void with_row_shape(int64_t cols, bool many, F f) {
  using std::integral_constant;
  if (cols <= 256) return f(integral_constant<int, 1>(), integral_constant<int, 1>());
  if (cols <= 512) return f(integral_constant<int, 1>(), integral_constant<int, 2>());
  if (cols <= 1024) return f(integral_constant<int, 1>(), integral_constant<int, 4>());
  if (cols <= 2048) return f(integral_constant<int, 4>(), integral_constant<int, 2>());
  if (cols <= 4096 && many) return f(integral_constant<int, 8>(), integral_constant<int, 2>());
  if (cols <= 4096) return f(integral_constant<int, 4>(), integral_constant<int, 4>());
  return f(integral_constant<int, 8>(), integral_constant<int, 4>());
}
constexpr int kForwardBlocks = 4;  // a CU
bool in_registers(int64_t cols) { return cols >= 4 && cols <= kMaxRegisterRow; }

template <int NW, int Q>
void launch_forward_rows(orca_hip_ctx* ctx, const NormForward& a, bool joint) {
  constexpr int TEAMS = kRowThreads<NW> / (64 * NW);
  const dim3 grid((unsigned)std::min<int64_t>((a.rows + TEAMS - 1) / TEAMS, (int64_t)ctx->num_cus * kForwardBlocks));
  auto kernel = norm_rows_kernel<NW, Q, NW == 8 && Q == 2>;  // of with_row_shape's two for 2049 to 4096 values
  if constexpr (!(NW == 8 && Q == 2) && !(NW == 4 && Q == 4))
    kernel = joint ? norm_rows_kernel<NW, Q, true> : norm_rows_kernel<NW, Q, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kRowThreads<NW>), 0, ctx->stream, a);
}
void launch_forward(orca_hip_ctx* ctx, const NormForward& a, bool joint) {
  if (!in_registers(a.cols)) {
    const dim3 grid((unsigned)std::min<int64_t>(a.rows, kMaxBlocks));
    hipLaunchKernelGGL(joint ? norm_stream_kernel<true> : norm_stream_kernel<false>, grid, dim3(kStream), 0, ctx->stream,
                       a);
  } else if (a.cols > 512 && a.cols <= 1024 && a.rows <= 4 * ctx->num_cus) {
    // four waves a row where one a row would leave CUs without any (joint 777 x 1003: 7.8 us for 9.4, but
    // 2048 x 1024 8.9 for 8.4)
    launch_forward_rows<4, 1>(ctx, a, joint);
  } else {
    // joint 300 x 3000: 9.4 us in eight waves, 9.8 in four, 8192 x 2100 73 and 77; norm 1024 x 4096 7.0 in four, 8.5 in
    // eight
    with_row_shape(a.cols, joint, [&](auto nw, auto q) {
      launch_forward_rows<decltype(nw)::value, decltype(q)::value>(ctx, a, joint);
    });
  }
  ORCA_HIP_CHECK(hipGetLastError());
}

// Blocks of a backward.  Two a CU: fewer leave memory idle, more make more partial sums (norm 8192 x 4096: 99 us with two
// a CU, 111 with one, 107 with four).  One where a CU holds no more: rows of more than 4096 (4096 x 8192 105 us, 107 with
// two), and a wave's rows of 513 to 1024 with both norms (2048 x 1024 with biases 22 for 30, without 20 for 27; 8192 x 1003
// 58 for 70 and 56 for 66).  Up to four of the smallest rows, 16 rows a block at least (131072 x 64 51 us, 71 with two;
// 131072 x 256 80 and 86; joint 30000 x 200 43 and 48).
int64_t backward_blocks(const orca_hip_ctx* ctx, int64_t rows, int64_t cols, bool both) {
  if (cols > 4096 || (cols > 512 && cols <= 1024 && both)) return ctx->num_cus;
  if (cols <= 256) return std::max<int64_t>(2 * ctx->num_cus, std::min<int64_t>(4 * ctx->num_cus, rows / 16));
  return 2 * ctx->num_cus;
}

// Each of a block's teams adds up its rows one after the other: so many at most, and up to twice as many in whole groups
// (2^25 rows of four columns, of one value each: off by up to 7e-6, and by 1.2e-4 in chains of 8192).  Beyond the usual
// blocks times that many rows there are more blocks; a vector of partial sums takes 1 / 512 of an operand's bytes then.
constexpr int64_t kMaxChain = 512;

template <int NW, int Q, bool BIAS>
auto backward_kernel(bool next, bool block, bool post) {
  if (!next) return post ? norm_backward_kernel<NW, Q, false, true, true, BIAS>
                         : norm_backward_kernel<NW, Q, false, true, false, false>;
  if (!block) return norm_backward_kernel<NW, Q, true, false, false, BIAS>;
  constexpr bool EIGHT = BIAS && NW == 4 && Q == 4;  // both norms with biases: with_row_shape's eight waves
  return post ? norm_backward_kernel<NW, Q, true, true, true, BIAS && !EIGHT>
              : norm_backward_kernel<NW, Q, true, true, false, BIAS>;
}
template <int NW, int Q>
void launch_backward_rows(orca_hip_ctx* ctx, const NormBackward& a, bool block, bool bias, unsigned blocks) {
  const bool post = a.post.kind != ORCA_HIP_NORM_NONE;
  void (*kernel)(NormBackward);
  if constexpr (NW == 8 && Q == 2)  // the shape for this one alone (with_row_shape)
    kernel = norm_backward_kernel<NW, Q, true, true, true, true>;
  else
    kernel = bias ? backward_kernel<NW, Q, true>(a.du, block, post) : backward_kernel<NW, Q, false>(a.du, block, post);
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kRowThreads<NW>), 0, ctx->stream, a);
}

void launch_finish(orca_hip_ctx* ctx, const NormFinish& f) {
  const int64_t outs = f.count + f.groups;
  if (!outs) return;
  hipLaunchKernelGGL(norm_finish_kernel, dim3((unsigned)((f.cols + 31) / 32), (unsigned)std::min<int64_t>(outs, 32768)),
                     dim3(512), 0, ctx->stream, f);
  ORCA_HIP_CHECK(hipGetLastError());
}

// Runs a backward; `to` are the results of the sums (null: not wanted).  dgate has `gate_rows` rows.
void launch_backward(orca_hip_ctx* ctx, NormBackward& a, float* const (&to)[kSums], int64_t gate_rows, const char* op) {
  if (!a.rows) {  // sums of nothing
    NormFinish fin{};
    fin.cols = a.cols;
    for (int i = 0; i < kSums; ++i)
      if (to[i] && i != kSumGate) fin.to[fin.count++] = to[i];
    if (to[kSumGate]) {
      fin.dgate = to[kSumGate];
      fin.lddgate = a.lddgate;
      fin.groups = gate_rows;
    }
    return launch_finish(ctx, fin);
  }
  a.gate_rows = gate_rows ? a.rows / gate_rows : a.rows;
  a.gate_each = to[kSumGate] && a.gate_rows == 1;
  const bool gate_sum = to[kSumGate] && !a.gate_each;
  a.gate_grouped = a.gate_rows != 1 && a.gate_rows != a.rows;
  a.groups = a.gate_grouped ? (int)(a.rows / a.gate_rows) : 1;
  a.group_rows = (int)(a.gate_grouped ? a.gate_rows : a.rows);
  const bool block = a.df || to[kSumGate] || to[kSumPostW] || to[kSumPostB];
  const bool registers = in_registers(a.cols);
  // What the split of the rows and their shape go by: the parameters, and not which results are wanted, but for a
  // bias's gradient of norms that have none: four waves would spill 36 registers on it (8192 x 4096: 198 us for 180).
  const bool both = a.du && a.post.kind != ORCA_HIP_NORM_NONE,
             heavy = both && (a.post.b || a.next.b || to[kSumPostB] || to[kSumNextB]);
  const int64_t strips = registers ? 1 : (a.cols + kStream * 4 - 1) / (kStream * 4);
  int64_t blocks = registers ? backward_blocks(ctx, a.rows, a.cols, both)
                             : std::max<int64_t>(1, 2 * ctx->num_cus / strips);
  const bool few = registers && a.groups == 1 && a.rows <= (a.cols <= 1024 ? 8 : 2);
  const int64_t span = kMaxChain * (registers && a.cols <= 1024 ? 4 : 1);  // rows that a block adds up
  const int64_t least_pieces = (a.group_rows + span - 1) / span;
  if (few) {
    // one block, without a launch for partial sums (norm 8 x 512: 6.1 us for 9.0, 2 x 4096 6.9 for 8.9; but 4 x 4096 10.4
    // for 8.5, joint 16 x 1000 25 for 16)
    blocks = a.per_group = 1;
  } else if (a.groups >= blocks && least_pieces == 1) {
    a.per_group = 1;
    blocks = std::max(blocks, (a.rows + span - 1) / span);
  } else {
    const int64_t least = registers ? a.cols <= 1024 ? 4 : 1 : 16;  // rows of a piece
    const int64_t most =
        std::max(least_pieces, std::min<int64_t>(blocks / a.groups, (a.group_rows + least - 1) / least));
    // no more pieces than the longest one's rows ask for: less to add up, and no later an end
    const int64_t longest = (a.group_rows + least * most - 1) / (least * most) * least;
    a.per_group = (int)((a.group_rows + longest - 1) / longest);
    blocks = (int64_t)a.groups * a.per_group;
  }
  // slots of the partial sums
  NormFinish fin{};
  fin.cols = a.cols;
  fin.blocks = blocks;
  fin.per_group = a.per_group;
  const bool direct = blocks == 1;
  const bool gate_slot = gate_sum && !(a.gate_grouped && a.per_group == 1);
  int slots = 0;
  int slot[kSums];
  for (int i = 0; i < kSums; ++i) slot[i] = to[i] && (i != kSumGate || gate_slot) ? slots++ : -1;
  std::unique_ptr<Scratch> ws, stats;
  const size_t step = (size_t)slots * a.cols;
  if (!direct && slots) ws = workspace(ctx, sizeof(float) * step * blocks, op);
  a.sum_step = direct ? 0 : (int64_t)step;
  fin.step = (int64_t)step;
  for (int i = 0; i < kSums; ++i) {
    a.sum[i] = nullptr;
    if (slot[i] < 0) continue;
    float* out = to[i];
    float* p = ws ? ws->as<float>() + (size_t)slot[i] * a.cols : nullptr;
    a.sum[i] = direct ? out : p;
    if (i == kSumGate && a.gate_grouped) {
      fin.gate_from = p;
      fin.dgate = out;
      fin.lddgate = a.lddgate;
      fin.groups = a.groups;
    } else {
      fin.from[fin.count] = p;
      fin.to[fin.count++] = out;
    }
  }
  if (registers) {
    const bool bias = a.post.b || to[kSumPostB] || to[kSumNextB];
    with_row_shape(a.cols, heavy, [&](auto nw, auto q) {
      launch_backward_rows<decltype(nw)::value, decltype(q)::value>(ctx, a, block, bias, (unsigned)blocks);
    });
    ORCA_HIP_CHECK(hipGetLastError());
    if (!direct) launch_finish(ctx, fin);
    return;
  }
  if (a.du || (block && a.post.kind != ORCA_HIP_NORM_NONE)) {
    stats = workspace(ctx, sizeof(float) * kRowStats * a.rows, op);
    a.stats = stats->as<float>();
    hipLaunchKernelGGL(norm_stats_kernel, dim3((unsigned)std::min<int64_t>(a.rows, kMaxBlocks)), dim3(kStream), 0,
                       ctx->stream, a, block);
    ORCA_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(norm_strip_kernel, dim3((unsigned)(strips * blocks)), dim3(kStream), 0, ctx->stream, a, block);
  ORCA_HIP_CHECK(hipGetLastError());
  if (!direct) launch_finish(ctx, fin);
}

}  // namespace
}  // namespace orca_hip

using namespace orca_hip;

extern "C" {

int orca_hip_norm(orca_hip_ctx* ctx, size_t rows, size_t cols, const float* x, size_t ldx,
                  const orca_hip_norm_params* norm, float* y, size_t ldy, void* y8) {
  return guard([&] {
    const char* op = "norm";
    check_sizes(op, {rows, cols});
    if (!norm) fail(ORCA_HIP_ERR_INTERNAL, "norm: null parameters");
    check_norm(op, *norm, false);
    check_ld("norm (x)", ldx, cols);
    check_ld("norm (y)", ldy, cols);
    if (rows && cols && (!x || !y)) fail(ORCA_HIP_ERR_INTERNAL, "norm: null operand");
    const Span xs = matrix_span(x, rows, cols, ldx), ys = matrix_span(y, rows, cols, ldy),
               ws = vector_span(norm->weight, cols), bs = vector_span(norm->bias, cols),
               y8s = buffer_span(y8, act8_layout(rows, cols).bytes);
    for (const Span& in : {ws, bs}) check_apart(op, ys, in);
    for (const Span& in : {xs, ws, bs}) check_apart(op, y8s, in);
    if (x != y || ldx != ldy) check_apart(op, ys, xs);  // y over x, row by row, is in order
    check_apart(op, y8s, ys);
    act8_aligned(y8, op);
    bind(ctx);
    if (!rows || !cols) return;
    check_operands(ctx, op, {{xs, "x"}, {ws, "weight"}, {bs, "bias"}, {ys, "y"}, {y8s, "y8"}});
    NormForward a{};
    a.rows = (int64_t)rows;
    a.cols = (int64_t)cols;
    a.x = x;
    a.ldx = (int64_t)ldx;
    a.u = y;
    a.ldu = (int64_t)ldy;
    a.u8 = act8_at(y8, rows, cols);
    a.next = norm_of(*norm);
    ProfScope prof(ctx, op, 7.0 * rows * cols, 8.0 * rows * cols + (double)(y8 ? y8s.bytes() : 0));
    launch_forward(ctx, a, false);
  });
}

int orca_hip_norm_backward(orca_hip_ctx* ctx, size_t rows, size_t cols, const float* dy, size_t lddy, const float* x,
                           size_t ldx, const orca_hip_norm_params* norm, const float* dx_add, size_t ldadd, float* dx,
                           size_t lddx, float* dweight, float* dbias) {
  return guard([&] {
    const char* op = "norm_backward";
    check_sizes(op, {rows, cols});
    if (!norm) fail(ORCA_HIP_ERR_INTERNAL, "norm_backward: null parameters");
    check_norm(op, *norm, false);
    check_ld("norm_backward (dy)", lddy, cols);
    check_ld("norm_backward (x)", ldx, cols);
    if (dx) check_ld("norm_backward (dx)", lddx, cols);
    if (dx && dx_add) check_ld("norm_backward (dx_add)", ldadd, cols);
    if (rows && cols && (!dy || !x)) fail(ORCA_HIP_ERR_INTERNAL, "norm_backward: null operand");
    const Span dys = matrix_span(dy, rows, cols, lddy), xs = matrix_span(x, rows, cols, ldx),
               ws = vector_span(norm->weight, cols), add = matrix_span(dx ? dx_add : nullptr, rows, cols, ldadd),
               dxs = matrix_span(dx, rows, cols, lddx), dws = vector_span(dweight, cols), dbs = vector_span(dbias, cols);
    const Span outs[3] = {dxs, dws, dbs};
    for (int i = 0; i < 3; ++i) {
      for (const Span& in : {dys, xs, ws}) check_apart(op, outs[i], in);
      // dx over dx_add, row by row, is in order (a gradient added up in place)
      if (!(i == 0 && dx_add == dx && ldadd == lddx)) check_apart(op, outs[i], add);
      for (int j = 0; j < i; ++j) check_apart(op, outs[i], outs[j]);
    }
    bind(ctx);
    check_operands(ctx, op, {{dys, "dy"}, {xs, "x"}, {ws, "weight"}, {add, "dx_add"}, {dxs, "dx"}, {dws, "dweight"},
                             {dbs, "dbias"}});
    if (!cols || (!dx && !dweight && !dbias)) return;
    NormBackward a{};
    a.rows = (int64_t)rows;
    a.cols = (int64_t)cols;
    a.dy = static_cast<const float*>(add.p);
    a.lddy = (int64_t)ldadd;
    a.du = dy;
    a.lddu = (int64_t)lddy;
    a.y = x;
    a.ldy = (int64_t)ldx;
    a.next = norm_of(*norm);
    a.rs = 1.0f;
    a.dx = dx;
    a.lddx = (int64_t)lddx;
    float* const to[kSums] = {nullptr, nullptr, nullptr, dweight, dbias};
    ProfScope prof(ctx, op, 16.0 * rows * cols, 4.0 * (2 + (dx != nullptr) + (add.p != nullptr)) * rows * cols);
    launch_backward(ctx, a, to, 0, op);
  });
}

int orca_hip_residual_norm(orca_hip_ctx* ctx, size_t rows, size_t cols, const float* x, size_t ldx, const float* f,
                           size_t ldf, const orca_hip_residual_block* block, float* y, size_t ldy, float* u,
                           size_t ldu, void* u8) {
  return guard([&] {
    const char* op = "residual_norm";
    check_sizes(op, {rows, cols});
    if (!block) fail(ORCA_HIP_ERR_INTERNAL, "residual_norm: null parameters");
    const orca_hip_residual_block& p = *block;
    check_block(op, "residual_norm (gate)", rows, cols, p);
    const bool next = p.next.kind != ORCA_HIP_NORM_NONE;
    check_ld("residual_norm (x)", ldx, cols);
    check_ld("residual_norm (f)", ldf, cols);
    check_ld("residual_norm (y)", ldy, cols);
    if (next) check_ld("residual_norm (u)", ldu, cols);
    if (!next && (u || u8)) fail(ORCA_HIP_ERR_INTERNAL, "residual_norm: u without a next norm");
    if (rows && cols && (!x || !f || !y || (next && !u))) fail(ORCA_HIP_ERR_INTERNAL, "residual_norm: null operand");
    const Norm post = norm_of(p.post), nx = norm_of(p.next);
    const Span xs = matrix_span(x, rows, cols, ldx), fs = matrix_span(f, rows, cols, ldf),
               ys = matrix_span(y, rows, cols, ldy), us = matrix_span(u, rows, cols, ldu),
               u8s = buffer_span(u8, act8_layout(rows, cols).bytes),
               gate = matrix_span(p.gate, p.gate ? p.groups : 0, cols, p.ldgate), pw = vector_span(post.w, cols),
               pb = vector_span(post.b, cols), nw = vector_span(nx.w, cols), nb = vector_span(nx.b, cols);
    const Span outs[3] = {ys, us, u8s};
    for (int i = 0; i < 3; ++i) {
      for (const Span& in : {fs, gate, pw, pb, nw, nb}) check_apart(op, outs[i], in);
      // y over x, element by element, is in order
      if (!(i == 0 && x == y && ldx == ldy)) check_apart(op, outs[i], xs);
      for (int j = 0; j < i; ++j) check_apart(op, outs[i], outs[j]);
    }
    act8_aligned(u8, op);
    bind(ctx);
    if (!rows || !cols) return;
    check_operands(ctx, op, {{xs, "x"}, {fs, "f"}, {gate, "gate"}, {pw, "post weight"}, {pb, "post bias"},
                             {nw, "next weight"}, {nb, "next bias"}, {ys, "y"}, {us, "u"}, {u8s, "u8"}});
    NormForward a{};
    a.rows = (int64_t)rows;
    a.cols = (int64_t)cols;
    a.x = x;
    a.ldx = (int64_t)ldx;
    a.f = f;
    a.ldf = (int64_t)ldf;
    a.y = y;
    a.ldy = (int64_t)ldy;
    a.u = u;
    a.ldu = (int64_t)ldu;
    a.u8 = act8_at(u8, rows, cols);
    a.post = post;
    a.next = nx;
    a.gate = p.gate;
    a.ldgate = (int64_t)p.ldgate;
    a.gate_rows = p.gate ? (int64_t)(rows / p.groups) : 1;
    a.rs = p.residual_scale;
    a.bs = p.block_scale;
    a.drop = dropout_of(p.p, p.seed, p.offset);
    ProfScope prof(ctx, op, 12.0 * rows * cols, 4.0 * (3 + next) * rows * cols + (double)(u8 ? u8s.bytes() : 0));
    launch_forward(ctx, a, true);
  });
}

int orca_hip_residual_norm_backward(orca_hip_ctx* ctx, size_t rows, size_t cols, const float* dy, size_t lddy,
                                    const float* du, size_t lddu, const float* f, size_t ldf, const float* y,
                                    size_t ldy, const orca_hip_residual_block* block,
                                    const orca_hip_residual_grads* grads) {
  return guard([&] {
    const char* op = "residual_norm_backward";
    check_sizes(op, {rows, cols});
    if (!block || !grads) fail(ORCA_HIP_ERR_INTERNAL, "residual_norm_backward: null parameters");
    const orca_hip_residual_block& p = *block;
    const orca_hip_residual_grads& o = *grads;
    check_block(op, "residual_norm_backward (gate)", rows, cols, p);
    const bool post = p.post.kind != ORCA_HIP_NORM_NONE;
    if (du && p.next.kind == ORCA_HIP_NORM_NONE)
      fail(ORCA_HIP_ERR_INTERNAL, "residual_norm_backward: du without a next norm");
    if (!du && (o.dnext_weight || o.dnext_bias))
      fail(ORCA_HIP_ERR_INTERNAL, "residual_norm_backward: the next norm's gradients need du");
    if (!post && (o.dpost_weight || o.dpost_bias))
      fail(ORCA_HIP_ERR_INTERNAL, "residual_norm_backward: gradients of a post norm that is not there");
    if (o.dgate && !p.gate) fail(ORCA_HIP_ERR_INTERNAL, "residual_norm_backward: a gradient without its gate");
    const bool through = o.df || o.dgate || o.dpost_weight || o.dpost_bias;  // something of the block is wanted
    const bool reads_f = (through && post) || o.dgate;
    if (rows && cols && !dy && !du) fail(ORCA_HIP_ERR_INTERNAL, "residual_norm_backward: one of dy and du is needed");
    if (rows && cols && ((du && !y) || (reads_f && !f)))
      fail(ORCA_HIP_ERR_INTERNAL, "residual_norm_backward: null operand");
    if (dy) check_ld("residual_norm_backward (dy)", lddy, cols);
    if (du) check_ld("residual_norm_backward (du)", lddu, cols);
    if (du) check_ld("residual_norm_backward (y)", ldy, cols);
    if (reads_f) check_ld("residual_norm_backward (f)", ldf, cols);
    if (o.dx) check_ld("residual_norm_backward (dx)", o.lddx, cols);
    if (o.df) check_ld("residual_norm_backward (df)", o.lddf, cols);
    if (o.dgate) check_ld("residual_norm_backward (dgate)", o.lddgate, cols);
    const Norm pn = norm_of(p.post), nx = norm_of(p.next);
    const Span dys = matrix_span(dy, rows, cols, lddy), dus = matrix_span(du, rows, cols, lddu),
               fs = matrix_span(reads_f ? f : nullptr, rows, cols, ldf),
               ys = matrix_span(du ? y : nullptr, rows, cols, ldy),
               gate = matrix_span(p.gate, p.gate ? p.groups : 0, cols, p.ldgate), pw = vector_span(pn.w, cols),
               pb = vector_span(pn.b, cols), nw = vector_span(nx.w, cols),
               dxs = matrix_span(o.dx, rows, cols, o.lddx), dfs = matrix_span(o.df, rows, cols, o.lddf),
               dgs = matrix_span(o.dgate, o.dgate ? p.groups : 0, cols, o.lddgate),
               dpw = vector_span(o.dpost_weight, cols), dpb = vector_span(o.dpost_bias, cols),
               dnw = vector_span(o.dnext_weight, cols), dnb = vector_span(o.dnext_bias, cols);
    const Span outs[7] = {dxs, dfs, dgs, dpw, dpb, dnw, dnb};
    for (int i = 0; i < 7; ++i) {
      for (const Span& in : {dus, fs, ys, gate, pw, pb, nw}) check_apart(op, outs[i], in);
      // dx over dy, element by element, is in order
      if (!(i == 0 && o.dx == dy && o.lddx == lddy)) check_apart(op, outs[i], dys);
      for (int j = 0; j < i; ++j) check_apart(op, outs[i], outs[j]);
    }
    bind(ctx);
    check_operands(ctx, op, {{dys, "dy"}, {dus, "du"}, {fs, "f"}, {ys, "y"}, {gate, "gate"}, {pw, "post weight"},
                             {pb, "post bias"}, {nw, "next weight"}, {dxs, "dx"}, {dfs, "df"}, {dgs, "dgate"},
                             {dpw, "dpost_weight"}, {dpb, "dpost_bias"}, {dnw, "dnext_weight"}, {dnb, "dnext_bias"}});
    if (!cols || (!through && !o.dx && !o.dnext_weight && !o.dnext_bias)) return;
    NormBackward a{};
    a.rows = (int64_t)rows;
    a.cols = (int64_t)cols;
    a.dy = dy;
    a.lddy = (int64_t)lddy;
    a.du = du;
    a.lddu = (int64_t)lddu;
    a.f = static_cast<const float*>(fs.p);
    a.ldf = (int64_t)ldf;
    a.y = y;
    a.ldy = (int64_t)ldy;
    a.post = pn;
    a.next = nx;
    a.gate = p.gate;
    a.ldgate = (int64_t)p.ldgate;
    a.rs = p.residual_scale;
    a.bs = p.block_scale;
    a.drop = dropout_of(p.p, p.seed, p.offset);
    a.dx = o.dx;
    a.lddx = (int64_t)o.lddx;
    a.df = o.df;
    a.lddf = (int64_t)o.lddf;
    a.dgate = o.dgate;
    a.lddgate = (int64_t)o.lddgate;
    float* const to[kSums] = {o.dgate, o.dpost_weight, o.dpost_bias, o.dnext_weight, o.dnext_bias};
    ProfScope prof(ctx, op, 32.0 * rows * cols,
                   4.0 * ((dy != nullptr) + 2 * (du != nullptr) + reads_f + (o.dx != nullptr) + (o.df != nullptr)) *
                       rows * cols);
    launch_backward(ctx, a, to, p.gate ? (int64_t)p.groups : 0, op);
  });
}

}  // extern "C"
