// The row-scaled producers: operators whose e4m3 output carries one scale per row (token, or output channel of a weight)
// instead of one per tensor. A row's maximum is known to the threads that hold the row, so there is no fold over the chip
// and no second pass: each kernel reads its inputs once and writes its outputs once, and one row alone is one short launch.
//
//   row cast      a = max(max|h|, 1e-12), s = RN(a / 448), q = e4m3(min(max(RN(h RN(448 / a)), -448), 448))
//   norm          x_new = bf16(x + gate a); rstd = 1 / sqrt(mean(x_new^2) + eps);
//                 h = (w (x_new rstd)) (1 + scale) + shift, cast by row
//   its backward  t = x_new rstd, dt = dh w, dx = bf16(rstd (dt - t mean(dt t)) + dx_new), dw = sum over rows of dh t
//   activation's backward  dz = dy act'(z) as bf16, and (dz sw) cast by row
//
// h and dz sw are fp32 until the one rounding to e4m3: the tensorwise norm sites (norm.hip) round n and h to bf16 because the
// reference's ops hand them on in bf16; here nothing between the row's statistics and its bytes is held in memory.
// A NaN anywhere in a row makes the row's maximum, and so its scale, NaN (the maximum of the magnitudes' bit patterns: a
// NaN's is above infinity's): a product of the row is then NaN. The tensorwise casts ignore NaN, as the reference's.
// An infinity makes the scale infinite.
//
// A team of T threads holds a row, 8 elements (16 bytes of bf16) a thread and step: a wave for rows of up to 2048, four waves
// up to 8192, sixteen above. What bounds them is memory; each vector of a row is requested before any is used.
#include "gpic_act.h"
#include "gpic_rows.h"

namespace gpic {

struct CastArgs {
  const void *x;   // [rows, C] bf16, or fp32 (f32)
  uint8_t *q;
  float *s;
  int64_t rows, ld;
  int f32;
};

// The row cast of p's rows first, first + step, ... by one team. red: two sets of T / 64 words, in turn.
template <int T, int kV>
__device__ __forceinline__ void cast_team(const CastArgs &p, bool f32, int C, int64_t first, int64_t step,
                                          uint32_t (&red)[2][T > 64 ? T / 64 : 1]) {
  const int t = threadIdx.x % T, nv = C / 8;
  int turn = 0;
  for (int64_t row = first; row < p.rows; row += step, turn ^= 1) {
    float H[kV][8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      if (v < nv) load8(p.x, f32, row * p.ld + 8 * v, H[j]);
    }
#pragma unroll
    for (int j = 0; j < kV; j++)
      if (t + T * j < nv) m = absmax8(H[j], m);
    float scale, dequant;
    scales_from_amax(team_max<T>(m, red[turn]), scale, dequant);
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      if (v < nv) *reinterpret_cast<u32x2 *>(p.q + row * C + 8 * v) = cast8(H[j], scale);
    }
    if (t == 0) p.s[row] = dequant;
  }
}

// The workgroup's index among `blocks` from blockIdx.x - first, as a team's first row and the rows between two of its rows.
template <int T>
__device__ __forceinline__ int64_t team_row_in(int first) {
  constexpr int R = kWG<T> / T;
  return ((int64_t)blockIdx.x - first) * R + (R == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / T));
}

// Bound by memory: [32768 x 4096] bf16 71 us, 5.7 TB/s of the 3 bytes an element; [8192 x 1024] fp32 8.2 us, 5.1 TB/s (a copy of
// 1 GiB: 5.1).
// One matrix by the first `blocks` workgroups, another (a linear's input and its weight: rows of one length) by the rest.
// (kKind: one bf16 matrix, one fp32, or two: instances of their own, as for the norm, whose plain one the test and the second
// set of arguments cost 6%)
enum { kOneBF16, kOneF32, kTwo };
template <int T, int kV, int kKind>
__global__ __launch_bounds__(kWG<T>) void tcast_rows_kernel(CastArgs a, CastArgs b, int C, int blocks) {
  __shared__ uint32_t red[2][T > 64 ? T / 64 : 1];
  constexpr int R = kWG<T> / T;
  if constexpr (kKind != kTwo) {
    cast_team<T, kV>(a, kKind == kOneF32, C, team_row<T>(), team_step<T>(), red);
  } else {
    const bool first = (int)blockIdx.x < blocks;
    const CastArgs p = first ? a : b;
    cast_team<T, kV>(p, p.f32, C, team_row_in<T>(first ? 0 : blocks),
                     (int64_t)(first ? blocks : (int)gridDim.x - blocks) * R, red);
  }
}

struct NormRowsArgs {
  const uint16_t *x, *a, *gate, *shift, *scale;
  const void *w;
  uint16_t *xn, *h;
  float *rstd, *s;
  uint8_t *q;
  int64_t rows, ntok, ldx, lda, sg, ssh, ssc;
  int C, w32, chunk;   // chunk: rows of a team
  float eps;
};

// Bound by memory, one row alone by the launch: x_new and the bytes of [32768 x 1024] with residual, gate, shift and scale, 7 bytes
// an element, 46 us, 5.1 TB/s; one row 2.6 us.
// A team takes `chunk` rows one after another: the row after the current one is requested before the current one's sums, and
// w, and gate, shift and scale while the batch entry stays the same, are kept in registers.
template <int T, int kV, bool kRes, bool kMod, bool kWeight>
__global__ __launch_bounds__(kWG<T>) void rmsnorm_rows_kernel(NormRowsArgs p, CastArgs weight, int blocks) {
  __shared__ float red_s[T > 64 ? T / 64 : 1];
  __shared__ uint32_t red_w[2][T > 64 ? T / 64 : 1];
  uint32_t (&red_m)[T > 64 ? T / 64 : 1] = red_w[0];
  if (kWeight && (int)blockIdx.x >= blocks) {   // (the weight of the linear that reads the norm: its cast, beside it)
    cast_team<T, kV>(weight, weight.f32, p.C, team_row_in<T>(blocks), (int64_t)((int)gridDim.x - blocks) * (kWG<T> / T), red_w);
    return;
  }
  const int t = threadIdx.x % T, nv = p.C / 8;
  int64_t row = team_row<T>() * p.chunk;
  const int64_t end = min(row + p.chunk, p.rows);
  if (row >= end) return;
  u32x4 X[kV], A[kV], G[kV], SH[kV], SC[kV];
  float W[kV][8];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      X[j] = A[j] = u32x4{0u, 0u, 0u, 0u};
      if (v < nv) {
        X[j] = ld16(p.x + r * p.ldx + 8 * v);
        if (kRes) A[j] = ld16(p.a + r * p.lda + 8 * v);
      }
    }
  };
  fetch(row);
#pragma unroll
  for (int j = 0; j < kV; j++)
    if (t + T * j < nv) load8(p.w, p.w32, 8 * (t + T * j), W[j]);
  const bool gated = kRes && p.gate;
  int64_t batch_end = row;   // the first row of the next batch entry
  for (; row < end; row++) {
    if ((kMod || gated) && row == batch_end) {
      const uint32_t b = (uint32_t)row / (uint32_t)p.ntok;
      batch_end = (int64_t)(b + 1) * p.ntok;
#pragma unroll
      for (int j = 0; j < kV; j++) {
        const int v = t + T * j;
        if (v < nv) {
          if (gated) G[j] = ld16(p.gate + b * p.sg + 8 * v);
          if (kMod) {
            SH[j] = ld16(p.shift + b * p.ssh + 8 * v);
            SC[j] = ld16(p.scale + b * p.ssc + 8 * v);
          }
        }
      }
    }
    u32x4 V[kV];   // x_new
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < kV; j++) {
      float x[8];
      unpack8(X[j], x);
      V[j] = X[j];
      if (kRes) {
        float av[8];
        unpack8(A[j], av);
        if (gated) {
          float g[8];
          unpack8(G[j], g);
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf(g[e], av[e], x[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] += av[e];
        }
        V[j] = pack8(x);
        unpack8(V[j], x);
      }
      if (t + T * j < nv) {   // (past the row's end: zeros times whatever G holds there)
#pragma unroll
        for (int e = 0; e < 8; e++) ss = __builtin_fmaf(x[e], x[e], ss);
      }
    }
    if (row + 1 < end) fetch(row + 1);
    if (kRes) {
#pragma unroll
      for (int j = 0; j < kV; j++) {
        const int v = t + T * j;
        if (v < nv) *reinterpret_cast<u32x4 *>(p.xn + row * p.C + 8 * v) = V[j];
      }
    }
    ss = team_sum<T>(ss, red_s);
    const float rstd = __fdiv_rn(1.0f, __builtin_sqrtf(__fdiv_rn(ss, (float)p.C) + p.eps));
    float H[kV][8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      if (v < nv) {
        float x[8];
        unpack8(V[j], x);
#pragma unroll
        for (int e = 0; e < 8; e++) H[j][e] = W[j][e] * (x[e] * rstd);
        if (kMod) {
          float sh[8], sc[8];
          unpack8(SH[j], sh);
          unpack8(SC[j], sc);
#pragma unroll
          for (int e = 0; e < 8; e++) H[j][e] = __builtin_fmaf(H[j][e], 1.0f + sc[e], sh[e]);
        }
        m = absmax8(H[j], m);
        if (p.h) *reinterpret_cast<u32x4 *>(p.h + row * p.C + 8 * v) = pack8(H[j]);
      }
    }
    float scale, dequant;
    scales_from_amax(team_max<T>(m, red_m), scale, dequant);
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      if (v < nv) *reinterpret_cast<u32x2 *>(p.q + row * p.C + 8 * v) = cast8(H[j], scale);
    }
    if (t == 0) {
      p.s[row] = dequant;
      p.rstd[row] = rstd;
    }
  }
}

// A 64 x 64 tile of qt[c, r] = q[r, c] by 256 threads, 16 bytes each in and out; columns rows .. ldt - 1 of qt zero. on: whether
// there is a tile (uniform over the 256 threads; all of a workgroup's meet at the barrier).
struct TransposeTile {
  uint8_t b[64][80];   // (80: 16-byte rows on different banks)
};
__device__ __forceinline__ void transpose_tile(const uint8_t *q, int64_t rows, int64_t cols, uint8_t *qt, int64_t ldt,
                                               int64_t tile_r, int64_t tile_c, bool on, TransposeTile &tile) {
  const int64_t r0 = tile_r * 64, c0 = tile_c * 64;
  const int i = (threadIdx.x & 255) >> 2, k = 16 * (threadIdx.x & 3);
  u32x4 v{0u, 0u, 0u, 0u};
  if (on && r0 + i < rows && c0 + k < cols) v = ld16(q + (r0 + i) * cols + c0 + k);
  *reinterpret_cast<u32x4 *>(&tile.b[i][k]) = v;
  __syncthreads();
  if (on && c0 + i < cols && r0 + k < ldt) {
    uint32_t o[4];
#pragma unroll
    for (int w = 0; w < 4; w++)
      o[w] = (uint32_t)tile.b[k + 4 * w][i] | (uint32_t)tile.b[k + 4 * w + 1][i] << 8 |
             (uint32_t)tile.b[k + 4 * w + 2][i] << 16 | (uint32_t)tile.b[k + 4 * w + 3][i] << 24;
    *reinterpret_cast<u32x4 *>(qt + (c0 + i) * ldt + r0 + k) = u32x4{o[0], o[1], o[2], o[3]};
  }
}

// Bound by memory: 7 bytes an element, [16384 x 7168] with db and the weight's transpose 166 us, 5.2 TB/s of what it moves; the
// derivative's arithmetic passes under the loads ([6592 x 4096] 39 us).
// The epilogue's backward, and beside it, in workgroups of their own, the transposed bytes of the weight that the dgrad reads
// (independent work: a launch less in the chain). kDb: each thread also sums its columns' dz, as rounded, over its rows, for
// column_sum_kernel: the same order in every run.
struct ActBwdArgs {
  const uint16_t *dy, *z;
  const float *sw;
  const uint8_t *wq;   // [N, K]: transposed by the workgroups past row_blocks
  uint8_t *wqt;        // [K, ldt]
  uint16_t *dz;
  uint8_t *q;
  float *s, *P;        // P: [row_blocks, N] partial sums (kDb)
  int64_t rows, lddy, ldz, K, ldt, tiles_c, tiles;
  int N, act, row_blocks;
};

template <int T, int kV, bool kDb>
__global__ __launch_bounds__(kWG<T>) void act_bwd_rows_kernel(ActBwdArgs p) {
  constexpr int R = kWG<T> / T;
  __shared__ uint32_t red_m[2][T > 64 ? T / 64 : 1];
  __shared__ TransposeTile tile[kWG<T> / 256];
  __shared__ __attribute__((aligned(16))) float part[kDb && R > 1 ? T * kV * 8 : 4];
  if ((int)blockIdx.x >= p.row_blocks) {
    const int sub = threadIdx.x >> 8;
    const int64_t i = (int64_t)((int)blockIdx.x - p.row_blocks) * (kWG<T> / 256) + sub;
    transpose_tile(p.wq, p.N, p.K, p.wqt, p.ldt, i / p.tiles_c, i % p.tiles_c, i < p.tiles, tile[sub]);
    return;
  }
  const int t = threadIdx.x % T, nv = p.N / 8;
  float D[kV][8];
#pragma unroll
  for (int j = 0; j < kV; j++)
#pragma unroll
    for (int e = 0; e < 8; e++) D[j][e] = 0.0f;
  u32x4 Y[kV], Z[kV];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      if (v < nv) {
        Y[j] = ld16(p.dy + r * p.lddy + 8 * v);
        if (p.act) Z[j] = ld16(p.z + r * p.ldz + 8 * v);
      }
    }
  };
  int64_t row = team_row<T>();
  const int64_t step = (int64_t)p.row_blocks * R;
  if (row < p.rows) fetch(row);
  for (int turn = 0; row < p.rows; row += step, turn ^= 1) {
    float H[kV][8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      if (v < nv) {
        float d[8], z[8];
        unpack8(Y[j], d);
        if (p.act) {
          unpack8(Z[j], z);
#pragma unroll
          for (int e = 0; e < 8; e++) d[e] *= act_bwd(z[e], p.act);
          Y[j] = pack8(d);
          *reinterpret_cast<u32x4 *>(p.dz + row * p.N + 8 * v) = Y[j];
        }
        if (kDb) {
          float r[8];
          unpack8(Y[j], r);
#pragma unroll
          for (int e = 0; e < 8; e++) D[j][e] += r[e];
        }
        float w[8];
        load8(p.sw, true, 8 * v, w);
#pragma unroll
        for (int e = 0; e < 8; e++) H[j][e] = d[e] * w[e];
        m = absmax8(H[j], m);
      }
    }
    if (row + step < p.rows) fetch(row + step);   // (the next row is under way during this one's maximum and stores)
    float scale, dequant;
    scales_from_amax(team_max<T>(m, red_m[turn]), scale, dequant);
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      if (v < nv) *reinterpret_cast<u32x2 *>(p.q + row * p.N + 8 * v) = cast8(H[j], scale);
    }
    if (t == 0) p.s[row] = dequant;
  }
  if constexpr (kDb) store_column_partials<T, kV>(D, part, p.P, p.N);
}

struct NormBwdRowsArgs {
  const uint16_t *dh, *dxn, *xs;
  const void *w;
  const float *rstd;
  uint16_t *dx;
  float *P;   // [gridDim.x, C] partial sums of dw
  int64_t rows;
  int C, w32;
};

// Bound by memory: 8 bytes an element with dx_new, [16381 x 4096] 96 us, 5.7 TB/s, and 5 us for the column sums; [6528 x 1024] 11
// and 4.
// The rows of a workgroup in their order, each thread's columns' dw in registers; a workgroup's teams are added in their
// order, then the workgroups in theirs (column_sum_kernel): the same sums in every run.
template <int T, int kV>
__global__ __launch_bounds__(kWG<T>) void rmsnorm_rows_bwd_kernel(NormBwdRowsArgs p) {
  constexpr int R = kWG<T> / T;
  __shared__ float red_s[2][T > 64 ? T / 64 : 1];
  __shared__ __attribute__((aligned(16))) float part[R > 1 ? T * kV * 8 : 4];
  const int t = threadIdx.x % T, nv = p.C / 8;
  float W[kV][8], D[kV][8];
#pragma unroll
  for (int j = 0; j < kV; j++) {
    const int v = t + T * j;
#pragma unroll
    for (int e = 0; e < 8; e++) W[j][e] = D[j][e] = 0.0f;
    if (v < nv) load8(p.w, p.w32, 8 * v, W[j]);
  }
  const float rC = 1.0f / (float)p.C;
  int turn = 0;
  for (int64_t row = team_row<T>(); row < p.rows; row += team_step<T>(), turn ^= 1) {
    u32x4 Y[kV], X[kV], N[kV];
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      Y[j] = X[j] = N[j] = u32x4{0u, 0u, 0u, 0u};
      if (v < nv) {
        Y[j] = ld16(p.dh + row * p.C + 8 * v);
        X[j] = ld16(p.xs + row * p.C + 8 * v);
        if (p.dxn) N[j] = ld16(p.dxn + row * p.C + 8 * v);
      }
    }
    const float rs = p.rstd[row];
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kV; j++) {
      float d[8], x[8];
      unpack8(Y[j], d);
      unpack8(X[j], x);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float tt = x[e] * rs;
        sum = __builtin_fmaf(d[e] * W[j][e], tt, sum);
        D[j][e] = __builtin_fmaf(d[e], tt, D[j][e]);
      }
    }
    const float mean = team_sum<T>(sum, red_s[turn]) * rC;
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      if (v < nv) {
        float d[8], x[8], n[8];
        unpack8(Y[j], d);
        unpack8(X[j], x);
        unpack8(N[j], n);
#pragma unroll
        for (int e = 0; e < 8; e++)
          n[e] = __builtin_fmaf(rs, __builtin_fmaf(-(x[e] * rs), mean, d[e] * W[j][e]), n[e]);
        *reinterpret_cast<u32x4 *>(p.dx + row * p.C + 8 * v) = pack8(n);
      }
    }
  }
  store_column_partials<T, kV>(D, part, p.P, p.C);
}

// out[c] = sum over g of P[g, c] (column_sum16)
__global__ __launch_bounds__(256) void column_sum_kernel(const float *__restrict__ P, int G, int C, void *__restrict__ out,
                                                         int out32) {
  __shared__ float4 red[64][4];
  float4 a;
  const int c = blockIdx.x * 16 + 4 * (threadIdx.x & 3);
  if (!column_sum16(P, G, C, red, a)) return;
  if (out32) *reinterpret_cast<float4 *>(static_cast<float *>(out) + c) = a;
  else
    *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(out) + c) = u32x2{pack_bf16(a.x, a.y), pack_bf16(a.z, a.w)};
}

// ------------------------------------------------------------------------------------------- host side

// Workgroups of the epilogue's backward: with db each leaves a partial row of it, so no more than fill the device. us, 256 / 512 /
// 768 / 1024: [6592 x 4096] 66 / 43.2 / 39.6 / 40.7, [32768 x 4096] 322 / 198 / 185 / 180, [16384 x 7168] (512 threads each)
// 191 / 165 / 196 / 172. Without db a workgroup a row: [32768 x 4096] 166, 2048 workgroups 189.
static int act_bwd_blocks(int64_t rows, int64_t N, bool db) {
  const int teams = N <= 1024 ? 4 : 1;
  return (int)std::min<int64_t>((rows + teams - 1) / teams, db ? N <= 4096 ? 768 : 512 : kMaxRowBlocks);
}

// Workgroups of the norm's backward: each leaves a partial row of dw. us, 256 / 512 / 1024: [6528 x 1024] 15.5 / 14.1 / 16.0,
// [16381 x 4096] 113 / 102 / 111, [4096 x 8192] 57 / 51 / 61.
static int norm_bwd_blocks(int64_t rows, int64_t C) {
  const int teams = C <= 2048 ? 4 : 1;
  return (int)std::min<int64_t>((rows + teams - 1) / teams, 512);
}

}  // namespace gpic

using namespace gpic;

extern "C" {

// A matrix to cast by rows: its status, and whether there is anything to do.
static int cast_ok(const void *x, int dtype, int64_t ldx, int64_t rows, int64_t cols, int64_t most, const uint8_t *q,
                   const float *s) {
  if (rows < 0 || cols <= 0 || (rows > 0 && (!x || !q || !s))) return GPIC_EINVAL;
  if (!dtype_ok(dtype)) return GPIC_EDTYPE;
  if (cols % 8 || cols > most || ldx % 8 || ldx < cols) return GPIC_ESHAPE;
  if (!aligned16(x) || !aligned16(q)) return GPIC_EALIGN;
  return GPIC_OK;
}

int gpic_fp8_tcast_rows(const void *x, int dtype, int64_t ldx, int64_t rows, int64_t cols, uint8_t *q, float *s,
                        const void *x2, int dtype2, int64_t ldx2, int64_t rows2, uint8_t *q2, float *s2, void *stream) {
  status_scope();
  int e = cast_ok(x, dtype, ldx, rows, cols, kMaxRowC, q, s);
  if (e == GPIC_OK && x2) e = cast_ok(x2, dtype2, ldx2, rows2, cols, kMaxRowC, q2, s2);
  if (e != GPIC_OK) return e;
  if (!x2) rows2 = 0;
  if (rows + rows2 == 0) return GPIC_OK;
  const CastArgs a{x, q, s, rows, ldx, dtype == GPIC_DTYPE_F32}, b{x2, q2, s2, rows2, ldx2, dtype2 == GPIC_DTYPE_F32};
  with_team(cols, [&](auto T, auto V) {
    constexpr int t = decltype(T)::value, v = decltype(V)::value;
    const unsigned ga = row_blocks(rows, kWG<t> / t), gb = row_blocks(rows2, kWG<t> / t);
    auto *k = x2 ? tcast_rows_kernel<t, v, kTwo> : a.f32 ? tcast_rows_kernel<t, v, kOneF32> : tcast_rows_kernel<t, v, kOneBF16>;
    k<<<ga + gb, kWG<t>, 0, (hipStream_t)stream>>>(a, b, (int)cols, (int)ga);
  });
  return (int)hipGetLastError();
}

int gpic_fp8_rmsnorm_rows(const uint16_t *x, int64_t ldx, const uint16_t *a, int64_t lda, const uint16_t *gate, int64_t sg,
                          const void *w, int w_dtype, const uint16_t *shift, int64_t ssh, const uint16_t *scale,
                          int64_t ssc, int64_t rows, int64_t ntok, int64_t C, float eps, uint16_t *xn, uint16_t *h,
                          float *rstd, uint8_t *q, float *s, const void *wt, int wt_dtype, int64_t N, uint8_t *wq, float *sw,
                          void *stream) {
  status_scope();
  if (rows < 0 || C <= 0 || ntok <= 0 || !shift != !scale) return GPIC_EINVAL;
  if (rows > 0 && (!x || !w || !rstd || !q || !s || (a && !xn) || (gate && !a))) return GPIC_EINVAL;   // (no rows: null)
  if (!dtype_ok(w_dtype)) return GPIC_EDTYPE;
  if (C % 8 || C > kMaxNormC || rows >= (int64_t(1) << 31) || rows % ntok || ldx % 8 || ldx < C || (a && (lda % 8 || lda < C)) ||
      (gate && (sg % 8 || sg < C)) || (shift && (ssh % 8 || ssh < C || ssc % 8 || ssc < C)))
    return GPIC_ESHAPE;
  if (!aligned16(x) || !aligned16(a) || !aligned16(gate) || !aligned16(w) || !aligned16(shift) || !aligned16(scale) ||
      !aligned16(xn) || !aligned16(h) || !aligned16(q))
    return GPIC_EALIGN;
  if (wt) {
    const int e = cast_ok(wt, wt_dtype, C, N, C, kMaxNormC, wq, sw);
    if (e != GPIC_OK) return e;
  } else {
    N = 0;
  }
  if (rows + N == 0) return GPIC_OK;
  const CastArgs weight{wt, wq, sw, N, C, wt_dtype == GPIC_DTYPE_F32};
  const NormRowsArgs p{x, a, gate, shift, scale, w, xn, h, rstd, s, q, rows, ntok, ldx, lda, sg, ssh, ssc,
                       (int)C, w_dtype == GPIC_DTYPE_F32, 1, eps};
  const hipStream_t st = (hipStream_t)stream;
  with_team(C, [&](auto T, auto V) {
    constexpr int t = decltype(T)::value, v = decltype(V)::value;
    if constexpr (t * v * 8 <= kMaxNormC) {
      NormRowsArgs q = p;
      q.chunk = norm_chunk(rows, kWG<t> / t, a ? (gate || shift ? 2 : 1) : shift ? 4 : 2);
      const unsigned g = (unsigned)((rows + (int64_t)q.chunk * (kWG<t> / t) - 1) / ((int64_t)q.chunk * (kWG<t> / t)));
      auto pick = [&](auto two) {
        constexpr bool w = decltype(two)::value;
        return a ? (shift ? rmsnorm_rows_kernel<t, v, true, true, w> : rmsnorm_rows_kernel<t, v, true, false, w>)
                 : (shift ? rmsnorm_rows_kernel<t, v, false, true, w> : rmsnorm_rows_kernel<t, v, false, false, w>);
      };
      auto *k = wt ? pick(std::true_type()) : pick(std::false_type());
      k<<<g + row_blocks(N, kWG<t> / t), kWG<t>, 0, st>>>(q, weight, (int)g);
    }
  });
  return (int)hipGetLastError();
}

size_t gpic_fp8_rmsnorm_rows_bwd_workspace_bytes(int64_t rows, int64_t C) {
  if (rows <= 0 || C <= 0) return 0;
  return (size_t)norm_bwd_blocks(rows, C) * C * sizeof(float);
}

int gpic_fp8_rmsnorm_rows_bwd(const uint16_t *dh, const uint16_t *dxn, const uint16_t *xs, const void *w, int w_dtype,
                              const float *rstd, int64_t rows, int64_t C, uint16_t *dx, void *dw, int dw_dtype, void *ws,
                              size_t ws_bytes, void *stream) {
  status_scope();
  if (rows < 0 || C <= 0 || !dw || !w || (rows > 0 && (!dh || !xs || !rstd || !dx))) return GPIC_EINVAL;
  if (!dtype_ok(w_dtype) || !dtype_ok(dw_dtype)) return GPIC_EDTYPE;
  if (C % 8 || C > kMaxNormC) return GPIC_ESHAPE;
  if (!aligned16(dh) || !aligned16(dxn) || !aligned16(xs) || !aligned16(w) || !aligned16(dx) || !aligned16(dw) ||
      !aligned16(ws))
    return GPIC_EALIGN;
  if (ws_bytes < gpic_fp8_rmsnorm_rows_bwd_workspace_bytes(rows, C) || (rows > 0 && !ws)) return GPIC_EWORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  const int g = rows ? norm_bwd_blocks(rows, C) : 0;
  const NormBwdRowsArgs p{dh, dxn, xs, w, rstd, dx, static_cast<float *>(ws), rows, (int)C, w_dtype == GPIC_DTYPE_F32};
  if (g > 0)
    with_team(C, [&](auto T, auto V) {
      constexpr int t = decltype(T)::value, v = decltype(V)::value;
      if constexpr (t * v * 8 <= kMaxNormC) rmsnorm_rows_bwd_kernel<t, v><<<g, kWG<t>, 0, st>>>(p);
    });
  column_sum_kernel<<<(unsigned)((C + 15) / 16), 256, 0, st>>>(static_cast<const float *>(ws), g, (int)C, dw,
                                                               dw_dtype == GPIC_DTYPE_F32);
  return (int)hipGetLastError();
}

size_t gpic_fp8_act_bwd_rows_workspace_bytes(int64_t rows, int64_t N) {
  if (rows <= 0 || N <= 0) return 0;
  return (size_t)act_bwd_blocks(rows, N, true) * N * sizeof(float);
}

int gpic_fp8_act_bwd_rows(const uint16_t *dy, int64_t lddy, const uint16_t *z, int64_t ldz, int act, const float *sw,
                          int64_t rows, int64_t N, uint16_t *dz, uint8_t *q, float *s, const uint8_t *wq, int64_t K,
                          uint8_t *wqt, int64_t ldt, void *db, int db_dtype, void *ws, size_t ws_bytes, void *stream) {
  status_scope();
  if (rows < 0 || N <= 0 || act < GPIC_ACT_NONE || act > GPIC_ACT_GELU_TANH || !wq != !wqt || (wq && K < 0)) return GPIC_EINVAL;
  if (rows > 0 && (!dy || !sw || !q || !s || (act && (!z || !dz)))) return GPIC_EINVAL;
  if (db && !dtype_ok(db_dtype)) return GPIC_EDTYPE;
  if (N % 8 || N > kMaxRowC || lddy % 8 || lddy < N || (act && (ldz % 8 || ldz < N))) return GPIC_ESHAPE;
  if (wq && (K % 16 || ldt % 16 || ldt < N)) return GPIC_ESHAPE;
  if (!aligned16(dy) || !aligned16(sw) || !aligned16(q) || (act && (!aligned16(z) || !aligned16(dz))) || !aligned16(wq) ||
      !aligned16(wqt) || !aligned16(db) || !aligned16(ws))
    return GPIC_EALIGN;
  if (db && (ws_bytes < gpic_fp8_act_bwd_rows_workspace_bytes(rows, N) || (rows > 0 && !ws))) return GPIC_EWORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  const int64_t tc = wq ? (K + 63) / 64 : 1, tiles = wq ? (ldt + 63) / 64 * tc : 0;
  if (tiles >= (int64_t(1) << 23)) return GPIC_ESHAPE;   // (a launch's threads are counted in 32 bits)
  const int g = rows ? act_bwd_blocks(rows, N, db != nullptr) : 0;
  if (g == 0 && tiles == 0 && !db) return GPIC_OK;
  const ActBwdArgs p{dy, z, sw, wq, wqt, dz, q, s, static_cast<float *>(ws), rows, lddy, ldz, K, ldt, tc, tiles,
                     (int)N, act, g};
  if (g > 0 || tiles > 0)
    with_short_team(N, [&](auto T, auto V) {
      constexpr int t = decltype(T)::value, v = decltype(V)::value, sub = kWG<t> / 256;
      auto *k = db ? act_bwd_rows_kernel<t, v, true> : act_bwd_rows_kernel<t, v, false>;
      k<<<(unsigned)(g + (tiles + sub - 1) / sub), kWG<t>, 0, st>>>(p);
    });
  if (db)
    column_sum_kernel<<<(unsigned)((N + 15) / 16), 256, 0, st>>>(static_cast<const float *>(ws), g, (int)N, db,
                                                                 db_dtype == GPIC_DTYPE_F32);
  return (int)hipGetLastError();
}

}  // extern "C"
