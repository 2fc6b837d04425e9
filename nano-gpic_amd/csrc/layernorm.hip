// Layer norm, forward and backward, of rows x (+ a), beside the root-mean-square norms of rows.hip:
//
//   forward   x_new = x + a (rounded to the type);  mu = mean(x_new);  rstd = 1 / sqrt(mean((x_new - mu)^2) + eps)
//             t = (x_new - mu) rstd;  h = t w + b, rounded once: to the inputs' type, or to e4m3 with the row's scale
//   backward  dt = dh w;  dx = rstd (dt - mean(dt) - t mean(dt t)) + dx_new;  dw = sum over rows of dh t;  db = sum of dh
//
// Everything between loads and stores is fp32. The deviations are taken from a first mean and their own mean is taken off again
// (mu = mu0 + mean(x - mu0)), so that a row far from zero loses no more than its inputs' own rounding to the first sum's.
// Each kernel reads its inputs once and writes its outputs once; memory bounds them, and one row alone the launch. The teams and
// what they hold are rows.hip's.
#include "gpic_rows.h"

namespace gpic {

// Two sums over a team (as team_sum): red has two words a wave.
template <int T>
__device__ __forceinline__ void team_sum2(float &a, float &b, float2 *red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    a += __shfl_xor(a, o, 64);
    b += __shfl_xor(b, o, 64);
  }
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = float2{a, b};
    lds_barrier();
    a = red[0].x, b = red[0].y;
#pragma unroll
    for (int i = 1; i < T / 64; i++) a += red[i].x, b += red[i].y;
  }
}

struct LayerNormArgs {
  const void *x, *a, *w, *b;
  void *xn, *h;
  float *mean, *rstd, *s;
  uint8_t *q;
  int64_t rows, ldx, lda;
  int C, wt, bt, chunk;   // wt, bt: w's and b's types; chunk: rows of a team
  float eps;
};

// Bound by memory: x_new and the bytes of [32768 x 1024] with residual, 7 bytes an element, 46 us, 5.1 TB/s; [8191 x 4096] fp32 52
// us, 5.1 TB/s; one row 3.9 us (the sum, the deviations' and the maximum one after another).
// A team takes `chunk` rows one after another; the row after the current one is requested before the current one's sums, and w
// and b are kept in registers. kQ: h goes to q, s (and to h only if it is asked for).
template <int T, int kV, int E, bool kRes, bool kQ>
__global__ __launch_bounds__(kWG<T>) void layer_norm_kernel(LayerNormArgs p) {
  __shared__ float red_s[T > 64 ? T / 64 : 1];
  __shared__ float2 red_d[T > 64 ? T / 64 : 1];
  __shared__ uint32_t red_m[T > 64 ? T / 64 : 1];
  const int t = threadIdx.x % T, nv = p.C / 8;
  int64_t row = team_row<T>() * p.chunk;
  const int64_t end = min(row + p.chunk, p.rows);
  if (row >= end) return;
  Raw8<E> X[kV], A[kV];
  float W[kV][8], Bv[kV][8];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      X[j] = A[j] = zero8<E>();
      if (v < nv) {
        X[j] = raw8<E>(p.x, r * p.ldx + 8 * v);
        if (kRes) A[j] = raw8<E>(p.a, r * p.lda + 8 * v);
      }
    }
  };
  fetch(row);
#pragma unroll
  for (int j = 0; j < kV; j++) {
    const int v = t + T * j;
#pragma unroll
    for (int e = 0; e < 8; e++) W[j][e] = 1.0f, Bv[j][e] = 0.0f;
    if (v < nv) {
      if (p.w) load8_as(p.w, p.wt, 8 * v, W[j]);
      if (p.b) load8_as(p.b, p.bt, 8 * v, Bv[j]);
    }
  }
  const float C = (float)p.C;
  for (; row < end; row++) {
    float D[kV][8];
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kV; j++) {
      values8<E>(X[j], D[j]);
      if (kRes) {
        float av[8];
        values8<E>(A[j], av);
#pragma unroll
        for (int e = 0; e < 8; e++) D[j][e] += av[e];
        const Raw8<E> n = round8<E>(D[j]);
        values8<E>(n, D[j]);
        const int v = t + T * j;
        if (v < nv) store8<E>(p.xn, row * p.C + 8 * v, n);
      }
#pragma unroll
      for (int e = 0; e < 8; e++) sum += D[j][e];   // (zeros past the row's end)
    }
    if (row + 1 < end) fetch(row + 1);
    const float mu0 = __fdiv_rn(team_sum<T>(sum, red_s), C);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < kV; j++)
      if (t + T * j < nv) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float d = D[j][e] - mu0;
          D[j][e] = d;
          s1 += d;
          s2 = __builtin_fmaf(d, d, s2);
        }
      }
    team_sum2<T>(s1, s2, red_d);
    const float m1 = __fdiv_rn(s1, C);
    const float var = fmaxf(__builtin_fmaf(-m1, m1, __fdiv_rn(s2, C)), 0.0f);
    // (a NaN in the row: fmaxf drops the variance's, t = (x - mu) rstd keeps the deviations')
    const float rstd = __fdiv_rn(1.0f, __builtin_sqrtf(var + p.eps));
    const float off = -m1 * rstd;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      if (v < nv) {
#pragma unroll
        for (int e = 0; e < 8; e++) D[j][e] = __builtin_fmaf(__builtin_fmaf(D[j][e], rstd, off), W[j][e], Bv[j][e]);
        if (kQ) m = absmax8(D[j], m);
        if (!kQ || p.h) store8<E>(p.h, row * p.C + 8 * v, round8<E>(D[j]));
      }
    }
    if constexpr (kQ) {
      float scale, dequant;
      scales_from_amax(team_max<T>(m, red_m), scale, dequant);
#pragma unroll
      for (int j = 0; j < kV; j++) {
        const int v = t + T * j;
        if (v < nv) *reinterpret_cast<u32x2 *>(p.q + row * p.C + 8 * v) = cast8(D[j], scale);
      }
      if (t == 0) p.s[row] = dequant;
    }
    if (t == 0 && p.mean) p.mean[row] = mu0 + m1, p.rstd[row] = rstd;
  }
}

struct LayerNormBwdArgs {
  const void *dh, *dxn, *xs, *w;
  const float *mean, *rstd;
  void *dx;
  float *P;   // [2, gridDim.x, C] partial sums of dw, then db
  int64_t rows;
  int C, wt;
};

// Bound by memory: [8191 x 4096] fp32 79 us, 5.3 TB/s, and 7 us for the column sums; [6528 x 1024] bf16 with dx_new 15.6 and 3.8.
// The rows of a workgroup in their order, each thread's columns' dw and db in registers; a workgroup's teams are added in their
// order, then the workgroups in theirs (column_sums_kernel): the same sums in every run.
template <int T, int kV, int E>
__global__ __launch_bounds__(kWG<T>) void layer_norm_bwd_kernel(LayerNormBwdArgs p) {
  constexpr int R = kWG<T> / T;
  __shared__ float2 red[2][T > 64 ? T / 64 : 1];
  __shared__ __attribute__((aligned(16))) float part[R > 1 ? T * kV * 8 : 4];
  const int t = threadIdx.x % T, nv = p.C / 8;
  float W[kV][8], DW[kV][8], DB[kV][8];
#pragma unroll
  for (int j = 0; j < kV; j++) {
    const int v = t + T * j;
#pragma unroll
    for (int e = 0; e < 8; e++) W[j][e] = 1.0f, DW[j][e] = DB[j][e] = 0.0f;
    if (v < nv && p.w) load8_as(p.w, p.wt, 8 * v, W[j]);
  }
  const float C = (float)p.C;
  int turn = 0;
  for (int64_t row = team_row<T>(); row < p.rows; row += team_step<T>(), turn ^= 1) {
    Raw8<E> Y[kV], X[kV], N[kV];
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      Y[j] = X[j] = N[j] = zero8<E>();
      if (v < nv) {
        Y[j] = raw8<E>(p.dh, row * p.C + 8 * v);
        X[j] = raw8<E>(p.xs, row * p.C + 8 * v);
        if (p.dxn) N[j] = raw8<E>(p.dxn, row * p.C + 8 * v);
      }
    }
    const float mu = p.mean[row], rs = p.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < kV; j++)
      if (t + T * j < nv) {
        float d[8], x[8];
        values8<E>(Y[j], d);
        values8<E>(X[j], x);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float tt = (x[e] - mu) * rs, dt = d[e] * W[j][e];
          s1 += dt;
          s2 = __builtin_fmaf(dt, tt, s2);
          DW[j][e] = __builtin_fmaf(d[e], tt, DW[j][e]);
          DB[j][e] += d[e];
        }
      }
    team_sum2<T>(s1, s2, red[turn]);
    const float m1 = __fdiv_rn(s1, C), m2 = __fdiv_rn(s2, C);
#pragma unroll
    for (int j = 0; j < kV; j++) {
      const int v = t + T * j;
      if (v < nv) {
        float d[8], x[8], n[8];
        values8<E>(Y[j], d);
        values8<E>(X[j], x);
        values8<E>(N[j], n);
#pragma unroll
        for (int e = 0; e < 8; e++)
          n[e] = __builtin_fmaf(rs, __builtin_fmaf(-((x[e] - mu) * rs), m2, __builtin_fmaf(d[e], W[j][e], -m1)), n[e]);
        store8<E>(p.dx, row * p.C + 8 * v, round8<E>(n));
      }
    }
  }
  store_column_partials<T, kV>(DW, part, p.P, p.C);
  __syncthreads();
  store_column_partials<T, kV>(DB, part, p.P + (int64_t)gridDim.x * p.C, p.C);
}

__device__ __forceinline__ void store_vec4(void *p, int dtype, int64_t c, const float4 &v) {
  if (dtype == GPIC_DTYPE_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(p) + c) = v;
  } else if (dtype == GPIC_DTYPE_BF16) {
    *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p) + c) = u32x2{pack_bf16(v.x, v.y), pack_bf16(v.z, v.w)};
  } else {
    typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
    *reinterpret_cast<f16x4_t *>(static_cast<_Float16 *>(p) + c) =
        f16x4_t{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
  }
}

// dw (blockIdx.y 0) and db (1): the sums over the workgroups of P [2, G, C], as column_sum_kernel's.
__global__ __launch_bounds__(256) void column_sums_kernel(const float *__restrict__ P, int G, int C, void *dw, int dwt, void *db,
                                                          int dbt) {
  __shared__ float4 red[64][4];
  float4 a;
  void *out = blockIdx.y ? db : dw;
  const int c = blockIdx.x * 16 + 4 * (threadIdx.x & 3);
  if (!column_sum16(P + (int64_t)blockIdx.y * G * C, G, C, red, a) || !out) return;
  store_vec4(out, blockIdx.y ? dbt : dwt, c, a);
}

// ------------------------------------------------------------------------------------------- host side

static bool dtype3_ok(int d) { return d == GPIC_DTYPE_BF16 || d == GPIC_DTYPE_F32 || d == GPIC_DTYPE_F16; }

// f(E) with the type as a constant
template <class F>
static void with_dtype(int dtype, F f) {
  if (dtype == GPIC_DTYPE_BF16) f(std::integral_constant<int, 0>());
  else if (dtype == GPIC_DTYPE_F32) f(std::integral_constant<int, 1>());
  else f(std::integral_constant<int, 2>());
}

// Workgroups of the backward: each leaves a partial row of dw and of db.
static int layer_norm_bwd_blocks(int64_t rows, int64_t C) {
  const int teams = C <= 1024 ? 4 : 1;
  return (int)std::min<int64_t>((rows + teams - 1) / teams, 512);
}

}  // namespace gpic

using namespace gpic;

extern "C" {

int gpic_fp8_layer_norm(const void *x, int dtype, int64_t ldx, const void *a, int64_t lda, const void *w, int w_dtype,
                        const void *b, int b_dtype, int64_t rows, int64_t C, float eps, void *xn, void *h, float *mean,
                        float *rstd, uint8_t *q, float *s, void *stream) {
  status_scope();
  if (rows < 0 || C <= 0 || !mean != !rstd || !q != !s) return GPIC_EINVAL;
  if (rows > 0 && (!x || (a && !xn) || (!h && !q))) return GPIC_EINVAL;
  if (!dtype3_ok(dtype) || (w && !dtype3_ok(w_dtype)) || (b && !dtype3_ok(b_dtype)) || (q && dtype != GPIC_DTYPE_BF16))
    return GPIC_EDTYPE;
  if (C % 8 || C > kMaxNormC || rows >= (int64_t(1) << 31) || ldx % 8 || ldx < C || (a && (lda % 8 || lda < C)))
    return GPIC_ESHAPE;
  if (!aligned16(x) || !aligned16(a) || !aligned16(w) || !aligned16(b) || !aligned16(xn) || !aligned16(h) || !aligned16(q))
    return GPIC_EALIGN;
  if (rows == 0) return GPIC_OK;
  LayerNormArgs p{x, a, w, b, xn, h, mean, rstd, s, q, rows, ldx, lda, (int)C, w_dtype, b_dtype, 1, eps};
  const hipStream_t st = (hipStream_t)stream;
  with_team(C, [&](auto T, auto V) {
    constexpr int t = decltype(T)::value, v = decltype(V)::value;
    if constexpr (t * v * 8 <= kMaxNormC) {
      constexpr int teams = kWG<t> / t;
      p.chunk = norm_chunk(rows, teams, a ? 1 : 2);
      const unsigned g = (unsigned)((rows + (int64_t)p.chunk * teams - 1) / ((int64_t)p.chunk * teams));
      with_dtype(dtype, [&](auto E) {
        constexpr int e = decltype(E)::value;
        auto *k = a ? layer_norm_kernel<t, v, e, true, false> : layer_norm_kernel<t, v, e, false, false>;
        if constexpr (e == 0)
          if (q) k = a ? layer_norm_kernel<t, v, 0, true, true> : layer_norm_kernel<t, v, 0, false, true>;
        k<<<g, kWG<t>, 0, st>>>(p);
      });
    }
  });
  return (int)hipGetLastError();
}

size_t gpic_fp8_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t C) {
  if (rows <= 0 || C <= 0) return 0;
  return (size_t)layer_norm_bwd_blocks(rows, C) * C * 2 * sizeof(float);
}

int gpic_fp8_layer_norm_bwd(const void *dh, const void *dxn, const void *xs, int dtype, const void *w, int w_dtype,
                            const float *mean, const float *rstd, int64_t rows, int64_t C, void *dx, void *dw, int dw_dtype,
                            void *db, int db_dtype, void *ws, size_t ws_bytes, void *stream) {
  status_scope();
  if (rows < 0 || C <= 0 || (rows > 0 && (!dh || !xs || !mean || !rstd || !dx))) return GPIC_EINVAL;
  if (!dtype3_ok(dtype) || (w && !dtype3_ok(w_dtype)) || (dw && !dtype3_ok(dw_dtype)) || (db && !dtype3_ok(db_dtype)))
    return GPIC_EDTYPE;
  if (C % 8 || C > kMaxNormC || rows >= (int64_t(1) << 31)) return GPIC_ESHAPE;
  if (!aligned16(dh) || !aligned16(dxn) || !aligned16(xs) || !aligned16(w) || !aligned16(dx) || !aligned16(dw) ||
      !aligned16(db) || !aligned16(ws))
    return GPIC_EALIGN;
  if (ws_bytes < gpic_fp8_layer_norm_bwd_workspace_bytes(rows, C) || (rows > 0 && !ws)) return GPIC_EWORKSPACE;
  const hipStream_t st = (hipStream_t)stream;
  const int g = rows ? layer_norm_bwd_blocks(rows, C) : 0;
  const LayerNormBwdArgs p{dh, dxn, xs, w, mean, rstd, dx, static_cast<float *>(ws), rows, (int)C, w_dtype};
  if (g > 0)
    with_short_team(C, [&](auto T, auto V) {
      constexpr int t = decltype(T)::value, v = decltype(V)::value;
      if constexpr (t * v * 8 <= kMaxNormC)
        with_dtype(dtype, [&](auto E) { layer_norm_bwd_kernel<t, v, decltype(E)::value><<<g, kWG<t>, 0, st>>>(p); });
    });
  if (dw || db)
    column_sums_kernel<<<dim3((unsigned)((C + 15) / 16), db ? 2 : 1), 256, 0, st>>>(p.P, g, (int)C, dw, dw_dtype, db, db_dtype);
  return (int)hipGetLastError();
}

}  // extern "C"
