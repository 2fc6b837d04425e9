// Low-rank adapters of many requests beside a shared projection:
//
//   out[m] = y[m] + s_i (x[m] A_i^T) B_i^T, i = ids[m / per];  rows whose id is none of 0 .. n - 1: out[m] = y[m]
//   x [M, K], A [n, R, K], B [n, N, R], y (the shared projection's output), out [M, N], bf16 or fp16; s [n] fp32
//
// Two launches: t = x A_i^T (fp32, [splits, M, R]: parts of K by different workgroups), then the product with B_i added to y and
// rounded once. Both are bound by memory: x, y, out and the adapters in use once, since R is far below the matrix instructions'
// balance; few rows by the launches and the adapters' bytes.
// A tile of rows may hold rows of any adapters, in any order: it is passed over once for each adapter that occurs in it, all of its
// rows multiplied and those of the pass kept, so what an adapter holds reaches no row but its own. Passes of one tile are
// independent: few rows spread them over workgroups of their own.
// t stays exact to 2^-16 and better: the second product reads it as the sum of two 16-bit numbers, its rounding and what the
// rounding left, beside each other on the reduction, which costs little for a rank this small.
#include <algorithm>
#include <type_traits>

#include "gpic_device.h"
#include "gpic_launch.h"
#include "gpic_mfma.h"

namespace gpic {

constexpr int kMaxRank = 128;

struct LoraArgs {
  const uint16_t *y, *x, *A, *B;
  const float *s;
  const void *ids;
  uint16_t *out;
  float *t;
  int64_t M, per, ldx, ldy;
  int N, K, R, n, wide_ids;       // wide_ids: 64-bit ids
  int splits, groups, col_blocks, cols;   // parts of K; workgroups that share a tile's passes; column blocks, of cols each
};

// The adapter of row m, or -1.
__device__ __forceinline__ int adapter_of(const LoraArgs &p, int64_t m) {
  if (m >= p.M) return -1;
  const int64_t i = p.wide_ids ? static_cast<const int64_t *>(p.ids)[m / p.per] : static_cast<const int *>(p.ids)[m / p.per];
  return i >= 0 && i < p.n ? (int)i : -1;
}

// Sixteen bytes of a row from element 8 c, zeros where off.
__device__ __forceinline__ s16x8 chunk16(const uint16_t *row, int c, bool on) {
  s16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
  if (on) z = *reinterpret_cast<const s16x8 *>(row + 8 * c);
  return z;
}

// t of 16 RT rows (NT tiles of 16 of the rank): the workgroups' parts of K, and in them the four waves', added in their order.
template <bool F16, int RT, int NT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraArgs p) {
  __shared__ float red[16 * RT][16 * NT + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * 16 * RT;
  const int split = blockIdx.y, group = blockIdx.z;
  const int id = lane < 16 * RT ? adapter_of(p, row0 + lane) : -1;
  const int steps = (p.K + 31) / 32, per = (steps + 4 * p.splits - 1) / (4 * p.splits);
  const int first = (split * 4 + wave) * per, end = min(steps, first + per);
  uint64_t todo = __ballot(id >= 0);
  for (int pass = 0; todo; pass++) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
    const uint64_t mine = __ballot(id == cur);
    todo &= ~mine;
    if (pass % p.groups != group) continue;
    f32x4_t acc[RT][NT];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const uint16_t *A = p.A + (int64_t)cur * p.R * p.K;
#pragma unroll 2
    for (int s = first; s < end; s++) {
      const int c = 4 * s + g;
      const bool in = 8 * c < p.K;
      s16x8 a[RT], b[NT];
#pragma unroll
      for (int i = 0; i < RT; i++)
        a[i] = chunk16(p.x + (row0 + 16 * i + l15) * p.ldx, c, in && (mine >> (16 * i + l15) & 1));
#pragma unroll
      for (int j = 0; j < NT; j++) b[j] = chunk16(A + (int64_t)(16 * j + l15) * p.K, c, in && 16 * j + l15 < p.R);
#pragma unroll
      for (int i = 0; i < RT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = mfma16<F16>(a[i], b[j], acc[i][j]);
    }
    for (int w = 0; w < 4; w++) {
      if (wave == w) {
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
          for (int j = 0; j < NT; j++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
              float &r = red[16 * i + 4 * g + v][16 * j + l15];
              r = w ? r + acc[i][j][v] : acc[i][j][v];
            }
      }
      __syncthreads();
    }
    for (int e = threadIdx.x; e < 16 * RT * p.R; e += 256) {
      const int m = e / p.R, r = e - m * p.R;
      if (mine >> m & 1) p.t[((int64_t)split * p.M + row0 + m) * p.R + r] = red[m][r];
    }
    __syncthreads();
  }
}

// out of 16 RT rows and p.cols columns: a wave 32 columns at a time, which the order of B's rows gives a lane as 8 beside each
// other (16 bytes of y and out). NS: steps of 32 over the rank's rounded and left-over halves.
template <bool F16, int RT, int NS>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs p) {
  constexpr int RP = 16 * NS;   // the rank, rounded up to tiles
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const int64_t row0 = (int64_t)blockIdx.x * 16 * RT;
  const int group = blockIdx.z;
  const int id = lane < 16 * RT ? adapter_of(p, row0 + lane) : -1;
  uint64_t todo = __ballot(lane < 16 * RT && row0 + lane < p.M);
  const int c0 = blockIdx.y * p.cols, c1 = min(p.N, c0 + p.cols);
  for (int pass = 0; todo; pass++) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
    const uint64_t mine = __ballot(id == cur) & todo;   // (rows without an adapter are a pass too)
    todo &= ~mine;
    if (pass % p.groups != group) continue;
    s16x8 tf[RT][NS];
    float up[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {
      float t[NS][8], most = 0.0f;
      const bool on = cur >= 0 && (mine >> (16 * i + l15) & 1);
#pragma unroll
      for (int k = 0; k < NS; k++) {
        const int kk = 32 * k + 8 * g, r = kk < RP ? kk : kk - RP;
#pragma unroll
        for (int e = 0; e < 8; e++) t[k][e] = 0.0f;
        if (on && r < p.R)
          for (int s = 0; s < p.splits; s++) {
            const float4 *src = reinterpret_cast<const float4 *>(p.t + ((int64_t)s * p.M + row0 + 16 * i + l15) * p.R + r);
            const float4 a = src[0], b = src[1];
            t[k][0] += a.x, t[k][1] += a.y, t[k][2] += a.z, t[k][3] += a.w;
            t[k][4] += b.x, t[k][5] += b.y, t[k][6] += b.z, t[k][7] += b.w;
          }
#pragma unroll
        for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(t[k][e]));
      }
      // (fp16: the row's largest brought to 2^8 .. 2^9 by a power of two, taken off the fp32 sums again)
      up[i] = 1.0f;
      float f = 1.0f;
      if (F16) {
        most = fmaxf(most, __shfl_xor(most, 16, 64));
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        if (most > 0.0f && most < kInf) {
          const int e = min(max((int)(__float_as_uint(most) >> 23 & 255) - 127 - 8, -100), 100);
          f = __builtin_ldexpf(1.0f, -e), up[i] = __builtin_ldexpf(1.0f, e);
        }
      }
#pragma unroll
      for (int k = 0; k < NS; k++) {
        const bool low = 32 * k + 8 * g >= RP;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          v[e] = t[k][e] * f;
          const float h = round16<F16>(v[e]);
          if (low) v[e] = fabsf(h) < kInf ? v[e] - h : 0.0f;   // (nothing is left over of an infinity)
        }
        tf[i][k] = __builtin_bit_cast(s16x8, u32x4{pack16<F16>(v[0], v[1]), pack16<F16>(v[2], v[3]), pack16<F16>(v[4], v[5]),
                                                   pack16<F16>(v[6], v[7])});
      }
    }
    const uint16_t *B = p.B + (int64_t)max(cur, 0) * p.N * p.R;
    const float s = cur >= 0 ? (p.s ? p.s[cur] : 1.0f) : 0.0f;
    for (int c = c0 + 32 * wave; c < c1; c += 128) {
      f32x4_t acc[RT][2];
#pragma unroll
      for (int i = 0; i < RT; i++) acc[i][0] = acc[i][1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      const int col = c + 8 * g;
      u32x4 Y[RT];
#pragma unroll
      for (int i = 0; i < RT; i++) {
        Y[i] = u32x4{0u, 0u, 0u, 0u};
        if ((mine >> (16 * i + l15) & 1) && col < c1)
          Y[i] = *reinterpret_cast<const u32x4 *>(p.y + (row0 + 16 * i + l15) * p.ldy + col);
      }
      if (cur >= 0) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int n = c + 8 * (l15 >> 2) + 4 * h + (l15 & 3);
#pragma unroll
          for (int k = 0; k < NS; k++) {
            const int kk = 32 * k + 8 * g, r = kk < RP ? kk : kk - RP;
            const s16x8 b = chunk16(B + (int64_t)n * p.R, r / 8, n < c1 && r < p.R);
#pragma unroll
            for (int i = 0; i < RT; i++) acc[i][h] = mfma16<F16>(b, tf[i][k], acc[i][h]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < RT; i++) {
        if (!(mine >> (16 * i + l15) & 1) || col >= c1) continue;
        if (cur >= 0) {
          float f[8];
          floats8<F16>(__builtin_bit_cast(s16x8, Y[i]), f);
#pragma unroll
          for (int e = 0; e < 8; e++) f[e] = __builtin_fmaf(acc[i][e >> 2][e & 3] * up[i], s, f[e]);
          Y[i] = u32x4{pack16<F16>(f[0], f[1]), pack16<F16>(f[2], f[3]), pack16<F16>(f[4], f[5]), pack16<F16>(f[6], f[7])};
        }
        *reinterpret_cast<u32x4 *>(p.out + (row0 + 16 * i + l15) * p.N + col) = Y[i];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------- host side

struct LoraPlan {
  int rt, nt, splits, groups, cols;
};
static LoraPlan lora_plan(int64_t M, int64_t K, int64_t N, int64_t R, int64_t n) {
  LoraPlan a;
  a.nt = R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8;
  a.rt = M >= 2048 ? 4 : 1;
  const int64_t tiles = (M + 16 * a.rt - 1) / (16 * a.rt);
  a.groups = M <= 256 ? (int)std::min<int64_t>(std::min<int64_t>(n, M), 4) : 1;
  const int64_t want = 512 / (tiles * a.groups), most = K / 512;   // (a wave 128 of K at least)
  a.splits = (int)std::max<int64_t>(std::min<int64_t>(std::min(want, most), 8), 1);
  a.cols = 128;
  while (a.cols < 1024 && tiles * a.groups * ((N + 2 * a.cols - 1) / (2 * a.cols)) >= 1024) a.cols *= 2;
  return a;
}

template <class F>
static void with_rank(int nt, F f) {
  if (nt == 1) f(std::integral_constant<int, 1>());
  else if (nt == 2) f(std::integral_constant<int, 2>());
  else if (nt == 4) f(std::integral_constant<int, 4>());
  else f(std::integral_constant<int, 8>());
}

}  // namespace gpic

using namespace gpic;

extern "C" {

size_t gpic_fp8_lora_rows_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t R, int64_t n) {
  if (M <= 0 || N <= 0 || K <= 0 || R <= 0 || n <= 0 || R > kMaxRank) return 0;
  return (size_t)lora_plan(M, K, N, R, n).splits * M * R * sizeof(float);
}

int gpic_fp8_lora_rows(const uint16_t *y, int64_t ldy, const uint16_t *x, int64_t ldx, const uint16_t *A, const uint16_t *B,
                       const float *scales, const void *ids, int wide_ids, int64_t per, int dtype, int64_t M, int64_t N, int64_t K,
                       int64_t R, int64_t n, uint16_t *out, void *ws, size_t ws_bytes, void *stream) {
  status_scope();
  if (M < 0 || N <= 0 || K <= 0 || R <= 0 || n <= 0 || per <= 0) return GPIC_EINVAL;
  if (M > 0 && (!y || !x || !A || !B || !ids || !out)) return GPIC_EINVAL;
  if (dtype != GPIC_DTYPE_BF16 && dtype != GPIC_DTYPE_F16) return GPIC_EDTYPE;
  const int64_t most = int64_t(1) << 30;
  if (N % 8 || K % 8 || R % 8 || R > kMaxRank || ldx % 8 || ldx < K || ldy % 8 || ldy < N || M >= most || N >= most || K >= most ||
      n >= most)
    return GPIC_ESHAPE;
  if (!aligned16(y) || !aligned16(x) || !aligned16(A) || !aligned16(B) || !aligned16(out) || !aligned16(ws)) return GPIC_EALIGN;
  if (M == 0) return GPIC_OK;
  if (ws_bytes < gpic_fp8_lora_rows_workspace_bytes(M, N, K, R, n) || !ws) return GPIC_EWORKSPACE;
  const LoraPlan a = lora_plan(M, K, N, R, n);
  const int64_t tiles = (M + 16 * a.rt - 1) / (16 * a.rt), blocks = (N + a.cols - 1) / a.cols;
  if (blocks > 65535 || tiles * std::max<int64_t>(blocks, a.splits) * a.groups >= (int64_t(1) << 24)) return GPIC_ESHAPE;
  const LoraArgs p{y, x, A, B, scales, ids, out, static_cast<float *>(ws), M, per, ldx, ldy, (int)N, (int)K, (int)R, (int)n,
                   wide_ids, a.splits, a.groups, (int)blocks, a.cols};
  const hipStream_t st = (hipStream_t)stream;
  const dim3 shrink((unsigned)tiles, (unsigned)a.splits, (unsigned)a.groups), expand((unsigned)tiles, (unsigned)blocks, (unsigned)a.groups);
  auto launch = [&](auto f16) {
    constexpr bool F = decltype(f16)::value;
    with_rank(a.nt, [&](auto nt) {
      constexpr int T = decltype(nt)::value;
      if (a.rt == 4) {
        lora_shrink_kernel<F, 4, T><<<shrink, 256, 0, st>>>(p);
        lora_expand_kernel<F, 4, T><<<expand, 256, 0, st>>>(p);
      } else {
        lora_shrink_kernel<F, 1, T><<<shrink, 256, 0, st>>>(p);
        lora_expand_kernel<F, 1, T><<<expand, 256, 0, st>>>(p);
      }
    });
  };
  if (dtype == GPIC_DTYPE_F16) launch(std::true_type());
  else launch(std::false_type());
  return (int)hipGetLastError();
}

}  // extern "C"
