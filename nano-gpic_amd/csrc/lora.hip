// Low-rank adapters of many requests beside a shared projection:
//
//   out[m] = y[m] + s_i (x[m] A_i^T) B_i^T, i = ids[m / per];  rows whose id is none of 0 .. n - 1: out[m] = y[m]
//   x [M, K], A [n, R, K], B [n, N, R], y (the shared projection's output), out [M, N], bf16 or fp16; s [n] fp32
//
// Two launches: t = x A_i^T, then the product with B_i added to y and rounded once. Both are bound by memory: x, y, out and the
// adapters in use once, since R is far below the matrix instructions' balance; few rows by the launches and the adapters' bytes.
// A tile of rows may hold rows of any adapters, in any order: it is passed over once for each adapter that occurs in it, all of its
// rows multiplied and those of the pass kept, so what an adapter holds reaches no row but its own. Passes of one tile are
// independent: few rows spread them over workgroups of their own.
// t stays exact to 2^-16 and better: the second product reads it as the sum of two 16-bit numbers, its rounding and what the
// rounding left, beside each other on the reduction, which costs little for a rank this small. Many rows: the first launch leaves
// them so, [M, 2 RP] (RP: the rank in tiles of 16). Few rows: it leaves fp32 parts of K by different workgroups, [splits, M, R].
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
  void *t;
  float *up;   // fp16: the factors of t's rows
  int64_t ldx, ldy;
  int M, per, N, K, R, n, wide_ids;   // wide_ids: 64-bit ids
  int splits, groups, cols;           // parts of K; workgroups that share a tile's passes; columns of a workgroup
};
constexpr int kMaxSplits = 4;

// The adapter of row m, or -1.
__device__ __forceinline__ int adapter_of(const LoraArgs &p, int m) {
  if (m >= p.M) return -1;
  const uint32_t at = p.per == 1 ? (uint32_t)m : (uint32_t)m / (uint32_t)p.per;
  const int64_t i = p.wide_ids ? static_cast<const int64_t *>(p.ids)[at] : static_cast<const int *>(p.ids)[at];
  return i >= 0 && i < p.n ? (int)i : -1;
}

// Sixteen bytes of a row from element 8 c, zeros where off.
__device__ __forceinline__ s16x8 chunk16(const uint16_t *row, int c, bool on) {
  s16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
  if (on) z = *reinterpret_cast<const s16x8 *>(row + 8 * c);
  return z;
}

// Eight values of t as 16-bit numbers: their rounding, or (low) what it left.
template <bool F16>
__device__ __forceinline__ s16x8 half_of(const float (&t)[8], bool low) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const float h = round16<F16>(t[e]);
    v[e] = !low ? t[e] : fabsf(h) < kInf ? t[e] - h : 0.0f;   // (nothing is left over of an infinity)
  }
  return __builtin_bit_cast(s16x8, u32x4{pack16<F16>(v[0], v[1]), pack16<F16>(v[2], v[3]), pack16<F16>(v[4], v[5]),
                                         pack16<F16>(v[6], v[7])});
}
// fp16: the power of two that brings a row's largest value of t to 2^8 .. 2^9, and its inverse, which goes to the fp32 sums.
__device__ __forceinline__ void row_factor(float most, float &down, float &up) {
  down = up = 1.0f;
  if (most > 0.0f && most < kInf) {
    const int e = min(max((int)(__float_as_uint(most) >> 23 & 255) - 127 - 8, -100), 100);
    down = __builtin_ldexpf(1.0f, -e), up = __builtin_ldexpf(1.0f, e);
  }
}

// t of 16 RT rows (NT tiles of 16 of the rank): the workgroups' parts of K (kParts), and in them the four waves', added in their
// order. The next step's loads are under way during a step's products.
template <bool F16, int RT, int NT, bool kParts>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraArgs p) {
  __shared__ float red[16 * RT][16 * NT + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const int row0 = blockIdx.x * 16 * RT;
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
    s16x8 a[RT], b[NT];
    auto fetch = [&](int s) {
      const int c = 4 * s + g;
      const bool in = s < end && 8 * c < p.K;
#pragma unroll
      for (int i = 0; i < RT; i++)
        a[i] = chunk16(p.x + (int64_t)(row0 + 16 * i + l15) * p.ldx, c, in && (mine >> (16 * i + l15) & 1));
#pragma unroll
      for (int j = 0; j < NT; j++) b[j] = chunk16(A + (int64_t)(16 * j + l15) * p.K, c, in && 16 * j + l15 < p.R);
    };
    fetch(first);
    for (int s = first; s < end; s++) {
      s16x8 an[RT], bn[NT];
#pragma unroll
      for (int i = 0; i < RT; i++) an[i] = a[i];
#pragma unroll
      for (int j = 0; j < NT; j++) bn[j] = b[j];
      fetch(s + 1);
#pragma unroll
      for (int i = 0; i < RT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = mfma16<F16>(an[i], bn[j], acc[i][j]);
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
    if constexpr (kParts) {
      for (int e = threadIdx.x; e < 16 * RT * p.R; e += 256) {
        const int m = e / p.R, r = e - m * p.R;
        if (mine >> m & 1) static_cast<float *>(p.t)[((int64_t)split * p.M + row0 + m) * p.R + r] = red[m][r];
      }
    } else {
      const int c = threadIdx.x & 15;   // (16 threads a row, 8 of the rank each)
      for (int m = threadIdx.x >> 4; m < 16 * RT; m += 16) {
        float t[8], most = 0.0f, down = 1.0f, up = 1.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) t[e] = c < 2 * NT ? red[m][8 * c + e] : 0.0f;
        if (F16) {
#pragma unroll
          for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(t[e]));
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
          row_factor(most, down, up);
#pragma unroll
          for (int e = 0; e < 8; e++) t[e] *= down;
        }
        if (!(mine >> m & 1)) continue;
        uint16_t *o = static_cast<uint16_t *>(p.t) + (int64_t)(row0 + m) * 32 * NT + 8 * c;
        if (c < 2 * NT) {
          *reinterpret_cast<s16x8 *>(o) = half_of<F16>(t, false);
          *reinterpret_cast<s16x8 *>(o + 16 * NT) = half_of<F16>(t, true);
        }
        if (F16 && c == 0) p.up[row0 + m] = up;
      }
    }
    __syncthreads();
  }
}

// out of 16 RT rows and p.cols columns: a wave 32 columns at a time, which the order of B's rows gives a lane as 8 beside each
// other (16 bytes of y and out); the next columns' loads are under way during a step's products. NS: steps of 32 over t's two
// halves, which meet the same chunks of B.
template <bool F16, int RT, int NS, bool kParts>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs p) {
  constexpr int RP = 16 * NS;             // the rank in tiles of 16
  constexpr int NB = NS > 1 ? NS / 2 : 1;   // steps over B's chunks (a rank of one tile: both halves in one step)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const int row0 = blockIdx.x * 16 * RT;
  const int group = blockIdx.z;
  const int id = lane < 16 * RT ? adapter_of(p, row0 + lane) : -1;
  uint64_t todo = __ballot(lane < 16 * RT && row0 + lane < p.M);
  const int c0 = blockIdx.y * p.cols, c1 = min(p.N, c0 + p.cols);
  for (int pass = 0; todo; pass++) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
    const uint64_t mine = __ballot(id == cur) & todo;   // (rows without an adapter are a pass too)
    todo &= ~mine;
    if (pass % p.groups != group) continue;
    const uint16_t *B = p.B + (int64_t)max(cur, 0) * p.N * p.R;
    u32x4 Y[RT];
    s16x8 b[2][NB];
    auto fetch = [&](int c) {
      const int col = c + 8 * g;
#pragma unroll
      for (int i = 0; i < RT; i++) {
        Y[i] = u32x4{0u, 0u, 0u, 0u};
        if ((mine >> (16 * i + l15) & 1) && col < c1)
          Y[i] = *reinterpret_cast<const u32x4 *>(p.y + (int64_t)(row0 + 16 * i + l15) * p.ldy + col);
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int n = c + 8 * (l15 >> 2) + 4 * h + (l15 & 3);
#pragma unroll
        for (int k = 0; k < NB; k++) {
          const int r = NS > 1 ? 32 * k + 8 * g : 8 * (g & 1);
          b[h][k] = chunk16(B + (int64_t)n * p.R, r / 8, cur >= 0 && n < c1 && r < p.R);
        }
      }
    };
    int c = c0 + 32 * wave;
    fetch(c);
    s16x8 tf[RT][NS];
    float up[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {
      const int row = row0 + 16 * i + l15;
      const bool on = cur >= 0 && (mine >> (16 * i + l15) & 1);
      up[i] = 1.0f;
      if constexpr (kParts) {
        float t[NS][8], most = 0.0f, down = 1.0f;
#pragma unroll
        for (int k = 0; k < NS; k++) {
          const int kk = 32 * k + 8 * g, r = kk < RP ? kk : kk - RP;
          float4 part[kMaxSplits][2];
#pragma unroll
          for (int s = 0; s < kMaxSplits; s++) {
            part[s][0] = part[s][1] = float4{0.0f, 0.0f, 0.0f, 0.0f};
            if (on && r < p.R && s < p.splits) {
              const float4 *src = reinterpret_cast<const float4 *>(static_cast<const float *>(p.t) + ((int64_t)s * p.M + row) * p.R + r);
              part[s][0] = src[0], part[s][1] = src[1];
            }
          }
#pragma unroll
          for (int e = 0; e < 8; e++) {
            auto of = [&](int s) { return reinterpret_cast<const float *>(&part[s][0])[e]; };
            t[k][e] = of(0);
#pragma unroll
            for (int s = 1; s < kMaxSplits; s++) t[k][e] += of(s);
            most = fmaxf(most, fabsf(t[k][e]));
          }
        }
        if (F16) {
          most = fmaxf(most, __shfl_xor(most, 16, 64));
          most = fmaxf(most, __shfl_xor(most, 32, 64));
          row_factor(most, down, up[i]);
        }
#pragma unroll
        for (int k = 0; k < NS; k++) {
#pragma unroll
          for (int e = 0; e < 8; e++) t[k][e] *= down;
          tf[i][k] = half_of<F16>(t[k], 32 * k + 8 * g >= RP);
        }
      } else {
#pragma unroll
        for (int k = 0; k < NS; k++) tf[i][k] = chunk16(static_cast<const uint16_t *>(p.t) + (int64_t)row * 2 * RP, 4 * k + g, on);
        if (F16 && on) up[i] = p.up[row];
      }
    }
    const float s = cur >= 0 && p.s ? p.s[cur] : 1.0f;
    for (; c < c1; c += 128) {
      u32x4 Yc[RT];
      s16x8 bc[2][NB];
#pragma unroll
      for (int i = 0; i < RT; i++) Yc[i] = Y[i];
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int k = 0; k < NB; k++) bc[h][k] = b[h][k];
      if (c + 128 < c1) fetch(c + 128);
      const int col = c + 8 * g;
#pragma unroll
      for (int i = 0; i < RT; i++) {
        f32x4_t acc[2] = {f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int k = 0; k < NS; k++) acc[h] = mfma16<F16>(bc[h][k % NB], tf[i][k], acc[h]);
        if (!(mine >> (16 * i + l15) & 1) || col >= c1) continue;
        if (cur >= 0) {
          float f[8];
          floats8<F16>(__builtin_bit_cast(s16x8, Yc[i]), f);
#pragma unroll
          for (int e = 0; e < 8; e++) f[e] = __builtin_fmaf(F16 ? acc[e >> 2][e & 3] * up[i] : acc[e >> 2][e & 3], s, f[e]);
          Yc[i] = u32x4{pack16<F16>(f[0], f[1]), pack16<F16>(f[2], f[3]), pack16<F16>(f[4], f[5]), pack16<F16>(f[6], f[7])};
        }
        *reinterpret_cast<u32x4 *>(p.out + (int64_t)(row0 + 16 * i + l15) * p.N + col) = Yc[i];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------- host side

struct LoraPlan {
  int nt, shrink_rt, rt, splits, groups, cols;
};
static LoraPlan lora_plan(int64_t M, int64_t K, int64_t N, int64_t R, int64_t n) {
  LoraPlan a;
  a.nt = R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8;
  const bool few = M <= 256;
  a.shrink_rt = M >= 8192 ? 2 : 1;
  a.rt = M < 1024 ? 1 : a.nt == 8 ? 2 : 4;
  a.groups = few ? (int)std::min<int64_t>(std::min<int64_t>(n + 1, M), 16) : 1;
  a.splits = few ? (int)std::max<int64_t>(std::min<int64_t>(K / 512, kMaxSplits), 1) : 1;   // (a wave 128 of K at least)
  const int64_t tiles = (M + 16 * a.rt - 1) / (16 * a.rt);
  a.cols = 128;
  while (a.cols < 1024 && tiles * ((N + 2 * a.cols - 1) / (2 * a.cols)) >= 2048) a.cols *= 2;
  return a;
}
static size_t lora_t_bytes(const LoraPlan &a, int64_t M, int64_t R) {
  return a.splits > 1 ? (size_t)a.splits * M * R * sizeof(float) : (size_t)M * 32 * a.nt * sizeof(uint16_t);
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
  const LoraPlan a = lora_plan(M, K, N, R, n);
  return lora_t_bytes(a, M, R) + (size_t)M * sizeof(float);
}

int gpic_fp8_lora_rows(const uint16_t *y, int64_t ldy, const uint16_t *x, int64_t ldx, const uint16_t *A, const uint16_t *B,
                       const float *scales, const void *ids, int wide_ids, int64_t per, int dtype, int64_t M, int64_t N, int64_t K,
                       int64_t R, int64_t n, uint16_t *out, void *ws, size_t ws_bytes, void *stream) {
  status_scope();
  if (M < 0 || N <= 0 || K <= 0 || R <= 0 || n <= 0 || per <= 0) return GPIC_EINVAL;
  if (M > 0 && (!y || !x || !A || !B || !ids || !out)) return GPIC_EINVAL;
  if (dtype != GPIC_DTYPE_BF16 && dtype != GPIC_DTYPE_F16) return GPIC_EDTYPE;
  const int64_t most = int64_t(1) << 30;
  if (N % 8 || K % 8 || R % 8 || R > kMaxRank || per >= most || ldx % 8 || ldx < K || ldy % 8 || ldy < N || M >= most || N >= most || K >= most ||
      n >= most)
    return GPIC_ESHAPE;
  if (!aligned16(y) || !aligned16(x) || !aligned16(A) || !aligned16(B) || !aligned16(out) || !aligned16(ws)) return GPIC_EALIGN;
  if (M == 0) return GPIC_OK;
  if (ws_bytes < gpic_fp8_lora_rows_workspace_bytes(M, N, K, R, n) || !ws) return GPIC_EWORKSPACE;
  const LoraPlan a = lora_plan(M, K, N, R, n);
  const int64_t tiles = (M + 16 * a.rt - 1) / (16 * a.rt), blocks = (N + a.cols - 1) / a.cols;
  const int64_t stiles = (M + 16 * a.shrink_rt - 1) / (16 * a.shrink_rt);
  // (a launch's threads are counted in 32 bits)
  if (blocks > 65535 || tiles * blocks * a.groups >= (int64_t(1) << 24) || stiles * a.splits * a.groups >= (int64_t(1) << 24))
    return GPIC_ESHAPE;
  char *w = static_cast<char *>(ws);
  const LoraArgs p{y, x, A, B, scales, ids, out, w, reinterpret_cast<float *>(w + lora_t_bytes(a, M, R)), ldx, ldy, (int)M, (int)per,
                   (int)N, (int)K, (int)R, (int)n, wide_ids, a.splits, a.groups, a.cols};
  const hipStream_t st = (hipStream_t)stream;
  const dim3 shrink((unsigned)stiles, (unsigned)a.splits, (unsigned)a.groups),
      expand((unsigned)tiles, (unsigned)blocks, (unsigned)a.groups);
  auto launch = [&](auto f16) {
    constexpr bool F = decltype(f16)::value;
    with_rank(a.nt, [&](auto nt) {
      constexpr int T = decltype(nt)::value, W = T == 8 ? 2 : 4;
      if (a.splits > 1) lora_shrink_kernel<F, 1, T, true><<<shrink, 256, 0, st>>>(p);
      else if (a.shrink_rt == 2) lora_shrink_kernel<F, 2, T, false><<<shrink, 256, 0, st>>>(p);
      else lora_shrink_kernel<F, 1, T, false><<<shrink, 256, 0, st>>>(p);
      if (a.splits > 1) lora_expand_kernel<F, 1, T, true><<<expand, 256, 0, st>>>(p);
      else if (a.rt == W) lora_expand_kernel<F, W, T, false><<<expand, 256, 0, st>>>(p);
      else lora_expand_kernel<F, 1, T, false><<<expand, 256, 0, st>>>(p);
    });
  };
  if (dtype == GPIC_DTYPE_F16) launch(std::true_type());
  else launch(std::false_type());
  return (int)hipGetLastError();
}

}  // extern "C"
