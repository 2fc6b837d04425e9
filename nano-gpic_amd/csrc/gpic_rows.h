// What the row operators (rows.hip, layernorm.hip) share: a team of T threads holds a row, 8 elements a thread and step; its sums
// and maxima; the columns' sums over the rows; and how many teams and rows a launch takes.
#pragma once
#include <algorithm>
#include <type_traits>

#include "gpic_device.h"
#include "gpic_launch.h"

namespace gpic {

constexpr int kMaxNormC = 16384;    // the norm's widest row (16 elements a thread: the backward also holds w and dw of them)
constexpr int kMaxRowC = 32768;     // the casts' widest row
constexpr int kMaxRowBlocks = 16384;

__device__ __forceinline__ void unpack8(u32x4 v, float (&f)[8]) {
  f[0] = bf16_lo(v.x), f[1] = bf16_hi(v.x), f[2] = bf16_lo(v.y), f[3] = bf16_hi(v.y);
  f[4] = bf16_lo(v.z), f[5] = bf16_hi(v.z), f[6] = bf16_lo(v.w), f[7] = bf16_hi(v.w);
}
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  return u32x4{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])};
}
__device__ __forceinline__ u32x4 ld16(const void *p) { return *reinterpret_cast<const u32x4 *>(p); }

// Eight elements of a bf16 or (f32) fp32 vector at element c.
__device__ __forceinline__ void load8(const void *p, bool f32, int64_t c, float (&f)[8]) {
  if (f32) {
    const float4 x = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + c);
    const float4 y = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + c + 4);
    f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w, f[4] = y.x, f[5] = y.y, f[6] = y.z, f[7] = y.w;
  } else {
    unpack8(ld16(static_cast<const uint16_t *>(p) + c), f);
  }
}

// Eight elements of a row in memory, as loaded: dtype 0 bf16, 1 fp32, 2 fp16 (GPIC_DTYPE_*).
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x8_t __attribute__((ext_vector_type(8)));

template <int E>
struct Raw8 {
  u32x4 v[E == 1 ? 2 : 1];
};
template <int E>
__device__ __forceinline__ Raw8<E> raw8(const void *p, int64_t c) {
  Raw8<E> r;
  if constexpr (E == 1) {
    r.v[0] = ld16(static_cast<const float *>(p) + c), r.v[1] = ld16(static_cast<const float *>(p) + c + 4);
  } else {
    r.v[0] = ld16(static_cast<const uint16_t *>(p) + c);
  }
  return r;
}
template <int E>
__device__ __forceinline__ Raw8<E> zero8() {
  Raw8<E> r;
  r.v[0] = u32x4{0u, 0u, 0u, 0u};
  if constexpr (E == 1) r.v[1] = r.v[0];
  return r;
}
template <int E>
__device__ __forceinline__ void values8(const Raw8<E> &r, float (&f)[8]) {
  if constexpr (E == 0) {
    unpack8(r.v[0], f);
  } else if constexpr (E == 1) {
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = __uint_as_float(r.v[e >> 2][e & 3]);
  } else {
    const f16x8_t h = __builtin_bit_cast(f16x8_t, r.v[0]);
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = (float)h[e];
  }
}
// Rounded to the type, to nearest even (fp32: as they are).
template <int E>
__device__ __forceinline__ Raw8<E> round8(const float (&f)[8]) {
  Raw8<E> r;
  if constexpr (E == 0) {
    r.v[0] = pack8(f);
  } else if constexpr (E == 1) {
#pragma unroll
    for (int e = 0; e < 8; e++) r.v[e >> 2][e & 3] = __float_as_uint(f[e]);
  } else {
    f16x8_t h;
#pragma unroll
    for (int e = 0; e < 8; e++) h[e] = (_Float16)f[e];
    r.v[0] = __builtin_bit_cast(u32x4, h);
  }
  return r;
}
template <int E>
__device__ __forceinline__ void store8(void *p, int64_t c, const Raw8<E> &r) {
  if constexpr (E == 1) {
    *reinterpret_cast<u32x4 *>(static_cast<float *>(p) + c) = r.v[0];
    *reinterpret_cast<u32x4 *>(static_cast<float *>(p) + c + 4) = r.v[1];
  } else {
    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(p) + c) = r.v[0];
  }
}
// Eight values of a vector whose type the launch says (a norm's weight and bias).
__device__ __forceinline__ void load8_as(const void *p, int dtype, int64_t c, float (&f)[8]) {
  if (dtype == GPIC_DTYPE_F16) values8<2>(raw8<2>(p, c), f);
  else load8(p, dtype == GPIC_DTYPE_F32, c, f);
}

__device__ __forceinline__ u32x2 cast8(const float (&h)[8], float s) {
  return u32x2{e4m3x4(sat(h[0] * s), sat(h[1] * s), sat(h[2] * s), sat(h[3] * s)),
               e4m3x4(sat(h[4] * s), sat(h[5] * s), sat(h[6] * s), sat(h[7] * s))};
}

__device__ __forceinline__ uint32_t absmax8(const float (&h)[8], uint32_t m) {
#pragma unroll
  for (int e = 0; e < 8; e++) m = max(m, __float_as_uint(h[e]) & 0x7fffffffu);
  return m;
}

// Sum, or maximum, over a team of T threads (T == 64: one wave; else the whole workgroup, through LDS, the waves' values in
// their order), the result in every thread. red: T / 64 words for this use alone; two uses alternate over a row, so the
// barrier of one protects the words of the other from the next row's writes.
template <int T>
__device__ __forceinline__ float team_sum(float v, float *red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    lds_barrier();
    v = red[0];
#pragma unroll
    for (int i = 1; i < T / 64; i++) v += red[i];
  }
  return v;
}
template <int T>
__device__ __forceinline__ uint32_t team_max(uint32_t v, uint32_t *red) {
  v = wave_max_u32(v);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    lds_barrier();
    v = red[0];
#pragma unroll
    for (int i = 1; i < T / 64; i++) v = max(v, red[i]);
  }
  return v;
}

template <int T>
constexpr int kWG = T > 256 ? T : 256;   // threads of a workgroup: 256 / T teams, or one

// The team's first row and the rows between two of its rows.
template <int T>
__device__ __forceinline__ int64_t team_row() {
  constexpr int R = kWG<T> / T;
  if constexpr (R == 1) return blockIdx.x;
  return (int64_t)blockIdx.x * R + __builtin_amdgcn_readfirstlane(threadIdx.x / T);
}
template <int T>
__device__ __forceinline__ int64_t team_step() {
  return (int64_t)gridDim.x * (kWG<T> / T);
}

// The teams' column sums D of a workgroup, added in their order by the first, to row blockIdx.x of P [.., C]. part: T kV 8 words
// where a workgroup has several teams.
template <int T, int kV>
__device__ __forceinline__ void store_column_partials(float (&D)[kV][8], float *part, float *P, int C) {
  constexpr int R = kWG<T> / T;
  const int t = threadIdx.x % T, team = threadIdx.x / T;
  if constexpr (R > 1) {
    for (int i = 1; i < R; i++) {
      __syncthreads();
      if (team == i) {
#pragma unroll
        for (int j = 0; j < kV; j++)
#pragma unroll
          for (int e = 0; e < 8; e++) part[(j * 8 + e) * T + t] = D[j][e];
      }
      __syncthreads();
      if (team == 0) {
#pragma unroll
        for (int j = 0; j < kV; j++)
#pragma unroll
          for (int e = 0; e < 8; e++) D[j][e] += part[(j * 8 + e) * T + t];
      }
    }
    if (team != 0) return;
  }
#pragma unroll
  for (int j = 0; j < kV; j++) {
    const int v = t + T * j;
    if (v < C / 8) {
      float *o = P + (int64_t)blockIdx.x * C + 8 * v;
      *reinterpret_cast<float4 *>(o) = float4{D[j][0], D[j][1], D[j][2], D[j][3]};
      *reinterpret_cast<float4 *>(o + 4) = float4{D[j][4], D[j][5], D[j][6], D[j][7]};
    }
  }
}

// The sums over g of P[g, c] for the 16 columns from 16 blockIdx.x, in fp32 in a fixed order: 4 threads of a workgroup of 256 take
// them, its 64 groups every 64th row each, four requested at a time, and the groups are added in pairs. True in the threads that
// then hold the sums of four columns, from 16 blockIdx.x + 4 (threadIdx.x & 3).
__device__ __forceinline__ bool column_sum16(const float *__restrict__ P, int G, int C, float4 (&red)[64][4], float4 &a) {
  const int c4 = threadIdx.x & 3, g0 = threadIdx.x >> 2;
  const int c = blockIdx.x * 16 + 4 * c4;
  a = float4{0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [](float4 &x, const float4 &y) { x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w; };
  if (c < C)
    for (int g = g0; g < G; g += 256) {
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        v[i] = float4{0.0f, 0.0f, 0.0f, 0.0f};
        if (g + 64 * i < G) v[i] = *reinterpret_cast<const float4 *>(P + (int64_t)(g + 64 * i) * C + c);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) add(a, v[i]);
    }
  red[g0][c4] = a;
  for (int n = 32; n > 0; n >>= 1) {
    __syncthreads();
    if (g0 < n) {
      add(a, red[g0 + n][c4]);
      red[g0][c4] = a;
    }
  }
  return g0 == 0 && c < C;
}

// ------------------------------------------------------------------------------------------- host side

// Calls f(T, kV) with the team and the steps for rows of C elements (C <= 8 T kV): the smallest team that holds a row in four
// steps, since a wave alone needs no barrier. us, norm / cast / norm's backward: rows of 1024 by a wave 9.8 / 4.8 / 14.1 (6528
// rows), by four 12.8 / 7.0 / 18.8; 4096 by four waves 19.8 / 71.4 / 102 (4096, 32768, 16381 rows), by one 30.2 / 79.2 / 114; 8192
// by four 22.3 / 33 / 51.0 (2048, 8192, 4096 rows), by sixteen 28.3 / 36.4 / 56.1. (Rows of 2048 by four waves cost the cast 3%
// and the norm 6%.)
template <class F>
static void with_team(int64_t C, F f) {
  typedef std::integral_constant<int, 64> W;
  typedef std::integral_constant<int, 256> Q;
  typedef std::integral_constant<int, 1024> S;
  typedef std::integral_constant<int, 1> V1;
  typedef std::integral_constant<int, 2> V2;
  typedef std::integral_constant<int, 4> V4;
  if (C <= 512) f(W(), V1());
  else if (C <= 1024) f(W(), V2());
  else if (C <= 2048) f(W(), V4());
  else if (C <= 4096) f(Q(), V2());
  else if (C <= 8192) f(Q(), V4());
  else if (C <= 16384) f(S(), V2());
  else f(S(), V4());
}

// The same for the epilogue's backward, which holds dy, z, db and two rows' loads: at most two steps a thread up to 16384. us,
// with db, against twice the steps: [6592 x 2048] 24.0 / 27.2, [16384 x 7168] 165 / 184, [8192 x 8192] 99 / 113.
template <class F>
static void with_short_team(int64_t C, F f) {
  typedef std::integral_constant<int, 1> V1;
  typedef std::integral_constant<int, 2> V2;
  typedef std::integral_constant<int, 256> Q;
  if (C <= 512) f(std::integral_constant<int, 64>(), V1());
  else if (C <= 1024) f(std::integral_constant<int, 64>(), V2());
  else if (C <= 2048) f(Q(), V1());
  else if (C <= 4096) f(Q(), V2());
  else if (C <= 8192) f(std::integral_constant<int, 512>(), V2());
  else if (C <= 16384) f(std::integral_constant<int, 1024>(), V2());
  else f(std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
}

static unsigned row_blocks(int64_t rows, int teams) {
  return (unsigned)std::min<int64_t>((rows + teams - 1) / teams, kMaxRowBlocks);
}

static bool dtype_ok(int d) { return d == GPIC_DTYPE_BF16 || d == GPIC_DTYPE_F32; }

// Rows a team of the norm takes one after another: one while the workgroups would not fill the device, then up to `most`, by what
// it keeps from row to row. Short runs spread a launch's stores over its time, long ones read shift, scale and gate less often.
// us, at most 1 / 2 / 4 / 8 rows: [16384 x 4096] with a residual alone 82.4 / 85.0 / 88.4 / 92.6, with residual, gate, shift and
// scale 96.4 / 89.1 / 89.3 / 94.2, with shift and scale alone 48.5 / 42.4 / 39.7 / 39.8, with neither 34.7 / 33.9 / 33.8 / 35.5;
// [32768 x 1024] in that order 35.2 / 36.6 / 37.5 / 37.5, 39.5 / 38.0 / 39.0 / 39.0, 25.3 / 22.2 / 22.4 / 22.5 and four times 20
// (the rule's worst: [8192 x 8192] with all of them 95.3 at 2 against 92.7).
static int norm_chunk(int64_t rows, int teams, int most) {
  const int64_t c = std::min<int64_t>(rows / (2048 * teams), most);
  return (int)std::max<int64_t>(std::max<int64_t>(c, 1), rows / ((int64_t)teams << 21) + 1);
}

}  // namespace gpic
