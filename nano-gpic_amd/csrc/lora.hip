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
// them so, [M, 2 RP] (RP: the rank in tiles of 16). Few rows: it leaves fp32 parts of K by different workgroups, [splits, M, R];
// in between, where K is long, parts that a small launch adds and leaves as many rows'.
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
  const float *parts;   // what lora_pack_kernel adds
  float *up;   // fp16: the factors of t's rows
  int64_t ldx, ldy;
  int M, per, N, K, R, n, wide_ids;   // wide_ids: 64-bit ids
  int splits, groups, blocks, cols;   // parts of K; workgroups that share a tile's passes; column blocks, of cols columns each
};
constexpr int kMaxSplits = 4, kMaxPacked = 8;   // parts that the second product adds, that are packed

// The adapter of row m, or -1.
__device__ __forceinline__ int adapter_of(const LoraArgs &p, int m) {
  if (m >= p.M) return -1;
  const uint32_t at = p.per == 1 ? (uint32_t)m : (uint32_t)m / (uint32_t)p.per;
  const int64_t i = p.wide_ids ? static_cast<const int64_t *>(p.ids)[at] : static_cast<const int *>(p.ids)[at];
  return i >= 0 && i < p.n ? (int)i : -1;
}

// Sixteen bytes of a row from element 8 c, or zeros.
__device__ __forceinline__ s16x8 chunk16(const uint16_t *row, int c) { return *reinterpret_cast<const s16x8 *>(row + 8 * c); }
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

// A row's t in halves: 16 threads a row, 8 of the rank each (zeros past R); kept where `on`.
template <bool F16, int NT>
__device__ __forceinline__ void leave_halves(const LoraArgs &p, int row, bool on, float (&t)[8]) {
  const int c = threadIdx.x & 15;
  float most = 0.0f, down = 1.0f, up = 1.0f;
  if (F16) {
#pragma unroll
    for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(t[e]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    row_factor(most, down, up);
#pragma unroll
    for (int e = 0; e < 8; e++) t[e] *= down;
  }
  if (!on || c >= 2 * NT) return;
  uint16_t *o = static_cast<uint16_t *>(p.t) + (int64_t)row * 32 * NT + 8 * c;
  *reinterpret_cast<s16x8 *>(o) = half_of<F16>(t, false);
  *reinterpret_cast<s16x8 *>(o + 16 * NT) = half_of<F16>(t, true);
  if (F16 && c == 0) p.up[row] = up;
}

// One row 2.6 us, [1500 x 1024] to rank 32 5.6.
// t of 16 rows (NT tiles of 16 of the rank): the workgroups' parts of K (kParts), and in them the waves', added in their order.
template <int NT>
constexpr int kShrinkWaves = NT == 8 ? 4 : 8;

template <bool F16, int NT, bool kParts>
__global__ __launch_bounds__(64 * kShrinkWaves<NT>) void lora_shrink_kernel(LoraArgs p) {
  constexpr int W = kShrinkWaves<NT>;
  __shared__ float red[W][16][16 * NT + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const int row0 = blockIdx.x * 16;
  const int split = blockIdx.y, group = blockIdx.z;
  const int steps = (p.K + 63) / 64, per = (steps + W * p.splits - 1) / (W * p.splits);
  const int first = (split * W + wave) * per, end = min(steps, first + per), whole = min(end, p.K / 64);
  // 64 of K a step, 16 from 16 g for group g: whole lines of x and A at a time. Loads have no conditions, so that they stay in
  // flight behind the products of the step before: rows past the last and of other passes, and the rank's past R, are read from
  // rows that are there, and what they give is not kept. K's last step, where it is none of 64, loads zeros past K.
  const uint16_t *xr = p.x + (int64_t)min(row0 + l15, p.M - 1) * p.ldx;
  struct Step {
    s16x8 a[2], b[NT][2];
  };
  auto fetch_x = [&](int s, Step &f) {
#pragma unroll
    for (int h = 0; h < 2; h++) f.a[h] = chunk16(xr, 8 * s + 2 * g + h);
  };
  Step f0, f1;
  if (first < whole) fetch_x(first, f0);   // (before the ids are known, which A waits for)
  const int id = lane < 16 ? adapter_of(p, row0 + lane) : -1;
  uint64_t todo = __ballot(id >= 0);
  bool again = false;
  for (int pass = 0; todo; pass++) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
    const uint64_t mine = __ballot(id == cur);
    todo &= ~mine;
    if (pass % p.groups != group) continue;
    f32x4_t acc[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) acc[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const uint16_t *Ar[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) Ar[j] = p.A + ((int64_t)cur * p.R + min(16 * j + l15, p.R - 1)) * p.K;
    auto fetch_A = [&](int s, Step &f) {
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int j = 0; j < NT; j++) f.b[j][h] = chunk16(Ar[j], 8 * s + 2 * g + h);
    };
    auto fetch = [&](int s, Step &f) {
      fetch_x(s, f);
      fetch_A(s, f);
    };
    auto multiply = [&](const Step &f) {
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[j] = mfma16<F16>(f.a[h], f.b[j][h], acc[j]);
    };
    int s = first;
    if (s < whole) {
      if (again) fetch_x(s, f0);
      fetch_A(s, f0);
    }
    again = true;
    for (; s + 2 < whole; s += 2) {
      fetch(s + 1, f1);
      multiply(f0);
      fetch(s + 2, f0);
      multiply(f1);
    }
    if (s + 1 < whole) {
      fetch(s + 1, f1);
      multiply(f0);
      multiply(f1);
      s += 2;
    } else if (s < whole) {
      multiply(f0);
      s++;
    }
    if (s < end) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int c = 8 * s + 2 * g + h;
        f0.a[h] = chunk16(xr, c, 8 * c < p.K);
#pragma unroll
        for (int j = 0; j < NT; j++) f0.b[j][h] = chunk16(Ar[j], c, 8 * c < p.K);
      }
      multiply(f0);
    }
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int v = 0; v < 4; v++) red[wave][4 * g + v][16 * j + l15] = acc[j][v];
    __syncthreads();
    auto sum = [&](int m, int r) {
      float x = red[0][m][r];
#pragma unroll
      for (int w = 1; w < W; w++) x += red[w][m][r];
      return x;
    };
    if constexpr (kParts) {
      for (int e = threadIdx.x; e < 16 * p.R; e += 64 * W) {
        const int m = e / p.R, r = e - m * p.R;
        if (mine >> m & 1) static_cast<float *>(p.t)[((int64_t)split * p.M + row0 + m) * p.R + r] = sum(m, r);
      }
    } else {
      const int c = threadIdx.x & 15;
      for (int m = threadIdx.x >> 4; m < 16; m += 4 * W) {
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; e++) t[e] = 8 * c < p.R ? sum(m, 8 * c + e) : 0.0f;
        leave_halves<F16, NT>(p, row0 + m, mine >> m & 1, t);
      }
    }
    __syncthreads();
  }
}

// [16384 x 4096] to rank 32 41 us (beside the writing out of the second product's results), [2648 x 1024] to rank 64 9.9.
// The same for many rows, 64 a workgroup: x and A come past the registers into LDS, whole lines at a time and stages ahead, each
// wave multiplies 16 rows. (Rows across the lanes, as above, take the memory pipeline four times as long.)
template <int NT>
constexpr int kStages = NT <= 4 ? 5 : 4;

template <bool F16, int NT, bool kParts>
__global__ __launch_bounds__(256) void lora_shrink_staged_kernel(LoraArgs p) {
  constexpr int KC = 64, C = KC / 8;   // columns of a stage, and 16-byte chunks
  constexpr int S = kStages<NT>, AR = NT == 1 ? 32 : 16 * NT, kX = C / 4, kA = AR * C / 256, kLoads = kX + kA;   // loads a lane
  __shared__ __attribute__((aligned(16))) uint16_t xt[S][64 * KC], at[S][AR * KC];
  __shared__ float red[4][16][16 * NT + 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l15 = lane & 15, g = lane >> 4;
  const int row0 = blockIdx.x * 64, split = blockIdx.y, group = blockIdx.z;
  const int steps = (p.K + KC - 1) / KC, per = (steps + p.splits - 1) / p.splits, first = split * per, end = min(steps, first + per);
  const int whole = min(end, p.K / KC);
  // load u of a wave: 1 KiB of a tile, a lane one chunk
  auto row_of = [&](int u) { return (64 * (4 * u + wave) + lane) / C; };
  auto chunk_of = [&](int u) { return lane % C ^ swz<KC>(row_of(u)); };
  const uint16_t *xr[kX], *Ar[kA], *xs[kX];
#pragma unroll
  for (int u = 0; u < kX; u++)
    xs[u] = p.x + (int64_t)min(row0 + row_of(u), p.M - 1) * p.ldx + KC * first + 8 * chunk_of(u);
  // The next step's loads into a buffer, and on; in the last ones (past K or the last step) zeros, so that as many loads are
  // always in flight.
  auto request = [&](int s, int buf, auto whole) {
    auto load = [&](uint16_t *tile, int u, const uint16_t *&from) {
      const void *src = from;
      if constexpr (!decltype(whole)::value) src = s < end && KC * s + 8 * chunk_of(u) < p.K ? src : (const void *)&kZeros;
      to_lds(src, lds_at(tile) + 1024 * (4 * u + wave));
      from += KC;
    };
#pragma unroll
    for (int u = 0; u < kX; u++) load(xt[buf], u, xr[u]);
#pragma unroll
    for (int u = 0; u < kA; u++) load(at[buf], u, Ar[u]);
  };
  int place[KC / 32];
#pragma unroll
  for (int k = 0; k < KC / 32; k++) place[k] = l15 * KC + ((4 * k + g) ^ swz<KC>(l15)) * 8;
  const int id = adapter_of(p, row0 + lane);
  uint64_t todo = __ballot(id >= 0);
  for (int pass = 0; todo; pass++) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
    const uint64_t mine = __ballot(id == cur);
    todo &= ~mine;
    if (pass % p.groups != group) continue;
#pragma unroll
    for (int u = 0; u < kX; u++) xr[u] = xs[u];
#pragma unroll
    for (int u = 0; u < kA; u++) Ar[u] = p.A + ((int64_t)cur * p.R + min(row_of(u), p.R - 1)) * p.K + KC * first + 8 * chunk_of(u);
    f32x4_t acc[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) acc[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < S - 1; i++) request(first + i, i, std::false_type());
    int s = first, buf = 0;
    auto step = [&](auto whole) {
      staged_but<(S - 2) * kLoads>();
      __syncthreads();   // (stage s is there, and stage s - 1 read)
      request(s + S - 1, buf == 0 ? S - 1 : buf - 1, whole);
#pragma unroll
      for (int k = 0; k < KC / 32; k++) {
        const s16x8 a = *reinterpret_cast<const s16x8 *>(xt[buf] + wave * 16 * KC + place[k]);
#pragma unroll
        for (int j = 0; j < NT; j++)
          acc[j] = mfma16<F16>(a, *reinterpret_cast<const s16x8 *>(at[buf] + j * 16 * KC + place[k]), acc[j]);
      }
      buf = buf + 1 == S ? 0 : buf + 1;
    };
    for (; s + S - 1 < whole; s++) step(std::true_type());
    for (; s < end; s++) step(std::false_type());
    staged();
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
      for (int v = 0; v < 4; v++) red[wave][4 * g + v][16 * j + l15] = acc[j][v];
    __syncthreads();
    const int c = threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int m = 16 * i + (threadIdx.x >> 4);
      const bool on = mine >> m & 1;
      float t[8];
#pragma unroll
      for (int e = 0; e < 8; e++) t[e] = 8 * c < p.R ? red[i][threadIdx.x >> 4][8 * c + e] : 0.0f;
      if constexpr (kParts) {
        float *o = static_cast<float *>(p.t) + ((int64_t)split * p.M + row0 + m) * p.R + 8 * c;
        if (on && 8 * c < p.R) {
          *reinterpret_cast<f32x4_t *>(o) = f32x4_t{t[0], t[1], t[2], t[3]};
          *reinterpret_cast<f32x4_t *>(o + 4) = f32x4_t{t[4], t[5], t[6], t[7]};
        }
      } else {
        leave_halves<F16, NT>(p, row0 + m, on, t);
      }
    }
    __syncthreads();
  }
}

// The parts of t added in their order and left in halves. (Rows without an adapter have no parts: what is made of them is not used.)
template <bool F16, int NT>
__global__ __launch_bounds__(256) void lora_pack_kernel(LoraArgs p) {
  const int row = blockIdx.x * 16 + (threadIdx.x >> 4), c = threadIdx.x & 15;
  const bool on = row < p.M && 8 * c < p.R;
  float t[8];
#pragma unroll
  for (int e = 0; e < 8; e++) t[e] = 0.0f;
  for (int s = 0; on && s < p.splits; s++) {
    const float4 *src = reinterpret_cast<const float4 *>(p.parts + ((int64_t)s * p.M + row) * p.R + 8 * c);
    const float4 a = src[0], b = src[1];
    t[0] += a.x, t[1] += a.y, t[2] += a.z, t[3] += a.w, t[4] += b.x, t[5] += b.y, t[6] += b.z, t[7] += b.w;
  }
  leave_halves<F16, NT>(p, row, row < p.M, t);
}

// 2648 rows of rank 64 to 4096 columns 19 us, 64 rows of rank 16 on 32 adapters 6.5, one row 3.1.
// out of 16 RT rows and p.cols columns: a wave 32 columns at a time, which the order of B's rows gives a lane as 8 beside each
// other (16 bytes of y and out); the next columns' loads are under way during a step's products. NS: steps of 32 over t's two
// halves, which meet the same chunks of B.
template <bool F16, int RT, int NS, bool kParts>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs p) {
  constexpr int RP = 16 * NS;             // the rank in tiles of 16
  constexpr int NB = NS > 1 ? NS / 2 : 1;   // steps over B's chunks (a rank of one tile: both halves in one step)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  // (workgroups beside each other take columns beside each other: rows whose length is a power of two would otherwise meet in few
  // of the memory's channels)
  const int tile = blockIdx.x / p.blocks, block = blockIdx.x - tile * p.blocks;
  const int row0 = tile * 16 * RT;
  const int group = blockIdx.y;
  const int c0 = block * p.cols, c1 = min(p.N, c0 + p.cols);
  // (loads without conditions, as above: of rows past the last and of other passes nothing is kept; t is zero past R, and B's
  // chunks there are taken as zeros; a step that runs past the last column reads its last columns again)
  const uint16_t *yr[RT];
#pragma unroll
  for (int i = 0; i < RT; i++) yr[i] = p.y + (int64_t)min(row0 + 16 * i + l15, p.M - 1) * p.ldy;
  struct Step {
    u32x4 y[RT];
    s16x8 b[2][NB];
  };
  auto fetch_y = [&](int c, Step &f) {
#pragma unroll
    for (int i = 0; i < RT; i++) f.y[i] = *reinterpret_cast<const u32x4 *>(yr[i] + min(c + 8 * g, (c1 - 1) & ~7));
  };
  Step f0, f1;
  s16x8 tf[RT][NS];
  float up[RT];
  auto fetch_t = [&]() {
#pragma unroll
    for (int i = 0; i < RT; i++) {
      const int row = min(row0 + 16 * i + l15, p.M - 1);
      up[i] = 1.0f;
      if constexpr (kParts) {
        float t[NS][8], most = 0.0f, down = 1.0f;
#pragma unroll
        for (int k = 0; k < NS; k++) {
          const int kk = 32 * k + 8 * g, r = kk < RP ? kk : kk - RP;
          float4 part[kMaxSplits][2];
#pragma unroll
          for (int s = 0; s < kMaxSplits; s++) {
            const float4 *src = reinterpret_cast<const float4 *>(static_cast<const float *>(p.t) +
                                                                 ((int64_t)min(s, p.splits - 1) * p.M + row) * p.R + min(r, p.R - 8));
            part[s][0] = src[0], part[s][1] = src[1];
          }
#pragma unroll
          for (int e = 0; e < 8; e++) {
            auto of = [&](int s) { return reinterpret_cast<const float *>(&part[s][0])[e]; };
            t[k][e] = of(0);
#pragma unroll
            for (int s = 1; s < kMaxSplits; s++) t[k][e] += s < p.splits ? of(s) : 0.0f;
            if (r >= p.R) t[k][e] = 0.0f;
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
        for (int k = 0; k < NS; k++) tf[i][k] = chunk16(static_cast<const uint16_t *>(p.t) + (int64_t)row * 2 * RP, 4 * k + g);
        if (F16) up[i] = p.up[row];
      }
    }
  };
  if (!kParts) {   // (before the ids are known, which B waits for; few rows' workgroups may have no pass)
    if (c0 + 32 * wave < c1) fetch_y(c0 + 32 * wave, f0);
    fetch_t();
  }
  const int id = lane < 16 * RT ? adapter_of(p, row0 + lane) : -1;
  uint64_t todo = __ballot(lane < 16 * RT && row0 + lane < p.M);
  bool again = false;
  for (int pass = 0; todo; pass++) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
    const uint64_t mine = __ballot(id == cur) & todo;   // (rows without an adapter are a pass too)
    todo &= ~mine;
    if (pass % p.groups != group) continue;
    const uint16_t *B = p.B + (int64_t)max(cur, 0) * p.N * p.R;
    auto fetch_B = [&](int c, Step &f) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int n = min(c + 8 * (l15 >> 2) + 4 * h + (l15 & 3), c1 - 1);
#pragma unroll
        for (int k = 0; k < NB; k++) {
          const int r = NS > 1 ? 32 * k + 8 * g : 8 * (g & 1);
          f.b[h][k] = chunk16(B + (int64_t)n * p.R, min(r, p.R - 8) / 8);
        }
      }
    };
    auto fetch = [&](int c, Step &f) {
      fetch_y(c, f);
      fetch_B(c, f);
    };
    int c = c0 + 32 * wave;
    if (c < c1) {
      if (kParts || again) fetch_y(c, f0);
      fetch_B(c, f0);
    }
    if (kParts && !again) fetch_t();
    again = true;
    const float s = cur >= 0 && p.s ? p.s[cur] : 1.0f;
    auto put = [&](int c, Step &f) {
      const int col = c + 8 * g;
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int k = 0; k < NB; k++)
          if ((NS > 1 ? 32 * k + 8 * g : 8 * (g & 1)) >= p.R) f.b[h][k] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < RT; i++) {
        if (!(mine >> (16 * i) & 0xffff)) continue;   // (a row tile without rows of the pass)
        u32x4 out = f.y[i];
        if (cur >= 0) {
          f32x4_t acc[2] = {f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int k = 0; k < NS; k++) acc[h] = mfma16<F16>(f.b[h][k % NB], tf[i][k], acc[h]);
          float v[8];
          floats8<F16>(__builtin_bit_cast(s16x8, out), v);
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] = __builtin_fmaf(F16 ? acc[e >> 2][e & 3] * up[i] : acc[e >> 2][e & 3], s, v[e]);
          out = u32x4{pack16<F16>(v[0], v[1]), pack16<F16>(v[2], v[3]), pack16<F16>(v[4], v[5]), pack16<F16>(v[6], v[7])};
        }
        if ((mine >> (16 * i + l15) & 1) && col < c1)
          *reinterpret_cast<u32x4 *>(p.out + (int64_t)(row0 + 16 * i + l15) * p.N + col) = out;
      }
    };
    for (; c + 128 < c1; c += 256) {
      fetch(c + 128, f1);
      put(c, f0);
      if (c + 256 < c1) fetch(c + 256, f0);
      put(c + 128, f1);
    }
    if (c < c1) put(c, f0);
  }
}

// The same for many rows and ranks of at most two tiles: the product is t B^T with t's rows as the result's rows, and tile h of a
// step of 16 HT columns takes B's rows HT l15 + h: a lane then holds HT columns beside each other, and 16 lanes one run of a row
// of y and out, which the memory pipeline takes whole (rows across the lanes cost it four times as long). 16384 rows of rank 32,
// 4096 columns: 50 us against 62; larger ranks, whose B's fragments are as many as y's runs, lose by it (2648 rows of rank 64 22
// -> 26 us, 4096 of 128 17 -> 21).
// NS: steps of 32 over t's two halves, which meet the same chunks of B.
template <bool F16, int RT, int NS>
__global__ __launch_bounds__(256) void lora_expand_runs_kernel(LoraArgs p) {
  constexpr int RP = 16 * NS;               // the rank in tiles of 16
  constexpr int NB = NS > 1 ? NS / 2 : 1;   // steps over B's chunks (a rank of one tile: both halves in one step)
  constexpr int HT = 8;
  typedef uint32_t Run __attribute__((ext_vector_type(HT / 2)));   // HT columns of y
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  // (workgroups beside each other take columns beside each other: rows whose length is a power of two would otherwise meet in few
  // of the memory's channels)
  const int tile = blockIdx.x / p.blocks, block = blockIdx.x - tile * p.blocks;
  const int row0 = tile * 16 * RT;
  const int group = blockIdx.y;
  const int c0 = block * p.cols, c1 = min(p.N, c0 + p.cols);
  // (loads without conditions, as above: of rows past the last and of other passes nothing is kept; t is zero past R, and B's
  // chunks there are taken as zeros; a step that runs past the last column reads its last columns again)
  // (a tile's rows at 32-bit offsets from its first)
  const uint16_t *yt = p.y + (int64_t)row0 * p.ldy;
  uint16_t *ot = p.out + (int64_t)row0 * p.N;
  const int last = p.M - 1 - row0;
  auto fetch_y = [&](int c, int i, Run (&y)[4]) {
#pragma unroll
    for (int v = 0; v < 4; v++)
      y[v] = *reinterpret_cast<const Run *>(yt + ((uint32_t)min(16 * i + 4 * g + v, last) * (uint32_t)p.ldy +
                                                  (uint32_t)min(c + HT * l15, c1 - HT)));
  };
  Run y0[4], y1[4];
  s16x8 tf[RT][NS];
  float up[RT];
  if (c0 + 16 * HT * wave < c1) fetch_y(c0 + 16 * HT * wave, 0, y0);   // (before the ids are known, which B waits for; t too)
#pragma unroll
  for (int i = 0; i < RT; i++) {
    const int row = min(row0 + 16 * i + l15, p.M - 1);
#pragma unroll
    for (int k = 0; k < NS; k++) tf[i][k] = chunk16(static_cast<const uint16_t *>(p.t) + (int64_t)row * 2 * RP, 4 * k + g);
    up[i] = F16 ? p.up[row] : 1.0f;
  }
  const int id = lane < 16 * RT ? adapter_of(p, row0 + lane) : -1;
  uint64_t todo = __ballot(lane < 16 * RT && row0 + lane < p.M);
  bool again = false;
  for (int pass = 0; todo; pass++) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
    const uint64_t mine = __ballot(id == cur) & todo;   // (rows without an adapter are a pass too)
    todo &= ~mine;
    if (pass % p.groups != group) continue;
    auto part = [&](int i) { return (mine >> (16 * i) & 0xffff) != 0; };   // whether row tile i has rows of the pass
    const uint16_t *B = p.B + (int64_t)max(cur, 0) * p.N * p.R;
    const float s = cur >= 0 && p.s ? p.s[cur] : 1.0f;
    // The result's rows 4 g + v of a row tile lie in other lanes than t's row l15: their factors
    float sv[RT][4];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
      for (int v = 0; v < 4; v++) sv[i][v] = F16 ? __shfl(up[i], 4 * g + v, 64) : 1.0f;
    for (int c = c0 + 16 * HT * wave; c < c1; c += 64 * HT) {
      s16x8 b[HT][NB];
#pragma unroll
      for (int h = 0; h < HT; h++)
#pragma unroll
        for (int k = 0; k < NB; k++) {
          const int r = NS > 1 ? 32 * k + 8 * g : 8 * (g & 1);
          b[h][k] = *reinterpret_cast<const s16x8 *>(B + ((uint32_t)min(c + HT * l15 + h, c1 - 1) * (uint32_t)p.R + min(r, p.R - 8)));
        }
      if (part(0) && (again || c != c0 + 16 * HT * wave)) fetch_y(c, 0, y0);
#pragma unroll
      for (int h = 0; h < HT; h++)
#pragma unroll
        for (int k = 0; k < NB; k++)
          if ((NS > 1 ? 32 * k + 8 * g : 8 * (g & 1)) >= p.R) b[h][k] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < RT; i++) {
        Run(&y)[4] = i & 1 ? y1 : y0;
        if (i + 1 < RT && part(i + 1)) fetch_y(c, i + 1, i & 1 ? y0 : y1);
        if (!part(i)) continue;
        f32x4_t acc[HT];
#pragma unroll
        for (int h = 0; h < HT; h++) {
          acc[h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
          if (cur >= 0) {
#pragma unroll
            for (int k = 0; k < NS; k++) acc[h] = mfma16<F16>(tf[i][k], b[h][k % NB], acc[h]);
          }
        }
#pragma unroll
        for (int v = 0; v < 4; v++) {
          Run out = y[v];
          if (cur >= 0) {
#pragma unroll
            for (int h = 0; h < HT; h += 2) {
              const float lo = __builtin_fmaf(F16 ? acc[h][v] * sv[i][v] : acc[h][v], s, low16<F16>(out[h / 2]));
              const float hi = __builtin_fmaf(F16 ? acc[h + 1][v] * sv[i][v] : acc[h + 1][v], s, high16<F16>(out[h / 2]));
              out[h / 2] = pack16<F16>(lo, hi);
            }
          }
          if ((mine >> (16 * i + 4 * g + v) & 1) && c + HT * l15 < c1)
            *reinterpret_cast<Run *>(ot + ((uint32_t)(16 * i + 4 * g + v) * (uint32_t)p.N + (uint32_t)(c + HT * l15))) = out;
        }
      }
    }
    again = true;
  }
}

// ------------------------------------------------------------------------------------------- host side

struct LoraPlan {
  int nt, rt, splits, groups, cols;
  bool few, staged, runs;   // few rows: their parts go into the second product; staged, runs: the kernels of those names
};
// us, first + second product. Up to 256 rows the parts, few rows' columns and up to 16 workgroups for a tile's passes: 200 rows of
// rank 64, 2048 to 2048, 5.0 + 7.0, as many rows 11.6 + 4.2; 100 of rank 16, 1024 to 4096, 4.1 + 3.5 against 6.8 + 4.8; 500 of
// rank 16 the other way, 4.3 + 7.4 against 4.9 + 4.4. Two workgroups for a tile's passes while one would not fill the device: 500
// rows of rank 64, 4096 to 4096, 20.7 + 7.9 against 38.8 + 8.8, 4000 rows 24 + 22 against 25 + 19.
// First product, tiles from the registers / staged: 2648 rows x 1024 to rank 64 12.3 / 9.9, 5000 x 2048 to 32 18 / 16, 16384 x 256
// to 128 12.9 / 8.6, 16384 x 4096 to 32 45 / 41.5; but 1500 x 1024 to 32 5.6 / 6.7, 4096 x 512 to 16 4.2 / 5.3. Long K in parts
// while there are few tiles, and 4.3 to pack them: 4096 rows x 4096 to 32 18.4 / 9.4, 1000 x 8192 17.4 / 6.8, 4096 x 2048 to 128
// 20.5 / 12.7; 2500 x 2048 to 32 loses by it.
static LoraPlan lora_plan(int64_t M, int64_t K, int64_t N, int64_t R, int64_t n) {
  LoraPlan a;
  a.nt = R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8;
  const bool few = a.few = M <= 256;
  a.rt = M < 1024 ? 1 : a.nt == 8 ? 2 : 4;
  a.groups = few ? (int)std::min<int64_t>(std::min<int64_t>(n + 1, M), 16) : M < 4096 ? 2 : 1;
  a.staged = !few && (a.nt >= 4 || K >= 4096 || M * K >= (int64_t(1) << 23));
  int64_t splits = few ? std::min<int64_t>(K / 512, kMaxSplits) : 1;
  if (a.staged && K >= (a.nt == 8 ? 2048 : 4096)) splits = std::min<int64_t>({K / 512, 256 / ((M + 63) / 64), kMaxPacked});
  a.splits = (int)std::max<int64_t>(splits, 1);
  const int64_t tiles = (M + 16 * a.rt - 1) / (16 * a.rt);
  a.runs = a.rt == 4 && a.nt <= 2;
  a.cols = a.runs ? 512 : few ? 256 : 128;   // (a step of the workgroup's waves, few rows two)
  while (!few && a.cols < 1024 && tiles * ((N + 2 * a.cols - 1) / (2 * a.cols)) >= (a.runs ? 512 : 256)) a.cols *= 2;
  return a;
}
// t's halves (few rows: its parts), its rows' factors, and the parts that are packed: bytes before each, and of all
struct LoraSpace {
  size_t up, parts, all;
};
static LoraSpace lora_space(const LoraPlan &a, int64_t M, int64_t R) {
  const size_t parts = a.splits > 1 ? (size_t)a.splits * M * R * sizeof(float) : 0, halves = (size_t)M * 32 * a.nt * sizeof(uint16_t);
  LoraSpace s;
  s.up = a.few && parts ? parts : halves;
  s.parts = (s.up + M * sizeof(float) + 15) & ~size_t(15);
  s.all = s.parts + (a.few ? 0 : parts);
  return s;
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
  return lora_space(lora_plan(M, K, N, R, n), M, R).all;
}

int gpic_fp8_lora_rows(const uint16_t *y, int64_t ldy, const uint16_t *x, int64_t ldx, const uint16_t *A, const uint16_t *B,
                       const float *scales, const void *ids, int wide_ids, int64_t per, int dtype, int64_t M, int64_t N, int64_t K,
                       int64_t R, int64_t n, uint16_t *out, void *ws, size_t ws_bytes, void *stream) {
  status_scope();
  if (M < 0 || N <= 0 || K <= 0 || R <= 0 || n <= 0 || per <= 0) return GPIC_EINVAL;
  if (M > 0 && (!y || !x || !A || !B || !ids || !out)) return GPIC_EINVAL;
  if (dtype != GPIC_DTYPE_BF16 && dtype != GPIC_DTYPE_F16) return GPIC_EDTYPE;
  const int64_t most = int64_t(1) << 30, wide = int64_t(1) << 24;   // (a tile's offsets in 32 bits)
  if (N % 8 || K % 8 || R % 8 || R > kMaxRank || per >= most || ldx % 8 || ldx < K || ldy % 8 || ldy < N || M >= most || N >= wide ||
      K >= wide || ldx >= wide || ldy >= wide || n >= most)
    return GPIC_ESHAPE;
  if (!aligned16(y) || !aligned16(x) || !aligned16(A) || !aligned16(B) || !aligned16(out) || !aligned16(ws)) return GPIC_EALIGN;
  if (M == 0) return GPIC_OK;
  if (ws_bytes < gpic_fp8_lora_rows_workspace_bytes(M, N, K, R, n) || !ws) return GPIC_EWORKSPACE;
  const LoraPlan a = lora_plan(M, K, N, R, n);
  const int64_t tiles = (M + 16 * a.rt - 1) / (16 * a.rt), blocks = (N + a.cols - 1) / a.cols;
  const int64_t stiles = a.staged ? (M + 63) / 64 : (M + 15) / 16;
  // (a launch's threads are counted in 32 bits)
  if (tiles * blocks * a.groups >= (int64_t(1) << 24) || stiles * a.splits * a.groups >= (int64_t(1) << 24))
    return GPIC_ESHAPE;
  char *w = static_cast<char *>(ws);
  const LoraSpace space = lora_space(a, M, R);
  LoraArgs p{y, x, A, B, scales, ids, out, w, reinterpret_cast<const float *>(w + space.parts), reinterpret_cast<float *>(w + space.up),
             ldx, ldy, (int)M, (int)per, (int)N, (int)K, (int)R, (int)n, wide_ids, a.splits, a.groups, (int)blocks, a.cols};
  const hipStream_t st = (hipStream_t)stream;
  const dim3 shrink((unsigned)stiles, (unsigned)a.splits, (unsigned)a.groups),
      expand((unsigned)(tiles * blocks), (unsigned)a.groups);
  auto launch = [&](auto f16) {
    constexpr bool F = decltype(f16)::value;
    with_rank(a.nt, [&](auto nt) {
      constexpr int T = decltype(nt)::value;
      if (a.staged && a.splits > 1) {
        LoraArgs q = p;
        q.t = w + space.parts;
        lora_shrink_staged_kernel<F, T, true><<<shrink, 256, 0, st>>>(q);
        lora_pack_kernel<F, T><<<(unsigned)((M + 15) / 16), 256, 0, st>>>(p);
      } else if (a.staged) {
        lora_shrink_staged_kernel<F, T, false><<<shrink, 256, 0, st>>>(p);
      } else if (a.splits > 1) {
        lora_shrink_kernel<F, T, true><<<shrink, 64 * kShrinkWaves<T>, 0, st>>>(p);
      } else {
        lora_shrink_kernel<F, T, false><<<shrink, 64 * kShrinkWaves<T>, 0, st>>>(p);
      }
      if (a.few && a.splits > 1) lora_expand_kernel<F, 1, T, true><<<expand, 256, 0, st>>>(p);
      else if (a.rt == 1) lora_expand_kernel<F, 1, T, false><<<expand, 256, 0, st>>>(p);
      else if constexpr (T <= 2) lora_expand_runs_kernel<F, 4, T><<<expand, 256, 0, st>>>(p);
      else lora_expand_kernel<F, T == 8 ? 2 : 4, T, false><<<expand, 256, 0, st>>>(p);
    });
  };
  if (dtype == GPIC_DTYPE_F16) launch(std::true_type());
  else launch(std::false_type());
  return (int)hipGetLastError();
}

}  // extern "C"
