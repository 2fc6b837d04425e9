// Attention of queries to an encoder's states of another length, forward and backward, for gfx950.
//
//   S = scale q k^T over the valid keys of the query's batch entry;  P = softmax(S) (zeros where no key is valid);  o = P v
//   lse = log2 sum 2^(S log2 e) (kept for the backward; +inf where nothing is valid)
//   delta = sum(do o);  dv = P^T do;  dP = do v^T;  dS = P (dP - delta);  dq = scale dS k;  dk = scale dS^T q
//
// A key is valid below its batch entry's length and where its mask is true. Rows of k and v that are not are never used: they are
// taken as zeros when a tile is staged, so that an infinity or NaN in padding reaches nothing, and their gradients are zeros.
// The heads that share a key's head (H = G Hk) are rows beside each other: a (batch entry, key head) pair has G N rows of q.
//
// All products run on v_mfma_f32_16x16x32 (bf16 or fp16 operands, fp32 sums): lane l gives row (column) l & 15 and the 8 terms
// from 8 (l / 16), and holds rows 4 (l / 16) + v of column l & 15 of the result. Each kernel takes the product that yields P (or
// dS) with the index that is summed next as its rows, so that the result, rounded to 16 bits, is the next product's right operand
// as it lies in its lane: terms 8 g + e of group g = l / 16 are rows 4 g + e of two 16-row tiles (e < 4 the first's), and the left
// operand, read from the staged tile by columns (ds_read_b64_tr_b16: four rows' 16 columns, one column a lane), takes its rows in
// that same order. A softmax's maximum and sum are then over a lane's own values and two exchanges between the four groups.
//
// Staged tiles hold rows of DP elements (head dimensions up to DP, the rest zeros) in 16-byte chunks, chunk c of row r in place
// c ^ swz(r), where swz permutes the row's lowest bits so that both the reads by rows (16 rows, one chunk) and the reads by columns
// (8 rows, two chunks) touch every bank once.
#include <algorithm>
#include <type_traits>

#include "gpic_device.h"
#include "gpic_launch.h"
#include "gpic_mfma.h"

namespace gpic {

typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kTile = 64;   // rows of a staged tile

struct AttnArgs {
  const uint16_t *q, *k, *v, *o, *dout;
  uint16_t *out, *dq, *dk, *dv;
  int64_t qs[3], ks[3], vs[3], os[3], ds[3], dqs[3], dks[3], dvs[3];   // strides: batch entry, head, row
  const int *lens;                                                     // [B] or null
  const uint8_t *mask;                                                 // [B, L] or null
  int64_t ldm;
  float *lse, *delta, *rowmax, *part;
  int B, H, Hk, N, L, D, G, rows, tiles, splits;   // rows: G N; tiles: row (or key) tiles of a (batch entry, key head) pair
  int rtiles;                                      // row tiles of the dq kernel
  int budget, least;   // Runs: workgroups of a key head (0: no runs, `splits` for every pair), a run's least tiles
  float c, scale;                                  // c: scale log2 e
};

// Two result tiles as a right operand.
template <bool F16>
__device__ __forceinline__ s16x8 operand(f32x4_t a, f32x4_t b) {
  return __builtin_bit_cast(s16x8, u32x4{pack16<F16>(a[0], a[1]), pack16<F16>(a[2], a[3]), pack16<F16>(b[0], b[1]),
                                         pack16<F16>(b[2], b[3])});
}
// A result row, f times x, to 16 bits in memory (zeros unless `valid`), where `on`: the groups of 16 lanes hold 4 columns of a tile
// each; two tiles' exchanged between neighbouring groups are 8 beside each other, 16 bytes a store (8: the kernels take 4 to 12%
// longer, dk and dv most).
template <bool F16, int DT>
__device__ __forceinline__ void put_row(uint16_t *row, int D, const f32x4_t (&x)[DT], float f, bool on, bool valid = true) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int d = 0; d < DT; d += 2) {
    const auto lo = __builtin_amdgcn_permlane16_swap(pack16<F16>(x[d][0] * f, x[d][1] * f),
                                                     pack16<F16>(x[d + 1][0] * f, x[d + 1][1] * f), false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(pack16<F16>(x[d][2] * f, x[d][3] * f),
                                                     pack16<F16>(x[d + 1][2] * f, x[d + 1][3] * f), false, false);
    const int col = 16 * (d + (g & 1)) + 8 * (g >> 1);
    if (on && col < D) *reinterpret_cast<u32x4 *>(row + col) = valid ? u32x4{lo[0], hi[0], lo[1], hi[1]} : u32x4{0u, 0u, 0u, 0u};
  }
}
// Sum, or maximum, of a value over the four groups of 16 lanes, in every lane: two exchanges of half the lanes, in registers.
template <class F>
__device__ __forceinline__ float over_groups(float v, F f) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
  return over_groups(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float groups_max(float v) {
  return over_groups(v, [](float a, float b) { return fmaxf(a, b); });
}

// A lane's places in a staged tile (element offsets): for the read by rows of 16-row tile t and step ks, add t 16 DP to row[ks];
// for the read by columns of tile t and columns 16 dt.., add t 16 DP to col[dt].
template <int DP>
struct Places {
  int row[DP / 32], col[DP / 16];
  __device__ __forceinline__ Places(int lane) {
    const int l15 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int k = 0; k < DP / 32; k++) row[k] = l15 * DP + ((4 * k + g) ^ swz<DP>(l15)) * 8;
    const int r = 4 * g + (l15 >> 2);
#pragma unroll
    for (int d = 0; d < DP / 16; d++) col[d] = r * DP + ((2 * d + ((l15 >> 1) & 1)) ^ swz<DP>(r)) * 8 + (l15 & 1) * 4;
  }
};
template <int DP>
__device__ __forceinline__ s16x8 by_rows(const uint16_t *tile, int t, int place) {
  return *reinterpret_cast<const s16x8 *>(tile + t * 16 * DP + place);
}
// Columns of 16-row tiles t and t + 1
template <int DP>
__device__ __forceinline__ s16x8 by_columns(uint16_t *tile, int t, int place) {
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + t * 16 * DP + place));
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + (t + 1) * 16 * DP + place));
  return s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// How 256 threads stage a tile of kTile rows: kU loads each, load u of wave w to places 64 (4 u + w) + lane, of which place i is
// place i % kC of row i / kC and takes that row's chunk (i % kC) ^ swz(row).
template <int DP>
struct Stage {
  static constexpr int kC = DP / 8, kU = kTile * kC / 256;
  __device__ __forceinline__ static int row(int u) { return (64 * (4 * u + (int)(threadIdx.x >> 6)) + (int)(threadIdx.x & 63)) / kC; }
  __device__ __forceinline__ static int chunk(int u) { return ((int)(threadIdx.x & 63) % kC) ^ swz<DP>(row(u)); }
  __device__ __forceinline__ static void put(uint16_t *tile, int u, const uint16_t *src, bool on) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    to_lds(on ? (const void *)src : (const void *)&kZeros, lds_at(tile) + 1024 * (4 * u + w));
  }
};
// The same for rows at one stride: a lane's offsets are kept.
template <int DP>
struct RowStage {
  int64_t at[Stage<DP>::kU];
  __device__ __forceinline__ explicit RowStage(int64_t stride) {
#pragma unroll
    for (int u = 0; u < Stage<DP>::kU; u++) at[u] = Stage<DP>::row(u) * stride + 8 * Stage<DP>::chunk(u);
  }
  // Row i at base + i stride where bit i of rows is set; zeros elsewhere and past column D.
  __device__ __forceinline__ void load(uint16_t *tile, const uint16_t *base, uint64_t rows, int D) const {
#pragma unroll
    for (int u = 0; u < Stage<DP>::kU; u++)
      Stage<DP>::put(tile, u, base + at[u], (rows >> Stage<DP>::row(u) & 1) && 8 * Stage<DP>::chunk(u) < D);
  }
};

// The keys of a batch entry: those below len, and of them those whose mask is true.
struct Keys {
  const uint8_t *mask;
  int len;
  __device__ __forceinline__ Keys(const AttnArgs &p, int b) {
    len = p.lens ? min(max(p.lens[b], 0), p.L) : p.L;
    mask = p.mask ? p.mask + b * p.ldm : nullptr;
  }
  __device__ __forceinline__ bool valid(int j) const { return j < len && (!mask || mask[j]); }
  // Bit i: whether key j0 + i is valid
  __device__ __forceinline__ uint64_t tile(int j0) const { return __ballot(valid(j0 + (int)(threadIdx.x & 63))); }
  // The first tile at or after i (of kTile keys) that has a valid key, and its bits; at `end`, none.
  __device__ __forceinline__ int next(int i, int end, uint64_t &bits) const {
    for (; i < end; i++) {
      bits = tile(i * kTile);
      if (bits) return i;
    }
    return end;
  }
};

// The heads and rows of a (batch entry, key head) pair: row r is row r % N of head hk G + r / N.
__device__ __forceinline__ int64_t row_at(const AttnArgs &p, const int64_t (&s)[3], int b, int hk, int r) {
  const int h = p.G == 1 ? 0 : r / p.N;
  return b * s[0] + (hk * p.G + h) * s[1] + (r - h * p.N) * s[2];
}
// A row's 8 elements from 8 (4 ks + g), zeros past D and past the last row.
__device__ __forceinline__ s16x8 row_chunk(const uint16_t *row, int chunk, int D, bool on) {
  s16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
  if (on && 8 * chunk < D) z = *reinterpret_cast<const s16x8 *>(row + 8 * chunk);
  return z;
}

// The scores of a key tile as powers of two relative to a running maximum: p = 2^(c s - use). The maximum is brought up to date, and
// o and l shrunk, only when some row of the wave has passed its own by 2^8: p stays below that, which 16 bits hold as well, and
// most tiles skip it. The sum l is of p before its rounding: a sum of the rounded p, by a matrix instruction with ones, would move
// lse, and with it the backward's P, by as much as P's own rounding does. A lane sums its own keys, in four parts.
struct Softmax {
  float use = -kInf;
  // mx: the tile's maximum, the same in all groups. Whether the wave moves.
  __device__ __forceinline__ bool moves(float mx, float c) const { return __ballot(mx * c > use + kSlack) != 0; }
  // The factor for o and l.
  __device__ __forceinline__ float move(float mx, float c) {
    const float old = use;
    use = fmaxf(old, mx * c);
    return old == -kInf ? 0.0f : __builtin_amdgcn_exp2f(old - use);
  }
  // Of a row without a score above -inf so far, 0: its p are 0 all the same.
  __device__ __forceinline__ float base() const { return use == -kInf ? 0.0f : use; }
  static constexpr float kSlack = 8.0f;
};
// ------------------------------------------------------------------------------------------- forward

// Between memory, VALU and MFMA: 2 x 256 rows over up to 77 keys 5.0 us (latency); 128 x 16 heads of 256 over up to 320, dimension
// 64, 69 us (VALU two thirds busy, 3 TB/s); 4 x 16 of 1024 over 2048, dimension 128, 81 us, 0.85 PFLOP/s.
// A workgroup's four waves take 16 QT rows each and walk the pair's keys (or its split's part of them) by tiles of 64, k and v
// staged through two buffers: the next tile's loads are under way during the current one's products.
template <bool F16, int DP, int QT>
__global__ __launch_bounds__(256, 2) void attn_fwd_kernel(AttnArgs p) {
  constexpr int KS = DP / 32, DT = DP / 16;
  __shared__ __attribute__((aligned(16))) uint16_t kt[2][kTile * DP], vt[2][kTile * DP];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  const int rt = id % p.tiles, split = id / p.tiles % p.splits, pair = id / p.tiles / p.splits;
  const int b = pair / p.Hk, hk = pair - b * p.Hk;
  const Keys keys(p, b);
  const Places<DP> at(lane);
  const int row0 = rt * 64 * QT + wave * 16 * QT;
  s16x8 qf[QT][KS];
#pragma unroll
  for (int i = 0; i < QT; i++) {
    const int r = row0 + 16 * i + l15;
    const uint16_t *row = p.q + row_at(p, p.qs, b, hk, min(r, p.rows - 1));
#pragma unroll
    for (int k = 0; k < KS; k++) qf[i][k] = row_chunk(row, 4 * k + g, p.D, r < p.rows);
  }
  f32x4_t O[QT][DT], l4[QT];
  Softmax sm[QT];
#pragma unroll
  for (int i = 0; i < QT; i++) {
    l4[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int d = 0; d < DT; d++) O[i][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const uint16_t *kb = p.k + b * p.ks[0] + hk * p.ks[1], *vb = p.v + b * p.vs[0] + hk * p.vs[1];
  const int n = (keys.len + kTile - 1) / kTile, per = (n + p.splits - 1) / p.splits;
  const int end = min(n, (split + 1) * per);
  uint64_t bits = 0, nbits = 0;
  int i = keys.next(split * per, end, bits);
  const RowStage<DP> sk(p.ks[2]), sv(p.vs[2]);
  if (i < end) {
    sk.load(kt[0], kb + (int64_t)i * kTile * p.ks[2], bits, p.D);
    sv.load(vt[0], vb + (int64_t)i * kTile * p.vs[2], bits, p.D);
  }
  staged();
  __syncthreads();
  for (int cur = 0; i < end; cur ^= 1, bits = nbits) {
    const int j = keys.next(i + 1, end, nbits);
    if (j < end) {
      sk.load(kt[cur ^ 1], kb + (int64_t)j * kTile * p.ks[2], nbits, p.D);
      sv.load(vt[cur ^ 1], vb + (int64_t)j * kTile * p.vs[2], nbits, p.D);
    }
    f32x4_t S[QT][4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
#pragma unroll
      for (int q = 0; q < QT; q++) S[q][t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const s16x8 a = by_rows<DP>(kt[cur], t, at.row[k]);
#pragma unroll
        for (int q = 0; q < QT; q++) S[q][t] = mfma16<F16>(a, qf[q][k], S[q][t]);
      }
    }
    if (bits != ~0ull) {
      asm volatile("");   // (a branch: as selections in every tile it costs a third of the softmax)
#pragma unroll
      for (int t = 0; t < 4; t++) {
        const uint32_t on = (uint32_t)(bits >> (16 * t)) >> (4 * g);
#pragma unroll
        for (int q = 0; q < QT; q++)
#pragma unroll
          for (int v = 0; v < 4; v++) S[q][t][v] = on >> v & 1 ? S[q][t][v] : -kInf;
      }
    }
    s16x8 pf[QT][2];
#pragma unroll
    for (int q = 0; q < QT; q++) {
      float mx = -kInf;
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int v = 0; v < 4; v++) mx = fmaxf(mx, S[q][t][v]);
      mx = groups_max(mx);
      if (sm[q].moves(mx, p.c)) {
        const float f = sm[q].move(mx, p.c);
#pragma unroll
        for (int v = 0; v < 4; v++) {
          l4[q][v] *= f;
#pragma unroll
          for (int d = 0; d < DT; d++) O[q][d][v] *= f;
        }
      }
      const float use = sm[q].base();
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
          S[q][t][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[q][t][v], p.c, -use));
          l4[q][v] += S[q][t][v];
        }
      pf[q][0] = operand<F16>(S[q][0], S[q][1]);
      pf[q][1] = operand<F16>(S[q][2], S[q][3]);
    }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int d = 0; d < DT; d++) {
        const s16x8 a = by_columns<DP>(vt[cur], 2 * h, at.col[d]);
#pragma unroll
        for (int q = 0; q < QT; q++) O[q][d] = mfma16<F16>(a, pf[q][h], O[q][d]);
      }
    staged();
    __syncthreads();
    i = j;
  }
#pragma unroll
  for (int q = 0; q < QT; q++) {
    const int r = row0 + 16 * q + l15;
    const float l = groups_sum((l4[q][0] + l4[q][1]) + (l4[q][2] + l4[q][3]));
    const bool on = r < p.rows;
    if (p.splits > 1) {
      // (partial o, its maximum and sum: joined by attn_join_kernel)
      if (!on) continue;
      const int64_t at_row = ((int64_t)split * p.B * p.Hk + pair) * p.rows + r;
      float *o = p.part + at_row * (DP + 2);
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int v = 0; v < 4; v++) o[16 * d + 4 * g + v] = O[q][d][v];
      if (g == 0) o[DP] = l == 0.0f ? -kInf : sm[q].base(), o[DP + 1] = l;
      continue;
    }
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    put_row<F16, DT>(p.out + row_at(p, p.os, b, hk, min(r, p.rows - 1)), p.D, O[q], inv, on);
    if (p.lse && g == 0 && on)
      p.lse[(int64_t)pair * p.rows + r] = l == 0.0f ? kInf : sm[q].base() + __builtin_amdgcn_logf(l);
  }
}

// Requests of unlike lengths: a key head's tiles of 32 keys, entry after entry, dealt out in equal runs to `budget` workgroups
// (of `least` tiles at least; an entry without keys counts as a tile). A run that goes past an entry's end goes on in the next
// entry, and an entry's splits are the runs that meet it. Lane b of a wave holds where entry b begins and ends.
struct Runs {
  uint32_t run, begin, end, all;
  __device__ __forceinline__ explicit Runs(const AttnArgs &p) {
    const int lane = threadIdx.x & 63;
    const uint32_t n = lane < p.B ? max(((uint32_t)min(max(p.lens[lane], 0), p.L) + 31) / 32, 1u) : 0;
    end = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t below = __shfl_up(end, o, 64);
      if (lane >= o) end += below;
    }
    begin = end - n;
    all = __builtin_amdgcn_readlane(end, 63);
    run = max((all + p.budget - 1) / p.budget, (uint32_t)p.least);
  }
  // Of this lane's entry: the first run, and how many.
  __device__ __forceinline__ uint32_t first() const { return begin / run; }
  __device__ __forceinline__ uint32_t count() const { return end > begin ? (end - 1) / run - first() + 1 : 0; }
};

// Up to 16 rows a pair (a token's heads): memory bounds it, k and v once: 8 x 8 pairs over 8191 keys of dimension 128 54 us, 4.95
// TB/s, over up to as many, dealt out in runs, 28 us, 5.1 TB/s; 256 pairs over 4096 of 64 51 us, 5.2 TB/s. Each wave walks keys of
// its own, 32 a step: k goes from memory to the lanes as they multiply it, v through the wave's own staged tile, both requested a
// step ahead; no barrier until the waves' results are joined.
// attn_few: keys of tiles `from` to `to` of a pair, its split-th part.
template <bool F16, int DP>
__device__ __forceinline__ void attn_few(const AttnArgs &p, uint16_t (&vt)[4][32 * DP], float (&joined)[4][16][DP + 4], int b,
                                         int hk, int split, int from, int to) {
  constexpr int KS = DP / 32, DT = DP / 16, kC = DP / 8, kU = 32 * kC / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const int pair = b * p.Hk + hk;
  const Keys keys(p, b);
  const Places<DP> at(lane);
  s16x8 qf[KS];
  const uint16_t *row = p.q + row_at(p, p.qs, b, hk, min(l15, p.rows - 1));
#pragma unroll
  for (int k = 0; k < KS; k++) qf[k] = row_chunk(row, 4 * k + g, p.D, l15 < p.rows);
  f32x4_t O[DT], l4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int d = 0; d < DT; d++) O[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  Softmax sm;
  const uint16_t *kb = p.k + b * p.ks[0] + hk * p.ks[1], *vb = p.v + b * p.vs[0] + hk * p.vs[1];
  const int per = (to - from + 3) / 4, first = from + wave * per, end = min(to, first + per);
  s16x8 K[2][KS], Kn[2][KS];
  u32x4 V[kU];
  const uint16_t *kl = kb + l15 * p.ks[2] + 8 * g, *vl = vb + (lane / kC) * p.vs[2] + 8 * (lane % kC);
  auto fetch = [&](int i, uint32_t bits) {
    if (bits == ~0u && p.D == DP) {   // (whole: loads without conditions, which stay in flight together)
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int k = 0; k < KS; k++)
          Kn[t][k] = *reinterpret_cast<const s16x8 *>(kl + (int64_t)(32 * i + 16 * t) * p.ks[2] + 32 * k);
#pragma unroll
      for (int u = 0; u < kU; u++) V[u] = *reinterpret_cast<const u32x4 *>(vl + (int64_t)(32 * i + 64 / kC * u) * p.vs[2]);
      return;
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int k = 0; k < KS; k++)
        Kn[t][k] = row_chunk(kb + (int64_t)(32 * i + 16 * t + l15) * p.ks[2], 4 * k + g, p.D, bits >> (16 * t + l15) & 1);
#pragma unroll
    for (int u = 0; u < kU; u++) {
      const int w = lane + 64 * u, r = w / kC, c = w % kC;
      V[u] = __builtin_bit_cast(u32x4, row_chunk(vb + (int64_t)(32 * i + r) * p.vs[2], c, p.D, bits >> r & 1));
    }
  };
  auto next = [&](int i, uint32_t &bits) {
    for (; i < end; i++) {
      bits = (uint32_t)__ballot(lane < 32 && keys.valid(32 * i + lane));
      if (bits) return i;
    }
    return end;
  };
  uint32_t bits = 0, nbits = 0;
  int i = next(first, bits);
  if (i < end) fetch(i, bits);
  while (i < end) {
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int k = 0; k < KS; k++) K[t][k] = Kn[t][k];
#pragma unroll
    for (int u = 0; u < kU; u++) {
      const int w = lane + 64 * u, r = w / kC, c = w % kC;
      *reinterpret_cast<u32x4 *>(vt[wave] + r * DP + (c ^ swz<DP>(r)) * 8) = V[u];
    }
    const int j = next(i + 1, nbits);
    if (j < end) fetch(j, nbits);
    f32x4_t S[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
      S[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KS; k++) S[t] = mfma16<F16>(K[t][k], qf[k], S[t]);
    }
    float mx = -kInf;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int v = 0; v < 4; v++) {
        if (!(bits >> (16 * t + 4 * g + v) & 1)) S[t][v] = -kInf;
        mx = fmaxf(mx, S[t][v]);
      }
    mx = groups_max(mx);
    if (sm.moves(mx, p.c)) {
      const float f = sm.move(mx, p.c);
#pragma unroll
      for (int v = 0; v < 4; v++) l4[v] *= f;
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int v = 0; v < 4; v++) O[d][v] *= f;
    }
    const float use = sm.base();
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int v = 0; v < 4; v++) {
        S[t][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[t][v], p.c, -use));
        l4[v] += S[t][v];
      }
    const s16x8 pf = operand<F16>(S[0], S[1]);
#pragma unroll
    for (int d = 0; d < DT; d++) O[d] = mfma16<F16>(by_columns<DP>(vt[wave], 0, at.col[d]), pf, O[d]);
    i = j;
    bits = nbits;
  }
  const float l = groups_sum((l4[0] + l4[1]) + (l4[2] + l4[3]));
#pragma unroll
  for (int d = 0; d < DT; d++)
#pragma unroll
    for (int v = 0; v < 4; v++) joined[wave][l15][16 * d + 4 * g + v] = O[d][v];
  if (g == 0) joined[wave][l15][DP] = l == 0.0f ? -kInf : sm.base(), joined[wave][l15][DP + 1] = l;
  __syncthreads();
  for (int w = threadIdx.x; w < p.rows * DP; w += 256) {
    const int r = w / DP, d = w % DP;
    float m = -kInf, sum = 0.0f, o = 0.0f;
#pragma unroll
    for (int x = 0; x < 4; x++) m = fmaxf(m, joined[x][r][DP]);
#pragma unroll
    for (int x = 0; x < 4; x++) {
      if (joined[x][r][DP] == -kInf) continue;
      const float f = __builtin_amdgcn_exp2f(joined[x][r][DP] - m);
      sum = __builtin_fmaf(f, joined[x][r][DP + 1], sum);
      o = __builtin_fmaf(f, joined[x][r][d], o);
    }
    if (p.splits > 1) {
      float *out = p.part + (((int64_t)split * p.B * p.Hk + pair) * p.rows + r) * (DP + 2);
      out[d] = o;
      if (d == 0) out[DP] = m, out[DP + 1] = sum;
      continue;
    }
    const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
    if (d < p.D) p.out[row_at(p, p.os, b, hk, r) + d] = (uint16_t)pack16<F16>(o * inv, 0.0f);
    if (p.lse && d == 0) p.lse[(int64_t)pair * p.rows + r] = sum == 0.0f ? kInf : m + __builtin_amdgcn_logf(sum);
  }
}

template <bool F16, int DP, bool kRuns>
__global__ __launch_bounds__(256, 2) void attn_few_kernel(AttnArgs p) {
  __shared__ __attribute__((aligned(16))) uint16_t vt[4][32 * DP];
  __shared__ __attribute__((aligned(16))) float joined[4][16][DP + 4];
  const uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  if constexpr (kRuns) {
    const int hk = id / p.budget;
    const Runs runs(p);
    const uint32_t r = id - hk * p.budget, stop = min((r + 1) * runs.run, runs.all);
    for (uint32_t at = r * runs.run; at < stop;) {
      const int b = __builtin_ctzll(__ballot(at < runs.end));
      const uint32_t begin = __builtin_amdgcn_readlane(runs.begin, b),
                     upto = min(stop, (uint32_t)__builtin_amdgcn_readlane(runs.end, b));
      attn_few<F16, DP>(p, vt, joined, b, hk, r - begin / runs.run, at - begin, upto - begin);
      at = upto;
      __syncthreads();
    }
  } else {
    const int pair = id / p.splits, split = id - pair * p.splits, b = pair / p.Hk;
    const int n = (Keys(p, b).len + 31) / 32, per = (n + p.splits - 1) / p.splits;
    attn_few<F16, DP>(p, vt, joined, b, pair - b * p.Hk, split, min(n, split * per), min(n, (split + 1) * per));
  }
}

// The splits' parts of a row, joined in their order, by one wave: lane s holds split s's maximum and factor; the parts' columns are
// read two a lane, eight splits at a time.
template <bool F16, int DP>
__global__ __launch_bounds__(64) void attn_join_kernel(AttnArgs p) {
  const int64_t all = (int64_t)p.B * p.Hk * p.rows, row = blockIdx.x;
  const int lane = threadIdx.x;
  const float *x = p.part + row * (DP + 2);
  const int64_t step = all * (DP + 2);
  float2 ml = lane < p.splits ? *reinterpret_cast<const float2 *>(x + lane * step + DP) : float2{-kInf, 0.0f};
  const int pair = (int)(row / p.rows), r = (int)(row - (int64_t)pair * p.rows), b = pair / p.Hk;
  int splits = p.splits;
  if (p.budget) {
    splits = __builtin_amdgcn_readlane(Runs(p).count(), b);
    if (lane >= splits) ml = float2{-kInf, 0.0f};
  }
  float m = ml.x;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float f = ml.x == -kInf ? 0.0f : __builtin_amdgcn_exp2f(ml.x - m);
  float sum = ml.x == -kInf ? 0.0f : f * ml.y;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  constexpr int kV = DP / 64;   // (columns lane, lane + 64)
  float o[kV];
#pragma unroll
  for (int v = 0; v < kV; v++) o[v] = 0.0f;
  for (int s0 = 0; s0 < splits; s0 += 8) {
    float part[8][kV];
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
      for (int v = 0; v < kV; v++) part[i][v] = x[min(s0 + i, splits - 1) * step + lane + 64 * v];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float fs = __shfl(f, min(s0 + i, 63), 64);
      if (s0 + i < splits && fs != 0.0f) {
#pragma unroll
        for (int v = 0; v < kV; v++) o[v] = __builtin_fmaf(fs, part[i][v], o[v]);
      }
    }
  }
  const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
  uint16_t *out = p.out + row_at(p, p.os, b, pair - b * p.Hk, r);
#pragma unroll
  for (int v = 0; v < kV; v++)
    if (lane + 64 * v < p.D) out[lane + 64 * v] = (uint16_t)pack16<F16>(o[v] * inv, 0.0f);
  if (p.lse && lane == 0) p.lse[row] = sum == 0.0f ? kInf : m + __builtin_amdgcn_logf(sum);
}

// ------------------------------------------------------------------------------------------- backward

// fp16 holds nothing below 2^-24, where the probabilities of long states and their products with small gradients lie: P is held
// 2^10 times itself, and dS times a power of two that brings the gradients' largest row norm (for dq each row's own) to 16 .. 32.
// Exact factors, taken off the fp32 sums again.
constexpr float kPUp = 10.0f;
__device__ __forceinline__ float norm_factor(float norm2) {
  if (!(norm2 > 0.0f) || norm2 == kInf) return 1.0f;
  const int e = (int)((__float_as_uint(__builtin_sqrtf(norm2)) >> 23) & 255) - 127;
  return __builtin_ldexpf(1.0f, min(max(4 - e, -60), 60));
}

// 128 x 16 heads of 256 over up to 320 96 us; 4 x 16 of 1024 over 2048, dimension 128, 100 us, 1.03 PFLOP/s of its three products.
// dq, delta and (fp16) the largest row norm of the workgroup's do; the forward's walk over the keys.
template <bool F16, int DP, int QT>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(AttnArgs p) {
  constexpr int KS = DP / 32, DT = DP / 16;
  __shared__ __attribute__((aligned(16))) uint16_t kt[2][kTile * DP], vt[2][kTile * DP];
  __shared__ float norms[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  const int rt = id % p.tiles, split = id / p.tiles % p.splits, pair = id / p.tiles / p.splits;
  const int b = pair / p.Hk, hk = pair - b * p.Hk;
  const Keys keys(p, b);
  const Places<DP> at(lane);
  const int row0 = rt * 64 * QT + wave * 16 * QT;
  s16x8 qf[QT][KS], df[QT][KS];
  float delta[QT], lse[QT], up[QT];
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < QT; i++) {
    const int r = row0 + 16 * i + l15, rc = min(r, p.rows - 1);
    const bool on = r < p.rows;
    const uint16_t *qr = p.q + row_at(p, p.qs, b, hk, rc), *dr = p.dout + row_at(p, p.ds, b, hk, rc),
                   *orow = p.o + row_at(p, p.os, b, hk, rc);
    float sum = 0.0f, n2 = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; k++) {
      qf[i][k] = row_chunk(qr, 4 * k + g, p.D, on);
      df[i][k] = row_chunk(dr, 4 * k + g, p.D, on);
      float d[8], o[8];
      floats8<F16>(df[i][k], d);
      floats8<F16>(row_chunk(orow, 4 * k + g, p.D, on), o);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        sum = __builtin_fmaf(d[e], o[e], sum);
        if (F16) n2 = __builtin_fmaf(d[e], d[e], n2);
      }
    }
    delta[i] = groups_sum(sum);
    lse[i] = on ? p.lse[(int64_t)pair * p.rows + r] : kInf;
    up[i] = 1.0f;
    if (F16) {
      n2 = groups_sum(n2);
      up[i] = norm_factor(n2);
      most = fmaxf(most, n2);
    }
  }
  if (F16) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    if (lane == 0) norms[wave] = most;
    __syncthreads();
    if (threadIdx.x == 0 && split == 0)
      p.rowmax[pair * (int64_t)p.tiles + rt] = fmaxf(fmaxf(norms[0], norms[1]), fmaxf(norms[2], norms[3]));
  }
  f32x4_t dQ[QT][DT];
#pragma unroll
  for (int i = 0; i < QT; i++)
#pragma unroll
    for (int d = 0; d < DT; d++) dQ[i][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const uint16_t *kb = p.k + b * p.ks[0] + hk * p.ks[1], *vb = p.v + b * p.vs[0] + hk * p.vs[1];
  const int n = (keys.len + kTile - 1) / kTile, per = (n + p.splits - 1) / p.splits;
  const int end = min(n, (split + 1) * per);
  uint64_t bits = 0, nbits = 0;
  int i = keys.next(split * per, end, bits);
  const RowStage<DP> sk(p.ks[2]), sv(p.vs[2]);
  if (i < end) {
    sk.load(kt[0], kb + (int64_t)i * kTile * p.ks[2], bits, p.D);
    sv.load(vt[0], vb + (int64_t)i * kTile * p.vs[2], bits, p.D);
  }
  staged();
  __syncthreads();
  f32x4_t S[QT][2], P[QT][2];
  // P and dP of 32 keys of the tile, from the h-th half
  auto scores = [&](int cur, int h) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
#pragma unroll
      for (int q = 0; q < QT; q++) S[q][t] = P[q][t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const s16x8 a = by_rows<DP>(kt[cur], 2 * h + t, at.row[k]), c = by_rows<DP>(vt[cur], 2 * h + t, at.row[k]);
#pragma unroll
        for (int q = 0; q < QT; q++) {
          S[q][t] = mfma16<F16>(a, qf[q][k], S[q][t]);
          P[q][t] = mfma16<F16>(c, df[q][k], P[q][t]);
        }
      }
    }
    if (bits != ~0ull) {
      asm volatile("");   // (a branch, as in the forward)
      const uint32_t on = (uint32_t)(bits >> (32 * h)) >> (4 * g);
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int q = 0; q < QT; q++)
#pragma unroll
          for (int v = 0; v < 4; v++) S[q][t][v] = on >> (16 * t + v) & 1 ? S[q][t][v] : -kInf;
    }
#pragma unroll
    for (int q = 0; q < QT; q++)
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int v = 0; v < 4; v++) S[q][t][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[q][t][v], p.c, -lse[q]));
  };
  int j = i < end ? keys.next(i + 1, end, nbits) : end;
  if ((p.splits == 1 || n == 1) && i < end && j == end) {
    // One tile alone: delta as the sum of P dP. The few keys' dP are as large as delta, which the rounding of o would move by
    // as much as dS's own rounding does.
#pragma unroll
    for (int q = 0; q < QT; q++) delta[q] = 0.0f;
    for (int h = 0; h < 2; h++) {
      scores(0, h);
#pragma unroll
      for (int q = 0; q < QT; q++)
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int v = 0; v < 4; v++) delta[q] = __builtin_fmaf(S[q][t][v], P[q][t][v], delta[q]);
    }
#pragma unroll
    for (int q = 0; q < QT; q++) delta[q] = groups_sum(delta[q]);
  }
#pragma unroll
  for (int q = 0; q < QT; q++)
    if (g == 0 && split == 0 && row0 + 16 * q + l15 < p.rows) p.delta[(int64_t)pair * p.rows + row0 + 16 * q + l15] = delta[q];
  for (int cur = 0; i < end; cur ^= 1) {
    if (j < end) {
      sk.load(kt[cur ^ 1], kb + (int64_t)j * kTile * p.ks[2], nbits, p.D);
      sv.load(vt[cur ^ 1], vb + (int64_t)j * kTile * p.vs[2], nbits, p.D);
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      scores(cur, h);
      s16x8 sf[QT];
#pragma unroll
      for (int q = 0; q < QT; q++) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int v = 0; v < 4; v++) {
            const float x = S[q][t][v] * (P[q][t][v] - delta[q]);
            S[q][t][v] = F16 ? x * up[q] : x;
          }
        sf[q] = operand<F16>(S[q][0], S[q][1]);
      }
#pragma unroll
      for (int d = 0; d < DT; d++) {
        const s16x8 a = by_columns<DP>(kt[cur], 2 * h, at.col[d]);
#pragma unroll
        for (int q = 0; q < QT; q++) dQ[q][d] = mfma16<F16>(a, sf[q], dQ[q][d]);
      }
    }
    staged();
    __syncthreads();
    i = j, bits = nbits;
    if (i < end) j = keys.next(i + 1, end, nbits);
  }
#pragma unroll
  for (int q = 0; q < QT; q++) {
    const int r = row0 + 16 * q + l15;
    const float f = F16 ? p.scale / up[q] : p.scale;
    if (p.splits > 1) {   // (added by attn_dq_join_kernel)
      if (r >= p.rows) continue;
      float *part = p.part + (((int64_t)split * p.B * p.Hk + pair) * p.rows + r) * p.D;
#pragma unroll
      for (int d = 0; d < DT; d++)
        if (16 * d + 4 * g < p.D)
          *reinterpret_cast<f32x4_t *>(part + 16 * d + 4 * g) =
              f32x4_t{dQ[q][d][0] * f, dQ[q][d][1] * f, dQ[q][d][2] * f, dQ[q][d][3] * f};
      continue;
    }
    put_row<F16, DT>(p.dq + row_at(p, p.dqs, b, hk, min(r, p.rows - 1)), p.D, dQ[q], f, r < p.rows);
  }
}

// 128 x 16 heads of 256 over up to 320 124 us; 4 x 16 of 1024 over 2048, dimension 128, 163 us, 0.84 PFLOP/s of its four
// products: there LDS is read four times for 16 keys a wave, and 32 do not fit the registers.
// dk and dv of 64 KT keys: the waves' k and v stay in registers, the pair's rows (or the split's part of them) pass by in staged
// tiles of q and do. A shared key's gradient sums over its heads here, in a fixed order.
template <bool F16, int DP, int KT>
__global__ __launch_bounds__(256, 2) void attn_dkv_kernel(AttnArgs p) {
  constexpr int KS = DP / 32, DT = DP / 16;
  __shared__ __attribute__((aligned(16))) uint16_t qt[2][kTile * DP], dt[2][kTile * DP];
  __shared__ __attribute__((aligned(16))) float lse[2][kTile], delta[2][kTile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
  const uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  const int kt = id % p.tiles, split = id / p.tiles % p.splits, pair = id / p.tiles / p.splits;
  const int b = pair / p.Hk, hk = pair - b * p.Hk;
  const Keys keys(p, b);
  const Places<DP> at(lane);
  const int key0 = kt * 64 * KT + wave * 16 * KT;
  s16x8 kf[KT][KS], vf[KT][KS];
  bool on[KT];
  bool any = false;
#pragma unroll
  for (int i = 0; i < KT; i++) {
    const int j = key0 + 16 * i + l15;
    on[i] = keys.valid(j);
    any |= on[i];
    const int64_t jc = min(j, p.L - 1);
    const uint16_t *kr = p.k + b * p.ks[0] + hk * p.ks[1] + jc * p.ks[2], *vr = p.v + b * p.vs[0] + hk * p.vs[1] + jc * p.vs[2];
#pragma unroll
    for (int k = 0; k < KS; k++) {
      kf[i][k] = row_chunk(kr, 4 * k + g, p.D, on[i]);
      vf[i][k] = row_chunk(vr, 4 * k + g, p.D, on[i]);
    }
  }
  f32x4_t dK[KT][DT], dV[KT][DT];
#pragma unroll
  for (int i = 0; i < KT; i++)
#pragma unroll
    for (int d = 0; d < DT; d++) dK[i][d] = dV[i][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float up = 1.0f;
  if (F16) {   // (every row tile's largest norm: of the dq kernel's workgroups)
    const int n = p.rtiles;
    float m = 0.0f;
    for (int x = lane; x < n; x += 64) m = fmaxf(m, p.rowmax[pair * (int64_t)n + x]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    up = norm_factor(m);
  }
  // (tiles of a head's rows: one base a tile, where tiles across heads would need an address a row)
  const int nt = (p.N + kTile - 1) / kTile, n = p.G * nt, per = (n + p.splits - 1) / p.splits;
  int i = split * per;
  const int end = __syncthreads_or(any) ? min(n, i + per) : 0;
  const RowStage<DP> sq(p.qs[2]), sd(p.ds[2]);
  float sl = 0.0f;
  auto fetch = [&](int item, int buf) {
    const int h = item / nt, n0 = (item - h * nt) * kTile, rest = p.N - n0;
    const uint64_t rows = rest < kTile ? (1ull << rest) - 1 : ~0ull;
    sq.load(qt[buf], p.q + b * p.qs[0] + (hk * p.G + h) * p.qs[1] + n0 * p.qs[2], rows, p.D);
    sd.load(dt[buf], p.dout + b * p.ds[0] + (hk * p.G + h) * p.ds[1] + n0 * p.ds[2], rows, p.D);
    const int r = threadIdx.x & 63;
    if (threadIdx.x < 128) {
      const float *src = threadIdx.x < 64 ? p.lse : p.delta;
      sl = r < rest ? src[(int64_t)pair * p.rows + h * p.N + n0 + r] : threadIdx.x < 64 ? kInf : 0.0f;
      if (F16 && threadIdx.x < 64) sl -= kPUp;
    }
  };
  auto put = [&](int buf) {
    if (threadIdx.x < 64) lse[buf][threadIdx.x] = sl;
    else if (threadIdx.x < 128) delta[buf][threadIdx.x - 64] = sl;
    staged();
  };
  if (i < end) {
    fetch(i, 0);
    put(0);
  }
  __syncthreads();
  const float us = F16 ? up * __builtin_ldexpf(1.0f, -(int)kPUp) : 1.0f;
  for (int cur = 0; i < end; cur ^= 1, i++) {
    if (i + 1 < end) fetch(i + 1, cur ^ 1);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      f32x4_t S[KT][2], P[KT][2];
#pragma unroll
      for (int t = 0; t < 2; t++) {
#pragma unroll
        for (int x = 0; x < KT; x++) S[x][t] = P[x][t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < KS; k++) {
          const s16x8 a = by_rows<DP>(qt[cur], 2 * h + t, at.row[k]), c = by_rows<DP>(dt[cur], 2 * h + t, at.row[k]);
#pragma unroll
          for (int x = 0; x < KT; x++) {
            S[x][t] = mfma16<F16>(a, kf[x][k], S[x][t]);
            P[x][t] = mfma16<F16>(c, vf[x][k], P[x][t]);
          }
        }
        const f32x4_t ls = *reinterpret_cast<const f32x4_t *>(&lse[cur][32 * h + 16 * t + 4 * g]),
                      de = *reinterpret_cast<const f32x4_t *>(&delta[cur][32 * h + 16 * t + 4 * g]);
#pragma unroll
        for (int x = 0; x < KT; x++)
#pragma unroll
          for (int v = 0; v < 4; v++) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(S[x][t][v], p.c, -ls[v]));
            float d = P[x][t][v] - de[v];
            if (F16) d *= us;
            S[x][t][v] = e;
            P[x][t][v] = e * d;
          }
      }
      s16x8 pf[KT], sf[KT];
#pragma unroll
      for (int x = 0; x < KT; x++) {
        pf[x] = operand<F16>(S[x][0], S[x][1]);
        sf[x] = operand<F16>(P[x][0], P[x][1]);
      }
#pragma unroll
      for (int d = 0; d < DT; d++) {
        const s16x8 a = by_columns<DP>(dt[cur], 2 * h, at.col[d]), c = by_columns<DP>(qt[cur], 2 * h, at.col[d]);
#pragma unroll
        for (int x = 0; x < KT; x++) {
          dV[x][d] = mfma16<F16>(a, pf[x], dV[x][d]);
          dK[x][d] = mfma16<F16>(c, sf[x], dK[x][d]);
        }
      }
    }
    if (i + 1 < end) put(cur ^ 1);
    __syncthreads();
  }
  const float fk = F16 ? p.scale / up : p.scale, fv = F16 ? __builtin_ldexpf(1.0f, -(int)kPUp) : 1.0f;
#pragma unroll
  for (int x = 0; x < KT; x++) {
    const int j = key0 + 16 * x + l15;
    if (p.splits > 1) {
      if (j >= p.L) continue;
      float *o = p.part + (((int64_t)split * p.B * p.Hk + pair) * p.L + j) * 2 * p.D;
#pragma unroll
      for (int d = 0; d < DT; d++)
        if (16 * d + 4 * g < p.D) {
          f32x4_t a, c;
#pragma unroll
          for (int v = 0; v < 4; v++) a[v] = on[x] ? dK[x][d][v] * fk : 0.0f, c[v] = on[x] ? dV[x][d][v] * fv : 0.0f;
          *reinterpret_cast<f32x4_t *>(o + 16 * d + 4 * g) = a;
          *reinterpret_cast<f32x4_t *>(o + p.D + 16 * d + 4 * g) = c;
        }
      continue;
    }
    const int64_t jc = min(j, p.L - 1);
    put_row<F16, DT>(p.dk + b * p.dks[0] + hk * p.dks[1] + jc * p.dks[2], p.D, dK[x], fk, j < p.L, on[x]);
    put_row<F16, DT>(p.dv + b * p.dvs[0] + hk * p.dvs[1] + jc * p.dvs[2], p.D, dV[x], fv, j < p.L, on[x]);
  }
}

// The splits' dq added in their order: a thread four columns of one row.
template <bool F16>
__global__ __launch_bounds__(256) void attn_dq_join_kernel(AttnArgs p) {
  const int q = p.D / 4;
  const int64_t n4 = (int64_t)p.B * p.Hk * p.rows * q, x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x >= n4) return;
  f32x4_t a{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < p.splits; s++) a += *reinterpret_cast<const f32x4_t *>(p.part + 4 * (s * n4 + x));
  const int64_t row = x / q;
  const int c = (int)(x - row * q), pair = (int)(row / p.rows), r = (int)(row - (int64_t)pair * p.rows), b = pair / p.Hk;
  *reinterpret_cast<u32x2 *>(p.dq + row_at(p, p.dqs, b, pair - b * p.Hk, r) + 4 * c) =
      u32x2{pack16<F16>(a[0], a[1]), pack16<F16>(a[2], a[3])};
}

// The splits' dk and dv added in their order: a thread four columns of one key's dk or dv.
template <bool F16>
__global__ __launch_bounds__(256) void attn_dkv_join_kernel(AttnArgs p) {
  const int64_t n4 = (int64_t)p.B * p.Hk * p.L * 2 * (p.D / 4), x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x >= n4) return;
  f32x4_t a{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < p.splits; s++) a += *reinterpret_cast<const f32x4_t *>(p.part + 4 * (s * n4 + x));
  const int q = p.D / 4, c = (int)(x % q);
  int64_t r = x / q;
  const bool v = r & 1;
  r >>= 1;
  const int j = (int)(r % p.L), pair = (int)(r / p.L), b = pair / p.Hk, hk = pair - b * p.Hk;
  const int64_t (&s)[3] = v ? p.dvs : p.dks;
  *reinterpret_cast<u32x2 *>((v ? p.dv : p.dk) + b * s[0] + hk * s[1] + j * s[2] + 4 * c) =
      u32x2{pack16<F16>(a[0], a[1]), pack16<F16>(a[2], a[3])};
}

// ------------------------------------------------------------------------------------------- host side

constexpr int kMaxAttnD = 128;
constexpr float kLog2e = 1.44269504f;
constexpr int kFewRows = 16;
constexpr int kMaxSplits = 64;   // (a wave joins the forward's)
constexpr int64_t kMaxBlocks = int64_t(1) << 23;   // (a launch's threads are counted in 32 bits)

struct AttnPlan {
  bool few;
  int qt, tiles, splits;        // forward: 16-row tiles a wave, row tiles, key splits
  int budget, least;             // few rows of requests of unlike lengths: for Runs; splits is then a pair's most
  int bqt, btiles, bsplits;      // dq: the same
  int kt, ktiles, ksplits;       // dkv: 16-key tiles a wave, key tiles, splits of the rows
};
// Two 16-row tiles a wave where the workgroups still fill the device twice (us, one / two: 128 x 16 heads of 256 over up to 320
// 83 / 73 and dq 101 / 98; 2 x 4 pairs of 8188 rows over 4097, dimension 128, 215 / 155 and 244 / 193); two 16-key tiles for long
// states of dimension 64 (4 x 16 heads of 1024 over 1024 48 / 44; over states of up to 320, whose masked part it doubles,
// 135 / 161, and for 128 the registers do not hold them).
// Keys (dkv: rows) are split while there would be fewer workgroups than CUs: 100 rows of 4 pairs over 4000 keys 51 -> 9.4 + 4.2
// for the join, 320 of one pair over 8000 of dimension 128 170 -> 15 + 4; up to two a CU (32 pairs of 512 over 512, 128: dkv
// 22 -> 20.5 + 9.3) it costs what it gains. Few rows likewise (us, 256 / 512 / 1024 workgroups wanted: 64 pairs over up to 8191
// keys of dimension 128 43 / 46 / 45, 256 over 4096 of 64 51 / 65 / 63 with the join).
// Entries with lengths of their own are dealt out in runs (us with the join, splits or a workgroup for each pair / runs; lengths
// drawn evenly, then all full): 64 pairs over up to 8191 keys of dimension 128 46 / 38, 59 / 59; 256 146 / 128, 196 / 193; 480
// over 4096 136 / 107, 189 / 189; 256 over 4096 of 64 39 / 34, 51 / 55. Not where k and v are small, as going on in the next entry
// takes 4 and the join as much: 256 over 2048 of 64 20 / 21, 128 over 4096 23.8 / 22.2, 27 / 30, 16 of 128 14 / 18.
static AttnPlan attn_plan(bool lens, int64_t B, int64_t H, int64_t Hk, int64_t N, int64_t L, int64_t D) {
  AttnPlan a;
  const int64_t pairs = std::max<int64_t>(B * Hk, 1), rows = H / Hk * N;
  auto splits = [](int64_t blocks, int64_t most) {
    const int64_t want = 256 / std::max<int64_t>(blocks, 1);
    return (int)std::max<int64_t>(std::min<int64_t>(std::min(want, most), kMaxSplits), 1);
  };
  a.few = rows <= kFewRows;
  a.bqt = pairs * ((rows + 127) / 128) >= 512 ? 2 : 1;
  a.btiles = (int)((rows + 64 * a.bqt - 1) / (64 * a.bqt));
  a.bsplits = splits(pairs * a.btiles, (L + 511) / 512);
  a.qt = a.few ? 1 : a.bqt;
  a.tiles = a.few ? 1 : a.btiles;
  a.splits = a.few ? splits(pairs, (L + 255) / 256) : a.bsplits;
  a.budget = a.least = 0;
  if (a.few && lens && B > 1 && B <= 64 && Hk <= 64 && pairs < 512 && pairs * L * D >= (int64_t(3) << 24)) {
    a.budget = (int)(256 / Hk);
    const int64_t n = (L + 31) / 32;
    a.least = (int)std::max<int64_t>((n + kMaxSplits - 3) / (kMaxSplits - 2), 8);
    a.splits = (int)std::min<int64_t>(a.budget, (n - 2) / a.least + 2);   // (an entry may begin and end inside runs)
  }
  a.kt = D <= 64 && L >= 1024 && pairs * ((L + 127) / 128) >= 512 ? 2 : 1;
  a.ktiles = (int)((L + 64 * a.kt - 1) / (64 * a.kt));
  a.ksplits = splits(pairs * a.ktiles, (H / Hk * ((N + 63) / 64) + 3) / 4);
  return a;
}
static int attn_dp(int64_t D) { return D <= 64 ? 64 : 128; }

// The extents' status
static int attn_shape(int dtype, int64_t B, int64_t H, int64_t Hk, int64_t N, int64_t L, int64_t D) {
  if (B < 0 || H <= 0 || Hk <= 0 || N < 0 || L < 0 || D <= 0) return GPIC_EINVAL;
  if (dtype != GPIC_DTYPE_BF16 && dtype != GPIC_DTYPE_F16) return GPIC_EDTYPE;
  if (H % Hk || D % 8 || D > kMaxAttnD) return GPIC_ESHAPE;
  const int64_t most = int64_t(1) << 30;
  if (B > most || H > most || N > most || L > most || H / Hk * N > most || B * H > most) return GPIC_ESHAPE;
  if (B * Hk * ((H / Hk * N + 63) / 64) >= kMaxBlocks || B * Hk * ((L + 63) / 64) >= kMaxBlocks) return GPIC_ESHAPE;
  return GPIC_OK;
}
static int strides_ok(const void *p, const int64_t *s, int64_t (&out)[3]) {
  if (!s) return GPIC_EINVAL;
  for (int i = 0; i < 3; i++) {
    if (s[i] < 0) return GPIC_EINVAL;
    if (s[i] % 8) return GPIC_EALIGN;
    out[i] = s[i];
  }
  return aligned16(p) ? GPIC_OK : GPIC_EALIGN;
}

template <class F>
static void with_attn(int dtype, int64_t D, F f) {
  auto dp = [&](auto f16) {
    if (D <= 64) f(f16, std::integral_constant<int, 64>());
    else f(f16, std::integral_constant<int, 128>());
  };
  if (dtype == GPIC_DTYPE_F16) dp(std::true_type());
  else dp(std::false_type());
}

}  // namespace gpic

using namespace gpic;

extern "C" {

size_t gpic_fp8_attention_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int64_t L, int64_t D) {
  if (attn_shape(GPIC_DTYPE_BF16, B, H, Hk, N, L, D) != GPIC_OK || B * N == 0) return 0;
  const int splits = std::max(attn_plan(false, B, H, Hk, N, L, D).splits, attn_plan(true, B, H, Hk, N, L, D).splits);
  return splits > 1 ? (size_t)splits * B * H * N * (attn_dp(D) + 2) * sizeof(float) : 0;
}

int gpic_fp8_attention(const uint16_t *q, const int64_t *qs, const uint16_t *k, const int64_t *ks, const uint16_t *v,
                       const int64_t *vs, int dtype, const int *lens, const uint8_t *mask, int64_t ldm, int64_t B, int64_t H,
                       int64_t Hk, int64_t N, int64_t L, int64_t D, float scale, uint16_t *o, const int64_t *os, float *lse,
                       void *ws, size_t ws_bytes, void *stream) {
  status_scope();
  int e = attn_shape(dtype, B, H, Hk, N, L, D);
  if (e != GPIC_OK) return e;
  if (!(scale > 0.0f) || scale * kLog2e == kInf) return GPIC_EINVAL;
  if (B * N == 0) return GPIC_OK;
  if (!q || !o || (L > 0 && (!k || !v)) || (mask && ldm < 0)) return GPIC_EINVAL;
  AttnArgs p{};
  if ((e = strides_ok(q, qs, p.qs)) || (e = strides_ok(k, ks, p.ks)) || (e = strides_ok(v, vs, p.vs)) ||
      (e = strides_ok(o, os, p.os)))
    return e;
  if (!aligned16(ws)) return GPIC_EALIGN;
  if (ws_bytes < gpic_fp8_attention_workspace_bytes(B, H, Hk, N, L, D)) return GPIC_EWORKSPACE;
  const AttnPlan a = attn_plan(lens != nullptr, B, H, Hk, N, L, D);
  if (a.splits > 1 && !ws) return GPIC_EWORKSPACE;
  p.q = q, p.k = k, p.v = v, p.out = o, p.lens = lens, p.mask = mask, p.ldm = ldm, p.lse = lse;
  p.part = static_cast<float *>(ws);
  p.B = (int)B, p.H = (int)H, p.Hk = (int)Hk, p.N = (int)N, p.L = (int)L, p.D = (int)D, p.G = (int)(H / Hk);
  p.rows = p.G * p.N, p.tiles = a.tiles, p.splits = a.splits, p.scale = scale, p.c = scale * kLog2e;
  const hipStream_t st = (hipStream_t)stream;
  p.budget = a.budget, p.least = a.least;
  const unsigned grid = (unsigned)(a.budget ? Hk * a.budget : B * Hk * a.tiles * a.splits);
  with_attn(dtype, D, [&](auto f, auto dp) {
    constexpr bool F = decltype(f)::value;
    constexpr int DP = decltype(dp)::value;
    if (a.few && a.budget) attn_few_kernel<F, DP, true><<<grid, 256, 0, st>>>(p);
    else if (a.few) attn_few_kernel<F, DP, false><<<grid, 256, 0, st>>>(p);
    else if (a.qt == 2) attn_fwd_kernel<F, DP, 2><<<grid, 256, 0, st>>>(p);
    else attn_fwd_kernel<F, DP, 1><<<grid, 256, 0, st>>>(p);
    if (a.splits > 1) attn_join_kernel<F, DP><<<(unsigned)(B * Hk * p.rows), 64, 0, st>>>(p);
  });
  return (int)hipGetLastError();
}

// delta, the row tiles' largest norms, the splits' parts of dq, then of dk and dv: bytes before each, and of all
struct AttnBwdSpace {
  size_t rowmax, part, all;
};
static AttnBwdSpace attn_bwd_space(const AttnPlan &a, int64_t B, int64_t H, int64_t Hk, int64_t N, int64_t L, int64_t D) {
  auto up = [](size_t n) { return (n + 255) & ~size_t(255); };
  AttnBwdSpace s;
  s.rowmax = up((size_t)B * H * N * sizeof(float));
  s.part = s.rowmax + up((size_t)B * Hk * a.btiles * sizeof(float));
  // (dq's parts are joined before dk's and dv's are written: one place)
  s.all = s.part + std::max(a.bsplits > 1 ? (size_t)a.bsplits * B * H * N * D * sizeof(float) : 0,
                            a.ksplits > 1 ? (size_t)a.ksplits * B * Hk * L * 2 * D * sizeof(float) : 0);
  return s;
}

size_t gpic_fp8_attention_bwd_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t N, int64_t L, int64_t D) {
  if (attn_shape(GPIC_DTYPE_BF16, B, H, Hk, N, L, D) != GPIC_OK) return 0;
  return attn_bwd_space(attn_plan(false, B, H, Hk, N, L, D), B, H, Hk, N, L, D).all;
}

int gpic_fp8_attention_bwd(const uint16_t *dout, const int64_t *ds, const uint16_t *q, const int64_t *qs, const uint16_t *k,
                           const int64_t *ks, const uint16_t *v, const int64_t *vs, const uint16_t *o, const int64_t *os,
                           const float *lse, int dtype, const int *lens, const uint8_t *mask, int64_t ldm, int64_t B, int64_t H,
                           int64_t Hk, int64_t N, int64_t L, int64_t D, float scale, uint16_t *dq, const int64_t *dqs,
                           uint16_t *dk, const int64_t *dks, uint16_t *dv, const int64_t *dvs, void *ws, size_t ws_bytes,
                           void *stream) {
  status_scope();
  int e = attn_shape(dtype, B, H, Hk, N, L, D);
  if (e != GPIC_OK) return e;
  if (!(scale > 0.0f) || scale * kLog2e == kInf) return GPIC_EINVAL;
  if (!dk != !dv) return GPIC_EINVAL;
  const bool rows = B * N > 0, keys = B * L > 0;
  if (!rows && !keys) return GPIC_OK;
  if ((rows && (!q || !dout || !o || !lse || !dq)) || (keys && (!k || !v)) || (mask && ldm < 0)) return GPIC_EINVAL;
  AttnArgs p{};
  if ((e = strides_ok(dout, ds, p.ds)) || (e = strides_ok(q, qs, p.qs)) || (e = strides_ok(k, ks, p.ks)) ||
      (e = strides_ok(v, vs, p.vs)) || (e = strides_ok(o, os, p.os)) || (e = strides_ok(dq, dqs, p.dqs)) ||
      (dk && ((e = strides_ok(dk, dks, p.dks)) || (e = strides_ok(dv, dvs, p.dvs)))))
    return e;
  if (!aligned16(ws)) return GPIC_EALIGN;
  const AttnPlan a = attn_plan(false, B, H, Hk, N, L, D);
  const AttnBwdSpace space = attn_bwd_space(a, B, H, Hk, N, L, D);
  if (ws_bytes < space.all || (space.all && !ws)) return GPIC_EWORKSPACE;
  p.q = q, p.k = k, p.v = v, p.o = o, p.dout = dout, p.dq = dq, p.dk = dk, p.dv = dv, p.lens = lens, p.mask = mask, p.ldm = ldm;
  p.lse = const_cast<float *>(lse);
  char *w = static_cast<char *>(ws);
  p.delta = reinterpret_cast<float *>(w), p.rowmax = reinterpret_cast<float *>(w + space.rowmax);
  p.part = reinterpret_cast<float *>(w + space.part);
  p.B = (int)B, p.H = (int)H, p.Hk = (int)Hk, p.N = (int)N, p.L = (int)L, p.D = (int)D, p.G = (int)(H / Hk);
  p.rows = p.G * p.N, p.scale = scale, p.c = scale * kLog2e, p.rtiles = a.btiles;
  const hipStream_t st = (hipStream_t)stream;
  with_attn(dtype, D, [&](auto f, auto dp) {
    constexpr bool F = decltype(f)::value;
    constexpr int DP = decltype(dp)::value;
    if (rows) {
      p.tiles = a.btiles, p.splits = a.bsplits;
      const unsigned grid = (unsigned)(B * Hk * a.btiles * a.bsplits);
      if (a.bqt == 2) attn_dq_kernel<F, DP, 2><<<grid, 256, 0, st>>>(p);
      else attn_dq_kernel<F, DP, 1><<<grid, 256, 0, st>>>(p);
      if (a.bsplits > 1) attn_dq_join_kernel<F><<<(unsigned)((B * H * N * (D / 4) + 255) / 256), 256, 0, st>>>(p);
    }
    if (keys && dk) {
      p.tiles = a.ktiles, p.splits = a.ksplits;
      const unsigned grid = (unsigned)(B * Hk * a.ktiles * a.ksplits);
      if (a.kt == 2) attn_dkv_kernel<F, DP, 2><<<grid, 256, 0, st>>>(p);
      else attn_dkv_kernel<F, DP, 1><<<grid, 256, 0, st>>>(p);
      if (a.ksplits > 1)
        attn_dkv_join_kernel<F><<<(unsigned)((B * Hk * L * (D / 2) + 255) / 256), 256, 0, st>>>(p);
    }
  });
  return (int)hipGetLastError();
}

}  // extern "C"
