// Softmax attention with products in fp32: the kernels of 4-byte elements (and of 2-byte elements whose rows lie too far apart for
// the kernels of those).
//
// A wave keeps 16 or 32 rows (dk, dv: keys) and goes through what they meet in tiles of 16 that it loads from memory straight into
// registers: nothing is staged in LDS, and no wave waits for another before the end.  That works because a product of 16 x 16 x 4
// adds over four numbers, one per lane group, and does not mind which ones.  Of a tile that is contracted over its columns (S, dP)
// lane l takes row l % 16 and columns 16 j + 4 (l / 16) .. + 3; of one that is contracted over its rows (o, dq, dk, dv) rows
// 4 (l / 16) + e and columns 64 x + 4 (l % 16) .. + 3: both 16 bytes per load, and the accumulator of S, whose lane holds rows
// 4 (l / 16) + e of column l % 16, is the other operand of the second product as it stands.
//
// Bound: the fp32 matrix rate.  The waves of a work-group share its rows and take every KW-th tile, since short calls have few
// rows and many tiles; their sums are joined in LDS in the order of the waves.  2 x 4096 tokens, 16 heads on 4 of 64, causal: forward
// 0.70 ms, 98 TFLOP/s (a large product of this type reaches 154), backward 2.31 ms, 104 TFLOP/s with the scores formed twice.  2 x
// 1000 tokens, 4 heads on 2: 22 and 88 us.  (64 rows against 64, every operand staged in LDS: 0.89, 3.40 ms, 80 and 304 us.)
// 8 waves on the rows of a strip: 2 to 5 % more; tiles loaded two steps ahead: 3 % more.
#pragma once
#include "lmoe_attn_bwd.hpp"

namespace lmoe {

template <typename T> __device__ __forceinline__ f32x4 load4(const T* p) {
  const typename ET<T>::vec4 x = *(const typename ET<T>::vec4*)p;
  return f32x4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
}
// the two lane groups of 16 (of each half), then the two halves
__device__ __forceinline__ void pairs16(float x, float& a, float& b) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const u32x2 y = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  a = __builtin_bit_cast(float, (uint32_t)y[0]); b = __builtin_bit_cast(float, (uint32_t)y[1]);
}
__device__ __forceinline__ float column_max(float x) { float a, b; pairs16(x, a, b); return both_max(fmaxf(a, b)); }
__device__ __forceinline__ float column_sum(float x) { float a, b; pairs16(x, a, b); return both_sum(a + b); }

// of a tile of 16 rows, the lane's numbers: contracted over the columns
template <int W> struct ByCols {
  f32x4 x[W / 16];
  template <typename T> __device__ __forceinline__ void load(const T* row, int D, int g) {      // row: l % 16 of the tile
#pragma unroll
    for (int j = 0; j < W / 16; ++j) {
      const int c = 16 * j + 4 * g;
      x[j] = load4(row + (c < D ? c : 0));
      if (c >= D) x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
};
// ... contracted over the rows
template <int W> struct ByRows {
  f32x4 x[W / 64][4];
  template <typename T> __device__ __forceinline__ void load(const T* m, int64_t stride, int r0, int last, int D, int l) {   // rows r0 .. (none behind last)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int b = 0; b < W / 64; ++b) {
        const int c = 64 * b + 4 * (l & 15);
        x[b][e] = load4(m + (int64_t)min(r0 + 4 * (l >> 4) + e, last) * stride + (c < D ? c : 0));
        if (c >= D) x[b][e] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
  }
};
// acc (lane: row of y l % 16, rows of x 4 (l / 16) + e) += x y^T
template <int W> __device__ __forceinline__ f32x4 by_cols(const ByCols<W>& x, const ByCols<W>& y, f32x4 acc) {
#pragma unroll
  for (int j = 0; j < W / 16; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x[j][e], y.x[j][e], acc, 0, 0, 0);
  return acc;
}
// acc[b][d] (lane: column of p l % 16, columns 64 b + 4 (4 (l / 16) + e) + d of x) += x^T p
template <int W> __device__ __forceinline__ void by_rows(f32x4 (&acc)[W / 64][4], const ByRows<W>& x, f32x4 p) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int b = 0; b < W / 64; ++b)
#pragma unroll
      for (int d = 0; d < 4; ++d) acc[b][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x[b][e][d], p[e], acc[b][d], 0, 0, 0);
}
template <int W> __device__ __forceinline__ void zero_sums(f32x4 (&acc)[W / 64][4]) {
#pragma unroll
  for (int b = 0; b < W / 64; ++b)
#pragma unroll
    for (int d = 0; d < 4; ++d) acc[b][d] = f32x4{0.f, 0.f, 0.f, 0.f};
}
// such sums to row l % 16 of a tile of LDS
template <int W> __device__ __forceinline__ void put_sums(const f32x4 (&acc)[W / 64][4], float* row, int l) {
#pragma unroll
  for (int b = 0; b < W / 64; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) *(f32x4*)(row + 64 * b + 16 * (l >> 4) + 4 * e) = f32x4{acc[b][0][e], acc[b][1][e], acc[b][2][e], acc[b][3][e]};
}

constexpr int ANY_WAVES = 4;         // that share a strip of rows
constexpr int ANY_KV_WAVES = 8;      // ... of keys

template <typename T, int W, int RB, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * ANY_WAVES, 2) void k_attn_fwd_any(const lmoe_attn_args a, int fold) {
  constexpr int KW = ANY_WAVES, LD = W + 4;
  __shared__ __attribute__((aligned(16))) float s_o[KW][16 * RB][LD];
  __shared__ float s_m[KW][16 * RB], s_sum[KW][16 * RB];
  zero_behind<T>(a, a.o, a.HQ, a.V);
  AttnTile t;
  int h;
  if (!attn_place<CH, 16 * RB>(a, a.HQ, true, h, t, fold)) return;
  const int hk = h / (a.HQ / a.HKV), l = lane_id(), w = wave_id(), g = l >> 4, last = t.len - 1;
  const Score<CAP, BIAS, false> sc(a, h);
  const int end = a.causal ? min(t.len, max(t.r0 + 16 * RB, t.prefix)) : t.len, whole = a.causal ? min(t.len, max(t.r0 + 1, t.prefix)) : t.len;
  const T* kp = attn_row<T>(a.k, t.b, t.tok0, hk);
  const T* vp = attn_row<T>(a.v, t.b, t.tok0, hk);
  ByCols<W> q[RB], k;
  f32x4 o[RB][W / 64][4];
  int row[RB], sees[RB];                                           // sees: keys that the row sees
  float m[RB], sum[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    row[r] = t.r0 + 16 * r + (l & 15);
    sees[r] = a.causal ? min(t.len, max(row[r] + 1, t.prefix)) : t.len;
    q[r].load(attn_row<T>(a.q, t.b, t.tok0 + min(row[r], last), h), a.K, g);
    zero_sums<W>(o[r]);
    m[r] = M_LOW;
    sum[r] = 0.f;
  }
  auto keys = [&](int j0) { k.load(kp + (int64_t)min(j0 + (l & 15), last) * a.k.st, a.K, g); };
  keys(16 * w);
  for (int j0 = 16 * w; j0 < end; j0 += 16 * KW) {
    ByRows<W> v;
    v.load(vp, a.v.st, j0, last, a.V, l);
    f32x4 s[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) s[r] = by_cols<W>(k, q[r], f32x4{0.f, 0.f, 0.f, 0.f});
    keys(j0 + 16 * KW);                                            // (of the next step, under the rest of this one)
    const bool part = j0 + 16 > whole;                             // some of the tile's keys are hidden from some rows
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[r][e] = sc.of(s[r][e], CAP ? sc.squash(s[r][e]) : 0.f, (float)(row[r] - j0 - 4 * g - e));
        if (part) s[r][e] = e < sees[r] - j0 - 4 * g ? s[r][e] : -INFINITY;
        mx = fmaxf(mx, s[r][e]);
      }
      const float next = fmaxf(m[r], column_max(mx)), f = pow2(m[r] - next);
      m[r] = next;
      float part = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[r][e] = pow2(s[r][e] - next);
        part += s[r][e];
      }
      sum[r] = sum[r] * f + part;
#pragma unroll
      for (int b = 0; b < W / 64; ++b)
#pragma unroll
        for (int d = 0; d < 4; ++d) o[r][b][d] *= f;
    }
    if (part) {
      // A product with 0 for what the mask hides would make NaN of a hidden NaN or infinity: such numbers are left out here, and reach the
      // rows that see them by themselves.
      bool finite = true;
#pragma unroll
      for (int c = 0; c < W / 64; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const bool ok = fabsf(v.x[c][e][d]) < INFINITY;
            finite &= ok;
            v.x[c][e][d] = ok ? v.x[c][e][d] : 0.f;
          }
      if (__any(!finite))
        for (int j = j0; j < min(j0 + 16, t.len); ++j)
#pragma unroll
          for (int c = 0; c < W / 64; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int col = 64 * c + 16 * g + 4 * e;
              const f32x4 x = load4(vp + (int64_t)j * a.v.st + (col < a.V ? col : 0));
#pragma unroll
              for (int r = 0; r < RB; ++r)
#pragma unroll
                for (int d = 0; d < 4; ++d) o[r][c][d][e] += j < sees[r] && col < a.V && !(fabsf(x[d]) < INFINITY) ? x[d] : 0.f;
            }
    }
#pragma unroll
    for (int r = 0; r < RB; ++r) by_rows<W>(o[r], v, s[r]);
  }
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const float all = column_sum(sum[r]);
    put_sums<W>(o[r], s_o[w][16 * r + (l & 15)], l);
    if (g == 0) { s_m[w][16 * r + l] = m[r]; s_sum[w][16 * r + l] = all; }
  }
  __syncthreads();
  for (int r = threadIdx.x >> 4; r < min(16 * RB, t.len - t.r0); r += 4 * KW) {
    float f[KW], all = 0.f, top = M_LOW;
#pragma unroll
    for (int i = 0; i < KW; ++i) top = fmaxf(top, s_m[i][r]);
#pragma unroll
    for (int i = 0; i < KW; ++i) { f[i] = pow2(s_m[i][r] - top); all += s_sum[i][r] * f[i]; }
    const int c0 = 4 * (threadIdx.x & 15);
    if (a.lse && c0 == 0) a.lse[((int64_t)t.b * a.HQ + h) * a.T + t.tok0 + t.r0 + r] = top + __builtin_amdgcn_logf(all);
    T* const out = attn_row<T>(a.o, t.b, t.tok0 + t.r0 + r, h);
    const float inv = 1.0f / all;
    for (int c = c0; c < a.V; c += 64) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KW; ++i) x += *(const f32x4*)&s_o[i][r][c] * f[i];
      store4(out + c, x * inv);
      if constexpr (sizeof(T) == 2) {
        uint32_t z = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) z |= low_byte(x[e] * inv) << 8 * e;
        if (a.o_low) *(uint32_t*)(a.o_low + (((int64_t)t.b * a.HQ + h) * a.T + t.tok0 + t.r0 + r) * a.V + c) = z;
      }
    }
  }
}

// the sums of the waves' rows, times mul, to rows [0, nvalid) of dst
template <typename T, int KW, int ROWS, int LD> __device__ __forceinline__ void join_rows(const float (&sums)[KW][ROWS][LD], int off, float mul, T* dst, int64_t stride, int nvalid, int D) {
  for (int r = threadIdx.x >> 4; r < min(nvalid, ROWS); r += 4 * KW)
    for (int c = 4 * (threadIdx.x & 15); c < D; c += 64) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KW; ++i) x += *(const f32x4*)&sums[i][r][off + c];
      store4(dst + (int64_t)r * stride + c, x * mul);
    }
}

// dq of a strip of rows; delta of those rows beside it
template <typename T, int W, int RB, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * ANY_WAVES, 2) void k_attn_bwd_dq_any(const lmoe_attn_args a, int fold) {
  constexpr int KW = ANY_WAVES, LD = W + 4;
  __shared__ __attribute__((aligned(16))) float s_dq[KW][16 * RB][LD];
  zero_behind<T>(a, a.dq, a.HQ, a.K);
  AttnTile t;
  int h;
  if (!attn_place<CH, 16 * RB>(a, a.HQ, true, h, t, fold)) return;
  const int hk = h / (a.HQ / a.HKV), l = lane_id(), w = wave_id(), g = l >> 4, last = t.len - 1;
  const Score<CAP, BIAS, false> sc(a, h);
  const int end = a.causal ? min(t.len, max(t.r0 + 16 * RB, t.prefix)) : t.len, whole = a.causal ? min(t.len, max(t.r0 + 1, t.prefix)) : t.len;
  const T* kp = attn_row<T>(a.k, t.b, t.tok0, hk);
  const T* vp = attn_row<T>(a.v, t.b, t.tok0, hk);
  ByCols<W> q[RB], d_o[RB], k, v;
  f32x4 dq[RB][W / 64][4];
  int row[RB], sees[RB];
  float lse[RB], delta[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    row[r] = t.r0 + 16 * r + (l & 15);
    sees[r] = a.causal ? min(t.len, max(row[r] + 1, t.prefix)) : t.len;
    const int rc = min(row[r], last);
    q[r].load(attn_row<T>(a.o, t.b, t.tok0 + rc, h), a.V, g);
    d_o[r].load(attn_row<T>(a.d_o, t.b, t.tok0 + rc, h), a.V, g);
    const int64_t at = ((int64_t)t.b * a.HQ + h) * a.T + t.tok0 + rc;
    float d = 0.f;
#pragma unroll
    for (int j = 0; j < W / 16; ++j) {
      uint32_t low = 0;
      if (sizeof(T) == 2 && a.o_low && 16 * j + 4 * g < a.V) low = *(const uint32_t*)(a.o_low + at * a.V + 16 * j + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float o = sizeof(T) == 2 ? with_low((bf16)q[r].x[j][e], low, e) : q[r].x[j][e];
        d = __builtin_fmaf(o, d_o[r].x[j][e], d);
      }
    }
    delta[r] = column_sum(d);
    lse[r] = a.lse[at];
    if (w == 0 && g == 0 && row[r] < t.len) a.delta[at] = delta[r];
    q[r].load(attn_row<T>(a.q, t.b, t.tok0 + rc, h), a.K, g);
    zero_sums<W>(dq[r]);
  }
  auto keys = [&](int j0) {
    const int64_t j = min(j0 + (l & 15), last);
    k.load(kp + j * a.k.st, a.K, g);
    v.load(vp + j * a.v.st, a.V, g);
  };
  keys(16 * w);
  for (int j0 = 16 * w; j0 < end; j0 += 16 * KW) {
    ByRows<W> kr;
    kr.load(kp, a.k.st, j0, last, a.K, l);
    f32x4 s[RB], dp[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      s[r] = by_cols<W>(k, q[r], f32x4{0.f, 0.f, 0.f, 0.f});
      dp[r] = by_cols<W>(v, d_o[r], f32x4{0.f, 0.f, 0.f, 0.f});
    }
    keys(j0 + 16 * KW);
    const bool part = j0 + 16 > whole;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float th = CAP ? sc.squash(s[r][e]) : 0.f;
        float ds = pow2(sc.of(s[r][e], th, (float)(row[r] - j0 - 4 * g - e)) - lse[r]) * (dp[r][e] - delta[r]);
        if constexpr (CAP) ds *= 1.0f - th * th;
        s[r][e] = ds;
        if (part) s[r][e] = e < sees[r] - j0 - 4 * g ? ds : 0.f;
      }
      by_rows<W>(dq[r], kr, s[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < RB; ++r) put_sums<W>(dq[r], s_dq[w][16 * r + (l & 15)], l);
  __syncthreads();
  join_rows<T>(s_dq, 0, a.scale, attn_row<T>(a.dq, t.b, t.tok0 + t.r0, h), a.dq.st, t.len - t.r0, a.K);
}

// dk, dv of a strip of keys, over the rows of all query heads that share the key head.  parts > 1: that many work-groups share them, and
// leave fp32 sums for k_attn_join.
template <typename T, int W, int KB, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * ANY_KV_WAVES, 2) void k_attn_bwd_dkv_any(const lmoe_attn_args a, int fold, int parts) {
  constexpr int KW = ANY_KV_WAVES, LD = 2 * W + 4;
  __shared__ __attribute__((aligned(16))) float s_sum[KW][16 * KB][LD];
  if (blockIdx.y == 0) {
    zero_behind<T>(a, a.dk, a.HKV, a.K);
    zero_behind<T>(a, a.dv, a.HKV, a.V);
  }
  AttnTile t;
  int hk;
  if (!attn_place<CH, 16 * KB>(a, a.HKV, false, hk, t, fold)) return;
  const int G = a.HQ / a.HKV, l = lane_id(), w = wave_id(), g = l >> 4, last = t.len - 1;
  const int begin = a.causal && t.r0 >= t.prefix ? t.r0 : 0, tiles = (t.len - begin + 15) / 16;
  const int whole = a.causal && t.r0 + 16 * KB > t.prefix ? t.r0 + 16 * KB - 1 : 0;        // from it on rows see all keys of the strip
  ByCols<W> k[KB], v[KB], q, d_o;
  f32x4 dk[KB][W / 64][4], dv[KB][W / 64][4];
  int key[KB], from[KB];                                           // from: rows that see the key begin here
#pragma unroll
  for (int b = 0; b < KB; ++b) {
    key[b] = t.r0 + 16 * b + (l & 15);
    from[b] = a.causal && key[b] >= t.prefix ? key[b] : 0;
    const int kc = min(key[b], last);
    k[b].load(attn_row<T>(a.k, t.b, t.tok0 + kc, hk), a.K, g);
    v[b].load(attn_row<T>(a.v, t.b, t.tok0 + kc, hk), a.V, g);
    zero_sums<W>(dk[b]);
    zero_sums<W>(dv[b]);
  }
  // The stream: the tiles of a head, head by head.  Of the parts' waves each takes every so many-th (behind the last: one of the last head,
  // unused).
  const int stride = KW * parts, mine = blockIdx.y * KW + w;
  int x = mine % tiles, h = mine / tiles;
  float lse[4], delta[4];
  auto rows = [&] {
    const int hq = hk * G + min(h, G - 1), i0 = begin + 16 * x;
    const int64_t r = t.tok0 + min(i0 + (l & 15), last), at = ((int64_t)t.b * a.HQ + hq) * a.T + t.tok0;
    q.load(attn_row<T>(a.q, t.b, 0, hq) + r * a.q.st, a.K, g);
    d_o.load(attn_row<T>(a.d_o, t.b, 0, hq) + r * a.d_o.st, a.V, g);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = min(i0 + 4 * g + e, last);
      lse[e] = a.lse[at + i];
      delta[e] = a.delta[at + i];
    }
  };
  rows();
  while (h < G) {
    const int hq = hk * G + h, i0 = begin + 16 * x;
    const Score<CAP, BIAS, false> sc(a, hq);
    ByRows<W> y, z;
    y.load(attn_row<T>(a.d_o, t.b, t.tok0, hq), a.d_o.st, i0, last, a.V, l);
    f32x4 p[KB], ds[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      p[b] = by_cols<W>(q, k[b], f32x4{0.f, 0.f, 0.f, 0.f});
      ds[b] = by_cols<W>(d_o, v[b], f32x4{0.f, 0.f, 0.f, 0.f});
    }
    z.load(attn_row<T>(a.q, t.b, t.tok0, hq), a.q.st, i0, last, a.K, l);
    const bool part = i0 + 16 > t.len || i0 < whole;
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + 4 * g + e;
        const bool ok = !part || (i < t.len && i >= from[b]);
        const float th = CAP ? sc.squash(p[b][e]) : 0.f;
        p[b][e] = ok ? pow2(sc.of(p[b][e], th, (float)(i - key[b])) - lse[e]) : 0.f;
        float d = p[b][e] * (ds[b][e] - delta[e]);
        if constexpr (CAP) d *= 1.0f - th * th;
        ds[b][e] = ok ? d : 0.f;
      }
    for (x += stride; x >= tiles && h < G; x -= tiles) ++h;
    rows();                                                        // (of the next step, under the rest of this one)
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      by_rows<W>(dv[b], y, p[b]);
      by_rows<W>(dk[b], z, ds[b]);
    }
  }
#pragma unroll
  for (int b = 0; b < KB; ++b) {
    put_sums<W>(dk[b], s_sum[w][16 * b + (l & 15)], l);
    put_sums<W>(dv[b], s_sum[w][16 * b + (l & 15)] + W, l);
  }
  __syncthreads();
  const int n = t.len - t.r0;
  if (parts == 1) {
    join_rows<T>(s_sum, 0, a.scale, attn_row<T>(a.dk, t.b, t.tok0 + t.r0, hk), a.dk.st, n, a.K);
    join_rows<T>(s_sum, W, 1.0f, attn_row<T>(a.dv, t.b, t.tok0 + t.r0, hk), a.dv.st, n, a.V);
  } else {
    const int64_t D = a.K + a.V, row = ((int64_t)blockIdx.y * a.B * a.T + (int64_t)t.b * a.T + t.tok0 + t.r0) * a.HKV + hk;
    join_rows<float>(s_sum, 0, a.scale, a.ws + row * D, a.HKV * D, n, a.K);
    join_rows<float>(s_sum, W, 1.0f, a.ws + row * D + a.K, a.HKV * D, n, a.V);
  }
}

}  // namespace lmoe
