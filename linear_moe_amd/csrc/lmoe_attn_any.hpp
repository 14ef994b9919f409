// Softmax attention, the kernels for any element type: 64 rows against 64 rows, four waves of 16 rows, every operand of a
// product in LDS.  The path of 4-byte elements.
#pragma once
#include "lmoe_attn.hpp"

namespace lmoe {

// tile[64][LD] = rows [0, nvalid) of a matrix with D <= W columns, the rest zero.  Returns whether the thread saw a number that
// is not finite.
template <typename T, int W> __device__ __forceinline__ bool attn_load(T* tile, const T* src, int64_t stride, int nvalid, int D) {
  constexpr int VEC = ET<T>::VEC, VPR = W / VEC, LD = W + LPAD;
  typedef typename ET<T>::vec vec;
  bool odd = false;
#pragma unroll
  for (int p = 0; p < CH * VPR / NTHR; ++p) {
    const int idx = p * NTHR + threadIdx.x, r = idx / VPR, c = idx % VPR * VEC;
    vec x = ET<T>::zero();
    if (r < nvalid && c < D) x = *(const vec*)(src + (int64_t)r * stride + c);
    *(vec*)(tile + r * LD + c) = x;
#pragma unroll
    for (int i = 0; i < VEC; ++i) odd |= !(fabsf(ET<T>::to_f(x[i])) < INFINITY);
  }
  return odd;
}
// 16 rows of a wave's accumulators, times mul, to rows [0, nvalid) and columns [0, D) of dst
template <typename T, int NB> __device__ __forceinline__ void attn_store(const f32x4 (&acc)[1][NB], T* dst, int64_t stride, int nvalid, int D, const float (&mul)[4]) {
  const int l = lane_id();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * (l >> 4) + i;
#pragma unroll
    for (int ni = 0; ni < NB; ++ni) {
      const int c = 16 * ni + (l & 15);
      if (r < nvalid && c < D) dst[(int64_t)r * stride + c] = ET<T>::from_f(acc[0][ni][i] * mul[i]);
    }
  }
}
template <typename T, int W, bool CAP, bool BIAS>
__global__ __launch_bounds__(NTHR) void k_attn_fwd_any(const lmoe_attn_args a) {
  constexpr int LD = W + LPAD, PLD = CH + LPAD, NB = W / 16;
  __shared__ __attribute__((aligned(16))) T s_q[CH * LD], s_k[CH * LD], s_v[CH * LD], s_p[CH * PLD];
  zero_behind<T>(a, a.o, a.HQ, a.V);
  AttnTile t;
  int h;
  if (!attn_place<CH>(a, a.HQ, true, h, t)) return;
  const int hk = h / (a.HQ / a.HKV);
  const Score<CAP, BIAS, false> sc(a, h);
  const int l = lane_id(), w = wave_id(), row = t.r0 + 16 * w + 4 * (l >> 4);
  const int rows = min(CH, t.len - t.r0);
  attn_load<T, W>(s_q, attn_row<T>(a.q, t.b, t.tok0 + t.r0, h), a.q.st, rows, a.K);
  f32x4 o[1][NB];
  acc_zero(o);
  float m[4], sum[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { m[i] = M_LOW; sum[i] = 0.f; }
  const int end = a.causal ? min(t.len, max(t.r0 + CH, t.prefix)) : t.len;
  for (int j0 = 0; j0 < end; j0 += CH) {
    const int keys = min(CH, t.len - j0);
    __syncthreads();
    attn_load<T, W>(s_k, attn_row<T>(a.k, t.b, t.tok0 + j0, hk), a.k.st, keys, a.K);
    const bool odd = __syncthreads_or(attn_load<T, W>(s_v, attn_row<T>(a.v, t.b, t.tok0 + j0, hk), a.v.st, keys, a.V));
    f32x4 s[1][4];
    acc_zero(s);
    gemm_nt<T, 1, 4>(s, s_q, LD, 16 * w, s_k, LD, 0, 0, W);
    float old[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      old[i] = m[i];
      float mx = M_LOW;
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) {
        const int j = j0 + 16 * ni + (l & 15);
        const float qk = s[0][ni][i];
        const bool ok = j < t.len && (!a.causal || j <= row + i || j < t.prefix);
        s[0][ni][i] = ok ? sc.of(qk, CAP ? sc.squash(qk) : 0.f, (float)(row + i - j)) : -INFINITY;
        mx = fmaxf(mx, s[0][ni][i]);
      }
      m[i] = fmaxf(m[i], row16_max(mx));
      float ps = 0.f;
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) {
        const float p = pow2<false>(s[0][ni][i] - m[i]);
        ps += p;
        s[0][ni][i] = p;
      }
      const float f = pow2<false>(old[i] - m[i]);
      sum[i] = sum[i] * f + group_sum<16>(ps);
#pragma unroll
      for (int ni = 0; ni < NB; ++ni) o[0][ni][i] *= f;
    }
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) acc_to_lds<T>(s[0][ni], s_p, PLD, 16 * w, 16 * ni);
    __syncthreads();
    // A product with 0 for what the mask hides would make NaN of a hidden NaN or infinity: such numbers are added by themselves to
    // the rows that see them and leave the tile.
    if (odd && a.causal && j0 + CH > t.r0) {
      for (int j = 0; j < keys; ++j)
#pragma unroll
        for (int ni = 0; ni < NB; ++ni) {
          const float v = ET<T>::to_f(s_v[j * LD + 16 * ni + (l & 15)]);
          if (fabsf(v) < INFINITY) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (j0 + j <= row + i || j0 + j < t.prefix) o[0][ni][i] += ET<T>::to_f(s_p[(16 * w + 4 * (l >> 4) + i) * PLD + j]) * v;
        }
      __syncthreads();
      for (int i = threadIdx.x; i < CH * LD; i += NTHR)
        if (!(fabsf(ET<T>::to_f(s_v[i])) < INFINITY)) s_v[i] = (T)0.0f;
      __syncthreads();
    }
    gemm<T, 1, NB, false, true>(o, s_p, PLD, 16 * w, s_v, LD, 0, 0, CH);
  }
  float inv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    inv[i] = 1.0f / sum[i];
    if (a.lse && (l & 15) == 0 && row + i < t.len)
      a.lse[((int64_t)t.b * a.HQ + h) * a.T + t.tok0 + row + i] = m[i] + log2f(sum[i]);
  }
  attn_store<T, NB>(o, attn_row<T>(a.o, t.b, t.tok0 + t.r0 + 16 * w, h), a.o.st, rows - 16 * w, a.V, inv);
}

// dq of 64 rows; delta of those rows beside it
template <typename T, int W, bool CAP, bool BIAS>
__global__ __launch_bounds__(NTHR) void k_attn_bwd_dq_any(const lmoe_attn_args a) {
  constexpr int LD = W + LPAD, PLD = CH + LPAD, NB = W / 16;
  // (q, then keys; do, then values: the strips of q and do a wave needs stay with it as LDS tiles of their own)
  __shared__ __attribute__((aligned(16))) T s_q[CH * LD], s_k[CH * LD], s_v[CH * LD], s_do[CH * LD], s_p[CH * PLD];
  zero_behind<T>(a, a.dq, a.HQ, a.K);
  AttnTile t;
  int h;
  if (!attn_place<CH>(a, a.HQ, true, h, t)) return;
  const int hk = h / (a.HQ / a.HKV);
  const Score<CAP, BIAS, false> sc(a, h);
  const int l = lane_id(), w = wave_id(), row = t.r0 + 16 * w + 4 * (l >> 4);
  const int rows = min(CH, t.len - t.r0);
  attn_load<T, W>(s_q, attn_row<T>(a.q, t.b, t.tok0 + t.r0, h), a.q.st, rows, a.K);
  attn_load<T, W>(s_do, attn_row<T>(a.d_o, t.b, t.tok0 + t.r0, h), a.d_o.st, rows, a.V);
  attn_load<T, W>(s_k, attn_row<T>(a.o, t.b, t.tok0 + t.r0, h), a.o.st, rows, a.V);
  __syncthreads();
  float lse[4], delta[4];
  const int64_t at = ((int64_t)t.b * a.HQ + h) * a.T + t.tok0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 16 * w + 4 * (l >> 4) + i;
    float d = 0.f;
#pragma unroll
    for (int c = 0; c < W; c += 16) d += ET<T>::to_f(s_do[r * LD + c + (l & 15)]) * ET<T>::to_f(s_k[r * LD + c + (l & 15)]);
    delta[i] = group_sum<16>(d);
    lse[i] = a.lse[at + min(row + i, t.len - 1)];
    if ((l & 15) == 0 && row + i < t.len) a.delta[at + row + i] = delta[i];
  }
  f32x4 dq[1][NB];
  acc_zero(dq);
  const int end = a.causal ? min(t.len, max(t.r0 + CH, t.prefix)) : t.len;
  for (int j0 = 0; j0 < end; j0 += CH) {
    const int keys = min(CH, t.len - j0);
    __syncthreads();
    attn_load<T, W>(s_k, attn_row<T>(a.k, t.b, t.tok0 + j0, hk), a.k.st, keys, a.K);
    attn_load<T, W>(s_v, attn_row<T>(a.v, t.b, t.tok0 + j0, hk), a.v.st, keys, a.V);
    __syncthreads();
    f32x4 s[1][4], dp[1][4];
    acc_zero(s);
    acc_zero(dp);
    gemm_nt<T, 1, 4>(s, s_q, LD, 16 * w, s_k, LD, 0, 0, W);
    gemm_nt<T, 1, 4>(dp, s_do, LD, 16 * w, s_v, LD, 0, 0, W);
#pragma unroll
    for (int ni = 0; ni < 4; ++ni)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = j0 + 16 * ni + (l & 15);
        const float qk = s[0][ni][i], th = CAP ? sc.squash(qk) : 0.f;
        const bool ok = j < t.len && (!a.causal || j <= row + i || j < t.prefix);
        float ds = pow2<false>(sc.of(qk, th, (float)(row + i - j)) - lse[i]) * (dp[0][ni][i] - delta[i]);
        if constexpr (CAP) ds *= 1.0f - th * th;
        s[0][ni][i] = ok ? ds : 0.f;
      }
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) acc_to_lds<T>(s[0][ni], s_p, PLD, 16 * w, 16 * ni);
    __syncthreads();
    gemm<T, 1, NB, false, true>(dq, s_p, PLD, 16 * w, s_k, LD, 0, 0, CH);
  }
  const float mul[4] = {a.scale, a.scale, a.scale, a.scale};
  attn_store<T, NB>(dq, attn_row<T>(a.dq, t.b, t.tok0 + t.r0 + 16 * w, h), a.dq.st, rows - 16 * w, a.K, mul);
}

// dk, dv of 64 keys: over the rows of all query heads that share the key head, one after the other (no atomics)
template <typename T, int W, bool CAP, bool BIAS>
__global__ __launch_bounds__(NTHR) void k_attn_bwd_dkv_any(const lmoe_attn_args a) {
  constexpr int LD = W + LPAD, PLD = CH + LPAD, NB = W / 16;
  __shared__ __attribute__((aligned(16))) T s_q[CH * LD], s_k[CH * LD], s_v[CH * LD], s_do[CH * LD], s_p[CH * PLD];
  zero_behind<T>(a, a.dk, a.HKV, a.K);
  zero_behind<T>(a, a.dv, a.HKV, a.V);
  const int G = a.HQ / a.HKV;
  AttnTile t;
  int hk;
  if (!attn_place<CH>(a, a.HKV, false, hk, t)) return;
  const int l = lane_id(), w = wave_id(), key = t.r0 + 16 * w + 4 * (l >> 4);
  const int keys = min(CH, t.len - t.r0);
  attn_load<T, W>(s_k, attn_row<T>(a.k, t.b, t.tok0 + t.r0, hk), a.k.st, keys, a.K);
  attn_load<T, W>(s_v, attn_row<T>(a.v, t.b, t.tok0 + t.r0, hk), a.v.st, keys, a.V);
  f32x4 dk[1][NB], dv[1][NB];
  acc_zero(dk);
  acc_zero(dv);
  const int begin = a.causal && t.r0 >= t.prefix ? t.r0 : 0;
  for (int h = hk * G; h < (hk + 1) * G; ++h) {
    const Score<CAP, BIAS, false> sc(a, h);
    const int64_t at = ((int64_t)t.b * a.HQ + h) * a.T + t.tok0;
    for (int i0 = begin; i0 < t.len; i0 += CH) {
      const int rows = min(CH, t.len - i0);
      __syncthreads();
      attn_load<T, W>(s_q, attn_row<T>(a.q, t.b, t.tok0 + i0, h), a.q.st, rows, a.K);
      attn_load<T, W>(s_do, attn_row<T>(a.d_o, t.b, t.tok0 + i0, h), a.d_o.st, rows, a.V);
      __syncthreads();
      f32x4 s[1][4], dp[1][4];
      acc_zero(s);
      acc_zero(dp);
      gemm_nt<T, 1, 4>(s, s_k, LD, 16 * w, s_q, LD, 0, 0, W);
      gemm_nt<T, 1, 4>(dp, s_v, LD, 16 * w, s_do, LD, 0, 0, W);
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) {
        const int i = i0 + 16 * ni + (l & 15), ic = min(i, t.len - 1);
        const float lse = a.lse[at + ic], delta = a.delta[at + ic];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = key + e;
          const float qk = s[0][ni][e], th = CAP ? sc.squash(qk) : 0.f;
          const bool ok = i < t.len && (!a.causal || j <= i || j < t.prefix);
          const float p = ok ? pow2<false>(sc.of(qk, th, (float)(i - j)) - lse) : 0.f;
          float ds = p * (dp[0][ni][e] - delta);
          if constexpr (CAP) ds *= 1.0f - th * th;
          s[0][ni][e] = p;
          dp[0][ni][e] = ok ? ds : 0.f;
        }
      }
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) acc_to_lds<T>(s[0][ni], s_p, PLD, 16 * w, 16 * ni);
      __syncthreads();
      gemm<T, 1, NB, false, true>(dv, s_p, PLD, 16 * w, s_do, LD, 0, 0, CH);
      __syncthreads();
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) acc_to_lds<T>(dp[0][ni], s_p, PLD, 16 * w, 16 * ni);
      __syncthreads();
      gemm<T, 1, NB, false, true>(dk, s_p, PLD, 16 * w, s_q, LD, 0, 0, CH);
    }
  }
  const float one[4] = {1.f, 1.f, 1.f, 1.f}, mul[4] = {a.scale, a.scale, a.scale, a.scale};
  attn_store<T, NB>(dv, attn_row<T>(a.dv, t.b, t.tok0 + t.r0 + 16 * w, hk), a.dv.st, keys - 16 * w, a.V, one);
  attn_store<T, NB>(dk, attn_row<T>(a.dk, t.b, t.tok0 + t.r0 + 16 * w, hk), a.dk.st, keys - 16 * w, a.K, mul);
}

}  // namespace lmoe
