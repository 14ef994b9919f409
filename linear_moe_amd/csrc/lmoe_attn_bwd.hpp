// Softmax attention, backward pass on 2-byte elements: dq by rows, then dk and dv by keys, each with the scores formed again.
// (One kernel for all three would add dq up in memory, in an order that changes from run to run, or write every tile's share of
// it: T / 256 times the bytes of dq.  Two score products more cost less.)
#pragma once
#include "lmoe_attn_fwd.hpp"

namespace lmoe {

// dq of NW x 32 rows; delta of those rows beside it.  As the forward kernel: S^T = K Q^T and dP^T = V dO^T leave a lane with one row,
// whose lse and delta are one number, and dS^T as the B operand of dQ^T += K^T dS^T.
template <int W, int NW, bool CAP, bool BIAS>
__global__ __launch_bounds__(NW * 64, 2) void k_attn_bwd_dq(const lmoe_attn_args a) {
  constexpr int LD = W + LPAD, KS = W / 16, DB = W / 32, NT = NW * 64, ROWS = NW * 32, TILE = CH * LD;
  typedef RowStage<CH, W, NT> St;
  __shared__ __attribute__((aligned(16))) bf16 s_kv[4 * TILE];
  static_assert(ROWS * LD <= 4 * TILE, "the strips of the waves");
  zero_behind<bf16>(a, a.dq, a.HQ, a.K);
  AttnTile t;
  int h;
  if (!attn_place<ROWS>(a, a.HQ, true, h, t)) return;
  const int hk = h / (a.HQ / a.HKV), tid = threadIdx.x, l = lane_id(), w = wave_id(), g = l >> 5;
  const Score<CAP, BIAS, true> sc(a, h);
  const int w0 = t.r0 + 32 * w, rows = t.len - w0, row = w0 + (l & 31);
  const int64_t at = ((int64_t)t.b * a.HQ + h) * a.T + t.tok0;
  bf16x8 q[KS], d_o[KS];
  rows32<W>(d_o, attn_row<bf16>(a.d_o, t.b, t.tok0 + min(w0, t.len - 1), h), a.d_o.st, max(rows, 1), a.V, l);
  rows32<W>(q, attn_row<bf16>(a.o, t.b, t.tok0 + min(w0, t.len - 1), h), a.o.st, max(rows, 1), a.V, l);
  float delta = 0.f;
#pragma unroll
  for (int j = 0; j < KS; ++j) delta = dot_vec(q[j], d_o[j], delta);
  delta = both_sum(delta);
  const float lse = a.lse[at + min(row, t.len - 1)];
  if (g == 0 && row < t.len) a.delta[at + row] = delta;
  rows32<W>(q, attn_row<bf16>(a.q, t.b, t.tok0 + min(w0, t.len - 1), h), a.q.st, max(rows, 1), a.K, l);
  f32x16 dq[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) dq[b] = zero16();

  const int end = a.causal ? min(t.len, max(t.r0 + ROWS, t.prefix)) : t.len;
  const int wend = rows <= 0 ? 0 : a.causal ? min(t.len, max(w0 + 32, t.prefix)) : t.len;
  const int whole = a.causal ? max(w0 + 1, t.prefix) : t.len;
  const bf16* kp = attn_row<bf16>(a.k, t.b, t.tok0, hk);
  const bf16* vp = attn_row<bf16>(a.v, t.b, t.tok0, hk);

  auto block = [&](const bf16* sk, const bf16* sv, int j0, auto part_c) {
    constexpr bool PART = decltype(part_c)::value;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      __builtin_amdgcn_sched_barrier(0);
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int j = 0; j < KS; ++j) s = mfma32(*(const bf16x8*)(sk + (32 * b + (l & 31)) * LD + 16 * j + 8 * g), q[j], s);
#pragma unroll
      for (int j = 0; j < KS; ++j) dp = mfma32(*(const bf16x8*)(sv + (32 * b + (l & 31)) * LD + 16 * j + 8 * g), d_o[j], dp);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = j0 + 32 * b + row32(i) + 4 * g;
        const float th = CAP ? sc.squash(s[i]) : 0.f;
        float ds = pow2<true>(sc.of(s[i], th, (float)(row - j)) - lse) * (dp[i] - delta);
        if constexpr (CAP) ds *= __builtin_fmaf(-th, th, 1.0f);
        if constexpr (PART) ds = j < t.len && (!a.causal || j <= row || j < t.prefix) ? ds : 0.f;
        s[i] = ds;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const bf16x8 ds = frag_of_acc(s, x);
#pragma unroll
        for (int d = 0; d < DB; ++d) dq[d] = mfma32(frag32_t(sk, LD, 32 * b + 16 * x, 32 * d, l), ds, dq[d]);
      }
    }
  };

  St sk, sv;
  sk.load(kp, a.k.st, t.len, a.K, tid);
  sv.load(vp, a.v.st, t.len, a.V, tid);
  sk.store(s_kv, t.len, a.K, tid);
  sv.store(s_kv + TILE, t.len, a.V, tid);
  if (CH < end) {
    sk.load(kp + CH * a.k.st, a.k.st, t.len - CH, a.K, tid);
    sv.load(vp + CH * a.v.st, a.v.st, t.len - CH, a.V, tid);
  }
  for (int j0 = 0; j0 < end; j0 += CH) {
    const int cur = (j0 / CH) & 1;
    lds_barrier();
    if (j0 + CH < end) {
      sk.store(s_kv + (2 - 2 * cur) * TILE, t.len - j0 - CH, a.K, tid);
      sv.store(s_kv + (3 - 2 * cur) * TILE, t.len - j0 - CH, a.V, tid);
      if (j0 + 2 * CH < end) {
        sk.load(kp + (int64_t)(j0 + 2 * CH) * a.k.st, a.k.st, t.len - j0 - 2 * CH, a.K, tid);
        sv.load(vp + (int64_t)(j0 + 2 * CH) * a.v.st, a.v.st, t.len - j0 - 2 * CH, a.V, tid);
      }
    }
    const bf16 *ck = s_kv + 2 * cur * TILE, *cv = ck + TILE;
    if (j0 + CH <= whole && j0 + CH <= t.len) { if (rows > 0) block(ck, cv, j0, std::false_type()); }
    else if (j0 < wend) block(ck, cv, j0, std::true_type());
  }
  lds_barrier();
  if (rows > 0)
    store_rows32<W>(dq, a.scale, s_kv + w * 32 * LD, attn_row<bf16>(a.dq, t.b, t.tok0 + w0, h), a.dq.st, rows, a.K, l);
}

// dk, dv of NW x 32 keys, over the rows of all query heads that share the key head, one after the other.  A wave holds its 32 keys
// and values as B operands: S = Q K^T and dP = dO V^T leave a lane with one key, P and dS as the B operands of dV^T += dO^T P and
// dK^T += Q^T dS.  QR rows of q and do at a time lie in LDS, twice, with their lse and delta.  Rows behind the sequence come with
// lse = infinity, so that their p is 0.
template <int W, int NW, int QR, bool CAP, bool BIAS>
__global__ __launch_bounds__(NW * 64, W == 64 ? 2 : 1) void k_attn_bwd_dkv(const lmoe_attn_args a) {
  constexpr int LD = W + LPAD, KS = W / 16, DB = W / 32, NT = NW * 64, KEYS = NW * 32, TILE = QR * LD;
  typedef RowStage<QR, W, NT> St;
  constexpr int AREA = 4 * TILE > KEYS * LD ? 4 * TILE : KEYS * LD;
  __shared__ __attribute__((aligned(16))) bf16 s_qd[AREA];
  __shared__ __attribute__((aligned(16))) float s_row[2][2][QR];          // lse, delta
  zero_behind<bf16>(a, a.dk, a.HKV, a.K);
  zero_behind<bf16>(a, a.dv, a.HKV, a.V);
  AttnTile t;
  int hk;
  if (!attn_place<KEYS>(a, a.HKV, false, hk, t)) return;
  const int G = a.HQ / a.HKV, tid = threadIdx.x, l = lane_id(), w = wave_id(), g = l >> 5;
  const int w0 = t.r0 + 32 * w, keys = t.len - w0, key = w0 + (l & 31);
  bf16x8 k[KS], v[KS];
  rows32<W>(k, attn_row<bf16>(a.k, t.b, t.tok0 + min(w0, t.len - 1), hk), a.k.st, max(keys, 1), a.K, l);
  rows32<W>(v, attn_row<bf16>(a.v, t.b, t.tok0 + min(w0, t.len - 1), hk), a.v.st, max(keys, 1), a.V, l);
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) { dk[b] = zero16(); dv[b] = zero16(); }
  const int begin = a.causal && t.r0 >= t.prefix ? t.r0 : 0;
  const int wbegin = keys <= 0 ? t.len : a.causal && w0 >= t.prefix ? w0 : 0;             // the first row that sees one of the wave's keys
  const int whole = a.causal && w0 + 32 > t.prefix ? w0 + 31 : 0;                         // from it on rows see all of them

  auto block = [&](const Score<CAP, BIAS, true>& sc, const bf16* sq, const bf16* sd, const float* s_lse, const float* s_delta, int i0, auto part_c) {
    constexpr bool PART = decltype(part_c)::value;
#pragma unroll
    for (int b = 0; b < QR / 32; ++b) {
      if constexpr (W == 64) __builtin_amdgcn_sched_barrier(0);
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int j = 0; j < KS; ++j) s = mfma32(*(const bf16x8*)(sq + (32 * b + (l & 31)) * LD + 16 * j + 8 * g), k[j], s);
#pragma unroll
      for (int j = 0; j < KS; ++j) dp = mfma32(*(const bf16x8*)(sd + (32 * b + (l & 31)) * LD + 16 * j + 8 * g), v[j], dp);
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f32x4 lse = *(const f32x4*)(s_lse + 32 * b + row32(e) + 4 * g), delta = *(const f32x4*)(s_delta + 32 * b + row32(e) + 4 * g);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int i = i0 + 32 * b + row32(e + x) + 4 * g;
          const float th = CAP ? sc.squash(s[e + x]) : 0.f;
          float p = pow2<true>(sc.of(s[e + x], th, (float)(i - key)) - lse[x]);
          if constexpr (PART) p = key <= i || key < t.prefix ? p : 0.f;
          float ds = p * (dp[e + x] - delta[x]);
          if constexpr (CAP) ds *= __builtin_fmaf(-th, th, 1.0f);
          s[e + x] = p;
          dp[e + x] = ds;
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const bf16x8 p = frag_of_acc(s, x), ds = frag_of_acc(dp, x);
#pragma unroll
        for (int d = 0; d < DB; ++d) dv[d] = mfma32(frag32_t(sd, LD, 32 * b + 16 * x, 32 * d, l), p, dv[d]);
#pragma unroll
        for (int d = 0; d < DB; ++d) dk[d] = mfma32(frag32_t(sq, LD, 32 * b + 16 * x, 32 * d, l), ds, dk[d]);
      }
    }
  };

  // rows of the group's heads, one after the other: what is fetched next
  struct { int h, i; } next = {hk * G, begin};
  St sq, sd;
  float stat = 0.f;
  const int last = hk * G + G;
  auto fetch = [&] {
    sq.load(attn_row<bf16>(a.q, t.b, t.tok0 + next.i, next.h), a.q.st, t.len - next.i, a.K, tid);
    sd.load(attn_row<bf16>(a.d_o, t.b, t.tok0 + next.i, next.h), a.d_o.st, t.len - next.i, a.V, tid);
    if (tid < 2 * QR) {
      const int i = next.i + tid % QR;
      const float* p = (tid < QR ? a.lse : a.delta) + ((int64_t)t.b * a.HQ + next.h) * a.T + t.tok0;
      stat = i < t.len ? p[i] : tid < QR ? INFINITY : 0.f;
    }
  };
  auto put = [&](int buf, int i) {
    sq.store(s_qd + 2 * buf * TILE, t.len - i, a.K, tid);
    sd.store(s_qd + (2 * buf + 1) * TILE, t.len - i, a.V, tid);
    if (tid < 2 * QR) s_row[buf][tid / QR][tid % QR] = stat;
  };
  auto advance = [&] {
    next.i += QR;
    if (next.i >= t.len) { next.i = begin; ++next.h; }
  };
  fetch();
  put(0, next.i);
  int h = next.h, i0 = next.i, cur = 0;
  advance();
  if (next.h < last) fetch();
  Score<CAP, BIAS, true> sc(a, h);
  while (h < last) {
    lds_barrier();
    const int hn = next.h, in = next.i;
    if (hn < last) {
      put(cur ^ 1, in);
      advance();
      if (next.h < last) fetch();
    }
    const bf16 *cq = s_qd + 2 * cur * TILE, *cd = cq + TILE;
    if (i0 + QR > wbegin) {
      if (i0 >= whole) block(sc, cq, cd, s_row[cur][0], s_row[cur][1], i0, std::false_type());
      else block(sc, cq, cd, s_row[cur][0], s_row[cur][1], i0, std::true_type());
    }
    if (hn != h && hn < last) sc = Score<CAP, BIAS, true>(a, hn);
    h = hn; i0 = in; cur ^= 1;
  }
  lds_barrier();
  if (keys > 0) {
    store_rows32<W>(dv, 1.0f, s_qd + w * 32 * LD, attn_row<bf16>(a.dv, t.b, t.tok0 + w0, hk), a.dv.st, keys, a.V, l);
    __builtin_amdgcn_wave_barrier();
    store_rows32<W>(dk, a.scale, s_qd + w * 32 * LD, attn_row<bf16>(a.dk, t.b, t.tok0 + w0, hk), a.dk.st, keys, a.K, l);
  }
}

}  // namespace lmoe
