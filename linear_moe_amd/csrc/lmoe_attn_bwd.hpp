// Softmax attention, backward pass on 2-byte elements: dq by rows, then dk and dv by keys, each with the scores formed again.
// (One kernel for all three would add dq up in memory, in an order that changes from run to run, or write every tile's share of
// it: T / 256 times the bytes of dq.  Two score products more cost less.)
// Bound: the matrix rate (the matrix unit is busy for 59 % of the cycles of dq, 55 % of those of dk and dv, in which a third of the
// waves' time goes to waiting for LDS and the barrier; LDS itself is busy for 41 %).  4 x 8192 tokens, 16 heads on 4 of 128, causal: dq 1.44 ms,
// 1146 TFLOP/s, dk and dv 2.02 ms, 1089, counted with the scores each forms again; the whole by the five products that it cannot do
// without 790.
#pragma once
#include "lmoe_attn_fwd.hpp"

namespace lmoe {

// dq of 128 rows; delta of those rows beside it.  As the forward kernel: S^T = K Q^T and dP^T = V dO^T leave a lane with one row,
// whose lse and delta are one number, and dS^T as the B operand of dQ^T += K^T dS^T.
template <int W, int KG, int CAP, bool BIAS>
__global__ __launch_bounds__(KG * ATTN_WAVES * 64, 2) void k_attn_bwd_dq(const lmoe_attn_args a) {
  constexpr int KS = W / 16, DB = W / 32, TILE = CH * W, A1 = 3;
  __shared__ __attribute__((aligned(1024))) bf16 a_k0[KG * TILE], a_v0[KG * TILE], a_k1[KG * TILE], a_v1[KG * TILE];
  zero_behind<bf16>(a, a.dq, a.HQ, a.K);
  AttnTile t;
  int h;
  if (!attn_place<ATTN_ROWS>(a, a.HQ, true, h, t)) return;
  const int hk = h / (a.HQ / a.HKV), l = lane_id(), w = KG == 1 ? wave_id() : wave_id() % ATTN_WAVES, g = l >> 5;
  const int kg = KG == 1 ? 0 : wave_id() / ATTN_WAVES;
  bf16 *const s_k0 = a_k0 + kg * TILE, *const s_v0 = a_v0 + kg * TILE, *const s_k1 = a_k1 + kg * TILE, *const s_v1 = a_v1 + kg * TILE;
  const Score16<CAP, BIAS> sc(a, h);
  const int w0 = t.r0 + 32 * w, rows = t.len - w0, row_ = w0 + (l & 31);
  const int64_t first = ((int64_t)t.b * a.HQ + h) * a.T + t.tok0;
  const Swz<W> lane(l);
  bf16x8 q[KS], d_o[KS];
  rows32<W>(d_o, attn_row<bf16>(a.d_o, t.b, t.tok0 + min(w0, t.len - 1), h), a.d_o.st, max(rows, 1), a.V, l);
  rows32<W>(q, attn_row<bf16>(a.o, t.b, t.tok0 + min(w0, t.len - 1), h), a.o.st, max(rows, 1), a.V, l);
  float delta = 0.f;
  const int8_t* low = a.o_low + (first + min(row_, t.len - 1)) * a.V;
#pragma unroll
  for (int j = 0; j < KS; ++j) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    u32x2 x = {0, 0};
    if (a.o_low && 16 * j + 8 * g < a.V) x = *(const u32x2*)(low + 16 * j + 8 * g);
#pragma unroll
    for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(with_low(q[j][e], x[e / 4], e % 4), (float)d_o[j][e], delta);
  }
  delta = both_sum(delta);
  const float lse = a.lse[first + min(row_, t.len - 1)];
  if (kg == 0 && g == 0 && row_ < t.len) a.delta[first + row_] = delta;
  rows32<W>(q, attn_row<bf16>(a.q, t.b, t.tok0 + min(w0, t.len - 1), h), a.q.st, max(rows, 1), a.K, l);
  if (sc.negate) {
#pragma unroll
    for (int j = 0; j < KS; ++j) frag_negate(q[j]);
  }
  const float off = sc.b - lse;
  f32x16 dq[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) dq[b] = zero16();

  const int end = a.causal ? min(t.len, max(t.r0 + ATTN_ROWS, t.prefix)) : t.len;
  const int wend = rows <= 0 ? 0 : a.causal ? min(t.len, max(w0 + 32, t.prefix)) : t.len;
  const int wwhole = a.causal ? min(t.len, max(w0 + 1, t.prefix)) : t.len;        // all rows of the wave see the keys before it
  const bf16* kp = attn_row<bf16>(a.k, t.b, t.tok0, hk);
  const bf16* vp = attn_row<bf16>(a.v, t.b, t.tok0, hk);

  auto block = [&](const bf16* sk, const bf16* sv, int j0, auto issue) __attribute__((always_inline)) {
    const Swz<W> at = lane.fresh();
    const int row = fresh_index(row_);
    // (pieces are asked for A1 steps before their products, those of the second half under the last products of the first: 4 x 8192
    // tokens, 16 heads on 4 of 128, 1.44 ms, with each pair asked for right in front of its products 1.47; two or four steps: the same)
    bf16x8 kf[A1], vf[A1], kt[2 * DB];
    auto read = [&](int b, int j) { kf[j % A1] = at.frag(sk, b, j); vf[j % A1] = at.frag(sv, b, j); };
#pragma unroll
    for (int j = 0; j < A1; ++j) read(0, j);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      __builtin_amdgcn_sched_barrier(0);
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        s = mfma32(kf[j % A1], q[j], s);
        dp = mfma32(vf[j % A1], d_o[j], dp);
        if (j + A1 < KS) read(b, j + A1);
        __builtin_amdgcn_sched_barrier(0);
      }
      issue(2 * b);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int d = 0; d < DB; ++d) kt[x * DB + d] = at.frag_t(sk, 2 * b + x, d);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = j0 + 32 * b + row32(i) + 4 * g;
        float r;
        const float u = sc(s[i], (float)(row - j), r);
        float ds = pow2(__builtin_fmaf(u, sc.a, off)) * (dp[i] - delta);
        if constexpr (CAP) ds *= sc.fade(r);
        s[i] = ds;
      }
      if (j0 + 32 * b + 32 > wwhole) {
        const int sees = (a.causal ? min(t.len, max(row + 1, t.prefix)) : t.len) - (j0 + 32 * b + 4 * g);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = row32(i) < sees ? s[i] : 0.f;
      }
      issue(2 * b + 1);
      if (b == 0) {
#pragma unroll
        for (int j = 0; j < A1; ++j) read(1, j);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const bf16x8 ds = frag_of_acc(s, x);
#pragma unroll
        for (int d = 0; d < DB; ++d) dq[d] = mfma32(kt[x * DB + d], ds, dq[d]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  KeyTiles<W> load(a, kp, vp, t.len, end, w, l, KG * CH);
  auto tile = [&](bf16* ck, bf16* cv, bf16* nk, bf16* nv, int j0) __attribute__((always_inline)) {
    load.arrived(ck, cv, j0);
    auto issue = [&](int point) __attribute__((always_inline)) { load.next(nk, nv, j0, point); };
    if (j0 < wend) block(ck, cv, j0, issue);
    else { issue(0); issue(1); issue(2); issue(3); }
  };
  load.first(s_k0, s_v0, kg * CH);
  for (int j0 = 0; j0 < end; j0 += 2 * KG * CH) {
    tile(s_k0, s_v0, s_k1, s_v1, j0 + kg * CH);
    if (j0 + KG * CH < end) tile(s_k1, s_v1, s_k0, s_v0, j0 + (KG + kg) * CH);
  }
  wait_all_loads();                      // (none may arrive in an LDS that is another's)
  if constexpr (KG == 2) {
    const Handed<W> x(a_k0, a_v0, w, l);
    lds_barrier();
    if (kg == 1) x.put(dq);
    lds_barrier();
    if (kg == 1) return;
#pragma unroll
    for (int i = 0; i < 16 * DB; ++i) dq[i / 16][i % 16] += x.at(i);
  }
  if (rows > 0)
    store_rows32<W>(dq, a.scale, attn_row<bf16>(a.dq, t.b, t.tok0 + w0, h), a.dq.st, rows, a.K, l);
}

// the lane's numbers of a transposed block of 32 rows, times mul, as they are: four adjacent columns at a time
template <int W> __device__ __forceinline__ void store_sums(const f32x16 (&acc)[W / 32], float mul, float* row, int D, int g) {
#pragma unroll
  for (int b = 0; b < W / 32; ++b)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int c = 32 * b + row32(i) + 4 * g;
      if (c < D) *(f32x4*)(row + c) = f32x4{acc[b][i], acc[b][i + 1], acc[b][i + 2], acc[b][i + 3]} * mul;
    }
}

// dk, dv of NW x 32 keys, over the rows of all query heads that share the key head.  S = Q K^T and dP = dO V^T leave a lane with one
// key, P and dS as the B operands of dV^T += dO^T P and dK^T += Q^T dS.  A wave holds its keys as B operands in registers; its
// values, for which there is no room beside both sums, lie in LDS.  64 rows of q and do at a time lie there too, twice, with
// their lse and delta.  Rows behind the sequence come with lse = infinity, so that their p is 0.
// From the last row to the first, the heads of a row tile one after the other: the work-groups of a key head, whose rows begin at
// different places but end at one, read the same tiles at about the same time, and an XCD's L2 holds them for all.
// Where the keys are too few for the card, or unequal work, up to `parts` work-groups share a tile of them, each with its part of that
// stream (`least` of its pieces or more), and leave fp32 sums for k_attn_join; alone, a work-group leaves the gradients themselves.
// The stream of a tile of keys: 64-row tiles top .. begin / 64 of G heads
struct KeyStream {
  int begin, top, all, parts;
  __device__ __forceinline__ KeyStream(const lmoe_attn_args& a, const AttnTile& t, int most, int least) {
    begin = a.causal && t.r0 >= t.prefix ? t.r0 : 0;              // the first row that sees a key of the tile
    top = (t.len - 1) / CH;
    all = (top - begin / CH + 1) * (a.HQ / a.HKV);
    parts = least ? max(1, min(most, all / least)) : most;        // (0: all of them, whatever the stream)
  }
};
template <int W, int NW, int CAP, bool BIAS>
__global__ __launch_bounds__(NW * 64, W == 64 ? 3 : 2) void k_attn_bwd_dkv(const lmoe_attn_args a, int most, int least) {
  constexpr int KS = W / 16, DB = W / 32, KEYS = NW * 32, TILE = CH * W;
  constexpr int A1 = 2, A2 = 4;
  __shared__ __attribute__((aligned(1024))) bf16 s_q0[TILE], s_d0[TILE], s_q1[TILE], s_d1[TILE], s_v[KEYS * W];
  __shared__ __attribute__((aligned(16))) float s_row[2][2][CH];          // lse, delta
  if (blockIdx.y == 0) {
    zero_behind<bf16>(a, a.dk, a.HKV, a.K);
    zero_behind<bf16>(a, a.dv, a.HKV, a.V);
  }
  AttnTile t;
  int hk;
  if (!attn_place<KEYS>(a, a.HKV, false, hk, t)) return;
  const KeyStream of(a, t, most, least);
  const int parts = of.parts;
  if ((int)blockIdx.y >= parts) return;
  const int G = a.HQ / a.HKV, tid = threadIdx.x, l = lane_id(), w = wave_id(), g = l >> 5;
  const Swz<W> lane(l);
  const int w0 = t.r0 + 32 * w, keys = t.len - w0, key_ = w0 + (l & 31);
  bf16x8 k[KS];
  bf16* const sv = s_v + 32 * w * W;                                      // (of the wave's own: no barrier)
  rows32<W>(k, attn_row<bf16>(a.v, t.b, t.tok0 + min(w0, t.len - 1), hk), a.v.st, max(keys, 1), a.V, l);
#pragma unroll
  for (int j = 0; j < KS; ++j) *(bf16x8*)((char*)sv + (lane.rows ^ 32 * j)) = k[j];
  rows32<W>(k, attn_row<bf16>(a.k, t.b, t.tok0 + min(w0, t.len - 1), hk), a.k.st, max(keys, 1), a.K, l);
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) { dk[b] = zero16(); dv[b] = zero16(); }
  const int wbegin = keys <= 0 ? t.len : a.causal && w0 >= t.prefix ? w0 : 0;             // ... of the wave
  const int wwhole = a.causal && w0 + 32 > t.prefix ? w0 + 31 : 0;                         // from it on rows see all keys of the wave

  auto block = [&](const Score16<CAP, BIAS>& sc, const bf16* sq, const bf16* sd, const float* s_lse, const float* s_delta, int i0, auto issue) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < CH / 32; ++b) {
      const Swz<W> at = lane.fresh();
      const int key = fresh_index(key_);
      f32x16 s = zero16(), dp = zero16();
      __builtin_amdgcn_sched_barrier(0);
      // (128 columns: the pieces of a step are asked for two steps before their products, in this order.  Left to itself the compiler asks for
      // each right in front of its product and waits for it; with 64 it has registers for more, and three waves a SIMD: 2 x 8192
      // tokens, 16 heads on 4, backward 1.062 ms, in this order 1.075; of 128 with a cap 2.228 and 2.188)
      bf16x8 f[A1], y[A1], z[A1];
      auto read = [&](int j) { f[j % A1] = at.frag(sq, b, j); y[j % A1] = at.frag(sd, b, j); z[j % A1] = at.frag(sv, 0, j); };
#pragma unroll
      for (int j = 0; j < A1; ++j) read(j);
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        if constexpr (W == 128) __builtin_amdgcn_sched_barrier(0);
        s = mfma32(f[j % A1], k[j], s);
        dp = mfma32(y[j % A1], z[j % A1], dp);
        if (j + A1 < KS) read(j + A1);
      }
      __builtin_amdgcn_sched_barrier(0);
      issue(2 * b);
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f32x4 lse = *(const f32x4*)(s_lse + 32 * b + row32(e) + 4 * g), delta = *(const f32x4*)(s_delta + 32 * b + row32(e) + 4 * g);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int i = i0 + 32 * b + row32(e + x) + 4 * g;
          float r;
          const float u = sc(s[e + x], (float)(i - key), r);
          float p = pow2(__builtin_fmaf(u, sc.a, sc.b - lse[x]));
          float ds = p * (dp[e + x] - delta[x]);
          if constexpr (CAP) ds *= sc.fade(r);
          s[e + x] = p;
          dp[e + x] = ds;
        }
      }
      if (i0 + 32 * b < wwhole) {
        const int from = (key < t.prefix ? 0 : key) - (i0 + 32 * b + 4 * g);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[e] = row32(e) >= from ? s[e] : 0.f;
          dp[e] = row32(e) >= from ? dp[e] : 0.f;
        }
      }
      const bf16x8 p0 = frag_of_acc(s, 0), p1 = frag_of_acc(s, 1), ds0 = frag_of_acc(dp, 0), ds1 = frag_of_acc(dp, 1);
      issue(2 * b + 1);
      bf16x8 t[A2];
      auto read_t = [&](int n) { t[n % A2] = at.frag_t(n < 2 * DB ? sd : sq, 2 * b + n / DB % 2, n % DB); };
#pragma unroll
      for (int n = 0; n < A2; ++n) read_t(n);
#pragma unroll
      for (int n = 0; n < 4 * DB; ++n) {
        if constexpr (W == 128) __builtin_amdgcn_sched_barrier(0);
        if (n < 2 * DB) dv[n % DB] = mfma32(t[n % A2], n / DB % 2 ? p1 : p0, dv[n % DB]);
        else dk[n % DB] = mfma32(t[n % A2], n / DB % 2 ? ds1 : ds0, dk[n % DB]);
        if (n + A2 < 4 * DB) read_t(n + A2);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  typedef TileLoad<W, NW> Load;
  const Load lq(a.q.st, a.K, w, l), ld(a.d_o.st, a.V, w, l);
  // The stream: tiles of 64 rows from the last to the first, per tile the heads.  Of it the work-group takes pieces m0 .. m1 - 1.
  const int top = of.top, all = of.all;
  const int m0 = (int)((int64_t)all * blockIdx.y / parts), m1 = (int)((int64_t)all * (blockIdx.y + 1) / parts);
  struct Place { int m, h, i; } cur = {m0, m0 % G, (top - m0 / G) * CH}, next = cur;
  auto advance = [&](Place& x) { ++x.m; if (++x.h == G) { x.h = 0; x.i -= CH; } };
  float lse_ = 0.f, delta_ = 0.f;
  auto piece = [&](bf16* sq, bf16* sd, int i) __attribute__((always_inline)) {
    const int hq = hk * G + next.h;
    if (i < Load::PASSES) lq.load(sq, attn_row<bf16>(a.q, t.b, t.tok0 + next.i, hq), a.q.st, t.len - next.i, w, i);
    else ld.load(sd, attn_row<bf16>(a.d_o, t.b, t.tok0 + next.i, hq), a.d_o.st, t.len - next.i, w, i - Load::PASSES);
  };
  auto stats = [&] {
    if (tid < CH) {
      const int64_t row = ((int64_t)t.b * a.HQ + hk * G + next.h) * a.T + t.tok0 + next.i;
      const bool in = next.i + tid < t.len;
      lse_ = in ? (a.lse + row)[(uint32_t)tid] : INFINITY;
      delta_ = in ? (a.delta + row)[(uint32_t)tid] : 0.f;
    }
  };
  auto tile = [&](bf16* cq, bf16* cd, bf16* nq, bf16* nd, float (&rows)[2][CH]) __attribute__((always_inline)) {
    wait_all_loads();
    lq.clear(cq, t.len - cur.i, a.K, w, l);
    ld.clear(cd, t.len - cur.i, a.V, w, l);
    if (tid < CH) { rows[0][tid] = lse_; rows[1][tid] = delta_; }
    lds_barrier();
    if (next.m + 1 < m1) advance(next);                  // (behind the last piece: that one once more, so that there is no branch)
    stats();
    auto issue = [&](int point) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = point * 2 * Load::PASSES / 4; i < (point + 1) * 2 * Load::PASSES / 4; ++i) piece(nq, nd, i);
      __builtin_amdgcn_sched_barrier(0);
    };
    if (cur.i + CH > wbegin) {
      const Score16<CAP, BIAS> sc(a, hk * G + cur.h);
      block(sc, cq, cd, rows[0], rows[1], cur.i, issue);
    } else {
      issue(0); issue(1); issue(2); issue(3);
    }
    advance(cur);
  };
  if (CAP == NO_CAP && !BIAS && a.scale < 0.f) {
#pragma unroll
    for (int j = 0; j < KS; ++j) frag_negate(k[j]);
  }
  if (m0 < m1) {
#pragma unroll
    for (int i = 0; i < 2 * Load::PASSES; ++i) piece(s_q0, s_d0, i);
    stats();
  }
  while (cur.m < m1) {
    tile(s_q0, s_d0, s_q1, s_d1, s_row[0]);
    if (cur.m < m1) tile(s_q1, s_d1, s_q0, s_d0, s_row[1]);
  }
  wait_all_loads();                      // (none may arrive in an LDS that is another's)
  if (keys <= 0) return;
  if (parts == 1) {
    store_rows32<W>(dv, 1.0f, attn_row<bf16>(a.dv, t.b, t.tok0 + w0, hk), a.dv.st, keys, a.V, l);
    store_rows32<W>(dk, a.scale, attn_row<bf16>(a.dk, t.b, t.tok0 + w0, hk), a.dk.st, keys, a.K, l);
  } else {
    const int64_t rows = (int64_t)a.B * a.T * a.HKV, row = ((int64_t)t.b * a.T + t.tok0 + key_) * a.HKV + hk;
    float* sums = a.ws + ((int64_t)blockIdx.y * rows + row) * (a.K + a.V);
    if ((l & 31) < keys) {
      store_sums<W>(dk, a.scale, sums, a.K, g);
      store_sums<W>(dv, 1.0f, sums + a.K, a.V, g);
    }
  }
}

// dk and dv of a tile of KEYS keys that several work-groups shared, from their sums: [parts][B, T, HKV][K + V].
// A work-group takes JOIN_ROWS of the tile (blockIdx.y).
constexpr int JOIN_ROWS = 8;
template <typename T, int KEYS>
__global__ __launch_bounds__(NTHR) void k_attn_join(const lmoe_attn_args a, int most, int least) {
  AttnTile t;
  int hk;
  if (!attn_place<KEYS>(a, a.HKV, false, hk, t)) return;
  const int parts = KeyStream(a, t, most, least).parts, per = (a.K + a.V) / 4;
  if (parts == 1) return;
  const int64_t rows = (int64_t)a.B * a.T * a.HKV, first = ((int64_t)t.b * a.T + t.tok0 + t.r0) * a.HKV + hk;
  const int end = min((int)blockIdx.y * JOIN_ROWS + JOIN_ROWS, t.len - t.r0);
  for (int i = blockIdx.y * JOIN_ROWS * per + threadIdx.x; i < end * per; i += NTHR) {
    const int r = i / per, c = (i - r * per) * 4;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = 0; p < parts; ++p) x += *(const f32x4*)(a.ws + ((int64_t)p * rows + first + (int64_t)r * a.HKV) * (a.K + a.V) + c);
    store4(c < a.K ? attn_row<T>(a.dk, t.b, t.tok0 + t.r0 + r, hk) + c : attn_row<T>(a.dv, t.b, t.tok0 + t.r0 + r, hk) + c - a.K, x);
  }
}

}  // namespace lmoe
