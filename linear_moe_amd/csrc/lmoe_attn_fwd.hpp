// Softmax attention, forward pass on 2-byte elements.
//
// A work-group of NW waves takes NW x 32 rows of one query head; 64 keys and values at a time lie in LDS, twice: while the
// waves work on one pair of tiles, the next is written from registers into the other and the one after it is on its way
// into those registers.  A wave works on S^T = K Q^T (32 x 32 blocks of v_mfma_f32_32x32x16_bf16, q held in registers), so
// that a lane has one row of the scores (with its neighbour 32 lanes on): maximum, sum and scale factors are one number per
// lane.  O^T += V^T P^T takes P^T from the registers it is in (the contraction index may be numbered freely) and V^T through
// the transposing LDS read.
//
// The running maximum is raised (and O, sum scaled) only when a row exceeds it by more than 2^8: p <= 256 then, which changes
// neither the relative rounding of p nor that of the sums.
#pragma once
#include "lmoe_attn.hpp"

namespace lmoe {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}
// row of element i of a 32 x 32 accumulator block (its column is lane % 32)
__device__ __forceinline__ constexpr int row32(int i) { return (i & 3) + 8 * (i >> 2); }      // + 4 (lane / 32)
// the lane's number of the lane 32 further on (or back), both ways round
__device__ __forceinline__ void halves(float x, float& lo, float& hi) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  lo = __builtin_bit_cast(float, (uint32_t)r[0]); hi = __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ float both_max(float x) { float a, b; halves(x, a, b); return fmaxf(a, b); }
__device__ __forceinline__ float both_sum(float x) { float a, b; halves(x, a, b); return a + b; }

// A operand of a product that contracts over the rows of a tile (32 of its columns, from n0): the rows k0 + 4 g + {0..3} and
// k0 + 8 + 4 g + {0..3}, g = lane / 32 -- the numbering in which elements 8 s .. 8 s + 7 of an accumulator block are a B operand.
__device__ __forceinline__ bf16x8 frag32_t(const bf16* tile, int ld, int k0, int n0, int l) {
  const int s = l & 15;
  const bf16* p = tile + (k0 + 4 * (l >> 5) + (s >> 2)) * ld + n0 + 16 * ((l >> 4) & 1) + 4 * (s & 3);
  typedef __attribute__((address_space(3))) bf16x4 lds_b4;
  const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4*)p);
  const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4*)(p + 8 * ld));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// elements 8 s .. 8 s + 7 of an accumulator block as a B operand
__device__ __forceinline__ bf16x8 frag_of_acc(const f32x16& x, int s) {
  bf16x8 f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (bf16)x[8 * s + i];
  return f;
}

// ROWS rows of W columns on their way from memory to LDS, NT threads: rows at or behind nvalid and columns at or behind D
// arrive as zeros.
template <int ROWS, int W, int NT> struct RowStage {
  static constexpr int VPR = W / 8, PASSES = ROWS * VPR / NT, LD = W + LPAD;
  static_assert(PASSES * NT == ROWS * VPR, "whole passes");
  bf16x8 v[PASSES];
  __device__ __forceinline__ void load(const bf16* src, int64_t stride, int nvalid, int D, int tid) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int idx = p * NT + tid, c = idx % VPR * 8;
      const int r = min(idx / VPR, nvalid - 1);
      v[p] = *(const bf16x8*)(src + (int64_t)r * stride + (c < D ? c : 0));
    }
  }
  __device__ __forceinline__ void store(bf16* tile, int nvalid, int D, int tid) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int idx = p * NT + tid, r = idx / VPR, c = idx % VPR * 8;
      frag_keep_if(v[p], r < nvalid && c < D);
      *(bf16x8*)(tile + r * LD + c) = v[p];
    }
  }
};

// 32 rows of W columns as B operands (lane: row l % 32, columns 16 j + 8 (l / 32) ..), rows at or behind `rows` repeat the last
template <int W> __device__ __forceinline__ void rows32(bf16x8 (&f)[W / 16], const bf16* src, int64_t stride, int rows, int D, int l) {
  const bf16* p = src + (int64_t)min(l & 31, rows - 1) * stride + 8 * (l >> 5);
#pragma unroll
  for (int j = 0; j < W / 16; ++j) {
    f[j] = ET<bf16>::zero();
    if (16 * j + 8 * (l >> 5) < D) f[j] = *(const bf16x8*)(p + 16 * j);
  }
}

// a transposed block of 32 rows and W columns (acc[b]: columns 32 b ..) to rows [0, rows) and columns [0, D) of dst, through a
// strip of LDS that only this wave uses
template <int W> __device__ __forceinline__ void store_rows32(const f32x16 (&acc)[W / 32], float mul, bf16* strip, bf16* dst, int64_t stride, int rows, int D, int l) {
  constexpr int LD = W + LPAD;
#pragma unroll
  for (int b = 0; b < W / 32; ++b)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      bf16x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (bf16)(acc[b][i + e] * mul);
      *(bf16x4*)(strip + (l & 31) * LD + 32 * b + row32(i) + 4 * (l >> 5)) = x;
    }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
  for (int i = 0; i < 32 * (W / 8) / 64; ++i) {
    const int idx = i * 64 + l, r = idx / (W / 8), c = idx % (W / 8) * 8;
    if (r < rows && c < D) *(bf16x8*)(dst + (int64_t)r * stride + c) = *(const bf16x8*)(strip + r * LD + c);
  }
}

__device__ __forceinline__ bool all_finite(const bf16x8& f) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 w = __builtin_bit_cast(u32x4, f);
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) ok &= (w[i] & 0x7f80u) != 0x7f80u && (w[i] & 0x7f800000u) != 0x7f800000u;
  return ok;
}

template <int W, int NW, bool CAP, bool BIAS>
__global__ __launch_bounds__(NW * 64, 2) void k_attn_fwd(const lmoe_attn_args a) {
  constexpr int LD = W + LPAD, KS = W / 16, DB = W / 32, NT = NW * 64, ROWS = NW * 32, TILE = CH * LD;
  typedef RowStage<CH, W, NT> St;
  __shared__ __attribute__((aligned(16))) bf16 s_kv[4 * TILE];       // K, V of even tiles, of odd tiles
  static_assert(ROWS * LD <= 4 * TILE, "the strips of the waves");
  zero_behind<bf16>(a, a.o, a.HQ, a.V);
  AttnTile t;
  int h;
  if (!attn_place<ROWS>(a, a.HQ, true, h, t)) return;
  const int hk = h / (a.HQ / a.HKV), tid = threadIdx.x, l = lane_id(), w = wave_id(), g = l >> 5;
  const Score<CAP, BIAS, true> sc(a, h);
  const int w0 = t.r0 + 32 * w, rows = t.len - w0;                   // the wave's first row, its rows (may be none)
  const int row = w0 + (l & 31);
  bf16x8 q[KS];
  rows32<W>(q, attn_row<bf16>(a.q, t.b, t.tok0 + min(w0, t.len - 1), h), a.q.st, max(rows, 1), a.K, l);
  f32x16 o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) o[b] = zero16();
  float m = M_LOW, sum = 0.f;

  const int end = a.causal ? min(t.len, max(t.r0 + ROWS, t.prefix)) : t.len;       // keys that some row sees
  const int wend = rows <= 0 ? 0 : a.causal ? min(t.len, max(w0 + 32, t.prefix)) : t.len;
  const int whole = a.causal ? max(w0 + 1, t.prefix) : t.len;                      // keys before it: seen by all rows of the wave
  const bf16* kp = attn_row<bf16>(a.k, t.b, t.tok0, hk);
  const bf16* vp = attn_row<bf16>(a.v, t.b, t.tok0, hk);

  auto block = [&](const bf16* sk, const bf16* sv, int j0, auto part_c) {
    constexpr bool PART = decltype(part_c)::value;                   // some of the tile's keys are hidden from some rows
    f32x16 s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = zero16();
#pragma unroll
      for (int j = 0; j < KS; ++j) s[b] = mfma32(*(const bf16x8*)(sk + (32 * b + (l & 31)) * LD + 16 * j + 8 * g), q[j], s[b]);
    }
    float mx = M_LOW;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = j0 + 32 * b + row32(i) + 4 * g;
        float x = sc.of(s[b][i], CAP ? sc.squash(s[b][i]) : 0.f, (float)(row - j));
        if constexpr (PART) x = j < t.len && (!a.causal || j <= row || j < t.prefix) ? x : -INFINITY;
        s[b][i] = x;
        mx = fmaxf(mx, x);
      }
    mx = both_max(mx);
    if (__any(mx > m + 8.0f)) {
      const float next = mx > m + 8.0f ? mx : m, f = pow2<true>(m - next);      // (row by row: what a row gets depends on no other)
      m = next;
      sum *= f;
#pragma unroll
      for (int b = 0; b < DB; ++b) o[b] *= f;
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = pow2<true>(s[b][i] - m);
        sum += s[b][i];
      }
    bool finite = true;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const bf16x8 p = frag_of_acc(s[b], x);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          bf16x8 v = frag32_t(sv, LD, 32 * b + 16 * x, 32 * d, l);
          if constexpr (PART) {
            // A product with 0 for what the mask hides would make NaN of a hidden NaN or infinity: such numbers are left out here ...
            if (!all_finite(v)) {
              finite = false;
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = fabsf((float)v[e]) < INFINITY ? v[e] : (bf16)0.0f;
            }
          }
          o[d] = mfma32(v, p, o[d]);
        }
      }
    if constexpr (PART) {
      if (__any(!finite)) {                                          // ... and reach the rows that see them by themselves
        for (int j = 0; j < CH; ++j) {
          const bool ok = j0 + j < t.len && (!a.causal || j0 + j <= row || j0 + j < t.prefix);
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float x = (float)sv[j * LD + 32 * d + row32(i) + 4 * g];
              if (ok && !(fabsf(x) < INFINITY)) o[d][i] += x;
            }
        }
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
  sum = both_sum(sum);
  if (a.lse && g == 0 && row < t.len) a.lse[((int64_t)t.b * a.HQ + h) * a.T + t.tok0 + row] = m + __builtin_amdgcn_logf(sum);
  lds_barrier();
  if (rows > 0)
    store_rows32<W>(o, 1.0f / sum, s_kv + w * 32 * LD, attn_row<bf16>(a.o, t.b, t.tok0 + w0, h), a.o.st, rows, a.V, l);
}

}  // namespace lmoe
