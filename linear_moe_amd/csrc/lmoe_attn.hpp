// Softmax attention: what its kernels share.
//
//   x_ij = scale q_i . k_j                            (query head h reads key / value head h / (HQ / HKV))
//   x_ij = cap tanh(x_ij / cap)                       with a cap
//   s_ij = x_ij - slope_h |i - j|                     with slopes
//   allowed(i, j): same sequence and (not causal, or j <= i, or j < prefix of the sequence)
//   p_ij = 2^(log2(e) s_ij - lse_i),  lse_i = log2 sum_j e^{s_ij},   o_i = sum_j p_ij v_j
// Backward, with delta_i = do_i . o_i and dp_ij = do_i . v_j:
//   ds_ij = p_ij (dp_ij - delta_i) [(1 - tanh^2(x_ij / cap))]
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_{h, i} ds_ij q_i,   dv_j = sum_{h, i} p_ij do_i
// (stands where the reference's softmax layers call their attention core:
// linear_moe/sequence_modeling/attention/dot_product_attention.py:139-183).
//
// All exponents are to the base 2: log2(e) is a factor of the scale, the cap and the slope.  Statistics, the sums and the
// accumulators are fp32 (scores of 2^28 and more in size are past that: the rounding of one is a factor of 2^16 in its p).  Every row of a sequence is allowed to see itself (causal) or everything, so no row is empty;
// rows that a mask leaves nothing of inside one tile are handled by a finite lowest maximum (M_LOW): 2^(-inf - M_LOW) = 0.
#pragma once
#include <algorithm>

#include "lmoe_launch.hpp"
#include "lmoe_seq.hpp"

namespace lmoe {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float M_LOW = -1e30f;

// 1 - 2 / (1 + e^{2z}) is off by an ulp of 1 whatever tanh(z) itself is, and a score by an ulp of the cap: 1.2e-4 at a cap of 1024, a
// thirtieth of the rounding of p to a bfloat16.  The kernels on 2-byte elements take that form for caps up to it, and beyond it one whose
// error is relative (the near form would be off by 1.2e-3 in the score at a cap of 1e4, by 0.09 at 1e6).  It costs six operations more: 2 x
// 8192 tokens, 16 heads on 4 of 128, forward and backward 0.88 and 2.57 ms, with a near cap 0.69 to 0.77 and 2.18.
constexpr float CAP_NEAR = 1024.0f;
enum { NO_CAP, NEAR_CAP, FAR_CAP };
// Below 1/4 by the series, whose next term is 2^-27 of the sum; from there on the form above is off by 16 ulps of the number at most.
__device__ __forceinline__ float tanh_far(float z) {
  const float y = z * z;
  float x = __builtin_fmaf(y, 62.0f / 2835.0f, -17.0f / 315.0f);
  x = __builtin_fmaf(y, x, 2.0f / 15.0f);
  x = __builtin_fmaf(y, x, -1.0f / 3.0f);
  x = __builtin_fmaf(z * y, x, z);
  const float t = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * (2.0f * LOG2E))), 1.0f);
  return fabsf(z) < 0.25f ? x : t;
}
// (caps above 2^100 are as good as that one: the cap and scale / cap stay normal numbers)
__device__ __forceinline__ float cap_in_range(float softcap) { return fminf(softcap, 0x1p100f); }
// (finite for the least of caps as well: a product of 0 has a score of 0)
__device__ __forceinline__ float over_cap(float scale, float cap) {
  const float x = scale / cap;
  return fabsf(x) > 1e38f ? copysignf(1e38f, x) : x;
}

// What turns a product q . k into a score to the base 2.  CAP, BIAS: the call has a cap / slopes.
template <bool CAP, bool BIAS, bool FAST> struct Score {
  float mul;       // without a cap: scale log2(e);  with one: scale / cap
  float out;       // cap log2(e)
  float slope;     // slope log2(e)
  __device__ __forceinline__ Score(float scale, float softcap, const float* slopes, int h) {
    const float cap = cap_in_range(softcap);
    mul = CAP ? over_cap(scale, cap) : scale * LOG2E;
    out = cap * LOG2E;
    slope = BIAS ? slopes[h] * LOG2E : 0.f;
  }
  __device__ __forceinline__ Score(const lmoe_attn_args& a, int h) : Score(a.scale, a.softcap, a.slopes, h) {}
  // tanh(x / cap) of a product (fast: with the hardware's exponential and reciprocal)
  __device__ __forceinline__ float squash(float qk) const {
    if constexpr (FAST) return tanh_far(qk * mul);
    else return tanhf(qk * mul);
  }
  // dist = i - j, th = squash(qk) where there is a cap
  __device__ __forceinline__ float of(float qk, float th, float dist) const {
    float s = CAP ? th * out : qk * mul;
    if constexpr (BIAS) s = __builtin_fmaf(-slope, fabsf(dist), s);
    return s;
  }
};

// The same for the kernels on 2-byte elements, which keep a number u per pair that grows with the score, s = a u + b, so that a score
// less a maximum (or lse) is one multiply-add:  u = q . k (q negated for a negative scale);  with a cap up to CAP_NEAR
// u = -1 / (1 + e^{2x / cap}), tanh = 1 + 2 u, a = 2 b = 2 cap;  with one beyond u = tanh, a = cap, b = 0;  with slopes u = s.
template <int CAP, bool BIAS> struct Score16 {
  float mul, wide, slope, a, b;        // wide: cap times two, or the cap
  bool negate;
  __device__ __forceinline__ Score16(const lmoe_attn_args& x, int h) {
    const float cap = cap_in_range(x.softcap);
    negate = CAP == NO_CAP && !BIAS && x.scale < 0.f;
    mul = CAP == NEAR_CAP ? over_cap(x.scale, cap) * (2.0f * LOG2E) : CAP == FAR_CAP ? over_cap(x.scale, cap) : x.scale * LOG2E;
    wide = (CAP == FAR_CAP ? 1.0f : 2.0f) * cap * LOG2E;
    slope = BIAS ? x.slopes[h] * LOG2E : 0.f;
    // (a > 0 also for a scale of 0: a hidden score of -infinity stays one)
    a = BIAS ? 1.0f : CAP ? wide : fmaxf(fabsf(mul), 1e-37f);
    b = !BIAS && CAP == NEAR_CAP ? 0.5f * wide : 0.f;
  }
  // r: what fade() is made of; dist = i - j
  __device__ __forceinline__ float operator()(float qk, float dist, float& r) const {
    if constexpr (CAP == NEAR_CAP) r = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(qk * mul));
    if constexpr (CAP == FAR_CAP) r = tanh_far(qk * mul);
    if constexpr (BIAS) return __builtin_fmaf(-slope, fabsf(dist), CAP == NEAR_CAP ? __builtin_fmaf(r, wide, 0.5f * wide) : CAP == FAR_CAP ? r * wide : qk * mul);
    return CAP ? r : qk;
  }
  // the factor of the cap, 1 - tanh^2
  static __device__ __forceinline__ float fade(float r) { return CAP == NEAR_CAP ? -4.0f * __builtin_fmaf(r, r, r) : __builtin_fmaf(-r, r, 1.0f); }
};

// (to an ulp or so; what lies below 2^-126 becomes 0, beside numbers of which one is 1)
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// The sequence a tile of rows lies in, and the tile's first row inside it
struct AttnTile {
  int n, b;        // sequence, batch row
  int tok0, len;   // first token of the sequence inside the batch row, tokens of the sequence
  int r0;          // first row of the tile inside the sequence
  int prefix;      // tokens every row of the sequence sees (causal calls)
};
// Packed input of at most so many sequences is walked through by every work-group (64 sequences at a time) to find its tile; of
// more, the chunk map names 64-token chunks, a tile begins at every ROWS / 64-th of a sequence, and the work-groups of the
// other chunks leave.
constexpr int WALK_SEQS = 256;

// The tile of ROWS rows (a multiple of 64) and the head of H that the work-group takes.  from_end: the last tiles first (with a
// causal mask the late rows see most, and work-groups are dispatched in the order of their index; the keys of a causal call the
// other way round); of packed sequences the longest first, where the walk finds the tile.  The (row of the batch, head) pairs
// change fastest, so that neighbouring work-groups do alike; where their number allows it, an XCD (work-groups go round them) keeps
// the same pairs, and with them the same keys in its L2.  All lanes of the wave call it.
// STRIP < ROWS: the tile's strips of so many rows have work-groups of their own, one after the other; false for one without rows.
// fold: the strips (of one pair) behind the first so many come in the other order (attn_fold).
template <int ROWS, int STRIP = ROWS>
__device__ __forceinline__ bool attn_place(const lmoe_attn_args& a, int H, bool from_end, int& h, AttnTile& t, int fold = INT32_MAX) {
  const int pairs = a.cu_seqlens ? H : a.B * H, j = blockIdx.x / pairs, k = j < fold ? j : (int)gridDim.x / pairs - 1 - (j - fold);
  const int i = k / (ROWS / STRIP), strip = k % (ROWS / STRIP);
  int x = blockIdx.x - j * pairs;
  if (pairs % 8 == 0) x = (x & 7) * (pairs / 8) + (x >> 3);
  h = x % H;
  if (a.cu_seqlens && a.N <= WALK_SEQS) {
    int before = 0;
    for (int n0 = 0;; n0 += 64) {
      if (n0 >= a.N) return false;
      const int y = n0 + lane_id(), n = y < a.N ? (a.seq_order ? a.seq_order[y] : y) : 0;
      const int first = a.cu_seqlens[n], len = y < a.N ? a.cu_seqlens[n + 1] - first : 0, tiles = (len + ROWS - 1) / ROWS;
      int upto = tiles;                                    // tiles of the sequences up to the lane's
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int z = __shfl_up(upto, d, 64);
        if (lane_id() >= d) upto += z;
      }
      const uint64_t behind = __ballot(before + upto > i);
      if (behind) {
        const int l = __builtin_ctzll(behind), at = i - before - __shfl(upto, l, 64) + __shfl(tiles, l, 64);
        t.n = __shfl(n, l, 64); t.tok0 = __shfl(first, l, 64); t.len = __shfl(len, l, 64);
        t.r0 = (from_end ? (t.len + ROWS - 1) / ROWS - 1 - at : at) * ROWS;
        t.n = __builtin_amdgcn_readfirstlane(t.n); t.tok0 = __builtin_amdgcn_readfirstlane(t.tok0);
        t.len = __builtin_amdgcn_readfirstlane(t.len); t.r0 = __builtin_amdgcn_readfirstlane(t.r0);
        t.b = 0;
        break;
      }
      before += __shfl(upto, 63, 64);
    }
  } else if (a.cu_seqlens) {
    const int nt = a.nt_dev ? as_const(a.nt_dev)[0] : a.NT;
    const int c = from_end ? nt - 1 - i : i;
    if (c < 0 || c >= nt) return false;
    t.n = as_const(a.chunk_map)[2 * c];
    t.r0 = as_const(a.chunk_map)[2 * c + 1] * CH;
    if (t.r0 % ROWS) return false;
    t.b = 0;
    t.tok0 = as_const(a.cu_seqlens)[t.n];
    t.len = as_const(a.cu_seqlens)[t.n + 1] - t.tok0;
  } else {
    t.n = t.b = x / H;
    t.r0 = (from_end ? (a.T + ROWS - 1) / ROWS - 1 - i : i) * ROWS;
    t.tok0 = 0; t.len = a.T;
  }
  if constexpr (STRIP < ROWS) {
    t.r0 += (from_end ? ROWS / STRIP - 1 - strip : strip) * STRIP;
    if (t.r0 >= t.len) return false;
  }
  t.prefix = 0;
  if (a.prefix_lens) {
    const int p = as_const(a.prefix_lens)[t.n];
    t.prefix = p < 0 ? 0 : p > t.len ? t.len : p;
  }
  return true;
}
// tiles of a call, all rows of the batch together (packed input: no fewer)
template <int ROWS> inline int64_t attn_tiles(const lmoe_attn_args& a) {
  if (!a.cu_seqlens) return (int64_t)a.B * ((a.T + ROWS - 1) / ROWS);
  return a.N <= WALK_SEQS ? std::min<int64_t>((int64_t)a.T / ROWS + a.N, a.NT) : (int64_t)a.NT;
}
// Where the work-groups of a causal call come to a CU two at a time and all at once, the second of a CU is as much lighter than the
// average as the first is heavier if the second card-full comes lightest first (2 x 1000 tokens of fp32, 4 heads, forward: 25 -> 22 us).
inline int attn_fold(const lmoe_attn_args& a, int64_t groups, int H, int cus) {
  const int64_t pairs = (int64_t)a.B * H;
  return a.causal && !a.cu_seqlens && groups > cus && groups <= 2 * (int64_t)cus && cus % pairs == 0 ? (int)(cus / pairs) : INT32_MAX;
}
template <typename T> __device__ __forceinline__ void store4(T* p, f32x4 x) {
  typename ET<T>::vec4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = ET<T>::from_f(x[i]);
  *(typename ET<T>::vec4*)p = y;
}
template <typename T> __device__ __forceinline__ T* attn_row(const lmoe_tensor& x, int b, int t, int h) {
  return (T*)x.ptr + (int64_t)b * x.sb + (int64_t)t * x.st + (int64_t)h * x.sh;
}

// What the rounding of x to a bfloat16 leaves, in 2^-8 of its last place (of the bit pattern, so that it holds across a power of two
// as well), and the number again.  The backward pass takes delta = do . o from both: where few keys are seen, ds is a small
// difference of dp and delta, and the rounding of o alone would be as large in dq and dk as that of ds (documents of 8 tokens: off by
// 0.0029 of their size in place of 0.0024, 0.0017 of which is their own rounding).
__device__ __forceinline__ uint32_t low_byte(float x) {
  const int left = (int)(__builtin_bit_cast(uint32_t, x) - ((uint32_t)__builtin_bit_cast(uint16_t, (bf16)x) << 16));
  return (uint32_t)min((left + 128) >> 8, 127) & 0xff;
}
// byte i of low
__device__ __forceinline__ float with_low(bf16 x, uint32_t low, int i) {
  return __builtin_bit_cast(float, ((uint32_t)__builtin_bit_cast(uint16_t, x) << 16) + (uint32_t)((int)(low << (24 - 8 * i)) >> 24 << 8));
}

// Rows that belong to no sequence (packed input whose last offset is below T) are zero in the outputs: the work-groups of a
// launch share them.  out: [1, T, H, D] with D = V or K.
template <typename T> __device__ __forceinline__ void zero_behind(const lmoe_attn_args& a, const lmoe_tensor& x, int H, int D) {
  if (!a.cu_seqlens) return;
  const int end = as_const(a.cu_seqlens)[a.N];
  if (end >= a.T) return;
  const typename ET<T>::vec z = ET<T>::zero();
  const int per = H * (D / ET<T>::VEC);
  for (int t = end + blockIdx.x; t < a.T; t += gridDim.x)
    for (int i = threadIdx.x; i < per; i += blockDim.x) {
      const int h = i / (D / ET<T>::VEC), c = i % (D / ET<T>::VEC) * ET<T>::VEC;
      *(typename ET<T>::vec*)((T*)x.ptr + (int64_t)t * x.st + (int64_t)h * x.sh + c) = z;
    }
}

}  // namespace lmoe
