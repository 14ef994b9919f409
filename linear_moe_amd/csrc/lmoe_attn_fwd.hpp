// Softmax attention, forward pass on 2-byte elements.
//
// A work-group of four waves takes 128 rows of one query head; 64 keys and values at a time lie in LDS, twice: while the waves work
// on one pair of tiles, the next is loaded into the other.  Two work-groups share a CU, and no barrier holds them to one
// another: while one wave of a SIMD has the matrix unit, the other has the vector unit.  (One work-group of eight waves, 128 keys
// between two barriers: 2 x 8192 tokens, 16 heads of 128, 580 us in place of 556, of 64 362 in place of 322; with its two
// halves held half a step apart by barriers, and the tiles of one step in one phase, 20 % more.)
// A wave works on S^T = K Q^T (32 x 32 blocks of v_mfma_f32_32x32x16_bf16, q held in registers), so that a lane has one row of the
// scores (with its neighbour 32 lanes on): maximum, sum and scale factors are one number per lane.  O^T += V^T P^T takes P^T from
// the registers it is in (the contraction index may be numbered freely) and V^T through the transposing LDS read.
//
// Bound: the matrix rate and, as much, the vector unit's 32 exponentials and 170 other operations per 64 keys of a wave, which take it as
// long as the products take the matrix unit.  4 x 8192 tokens, 16 heads on 4 of 128, causal: 1.13 ms, 976 TFLOP/s (a product of 8192^3
// reaches 1133); with a cap, whose two more of the slow operations per score make the vector unit the longer, 760; heads of 64 840.
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

// A tile of rows of W columns in LDS, without padding: the 16-byte piece c of row r lies at piece c ^ f(r), so that neither 16 lanes that
// read one piece of 16 successive rows (A operands that contract over the columns) nor 32 lanes that read 64 bytes of four
// successive rows (the transposing read, for those that contract over the rows) meet in a bank.  (Rows padded by 16 bytes: the
// transposing reads lay in wait of each other for a quarter of the forward kernel's time.)
// Both kinds of address are a number per lane, xor a constant, plus a constant.
template <int W> struct Swz {
  static constexpr int RB = W * 2;
  static __device__ __forceinline__ int f(int r) { return W == 128 ? (r & 3) << 2 | (r >> 2 & 3) : (r >> 1 & 1) << 2 | (r >> 2 & 3); }
  int rows, cols;       // byte offsets of the lane
  __device__ __forceinline__ explicit Swz(int l) {
    rows = (l & 31) * RB + ((l >> 5 ^ f(l & 15)) << 4);
    const int s = l & 15, r = 4 * (l >> 5) + (s >> 2);
    cols = r * RB + ((2 * (l >> 4 & 1) + (s >> 1 & 1) ^ f(r)) << 4) + 8 * (s & 1);
  }
  // the same numbers, in a form the compiler cannot prove invariant: what is formed from them stays in the iteration, in place of
  // sixteen addresses in registers for the whole loop
  __device__ __forceinline__ Swz fresh() const {
    Swz x = *this;
    x.rows = fresh_index(x.rows); x.cols = fresh_index(x.cols);
    return x;
  }
  // row 32 b + l % 32, columns 16 j + 8 (l / 32) ..
  __device__ __forceinline__ bf16x8 frag(const bf16* tile, int b, int j) const {
    return *(const bf16x8*)((const char*)tile + (rows ^ 32 * j) + 32 * RB * b);
  }
  // 32 columns from 32 d, rows 16 x + 4 g + {0..3} and 16 x + 8 + 4 g + {0..3}, g = lane / 32 -- the numbering in which elements
  // 8 s .. 8 s + 7 of an accumulator block are a B operand
  __device__ __forceinline__ bf16x8 frag_t(const bf16* tile, int x, int d) const {
    typedef __attribute__((address_space(3))) bf16x4 lds_b4;
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4*)((const char*)tile + (cols ^ 64 * d) + 16 * RB * x));
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4*)((const char*)tile + (cols ^ 64 * d ^ 32) + 16 * RB * x + 8 * RB));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  static __device__ __forceinline__ const bf16* at(const bf16* tile, int r, int c) {
    return (const bf16*)((const char*)tile + r * RB + ((c >> 3 ^ f(r)) << 4) + 2 * (c & 7));
  }
};
// elements 8 s .. 8 s + 7 of an accumulator block as a B operand
__device__ __forceinline__ bf16x8 frag_of_acc(const f32x16& x, int s) {
  bf16x8 f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (bf16)x[8 * s + i];
  return f;
}

// Loads straight into LDS: a wave's instruction fills 1 KB, 16 bytes a lane, in the order of the lanes; the order of a row's pieces comes
// from the addresses the lanes read.  NW waves share a tile of 64 rows.  Rows at or behind nvalid repeat the last one and columns
// at or behind D the first, until clear() (once they have arrived) makes zeros of them.  Offsets inside a tile fit 32 bits: the
// launch sees to it.
typedef __attribute__((address_space(1))) const void global_void;
typedef __attribute__((address_space(3))) void lds_void;
template <int W, int NW> struct TileLoad {
  static constexpr int VPR = W / 8, RPI = 64 / VPR, PASSES = CH / RPI / NW;      // pieces per row, rows per instruction
  static_assert(PASSES * RPI * NW == CH && NW * RPI % 16 == 0, "whole passes; the order of the pieces repeats after 16 rows");
  int row, col;      // of the lane in the first pass
  uint32_t first;    // bytes
  __device__ __forceinline__ TileLoad(int64_t stride, int D, int w, int l) {
    row = w * RPI + l / VPR;
    col = (l % VPR ^ Swz<W>::f(row)) * 8;
    first = (col < D ? col : 0) * 2;
  }
  // pass p of the tile from src on (nvalid >= 1)
  __device__ __forceinline__ void load(bf16* tile, const bf16* src, int64_t stride, int nvalid, int w, int p) const {
    const uint32_t r = min(row + p * NW * RPI, nvalid - 1);
    __builtin_amdgcn_global_load_lds((global_void*)((const char*)src + (r * (uint32_t)(2 * stride) + first)), (lds_void*)(tile + (p * NW + w) * 512), 16, 0, 0);
  }
  __device__ __forceinline__ void clear(bf16* tile, int nvalid, int D, int w, int l) const {
    if (nvalid >= CH && D >= W) return;
#pragma unroll
    for (int p = 0; p < PASSES; ++p)
      if (row + p * NW * RPI >= nvalid || col >= D) *(bf16x8*)(tile + (p * NW + w) * 512 + l * 8) = ET<bf16>::zero();
  }
};

// The tiles of 64 keys and values that a work-group of ATTN_WAVES waves goes through.  The loads of a tile are spread over the products
// of the one before it, a quarter at each of four points: a CU takes 64 bytes a cycle, and waves that hand over a whole tile at once
// wait for each other in front of it.
constexpr int ATTN_WAVES = 4, ATTN_ROWS = 32 * ATTN_WAVES;
template <int W> struct KeyTiles {
  typedef TileLoad<W, ATTN_WAVES> Load;
  const lmoe_attn_args& a;
  const bf16 *kp, *vp;
  int len, last, step, w, l;       // last: first key of the last tile; step: keys from one tile to the next
  Load lk, lv;
  __device__ __forceinline__ KeyTiles(const lmoe_attn_args& a, const bf16* kp, const bf16* vp, int len, int end, int w, int l, int step = CH)
      : a(a), kp(kp), vp(vp), len(len), last((end - 1) / CH * CH), step(step), w(w), l(l), lk(a.k.st, a.K, w, l), lv(a.v.st, a.V, w, l) {}
  __device__ __forceinline__ void piece(bf16* sk, bf16* sv, int j0, int i) const {
    if (i < Load::PASSES) lk.load(sk, kp + (int64_t)j0 * a.k.st, a.k.st, len - j0, w, i);
    else lv.load(sv, vp + (int64_t)j0 * a.v.st, a.v.st, len - j0, w, i - Load::PASSES);
  }
  __device__ __forceinline__ void first(bf16* sk, bf16* sv, int j0 = 0) const {
#pragma unroll
    for (int i = 0; i < 2 * Load::PASSES; ++i) piece(sk, sv, min(j0, last), i);
  }
  // of the tile behind the one from j0 on (behind the last one: that once more, so that there is no branch)
  __device__ __forceinline__ void next(bf16* sk, bf16* sv, int j0, int point) const {
    const int j = min(j0 + step, last);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = point * 2 * Load::PASSES / 4; i < (point + 1) * 2 * Load::PASSES / 4; ++i) piece(sk, sv, j, i);
    __builtin_amdgcn_sched_barrier(0);
  }
  // the tile from j0 on is whole, for all waves
  __device__ __forceinline__ void arrived(bf16* sk, bf16* sv, int j0) const {
    wait_all_loads();
    lk.clear(sk, len - j0, a.K, w, l);
    lv.clear(sv, len - j0, a.V, w, l);
    lds_barrier();
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

// a transposed block of 32 rows and W columns (acc[b]: columns 32 b ..) to rows [0, rows) and columns [0, D) of dst: two lanes of a
// row exchange halves, so that each has 16 adjacent bytes
// low (or nullptr): [rows][D], what the rounding leaves (low_byte)
template <int W> __device__ __forceinline__ void store_rows32(const f32x16 (&acc)[W / 32], float mul, bf16* dst, int64_t stride, int rows, int D, int l, int8_t* low = nullptr) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  bf16* p = dst + (int64_t)(l & 31) * stride + 8 * (l >> 5);
#pragma unroll
  for (int b = 0; b < W / 32; ++b)
#pragma unroll
    for (int i = 0; i < 16; i += 8) {
      bf16x8 x;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (bf16)(acc[b][i + e] * mul);
      const u32x4 y = __builtin_bit_cast(u32x4, x);
      const u32x2 lo = __builtin_amdgcn_permlane32_swap(y[0], y[2], false, false), hi = __builtin_amdgcn_permlane32_swap(y[1], y[3], false, false);
      if ((l & 31) < rows && 32 * b + 2 * i + 8 * (l >> 5) < D) *(u32x4*)(p + 32 * b + 2 * i) = u32x4{lo[0], hi[0], lo[1], hi[1]};
      if (low) {
        uint32_t z[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e / 4] |= low_byte(acc[b][i + e] * mul) << 8 * (e % 4);
        const u32x2 q = __builtin_amdgcn_permlane32_swap(z[0], z[1], false, false);
        if ((l & 31) < rows && 32 * b + 2 * i + 8 * (l >> 5) < D) *(u32x2*)(low + (int64_t)(l & 31) * D + 32 * b + 2 * i + 8 * (l >> 5)) = q;
      }
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

// What the second group of waves of a work-group hands to the first: a block of 32 rows per wave, half of a lane's sums through either of
// two arrays of two tiles
template <int W> struct Handed {
  static constexpr int STRIDE = ATTN_WAVES * 64, HALF = W / 4;
  static_assert(HALF * STRIDE * 4 <= 2 * CH * W * 2, "half of the sums fit an array");
  float *const x, *const y;
  __device__ __forceinline__ Handed(bf16* p, bf16* q, int w, int l) : x((float*)p + (w * 64 + l)), y((float*)q + (w * 64 + l)) {}
  __device__ __forceinline__ float at(int i) const { return (i < HALF ? x : y)[i % HALF * STRIDE]; }
  __device__ __forceinline__ void put(const f32x16 (&acc)[W / 32]) const {
#pragma unroll
    for (int i = 0; i < 2 * HALF; ++i) (i < HALF ? x : y)[i % HALF * STRIDE] = acc[i / 16][i % 16];
  }
};

// KG: groups of ATTN_WAVES waves that go through the tiles of the same rows, each through every KG-th; the second hands its sums to the first.
template <int W, int KG, int CAP, bool BIAS>
__global__ __launch_bounds__(KG * ATTN_WAVES * 64, 2) void k_attn_fwd(const lmoe_attn_args a) {
  static_assert(KG == 1 || KG == 2, "one joins the other");
  constexpr int KS = W / 16, DB = W / 32, TILE = CH * W;
  // (arrays of their own, so that the compiler sees that reads of one tile need not wait for loads into the other)
  __shared__ __attribute__((aligned(1024))) bf16 a_k0[KG * TILE], a_v0[KG * TILE], a_k1[KG * TILE], a_v1[KG * TILE];
  zero_behind<bf16>(a, a.o, a.HQ, a.V);
  AttnTile t;
  int h;
  if (!attn_place<ATTN_ROWS>(a, a.HQ, true, h, t)) return;
  const int hk = h / (a.HQ / a.HKV), l = lane_id(), w = KG == 1 ? wave_id() : wave_id() % ATTN_WAVES, g = l >> 5;
  const int kg = KG == 1 ? 0 : wave_id() / ATTN_WAVES;
  bf16 *const s_k0 = a_k0 + kg * TILE, *const s_v0 = a_v0 + kg * TILE, *const s_k1 = a_k1 + kg * TILE, *const s_v1 = a_v1 + kg * TILE;
  const Score16<CAP, BIAS> sc(a, h);
  const Swz<W> lane(l);
  const int w0 = t.r0 + 32 * w, rows = t.len - w0;                   // the wave's first row, its rows (may be none)
  const int row_ = w0 + (l & 31);
  bf16x8 q[KS];
  rows32<W>(q, attn_row<bf16>(a.q, t.b, t.tok0 + min(w0, t.len - 1), h), a.q.st, max(rows, 1), a.K, l);
  if (sc.negate) {
#pragma unroll
    for (int j = 0; j < KS; ++j) frag_negate(q[j]);
  }
  f32x16 o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) o[b] = zero16();
  float m = M_LOW, sum = 0.f;

  const int end = a.causal ? min(t.len, max(t.r0 + ATTN_ROWS, t.prefix)) : t.len;       // keys that some row sees
  const int wend = rows <= 0 ? 0 : a.causal ? min(t.len, max(w0 + 32, t.prefix)) : t.len;
  const int whole = min(a.causal ? max(t.r0 + 1, t.prefix) : t.len, end);          // keys before it: seen by all rows
  const bf16* kp = attn_row<bf16>(a.k, t.b, t.tok0, hk);
  const bf16* vp = attn_row<bf16>(a.v, t.b, t.tok0, hk);

  // Fragments are read a phase ahead of their products: the second half of K under the products of the first, half of V before the
  // exponentials, the rest of it under the products of that half.
  auto block = [&](const bf16* sk, const bf16* sv, int j0, auto issue, auto part_c) __attribute__((always_inline)) {
    constexpr bool PART = decltype(part_c)::value;                   // some of the tile's keys are hidden from some rows
    const Swz<W> at = lane.fresh();
    const int row = fresh_index(row_);
    f32x16 s[2];
    bf16x8 kf[2][KS];
    auto read_k = [&](int b) {
#pragma unroll
      for (int j = 0; j < KS; ++j) kf[b][j] = at.frag(sk, b, j);
    };
    bf16x8 vf[2][2 * DB];
    auto read_v = [&](int b) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int d = 0; d < DB; ++d) vf[b][x * DB + d] = at.frag_t(sv, 2 * b + x, d);
    };
    read_k(0);
    __builtin_amdgcn_sched_barrier(0);
    read_k(1);
    s[0] = zero16(); s[1] = zero16();
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      s[0] = mfma32(kf[0][j], q[j], s[0]);
      s[1] = mfma32(kf[1][j], q[j], s[1]);
      if (j == KS / 2) issue(0);
    }
    issue(1);
    __builtin_amdgcn_sched_barrier(0);
    read_v(0);
    float mx = -INFINITY;
    const int sees = (a.causal ? min(t.len, max(row + 1, t.prefix)) : t.len) - j0;           // (keys from j0 on)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = j0 + 32 * b + row32(i) + 4 * g;
        float r, x = sc(s[b][i], (float)(row - j), r);
        if constexpr (PART) x = 32 * b + row32(i) < sees - 4 * g ? x : -INFINITY;
        s[b][i] = x;
        mx = fmaxf(mx, x);
      }
    const float next = fmaxf(m, __builtin_fmaf(sc.a, both_max(mx), sc.b)), f = pow2(m - next), off = sc.b - next;
    m = next;
    float part = 0.f;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = pow2(__builtin_fmaf(s[b][i], sc.a, off));
        part += s[b][i];
      }
    sum = __builtin_fmaf(sum, f, part);
#pragma unroll
    for (int b = 0; b < DB; ++b) o[b] *= f;
    __builtin_amdgcn_sched_barrier(0);
    read_v(1);
    issue(2);
    bool finite = true;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (b == 1) issue(3);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const bf16x8 p = frag_of_acc(s[b], x);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          bf16x8 v = vf[b][x * DB + d];
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
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (PART) {
      if (__any(!finite)) {                                          // ... and reach the rows that see them by themselves
        for (int j = 0; j < CH; ++j) {
          const bool ok = j < sees;
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float x = (float)*at.at(sv, j, 32 * d + row32(i) + 4 * g);
              if (ok && !(fabsf(x) < INFINITY)) o[d][i] += x;
            }
        }
      }
    }
  };

  KeyTiles<W> load(a, kp, vp, t.len, end, w, l, KG * CH);
  auto tile = [&](bf16* ck, bf16* cv, bf16* nk, bf16* nv, int j0, auto part_c) __attribute__((always_inline)) {
    load.arrived(ck, cv, j0);
    auto issue = [&](int point) __attribute__((always_inline)) { load.next(nk, nv, j0, point); };
    if (!decltype(part_c)::value || j0 < wend) block(ck, cv, j0, issue, part_c);
    else { issue(0); issue(1); issue(2); issue(3); }
  };
  load.first(s_k0, s_v0, kg * CH);
  // (two loops: with both bodies in one, the accumulators move between them.  The groups take the same number of steps, a last one for
  // nothing where the tiles do not come out even.)
  int j0 = 0;
  for (; j0 + 2 * KG * CH <= whole; j0 += 2 * KG * CH) {
    tile(s_k0, s_v0, s_k1, s_v1, j0 + kg * CH, std::false_type());
    tile(s_k1, s_v1, s_k0, s_v0, j0 + (KG + kg) * CH, std::false_type());
  }
  for (; j0 < end; j0 += 2 * KG * CH) {
    tile(s_k0, s_v0, s_k1, s_v1, j0 + kg * CH, std::true_type());
    if (j0 + KG * CH < end) tile(s_k1, s_v1, s_k0, s_v0, j0 + (KG + kg) * CH, std::true_type());
  }
  wait_all_loads();                      // (none may arrive in an LDS that is another's)
  sum = both_sum(sum);
  if constexpr (KG == 2) {
    const Handed<W> x(a_k0, a_v0, w, l);
    float* const st = (float*)a_k1 + (w * 64 + l);
    lds_barrier();
    if (kg == 1) { x.put(o); st[0] = m; st[x.STRIDE] = sum; }
    lds_barrier();
    if (kg == 1) return;
    const float m1 = st[0], next = fmaxf(m, m1), f0 = pow2(m - next), f1 = pow2(m1 - next);
#pragma unroll
    for (int i = 0; i < 16 * DB; ++i) o[i / 16][i % 16] = o[i / 16][i % 16] * f0 + x.at(i) * f1;
    sum = sum * f0 + st[x.STRIDE] * f1;
    m = next;
  }
  if (a.lse && g == 0 && row_ < t.len) a.lse[((int64_t)t.b * a.HQ + h) * a.T + t.tok0 + row_] = m + __builtin_amdgcn_logf(sum);
  if (rows > 0)
    store_rows32<W>(o, 1.0f / sum, attn_row<bf16>(a.o, t.b, t.tok0 + w0, h), a.o.st, rows, a.V, l,
                    a.o_low ? a.o_low + (((int64_t)t.b * a.HQ + h) * a.T + t.tok0 + w0) * a.V : nullptr);
}

}  // namespace lmoe
