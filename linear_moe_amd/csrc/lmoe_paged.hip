// One new token per sequence over a paged cache of keys and values (include/lmoe.h, lmoe_paged_args), and the writing of the
// cache.
//
// k_paged_attn: a work-group of four or eight waves takes up to 16 query heads of one key head and a stretch of the sequence's cache;
// each wave takes 32 positions at a time.  Everything a product needs lies in the wave's registers as it comes from memory:
//   S^T [32 keys][16 heads] = K Q^T:  the rows of K are the A operand (lane l: key l % 16, eight columns), 16 keys twice;
//     the result leaves lane l with head l % 16 and the keys 4g + e and 16 + 4g + e (g = l / 16, e = 0..3);
//   O^T [V columns][16 heads] += V^T P^T:  P^T as it is (the contraction index may be numbered freely, so those eight keys are the
//     lane's share), and V^T from the lane's own loads: lane l loads those eight keys at columns VW n .. VW n + VW - 1
//     (n = l % 16, VW = W / 16), so element i of all eight is the A operand whose row n is column VW n + i.
// So there is no LDS traffic and no barrier per step, and 16 lanes read 256 adjacent bytes of a value row.
// HBM-bound: the keys and values of the live tokens are read once for all heads that share them.
// The stretches of a sequence are joined by k_paged_join where there is more than one.
#include "lmoe_attn.hpp"

namespace lmoe {

constexpr int PSTEP = 32;              // positions a wave takes at a time
constexpr int PHEADS = 16;             // query heads of a work-group
constexpr int PSPLITS = 2048;          // stretches of a sequence at most

struct PagedPlan {
  int splits;      // stretches per sequence at most
  int chunk;       // positions of a stretch at least
  int waves;       // of a work-group
  int blocks;      // work-groups that share a key head's query heads
  uint32_t div_m;  // j / S = (umulhi(j, div_m) + j) >> div_s for 0 <= j < 2^31
  int div_s;
};
static PagedPlan paged_plan(const lmoe_paged_args& a) {
  PagedPlan p;
  p.blocks = (a.HQ / a.HKV + PHEADS - 1) / PHEADS;
  const int64_t bound = (int64_t)a.M * a.S + 1, groups = (int64_t)a.N * a.HKV * p.blocks;
  // A short cache: one stretch of eight waves, at most four steps each, and no second launch (one sequence of 500 tokens, 16 / 4
  // heads of 128: 9.2 us, in stretches of 256 and joined 13).  4-byte elements have no registers for eight waves.
  // Else stretches of one length, whatever the call: us for stretches of 256, 384, 512, 1024 positions (64 sequences of 1024 to 4096
  // tokens, 32 / 8 heads of 128; 2 of 32 K and 128 K, 16 / 4 heads of 128; 9 of 750 to 3001 tokens, 12 / 3 heads of 64,
  // 4-byte elements): 140 135 134 136; 80 76 74 78; 20.3 17.4 19.9 31.1.
  // (a launch has less than 2^32 threads: of 2^23 work-groups and more, which N * HQ < 2^24 allows, none has 512)
  p.waves = a.dtype == LMOE_BF16 && bound <= 1024 && groups < 1 << 23 ? 8 : 4;
  const int64_t chunk = p.waves == 8 ? 1024 : a.dtype == LMOE_BF16 ? 512 : 384;
  int64_t splits = (bound + chunk - 1) / chunk;
  const int64_t most = groups * PSPLITS <= 16384 ? PSPLITS : groups >= 16384 ? 1 : 16384 / groups;
  p.splits = (int)(splits < most ? splits : most);
  p.chunk = (int)chunk;
  p.div_s = 0;
  while ((1ll << p.div_s) < a.S) ++p.div_s;
  p.div_m = (uint32_t)((((1ull << p.div_s) - (uint64_t)a.S) << 32) / (uint64_t)a.S + 1);
  return p;
}
int64_t paged_attn_floats(const lmoe_paged_args& a) {
  const PagedPlan p = paged_plan(a);
  // per (sequence, head, stretch): V columns; behind them all the maxima and sums
  return p.splits > 1 ? (int64_t)a.N * a.HQ * p.splits * (a.V + 2) : 0;
}

// Tokens the new one attends to in the cache, and the length of a stretch
struct PagedSeq { int len, chunk, used; };
__device__ __forceinline__ PagedSeq paged_seq(const lmoe_paged_args& a, const PagedPlan& p, int n) {
  PagedSeq s;
  const int step = p.waves * PSTEP;
  const int len = as_const(a.lens)[n], room = a.M * a.S;
  s.len = len < 0 ? 0 : len > room ? room : len;
  const int total = s.len + (a.kn.ptr ? 1 : 0);
  const int per = (total + p.splits - 1) / p.splits;
  s.chunk = per <= p.chunk ? p.chunk : (per + step - 1) / step * step;
  s.used = (total + s.chunk - 1) / s.chunk;
  return s;
}

template <typename T, int W> struct PagedTile {
  static constexpr int KS = W / 32, VW = W / 16, PIECE = VW < ET<T>::VEC ? VW : ET<T>::VEC;
  typedef T piece __attribute__((ext_vector_type(PIECE)));
  typename ET<T>::frag k[2][KS];
  piece v[8][VW / PIECE];
  uint32_t live;         // which of the 32 positions exist
};

template <typename T> __device__ __forceinline__ typename ET<T>::frag zero_frag() {
  typename ET<T>::frag f;
  if constexpr (sizeof(T) == 2) f = ET<T>::zero(); else { f.lo = ET<T>::zero(); f.hi = ET<T>::zero(); }
  return f;
}
// eight columns from d of a row of D (a multiple of 16 bytes), zeros behind its end
template <typename T, bool ALL> __device__ __forceinline__ typename ET<T>::frag load_cols(const T* row, int d, int D) {
  if constexpr (ALL) return ET<T>::load_frag(row + d);
  typename ET<T>::frag f = zero_frag<T>();
  if constexpr (sizeof(T) == 2) { if (d < D) f = ET<T>::load_frag(row + d); }
  else { if (d < D) f.lo = *(const f32x4*)(row + d); if (d + 4 < D) f.hi = *(const f32x4*)(row + d + 4); }
  return f;
}

// ALL: the head dimension of q and k is W.
template <typename T, int W, int NW, bool CAP, bool BIAS, bool ALL>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 ? 2 : 1) void k_paged_attn(const lmoe_paged_args a, const PagedPlan p) {
  typedef PagedTile<T, W> Tile;
  constexpr int KS = Tile::KS, VW = Tile::VW, PIECE = Tile::PIECE;
  constexpr bool FAST = sizeof(T) == 2;
  constexpr int PGROUP = NW * PSTEP;        // positions the work-group takes at a time
  typedef typename Tile::piece piece;
  __shared__ __attribute__((aligned(16))) float s_o[NW][PHEADS][W + 4];
  __shared__ float s_m[NW][PHEADS], s_l[NW][PHEADS];
  // The stretches of one head follow each other in the grid, so that an XCD (work-groups go round them) has stretches of all
  // heads: with the heads next to each other, each XCD had some heads only, and those of the longest sequence took their
  // XCDs' time (the two documents of the comment above: 94 -> 74 us).
  const int part = blockIdx.x % p.splits, group = blockIdx.x / p.splits;
  const int n = group / (a.HKV * p.blocks), hb = group % (a.HKV * p.blocks), hk = hb / p.blocks, G = a.HQ / a.HKV;
  const int h0 = hb % p.blocks * PHEADS, heads = min(PHEADS, G - h0);      // of the key head's group
  const PagedSeq sq = paged_seq(a, p, n);
  const int total = sq.len + (a.kn.ptr ? 1 : 0), begin = part * sq.chunk;
  if (begin >= total && part > 0) return;
  const int end = min(total, begin + sq.chunk);
  const int l = lane_id(), w = wave_id(), c = l & 15, g = l >> 4;
  const int32_t* table = a.table + (int64_t)n * a.table_stride;
  const T* kp = (const T*)a.kp.ptr + (int64_t)hk * a.kp.sh;
  const T* vp = (const T*)a.vp.ptr + (int64_t)hk * a.vp.sh;
  const T* kn = a.kn.ptr ? (const T*)a.kn.ptr + (int64_t)n * a.kn.sb + (int64_t)hk * a.kn.sh : nullptr;
  const T* vn = a.kn.ptr ? (const T*)a.vn.ptr + (int64_t)n * a.vn.sb + (int64_t)hk * a.vn.sh : nullptr;

  // Where the lane's position (j0 + l % 32) lies.  A page number is asked for two steps before its rows are used and one before they
  // are asked for, in front of the rows of the step between: loads return in order, so that waiting for it waits for no rows.
  struct Where { int id, slot; };
  auto ask = [&](int j0) {
    Where x = {-1, 0};
    const int j = j0 + (l & 31);
    if (j < min(sq.len, end)) {
      const int col = (int)((__umulhi((uint32_t)j, p.div_m) + (uint32_t)j) >> p.div_s);
      x.slot = j - col * a.S;
      x.id = table[col];
    }
    return x;
  };
  auto load = [&](Tile& t, int j0, const Where& x) {
    // offsets of the lane's position, and the other lanes' through the LDS crossbar.  The new token: its own rows.
    const bool there = x.id >= 0 && x.id < a.P, fresh = j0 + (l & 31) == sq.len && sq.len < end;
    const int id = there ? x.id : 0;
    const T* kr = fresh ? kn : kp + (int64_t)id * a.kp.sb + (int64_t)x.slot * a.kp.st;
    const T* vr = fresh ? vn : vp + (int64_t)id * a.vp.sb + (int64_t)x.slot * a.vp.st;
    t.live = (uint32_t)__ballot(there || fresh);
    const uint64_t ki = (uint64_t)(uintptr_t)kr, vi = (uint64_t)(uintptr_t)vr;
    auto of = [&](uint64_t v, int lane) {
      const uint32_t lo = __shfl((int)(uint32_t)v, lane, 64), hi = __shfl((int)(uint32_t)(v >> 32), lane, 64);
      return (const T*)(uintptr_t)((uint64_t)hi << 32 | lo);
    };
    const T* kq[2];
    const T* vq[8];
#pragma unroll
    for (int b = 0; b < 2; ++b) kq[b] = of(ki, 16 * b + c);
#pragma unroll
    for (int e = 0; e < 8; ++e) vq[e] = of(vi, 16 * (e >> 2) + 4 * g + (e & 3));
    const int vc = VW * c;
    if (t.live == ~0u) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < KS; ++j) t.k[b][j] = load_cols<T, ALL>(kq[b], 32 * j + 8 * g, a.K);
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < VW; i += PIECE)
          // (columns behind the head dimension: any of the row, they are not stored)
          t.v[e][i / PIECE] = *(const piece*)(vq[e] + (vc + i < a.V ? vc + i : 0));
    } else {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          t.k[b][j] = zero_frag<T>();
          if (t.live >> (16 * b + c) & 1) t.k[b][j] = load_cols<T, ALL>(kq[b], 32 * j + 8 * g, a.K);
        }
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < VW; i += PIECE) {
          piece y;
#pragma unroll
          for (int z = 0; z < PIECE; ++z) y[z] = (T)0.0f;
          if (t.live >> (16 * (e >> 2) + 4 * g + (e & 3)) & 1) y = *(const piece*)(vq[e] + (vc + i < a.V ? vc + i : 0));
          t.v[e][i / PIECE] = y;
        }
    }
  };

  int j0 = begin + PSTEP * w;
  Where at = ask(j0), ahead = ask(j0 + PGROUP);

  // the new token into its page: by the work-group whose stretch ends with it
  if (kn && end == total && h0 == 0) {
    const int page = sq.len / a.S, slot = sq.len % a.S;
    const bool there = as_const(a.lens)[n] == sq.len && page < a.M;
    const int id = there ? as_const(table)[page] : -1;
    if (id >= 0 && id < a.P) {
      T* kd = (T*)a.kp.ptr + (int64_t)id * a.kp.sb + (int64_t)slot * a.kp.st + (int64_t)hk * a.kp.sh;
      T* vd = (T*)a.vp.ptr + (int64_t)id * a.vp.sb + (int64_t)slot * a.vp.st + (int64_t)hk * a.vp.sh;
      if ((int)threadIdx.x < a.K) kd[threadIdx.x] = kn[threadIdx.x];
      else if (threadIdx.x >= 128 && (int)threadIdx.x - 128 < a.V) vd[threadIdx.x - 128] = vn[threadIdx.x - 128];
    }
  }

  typename ET<T>::frag q[KS];
  const int hq = hk * G + h0 + min(c, heads - 1);
  {
    const T* row = (const T*)a.q.ptr + (int64_t)n * a.q.sb + (int64_t)hq * a.q.sh;
#pragma unroll
    for (int j = 0; j < KS; ++j) q[j] = load_cols<T, ALL>(row, 32 * j + 8 * g, a.K);
  }
  const Score<CAP, BIAS, FAST> sc(a.scale, a.softcap, a.slopes, hq);

  f32x4 o[VW];
#pragma unroll
  for (int i = 0; i < VW; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = M_LOW, sum = 0.f;
  auto take = [&](const Tile& t, int j0) {
    f32x4 s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KS; ++j) ET<T>::mma(s[b], t.k[b][j], q[j]);
    }
    float mx = M_LOW;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = j0 + 16 * b + 4 * g + e;
        const float x = sc.of(s[b][e], CAP ? sc.squash(s[b][e]) : 0.f, (float)(total - 1 - j));
        s[b][e] = t.live >> (16 * b + 4 * g + e) & 1 ? x : -INFINITY;
        mx = fmaxf(mx, s[b][e]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float next = fmaxf(m, mx), f = pow2(m - next);
    m = next;
    sum *= f;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[b][e] = pow2(s[b][e] - m);
        sum += s[b][e];
      }
    // (P rounded to the element type, as the products take it; the sum is of the numbers before)
    typename ET<T>::frag pf;
    if constexpr (FAST) pf = frag_of_blocks(s[0], s[1]); else { pf.lo = s[0]; pf.hi = s[1]; }
#pragma unroll
    for (int i = 0; i < VW; ++i) {
      o[i] *= f;
      typename ET<T>::frag vf;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const T x = t.v[e][i / PIECE][i % PIECE];
        if constexpr (FAST) vf[e] = x; else { if (e < 4) vf.lo[e] = x; else vf.hi[e - 4] = x; }
      }
      ET<T>::mma(o[i], vf, pf);
    }
  };

  Tile t[2];
  if (j0 < end) load(t[0], j0, at);
  while (j0 < end) {
    at = ahead;
    ahead = ask(j0 + 2 * PGROUP);
    if (j0 + PGROUP < end) load(t[1], j0 + PGROUP, at);
    take(t[0], j0);
    j0 += PGROUP;
    if (j0 >= end) break;
    at = ahead;
    ahead = ask(j0 + 2 * PGROUP);
    if (j0 + PGROUP < end) load(t[0], j0 + PGROUP, at);
    take(t[1], j0);
    j0 += PGROUP;
  }

  // the waves together: lane (c, g) holds head c, columns VW (4g + r) + i
  sum += __shfl_xor(sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  if (g == 0) { s_m[w][c] = m; s_l[w][c] = sum; }
#pragma unroll
  for (int i = 0; i < VW; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) s_o[w][c][VW * (4 * g + r) + i] = o[i][r];
  __syncthreads();
  for (int idx = threadIdx.x; idx < heads * W; idx += NW * 64) {
    const int hh = idx / W, d = idx % W;
    if (d >= a.V) continue;
    float mm = M_LOW;
#pragma unroll
    for (int y = 0; y < NW; ++y) mm = fmaxf(mm, s_m[y][hh]);
    float ll = 0.f, x = 0.f;
#pragma unroll
    for (int y = 0; y < NW; ++y) {
      const float f = pow2(s_m[y][hh] - mm);
      ll += f * s_l[y][hh];
      x += f * s_o[y][hh][d];
    }
    const int h = hk * G + h0 + hh;
    if (sq.used <= 1) {
      ((T*)a.o.ptr)[(int64_t)n * a.o.sb + (int64_t)h * a.o.sh + d] = ET<T>::from_f(ll != 0.f ? x / ll : 0.f);
    } else {
      const int64_t at = ((int64_t)n * a.HQ + h) * p.splits + part, rows = (int64_t)a.N * a.HQ * p.splits;
      a.ws[at * a.V + d] = x;
      if (d == 0) *(f32x2*)(a.ws + rows * a.V + 2 * at) = f32x2{mm, ll};
    }
  }
}

// The stretches of one (sequence, head) joined: o = sum 2^(m_s - m) x_s / sum 2^(m_s - m) l_s.  Eight rows of 32 lanes, four columns a
// lane; a row takes every eighth stretch.
template <typename T>
__global__ __launch_bounds__(NTHR) void k_paged_join(const lmoe_paged_args a, const PagedPlan p) {
  __shared__ float s_f[PSPLITS], s_r[NTHR / 64];
  __shared__ __attribute__((aligned(16))) f32x4 s_x[8][32];
  const int n = blockIdx.x / a.HQ, h = blockIdx.x % a.HQ, tid = threadIdx.x;
  const PagedSeq sq = paged_seq(a, p, n);
  if (sq.used <= 1) return;
  const int64_t at = ((int64_t)n * a.HQ + h) * p.splits, rows = (int64_t)a.N * a.HQ * p.splits;
  const f32x2* ml = (const f32x2*)(a.ws + rows * a.V) + at;
  float m = M_LOW;
  for (int s = tid; s < sq.used; s += NTHR) m = fmaxf(m, ml[s][0]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  if ((tid & 63) == 0) s_r[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_r[0], s_r[1]), fmaxf(s_r[2], s_r[3]));
  float ll = 0.f;
  for (int s = tid; s < sq.used; s += NTHR) {
    const f32x2 y = ml[s];
    const float f = pow2(y[0] - m);
    s_f[s] = f;
    ll += f * y[1];
  }
  ll = wave_sum(ll);
  __syncthreads();                       // s_r has been read, s_f is whole
  if ((tid & 63) == 0) s_r[tid >> 6] = ll;
  const int c = tid & 31, r = tid >> 5;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  if (4 * c < a.V) {
    const float* ws = a.ws + at * a.V + 4 * c;
#pragma unroll 4
    for (int s = r; s < sq.used; s += 8) x += s_f[s] * *(const f32x4*)(ws + (int64_t)s * a.V);
  }
  s_x[r][c] = x;
  __syncthreads();
  if (r == 0 && 4 * c < a.V) {
    ll = (s_r[0] + s_r[1]) + (s_r[2] + s_r[3]);
#pragma unroll
    for (int y = 1; y < 8; ++y) x += s_x[y][c];
    typename ET<T>::vec4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = ET<T>::from_f(ll != 0.f ? x[i] / ll : 0.f);
    *(typename ET<T>::vec4*)((T*)a.o.ptr + (int64_t)n * a.o.sb + (int64_t)h * a.o.sh + 4 * c) = y;
  }
}

template <typename T, int W, int NW, bool ALL> static void paged_parts(const lmoe_paged_args& a, const PagedPlan& p, hipStream_t st) {
  const dim3 grid((uint32_t)((int64_t)a.N * a.HKV * p.blocks * p.splits)), block(64 * NW);
  if (a.softcap > 0.f) {
    if (a.slopes) hipLaunchKernelGGL((k_paged_attn<T, W, NW, true, true, ALL>), grid, block, 0, st, a, p);
    else hipLaunchKernelGGL((k_paged_attn<T, W, NW, true, false, ALL>), grid, block, 0, st, a, p);
  } else if (a.slopes) hipLaunchKernelGGL((k_paged_attn<T, W, NW, false, true, ALL>), grid, block, 0, st, a, p);
  else hipLaunchKernelGGL((k_paged_attn<T, W, NW, false, false, ALL>), grid, block, 0, st, a, p);
}
template <typename T, int W> static void paged_decode(const lmoe_paged_args& a, hipStream_t st) {
  const PagedPlan p = paged_plan(a);
  if constexpr (sizeof(T) == 2) {
    if (p.waves == 8) {
      if (a.K == W) paged_parts<T, W, 8, true>(a, p, st); else paged_parts<T, W, 8, false>(a, p, st);
    }
  }
  if (p.waves == 4) {
    if (a.K == W) paged_parts<T, W, 4, true>(a, p, st); else paged_parts<T, W, 4, false>(a, p, st);
  }
  if (p.splits > 1) hipLaunchKernelGGL((k_paged_join<T>), dim3((uint32_t)((int64_t)a.N * a.HQ)), dim3(NTHR), 0, st, a, p);
}
void launch_paged_decode(const lmoe_paged_args& a, hipStream_t st) {
  const bool narrow = a.K <= 64 && a.V <= 64;
  if (a.dtype == LMOE_BF16) { if (narrow) paged_decode<bf16, 64>(a, st); else paged_decode<bf16, 128>(a, st); }
  else if (narrow) paged_decode<float, 64>(a, st);
  else paged_decode<float, 128>(a, st);
}

// ------------------------------------------------------------------------- //
// the cache is written: a wave per token, 16 bytes per lane
// ------------------------------------------------------------------------- //
template <typename T> __global__ __launch_bounds__(NTHR) void k_paged_append(const lmoe_paged_args a) {
  constexpr int VEC = ET<T>::VEC;
  typedef typename ET<T>::vec vec;
  const int64_t tok = (int64_t)blockIdx.x * (NTHR / 64) + wave_id();
  const int l = lane_id();
  if (tok >= (int64_t)a.B * a.T) return;
  int n, b, t, at;       // sequence; row and token in memory; token inside the sequence
  if (a.cu_seqlens) {
    // the last sequence that begins at or before the token (of several, all but the last are empty): 64 candidates a round
    b = 0; t = (int)tok;
    if (t >= a.cu_seqlens[a.N] || t < a.cu_seqlens[0]) return;
    int lo = 0, hi = a.N;
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64, i = lo + l * step;
      const int cnt = __popcll(__ballot(i < hi && a.cu_seqlens[min(i, a.N)] <= t));
      lo += (cnt - 1) * step;
      hi = min(hi, lo + step);
    }
    n = lo;
    at = t - a.cu_seqlens[n];
  } else {
    n = b = (int)(tok / a.T);
    t = at = (int)(tok - (int64_t)b * a.T);
  }
  const int64_t pos = (int64_t)a.lens[n] + at;
  if (a.lens[n] < 0 || pos >= (int64_t)a.M * a.S) return;
  const int id = a.table[(int64_t)n * a.table_stride + (int)pos / a.S], slot = (int)pos % a.S;
  if (id < 0 || id >= a.P) return;
  auto copy = [&](const lmoe_tensor& from, const lmoe_tensor& to, int D) {
    const T* s = (const T*)from.ptr + (int64_t)b * from.sb + (int64_t)t * from.st;
    T* d = (T*)to.ptr + (int64_t)id * to.sb + (int64_t)slot * to.st;
    const int per = D / VEC;
    for (int i = l; i < a.HKV * per; i += 64) {
      const int h = i / per, c = i % per * VEC;
      *(vec*)(d + (int64_t)h * to.sh + c) = *(const vec*)(s + (int64_t)h * from.sh + c);
    }
  };
  copy(a.kn, a.kp, a.K);
  copy(a.vn, a.vp, a.V);
}
void launch_paged_append(const lmoe_paged_args& a, hipStream_t st) {
  const dim3 grid((uint32_t)(((int64_t)a.B * a.T + NTHR / 64 - 1) / (NTHR / 64)));
  if (a.dtype == LMOE_BF16) hipLaunchKernelGGL((k_paged_append<bf16>), grid, dim3(NTHR), 0, st, a);
  else hipLaunchKernelGGL((k_paged_append<float>), grid, dim3(NTHR), 0, st, a);
}

}  // namespace lmoe
