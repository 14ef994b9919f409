// Norm and rotation of queries and keys (include/lmoe.h, lmoe_rope_args).
//
//   r = (mean x^2 + eps)^-1/2,  y = x r w,  z_a = y_a c - y_b s,  z_b = y_b c + y_a s
// Backward, with g the gradient of z turned back (the rotation by the negative angle) and x^ = x r:
//   dw = sum over rows of g x^,   dx = r (g w - x^ mean(g w x^))
// (the reference's rotary: linear_moe/model/common_modules/rotary.py:40-98).
//
// HBM-bound: x is read and z written once; backward x and the gradient read and dx written once.  A row is held by L lanes, a lane's
// columns being V of the first and V of the second members of V pairs, so that no column crosses lanes for the rotation.  A lane
// keeps its columns' weights over the whole call and a token's angles over the heads of a token that it takes.
// The sums of dw: fp32 in the lane's registers over all its rows, then lanes, waves and work-groups in a fixed order.
#include <algorithm>

#include "lmoe_common.hpp"
#include "lmoe_launch.hpp"

namespace lmoe {

constexpr int ROPE_HEADS = 4;          // heads of a token that a lane has in flight
constexpr int ROPE_GROUPS = 2048, ROPE_BWD_GROUPS = 1024;        // work-groups of a launch at most (or what one token needs)

struct RopePlan {
  int lanes;       // of a row
  int chunks;      // of a row: V pairs each
  int runs;        // lane groups that share a token's heads
  int heads;       // of them all
  uint32_t grid;
};

template <typename T, int V> struct RopeVec { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct RopeVec<T, 1> { typedef T type; };

// V columns each of the first (x[0 .. V - 1]) and second members of a lane's pairs
template <typename T, int V, bool INTER> __device__ __forceinline__ void rope_load(float (&x)[2 * V], const T* row, int a, int b) {
  typedef typename RopeVec<T, V>::type vec;
  const vec lo = *(const vec*)(row + a), hi = *(const vec*)(row + b);
  float y[2 * V];
  if constexpr (V == 1) { y[0] = (float)lo; y[1] = (float)hi; }
  else {
#pragma unroll
    for (int i = 0; i < V; ++i) { y[i] = (float)lo[i]; y[V + i] = (float)hi[i]; }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) { x[i] = INTER ? y[2 * i] : y[i]; x[V + i] = INTER ? y[2 * i + 1] : y[V + i]; }
}
template <typename T, int V, bool INTER> __device__ __forceinline__ void rope_store(T* row, int a, int b, const float (&x)[2 * V]) {
  typedef typename RopeVec<T, V>::type vec;
  float y[2 * V];
#pragma unroll
  for (int i = 0; i < V; ++i) { y[INTER ? 2 * i : i] = x[i]; y[INTER ? 2 * i + 1 : V + i] = x[V + i]; }
  vec lo, hi;
  if constexpr (V == 1) { lo = (T)y[0]; hi = (T)y[1]; }
  else {
#pragma unroll
    for (int i = 0; i < V; ++i) { lo[i] = (T)y[i]; hi[i] = (T)y[V + i]; }
  }
  *(vec*)(row + a) = lo;
  *(vec*)(row + b) = hi;
}
// the weights of a lane's columns (1 without them)
template <int V, bool INTER> __device__ __forceinline__ void rope_weights(float (&w)[2 * V], const void* p, int dtype, int a, int b) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int ia = INTER ? a + 2 * i : a + i, ib = INTER ? a + 2 * i + 1 : b + i;
    w[i] = !p ? 1.f : dtype == LMOE_F32 ? ((const float*)p)[ia] : (float)((const bf16*)p)[ia];
    w[V + i] = !p ? 1.f : dtype == LMOE_F32 ? ((const float*)p)[ib] : (float)((const bf16*)p)[ib];
  }
}

template <int L> __device__ __forceinline__ float lanes_of_row(float x) {
#pragma unroll
  for (int d = 1; d < L; d <<= 1) x += __shfl_xor(x, d, 64);
  return x;
}

// The position of token t (of row b), and whether it belongs to a sequence
__device__ __forceinline__ bool rope_position(const lmoe_rope_args& a, int b, int t, int& pos) {
  int n = b, at = t;
  if (a.cu_seqlens) {
    if (t < a.cu_seqlens[0] || t >= a.cu_seqlens[a.N]) return false;
    int lo = 0, hi = a.N;                       // the last sequence that begins at or before the token (of several, all but it are empty)
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (a.cu_seqlens[m] <= t) lo = m; else hi = m;
    }
    n = lo;
    at = t - a.cu_seqlens[n];
  }
  // (in 64 bits: an offset may be any number)
  int64_t p = a.positions ? a.positions[b * a.pos_stride + t] : (int64_t)at + (a.offsets ? a.offsets[n] : 0);
  pos = p >= 0 && p < a.L ? (int)p : -1;
  return true;
}

template <typename T, int V, int L, int NC, bool INTER, bool BWD>
__global__ __launch_bounds__(NTHR) void k_qk_norm_rope(const lmoe_rope_args a, const RopePlan p) {
  constexpr int HB = NC > 1 ? 1 : ROPE_HEADS;
  const int l = threadIdx.x % L;
  const int64_t group = (int64_t)blockIdx.x * (NTHR / L) + threadIdx.x / L, groups = (int64_t)gridDim.x * (NTHR / L) / p.runs;      // tokens at a time
  const int run = (int)(group % p.runs);
  const int half = a.R / 2, rest = (a.D - a.R) / 2;
  int ca[NC], cb[NC], cr[NC];          // columns of the pairs' members, row of the angles (-1: not rotated)
  bool on[NC];
  float wq[NC][2 * V], wk[NC][2 * V], sq[NC][2 * V], sk[NC][2 * V];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = (l + j * L) * V;
    on[j] = l + j * L < p.chunks;
    cr[j] = on[j] && c < half ? c : -1;
    ca[j] = INTER ? 2 * c : c < half ? c : c + half;
    cb[j] = INTER ? 2 * c + V : c < half ? c + half : c + half + rest;
    if (!on[j]) ca[j] = cb[j] = 0;
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) { wq[j][i] = wk[j][i] = 1.f; sq[j][i] = sk[j][i] = 0.f; }
    if (on[j]) {
      rope_weights<V, INTER>(wq[j], a.qw, a.w_dtype, ca[j], cb[j]);
      rope_weights<V, INTER>(wk[j], a.kw, a.w_dtype, ca[j], cb[j]);
    }
  }
  const float over = 1.0f / (float)a.D;
  const int64_t tokens = (int64_t)a.B * a.T;
  const int64_t first = group / p.runs;
  // (a group past the last whole set of runs has nothing to do; its lanes stay: sums over a row need them all)
  for (int64_t tok0 = 0; tok0 < tokens; tok0 += groups) {
    const int64_t tok = tok0 + first;
    const bool mine = first < groups && tok < tokens;
    const int b = mine ? (int)(tok / a.T) : 0, t = mine ? (int)(tok - (int64_t)b * a.T) : 0;
    int pos = -1;
    const bool live = mine && rope_position(a, b, t, pos);
    float c[NC][V], s[NC][V];
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool turn = pos >= 0 && cr[j] >= 0;
        c[j][i] = turn ? a.cos[(int64_t)pos * half + cr[j] + i] : 1.f;
        s[j][i] = turn ? a.sin[(int64_t)pos * half + cr[j] + i] : 0.f;
      }
    for (int h0 = run; h0 < p.heads; h0 += HB * p.runs) {
      float x[HB][NC][2 * V], g[HB][NC][2 * V];
#pragma unroll
      for (int y = 0; y < HB; ++y) {
        const int h = h0 + y * p.runs;
        const bool q = h < a.HQ;
        const lmoe_tensor& from = q ? a.q : a.k;
        const lmoe_tensor& grad = q ? a.dzq : a.dzk;
        const int64_t hh = q ? h : h - a.HQ;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) x[y][j][i] = g[y][j][i] = 0.f;
          if (!live || h >= p.heads || !on[j]) continue;
          if (!BWD || a.norm) rope_load<T, V, INTER>(x[y][j], (const T*)from.ptr + b * from.sb + t * from.st + hh * from.sh, ca[j], cb[j]);
          if (BWD) rope_load<T, V, INTER>(g[y][j], (const T*)grad.ptr + b * grad.sb + t * grad.st + hh * grad.sh, ca[j], cb[j]);
        }
      }
#pragma unroll
      for (int y = 0; y < HB; ++y) {
        const int h = h0 + y * p.runs;
        const bool q = h < a.HQ;
        float r = 1.f;
        if (a.norm) {
          float ss = 0.f;
#pragma unroll
          for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) ss += x[y][j][i] * x[y][j][i];
          r = rsqrt_fast(lanes_of_row<L>(ss) * over + a.eps);
        }
        float z[NC][2 * V];
        if constexpr (!BWD) {
#pragma unroll
          for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float ya = x[y][j][i] * r * (q ? wq[j][i] : wk[j][i]), yb = x[y][j][V + i] * r * (q ? wq[j][V + i] : wk[j][V + i]);
              z[j][i] = ya * c[j][i] - yb * s[j][i];
              z[j][V + i] = yb * c[j][i] + ya * s[j][i];
            }
        } else {
          float m = 0.f;
#pragma unroll
          for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float ga = g[y][j][i] * c[j][i] + g[y][j][V + i] * s[j][i], gb = g[y][j][V + i] * c[j][i] - g[y][j][i] * s[j][i];
              const float xa = x[y][j][i] * r, xb = x[y][j][V + i] * r;
              if (q) { sq[j][i] += ga * xa; sq[j][V + i] += gb * xb; }
              else { sk[j][i] += ga * xa; sk[j][V + i] += gb * xb; }
              z[j][i] = ga * (q ? wq[j][i] : wk[j][i]);
              z[j][V + i] = gb * (q ? wq[j][V + i] : wk[j][V + i]);
              m += z[j][i] * xa + z[j][V + i] * xb;
              x[y][j][i] = xa; x[y][j][V + i] = xb;
            }
          if (a.norm) {
            m = lanes_of_row<L>(m) * over;
#pragma unroll
            for (int j = 0; j < NC; ++j)
#pragma unroll
              for (int i = 0; i < 2 * V; ++i) z[j][i] = r * (z[j][i] - x[y][j][i] * m);
          }
        }
        if (!mine || h >= p.heads) continue;
        const lmoe_tensor& to = BWD ? (q ? a.dq : a.dk) : (q ? a.zq : a.zk);
        T* row = (T*)to.ptr + b * to.sb + t * to.st + (int64_t)(q ? h : h - a.HQ) * to.sh;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          if (!on[j]) continue;
          if (!live) {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) z[j][i] = 0.f;
          }
          rope_store<T, V, INTER>(row, ca[j], cb[j], z[j]);
        }
      }
    }
  }
  if constexpr (BWD) {
    // dw: the lane groups of a wave, then the waves, then a row of ws per work-group
    if (!a.ws) return;
    __shared__ float part[NTHR / 64][2][256];
    const int w = wave_id();
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) {
        float x = sq[j][i], y = sk[j][i];
#pragma unroll
        for (int d = L; d < 64; d <<= 1) { x += __shfl_xor(x, d, 64); y += __shfl_xor(y, d, 64); }
        if (lane_id() < L && on[j]) {
          const int e = i < V ? i : i - V, col = INTER ? ca[j] + 2 * e + (i >= V) : (i < V ? ca[j] : cb[j]) + e;
          part[w][0][col] = x;
          part[w][1][col] = y;
        }
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += NTHR) {
      const int which = i / a.D, col = i % a.D;
      a.ws[(int64_t)blockIdx.x * 2 * a.D + i] = (part[0][which][col] + part[1][which][col]) + (part[2][which][col] + part[3][which][col]);
    }
  }
}

// dw: the rows of ws, a work-group per 32 columns (of dqw and dkw in a row), 8 rows at a time
__global__ __launch_bounds__(NTHR) void k_qk_norm_dw(const lmoe_rope_args a, int rows) {
  __shared__ float s[8][32];
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
  float x = 0.f;
  if (col < 2 * a.D)
    for (int i = r; i < rows; i += 8) x += a.ws[(int64_t)i * 2 * a.D + col];
  s[r][c] = x;
  __syncthreads();
  if (r || col >= 2 * a.D) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) x += s[i][c];
  void* to = col < a.D ? a.dqw : a.dkw;
  const int at = col < a.D ? col : col - a.D;
  if (!to) return;
  if (a.w_dtype == LMOE_F32) ((float*)to)[at] = x; else ((bf16*)to)[at] = (bf16)x;
}

// Whether every row can be read in 16-byte pieces that hold whole pairs' members
static bool rope_wide(const lmoe_rope_args& a) {
  const int v = a.dtype == LMOE_BF16 ? 8 : 4;
  if (a.interleaved ? a.R % (2 * v) || a.D % (2 * v) : a.R % (2 * v) || (a.D - a.R) % (2 * v)) return false;
  const lmoe_tensor* all[] = {&a.q, &a.k, &a.zq, &a.zk, &a.dzq, &a.dzk, &a.dq, &a.dk};
  for (const lmoe_tensor* t : all)
    if (t->ptr && (((uintptr_t)t->ptr & 15) || (t->sb | t->st | t->sh) % v)) return false;
  return true;
}
static RopePlan rope_plan(const lmoe_rope_args& a, bool bwd) {
  RopePlan p;
  const int v = rope_wide(a) ? (a.dtype == LMOE_BF16 ? 8 : 4) : 1;
  p.chunks = a.D / (2 * v);
  p.lanes = 4;
  while (p.lanes < 64 && p.lanes < p.chunks) p.lanes *= 2;
  if (v == 1) p.lanes = 64;
  p.heads = a.HQ + a.HKV;
  const int64_t tokens = (int64_t)a.B * a.T, per = NTHR / p.lanes;
  // a head for each lane group while that leaves the card empty, else several
  const bool few = tokens * p.heads <= 256 * 8 * per;
  p.runs = few || v == 1 ? p.heads : (p.heads + ROPE_HEADS - 1) / ROPE_HEADS;
  const int64_t want = (tokens * p.runs + per - 1) / per, least = (p.runs + per - 1) / per;
  p.grid = (uint32_t)std::max(std::min<int64_t>(want, bwd ? ROPE_BWD_GROUPS : ROPE_GROUPS), least);
  return p;
}
// (as many rows as a call of these sizes has work-groups at most, however its tensors lie)
int64_t rope_floats(const lmoe_rope_args& a) {
  const int64_t heads = (int64_t)a.HQ + a.HKV, rows = (int64_t)a.B * a.T * heads;
  return std::max(std::min<int64_t>(ROPE_BWD_GROUPS, rows), heads) * 2 * a.D;
}

template <typename T, int V, int L, int NC, bool BWD> static void rope_launch(const lmoe_rope_args& a, const RopePlan& p, hipStream_t st) {
  if (a.interleaved) hipLaunchKernelGGL((k_qk_norm_rope<T, V, L, NC, true, BWD>), dim3(p.grid), dim3(NTHR), 0, st, a, p);
  else hipLaunchKernelGGL((k_qk_norm_rope<T, V, L, NC, false, BWD>), dim3(p.grid), dim3(NTHR), 0, st, a, p);
}
template <typename T, bool BWD> static void rope_typed(const lmoe_rope_args& a, const RopePlan& p, hipStream_t st) {
  constexpr int V = ET<T>::VEC;
  if (p.chunks * 2 * V != a.D || !rope_wide(a)) rope_launch<T, 1, 64, 2, BWD>(a, p, st);
  else if (p.lanes == 4) rope_launch<T, V, 4, 1, BWD>(a, p, st);
  else if (p.lanes == 8) rope_launch<T, V, 8, 1, BWD>(a, p, st);
  else if (p.lanes == 16) rope_launch<T, V, 16, 1, BWD>(a, p, st);
  else if constexpr (V == 4) rope_launch<T, V, 32, 1, BWD>(a, p, st);
}
void launch_qk_norm_rope(const lmoe_rope_args& a, bool bwd, hipStream_t st) {
  const RopePlan p = rope_plan(a, bwd);
  if (a.dtype == LMOE_BF16) { if (bwd) rope_typed<bf16, true>(a, p, st); else rope_typed<bf16, false>(a, p, st); }
  else if (bwd) rope_typed<float, true>(a, p, st);
  else rope_typed<float, false>(a, p, st);
  if (bwd && (a.dqw || a.dkw))
    hipLaunchKernelGGL(k_qk_norm_dw, dim3((2 * a.D + 31) / 32), dim3(NTHR), 0, st, a, (int)p.grid);
}

}  // namespace lmoe
