// Attention of one new token over a paged cache: what its kernels for elements of 2 and 4 bytes (lmoe_paged.hip) and for a cache in
// 4 bits (lmoe_paged4.hip) share.
#pragma once
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


// the stretches of every sequence joined, where there are several (lmoe_paged.hip)
void launch_paged_join(const lmoe_paged_args& a, const PagedPlan& p, hipStream_t st);

}  // namespace lmoe
