// Softmax attention: instances and dispatch (kernels in lmoe_attn_any.hpp).
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "lmoe_attn_any.hpp"
#include "lmoe_attn_bwd.hpp"

namespace lmoe {

int64_t attn_groups(const lmoe_attn_args& a) { return attn_tiles<CH>(a) * a.HQ; }

template <typename T, int W, bool CAP, bool BIAS> struct AttnAny {
  static void fwd(const lmoe_attn_args& a, hipStream_t st) {
    hipLaunchKernelGGL((k_attn_fwd_any<T, W, CAP, BIAS>), dim3(attn_tiles<CH>(a) * a.HQ), dim3(NTHR), 0, st, a);
  }
  static void bwd(const lmoe_attn_args& a, hipStream_t st) {
    hipLaunchKernelGGL((k_attn_bwd_dq_any<T, W, CAP, BIAS>), dim3(attn_tiles<CH>(a) * a.HQ), dim3(NTHR), 0, st, a);
    if (a.dk.ptr) hipLaunchKernelGGL((k_attn_bwd_dkv_any<T, W, CAP, BIAS>), dim3(attn_tiles<CH>(a) * a.HKV), dim3(NTHR), 0, st, a);
  }
};

// Keys of a work-group of k_attn_bwd_dkv: as many waves as have registers for both sums on a CU, eight with 128 columns (two per SIMD;
// its 64 KB of values leave no second work-group room), four with 64 (two work-groups per CU).  2 x 8192 tokens of 16 heads,
// backward: 8 and 4 waves, 128 columns 1.73 and 2.28 ms, 64 columns 1.04 and 0.94.
constexpr int attn_kv_waves(int W) { return W == 128 ? 8 : 4; }
// Work-groups that share the rows of a tile of keys (k_attn_bwd_dkv)
static int attn_parts(const lmoe_attn_args& a) {
  if (a.dtype != LMOE_BF16) return 1;
  const int W = a.K <= 64 && a.V <= 64 ? 64 : 128, keys = 32 * attn_kv_waves(W), per_cu = W == 128 ? 1 : 2;
  const int64_t rows = a.cu_seqlens ? a.T : (int64_t)a.B * a.T;
  const int64_t groups = std::max<int64_t>(rows / keys, 1) * a.HKV, want = 2 * per_cu * (int64_t)cu_count() * (a.cu_seqlens ? 2 : 1);
  const int64_t pieces = ((int64_t)a.T + CH - 1) / CH * (a.HQ / a.HKV);
  return (int)std::max<int64_t>(1, std::min(std::min<int64_t>((want + groups - 1) / groups, 16), pieces / 4));
}
int64_t attn_bwd_floats(const lmoe_attn_args& a) {
  const int parts = a.dk.ptr ? attn_parts(a) : 1;
  return parts > 1 ? (int64_t)parts * a.B * a.T * a.HKV * (a.K + a.V) : 0;
}

template <typename T, int W, bool CAP, bool BIAS> struct Attn16 {
  static void fwd(const lmoe_attn_args& a, hipStream_t st) {
    hipLaunchKernelGGL((k_attn_fwd<W, CAP, BIAS>), dim3(attn_tiles<ATTN_ROWS>(a) * a.HQ), dim3(64 * ATTN_WAVES), 0, st, a);
  }
  static void bwd(const lmoe_attn_args& a, hipStream_t st) {
    hipLaunchKernelGGL((k_attn_bwd_dq<W, CAP, BIAS>), dim3(attn_tiles<ATTN_ROWS>(a) * a.HQ), dim3(64 * ATTN_WAVES), 0, st, a);
    if (!a.dk.ptr) return;
    constexpr int NW = attn_kv_waves(W);
    const int parts = attn_parts(a);
    hipLaunchKernelGGL((k_attn_bwd_dkv<W, NW, CAP, BIAS>), dim3(attn_tiles<32 * NW>(a) * a.HKV, parts), dim3(64 * NW), 0, st, a, parts);
    if (parts == 1) return;
    const int64_t blocks = ((int64_t)a.B * a.T * a.HKV * (a.K + a.V) / 4 + NTHR - 1) / NTHR;
    hipLaunchKernelGGL(k_attn_join, dim3(std::min<int64_t>(blocks, 8 * cu_count())), dim3(NTHR), 0, st, a, parts);
  }
};

template <template <typename, int, bool, bool> class F, typename T, int W> static void by_score(const lmoe_attn_args& a, bool bwd, hipStream_t st) {
  auto run = [&](auto f) { if (bwd) f.bwd(a, st); else f.fwd(a, st); };
  if (a.softcap > 0.f) { if (a.slopes) run(F<T, W, true, true>()); else run(F<T, W, true, false>()); }
  else if (a.slopes) run(F<T, W, false, true>());
  else run(F<T, W, false, false>());
}
static void attn(const lmoe_attn_args& a, bool bwd, hipStream_t st) {
  const bool narrow = a.K <= 64 && a.V <= 64;
  // (the kernels on 2-byte elements reach the rows of a tile by 32-bit offsets)
  int64_t stride = 0;
  for (const lmoe_tensor* x : {&a.q, &a.k, &a.v, &a.d_o}) stride = std::max(stride, std::abs(x->st));
  if (a.dtype == LMOE_BF16 && stride >= (1 << 24)) { if (narrow) by_score<AttnAny, bf16, 64>(a, bwd, st); else by_score<AttnAny, bf16, 128>(a, bwd, st); }
  else if (a.dtype == LMOE_BF16) { if (narrow) by_score<Attn16, bf16, 64>(a, bwd, st); else by_score<Attn16, bf16, 128>(a, bwd, st); }
  else if (narrow) by_score<AttnAny, float, 64>(a, bwd, st);
  else by_score<AttnAny, float, 128>(a, bwd, st);
}
void launch_attn_fwd(const lmoe_attn_args& a, hipStream_t st) { attn(a, false, st); }
void launch_attn_bwd(const lmoe_attn_args& a, hipStream_t st) { attn(a, true, st); }

}  // namespace lmoe
