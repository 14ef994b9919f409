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

template <typename T, int W, bool CAP, bool BIAS> struct Attn16 {
  static void fwd(const lmoe_attn_args& a, hipStream_t st) {
    if (a.T > 1024) hipLaunchKernelGGL((k_attn_fwd<W, 8, CAP, BIAS>), dim3(attn_tiles<256>(a) * a.HQ), dim3(512), 0, st, a);
    else hipLaunchKernelGGL((k_attn_fwd<W, 4, CAP, BIAS>), dim3(attn_tiles<128>(a) * a.HQ), dim3(256), 0, st, a);
  }
  static void bwd(const lmoe_attn_args& a, hipStream_t st) {
    if (a.T > 1024) hipLaunchKernelGGL((k_attn_bwd_dq<W, 8, CAP, BIAS>), dim3(attn_tiles<256>(a) * a.HQ), dim3(512), 0, st, a);
    else hipLaunchKernelGGL((k_attn_bwd_dq<W, 4, CAP, BIAS>), dim3(attn_tiles<128>(a) * a.HQ), dim3(256), 0, st, a);
    if (!a.dk.ptr) return;
    if (a.T > 1024) hipLaunchKernelGGL((k_attn_bwd_dkv<W, 8, CAP, BIAS>), dim3(attn_tiles<256>(a) * a.HKV), dim3(512), 0, st, a);
    else hipLaunchKernelGGL((k_attn_bwd_dkv<W, 4, CAP, BIAS>), dim3(attn_tiles<128>(a) * a.HKV), dim3(256), 0, st, a);
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
