// Softmax attention: instances and dispatch.
#include <algorithm>
#include <type_traits>

#include "lmoe_attn_any.hpp"
#include "lmoe_attn_bwd.hpp"

namespace lmoe {

// the kernels on 2-byte elements reach the rows of a tile by unsigned 32-bit offsets
static bool fits16(const lmoe_attn_args& a) {
  for (const lmoe_tensor* x : {&a.q, &a.k, &a.v, &a.d_o})
    if (x->st < 0 || x->st >= 1 << 24) return false;
  return a.dtype == LMOE_BF16;
}
// (without them: four strips to 64 rows, 512 threads each; with them 256, but 512 for tiles of 256 keys.  Of more than WALK_SEQS documents
// a tile of any size has as many work-groups as one of 64 rows.)
int64_t attn_groups(const lmoe_attn_args& a) {
  if (!fits16(a)) return attn_tiles<CH>(a) * a.HQ * 8;
  return std::max(attn_tiles<CH>(a) * a.HQ, a.dk.ptr ? 2 * attn_tiles<256>(a) * a.HKV : 0);
}

// Work-groups that share the rows of a strip of keys (k_attn_bwd_dkv_any): two where there are too few strips for the unequal work of a
// causal call to come out even, or for half of the card.  Backward with 1 / 2 / 3 / 4 work-groups, us: 2 x 1000 tokens, 4 heads on 2 of
// 64 98 / 88 / 101 / 101, of 128 191 / 160 / 182 / 178; 1 x 2048 190 / 162 / 177 / 172, not causal 206 / 215 / 220 / 226; 1 x 500, 16 on 4
// of 128 159 / 113 / 109 / 113.
static int any_parts(const lmoe_attn_args& a) {
  const int64_t strips = (int64_t)a.B * ((a.T + 15) / 16) * a.HKV;
  return a.T >= 256 && strips <= (a.causal ? cu_count() : cu_count() / 2) ? 2 : 1;
}
// A strip of 32 rows reads each tile half as often as two of 16, which with 64 columns gains where the strips fill the card all the same:
// 8 x 2048 tokens, 8 heads, forward 413 us in place of 448, backward 1307 in place of 1652; 2 x 1000, 4 heads on 2, 31 and 127 in
// place of 25 and 100.  (With 128 columns there are no registers for 32.)
template <typename T, int W, int CAP, bool BIAS> struct AttnAny {
  static bool wide(const lmoe_attn_args& a, int H) { return (int64_t)a.B * a.T * H / 32 >= 2 * cu_count(); }
  template <int RB> static void fwd_strips(const lmoe_attn_args& a, hipStream_t st) {
    const int64_t groups = attn_tiles<CH>(a) * a.HQ * (CH / 16 / RB);
    hipLaunchKernelGGL((k_attn_fwd_any<T, W, RB, CAP != NO_CAP, BIAS>), dim3(groups), dim3(64 * ANY_WAVES), 0, st, a, attn_fold(a, groups, a.HQ, cu_count()));
  }
  template <int RB> static void dq_strips(const lmoe_attn_args& a, hipStream_t st) {
    const int64_t groups = attn_tiles<CH>(a) * a.HQ * (CH / 16 / RB);
    hipLaunchKernelGGL((k_attn_bwd_dq_any<T, W, RB, CAP != NO_CAP, BIAS>), dim3(groups), dim3(64 * ANY_WAVES), 0, st, a, attn_fold(a, groups, a.HQ, cu_count()));
  }
  template <int KB> static void dkv_strips(const lmoe_attn_args& a, hipStream_t st) {
    const int64_t groups = attn_tiles<CH>(a) * a.HKV * (CH / 16 / KB);
    const int parts = any_parts(a);
    hipLaunchKernelGGL((k_attn_bwd_dkv_any<T, W, KB, CAP != NO_CAP, BIAS>), dim3(groups, parts), dim3(64 * ANY_KV_WAVES), 0, st, a, attn_fold(a, groups, a.HKV, cu_count()), parts);
    if (parts > 1) hipLaunchKernelGGL((k_attn_join<T, CH>), dim3(attn_tiles<CH>(a) * a.HKV, CH / JOIN_ROWS), dim3(NTHR), 0, st, a, parts, 0);
  }
  static void fwd(const lmoe_attn_args& a, hipStream_t st) {
    if constexpr (W == 64) { if (wide(a, a.HQ)) return fwd_strips<2>(a, st); }
    fwd_strips<1>(a, st);
  }
  static void bwd(const lmoe_attn_args& a, hipStream_t st) {
    if constexpr (W == 64) {
      if (wide(a, a.HQ)) dq_strips<2>(a, st); else dq_strips<1>(a, st);
      if (a.dk.ptr) { if (wide(a, a.HKV)) dkv_strips<2>(a, st); else dkv_strips<1>(a, st); }
    } else {
      dq_strips<1>(a, st);
      if (a.dk.ptr) dkv_strips<1>(a, st);
    }
  }
};

// Keys of a work-group of k_attn_bwd_dkv: as many waves as have registers for both sums on a CU, eight with 128 columns (two per SIMD;
// its 64 KB of values leave no second work-group room), four with 64 (three work-groups per CU).  2 x 8192 tokens of 16 heads,
// backward: 8 and 4 waves, 128 columns 1.73 and 2.28 ms, 64 columns 1.04 and 0.94.
constexpr int attn_kv_waves(int W) { return W == 128 ? 8 : 4; }
// Work-groups that share the rows of a tile of keys (k_attn_bwd_dkv), at most, and the pieces of its stream that each has at least.
// So many that the card is full; where it is, the tiles of a causal call are unequal work all the same, those of documents more so:
// two (64 columns: four) for long streams, four for documents of 96 pieces or more where the tiles fill the card twice at most (beyond
// that the longest documents, which come first, leave enough behind them).  Each part costs its sums' way through memory, and room for
// them whether a document is long enough or not: 1 GiB at the very most with these limits.
// Backward in us, 128 columns, 16 heads on 4, with 1 / 2 / 4 / 8 parts: 1 x 1024 tokens 243 / 155 / 106 / 86 (16 parts: 83), 1 x 4096
// 929 / 549 / 365 / 384, 8 x 1024 275 / 203 / 214 / 265, 2 x 8192 2411 / 1844 / 1911 / 2017; 16 on 16, 8 x 1024 162 / 278 / 420 / 686.
// 64 columns, 16 on 4, 2 x 8192 1316 / 1136 / 1034 / 1072.  16384 tokens in documents of which the longest has 5990, one part / two
// of 4 pieces or more / four of 48: 16 on 4 1677 / 1281 / 1270, 16 on 16 1142 / 1313 / 1159; in 16 equal ones 388 / 448 / 394.  7, 23
// and 60 unequal ones, one part / four of 48: 16 on 8 (tiles twice the CUs) 1223 / 1265, 815 / 764, 389 / 423; 12 on 12 (three
// times) 913 / 1045, 510 / 543, 267 / 325; 32768 tokens, 16 on 8 (four times) 4549 / 4793, 2264 / 2485, 951 / 1101.
struct Parts { int most, least; };
static Parts attn_parts(const lmoe_attn_args& a) {
  if (!fits16(a)) return {any_parts(a), 0};
  const int W = a.K <= 64 && a.V <= 64 ? 64 : 128, keys = 32 * attn_kv_waves(W);
  const int64_t groups = (a.cu_seqlens ? std::max<int64_t>(a.T / keys, 1) : (int64_t)a.B * ((a.T + keys - 1) / keys)) * a.HKV;
  const int64_t full = (W == 128 ? 1 : 2) * (int64_t)cu_count(), pieces = ((int64_t)a.T + CH - 1) / CH * (a.HQ / a.HKV);
  int64_t parts = (full + groups - 1) / groups;
  const int least = parts == 1 && a.cu_seqlens ? 48 : 4;
  if (a.cu_seqlens) parts = parts > 1 ? parts : groups <= 2 * full ? 4 : 1;
  else for (int i = W == 128 ? 1 : 2; i > 0 && groups * parts < (W == 128 ? 2 : 4) * full && pieces / parts >= 128; --i) parts *= 2;
  return {(int)std::max<int64_t>(1, std::min(std::min<int64_t>(parts, 16), pieces / least)), least};
}
int64_t attn_bwd_floats(const lmoe_attn_args& a) {
  const int parts = a.dk.ptr ? attn_parts(a).most : 1;
  return parts > 1 ? (int64_t)parts * a.B * a.T * a.HKV * (a.K + a.V) : 0;
}

// Whether two groups of waves share the rows of a work-group (k_attn_fwd, k_attn_bwd_dq): where the card is not full without, or
// just so, and the rows see many keys.  Forward, us with one group and with two, 16 heads of 128: 1 x 448 tokens 15.3 15.6, 1 x 512
// 18.4 17.3, 1 x 1024 28.6 24.8, 1 x 2048 50.6 41.2, 1 x 4096 107 91, 1 x 8192 321 321; 4 x 1024 35.9 41.7, 2 x 2048 60.6 57.1;
// not causal 1 x 2048 49.9 42.7, 1 x 4096 168 179.  8 heads of 64: 1 x 256 9.1 9.6, 1 x 2048 34.8 27.9, 1 x 4096 63.6 49.7.
static bool two_groups(const lmoe_attn_args& a, int64_t groups) {
  return (groups <= cu_count() && a.T >= 384) || (a.causal && groups <= 2 * cu_count() && a.T >= 2048);
}

template <typename T, int W, int CAP, bool BIAS> struct Attn16 {
  static void fwd(const lmoe_attn_args& a, hipStream_t st) {
    const int64_t groups = attn_tiles<ATTN_ROWS>(a) * a.HQ;
    if (two_groups(a, groups)) hipLaunchKernelGGL((k_attn_fwd<W, 2, CAP, BIAS>), dim3(groups), dim3(128 * ATTN_WAVES), 0, st, a);
    else hipLaunchKernelGGL((k_attn_fwd<W, 1, CAP, BIAS>), dim3(groups), dim3(64 * ATTN_WAVES), 0, st, a);
  }
  static void bwd(const lmoe_attn_args& a, hipStream_t st) {
    const int64_t groups = attn_tiles<ATTN_ROWS>(a) * a.HQ;
    if (two_groups(a, groups)) hipLaunchKernelGGL((k_attn_bwd_dq<W, 2, CAP, BIAS>), dim3(groups), dim3(128 * ATTN_WAVES), 0, st, a);
    else hipLaunchKernelGGL((k_attn_bwd_dq<W, 1, CAP, BIAS>), dim3(groups), dim3(64 * ATTN_WAVES), 0, st, a);
    if (!a.dk.ptr) return;
    constexpr int NW = attn_kv_waves(W);
    const Parts p = attn_parts(a);
    const dim3 tiles(attn_tiles<32 * NW>(a) * a.HKV);
    hipLaunchKernelGGL((k_attn_bwd_dkv<W, NW, CAP, BIAS>), dim3(tiles.x, p.most), dim3(64 * NW), 0, st, a, p.most, p.least);
    if (p.most > 1) hipLaunchKernelGGL((k_attn_join<bf16, 32 * NW>), dim3(tiles.x, 32 * NW / JOIN_ROWS), dim3(NTHR), 0, st, a, p.most, p.least);
  }
};

template <template <typename, int, int, bool> class F, typename T, int W, int FAR> static void by_score(const lmoe_attn_args& a, bool bwd, hipStream_t st) {
  auto run = [&](auto f) { if (bwd) f.bwd(a, st); else f.fwd(a, st); };
  if (a.softcap > CAP_NEAR) { if (a.slopes) run(F<T, W, FAR, true>()); else run(F<T, W, FAR, false>()); }
  else if (a.softcap > 0.f) { if (a.slopes) run(F<T, W, NEAR_CAP, true>()); else run(F<T, W, NEAR_CAP, false>()); }
  else if (a.slopes) run(F<T, W, NO_CAP, true>());
  else run(F<T, W, NO_CAP, false>());
}
// (the kernels with products in fp32 have one form for all caps)
template <typename T, int W> static void by_score_any(const lmoe_attn_args& a, bool bwd, hipStream_t st) { by_score<AttnAny, T, W, NEAR_CAP>(a, bwd, st); }
static void attn(const lmoe_attn_args& a, bool bwd, hipStream_t st) {
  const bool narrow = a.K <= 64 && a.V <= 64;
  if (fits16(a)) { if (narrow) by_score<Attn16, bf16, 64, FAR_CAP>(a, bwd, st); else by_score<Attn16, bf16, 128, FAR_CAP>(a, bwd, st); }
  else if (a.dtype == LMOE_BF16) { if (narrow) by_score_any<bf16, 64>(a, bwd, st); else by_score_any<bf16, 128>(a, bwd, st); }
  else if (narrow) by_score_any<float, 64>(a, bwd, st);
  else by_score_any<float, 128>(a, bwd, st);
}
void launch_attn_fwd(const lmoe_attn_args& a, hipStream_t st) { attn(a, false, st); }
void launch_attn_bwd(const lmoe_attn_args& a, hipStream_t st) { attn(a, true, st); }

}  // namespace lmoe
