// The pages of a cache: given back, shared, given out (and copied, where a shared one is to be written), moved together
// (include/lmoe.h, lmoe_pages_args).
//
// Who gets which page is decided by one work-group (k_pages_reserve, k_pages_compact: integer work on the table's asked columns and on
// refs, bound by latency); what it decided is a list of copies that k_pages_copy carries out with the whole card, HBM-bound at two bytes
// moved for one of a page.  Counts are kept by integer atomics, whose order changes no result; places in a list come from scans.
#include <algorithm>

#include "lmoe_common.hpp"
#include "lmoe_launch.hpp"

namespace lmoe {

constexpr int PAGES_NTHR = 1024, PAGES_WAVES = PAGES_NTHR / 64;
constexpr int PAGES_VEC = 16;                 // numbers of refs that a thread takes at a time
constexpr int COPY_BUFS = 32;                 // tensors of a launch of the copies
constexpr int COPY_UNIT = 16384;              // bytes of a page that a work-group takes at a time

// What ws holds for reserve and compact
struct PagesWs {
  int32_t* count;                       // copies to make
  int32_t *src, *dst;                   // [P] their pages
  int32_t* list;                        // [P] free pages
  int32_t *claims, *last, *failed;      // [P] of a shared page: asked entries, the last of them, whether one gets no copy
  int32_t* need;                        // [N] pages that the rows up to a row need
};
__host__ __device__ inline PagesWs pages_ws(const lmoe_pages_args& a) {
  PagesWs w;
  int32_t* p = a.ws;
  w.count = p; p += 16;
  w.list = p; p += a.P;
  w.claims = p; p += a.P;
  w.last = p; p += a.P;
  w.failed = p; p += a.P;
  w.src = p; p += a.P;
  w.dst = p; p += a.P;
  w.need = p;
  return w;
}
int64_t pages_ints(const lmoe_pages_args& a) { return 16 + 6 * (int64_t)a.P + a.N; }
int64_t fork_ints(const lmoe_pages_args& a) { return (int64_t)a.F * (a.M + 1); }

// memory that other waves of the work-group wrote, or that atomics count in: past this CU's cache
__device__ __forceinline__ int32_t seen(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void put(int32_t* p, int32_t x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// sum over the threads in front of this one, and over all (every thread of the work-group calls it)
__device__ __forceinline__ int scan(int x, int& total, int* s_wave) {
  int y = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int z = __shfl_up(y, d, 64);
    if (lane_id() >= d) y += z;
  }
  __syncthreads();                         // s_wave of the scan before has been read
  if (lane_id() == 63) s_wave[threadIdx.x >> 6] = y;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < PAGES_WAVES; ++i) {
    const int z = s_wave[i];
    if (i < (int)(threadIdx.x >> 6)) before += z;
    total += z;
  }
  return before + y - x;
}

// The numbers p in [begin, end) with (refs[p] > 0) == used, in their order, into list[0 .. most - 1]; how many there are (counting stops
// behind the one that fills the list)
__device__ __forceinline__ int listed(const int32_t* refs, int begin, int end, bool used, int32_t* list, int most, int* s_wave) {
  int before = 0;
  for (int p0 = begin; p0 < end && before < most; p0 += PAGES_NTHR * PAGES_VEC) {
    const int first = p0 + (int)threadIdx.x * PAGES_VEC;
    uint32_t hit = 0;
#pragma unroll
    for (int i = 0; i < PAGES_VEC; ++i)
      if (first + i < end && (refs[first + i] > 0) == used) hit |= 1u << i;
    int total, at = before + scan(__popc(hit), total, s_wave);
#pragma unroll
    for (int i = 0; i < PAGES_VEC; ++i)
      if (hit >> i & 1) { if (at < most) put(list + at, first + i); ++at; }
    before += total;
  }
  return before;
}

// ---- given back ----
__global__ __launch_bounds__(NTHR) void k_pages_free(const lmoe_pages_args a) {
  const int row = a.rows[blockIdx.x];
  if (row < 0 || row >= a.N) return;
  int32_t* t = a.table + (int64_t)row * a.table_stride;
  for (int c = threadIdx.x; c < a.M; c += NTHR) {
    const int e = t[c];
    if (e < 0 || e >= a.P) continue;
    const int was = atomicExch(t + c, -1);              // (a row that is listed twice gives its pages back once)
    if (was >= 0 && was < a.P) atomicSub(a.refs + was, 1);
  }
  if (threadIdx.x == 0) a.lens[row] = 0;
}

// ---- shared ----
__global__ __launch_bounds__(NTHR) void k_pages_snapshot(const lmoe_pages_args a) {
  const int row = a.src[blockIdx.x];
  if (row < 0 || row >= a.N) return;
  const int32_t* t = a.table + (int64_t)row * a.table_stride;
  int32_t* to = a.ws + (int64_t)blockIdx.x * (a.M + 1);
  for (int c = threadIdx.x; c < a.M; c += NTHR) to[c] = t[c];
  if (threadIdx.x == 0) to[a.M] = a.lens[row];
}
__global__ __launch_bounds__(NTHR) void k_pages_fork(const lmoe_pages_args a) {
  const int i = blockIdx.x, to = a.rows[i], from = a.src[i];
  if (to < 0 || to >= a.N || from < 0 || from >= a.N) return;
  bool again = false;                                    // a later one for the same row
  for (int j = i + 1 + threadIdx.x; j < a.F; j += NTHR) again |= a.rows[j] == to && a.src[j] >= 0 && a.src[j] < a.N;
  if (__syncthreads_or(again)) return;
  int32_t* t = a.table + (int64_t)to * a.table_stride;
  const int32_t* s = a.ws + (int64_t)i * (a.M + 1);
  for (int c = threadIdx.x; c < a.M; c += NTHR) {
    const int old = t[c], now = s[c];
    if (old == now) continue;
    if (old >= 0 && old < a.P) atomicSub(a.refs + old, 1);
    if (now >= 0 && now < a.P) atomicAdd(a.refs + now, 1);
    t[c] = now;
  }
  if (threadIdx.x == 0) a.lens[to] = s[a.M];
}

// ---- given out ----
// Columns of row n that are to be writable: first .. last (none: last < first); false where the table ends before
__device__ __forceinline__ bool asked(const lmoe_pages_args& a, int n, int& first, int& last) {
  const int64_t len = max(a.lens[n], 0), t = a.tokens ? a.tokens[n] : a.each;
  first = 0; last = -1;
  if (t <= 0) return true;
  const int64_t end = (len + t - 1) / a.S;
  if (end >= a.M) return false;
  first = (int)(len / a.S);
  last = (int)end;
  return true;
}
// In the order of rows and columns, as if one after the other: an entry that names a page of refs r, of which e entries in front
// of it are asked for too, has to be copied if r - e > 1, for those have taken their copies by then.  So of the asked entries of a page all are
// copied, but the last where there are r of them.
__global__ __launch_bounds__(PAGES_NTHR) void k_pages_reserve(const lmoe_pages_args a) {
  __shared__ int s_wave[PAGES_WAVES];
  const PagesWs w = pages_ws(a);
  const int wave = wave_id(), l = lane_id();
  auto each = [&](auto f) {                              // a wave per row, its columns over the lanes
    for (int n = wave; n < a.N; n += PAGES_WAVES) {
      int first, last;
      if (asked(a, n, first, last)) f(n, first, last);
    }
  };
  auto entry = [&](int n, int c) { return a.table[(int64_t)n * a.table_stride + c]; };
  auto is_page = [&](int x) { return x >= 0 && x < a.P; };
  if (threadIdx.x == 0) put(w.count, 0);
  each([&](int n, int first, int last) {
    for (int c = first + l; c <= last; c += 64) {
      const int x = entry(n, c);
      if (is_page(x) && a.refs[x] > 1) { put(w.claims + x, 0); put(w.last + x, -1); put(w.failed + x, 0); }
    }
  });
  __syncthreads();
  each([&](int n, int first, int last) {
    for (int c = first + l; c <= last; c += 64) {
      const int x = entry(n, c);
      if (is_page(x) && a.refs[x] > 1) { atomicAdd(w.claims + x, 1); atomicMax(w.last + x, n * a.M + c); }
    }
  });
  __syncthreads();
  auto shared = [&](int x) { return is_page(x) && a.refs[x] > 1; };
  auto kept = [&](int n, int c, int x) { return seen(w.claims + x) == a.refs[x] && seen(w.last + x) == n * a.M + c; };
  for (int n = threadIdx.x; n < a.N; n += PAGES_NTHR) put(w.need + n, 0);
  __syncthreads();
  each([&](int n, int first, int last) {
    int need = 0;
    for (int c0 = first; c0 <= last; c0 += 64) {
      const int c = c0 + l, x = c <= last ? entry(n, c) : -1;
      need += __popcll(__ballot(c <= last && (!is_page(x) || (shared(x) && !kept(n, c, x)))));
    }
    if (l == 0) put(w.need + n, need);
  });
  __syncthreads();
  // how many pages up to each row
  int all = 0;
  for (int n0 = 0; n0 < a.N; n0 += PAGES_NTHR) {
    const int n = n0 + threadIdx.x, need = n < a.N ? seen(w.need + n) : 0;
    int total;
    const int at = all + scan(need, total, s_wave);
    if (n < a.N) put(w.need + n, at);
    all += total;
  }
  const int free = listed(a.refs, 0, a.P, false, w.list, min(all, a.P), s_wave);
  __syncthreads();
  // rows that the free pages do not reach: the pages they do not copy stay shared
  auto before = [&](int n) { return seen(w.need + n); };
  auto upto = [&](int n) { return n + 1 < a.N ? seen(w.need + n + 1) : all; };
  auto reached = [&](int n) { return upto(n) <= free || upto(n) == before(n); };
  if (all > free) {
    each([&](int n, int first, int last) {
      if (reached(n)) return;
      for (int c = first + l; c <= last; c += 64) {
        const int x = entry(n, c);
        if (shared(x) && !kept(n, c, x)) put(w.failed + x, 1);
      }
    });
    __syncthreads();
  }
  for (int n = wave; n < a.N; n += PAGES_WAVES) {
    int first, last;
    bool fits = asked(a, n, first, last);
    if (fits && all > free) {
      fits = reached(n);
      for (int c0 = first; fits && c0 <= last; c0 += 64) {
        const int c = c0 + l, x = c <= last ? entry(n, c) : -1;
        if (__ballot(c <= last && shared(x) && kept(n, c, x) && seen(w.failed + x))) fits = false;
      }
    }
    if (l == 0) a.fits[n] = fits;
    // (refs of a shared page stays as it is until every wave has decided by it)
    int at = before(n);
    for (int c0 = first; fits && c0 <= last; c0 += 64) {
      const int c = c0 + l, x = c <= last ? entry(n, c) : -1;
      const bool copy = c <= last && shared(x) && !kept(n, c, x), take = copy || (c <= last && !is_page(x));
      const uint64_t mask = __ballot(take);
      if (take) {
        const int page = seen(w.list + at + __popcll(mask & ((1ull << l) - 1)));
        a.table[(int64_t)n * a.table_stride + c] = page;
        a.refs[page] = 1;                                // (free or given out: no page is shared by it)
        if (copy) {
          const int i = atomicAdd(w.count, 1);           // (the order of the copies changes nothing)
          put(w.src + i, x);
          put(w.dst + i, page);
        }
      }
      at += __popcll(mask);
    }
  }
  __syncthreads();
  const int copies = seen(w.count);
  for (int i = threadIdx.x; i < copies; i += PAGES_NTHR) atomicSub(a.refs + seen(w.src + i), 1);
}

// ---- moved together ----
__global__ __launch_bounds__(PAGES_NTHR) void k_pages_compact(const lmoe_pages_args a) {
  __shared__ int s_wave[PAGES_WAVES];
  const PagesWs w = pages_ws(a);
  int used = 0;
  for (int p = threadIdx.x; p < a.P; p += PAGES_NTHR) {
    used += a.refs[p] > 0;
    put(a.moved + p, p);
  }
  int live;
  scan(used, live, s_wave);
  // as many free numbers below as used pages above
  const int count = listed(a.refs, 0, live, false, w.dst, live, s_wave);
  listed(a.refs, live, a.P, true, w.src, count, s_wave);
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += PAGES_NTHR) {
    const int from = seen(w.src + i), to = seen(w.dst + i);
    put(a.moved + from, to);
    a.refs[to] = a.refs[from];
    a.refs[from] = 0;
  }
  if (threadIdx.x == 0) { a.live[0] = live; put(w.count, count); }
}
__global__ __launch_bounds__(NTHR) void k_pages_renamed(const lmoe_pages_args a) {
  const int64_t all = (int64_t)a.N * a.M;
  for (int64_t i = (int64_t)blockIdx.x * NTHR + threadIdx.x; i < all; i += (int64_t)gridDim.x * NTHR) {
    int32_t* t = a.table + i / a.M * a.table_stride + i % a.M;
    const int x = *t;
    if (x >= 0 && x < a.P) *t = a.moved[x];
  }
}

// ---- the copies ----
struct PageBufs {
  int n;
  lmoe_page_buf b[COPY_BUFS];
  int32_t units[COPY_BUFS + 1];        // units of a page up to each tensor
  int32_t per[COPY_BUFS];              // units of a run
  int8_t vec[COPY_BUFS];               // bytes of a piece: 16, 4 or 1
};
template <typename P> __device__ __forceinline__ void copy_run(uint8_t* to, const uint8_t* from, int64_t bytes) {
  constexpr int U = 4;
  const int64_t n = bytes / sizeof(P);
  for (int64_t i0 = threadIdx.x; i0 < n; i0 += U * NTHR) {
    P x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) if (i0 + u * NTHR < n) x[u] = ((const P*)from)[i0 + u * NTHR];
#pragma unroll
    for (int u = 0; u < U; ++u) if (i0 + u * NTHR < n) ((P*)to)[i0 + u * NTHR] = x[u];
  }
}
__global__ __launch_bounds__(NTHR) void k_pages_copy(const lmoe_pages_args a, const PageBufs bufs) {
  const PagesWs w = pages_ws(a);
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const int count = w.count[0], per_page = bufs.units[bufs.n];
  for (int64_t x = blockIdx.x; x < (int64_t)count * per_page; x += gridDim.x) {
    const int i = (int)(x / per_page), u = (int)(x % per_page);
    int k = 0;
    while (u >= bufs.units[k + 1]) ++k;
    const lmoe_page_buf& b = bufs.b[k];
    const int y = u - bufs.units[k], run = y / bufs.per[k];
    const int64_t at = (int64_t)(y % bufs.per[k]) * COPY_UNIT;
    const int64_t off = run / b.rows1 * b.stride0 + run % b.rows1 * b.stride1 + at, bytes = min((int64_t)COPY_UNIT, b.bytes - at);
    const uint8_t* from = (const uint8_t*)b.ptr + w.src[i] * b.page_stride + off;
    uint8_t* to = (uint8_t*)b.ptr + w.dst[i] * b.page_stride + off;
    if (bufs.vec[k] == 16) copy_run<u32x4>(to, from, bytes);
    else if (bufs.vec[k] == 4) copy_run<uint32_t>(to, from, bytes);
    else copy_run<uint8_t>(to, from, bytes);
  }
}

void launch_pages_free(const lmoe_pages_args& a, hipStream_t st) {
  hipLaunchKernelGGL(k_pages_free, dim3(a.F), dim3(NTHR), 0, st, a);
}
void launch_pages_fork(const lmoe_pages_args& a, hipStream_t st) {
  hipLaunchKernelGGL(k_pages_snapshot, dim3(a.F), dim3(NTHR), 0, st, a);
  hipLaunchKernelGGL(k_pages_fork, dim3(a.F), dim3(NTHR), 0, st, a);
}
static void pages_copies(const lmoe_pages_args& a, int64_t most, hipStream_t st) {
  for (int k0 = 0; k0 < a.n_bufs; k0 += COPY_BUFS) {
    PageBufs p;
    p.n = std::min(COPY_BUFS, a.n_bufs - k0);
    p.units[0] = 0;
    for (int k = 0; k < p.n; ++k) {
      const lmoe_page_buf& b = p.b[k] = a.bufs[k0 + k];
      p.per[k] = (int32_t)((b.bytes + COPY_UNIT - 1) / COPY_UNIT);
      p.units[k + 1] = p.units[k] + (int32_t)((int64_t)b.rows0 * b.rows1 * p.per[k]);
      const uint64_t bits = (uintptr_t)b.ptr | (uint64_t)(b.page_stride | b.stride0 | b.stride1 | b.bytes);
      p.vec[k] = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
    }
    const int64_t units = most * p.units[p.n];
    if (units > 0) hipLaunchKernelGGL(k_pages_copy, dim3((uint32_t)std::min<int64_t>(units, 2048)), dim3(NTHR), 0, st, a, p);
  }
}
void launch_pages_reserve(const lmoe_pages_args& a, hipStream_t st) {
  hipLaunchKernelGGL(k_pages_reserve, dim3(1), dim3(PAGES_NTHR), 0, st, a);
  pages_copies(a, std::min<int64_t>(a.P, (int64_t)a.N * a.M), st);
}
void launch_pages_compact(const lmoe_pages_args& a, hipStream_t st) {
  hipLaunchKernelGGL(k_pages_compact, dim3(1), dim3(PAGES_NTHR), 0, st, a);
  const int64_t all = (int64_t)a.N * a.M;
  if (all) hipLaunchKernelGGL(k_pages_renamed, dim3((uint32_t)std::min<int64_t>((all + NTHR - 1) / NTHR, 1024)), dim3(NTHR), 0, st, a);
  pages_copies(a, a.P / 2, st);
}

}  // namespace lmoe
