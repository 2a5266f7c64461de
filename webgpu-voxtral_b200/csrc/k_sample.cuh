// k_sample.cuh — one token drawn from each row of logits: temperature, min-p, top-k, top-p,
// and a uniform number that the caller gives.
//
// With x the row's logits, w_i = exp((x_i - max x) / T) (0 for -inf and NaN).  The kept tokens
// are a run at the head of the descending order (equal logits in index order):
//   min-p  drops w_i < min_p;
//   top-k  keeps the first k of what is left;
//   top-p  keeps the shortest run whose mass reaches top_p of the mass of what is left.
// The draw is the first token, in that order, whose running mass reaches u x (kept mass).
//
// Masses are whole numbers, round(w 2^44), w in f64 (sums of up to 2^18 of them fit 64 bits):
// their order of addition does not matter, so the result is the same in every run, and a
// boundary is off by less than 2^-44 of the most likely token a token.  f32 weights would move
// boundaries by 2^-24, which at 131072 tokens of about equal weight changes one draw in a
// hundred.
//
// No sort of the row.  A cluster of 1 to 8 CTAs shares a row (kept in shared memory where the
// slices are small, read again from L2 where not).  After the pass for the maximum, one pass puts
// each survivor's count and mass into one of 2048 bins, linear in the logit; running sums over the
// bins (each CTA sums a share of them over the cluster) find the bin in which a count or mass is
// reached.  Where the whole head up to that bin is at most 512 tokens it is gathered into one
// CTA, sorted exactly, and all three limits are found in the sorted list; with top-k that head is
// found from counts alone, so only its tokens need an exponential.  Otherwise the tokens of the
// bin in question are gathered, binned again by their order key (logit, then index) and the few of
// one such bin sorted.  A bin of more than 1024 tokens is first binned again over the cluster by the
// same key; runs of equal logits need nothing of their own, as their keys differ in the index.
//
// Bound: not HBM (200 rows of 131072 f32 logits would take 16 us) but the pass of the masses, about
// 45 instructions and two or three shared-memory atomics a logit.  One B200: those 200 rows 143 us
// with top-p 0.95, 67 us with top-k 50; 64 rows of 131072 bf16 logits with all filters 34 us (in a captured graph).
#pragma once
#include <cooperative_groups.h>

#include <type_traits>

#include "vx_ops.cuh"

namespace vx {
namespace sample {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kBins = 2048;
constexpr int kSub = kThreads;         // second-level bins, one a thread
constexpr int kHead = kThreads;        // tokens sorted at once, one a thread
constexpr int kList = 1024;            // tokens gathered at once
constexpr int kFew = 96;               // tokens of a list that are sorted rather than binned again
constexpr int kMaxCols = 262144;
constexpr int kResident = 16384;       // logits that a CTA keeps in shared memory, at most
constexpr int kMaxCluster = 8;
constexpr float kRangeLog2 = 45.f;     // w below 2^-45 rounds to mass 0

struct Params {
  const void* logits;
  long long stride;
  const double* u;
  const float *temperature, *top_p, *min_p;   // by row, or null: the value below for every row
  const int32_t* top_k;
  float temperature1, top_p1, min_p1;
  int top_k1;
  int32_t* out;
  int n, slice;
  int resident;   // the slice is kept in shared memory
};

// Where a running count or mass reaches a target.
struct Hit {
  uint32_t bin, cnt_before, cnt;
  u64 mass_before;
};
template <int N>
struct Bins {
  uint32_t cnt[N], lo[N], hi[N];       // counts, and masses in two words
};
struct Smem {
  Bins<kBins> bins;                    // this CTA's part of the row; then running sums of its share of bins
  Bins<kSub> sub;
  u64 list[kList], list2[kList];
  double exp2_tab[64];                 // 2^(j / 64)
  u64 scan64[16];
  uint32_t scan32[16];
  float2 red[16];
  float2 range_of[kMaxCluster];        // each CTA's largest and smallest, and the totals of each one's share of bins
  uint32_t tot_cnt[kMaxCluster];
  u64 tot_mass[kMaxCluster];
  u64 key_min, key_max;
  uint32_t n_list, n_list2, n_own, at;
  Hit hit, list_hit;
  uint32_t share_cnt;                  // what lies before this CTA's share of bins
  u64 share_mass;
  u64 res_mass;
  int res_idx;
  alignas(16) float x[4];              // the CTA's slice of the row
};

// Descending order of the logits, then the index: ascending keys.
__device__ __forceinline__ uint32_t desc_bits(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ u64 order_key(float x, int i) { return ((u64)desc_bits(x) << 32) | (uint32_t)i; }
__device__ __forceinline__ float key_logit(u64 k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float((b & 0x80000000u) ? b : ~b & 0x7fffffffu);
}

// Running sums of counts and masses over the threads, this thread's included.
__device__ __forceinline__ void block_scan(Smem& s, uint32_t& c, u64& m) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, c, o);
    const u64 z = __shfl_up_sync(0xffffffffu, m, o);
    if (lane >= o) {
      c += y;
      m += z;
    }
  }
  if (lane == 31) {
    s.scan32[w] = c;
    s.scan64[w] = m;
  }
  __syncthreads();
  // the warps' totals, 16 of them, summed by every warp for itself
  uint32_t cw = lane < kThreads / 32 ? s.scan32[lane] : 0u;
  u64 mw = lane < kThreads / 32 ? s.scan64[lane] : 0ull;
#pragma unroll
  for (int o = 1; o < kThreads / 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, cw, o);
    const u64 z = __shfl_up_sync(0xffffffffu, mw, o);
    if (lane >= o) {
      cw += y;
      mw += z;
    }
  }
  cw = __shfl_sync(0xffffffffu, cw, (w + 31) & 31);
  mw = __shfl_sync(0xffffffffu, mw, (w + 31) & 31);
  if (w) {
    c += cw;
    m += mw;
  }
  __syncthreads();
}
__device__ __forceinline__ u64 block_scan(Smem& s, u64 m) {
  uint32_t c = 0;
  block_scan(s, c, m);
  return m;
}

// The cluster of C CTAs that holds a row; one CTA needs no more than its own barrier.
template <int C>
__device__ __forceinline__ void cluster_barrier() {
  if constexpr (C == 1) __syncthreads();
  else cg::this_cluster().sync();
}
template <int C>
__device__ __forceinline__ Smem* of_rank(Smem& s, int q) {
  if constexpr (C == 1) return &s;
  else return cg::this_cluster().map_shared_rank(&s, q);
}
template <int C>
__device__ __forceinline__ int my_rank() {
  if constexpr (C == 1) return 0;
  else return (int)cg::this_cluster().block_rank();
}

struct Row {
  float mx, cut, scale;                // bin (mx - x) * scale; nothing further than cut below mx survives
  int sure;                            // every logit of the bins below this one survives
  double mxd, c64, min_p44;            // 64 log2(e) / T; min_p 2^44
};
// 2^(j / 64), rounded.
__device__ const double kExp2[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};
// round(w 2^44) of a logit within 2^-60 of the largest.  2^(t / 64) by the table and the Taylor sum
// of the rest, |r| <= 1/2 of a 64th (table-driven exponential, Tang 1989): the fifth power's term is
// below 4e-14.
__device__ __forceinline__ double weight44(const Smem& s, const Row& r, float x) {
  constexpr double a = 0.010830424696249145;   // ln 2 / 64
  const double t = ((double)x - r.mxd) * r.c64;
  const double shifted = t + 6755399441055744.0;   // 1.5 * 2^52: the nearest whole number in the low bits
  const int n = __double2loint(shifted);
  const double f = t - (shifted - 6755399441055744.0);
  const double poly = fma(f, fma(f, fma(f, fma(f, a * a * a * a / 24.0, a * a * a / 6.0), a * a / 2.0), a), 1.0);
  const double v = s.exp2_tab[n & 63] * poly;
  // times 2^(n / 64 + 44) in the exponent field
  return __hiloint2double(__double2hiint(v) + (((n >> 6) + 44) << 20), __double2loint(v));
}
__device__ __forceinline__ u64 whole(double w44) {   // + 2^52: whole in the mantissa
  return (u64)__double_as_longlong(w44 + 4503599627370496.0) & 0xfffffffffffffull;
}
// Mass of a logit of bin b >= 0, 0 where min-p drops it.
__device__ __forceinline__ u64 mass_of(const Smem& s, const Row& r, float x, int b) {
  const double w = weight44(s, r, x);
  return b < r.sure || w >= r.min_p44 ? whole(w) : 0ull;
}
// Mass of a token that is known to survive.
__device__ __forceinline__ u64 mass_of(const Smem& s, const Row& r, float x) { return whole(weight44(s, r, x)); }
// Bin of a logit, -1 for one that cannot survive (the exact test is mass_of's).
__device__ __forceinline__ int bin_of(const Row& r, float x) {
  const float d = r.mx - x;
  return d <= r.cut ? (int)(d * r.scale) : -1;
}
// Smallest distance from the maximum that falls into bin b or a later one.
__device__ __forceinline__ float bin_edge(const Row& r, int b) {
  if (b <= 0) return 0.f;
  if (b >= kBins) return INFINITY;
  float d = (float)b / r.scale;
  for (int i = 0; i < 4 && d > 0.f && __uint_as_float(__float_as_uint(d) - 1) * r.scale >= (float)b; ++i) d = __uint_as_float(__float_as_uint(d) - 1);
  for (int i = 0; i < 4 && d * r.scale < (float)b; ++i) d = __uint_as_float(__float_as_uint(d) + 1);
  return d;
}
// Whether a logit of bin b survives.
__device__ __forceinline__ bool survives(const Smem& s, const Row& r, float x, int b) {
  return b < r.sure || mass_of(s, r, x, b) > 0;
}

template <int N>
__device__ __forceinline__ void bins_clear(Bins<N>& b) {
  for (int i = threadIdx.x; i < N; i += kThreads) b.cnt[i] = b.lo[i] = b.hi[i] = 0;
}
template <int N>
__device__ __forceinline__ void bins_add(Bins<N>& b, int i, u64 m) {
  atomicAdd(&b.cnt[i], 1u);
  const uint32_t l = (uint32_t)m, old = atomicAdd(&b.lo[i], l);
  const uint32_t h = (uint32_t)(m >> 32) + (old + l < old ? 1u : 0u);
  if (h) atomicAdd(&b.hi[i], h);
}

// Running sums of the row's bins: this CTA's share of them, [rank kBins / C, ...), replaces its bins.
// Gives the row's total count and mass.
template <int C>
__device__ void sum_bins(Smem& s, uint32_t& cnt_all, u64& mass_all) {
  constexpr int share = kBins / C, per = (share + kThreads - 1) / kThreads;   // bins a thread
  const int t = threadIdx.x, rank = my_rank<C>();
  const bool on = t * per < share;
  cluster_barrier<C>();
  uint32_t c[per];
  u64 m[per];
#pragma unroll
  for (int j = 0; j < per; ++j) {
    uint32_t cq[C], lq[C], hq[C];
#pragma unroll
    for (int q = 0; q < C; ++q) {
      const Smem* o = of_rank<C>(s, q);
      const int b = rank * share + (on ? t * per + j : 0);
      cq[q] = o->bins.cnt[b];
      lq[q] = o->bins.lo[b];
      hq[q] = o->bins.hi[b];
    }
    c[j] = 0;
    m[j] = 0;
#pragma unroll
    for (int q = 0; q < C; ++q) {
      c[j] += on ? cq[q] : 0u;
      m[j] += on ? ((u64)hq[q] << 32) + lq[q] : 0ull;
    }
  }
  uint32_t c_to = 0;
  u64 m_to = 0;
#pragma unroll
  for (int j = 0; j < per; ++j) {
    c_to += c[j];
    m_to += m[j];
  }
  uint32_t c_before = c_to;
  u64 m_before = m_to;
  block_scan(s, c_to, m_to);
  if (t == kThreads - 1)
#pragma unroll
    for (int q = 0; q < C; ++q) {
      Smem* o = of_rank<C>(s, q);
      o->tot_cnt[rank] = c_to;
      o->tot_mass[rank] = m_to;
    }
  cluster_barrier<C>();                        // the totals are there, and every CTA has read the others' bins
  c_before = c_to - c_before;
  m_before = m_to - m_before;
  cnt_all = 0;
  mass_all = 0;
  uint32_t c_share = 0;
  u64 m_share = 0;
#pragma unroll
  for (int q = 0; q < C; ++q) {
    if (q < rank) {
      c_share += s.tot_cnt[q];
      m_share += s.tot_mass[q];
    }
    cnt_all += s.tot_cnt[q];
    mass_all += s.tot_mass[q];
  }
  if (t == 0) {
    s.share_cnt = c_share;
    s.share_mass = m_share;
  }
  c_before += c_share;
  m_before += m_share;
  if (on)
#pragma unroll
    for (int j = 0; j < per; ++j) {
      c_before += c[j];
      m_before += m[j];
      s.bins.cnt[t * per + j] = c_before;
      s.bins.lo[t * per + j] = (uint32_t)m_before;
      s.bins.hi[t * per + j] = (uint32_t)(m_before >> 32);
    }
  __syncthreads();
}
// The bin in which the target is reached, in s.hit of every CTA.
template <int C>
__device__ void find_bin(Smem& s, bool by_count, u64 target) {
  constexpr int share = kBins / C;
#pragma unroll
  for (int b = threadIdx.x; b < share; b += kThreads) {
    const uint32_t c1 = s.bins.cnt[b], c0 = b ? s.bins.cnt[b - 1] : s.share_cnt;
    const u64 m1 = ((u64)s.bins.hi[b] << 32) + s.bins.lo[b];
    const u64 m0 = b ? ((u64)s.bins.hi[b - 1] << 32) + s.bins.lo[b - 1] : s.share_mass;
    const u64 from = by_count ? (u64)c0 : m0, to = by_count ? (u64)c1 : m1;
    if (from < target && to >= target)
#pragma unroll
      for (int q = 0; q < C; ++q) of_rank<C>(s, q)->hit = Hit{(uint32_t)(my_rank<C>() * share + b), c0, c1 - c0, m0};
  }
  cluster_barrier<C>();
}

// The CTA's slice of the row: in shared memory, or read again from global memory (L2) each time.
template <typename T>
struct Slice {
  const T* g;
  int n;
  bool resident, wide;                 // wide: four logits in one load
  bool inf;                            // the row holds +inf: those draw as logits 0, the others not at all
};
__device__ __forceinline__ float clean(float x) {
  x += 0.f;                            // -0 counts as 0
  return x == x ? x : -INFINITY;       // NaN is never drawn
}
// Calls f(x, i) for the logits of the slice, x[0..3] at i (-inf past the end).  Four loads a thread are
// on their way before the first is used: neither the branches of a ragged end nor what f does to
// shared memory stand between them.  Ordinary loads: the kernel before may still be writing the logits when
// this one starts, and the read-only path holds only for what nobody writes while a kernel is there.
template <typename T, bool FIRST, typename F>
__device__ __forceinline__ void each_four(const Smem& s, const Slice<T>& sl, F f) {
  constexpr int U = 4, STEP = 4 * kThreads;
  for (int i0 = 4 * threadIdx.x; i0 < sl.n; i0 += U * STEP) {
    float x[U][4];
    const bool all = i0 + (U - 1) * STEP + 4 <= sl.n;
    if (!FIRST && sl.resident) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // past the end: the last four again, not used
        const float4 q = *reinterpret_cast<const float4*>(&s.x[min(i0 + u * STEP, (sl.n - 1) & ~3)]);
        x[u][0] = q.x; x[u][1] = q.y; x[u][2] = q.z; x[u][3] = q.w;
      }
    } else {
      if (sl.wide && all) {
        typedef typename std::conditional<sizeof(T) == 4, float4, uint2>::type Four;
        Four q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = *reinterpret_cast<const Four*>(sl.g + i0 + u * STEP);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if constexpr (sizeof(T) == 4) {
            x[u][0] = q[u].x; x[u][1] = q[u].y; x[u][2] = q[u].z; x[u][3] = q[u].w;
          } else {
            const float2 a = ops::Elem<T>::unpack(q[u].x), b = ops::Elem<T>::unpack(q[u].y);
            x[u][0] = a.x; x[u][1] = a.y; x[u][2] = b.x; x[u][3] = b.y;
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) x[u][j] = i0 + u * STEP + j < sl.n ? ops::Elem<T>::to_f32(sl.g[i0 + u * STEP + j]) : -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][j] = clean(x[u][j]);
      if (!FIRST && sl.inf)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) x[u][j] = x[u][j] == INFINITY ? 0.f : -INFINITY;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (all || i0 + u * STEP < sl.n) f(x[u], i0 + u * STEP);
  }
}

// Puts the cluster's tokens of the bins [bin0, bin1] whose order keys are in [k0, k1] into the list of
// CTA 0, whose n_list is 0: first into a list of the CTA's own, then those together.
template <typename T, int C>
__device__ __forceinline__ void gather(Smem& s, const Row& r, const Slice<T>& sl, int base, int bin0, int bin1, u64 k0, u64 k1) {
  if constexpr (C > 1) {
    if (threadIdx.x == 0) s.n_own = 0;
    __syncthreads();
  }
  uint32_t* count = C > 1 ? &s.n_own : &s.n_list;
  u64* list = C > 1 ? s.list2 : s.list;
  // the bins as a range [d0, d1) of distances from the maximum; the exact tests where they may matter
  const float d0 = bin_edge(r, bin0), d1 = fminf(bin_edge(r, bin1 + 1), nextafterf(r.cut, INFINITY));
  const bool keys = k0 > 0 || k1 < ~0ull, border = bin1 >= r.sure;
  each_four<T, false>(s, sl, [&](const float (&x)[4], int i) {
    float d[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j] = r.mx - x[j];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (d[j] >= d0 && d[j] < d1) {
        const u64 k = order_key(x[j], base + i + j);
        if (keys && (k < k0 || k > k1)) continue;
        if (border && !survives(s, r, x[j], bin_of(r, x[j]))) continue;
        const uint32_t at = atomicAdd(count, 1u);
        if (at < (uint32_t)kList) list[at] = k;
      }
  });
  if constexpr (C > 1) {
    __syncthreads();
    const uint32_t own = min(s.n_own, (uint32_t)kList);
    Smem* head = of_rank<C>(s, 0);
    if (threadIdx.x == 0) s.at = own ? atomicAdd(&head->n_list, own) : 0u;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < own; i += kThreads)
      if (s.at + i < (uint32_t)kList) head->list[s.at + i] = s.list2[i];
  }
  cluster_barrier<C>();
}

// Sorts `c` (at most one a thread) distinct keys: each counts the smaller ones.  Gives this thread's
// key of the sorted order (~0 past the end).
__device__ u64 sorted(Smem& s, const u64* list, int c) {
  const int t = threadIdx.x;
  // several threads share a key's comparisons where there are few keys
  int ways = 1;
  while (ways < 16 && c * ways * 2 <= kThreads) ways *= 2;
  const int e = t / ways, part = t % ways;
  const u64 mine = e < c ? list[e] : ~0ull;
  uint32_t less = 0;
  for (int i = part; i < c; i += ways) less += list[i] < mine;
  for (int o = ways >> 1; o > 0; o >>= 1) less += __shfl_xor_sync(0xffffffffu, less, o);
  __syncthreads();                             // all have read the list before it may be the target
  if (part == 0 && e < c) s.list2[less] = mine;
  __syncthreads();
  const u64 k = t < c ? s.list2[t] : ~0ull;
  __syncthreads();
  return k;
}

// In CTA 0, whose list holds the c <= kList tokens of hit: the first whose running count or mass
// reaches the target.  Index and running mass to res_idx / res_mass of every CTA.
template <int C>
__device__ void resolve_list(Smem& s, const Row& r, int c, uint32_t cnt_before, u64 mass_before, bool by_count, u64 target) {
  const int t = threadIdx.x;
  for (int level = 0; level < 8 && c > kFew; ++level) {
    // bins over the span of the keys; the tokens of the bin in question replace the list.  A bin
    // holds less than a 256th of the span, so eight rounds end at single keys
    if (t == 0) {
      s.key_min = ~0ull;
      s.key_max = 0;
      s.n_list2 = 0;
    }
    bins_clear(s.sub);
    __syncthreads();
    u64 key[kList / kThreads], lo = ~0ull, hi = 0;
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j) {
      const int i = t + j * kThreads;
      key[j] = i < c ? s.list[i] : ~0ull;
      if (i < c) {
        lo = min(lo, key[j]);
        hi = max(hi, key[j]);
      }
    }
    for (int o = 16; o > 0; o >>= 1) {
      lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if ((t & 31) == 0) {
      atomicMin(&s.key_min, lo);
      atomicMax(&s.key_max, hi);
    }
    __syncthreads();
    lo = s.key_min;
    const int shift = max(0, 64 - __clzll((long long)(s.key_max - lo)) - 9);
    u64 mass[kList / kThreads];
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j)
      if (t + j * kThreads < c) {
        mass[j] = mass_of(s, r, key_logit(key[j]));
        bins_add(s.sub, (int)((key[j] - lo) >> shift), mass[j]);
      }
    __syncthreads();
    const uint32_t bc = s.sub.cnt[t];
    const u64 bm = ((u64)s.sub.hi[t] << 32) + s.sub.lo[t];
    uint32_t c_to = bc;
    u64 m_to = bm;
    block_scan(s, c_to, m_to);
    c_to += cnt_before;
    m_to += mass_before;
    const u64 to = by_count ? (u64)c_to : m_to, from = to - (by_count ? (u64)bc : bm);
    if (from < target && to >= target) s.list_hit = Hit{(uint32_t)t, c_to - bc, bc, m_to - bm};
    __syncthreads();
    const Hit h = s.list_hit;
#pragma unroll
    for (int j = 0; j < kList / kThreads; ++j)
      if (t + j * kThreads < c && (uint32_t)((key[j] - lo) >> shift) == h.bin) s.list[atomicAdd(&s.n_list2, 1u)] = key[j];
    __syncthreads();
    c = (int)h.cnt;
    cnt_before = h.cnt_before;
    mass_before = h.mass_before;
  }
  c = min(c, kThreads);
  const u64 key = sorted(s, s.list, c);
  const u64 m = t < c ? mass_of(s, r, key_logit(key)) : 0ull;
  const u64 to_m = mass_before + block_scan(s, m);
  const u64 to = by_count ? (u64)cnt_before + t + 1 : to_m, from = by_count ? to - 1 : to - m;
  if (t < c && from < target && to >= target)
#pragma unroll
    for (int q = 0; q < C; ++q) {
      Smem* o = of_rank<C>(s, q);
      o->res_idx = (int)(uint32_t)key;
      o->res_mass = to_m;
    }
}

// First token in order whose running count (by_count) or mass reaches the target; the row's bins
// hold it.  Gives its index and the running mass up to and with it, in every CTA.
// Arguments by value, and shared memory by its own name: what is reached through a reference is read
// again after every store.
template <typename T, int C>
__device__ __noinline__ void select(const Row r, const Slice<T> sl, int base, bool by_count, u64 target) {
  extern __shared__ __align__(16) unsigned char raw[];
  Smem& s = *reinterpret_cast<Smem*>(raw);
  const int t = threadIdx.x;
  find_bin<C>(s, by_count, target);
  Hit h = s.hit;
  const int bin = (int)h.bin;
  u64 k0 = 0, k1 = ~0ull;                      // order keys of the tokens in question, inside the bin
  const auto member = [&](float x, int i) {
    if (bin_of(r, x) != bin) return false;
    const u64 k = order_key(x, i);
    return k >= k0 && k <= k1 && survives(s, r, x, bin);
  };
  // each level takes 9 bits off the span, so the sixth leaves fewer than a list holds
  for (int level = 0; level < 8 && h.cnt > (uint32_t)kList; ++level) {
    if (t == 0) {
      s.key_min = ~0ull;
      s.key_max = 0;
    }
    bins_clear(s.sub);
    __syncthreads();
    u64 lo = ~0ull, hi = 0;
    each_four<T, false>(s, sl, [&](const float (&x)[4], int i) {
#pragma unroll 1
      for (int j = 0; j < 4; ++j)
        if (member(x[j], base + i + j)) {
          const u64 k = order_key(x[j], base + i + j);
          lo = min(lo, k);
          hi = max(hi, k);
        }
    });
    for (int o = 16; o > 0; o >>= 1) {
      lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if ((t & 31) == 0) {
      atomicMin(&s.key_min, lo);
      atomicMax(&s.key_max, hi);
    }
    cluster_barrier<C>();
    for (int q = 0; q < C; ++q) {
      const Smem* o = of_rank<C>(s, q);
      lo = min(lo, o->key_min);
      hi = max(hi, o->key_max);
    }
    k0 = lo;
    k1 = hi;
    const int shift = max(0, 64 - __clzll((long long)(k1 - k0)) - 9);
    each_four<T, false>(s, sl, [&](const float (&x)[4], int i) {
#pragma unroll 1
      for (int j = 0; j < 4; ++j)
        if (member(x[j], base + i + j)) bins_add(s.sub, (int)((order_key(x[j], base + i + j) - k0) >> shift), mass_of(s, r, x[j]));
    });
    cluster_barrier<C>();
    uint32_t c = 0;
    u64 m = 0;
    for (int q = 0; q < C; ++q) {
      const Smem* o = of_rank<C>(s, q);
      c += o->sub.cnt[t];
      m += ((u64)o->sub.hi[t] << 32) + o->sub.lo[t];
    }
    uint32_t c_to = c;
    u64 m_to = m;
    block_scan(s, c_to, m_to);
    c_to += h.cnt_before;
    m_to += h.mass_before;
    const u64 to = by_count ? (u64)c_to : m_to, from = to - (by_count ? (u64)c : m);
    if (from < target && to >= target) s.hit = Hit{(uint32_t)t, c_to - c, c, m_to - m};   // the same in every CTA
    cluster_barrier<C>();
    h = s.hit;
    k0 += (u64)h.bin << shift;
    k1 = min(k1, k0 + ((1ull << shift) - 1ull));
  }
  gather<T, C>(s, r, sl, base, bin, bin, k0, k1);
  if (my_rank<C>() == 0) {
    resolve_list<C>(s, r, (int)min(h.cnt, (uint32_t)kList), h.cnt_before, h.mass_before, by_count, target);
    if (t == 0) s.n_list = 0;
  }
  cluster_barrier<C>();
}

// Largest and smallest finite logit of the slice; fills the resident copy.
template <typename T>
__device__ __forceinline__ void scan_slice(Smem& s, const Slice<T>& sl, float& mx, float& mn) {
  mx = -INFINITY;
  mn = INFINITY;
  each_four<T, true>(s, sl, [&](const float (&x)[4], int i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      mx = fmaxf(mx, x[j]);
      mn = fminf(mn, x[j] == -INFINITY ? INFINITY : x[j]);
    }
    if (sl.resident) *reinterpret_cast<float4*>(&s.x[i]) = make_float4(x[0], x[1], x[2], x[3]);
  });
}

template <typename T, int C>
__global__ void __launch_bounds__(kThreads, 2) k_sample(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) unsigned char raw[];
  Smem& s = *reinterpret_cast<Smem*>(raw);
  const int t = threadIdx.x;
  const long long row = blockIdx.x / C;
  const int rank = my_rank<C>(), base = rank * p.slice;
  Slice<T> sl;
  sl.g = (const T*)p.logits + row * p.stride + base;
  sl.n = max(0, min(p.slice, p.n - base));
  sl.resident = p.resident;
  sl.wide = reinterpret_cast<uintptr_t>(sl.g) % (4 * sizeof(T)) == 0;
  sl.inf = false;
  if (t < 64) s.exp2_tab[t] = kExp2[t];
  bins_clear(s.bins);
  if (t == 0) s.n_list = 0;
  if constexpr (C > 1) cg::this_cluster().barrier_arrive();
  griddep_launch();
  griddep_wait();

  // ---- the row's largest and smallest logit
  float mx, mn;
  scan_slice(s, sl, mx, mn);
  mx = warp_max(mx);
  mn = -warp_max(-mn);
  if ((t & 31) == 0) s.red[t >> 5] = make_float2(mx, mn);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    mx = fmaxf(mx, s.red[i].x);
    mn = fminf(mn, s.red[i].y);
  }
  if constexpr (C > 1) {
    cg::this_cluster().barrier_wait();         // every CTA runs, so that its memory may be written
    if (t < C) of_rank<C>(s, t)->range_of[rank] = make_float2(mx, mn);
    cluster_barrier<C>();
#pragma unroll
    for (int q = 0; q < C; ++q) {
      mx = fmaxf(mx, s.range_of[q].x);
      mn = fminf(mn, s.range_of[q].y);
    }
  }
  if (mx == -INFINITY) {   // nothing to draw from
    if (rank == 0 && t == 0) p.out[row] = -1;
    return;
  }
  if (mx == INFINITY) {
    sl.inf = true;
    mx = mn = 0.f;
    if (sl.resident)
      for (int i = t; i < sl.n; i += kThreads) s.x[i] = s.x[i] == INFINITY ? 0.f : -INFINITY;
    __syncthreads();
  }

  Row r;
  double temp = (double)(p.temperature ? p.temperature[row] : p.temperature1);
  int k = p.top_k ? p.top_k[row] : p.top_k1;
  const double top_p = (double)(p.top_p ? p.top_p[row] : p.top_p1);
  const double min_p = fmin(1.0, (double)(p.min_p ? p.min_p[row] : p.min_p1));
  const double u = p.u[row];
  if (!(temp > 0.0)) {   // greedy
    temp = 1.0;
    k = 1;
  }
  temp = fmin(temp, 1e30);                     // uniform by then
  r.mx = mx;
  r.mxd = (double)mx;
  r.c64 = 64.0 * 1.4426950408889634 / temp;
  r.min_p44 = min_p * 17592186044416.0;
  // how far below the maximum a logit can survive: until its mass rounds to 0, or to min-p; and at
  // least to 0.999 of that, so that the bins there need no exact test
  const double to_logit = temp * 0.6931471805599453;
  const double far = min_p > 0.0 ? fmin(-log2(min_p), (double)kRangeLog2) : (double)kRangeLog2;
  const float span = fmaxf(mx - mn, 1e-30f);                   // bins need not reach past the smallest
  r.cut = fminf((float)(far * to_logit * 1.001 + 1e-6 * to_logit), span);
  // finite: below a cut of 6e-36 (temperatures under 2e-37, or any with min-p near 1) the bins are wider
  // than they need be, which costs an exact pass over more tokens and changes no result
  r.scale = fminf((float)(kBins - 1) / r.cut, 3.402823466e38f);
  const float sure = fminf((float)(far * to_logit * 0.999), span) * r.scale;
  r.sure = sure < (float)(kBins - 1) ? (int)sure : mx - mn < (float)(far * to_logit * 0.999) ? kBins : kBins - 1;
  const auto reach = [](double share, u64 of) {   // the whole-number mass that `share` of `of` asks for
    if (!(share > 0.0)) return (u64)1;
    const u64 v = (u64)ceil(share * (double)of);
    return v < 1 ? (u64)1 : v > of ? of : v;
  };

  // ---- the head that decides: up to the bin of the k-th token (from counts alone), of the top-p
  // mass, or of the draw
  bool cut_k = k > 0 && k < p.n;
  const bool cut_p = top_p < 1.0;
  uint32_t total;
  u64 kept;
  int head = 0x7fffffff;
  if (cut_k && k <= kHead) {
    each_four<T, false>(s, sl, [&](const float (&x)[4], int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b = bin_of(r, x[j]);
        if (b >= 0) atomicAdd(&s.bins.cnt[b], 1u);
      }
    });
    sum_bins<C>(s, total, kept);
    if (total <= (uint32_t)kHead) {
      head = (int)total;
      if (t == 0) s.hit.bin = kBins - 1;
      __syncthreads();
    } else {
      find_bin<C>(s, true, (u64)k);           // total > kHead >= k: it is there
      head = (int)(s.hit.cnt_before + s.hit.cnt);
    }
    if (head > kHead) {                        // many equal or near-equal logits around the k-th
      cluster_barrier<C>();
      bins_clear(s.bins);
      __syncthreads();
    }
  }
  if (head > kHead) {
    each_four<T, false>(s, sl, [&](const float (&x)[4], int) {
      int b[4];
      double w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        b[j] = bin_of(r, x[j]);
        w[j] = weight44(s, r, x[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 m = b[j] < r.sure || w[j] >= r.min_p44 ? whole(w[j]) : 0ull;
        if (b[j] >= 0 && m) bins_add(s.bins, b[j], m);
      }
    });
    sum_bins<C>(s, total, kept);
    cut_k = cut_k && (uint32_t)k < total;
    find_bin<C>(s, cut_k, cut_k ? (u64)k : reach(cut_p ? top_p : u, kept));
    head = (int)(s.hit.cnt_before + s.hit.cnt);
  }
  if (head <= kHead) {
    const int last = (int)s.hit.bin;
    gather<T, C>(s, r, sl, base, 0, last, 0ull, ~0ull);
    if (rank == 0) {
      const int c = (int)s.n_list;             // exact survivors: at most `head`
      const u64 key = sorted(s, s.list, c);
      const u64 m = t < c ? mass_of(s, r, key_logit(key)) : 0ull;
      const u64 to = block_scan(s, m), from = to - m;
      if (cut_k || last == kBins - 1) {        // the list holds all that is left
        if (t == min(c, cut_k ? k : c) - 1) s.res_mass = to;
        __syncthreads();
        kept = s.res_mass;
        __syncthreads();
      }
      if (cut_p) {
        const u64 g = reach(top_p, kept);
        if (from < g && to >= g) s.res_mass = to;
        __syncthreads();
        kept = s.res_mass;
        __syncthreads();
      }
      const u64 g = reach(u, kept);
      if (from < g && to >= g) p.out[row] = (int32_t)(uint32_t)key;
    }
    return;
  }
  if (cut_k) {
    select<T, C>(r, sl, base, true, (u64)k);
    kept = s.res_mass;
  }
  if (cut_p) {
    select<T, C>(r, sl, base, false, reach(top_p, kept));
    kept = s.res_mass;
  }
  select<T, C>(r, sl, base, false, reach(u, kept));
  if (rank == 0 && t == 0) p.out[row] = s.res_idx;
}

}  // namespace sample
}  // namespace vx
