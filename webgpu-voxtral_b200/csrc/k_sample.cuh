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
// No sort of the row.  The row lies in the shared memory of a cluster of 1 to 8 CTAs.  One pass
// puts each survivor's count and mass into one of 1024 bins, linear in log w; sums over the bins
// find the bin in which a count or mass is reached.  Where the whole head up to that bin is at
// most 2048 tokens it is gathered and sorted exactly, and all three limits are found in the
// sorted list.  Otherwise only the tokens of the bin in question are; a bin with more than 2048
// is binned again by the bits of the logits, down to a run of equal logits, where the order is
// the index order.
#pragma once
#include <cooperative_groups.h>

#include "vx_ops.cuh"

namespace vx {
namespace sample {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kBins = kThreads;        // one a thread
constexpr int kList = 2 * kThreads;    // tokens sorted at once, two a thread
constexpr int kMaxSlice = 32768;       // logits a CTA holds
constexpr int kMaxCluster = 8;
constexpr float kRangeLog2 = 45.f;     // w below 2^-45 rounds to mass 0

struct Params {
  const void* logits;
  long long stride;
  const double* u;
  const float *temperature, *top_p, *min_p;   // by row, or null: the value below for every row
  const int32_t* top_k;
  double temperature1, top_p1, min_p1;
  int top_k1;
  int32_t* out;
  int n, slice;
};

struct Smem {
  uint32_t cnt[kBins], lo[kBins], hi[kBins];   // this CTA's bins: count, mass in two words
  u64 mass_to[kBins];                          // whole row: mass and count up to and with the bin
  uint32_t cnt_to[kBins];
  u64 list[kList];
  u64 scan64[32];
  uint32_t scan32[32];
  float red[32];
  float cta_max;
  uint32_t key_min, key_max;
  uint32_t n_list, eq_count;
  // where a target was reached (one thread writes, all read)
  int hit_bin;
  uint32_t hit_cnt_before, hit_cnt;
  u64 hit_mass_before;
  int res_idx;
  u64 res_mass;
  float x[1];                                  // the CTA's slice of the row
};

__device__ __forceinline__ uint32_t desc_key(float x) {   // ascending in the descending order of x
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ float from_desc_key(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k : ~k & 0x7fffffffu);
}

template <typename T>
__device__ __forceinline__ T block_incl_scan(T v, T* sh) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) sh[w] = v;
  __syncthreads();
  if (w == 0) {
    T s = sh[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    sh[lane] = s;
  }
  __syncthreads();
  if (w) v += sh[w - 1];
  __syncthreads();
  return v;
}

struct Row {
  float mx, bin_scale, cut_log2;   // bin = -(x - mx) * bin_scale; nothing below cut_log2 survives
  double inv_t, min_p;
  float c;                         // log2(e) / T
};
__device__ __forceinline__ u64 mass_of(const Row& r, float x) {
  const double w = x == r.mx ? 1.0 : exp(((double)x - (double)r.mx) * r.inv_t);
  return w >= r.min_p ? (u64)__double2ull_rn(w * 17592186044416.0) : 0ull;
}
// Bin of a logit, -1 for one that cannot survive (the exact test is mass_of's).
__device__ __forceinline__ int bin_of(const Row& r, float x) {
  if (x == r.mx) return 0;
  const float t = (r.mx - x) * r.c;
  if (!(t <= r.cut_log2)) return -1;
  return min(kBins - 1, (int)(t * r.bin_scale));
}

__device__ __forceinline__ void bins_clear(Smem& s) {
  s.cnt[threadIdx.x] = s.lo[threadIdx.x] = s.hi[threadIdx.x] = 0;
}
__device__ __forceinline__ void bins_add(Smem& s, int b, u64 m) {
  atomicAdd(&s.cnt[b], 1u);
  const uint32_t l = (uint32_t)m, old = atomicAdd(&s.lo[b], l);
  const uint32_t h = (uint32_t)(m >> 32) + (old + l < old ? 1u : 0u);
  if (h) atomicAdd(&s.hi[b], h);
}
// This thread's bin over the whole cluster, then its running sums.
__device__ __forceinline__ void bins_sum(Smem& s, cg::cluster_group& cl, uint32_t& cnt, u64& mass, uint32_t& cnt_to, u64& mass_to) {
  cl.sync();
  cnt = 0;
  mass = 0;
  for (unsigned r = 0; r < cl.num_blocks(); ++r) {
    const Smem* o = cl.map_shared_rank(&s, r);
    cnt += o->cnt[threadIdx.x];
    mass += ((u64)o->hi[threadIdx.x] << 32) + o->lo[threadIdx.x];
  }
  cl.sync();   // every CTA has read the others' bins
  cnt_to = block_incl_scan<uint32_t>(cnt, s.scan32);
  mass_to = block_incl_scan<u64>(mass, s.scan64);
}

// Sorts the first n of the list (ascending, kList at most) in this CTA.
__device__ void sort_list(Smem& s, int n) {
  int n2 = 2;
  while (n2 < n) n2 <<= 1;
  for (int i = threadIdx.x; i < n2; i += kThreads)
    if (i >= n) s.list[i] = ~0ull;
  __syncthreads();
  for (int k = 2; k <= n2; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      const int t = threadIdx.x;
      if (t < n2 / 2) {
        const int a = ((t & ~(j - 1)) << 1) | (t & (j - 1)), b = a | j;
        const u64 x = s.list[a], y = s.list[b];
        if ((x > y) == ((a & k) == 0)) {
          s.list[a] = y;
          s.list[b] = x;
        }
      }
      __syncthreads();
    }
}

// Puts the cluster's tokens for which `take` holds into the list of CTA 0.
template <typename F>
__device__ void gather(Smem& s, cg::cluster_group& cl, int base, int n, F take) {
  Smem* head = cl.map_shared_rank(&s, 0);
  if (cl.block_rank() == 0 && threadIdx.x == 0) s.n_list = 0;
  cl.sync();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float x = s.x[i];
    if (take(x)) head->list[atomicAdd(&head->n_list, 1u) & (kList - 1)] = ((u64)desc_key(x) << 32) | (uint32_t)(base + i);
  }
  cl.sync();
}

// First token in order whose running count (by_count) or mass reaches the target; the row's
// bins hold it.  Gives its index and the running mass up to and with it, in every CTA.
__device__ void select(Smem& s, cg::cluster_group& cl, const Row& r, int base, int n, bool by_count, u64 target) {
  const int t = threadIdx.x;
  {
    const u64 to = by_count ? (u64)s.cnt_to[t] : s.mass_to[t];
    const u64 from = t ? (by_count ? (u64)s.cnt_to[t - 1] : s.mass_to[t - 1]) : 0ull;
    if (from < target && to >= target) {
      s.hit_bin = t;
      s.hit_cnt_before = t ? s.cnt_to[t - 1] : 0u;
      s.hit_cnt = s.cnt_to[t] - s.hit_cnt_before;
      s.hit_mass_before = t ? s.mass_to[t - 1] : 0ull;
    }
  }
  __syncthreads();
  const int bin = s.hit_bin;
  uint32_t k0 = 0, k1 = 0xffffffffu;   // desc_key range of the tokens in question, inside the bin
  const auto member = [&](float x) {
    const uint32_t k = desc_key(x);
    return bin_of(r, x) == bin && k >= k0 && k <= k1 && mass_of(r, x) > 0;
  };
  // every level takes 10 bits off the span, so the fourth leaves single logits
  for (int level = 0; level < 8; ++level) {
    const uint32_t cnt = s.hit_cnt, cnt_before = s.hit_cnt_before;
    const u64 mass_before = s.hit_mass_before;
    __syncthreads();
    if (cnt <= (uint32_t)kList) {
      gather(s, cl, base, n, member);
      if (cl.block_rank() == 0) {
        const int c = (int)cnt;
        sort_list(s, c);
        u64 m0 = 0, m1 = 0;
        if (2 * t < c) m0 = mass_of(r, from_desc_key((uint32_t)(s.list[2 * t] >> 32)));
        if (2 * t + 1 < c) m1 = mass_of(r, from_desc_key((uint32_t)(s.list[2 * t + 1] >> 32)));
        const u64 to1 = mass_before + block_incl_scan<u64>(m0 + m1, s.scan64), to0 = to1 - m1;
        const u64 c0 = by_count ? cnt_before + 2ull * t : to0 - m0, c1 = by_count ? c0 + 1 : to0, c2 = by_count ? c0 + 2 : to1;
        const bool in0 = 2 * t < c && c0 < target && c1 >= target, in1 = 2 * t + 1 < c && c1 < target && c2 >= target;
        if (in0 || in1)
          for (unsigned q = 0; q < cl.num_blocks(); ++q) {
            Smem* o = cl.map_shared_rank(&s, q);
            o->res_idx = (int)(uint32_t)s.list[2 * t + (in0 ? 0 : 1)];
            o->res_mass = in0 ? to0 : to1;
          }
      }
      cl.sync();
      return;
    }
    // too many: the span of their logits, then bins over it
    if (t == 0) {
      s.key_min = 0xffffffffu;
      s.key_max = 0;
    }
    bins_clear(s);
    __syncthreads();
    uint32_t lo = 0xffffffffu, hi = 0;
    for (int i = t; i < n; i += kThreads)
      if (member(s.x[i])) {
        const uint32_t k = desc_key(s.x[i]);
        lo = min(lo, k);
        hi = max(hi, k);
      }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if ((t & 31) == 0) {
      atomicMin(&s.key_min, lo);
      atomicMax(&s.key_max, hi);
    }
    cl.sync();
    for (unsigned q = 0; q < cl.num_blocks(); ++q) {
      const Smem* o = cl.map_shared_rank(&s, q);
      lo = min(lo, o->key_min);
      hi = max(hi, o->key_max);
    }
    cl.sync();
    k0 = lo;
    k1 = hi;
    if (k0 == k1) {
      // a run of equal logits: its m-th token in index order
      const u64 w = mass_of(r, from_desc_key(k0)), need = target - (by_count ? (u64)cnt_before : mass_before);
      u64 m = by_count ? need : (need + w - 1) / w;
      if (m > cnt) m = cnt;
      const int per = (n + kThreads - 1) / kThreads, i0 = min(n, t * per), i1 = min(n, i0 + per);
      uint32_t mine = 0;
      for (int i = i0; i < i1; ++i) mine += desc_key(s.x[i]) == k0;
      const uint32_t incl = block_incl_scan<uint32_t>(mine, s.scan32);
      if (t == kThreads - 1) s.eq_count = incl;
      cl.sync();
      uint32_t before = 0;
      for (unsigned q = 0; q < cl.block_rank(); ++q) before += cl.map_shared_rank(&s, q)->eq_count;
      const uint32_t excl = before + incl - mine;
      if (excl < m && m <= (u64)excl + mine) {
        uint32_t left = (uint32_t)m - excl;
        int at = i0;
        for (int i = i0; i < i1; ++i)
          if (desc_key(s.x[i]) == k0 && --left == 0) at = i;
        for (unsigned q = 0; q < cl.num_blocks(); ++q) {
          Smem* o = cl.map_shared_rank(&s, q);
          o->res_idx = base + at;
          o->res_mass = mass_before + m * w;
        }
      }
      cl.sync();
      return;
    }
    const int bits = 32 - __clz(k1 - k0), shift = max(0, bits - 10);
    for (int i = t; i < n; i += kThreads)
      if (member(s.x[i])) bins_add(s, (int)((desc_key(s.x[i]) - k0) >> shift), mass_of(r, s.x[i]));
    uint32_t c, c_to;
    u64 ms, m_to;
    bins_sum(s, cl, c, ms, c_to, m_to);
    const u64 to = by_count ? (u64)cnt_before + c_to : mass_before + m_to, from = to - (by_count ? (u64)c : ms);
    if (from < target && to >= target) {
      s.key_min = k0 + ((uint32_t)t << shift);
      s.hit_cnt_before = cnt_before + c_to - c;
      s.hit_cnt = c;
      s.hit_mass_before = mass_before + m_to - ms;
    }
    __syncthreads();
    k0 = s.key_min;
    k1 = min(k1, k0 + ((1u << shift) - 1u));
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) k_sample(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) unsigned char raw[];
  Smem& s = *reinterpret_cast<Smem*>(raw);
  cg::cluster_group cl = cg::this_cluster();
  const int t = threadIdx.x;
  const long long row = blockIdx.x / cl.num_blocks();
  const int base = (int)cl.block_rank() * p.slice, n = max(0, min(p.slice, p.n - base));
  griddep_launch();
  griddep_wait();

  // ---- the slice and the row's maximum (NaN as -inf, -0 as 0)
  const T* src = (const T*)p.logits + row * p.stride + base;
  float mx = -INFINITY;
  for (int i = t; i < n; i += kThreads) {
    float x = ops::Elem<T>::to_f32(src[i]) + 0.f;
    if (!(x == x)) x = -INFINITY;
    s.x[i] = x;
    mx = fmaxf(mx, x);
  }
  mx = warp_max(mx);
  if ((t & 31) == 0) s.red[t >> 5] = mx;
  bins_clear(s);
  __syncthreads();
  if (t < 32) {
    mx = warp_max(s.red[t]);
    if (t == 0) s.cta_max = mx;
  }
  cl.sync();
  for (unsigned q = 0; q < cl.num_blocks(); ++q) mx = fmaxf(mx, cl.map_shared_rank(&s, q)->cta_max);

  Row r;
  double temp = p.temperature ? (double)p.temperature[row] : p.temperature1;
  int k = p.top_k ? p.top_k[row] : p.top_k1;
  const double top_p = p.top_p ? (double)p.top_p[row] : p.top_p1;
  const double u = p.u[row];
  if (!(temp > 0.0)) {   // greedy
    temp = 1.0;
    k = 1;
  }
  r.mx = mx;
  r.inv_t = 1.0 / temp;
  r.min_p = fmin(1.0, p.min_p ? (double)p.min_p[row] : p.min_p1);
  r.c = (float)(1.4426950408889634 / temp);
  r.cut_log2 = kRangeLog2;
  if (r.min_p > 0.0) r.cut_log2 = fminf(kRangeLog2, (float)-log2(r.min_p) * 1.0001f + 0.001f);
  r.bin_scale = (float)kBins / r.cut_log2;
  if (mx == -INFINITY) {   // nothing to draw from
    cl.sync();
    if (cl.block_rank() == 0 && t == 0) p.out[row] = -1;
    return;
  }

  // ---- bins of the row
  for (int i = t; i < n; i += kThreads) {
    const float x = s.x[i];
    const int b = bin_of(r, x);
    if (b >= 0) {
      const u64 m = mass_of(r, x);
      if (m) bins_add(s, b, m);
    }
  }
  {
    uint32_t c, c_to;
    u64 m, m_to;
    bins_sum(s, cl, c, m, c_to, m_to);
    s.cnt_to[t] = c_to;
    s.mass_to[t] = m_to;
  }
  __syncthreads();
  const uint32_t total = s.cnt_to[kBins - 1];
  u64 kept = s.mass_to[kBins - 1];
  const bool cut_k = k > 0 && (uint32_t)k < total, cut_p = top_p < 1.0;
  const auto reach = [](double share, u64 of) {   // the whole-number mass that `share` of `of` asks for
    if (!(share > 0.0)) return (u64)1;
    const u64 v = (u64)ceil(share * (double)of);
    return v < 1 ? (u64)1 : v > of ? of : v;
  };

  // ---- the head that decides: up to the bin of the k-th token, of the top-p mass, or of the draw
  const u64 target0 = cut_k ? (u64)k : reach(cut_p ? top_p : u, kept);
  {
    const u64 to = cut_k ? (u64)s.cnt_to[t] : s.mass_to[t], from = t ? (cut_k ? (u64)s.cnt_to[t - 1] : s.mass_to[t - 1]) : 0ull;
    if (from < target0 && to >= target0) s.hit_bin = t;
  }
  __syncthreads();
  const int last = s.hit_bin;
  const int head = (int)s.cnt_to[last];
  __syncthreads();
  if (head <= kList) {
    gather(s, cl, base, n, [&](float x) {
      const int b = bin_of(r, x);
      return b >= 0 && b <= last && mass_of(r, x) > 0;
    });
    if (cl.block_rank() == 0) {
      sort_list(s, head);
      u64 m0 = 0, m1 = 0;
      if (2 * t < head) m0 = mass_of(r, from_desc_key((uint32_t)(s.list[2 * t] >> 32)));
      if (2 * t + 1 < head) m1 = mass_of(r, from_desc_key((uint32_t)(s.list[2 * t + 1] >> 32)));
      const u64 to1 = block_incl_scan<u64>(m0 + m1, s.scan64), to0 = to1 - m1, from0 = to0 - m0;
      if (cut_k) {
        if (k - 1 == 2 * t) s.res_mass = to0;
        if (k - 1 == 2 * t + 1) s.res_mass = to1;
        __syncthreads();
        kept = s.res_mass;
        __syncthreads();
      }
      if (cut_p) {
        const u64 g = reach(top_p, kept);
        if (from0 < g && to0 >= g) s.res_mass = to0;
        if (to0 < g && to1 >= g) s.res_mass = to1;
        __syncthreads();
        kept = s.res_mass;
        __syncthreads();
      }
      const u64 g = reach(u, kept);
      if (from0 < g && to0 >= g) p.out[row] = (int32_t)(uint32_t)s.list[2 * t];
      if (to0 < g && to1 >= g) p.out[row] = (int32_t)(uint32_t)s.list[2 * t + 1];
    }
    return;
  }
  if (cut_k) {
    select(s, cl, r, base, n, true, (u64)k);
    kept = s.res_mass;
  }
  if (cut_p) {
    select(s, cl, r, base, n, false, reach(top_p, kept));
    kept = s.res_mass;
  }
  select(s, cl, r, base, n, false, reach(u, kept));
  if (cl.block_rank() == 0 && t == 0) p.out[row] = s.res_idx;
}

}  // namespace sample
}  // namespace vx
