// k_rope_append.cuh — rotary positions on q and k, and k / v appended to a paged cache.
//
// For a token at (rotary) position p, with frequency f_i of pair i:
//   (a, b) -> (a cos(p f_i) - b sin(p f_i), a sin(p f_i) + b cos(p f_i)),
// pairs (2i, 2i+1) (interleaved) or (i, i + rot/2); values past rot_dim pass through.
// q goes to q_out in the cache's type, k and v to slot c % page_size of the page that
// page_table[seq][c / page_size] names, c the position in the cache (p itself unless given apart).
//
// The angle is reduced in 64 bits: p f_i / 2 pi as a double, its nearest whole number taken
// off, and only the remainder (under half a turn) rounded to f32 for sincospif.  In f32 the
// product p f_i of position 100,000 is already off by up to 2^-8 rad.
//
// Bound: HBM (each value read once and written once), launch latency when the batch is
// small.  A CTA takes one token and forms its cosines and sines once for all heads.  One B200: 9711 tokens
// of 32 + 8 + 8 heads of 128 in f16 (239 MB) 41 us = 0.90 of the measured copy rate; one token 2.8 us.
#pragma once
#include "vx_ops.cuh"

namespace vx {
namespace append {

constexpr int kMaxPairs = 256;   // rot_dim <= 512

struct Params {
  const void *q, *k, *v;
  void *q_out, *k_pages, *v_pages;
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head, qo_tok, qo_head;      // element strides
  long long kp_page, kp_head, kp_slot, vp_page, vp_head, vp_slot;
  const int32_t *page_table, *seq_ids, *positions, *rope_positions;
  const float* freq;
  int32_t* status;
  long long table_stride;
  int n_tokens, n_heads, n_kv, head_dim, rot_dim, page_size, n_pages, n_seqs, max_pages;
};

// 8 consecutive values of a row, 16-byte loads and stores.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = ops::Elem<T>::unpack(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  using E = ops::Elem<T>;
  *reinterpret_cast<uint4*>(p) = make_uint4(E::pack(x[0], x[1]), E::pack(x[2], x[3]), E::pack(x[4], x[5]), E::pack(x[6], x[7]));
}

// A unit is 16 values of one head: 16 in a row, or (split pairs) 8 of the first half and the
// 8 of the second half that they turn with.
template <typename TI, typename TC, bool INTERLEAVED>
__global__ void __launch_bounds__(256) k_rope_append(const __grid_constant__ Params p) {
  __shared__ float cs[kMaxPairs], sn[kMaxPairs];
  griddep_launch();
  griddep_wait();
  const int t = blockIdx.x;
  const int pos = p.positions[t], seq = p.seq_ids[t], turn_pos = p.rope_positions ? p.rope_positions[t] : pos;
  if (pos < 0) return;   // padding
  const int lp = pos / p.page_size, slot = pos % p.page_size;
  const bool in_table = seq >= 0 && seq < p.n_seqs && lp < p.max_pages;
  const int page = in_table ? p.page_table[(long long)seq * p.table_stride + lp] : -1;
  if (page < 0 || page >= p.n_pages) {
    if (threadIdx.x == 0) ops::report(p.status, kDevBadIndex);
    return;
  }
  for (int i = threadIdx.x; i < p.rot_dim / 2; i += blockDim.x) {
    const double turns = (double)turn_pos * (double)p.freq[i] * 0.15915494309189533577;   // / (2 pi)
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = c;
    sn[i] = s;
  }
  __syncthreads();
  const int per_head = p.head_dim / 16, rot_units = p.rot_dim / 16;
  const int n_q = p.n_heads * per_head, n_k = p.n_kv * per_head, units = n_q + 2 * n_k;
  for (int u = threadIdx.x; u < units; u += blockDim.x) {
    const TI* src;
    TC* dst;
    int r = u;
    bool turn = true;
    if (u < n_q) {
      const int h = r / per_head;
      r -= h * per_head;
      src = (const TI*)p.q + t * p.q_tok + h * p.q_head;
      dst = (TC*)p.q_out + t * p.qo_tok + h * p.qo_head;
    } else if (u < n_q + n_k) {
      r -= n_q;
      const int h = r / per_head;
      r -= h * per_head;
      src = (const TI*)p.k + t * p.k_tok + h * p.k_head;
      dst = (TC*)p.k_pages + page * p.kp_page + h * p.kp_head + slot * p.kp_slot;
    } else {
      r -= n_q + n_k;
      const int h = r / per_head;
      r -= h * per_head;
      src = (const TI*)p.v + t * p.v_tok + h * p.v_head;
      dst = (TC*)p.v_pages + page * p.vp_page + h * p.vp_head + slot * p.vp_slot;
      turn = false;
    }
    turn = turn && r < rot_units;
    const int d0 = !INTERLEAVED && turn ? 8 * r : 16 * r;
    const int d1 = !INTERLEAVED && turn ? d0 + p.rot_dim / 2 : d0 + 8;
    float a[8], b[8];
    load8<TI>(src + d0, a);
    load8<TI>(src + d1, b);
    if (turn) {
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float c0 = cs[8 * r + i / 2], s0 = sn[8 * r + i / 2], c1 = cs[8 * r + 4 + i / 2], s1 = sn[8 * r + 4 + i / 2];
          const float x = a[i], y = a[i + 1], z = b[i], w = b[i + 1];
          a[i] = x * c0 - y * s0;
          a[i + 1] = x * s0 + y * c0;
          b[i] = z * c1 - w * s1;
          b[i + 1] = z * s1 + w * c1;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float c = cs[8 * r + i], s = sn[8 * r + i], x = a[i], y = b[i];
          a[i] = x * c - y * s;
          b[i] = x * s + y * c;
        }
      }
    }
    store8<TC>(dst + d0, a);
    store8<TC>(dst + d1, b);
  }
}

}  // namespace append
}  // namespace vx
