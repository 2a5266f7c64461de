// k_prefix_attn.cuh — attention over a paged K/V cache for a batch whose sequences share a
// prefix.
//
// Sequence b has n_q[b] query tokens and keys at positions [0, prefix_len + suffix_len[b]): the
// first prefix_len of them sit in pages that every sequence shares, the others in its own.
// Query token i stands at position prefix_len + suffix_len[b] - n_q[b] + i and sees the keys
// up to and including that position:
//   o = sum_p exp(q.k_p * scale - m) v_p / sum_p exp(q.k_p * scale - m),  m = the row's maximum.
// A row that sees no key gives 0.
//
// Softmax splits over ranges of keys: a range leaves (m, l, o) of its own keys, and ranges join
// by o = sum_r e^(m_r - m) o_r / sum_r e^(m_r - m) l_r.  Everything but the operands of the
// matrix products is f32; the weights are rounded to the cache's type for the product with V
// (half a step of 2^-11 / 2^-8 of a weight, as large as the rounding of V itself and averaged
// over the keys), their sum l is not.
#pragma once
#include "vx_ops.cuh"
#include "vx_tcgen05.cuh"

namespace vx {
namespace pattn {

constexpr float kLog2e = 1.4426950408889634f;

struct Pages {
  const void* base;
  long long page, head, slot;   // element strides
};
struct Params {
  const void* q;
  void* out;
  long long q_tok, q_head, o_tok, o_head;
  Pages k, v;
  const int32_t *prefix_pages, *page_table, *suffix_lens, *cu_q;   // cu_q null: one token each
  long long table_stride;
  int32_t* status;
  float *part_o, *part_ml;   // [split][n_tokens * n_heads][D] / [..][2]
  int n_tokens, n_seqs, n_heads, n_kv, group;
  int prefix_len, page_size, n_pages, max_pages;
  float scale_log2;          // scale * log2(e): weights are 2^(s * scale_log2 - m)
  int splits, split0;        // this launch's key ranges are partials [split0, split0 + splits)
  int direct;                // one range in all: write out, no partials
  int own_only;              // skip the prefix keys
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                 uint32_t b1) {
  mma_16816(d, a0, a1, a2, a3, b0, b1);
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
typedef unsigned long long f32x2;   // two f32 in a register pair: one instruction for both
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------- short row tiles
// A CTA takes up to 8 NT query rows of one sequence that share a K/V head (row = query token
// x group + head of the group) and one range of their keys.  Its 4 warps take 16-key blocks
// in turn, each through a ring of its own (cp.async, no block-wide barrier in the loop).
// Scores are formed transposed, S^T = K Q^T (16 keys x 8 rows an MMA), so that 4 query heads
// fill half of an MMA's rows and not a quarter; P^T comes from S^T by an 8x8 register transpose
// and O^T = V^T P^T.
constexpr int kRowWarps = 4;
constexpr int kRowStages = 3;
template <int D>
constexpr int row_smem() {
  return kRowWarps * kRowStages * 2 * 16 * D * 2;
}

// Tile `z` of the grid: its sequence and the tile's number in it (warp-wide, all lanes).
__device__ __forceinline__ bool find_tile(const Params& p, int z, int rows, int lane, int& b, int& i) {
  if (!p.cu_q) {
    const int per = (p.group + rows - 1) / rows;
    b = z / per;
    i = z - b * per;
    return b < p.n_seqs;
  }
  int before = 0;
  for (int b0 = 0; b0 < p.n_seqs; b0 += 32) {
    int n = 0;
    if (b0 + lane < p.n_seqs) n = (max(0, p.cu_q[b0 + lane + 1] - p.cu_q[b0 + lane]) * p.group + rows - 1) / rows;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + incl > z);
    if (hit) {
      const int l = __ffs(hit) - 1;
      b = b0 + l;
      i = z - before - (__shfl_sync(0xffffffffu, incl, l) - __shfl_sync(0xffffffffu, n, l));
      return true;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kRowWarps * 32) k_attn_rows(const __grid_constant__ Params p) {
  using E = ops::Elem<T>;
  constexpr int ROWS = 8 * NT, KK = D / 16, CH = D / 8, TILE = 16 * D * 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kRowWarps][ROWS], s_l[kRowWarps][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.z, kvh = blockIdx.y;
  griddep_launch();
  griddep_wait();
  int b, ti;
  if (!find_tile(p, blockIdx.x, ROWS, lane, b, ti)) return;
  const int tok0 = p.cu_q ? p.cu_q[b] : b;
  const int nq = p.cu_q ? p.cu_q[b + 1] - tok0 : 1;
  const int cap = p.max_pages * p.page_size, given = p.suffix_lens[b];
  const int own = max(0, min(given, cap));
  if (given > cap && threadIdx.x == 0) ops::report(p.status, kDevBadIndex);   // keys that the page table does not hold
  const int n_rows = min(ROWS, nq * p.group - ti * ROWS);
  if (tok0 < 0 || n_rows <= 0 || tok0 + nq > p.n_tokens) {   // offsets that the batch does not hold
    if (threadIdx.x == 0) ops::report(p.status, kDevBadIndex);
    return;
  }
  const int first_lim = p.prefix_len + own - nq + 1;   // keys that query token 0 sees
  // 16-key blocks of this tile: the prefix's, then the sequence's own
  const int last_lim = max(0, first_lim + (ti * ROWS + n_rows - 1) / p.group);
  const int pre_blocks = (min(p.prefix_len, last_lim) + 15) / 16;
  const int blk0 = p.own_only ? pre_blocks : 0;
  const int n_blocks = pre_blocks + (max(0, last_lim - p.prefix_len) + 15) / 16 - blk0;
  const int per = max(((n_blocks + p.splits - 1) / p.splits + kRowWarps - 1) / kRowWarps * kRowWarps, 4 * kRowWarps);
  const int begin = blk0 + split * per, end = min(blk0 + n_blocks, begin + per);

  // query fragments (B operand): lane holds row lane / 4, values 2 (lane % 4) + {0, 1, 8, 9} of each 16
  uint32_t qf[NT][KK][2];
  int lim[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = ti * ROWS + n * 8 + (lane >> 2);
    const bool live = n * 8 + (lane >> 2) < n_rows;
    const int j = r / p.group, g = r - j * p.group;
    const T* src = (const T*)p.q + (long long)(tok0 + j) * p.q_tok + (long long)(kvh * p.group + g) * p.q_head + 2 * (lane & 3);
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      qf[n][k][0] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * k) : 0u;
      qf[n][k][1] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8) : 0u;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = n * 8 + 2 * (lane & 3) + e;
      lim[n][e] = c < n_rows ? first_lim + (ti * ROWS + c) / p.group : 0;
    }
  }

  const uint32_t ring = smem_u32(smem) + warp * (kRowStages * 2 * TILE);
  const T* kb = (const T*)p.k.base + kvh * p.k.head;
  const T* vb = (const T*)p.v.base + kvh * p.v.head;
  auto issue = [&](int blk, int st) {
    if (blk < end) {
      const bool pre = blk < pre_blocks;
      const int key = 16 * (pre ? blk : blk - pre_blocks);
      const int n = (pre ? p.prefix_len : own) - key;   // keys of the block that exist
      const int lp = key / p.page_size;
      int page = -1;
      if (pre) page = p.prefix_pages[lp];
      else if (lp < p.max_pages) page = p.page_table[(long long)b * p.table_stride + lp];
      const bool ok = page >= 0 && page < p.n_pages;
      if (!ok) {
        ops::report(p.status, kDevBadIndex);
        page = 0;
      }
      const int slot = key % p.page_size;
      const T* ks = kb + page * p.k.page + slot * p.k.slot;
      const T* vs = vb + page * p.v.page + slot * p.v.slot;
      const uint32_t dst = ring + st * 2 * TILE;
#pragma unroll
      for (int c = 0; c < 16 * CH / 32; ++c) {
        const int x = c * 32 + lane, row = x / CH, col = x % CH;
        const uint32_t at = dst + row * (D * 2) + ((col ^ (row & 7)) << 4);
        const bool live = ok && row < n;
        cp16(at, live ? ks + row * p.k.slot + col * 8 : ks, live);
        cp16(at + TILE, live ? vs + row * p.v.slot + col * 8 : vs, live);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  float m[NT][2], l[NT][2], o[NT][KK][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.f;
#pragma unroll
    for (int d = 0; d < KK; ++d) o[n][d][0] = o[n][d][1] = o[n][d][2] = o[n][d][3] = 0.f;
  }
#pragma unroll
  for (int s = 0; s < kRowStages - 1; ++s) issue(begin + warp + s * kRowWarps, s);
  int st = 0;
  for (int blk = begin + warp; blk < end; blk += kRowWarps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRowStages - 2) : "memory");
    __syncwarp();
    issue(blk + (kRowStages - 1) * kRowWarps, st == 0 ? kRowStages - 1 : st - 1);
    const uint32_t kt = ring + st * 2 * TILE, vt = kt + TILE;
    st = st + 1 == kRowStages ? 0 : st + 1;
    const int mat = lane >> 3, r8 = lane & 7;
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      const int row = (mat & 1) * 8 + r8, col = 2 * k + (mat >> 1);
      uint32_t a0, a1, a2, a3;
      ldmatrix_x4(a0, a1, a2, a3, kt + row * (D * 2) + ((col ^ (row & 7)) << 4));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma16816<T>(s[n], a0, a1, a2, a3, qf[n][k][0], qf[n][k][1]);
    }
    // lane holds keys lane / 4 and + 8, rows 2 (lane % 4) and + 1 of each tile of 8
    const bool pre = blk < pre_blocks;
    const int key = 16 * (pre ? blk : blk - pre_blocks) + (lane >> 2);
    const int left = (pre ? p.prefix_len : own) - key;      // > 0: the key exists
    const int pos = (pre ? 0 : p.prefix_len) + key;
    uint32_t pb[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[4], corr[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        x[e] = left > 0 && pos < lim[n][e] ? s[n][e] * p.scale_log2 : -INFINITY;
        x[e + 2] = left > 8 && pos + 8 < lim[n][e] ? s[n][e + 2] * p.scale_log2 : -INFINITY;
        float mx = fmaxf(x[e], x[e + 2]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float m_new = fmaxf(m[n][e], mx);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        corr[e] = ex2(m[n][e] - m_use);
        m[n][e] = m_new;
        x[e] = ex2(x[e] - m_use);
        x[e + 2] = ex2(x[e + 2] - m_use);
        l[n][e] = l[n][e] * corr[e] + x[e] + x[e + 2];
      }
      if (!__all_sync(0xffffffffu, corr[0] == 1.f && corr[1] == 1.f)) {
#pragma unroll
        for (int d = 0; d < KK; ++d) {
          o[n][d][0] *= corr[0];
          o[n][d][1] *= corr[1];
          o[n][d][2] *= corr[0];
          o[n][d][3] *= corr[1];
        }
      }
      pb[n][0] = movmatrix_trans(E::pack(x[0], x[1]));
      pb[n][1] = movmatrix_trans(E::pack(x[2], x[3]));
    }
#pragma unroll
    for (int d = 0; d < KK; ++d) {
      const int row = (mat >> 1) * 8 + r8, col = 2 * d + (mat & 1);
      uint32_t a0, a1, a2, a3;
      ldmatrix_x4_trans(a0, a1, a2, a3, vt + row * (D * 2) + ((col ^ (row & 7)) << 4));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma16816<T>(o[n][d], a0, a1, a2, a3, pb[n][0], pb[n][1]);
    }
    __syncwarp();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // ---- the 4 warps' states join in shared memory
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
      if (lane < 4) {
        s_m[warp][n * 8 + 2 * lane + e] = m[n][e];
        s_l[warp][n * 8 + 2 * lane + e] = l[n][e];
      }
    }
  __syncthreads();   // the rings are free
  float* so = reinterpret_cast<float*>(smem);   // [warp][ROWS][D]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int d = 0; d < KK; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        so[(warp * ROWS + n * 8 + 2 * (lane & 3) + (e & 1)) * D + d * 16 + (lane >> 2) + (e >> 1) * 8] = o[n][d][e];
  __syncthreads();
  for (int x = threadIdx.x; x < n_rows * (D / 4); x += kRowWarps * 32) {
    const int r = x / (D / 4), d = (x - r * (D / 4)) * 4;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) M = fmaxf(M, s_m[w][r]);
    const float m_use = M == -INFINITY ? 0.f : M;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const float f = ex2(s_m[w][r] - m_use);
      const float4 v = *reinterpret_cast<const float4*>(so + (w * ROWS + r) * D + d);
      L += s_l[w][r] * f;
      acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
    }
    const int lr = ti * ROWS + r, j = lr / p.group, g = lr - j * p.group;
    const long long tok = tok0 + j;
    const int head = kvh * p.group + g;
    if (p.direct) {
      const float inv = L > 0.f ? 1.f / L : 0.f;
      *reinterpret_cast<uint2*>((T*)p.out + tok * p.o_tok + head * p.o_head + d) =
          make_uint2(E::pack(acc.x * inv, acc.y * inv), E::pack(acc.z * inv, acc.w * inv));
    } else {
      const long long row = (long long)(p.split0 + split) * p.n_tokens * p.n_heads + tok * p.n_heads + head;
      if (M != -INFINITY) *reinterpret_cast<float4*>(p.part_o + row * D + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * row) = make_float2(M, L);
    }
  }
}

// ---------------------------------------------------------------- tiles of 128 rows
// One CTA takes up to 256 query rows of one K/V head (two tiles of 128) against one range of
// 128-key tiles, on the tensor cores: S = Q K^T and O += P V as tcgen05.mma with f32 accumulators
// in TMEM, P written back into TMEM over S as the A operand of the second product.
//   OWN = false: the rows of all sequences against the shared prefix, which is so read and
//                multiplied once for the whole batch;
//   OWN = true:  the rows of one sequence against its prefix and own keys, causally.
// Warps 0-3 and 4-7 each do the softmax of one tile, a thread a row (no shuffles); warp 8 brings
// the pages in by TMA; one thread of warp 9 issues the products.  While one tile's softmax runs,
// the other tile's products do.  The reference exponent of a row only moves when its maximum grows
// by more than 2^8 (weights stay below 2^8, far inside f16's and f32's range), so that O in TMEM is
// hardly ever rescaled.
//
// Bound: for a wide batch the tensor cores and the exponentials (a 128 x 128 tile needs 1024 cycles
// of products at head_dim 128 and 1024 of ex2), for a narrow one the reading of K and V.
constexpr int kTile = 128;
constexpr int kTileThreads = 320;
template <int D>
struct TileCfg {
  static constexpr int kSlot = kTile * D * 2;                       // a K or V tile, or a tile of Q
  static constexpr int kSlots = D == 128 ? 5 : 8;
  static constexpr size_t kSmem = (size_t)(2 + kSlots) * kSlot + 1024 + 256;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
// One row from shared to global memory; returns when the shared memory has been read.
__device__ __forceinline__ void bulk_s2g(void* dst, uint32_t src, int bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <typename T, int D, bool OWN>
__global__ void __launch_bounds__(kTileThreads, 1) k_attn_tiles(const __grid_constant__ CUtensorMap kmap,
                                                                const __grid_constant__ CUtensorMap vmap,
                                                                const __grid_constant__ Params p) {
  using E = ops::Elem<T>;
  using C = TileCfg<D>;
  constexpr uint32_t kIdescQK = (1u << 4) | (E::kIdescType << 7) | (E::kIdescType << 10) | ((kTile >> 3) << 17) | ((kTile >> 4) << 24);
  constexpr uint32_t kIdescPV = (1u << 4) | (E::kIdescType << 7) | (E::kIdescType << 10) | (1u << 16) | ((D >> 3) << 17) | ((kTile >> 4) << 24);
  constexpr uint32_t kHalf = kTile * 128;   // bytes of 64 columns of a tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  uint8_t* ring = smem + 2 * C::kSlot;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + C::kSlots * C::kSlot);
  uint64_t* empty = full + C::kSlots;
  uint64_t* q_full = empty + C::kSlots;
  uint64_t* s_full = q_full + 1;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* tail = o_done + 1;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  volatile int* abort = &s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y, split = blockIdx.z;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 256);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kTile);
    }
    mbar_init(o_done, 1);
    mbar_init(tail, 1);
    fence_mbar_init();
    s_abort = 0;
    prefetch_tmap(&kmap);
    prefetch_tmap(&vmap);
  }
  griddep_launch();
  griddep_wait();

  // ---- the rows and keys of this CTA (the same in every thread)
  int b = 0, ti = blockIdx.x;
  int tok0 = 0, n_rows, own = 0, first_lim = p.prefix_len, last_lim = p.prefix_len;
  if (OWN) {
    if (!find_tile(p, blockIdx.x, 2 * kTile, lane, b, ti)) return;
    tok0 = p.cu_q[b];
    const int nq = p.cu_q[b + 1] - tok0;
    const int cap = p.max_pages * p.page_size, given = p.suffix_lens[b];
    own = max(0, min(given, cap));
    n_rows = min(2 * kTile, nq * p.group - ti * 2 * kTile);
    if ((given > cap || tok0 < 0 || n_rows <= 0 || tok0 + nq > p.n_tokens) && threadIdx.x == 0) ops::report(p.status, kDevBadIndex);
    if (tok0 < 0 || n_rows <= 0 || tok0 + nq > p.n_tokens) return;
    first_lim = p.prefix_len + own - nq + 1;
    last_lim = max(0, first_lim + (ti * 2 * kTile + n_rows - 1) / p.group);
  } else {
    n_rows = min((long long)2 * kTile, (long long)p.n_tokens * p.group - (long long)ti * 2 * kTile);
  }
  const int row0 = ti * 2 * kTile;                       // first row: token tok0 + row / group, head row % group
  const int n_pre = (min(p.prefix_len, last_lim) + kTile - 1) / kTile;
  const int n_all = n_pre + (max(0, last_lim - p.prefix_len) + kTile - 1) / kTile;
  const int per = (n_all + p.splits - 1) / p.splits;
  const int t0 = split * per, n = max(0, min(n_all, t0 + per) - t0);
  const int n_tiles = n_rows > kTile ? 2 : 1;

  if (warp == 9) tc::tmem_alloc(&s_tmem, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t t_s[2] = {tmem, tmem + 128}, t_o[2] = {tmem + 256, tmem + 384};

  if (warp == 8) {
    // ---- pages into the ring: K of tile 0, V of tile 0, K of tile 1, ...
    const int box = min(p.page_size, kTile);
    int issued = 0, tails = 0;
    bool ok = true;
    for (int it = 0; ok && it < 2 * n; ++it) {
      const int s = it % C::kSlots, t = t0 + (it >> 1);
      const bool is_v = it & 1;
      if (it >= C::kSlots) {
        int go = lane == 0 ? ops::wait_phase(&empty[s], (uint32_t)(it / C::kSlots - 1) & 1u, abort, p.status, kDevTimeoutEmpty) : 0;
        ok = __shfl_sync(0xffffffffu, go, 0);
        if (!ok) break;
      }
      const bool pre = t < n_pre;
      const int key = kTile * (pre ? t : t - n_pre), valid = min(kTile, (pre ? p.prefix_len : own) - key);
      const int boxes = (valid + box - 1) / box;
      // a tile that ends early: V's missing rows are zeroed (0 x NaN), K's scores are masked
      const bool zero = is_v && valid < kTile;
      uint64_t* bar = zero ? tail : &full[s];
      if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(boxes * box * D * 2));
      __syncwarp();
      const uint32_t dst = smem_u32(ring + s * C::kSlot);
      if (lane < boxes) {
        const int at = key + lane * box, lp = at / p.page_size;
        int page = -1;
        if (pre) page = p.prefix_pages[lp];
        else if (lp < p.max_pages) page = p.page_table[(long long)b * p.table_stride + lp];
        if (page < 0 || page >= p.n_pages) {
          ops::report(p.status, kDevBadIndex);
          page = p.n_pages;   // past the map's end: reads as zero
        }
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
          tma_load_4d(dst + h * kHalf + lane * box * 128, is_v ? &vmap : &kmap, h * 64, at % p.page_size, kvh, page, bar);
      }
      issued = it + 1;
      if (zero) {
        __syncwarp();
        ops::wait_landed(tail, tails & 1, p.status);
        ++tails;
        for (int x = lane; x < (kTile - valid) * 8 * (D / 64); x += 32) {
          const int h = x / ((kTile - valid) * 8), c = x % ((kTile - valid) * 8);
          *reinterpret_cast<uint4*>(ring + s * C::kSlot + h * kHalf + valid * 128 + c * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[s]);
      }
      __syncwarp();
    }
    // after a failure nobody may be waiting for the last copies: they land before the CTA ends
    if (!ok || *abort)
      for (int it = max(0, issued - C::kSlots); it < issued; ++it) ops::wait_landed(&full[it % C::kSlots], (uint32_t)(it / C::kSlots) & 1u, p.status);
  } else if (warp == 9) {
    if (lane == 0 && n > 0) {
      const uint32_t q_s = smem_u32(smem), r_s = smem_u32(ring);
      const auto qk = [&](int i, int slot) {
        const uint32_t q = q_s + i * C::kSlot, k = r_s + slot * C::kSlot;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * kHalf + (kk & 3) * 32;
          tc::tc_mma(t_s[i], tc::sw128_desc(q + off), tc::sw128_desc(k + off), kIdescQK, kk != 0);
        }
        tc::tc_commit(&s_full[i]);
      };
      bool ok = ops::wait_phase(q_full, 0, abort, p.status, kDevTimeoutFull) && ops::wait_phase(&full[0], 0, abort, p.status, kDevTimeoutFull);
      if (ok) {
        tc::tc_fence_after();
        for (int i = 0; i < n_tiles; ++i) qk(i, 0);
        tc::tc_commit(&empty[0]);
      }
      for (int j = 0; ok && j < n; ++j) {
        const int iv = 2 * j + 1, ik = iv + 1, sv = iv % C::kSlots, sk = ik % C::kSlots;
        for (int i = 0; ok && i < n_tiles; ++i) {
          ok = ops::wait_phase(&p_full[i], (uint32_t)j & 1u, abort, p.status, kDevTimeoutRed) &&
               (i || ops::wait_phase(&full[sv], (uint32_t)(iv / C::kSlots) & 1u, abort, p.status, kDevTimeoutFull));
          if (!ok) break;
          tc::tc_fence_after();
          const uint32_t v = r_s + sv * C::kSlot;
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk)
            tc::tc_mma_ta(t_o[i], t_s[i] + kk * 8, tc::sw128_mn_desc(v + kk * 2048, kHalf), kIdescPV, (j | kk) != 0);
          if (i == n_tiles - 1) tc::tc_commit(&empty[sv]);
          if (j + 1 < n) {
            if (i == 0) {
              ok = ops::wait_phase(&full[sk], (uint32_t)(ik / C::kSlots) & 1u, abort, p.status, kDevTimeoutFull);
              if (!ok) break;
              tc::tc_fence_after();
            }
            qk(i, sk);
            if (i == n_tiles - 1) tc::tc_commit(&empty[sk]);
          }
        }
      }
      tc::tc_commit(o_done);
      if (!ok) ops::wait_landed(o_done, 0, p.status);   // products already issued end before TMEM is freed
    }
  } else if (warp < 8) {
    // ---- Q into shared memory (128-byte swizzle), then the softmax of one tile
    const int wg = warp >> 2, row = threadIdx.x & (kTile - 1);
    {
      constexpr int CH = D / 8, STEP = kTile / CH;   // 16-byte chunks of a row; this thread's rows are STEP apart
      const int c = row % CH;
      int g = (row0 + wg * kTile + row / CH) % p.group;
      long long tok = tok0 + (row0 + wg * kTile + row / CH) / p.group;
      const int step_g = STEP % p.group, step_tok = STEP / p.group;
      const T* src = (const T*)p.q + (long long)kvh * p.group * p.q_head + c * 8;
      uint4 v[CH];
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const bool in = wg * kTile + row / CH + k * STEP < n_rows;
        v[k] = in ? *reinterpret_cast<const uint4*>(src + tok * p.q_tok + g * p.q_head) : make_uint4(0, 0, 0, 0);
        g += step_g;
        tok += step_tok;
        if (g >= p.group) {
          g -= p.group;
          ++tok;
        }
      }
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const int r = row / CH + k * STEP;
        *reinterpret_cast<uint4*>(smem + wg * C::kSlot + (c >> 3) * kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[k];
      }
    }
    fence_async_smem();
    mbar_arrive(q_full);

    if (wg < n_tiles) {
      const int lr = wg * kTile + row;   // this thread's row
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const int lim = OWN ? first_lim + (row0 + min(lr, n_rows - 1)) / p.group : p.prefix_len;   // keys that the row sees
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        ok = ops::wait_phase(&s_full[wg], (uint32_t)j & 1u, abort, p.status, kDevTimeoutAcc);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        float s[kTile];
        tc::tmem_ld128(t_s[wg] + lanes, s);
        const int t = t0 + j;
        const bool pre = t < n_pre;
        const int key = kTile * (pre ? t : t - n_pre);
        const int see = min((pre ? p.prefix_len : own), lim - (pre ? 0 : p.prefix_len)) - key;   // keys of this tile that count
        if (__any_sync(0xffffffffu, see < kTile)) {
#pragma unroll
          for (int i = 0; i < kTile; ++i)
            if (i >= see) s[i] = -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i + 8 <= kTile; i += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], s[i + 2 * k], s[i + 2 * k + 1]);
        mx[0] = max3(mx[0], s[kTile - 4], s[kTile - 3]);
        mx[1] = max3(mx[1], s[kTile - 2], s[kTile - 1]);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
        if (j == 0) {
          m = top;
        } else if (__any_sync(0xffffffffu, top > m + 8.f)) {
          const float m_new = fmaxf(m, top), f = ex2(m == m_new ? 0.f : m - m_new);
          l *= f;
          m = m_new;
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            float o[16];
            uint32_t u[16];
            tc::tmem_ld16(t_o[wg] + lanes + c, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(o[i] * f);
            tc::tmem_st16(t_o[wg] + lanes + c, u);
          }
        }
        const float m_use = m == -INFINITY ? 0.f : m;
        const f32x2 scale2 = pack2(p.scale_log2, p.scale_log2), off2 = pack2(-m_use, -m_use);
        f32x2 sum[2] = {pack2(l, 0.f), pack2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < kTile; c += 64) {
          uint32_t u[32];
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            float x, y;
            unpack2(fma2(pack2(s[c + i], s[c + i + 1]), scale2, off2), x, y);
            x = ex2(x);
            y = ex2(y);
            sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pack2(x, y));
            u[i >> 1] = E::pack(x, y);
          }
          tc::tmem_st32(t_s[wg] + lanes + c / 2, u);
        }
        {
          float x, y;
          unpack2(add2(sum[0], sum[1]), x, y);
          l = x + y;
        }
        tc::tmem_st_wait();
        tc::tc_fence_before();
        mbar_arrive(&p_full[wg]);
      }
      if (ok && n > 0) ok = __all_sync(0xffffffffu, ops::wait_phase(o_done, 0, abort, p.status, kDevTimeoutAcc));
      if (ok) {
        tc::tc_fence_after();
        const bool live = lr < n_rows;
        const long long tok = tok0 + (row0 + lr) / p.group;
        const int head = kvh * p.group + (row0 + lr) % p.group;
        const long long at = (long long)(p.split0 + split) * p.n_tokens * p.n_heads + tok * p.n_heads + head;
        const float inv = l > 0.f ? 1.f / l : 0.f;
        if (live && !p.direct) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(m, l);
        // rows to memory by one bulk copy each, staged in the ring (free now); 16 bytes of padding
        // keep the threads' rows on different banks
        const int row_bytes = p.direct ? D * 2 : D * 4;
        uint8_t* stage = ring + (size_t)lr * (row_bytes + 16);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          if (n > 0) {
            tc::tmem_ld32(t_o[wg] + lanes + c, o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
          }
          if (p.direct) {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4*>(stage + (c + i) * 2) =
                  make_uint4(E::pack(o[i] * inv, o[i + 1] * inv), E::pack(o[i + 2] * inv, o[i + 3] * inv),
                             E::pack(o[i + 4] * inv, o[i + 5] * inv), E::pack(o[i + 6] * inv, o[i + 7] * inv));
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(stage + (c + i) * 4) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        fence_async_smem();
        if (live && (p.direct || m != -INFINITY)) {
          void* dst = p.direct ? (void*)((T*)p.out + tok * p.o_tok + (long long)head * p.o_head) : (void*)(p.part_o + at * D);
          bulk_s2g(dst, smem_u32(stage), row_bytes);
        }
      }
    }
  }
  __syncwarp();
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- joining key ranges
// One warp per row (token, head): weights of the ranges from their (m, l), then the weighted
// sum of their o.  Ranges are added in order, so the result does not depend on timing.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_attn_join(const __grid_constant__ Params p) {
  using E = ops::Elem<T>;
  constexpr int V = D / 32;   // values a lane
  griddep_launch();
  griddep_wait();
  const long long rows = (long long)p.n_tokens * p.n_heads;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  float M = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) M = fmaxf(M, __ldcg(p.part_ml + 2 * (s * rows + row)));
  M = warp_max(M);
  const float m_use = M == -INFINITY ? 0.f : M;
  float L = 0.f, acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  for (int s0 = 0; s0 < p.splits; s0 += 32) {
    float f = 0.f;
    if (s0 + lane < p.splits) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + 2 * ((s0 + lane) * rows + row)));
      f = ml.x == -INFINITY ? 0.f : ex2(ml.x - m_use);
      L += ml.y * f;
    }
    const int n = min(32, p.splits - s0);
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float w = __shfl_sync(0xffffffffu, f, s);
      if (w == 0.f) continue;   // a range without keys left its o unwritten
      const float* o = p.part_o + ((s0 + s) * rows + row) * D + lane * V;
      if constexpr (V == 4) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(o));
        acc[0] += v.x * w; acc[1] += v.y * w; acc[2] += v.z * w; acc[3] += v.w * w;
      } else {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(o));
        acc[0] += v.x * w; acc[1] += v.y * w;
      }
    }
  }
  L = warp_sum(L);
  const float inv = L > 0.f ? 1.f / L : 0.f;
  const long long tok = row / p.n_heads;
  if (p.cu_q && (tok < p.cu_q[0] || tok >= p.cu_q[p.n_seqs])) return;   // no sequence's token
  const int head = (int)(row - tok * p.n_heads);
  T* dst = (T*)p.out + tok * p.o_tok + head * p.o_head + lane * V;
  if constexpr (V == 4) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(E::pack(acc[0] * inv, acc[1] * inv), E::pack(acc[2] * inv, acc[3] * inv));
  } else {
    *reinterpret_cast<uint32_t*>(dst) = E::pack(acc[0] * inv, acc[1] * inv);
  }
}

}  // namespace pattn
}  // namespace vx
