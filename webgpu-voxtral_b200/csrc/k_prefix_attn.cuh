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
// Two kernels and a join.  The tile kernel multiplies 128 query rows at a time on the tensor cores; with one
// query token a sequence it takes the rows of all sequences through the shared prefix, which is
// so read and multiplied once for the batch.  The row kernel takes up to 32 rows of one sequence
// through their keys at the rate of memory.  Which of them run, and on which keys, is plan_attention's choice
// (vx_ops.cu).  One B200, in a captured graph: 64 sequences of 32 heads on 8 K/V heads of 128 past 32768 shared
// keys 63 us (the prefix alone 49 us: 700 TFLOP/s, 134 MB read once), past 617 shared and 1 to 1500 own
// keys 25 us.
//
// Softmax splits over ranges of keys: a range leaves (m, l, o) of its own keys, and ranges join
// by o = sum_r e^(m_r - m) o_r / sum_r e^(m_r - m) l_r (online softmax, Milakov and Gimelshein 2018).  Everything but the operands of the
// matrix products is f32; the weights are rounded to the cache's type for the product with V
// (half a step of 2^-11 / 2^-8 of a weight, as large as the rounding of V itself and averaged
// over the keys), their sum l is not.  f16 weights end at 2^-25, which in a long tail adds up: 10^6 equal
// keys at 2^-26 of one strong key are 1.5 % of its result.  So a row's weights are taken relative to 2^-7
// (tile kernel, whose reference may lag by 2^8) or 2^-15 (row kernel) of its largest, which uses f16's
// range to 2^15: a weight is then off by 2^-32 of the largest at most.  The factor cancels against l.
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
  float* tile_o;             // partials of the tile kernel: [split][n_tokens * n_heads][D]
  float2* tile_ml;
  float* row_o;              // partials of the row kernel: [part][8 NT][D]
  float2* row_ml;
  int2* row_parts;           // [n_tokens * n_heads]: first and last partial row; last -1: none, -2: out is written
  int2* span;                // with cu_q and a join: the tokens [x, y) of the sequences that are held
  int n_tokens, n_seqs, n_heads, n_kv, group;
  int prefix_len, page_size, n_pages, max_pages;
  float scale_log2;          // scale * log2(e): weights are 2^(s * scale_log2 - m)
  int tile_parts;            // key ranges of the tile kernel (0: it does not run)
  int rows_run;              // whether the row kernel runs, and the rows of its tiles
  int own_only;              // the prefix is the shared tile kernel's: the row kernel and the one of whole sequences leave it out
  int part0;                 // this tile launch's first partial
  int parts;                 // and its key ranges
  int min_blocks;            // blocks a warp of the row kernel takes at least
  int direct;                // the tile kernel alone, with one key range: it writes out
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
// Powers of two by which a row's reference lies below its largest score, where its weights may grow to 2^room.
template <typename T>
constexpr float below_top(int room) {
  return sizeof(T) == 2 && ops::Elem<T>::kIdescType == 0 ? 15.f - room : 0.f;   // bf16 has f32's range
}
// Barrier of `threads` threads that tells all of them whether one came with `v`.
__device__ __forceinline__ bool named_bar_or(int id, int threads, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbarrier.cta.red.or.pred p, %2, %3, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Offsets begin at 0 or later, never go down and end within the batch: sequences then share no row, and
// have no more row tiles than the plan has room for.  The sequence whose beginning or end breaks that
// is refused with all after it; those in front of it are held.
__device__ __forceinline__ bool out_of_order(const Params& p, int b) {
  const int from = p.cu_q[b], to = p.cu_q[b + 1];
  return from < 0 || to < from || to > p.n_tokens;
}
// One thread says how many sequences are held: to the caller's status, and to the join.  (Every launch of
// a call finds and writes the same.)
__device__ __forceinline__ void tell_held(const Params& p, int n_seqs) {
  if (n_seqs < p.n_seqs) ops::report(p.status, kDevBadIndex);
  if (p.span) *p.span = make_int2(p.cu_q[0], p.cu_q[n_seqs]);
}
// Sequences that are held.  All threads of the block together: one pass over the offsets and, where they
// are in order, one barrier.
__device__ __forceinline__ int held_seqs(const Params& p) {
  __shared__ int s_first;
  if (!p.cu_q) return p.n_seqs;
  int first = p.n_seqs;
  for (int b = threadIdx.x; b < p.n_seqs && first == p.n_seqs; b += blockDim.x)
    if (out_of_order(p, b)) first = b;
  if (threadIdx.x == 0) s_first = p.n_seqs;
  if (__syncthreads_or(first < p.n_seqs)) {
    atomicMin(&s_first, first);
    __syncthreads();
    first = s_first;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) tell_held(p, first);
  return first;
}

// ---------------------------------------------------------------- short row tiles
// Up to 8 NT query rows of one sequence that share a K/V head are an item; its work is the 16-key
// blocks of its sequence.  All blocks of all items stand in one line (sequence, row tile, head, block)
// that the warps of the grid share out evenly, whatever the lengths are: a warp takes `per` blocks in a
// row, through a ring of its own (cp.async, no block-wide barrier in the loop), and leaves one partial
// for each item that it meets.  Warp w's part of item i is partial w + i: no two parts share a
// number, since from one part to the next w or i goes up, and the parts of an item follow one another.
// Scores are formed transposed, S^T = K Q^T (16 keys x 8 rows an MMA), so that 4 query heads
// fill half of an MMA's rows and not a quarter; P^T comes from S^T by an 8x8 register transpose
// and O^T = V^T P^T.
//
// Bound: the reading of K and V (HBM, or L2 where sequences read the same prefix).
constexpr int kRowStages = 3;
constexpr int kItemCost = 1;
// Warps of a CTA, one CTA an SM: as many as shared memory holds rings for (registers allow them too).
constexpr int row_warps(int d, int nt) {
  return d == 128 ? (nt == 1 ? 7 : nt == 2 ? 6 : 4) : (nt == 1 ? 14 : nt == 2 ? 12 : 8);
}
template <int D, int NT>
constexpr int row_warp_smem() {   // K and V of the stages, the query rows of as many items, what each stage holds
  return kRowStages * (2 * 16 * D * 2 + 8 * NT * D * 2 + 64);
}
template <int D, int NT>
constexpr int row_smem() {
  return row_warps(D, NT) * row_warp_smem<D, NT>();
}

// A sequence as the row kernel sees it (n_seqs: those of held_seqs).
struct Seq {
  int tok0, nq, own, tiles, blocks;   // query tokens, own keys, row tiles, 16-key blocks (prefix and own)
  // An item counts kItemCost blocks more than it has: what its start (q, page numbers) and its end (a
  // partial) take.  Otherwise the warps whose share is many short sequences are the last to be done.
  __device__ __forceinline__ int item_units() const { return blocks ? blocks + kItemCost : 0; }
  __device__ __forceinline__ long long units(int n_kv) const { return (long long)tiles * n_kv * item_units(); }
};
__device__ __forceinline__ Seq sequence(const Params& p, int n_seqs, int b, int rows) {
  Seq q{0, 0, 0, 0, 0};
  if (b >= n_seqs) return q;
  q.tok0 = p.cu_q ? p.cu_q[b] : b;
  q.nq = p.cu_q ? p.cu_q[b + 1] - q.tok0 : 1;
  const int cap = p.max_pages * p.page_size, given = p.suffix_lens[b];
  q.own = max(0, min(given, cap));
  if (given > cap) ops::report(p.status, kDevBadIndex);       // keys that the page table does not hold
  q.tiles = (q.nq * p.group + rows - 1) / rows;
  q.blocks = (p.own_only ? 0 : (p.prefix_len + 15) / 16) + (q.own + 15) / 16;
  return q;
}

// What a stage of the ring holds.
struct Stage {
  int keys, pos;            // keys of the block that exist, position of its first
  int flags;                // 1: first block of the warp's part, 2: its last, 4: the item's first, 8: the item's last
  int tok0, first_lim;      // the sequence's first query token, and the keys that it sees
  int row0, n_rows, kvh;    // the item
  int item, q_slot;
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(row_warps(D, NT) * 32, 1) k_attn_rows(const __grid_constant__ Params p) {
  using E = ops::Elem<T>;
  constexpr int ROWS = 8 * NT, KK = D / 16, CH = D / 8, TILE = 16 * D * 2, kRowWarps = row_warps(D, NT), RUN = kRowWarps * 32;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long s_sum[kRowWarps], s_start;
  __shared__ int s_items[kRowWarps], s_start_items, s_start_seq;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_launch();
  // After the tile kernel, of which nothing is read here, this kernel starts on the SMs that it leaves
  // free: the tile kernel lets it go only once what came before both is done.  It ends after it.
  if (!p.tile_parts) griddep_wait();

  // ---- the line: its length, and the run of sequences in which this CTA's part begins
  const int n_seqs = held_seqs(p), n_chunks = (n_seqs + RUN - 1) / RUN;
  long long total = 0;
  for (int c = 0; c < n_chunks; ++c) {
    const int b = c * RUN + threadIdx.x;
    const Seq q = sequence(p, n_seqs, b, ROWS);
    if (q.tiles && !q.blocks && b % (int)gridDim.x == (int)blockIdx.x)   // no keys: no part of any warp
      for (long long r = (long long)q.tok0 * p.n_heads; r < (long long)(q.tok0 + q.nq) * p.n_heads; ++r) p.row_parts[r] = make_int2(0, -1);
    long long u = q.units(p.n_kv);
    for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
    if (lane == 0) s_sum[warp] = u;
    __syncthreads();
    for (int w = 0; w < kRowWarps; ++w) total += s_sum[w];
    __syncthreads();
  }
  const long long warps = (long long)gridDim.x * kRowWarps;
  const long long per = max((total + warps - 1) / warps, (long long)p.min_blocks);
  const long long cta_first = (long long)blockIdx.x * kRowWarps * per;
  if (cta_first >= total) {
    if (p.tile_parts) griddep_wait();
    return;
  }
  if (n_chunks > 1) {
    long long before = 0;
    int items = 0;
    for (int c = 0; c < n_chunks; ++c) {
      const Seq q = sequence(p, n_seqs, c * RUN + threadIdx.x, ROWS);
      long long u = q.units(p.n_kv);
      int it = q.tiles * p.n_kv;
      for (int o = 16; o > 0; o >>= 1) {
        u += __shfl_xor_sync(0xffffffffu, u, o);
        it += __shfl_xor_sync(0xffffffffu, it, o);
      }
      if (lane == 0) {
        s_sum[warp] = u;
        s_items[warp] = it;
      }
      __syncthreads();
      long long sum = 0;
      int its = 0;
      for (int w = 0; w < kRowWarps; ++w) {
        sum += s_sum[w];
        its += s_items[w];
      }
      if (before + sum > cta_first || c == n_chunks - 1) {   // the same in every thread
        if (threadIdx.x == 0) {
          s_start = before;
          s_start_items = items;
          s_start_seq = c * RUN;
        }
        break;
      }
      before += sum;
      items += its;
      __syncthreads();
    }
  } else if (threadIdx.x == 0) {
    s_start = 0;
    s_start_items = s_start_seq = 0;
  }
  __syncthreads();

  const long long w_id = (long long)blockIdx.x * kRowWarps + warp;
  const long long u0 = w_id * per;
  long long u1 = min(total, u0 + per);
  if (u0 >= total) {                           // whole warps; no barrier follows
    if (p.tile_parts) griddep_wait();
    return;
  }

  // ---- the issuing side: where the warp stands in the line
  long long before = s_start;                  // units and items before sequence `chunk`
  int items = s_start_items, chunk = s_start_seq;
  Seq q{};
  int issued = 0, done = 0;                    // blocks
  int b = -1, in_item = 0, blk = 0, part_left = 0, q_count = 0, page_lane = 0, page_from = 0;
  bool part_starts = false;
  long long u = u0;
  uint8_t* mine = smem + warp * row_warp_smem<D, NT>();
  const uint32_t ring = smem_u32(mine), q_ring = ring + kRowStages * 2 * TILE;
  Stage* stages = reinterpret_cast<Stage*>(mine + kRowStages * (2 * TILE + ROWS * D * 2));
  int item_base = 0;                           // number of the sequence's first item

  // the sequence that holds unit u, all lanes together
  const auto locate = [&]() {
    while (true) {
      const Seq x = sequence(p, n_seqs, chunk + lane, ROWS);
      const long long n = x.units(p.n_kv);
      long long incl = n;
      int it = x.tiles * p.n_kv, it_incl = it;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, incl, o);
        const int z = __shfl_up_sync(0xffffffffu, it_incl, o);
        if (lane >= o) {
          incl += y;
          it_incl += z;
        }
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + incl > u);
      if (hit) {
        const int l = __ffs(hit) - 1;
        b = chunk + l;
        q.tok0 = __shfl_sync(0xffffffffu, x.tok0, l);
        q.nq = __shfl_sync(0xffffffffu, x.nq, l);
        q.own = __shfl_sync(0xffffffffu, x.own, l);
        q.tiles = __shfl_sync(0xffffffffu, x.tiles, l);
        q.blocks = __shfl_sync(0xffffffffu, x.blocks, l);
        item_base = items + __shfl_sync(0xffffffffu, it_incl - it, l);
        const long long off = u - (before + __shfl_sync(0xffffffffu, incl - n, l));
        const int iu = q.item_units();
        in_item = off <= 0x7fffffff ? (int)((unsigned)off / (unsigned)iu) : (int)(off / iu);
        blk = (int)(off - (long long)in_item * iu) - kItemCost;   // below 0: before the item's first block
        return;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
      items += __shfl_sync(0xffffffffu, it_incl, 31);
      chunk += 32;
      if (chunk >= n_seqs) {                   // not reached while the lengths stay what they were
        u1 = u;
        return;
      }
    }
  };
  const int pre_blocks = p.own_only ? 0 : (p.prefix_len + 15) / 16;
  const auto issue = [&](int st) {
    while (u < u1 && part_left == 0) {         // the next part: the rest of this item, or of this warp's units
      if (u == u0 || in_item + 1 >= q.tiles * p.n_kv) {
        const int was = b;
        locate();
        if (b != was || u == u0) page_from = -64;
      } else {
        ++in_item;
        blk = -kItemCost;
      }
      if (blk < 0) {                           // the item's cost before its first block
        const int skip = (int)min((long long)-blk, u1 - u);
        blk += skip;
        u += skip;
      }
      if (blk < 0 || u >= u1) break;
      part_left = (int)min((long long)(q.blocks - blk), u1 - u);
      part_starts = true;
    }
    {
      if (u < u1) {
        const int ti = in_item / p.n_kv, kvh = in_item - ti * p.n_kv;
        const bool pre = blk < pre_blocks;
        const int key = 16 * (pre ? blk : blk - pre_blocks);
        const int keys = (pre ? p.prefix_len : q.own) - key;
        // page numbers of 32 blocks at once, a block a lane
        if (blk < page_from || blk - page_from >= 32) {
          page_from = blk;
          const int bl = blk + lane;
          const bool bp = bl < pre_blocks;
          const int lp = 16 * (bp ? bl : bl - pre_blocks) / p.page_size;
          page_lane = -1;
          if (bl < q.blocks) {
            if (bp) page_lane = p.prefix_pages[lp];
            else if (lp < p.max_pages) page_lane = p.page_table[(long long)b * p.table_stride + lp];
            if (page_lane < 0 || page_lane >= p.n_pages) {
              ops::report(p.status, kDevBadIndex);
              page_lane = -1;
            }
          }
        }
        const int page = __shfl_sync(0xffffffffu, page_lane, blk - page_from);
        const bool ok = page >= 0;
        const int slot = key % p.page_size;
        const T* ks = (const T*)p.k.base + kvh * p.k.head + (ok ? page : 0) * p.k.page + slot * p.k.slot;
        const T* vs = (const T*)p.v.base + kvh * p.v.head + (ok ? page : 0) * p.v.page + slot * p.v.slot;
        const uint32_t dst = ring + st * 2 * TILE;
#pragma unroll
        for (int c = 0; c < 16 * CH / 32; ++c) {
          const int x = c * 32 + lane, row = x / CH, col = x % CH;
          const uint32_t at = dst + row * (D * 2) + ((col ^ (row & 7)) << 4);
          const bool live = ok && row < keys;
          cp16(at, live ? ks + row * p.k.slot + col * 8 : ks, live);
          cp16(at + TILE, live ? vs + row * p.v.slot + col * 8 : vs, live);
        }
        const int row0 = ti * ROWS, n_rows = min(ROWS, q.nq * p.group - row0);
        if (part_starts) {
          ++q_count;
#pragma unroll 1
          for (int x = lane; x < ROWS * CH; x += 32) {
            const int row = x / CH, col = x % CH;
            const bool live = row < n_rows;
            const int j = (row0 + row) / p.group, g = row0 + row - j * p.group;
            const T* src = (const T*)p.q + (live ? (long long)(q.tok0 + j) * p.q_tok + (long long)(kvh * p.group + g) * p.q_head + col * 8 : 0);
            cp16(q_ring + (q_count % kRowStages) * ROWS * D * 2 + row * (D * 2) + ((col ^ (row & 7)) << 4), src, live);
          }
        }
        if (lane == 0)
          stages[st] = Stage{keys, (pre ? 0 : p.prefix_len) + key,
                             (part_starts ? 1 : 0) | (part_left == 1 ? 2 : 0) | (blk == 0 ? 4 : 0) | (blk == q.blocks - 1 ? 8 : 0), q.tok0,
                             p.prefix_len + q.own - q.nq + 1, row0, n_rows, kvh, item_base + in_item, q_count % kRowStages};
        part_starts = false;
        ++blk;
        --part_left;
        ++u;
        ++issued;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  uint32_t qf[NT][KK][2];
  int lim[NT][2];
  float m[NT][2], l[NT][2], o[NT][KK][4];
#pragma unroll
  for (int s = 0; s < kRowStages - 1; ++s) issue(s);
  int st = 0;
  bool item_first = false;                     // the warp's part holds the item's first block
  for (; done < issued; ++done) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRowStages - 2) : "memory");
    __syncwarp();
    const Stage sg = stages[st];
    const uint32_t kt = ring + st * 2 * TILE, vt = kt + TILE;
    const int mat = lane >> 3, r8 = lane & 7;
    if (sg.flags & 1) {
      item_first = sg.flags & 4;
      // query fragments (B operand): lane holds row lane / 4, values 2 (lane % 4) + {0, 1, 8, 9} of each 16
      const uint32_t qs = q_ring + sg.q_slot * ROWS * D * 2;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < KK; k += 2) {
          const int row = n * 8 + r8, col = 2 * k + mat;
          ldmatrix_x4(qf[n][k][0], qf[n][k][1], qf[n][k + 1][0], qf[n][k + 1][1], qs + row * (D * 2) + ((col ^ (row & 7)) << 4));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = n * 8 + 2 * (lane & 3) + e;
          lim[n][e] = c < sg.n_rows ? sg.first_lim + (sg.row0 + c) / p.group : 0;
          m[n][e] = -INFINITY;
          l[n][e] = 0.f;
        }
#pragma unroll
        for (int d = 0; d < KK; ++d) o[n][d][0] = o[n][d][1] = o[n][d][2] = o[n][d][3] = 0.f;
      }
    }
    issue(st == 0 ? kRowStages - 1 : st - 1);
    st = st + 1 == kRowStages ? 0 : st + 1;
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
    const int left = sg.keys - (lane >> 2);      // > 0: the key exists
    const int pos = sg.pos + (lane >> 2);
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
        const float m_new = fmaxf(m[n][e], mx - below_top<T>(0));
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
    if (sg.flags & 2) {
      // the part is done: the rows' sums, and the result or a partial
      const bool whole = item_first && (sg.flags & 8) && !p.tile_parts;
      const long long part = w_id + sg.item;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
          l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
          l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
          const int c = n * 8 + 2 * (lane & 3) + e;
          if (c < sg.n_rows) {
            const int j = (sg.row0 + c) / p.group, g = sg.row0 + c - j * p.group;
            const long long tok = sg.tok0 + j;
            const int head = sg.kvh * p.group + g;
            const long long row = tok * p.n_heads + head;
            if (whole) {
              const float inv = l[n][e] > 0.f ? 1.f / l[n][e] : 0.f;
              T* dst = (T*)p.out + tok * p.o_tok + head * p.o_head + (lane >> 2);
#pragma unroll
              for (int d = 0; d < KK; ++d) {
                dst[d * 16] = E::from_f32(o[n][d][e] * inv);
                dst[d * 16 + 8] = E::from_f32(o[n][d][e + 2] * inv);
              }
              if (lane < 4) p.row_parts[row] = make_int2(0, -2);
            } else {
              float* dst = p.row_o + (part * ROWS + c) * D + (lane >> 2);
              if (m[n][e] != -INFINITY)
#pragma unroll
                for (int d = 0; d < KK; ++d) {
                  dst[d * 16] = o[n][d][e];
                  dst[d * 16 + 8] = o[n][d][e + 2];
                }
              if (lane < 4) {
                p.row_ml[part * ROWS + c] = make_float2(m[n][e], l[n][e]);
                // where the row's partials begin and end, ROWS apart
                if (item_first) p.row_parts[row].x = (int)(part * ROWS + c);
                if (sg.flags & 8) p.row_parts[row].y = (int)(part * ROWS + c);
              }
            }
          }
        }
    }
    __syncwarp();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (p.tile_parts) griddep_wait();
}

// Tile `z` of the held sequences of a ragged grid: its sequence and the tile's number in it.  `n_seqs`: how
// many are held, as far as the search came (warp-wide, all lanes).
__device__ __forceinline__ bool find_tile(const Params& p, int z, int rows, int lane, int& b, int& i, int& n_seqs) {
  int before = 0;
  n_seqs = p.n_seqs;
  for (int b0 = 0; b0 < n_seqs; b0 += 32) {
    const unsigned bad = __ballot_sync(0xffffffffu, b0 + lane < n_seqs && out_of_order(p, b0 + lane));
    if (bad) n_seqs = b0 + __ffs(bad) - 1;
    int n = 0;
    if (b0 + lane < n_seqs) n = ((p.cu_q[b0 + lane + 1] - p.cu_q[b0 + lane]) * p.group + rows - 1) / rows;
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

// ---------------------------------------------------------------- tiles of 128 rows
// One CTA takes up to 256 query rows of one K/V head (two tiles of 128) against one range of
// 128-key tiles, on the tensor cores: S = Q K^T and O += P V as tcgen05.mma with f32 accumulators
// in TMEM, P written back into TMEM over S as the A operand of the second product.
//   OWN = false: the rows of all sequences against the shared prefix, which is so read and
//                multiplied once for the whole batch;
//   OWN = true:  the rows of one sequence against its prefix and own keys, causally.
// Warps 0-7 and 8-15 each do the softmax of one tile, two threads a row (64 keys each; no shuffles);
// warp 16 brings the pages in by TMA; one thread of warp 17 issues the products.  While one tile's
// softmax runs, the other tile's products do.  The reference exponent of a row only moves when its maximum grows
// by more than 2^8 (weights stay below 2^8 or, in f16, 2^15, inside f16's and f32's range), so that O in TMEM is
// hardly ever rescaled.  (Both, the two tiles in turns and the reference that lags, are published
// techniques for attention on these tensor cores.)
//
// Bound: for a wide batch the tensor cores and the exponentials (a 128 x 128 tile needs 1024 cycles
// of products at head_dim 128, 512 at 64, and 1024 of ex2), for a narrow one the reading of K and V.
constexpr int kTile = 128;
constexpr int kTileThreads = 576;   // 16 warps of softmax, one that loads, one that multiplies
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
  __shared__ float s_row[2][kTile];    // between the two threads of a row
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ volatile int s_held, s_begin, s_end;   // OWN = false: the sequences that are held, their tokens
  volatile int* abort = &s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y, split = blockIdx.z;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 512);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 2 * kTile);
    }
    mbar_init(o_done, 1);
    mbar_init(tail, 1);
    fence_mbar_init();
    s_abort = 0;
    prefetch_tmap(&kmap);
    prefetch_tmap(&vmap);
  }
  // The kernel after this one may start once what came before both is done (griddep_launch follows the
  // wait).  After the shared prefix's kernel, of which nothing is read here, this one takes the SMs that
  // it leaves free, and ends after it.
  const bool beside = OWN && p.own_only;
  if (!beside) griddep_wait();
  griddep_launch();

  // ---- the rows and keys of this CTA (the same in every thread)
  int b = 0, ti = blockIdx.x;
  int tok0 = 0, n_rows, own = 0, first_lim = p.prefix_len, last_lim = p.prefix_len;
  if (OWN) {
    int n_seqs;
    const bool found = find_tile(p, blockIdx.x, 2 * kTile, lane, b, ti, n_seqs);
    // the last block finds its tile behind all others, if any: it has seen every offset that counts
    if (blockIdx.x == gridDim.x - 1 && (threadIdx.x | kvh | split) == 0) tell_held(p, n_seqs);
    if (!found) {
      if (beside) griddep_wait();
      return;
    }
    tok0 = p.cu_q[b];
    const int nq = p.cu_q[b + 1] - tok0;
    const int cap = p.max_pages * p.page_size, given = p.suffix_lens[b];
    own = max(0, min(given, cap));
    n_rows = min(2 * kTile, nq * p.group - ti * 2 * kTile);
    if (given > cap && threadIdx.x == 0) ops::report(p.status, kDevBadIndex);
    first_lim = p.prefix_len + own - nq + 1;
    last_lim = max(0, first_lim + (ti * 2 * kTile + n_rows - 1) / p.group);
  } else {
    n_rows = min((long long)2 * kTile, (long long)p.n_tokens * p.group - (long long)ti * 2 * kTile);
  }
  const int row0 = ti * 2 * kTile;                       // first row: token tok0 + row / group, head row % group
  const int n_pre = OWN && p.own_only ? 0 : (min(p.prefix_len, last_lim) + kTile - 1) / kTile;
  const int n_all = n_pre + (max(0, last_lim - p.prefix_len) + kTile - 1) / kTile;
  const int per = (n_all + p.parts - 1) / p.parts;
  const int t0 = split * per, n = max(0, min(n_all, t0 + per) - t0);
  const int n_tiles = n_rows > kTile ? 2 : 1;

  if (warp == 17) {
    tc::tmem_alloc(&s_tmem, 512);
    if (!OWN) {
      if (p.max_pages == 0) {   // no other kernel looks at the lengths: the blocks share them out
        const long long cta = (long long)blockIdx.x * gridDim.y * gridDim.z + kvh * gridDim.z + split, ctas = (long long)gridDim.x * gridDim.y * gridDim.z;
        for (long long b = cta * 32 + lane; b < p.n_seqs; b += ctas * 32)
          if (p.suffix_lens[b] > 0) ops::report(p.status, kDevBadIndex);
      }
      int n_seqs = p.n_seqs, begin = 0, end = p.n_tokens;
      if (p.cu_q) {
        for (int b0 = 0; b0 < n_seqs; b0 += 32) {
          const unsigned bad = __ballot_sync(0xffffffffu, b0 + lane < n_seqs && out_of_order(p, b0 + lane));
          if (bad) n_seqs = b0 + __ffs(bad) - 1;
        }
        begin = p.cu_q[0];
        end = p.cu_q[n_seqs];
        if ((blockIdx.x | kvh | split | lane) == 0) tell_held(p, n_seqs);
      }
      if (lane == 0) {
        s_held = n_seqs;
        s_begin = begin;
        s_end = end;
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t t_s[2] = {tmem, tmem + 128}, t_o[2] = {tmem + 256, tmem + 384};

  if (warp == 16) {
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
  } else if (warp == 17) {
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
  } else {
    // ---- Q into shared memory (128-byte swizzle), then the softmax of half the keys of one tile
    const int wg = warp >> 3, half = warp >> 2 & 1, row = threadIdx.x & (kTile - 1);
    {
      constexpr int CH = D / 8, STEP = 2 * kTile / CH, N = CH / 2;   // 16-byte chunks of a row; this thread's rows are STEP apart
      const int x = threadIdx.x & (2 * kTile - 1), c = x % CH, r0 = x / CH;
      int g = (row0 + wg * kTile + r0) % p.group;
      long long tok = tok0 + (row0 + wg * kTile + r0) / p.group;
      const int step_g = STEP % p.group, step_tok = STEP / p.group;
      const T* src = (const T*)p.q + (long long)kvh * p.group * p.q_head + c * 8;
      uint4 v[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        v[k] = wg * kTile + r0 + k * STEP < n_rows ? *reinterpret_cast<const uint4*>(src + tok * p.q_tok + g * p.q_head) : make_uint4(0, 0, 0, 0);
        g += step_g;
        tok += step_tok;
        if (g >= p.group) {
          g -= p.group;
          ++tok;
        }
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int r = r0 + k * STEP;
        *reinterpret_cast<uint4*>(smem + wg * C::kSlot + (c >> 3) * kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[k];
      }
    }
    fence_async_smem();
    mbar_arrive(q_full);

    if (wg < n_tiles) {
      constexpr int K = kTile / 2, DH = D / 2;
      const int lr = wg * kTile + row;   // this thread's row
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      int lim = OWN ? first_lim + (row0 + min(lr, n_rows - 1)) / p.group : p.prefix_len;   // keys that the row sees
      if (!OWN && p.cu_q) {
        // the row's sequence: where its queries reach into the prefix, they do not see all of it
        const int tok = (row0 + min(lr, n_rows - 1)) / p.group;
        int lo = 0, hi = s_held;               // cu_q[lo] <= tok < cu_q[hi], if it is any sequence's
        while (hi - lo > 1) {
          const int mid = (lo + hi) / 2;
          if (p.cu_q[mid] <= tok) lo = mid;
          else hi = mid;
        }
        const int own_keys = max(0, min(p.suffix_lens[lo], p.max_pages * p.page_size));
        lim = min(p.prefix_len, p.prefix_len + own_keys - p.cu_q[lo + 1] + tok + 1);
      }
      float m = -INFINITY, l = 0.f;
      // after a failed wait the threads of a tile go on to meet at the same barriers, without work
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        ok = __all_sync(0xffffffffu, ok && ops::wait_phase(&s_full[wg], (uint32_t)j & 1u, abort, p.status, kDevTimeoutAcc));
        tc::tc_fence_after();
        float s[K];
        tc::tmem_ld64(t_s[wg] + lanes + half * K, s);
        const int t = t0 + j;
        const bool pre = t < n_pre;
        const int key = kTile * (pre ? t : t - n_pre) + half * K;
        const int see = min((pre ? p.prefix_len : own), lim - (pre ? 0 : p.prefix_len)) - key;   // keys of this half that count
        if (__any_sync(0xffffffffu, see < K)) {
#pragma unroll
          for (int i = 0; i < K; ++i)
            if (i >= see) s[i] = -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i + 8 <= K; i += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], s[i + 2 * k], s[i + 2 * k + 1]);
        mx[0] = max3(mx[0], s[K - 4], s[K - 3]);
        mx[1] = max3(mx[1], s[K - 2], s[K - 1]);
        const float top = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), p.scale_log2, -below_top<T>(8));
        // The two halves' scores are in registers once all have met here, so the weights may take
        // their columns; and all know whether a row of the tile has outgrown its reference
        tc::tc_fence_before();
        if (named_bar_or(1 + wg, 2 * kTile, j == 0 || top > m + 8.f)) {
          if (half == 1) s_row[wg][row] = top;
          named_bar_sync(1 + wg, 2 * kTile);
          if (half == 0) s_row[wg][row] = fmaxf(m, fmaxf(top, s_row[wg][row]));
          named_bar_sync(1 + wg, 2 * kTile);
          const float m_new = s_row[wg][row], f = m == m_new ? 1.f : ex2(m - m_new);
          l *= f;
          m = m_new;
          tc::tc_fence_after();
          if (j > 0) {
            // scores in TMEM mean that the products before them are done: O may change
#pragma unroll 1
            for (int c = half * DH; c < (half + 1) * DH; c += 16) {
              float o[16];
              uint32_t u[16];
              tc::tmem_ld16(t_o[wg] + lanes + c, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(o[i] * f);
              tc::tmem_st16(t_o[wg] + lanes + c, u);
            }
          }
        }
        tc::tc_fence_after();
        const float m_use = m == -INFINITY ? 0.f : m;
        const f32x2 scale2 = pack2(p.scale_log2, p.scale_log2), off2 = pack2(-m_use, -m_use);
        f32x2 sum[2] = {pack2(l, 0.f), pack2(0.f, 0.f)};
        uint32_t u[K / 2];
#pragma unroll
        for (int i = 0; i < K; i += 2) {
          float x, y;
          unpack2(fma2(pack2(s[i], s[i + 1]), scale2, off2), x, y);
          x = ex2(x);
          y = ex2(y);
          sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pack2(x, y));
          u[i >> 1] = E::pack(x, y);
        }
        tc::tmem_st32(t_s[wg] + lanes + half * (K / 2), u);
        {
          float x, y;
          unpack2(add2(sum[0], sum[1]), x, y);
          l = x + y;
        }
        tc::tmem_st_wait();
        tc::tc_fence_before();
        mbar_arrive(&p_full[wg]);
      }
      if (n > 0) ok = __all_sync(0xffffffffu, ok && ops::wait_phase(o_done, 0, abort, p.status, kDevTimeoutAcc));
      named_bar_sync(1 + wg, 2 * kTile);       // the last maxima are read
      if (half == 1) s_row[wg][row] = l;
      named_bar_sync(1 + wg, 2 * kTile);
      if (half == 0) s_row[wg][row] = l + s_row[wg][row];
      named_bar_sync(1 + wg, 2 * kTile);
      l = s_row[wg][row];
      if (ok) {
        tc::tc_fence_after();
        const long long tok = tok0 + (row0 + lr) / p.group;
        const bool live = lr < n_rows && (OWN || (tok >= s_begin && tok < s_end));
        const int head = kvh * p.group + (row0 + lr) % p.group;
        const long long at = (long long)(p.part0 + split) * p.n_tokens * p.n_heads + tok * p.n_heads + head;
        const float inv = l > 0.f ? 1.f / l : 0.f;
        if (live && !p.direct && half == 0) p.tile_ml[at] = make_float2(m, l);
        // Through the ring (free now), so that a warp writes whole halves of rows; 16 bytes of padding
        // keep the threads' rows on different banks
        const int row_bytes = p.direct ? DH * 2 : DH * 4, pitch = row_bytes + 16;
        uint8_t* stage = ring + (size_t)warp * 32 * pitch;
#pragma unroll 1
        for (int c = 0; c < DH; c += 32) {
          float o[32];
          if (n > 0) {
            tc::tmem_ld32(t_o[wg] + lanes + half * DH + c, o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
          }
          if (p.direct) {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4*>(stage + lane * pitch + (c + i) * 2) =
                  make_uint4(E::pack(o[i] * inv, o[i + 1] * inv), E::pack(o[i + 2] * inv, o[i + 3] * inv),
                             E::pack(o[i + 4] * inv, o[i + 5] * inv), E::pack(o[i + 6] * inv, o[i + 7] * inv));
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(stage + lane * pitch + (c + i) * 4) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        __syncwarp();
        const bool written = live && (p.direct || m != -INFINITY);
        const long long dst = p.direct ? (tok * p.o_tok + (long long)head * p.o_head + half * DH) * 2 : (at * D + half * DH) * 4;
        char* to = p.direct ? (char*)p.out : (char*)p.tile_o;
        const unsigned all = __ballot_sync(0xffffffffu, written);
        const int chunks = row_bytes / 16, rows_at_once = 32 / chunks;   // a warp writes 2, 4 or 8 half rows at once
        const int sub = lane / chunks, col = lane % chunks;
#pragma unroll 4
        for (int r0 = 0; r0 < 32; r0 += rows_at_once) {
          const int r = r0 + sub;
          const long long off = __shfl_sync(0xffffffffu, dst, r);
          if (all >> r & 1) *reinterpret_cast<uint4*>(to + off + col * 16) = *reinterpret_cast<const uint4*>(stage + r * pitch + col * 16);
        }
      }
    }
  }
  __syncwarp();
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
  if (beside) griddep_wait();
}

// ---------------------------------------------------------------- joining key ranges
// One warp per row (token, head): the maximum over its partials, then the weighted sums in the
// order of the partials, so the result does not depend on timing.  U partials are on their way at
// a time: with many rows four, for the fewer registers (62 against 96 at D 128) that let more
// warps onto an SM (14000 rows of D 64 in a graph: 87.1 us for the whole call, with eight 91.8;
// 20480 rows of D 128: 86.9 and 93.0), with few rows eight, for the latency of their many partials
// (128 rows: 12.3 us, with four 13.4; 2048 rows: 25.4 and 26.1).
template <typename T, int D, int U>
__global__ void __launch_bounds__(128) k_attn_join(const __grid_constant__ Params p) {
  using E = ops::Elem<T>;
  constexpr int V = D / 32;   // values a lane
  griddep_launch();
  griddep_wait();
  const long long rows = (long long)p.n_tokens * p.n_heads;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const long long tok = row / p.n_heads;
  if (p.cu_q) {
    const int2 span = __ldcg(p.span);
    if (tok < span.x || tok >= span.y) return;   // no sequence's token, or a refused one's
  }
  int2 parts = make_int2(0, -1);
  if (p.rows_run) parts = __ldcg(p.row_parts + row);
  if (parts.y == -2) return;
  const int n_row = parts.y < 0 ? 0 : (parts.y - parts.x) / p.rows_run + 1, n = p.tile_parts + n_row;
  // partial s: the tile kernel's key ranges first
  const auto ml_of = [&](int s) {
    return s < p.tile_parts ? __ldcg(p.tile_ml + s * rows + row) : __ldcg(p.row_ml + parts.x + (long long)(s - p.tile_parts) * p.rows_run);
  };
  const auto o_of = [&](int s) {
    return (s < p.tile_parts ? p.tile_o + (s * rows + row) * D : p.row_o + (parts.x + (long long)(s - p.tile_parts) * p.rows_run) * D) + lane * V;
  };
  float M = -INFINITY;
  for (int s = lane; s < n; s += 32) M = fmaxf(M, ml_of(s).x);
  M = warp_max(M);
  const float m_use = M == -INFINITY ? 0.f : M;
  float L = 0.f, acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  for (int s0 = 0; s0 < n; s0 += 32) {
    float f = 0.f;
    if (s0 + lane < n) {
      const float2 ml = ml_of(s0 + lane);
      f = ml.x == -INFINITY ? 0.f : ex2(ml.x - m_use);
      L += ml.y * f;
    }
    const int k = min(32, n - s0);
    for (int s = 0; s < k; s += U) {
      float w[U], v[U][V];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        w[j] = __shfl_sync(0xffffffffu, f, (s + j) & 31);
        if (s + j >= k) w[j] = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = 0.f;
        if (w[j] != 0.f) {   // a range without keys left its o unwritten
          const float* o = o_of(s0 + s + j);
          if constexpr (V == 4) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(o));
            v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
          } else {
            const float2 x = __ldcg(reinterpret_cast<const float2*>(o));
            v[j][0] = x.x; v[j][1] = x.y;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += v[j][i] * w[j];
    }
  }
  L = warp_sum(L);
  const float inv = L > 0.f ? 1.f / L : 0.f;
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
