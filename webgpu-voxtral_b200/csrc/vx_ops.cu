// vx_ops.cu — host side of the serving operators that run on the caller's device memory:
// argument checks, launch shapes and launches (the kernels: k_rope_append.cuh,
// k_prefix_attn.cuh, k_sample.cuh).
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>
#include <atomic>

#include "../../include/voxtral_b200.h"
#include "k_prefix_attn.cuh"
#include "k_rope_append.cuh"
#include "k_sample.cuh"

namespace {

using namespace vx;

struct Err {
  char* buf;
  size_t n;
  int fail(int code, const char* fmt, ...) const {
    if (buf && n) {
      va_list ap;
      va_start(ap, fmt);
      vsnprintf(buf, n, fmt, ap);
      va_end(ap);
    }
    return code;
  }
  int ok() const {
    if (buf && n) buf[0] = 0;
    return VX_OK;
  }
};

constexpr int kMaxDevices = 64;
constexpr double kSharePrefixBytes = 50e6;

int sm_count() {
  static std::atomic<int> known[kMaxDevices];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  n = known[dev].load();
  if (!n && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) known[dev].store(n);
  return n;
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int elem_size(int dtype) { return dtype == 2 ? 4 : 2; }
bool row_strides(int dtype, int64_t a, int64_t b) {
  const int unit = 16 / elem_size(dtype);
  return a % unit == 0 && b % unit == 0;
}

// Shared memory beyond 48 KB needs an attribute, once per kernel and device.
template <typename K>
cudaError_t allow_smem(K kernel, std::atomic<int> (&done)[kMaxDevices], size_t bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (done[dev].load() >= (int)bytes) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done[dev].store((int)bytes);
  return e;
}

// Programmatic dependent launch: the kernel may be set up while the one before it drains and
// waits for its results in griddep_wait.
template <typename... P, typename... A>
cudaError_t launch_cluster(int cluster, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const A&... args) {
  return launch_cluster(1, kernel, grid, block, smem, stream, args...);
}

int check_cache(const vx_kv_pages& c, const Err& e) {
  if (!c.k || !c.v) return e.fail(VX_E_INVALID, "cache: k and v must be device pointers");
  if (c.dtype != 0 && c.dtype != 1) return e.fail(VX_E_INVALID, "cache: dtype %d (0 F16 or 1 BF16)", c.dtype);
  if (c.n_pages < 1 || c.n_kv_heads < 1 || c.page_size < 1 || c.n_kv_heads > 65535)
    return e.fail(VX_E_RANGE, "cache: %d pages of %d slots, %d heads", c.n_pages, c.page_size, c.n_kv_heads);
  if (!aligned(c.k) || !aligned(c.v) || !row_strides(0, c.k_page_stride, c.k_head_stride) || !row_strides(0, c.k_slot_stride, 0) ||
      !row_strides(0, c.v_page_stride, c.v_head_stride) || !row_strides(0, c.v_slot_stride, 0))
    return e.fail(VX_E_INVALID, "cache: rows must start on 16-byte boundaries");
  if (std::min({c.k_page_stride, c.k_head_stride, c.k_slot_stride, c.v_page_stride, c.v_head_stride, c.v_slot_stride}) < 0)
    return e.fail(VX_E_INVALID, "cache: negative strides");
  return VX_OK;
}

int launch_error(const Err& e, cudaError_t ce) {
  return e.fail(VX_E_CUDA, "launch: %s", cudaGetErrorString(ce));
}

// ------------------------------------------------------------------ rope + append
template <typename TI, typename TC>
cudaError_t launch_append(const append::Params& p, int interleaved, cudaStream_t s) {
  // Many tokens: two warps each, so that more of them are on their way in an SM (9711 tokens with 64, 128, 256
  // threads 41, 43, 52 us).  Few: six warps share one token's latency (one token 2.8 us with 192, 4.1 with 64).
  const dim3 grid(p.n_tokens), block(p.n_tokens >= 8 * sm_count() ? 64 : 192);
  return interleaved ? launch(append::k_rope_append<TI, TC, true>, grid, block, 0, s, p)
                     : launch(append::k_rope_append<TI, TC, false>, grid, block, 0, s, p);
}

// ------------------------------------------------------------------ attention
struct Plan {
  long long shared_pairs;   // tile kernel of all rows over the shared prefix: pairs of 128-row tiles; 0: not launched
  int shared_parts;
  long long own_pairs;      // tile kernel of each sequence's rows over its keys; 0: not launched
  int own_parts;
  int nt;                   // row kernel: tiles of 8 nt rows; 0: not launched
  int row_ctas;
  int64_t tile_rows, row_rows;   // partial rows of each kind
  bool join;                // there are partials
  int64_t bytes;
};

// Key ranges of the tile kernel: one CTA an SM, so the number that makes the slowest SM's share of the
// key tiles least.  A range's start and end (loading Q, writing the partial) count as four tiles
// (a tile of 2 x 128 rows takes 2.2 us), and each range's partial is written and read once more.  Where
// the row kernel runs beside it for `row_us`, the fewest ranges that take half as long leave it the most SMs:
// 64 sequences past 617 shared and 1 to 1500 own keys with 1, 2, 3, 5 ranges 25, 25, 27, 30 us in all.  row_us goes by what the page
// tables could hold, so a step with tables of a fixed width would wait for a row kernel that has little to
// do: fewer ranges may cost the tile kernel kGiveUs at most (64 sequences past 32768 shared keys: tables of 320,
// 8192, 32768, 131072 own keys 69, 71, 71, 71 us; by row_us alone 69, 87, 278, 539).
int tile_parts(long long items, long long tiles, double partial_bytes, double row_us, int sms) {
  constexpr double kTileUs = 2.2, kGiveUs = 4.0;
  const double join = 2.0 * partial_bytes / 6e6 / kTileUs;
  const auto us = [&](int s) {
    const double waves = (double)((items * s + sms - 1) / sms);
    return (waves * ((double)((tiles + s - 1) / s) + 4.0) + s * join) * kTileUs;
  };
  int best = 1;
  for (int s = 2; s <= 64 && s <= tiles; ++s)
    if (us(s) < us(best) * 0.999) best = s;
  const double most = std::min(row_us / 2, us(best) + kGiveUs);
  for (int s = 1; s < best; ++s)
    if (us(s) <= most) return s;
  return best;
}

int check_attention(const vx_shared_prefix_args& a, const Err& e) {
  const vx_kv_pages& c = a.cache;
  int rc = check_cache(c, e);
  if (rc) return rc;
  if (c.head_dim != 64 && c.head_dim != 128) return e.fail(VX_E_RANGE, "head_dim %d (64 or 128)", c.head_dim);
  if (c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1)))
    return e.fail(VX_E_RANGE, "page_size %d (16, 32, 64, 128 or 256)", c.page_size);
  if (a.n_tokens < 0 || a.n_seqs < 0) return e.fail(VX_E_RANGE, "%d tokens of %d sequences", a.n_tokens, a.n_seqs);
  if (a.n_heads < 1 || a.n_heads % c.n_kv_heads)
    return e.fail(VX_E_RANGE, "n_heads %d is not a multiple of n_kv_heads %d", a.n_heads, c.n_kv_heads);
  if (a.prefix_len < 0 || a.prefix_len > (1 << 30) || a.max_pages < 0 || (int64_t)a.max_pages * c.page_size > (1 << 30))
    return e.fail(VX_E_RANGE, "prefix_len %d, %d pages of %d own keys: at most 2^30 each", a.prefix_len, a.max_pages, c.page_size);
  // positions and limits are ints, up to a tile past the last key
  if ((int64_t)a.prefix_len + (int64_t)a.max_pages * c.page_size > 0x7fffff00)
    return e.fail(VX_E_RANGE, "prefix_len %d and %d pages of %d own keys: at most 2^31 - 256 together", a.prefix_len, a.max_pages, c.page_size);
  if (!(a.scale > 0.f) || a.scale > 1e30f) return e.fail(VX_E_RANGE, "scale %g must be positive", (double)a.scale);
  if (!a.cu_q && a.n_tokens != a.n_seqs)
    return e.fail(VX_E_INVALID, "%d tokens for %d sequences: cu_q is needed", a.n_tokens, a.n_seqs);
  return VX_OK;
}

// Launch shape of arguments that check_attention has let pass.
int plan_attention(const vx_shared_prefix_args& a, Plan& pl, const Err& e) {
  const vx_kv_pages& c = a.cache;
  const int group = a.n_heads / c.n_kv_heads, sms = sm_count();
  if (!sms) return e.fail(VX_E_CUDA, "no current CUDA device");
  const long long own_keys = (long long)a.max_pages * c.page_size, rows = (long long)a.n_tokens * group;
  pl = Plan{};
  const long long each = rows / std::max(1, a.n_seqs);   // rows a sequence
  // The row kernel reads the prefix again for every sequence (every 32 rows of one): from L2, 8 MB a us.
  // Where that would take longer than the tile kernel's start and end, the rows of all sequences
  // take the prefix together; not where the sequences' rows fill tiles by themselves, and partials of
  // the prefix and of the own keys would only add to the work.
  const double partial = (double)a.n_tokens * a.n_heads * c.head_dim * 4;
  const double again = (double)(a.cu_q ? rows / 32 + a.n_seqs : a.n_seqs) * a.prefix_len * c.n_kv_heads * c.head_dim * 4;
  // the row kernel beside it: its own start and end, and half the keys that the page tables can hold
  const double row_us = a.cu_q ? 0.0 : 8.0 + (double)a.n_seqs * own_keys * c.n_kv_heads * c.head_dim * 2 / 6.4e6;
  if (a.n_seqs > 1 && again > kSharePrefixBytes && each < 512) {
    pl.shared_pairs = (rows + 255) / 256;
    pl.shared_parts = tile_parts(pl.shared_pairs * c.n_kv_heads, (a.prefix_len + 127) / 128, partial, row_us, sms);
  }
  // The tile kernel multiplies 128 rows at once; of sequences with fewer than 64 the row kernel's tiles of
  // 32 waste less
  if (a.cu_q && own_keys + a.prefix_len && each >= 64) {
    pl.own_pairs = rows / 256 + a.n_seqs;
    const long long keys = (pl.shared_pairs ? 0 : (a.prefix_len + 127) / 128) + (own_keys + 127) / 128;
    pl.own_parts = keys ? tile_parts(pl.own_pairs * c.n_kv_heads, keys, partial, 0.0, sms) : 0;
    if (!keys) pl.own_pairs = 0;
  } else if (own_keys || !pl.shared_pairs) {
    pl.nt = a.cu_q || group > 16 ? 4 : group > 8 ? 2 : 1;
    // beside a tile kernel that leaves SMs free, those
    const long long busy = pl.shared_pairs * c.n_kv_heads * pl.shared_parts;
    pl.row_ctas = busy <= sms / 2 ? (int)(sms - busy) : sms;
  }
  const long long tile = 8 * pl.nt;
  const long long items = !pl.nt ? 0 : (a.cu_q ? rows / tile + a.n_seqs : a.n_seqs * ((group + tile - 1) / tile)) * c.n_kv_heads;
  const int parts = pl.shared_parts + pl.own_parts;
  pl.join = pl.nt || parts > 1;
  pl.tile_rows = pl.join ? (int64_t)parts * a.n_tokens * a.n_heads : 0;
  pl.row_rows = pl.nt ? ((int64_t)pl.row_ctas * pattn::row_warps(c.head_dim, pl.nt) + items) * tile : 0;
  if (std::max(pl.shared_pairs, pl.own_pairs) > 0x7fffffff || pl.row_rows > 0x7fffffff || (long long)a.n_tokens * a.n_heads > 0x7fffffff)
    return e.fail(VX_E_RANGE, "%d tokens of %d sequences are too many for one call", a.n_tokens, a.n_seqs);
  pl.bytes = (pl.tile_rows + pl.row_rows) * (c.head_dim + 2) * 4 + (pl.nt ? (int64_t)a.n_tokens * a.n_heads * 8 : 0) + (pl.join && a.cu_q ? 8 : 0);
  return VX_OK;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Map of a page pool: boxes of 64 values x up to 128 slots of one head of one page.
cudaError_t encode_pages(CUtensorMap* map, const vx_kv_pages& c, const pattn::Pages& g) {
  static std::atomic<void*> known{nullptr};
  void* fn = known.load();
  if (!fn) {
    cudaDriverEntryPointQueryResult q;
    const cudaError_t ce = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    if (ce != cudaSuccess) return ce;
    if (!fn || q != cudaDriverEntryPointSuccess) return cudaErrorNotSupported;
    known.store(fn);
  }
  const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.page_size, (cuuint64_t)c.n_kv_heads, (cuuint64_t)c.n_pages};
  cuuint64_t strides[3] = {(cuuint64_t)g.slot * 2, (cuuint64_t)g.head * 2, (cuuint64_t)g.page * 2};
  for (int i = 0; i < 3; ++i)
    if (dims[i + 1] == 1) strides[i] = 16;   // never stepped over; the caller's may be anything
  const cuuint32_t box[4] = {64, (cuuint32_t)std::min(c.page_size, 128), 1, 1}, es[4] = {1, 1, 1, 1};
  const CUresult r = ((EncodeTiledFn)fn)(map, c.dtype ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                                         const_cast<void*>(g.base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, int D, int NT>
cudaError_t launch_rows(const pattn::Params& p, int ctas, cudaStream_t s) {
  static std::atomic<int> done[kMaxDevices];
  constexpr int bytes = pattn::row_smem<D, NT>();
  cudaError_t ce = allow_smem(pattn::k_attn_rows<T, D, NT>, done, bytes);
  if (ce != cudaSuccess) return ce;
  return launch(pattn::k_attn_rows<T, D, NT>, dim3(ctas), dim3(pattn::row_warps(D, NT) * 32), bytes, s, p);
}
template <typename T, int D, bool OWN>
cudaError_t launch_tiles(pattn::Params p, const vx_kv_pages& c, long long pairs, int part0, int parts, cudaStream_t s) {
  p.part0 = part0;
  p.parts = parts;
  static std::atomic<int> done[kMaxDevices];
  constexpr size_t bytes = pattn::TileCfg<D>::kSmem;
  cudaError_t ce = allow_smem(pattn::k_attn_tiles<T, D, OWN>, done, bytes);
  CUtensorMap km, vm;
  if (ce == cudaSuccess) ce = encode_pages(&km, c, p.k);
  if (ce == cudaSuccess) ce = encode_pages(&vm, c, p.v);
  if (ce != cudaSuccess) return ce;
  return launch(pattn::k_attn_tiles<T, D, OWN>, dim3((unsigned)pairs, p.n_kv, parts), dim3(pattn::kTileThreads), bytes, s, km, vm, p);
}

template <typename T, int D>
cudaError_t launch_attention(const pattn::Params& p, const vx_kv_pages& c, const Plan& pl, cudaStream_t s) {
  cudaError_t ce = cudaSuccess;
  if (pl.shared_pairs) ce = launch_tiles<T, D, false>(p, c, pl.shared_pairs, 0, pl.shared_parts, s);
  if (ce == cudaSuccess && pl.own_pairs) ce = launch_tiles<T, D, true>(p, c, pl.own_pairs, pl.shared_parts, pl.own_parts, s);
  if (ce == cudaSuccess && pl.nt)
    ce = pl.nt == 1 ? launch_rows<T, D, 1>(p, pl.row_ctas, s)
         : pl.nt == 2 ? launch_rows<T, D, 2>(p, pl.row_ctas, s) : launch_rows<T, D, 4>(p, pl.row_ctas, s);
  if (ce != cudaSuccess || p.direct) return ce;
  const long long rows = (long long)p.n_tokens * p.n_heads;
  const dim3 grid((unsigned)((rows + 3) / 4));
  // Above 8192 rows there are 55 warps an SM and more: occupancy counts, below it latency.
  return rows >= 8192 ? launch(pattn::k_attn_join<T, D, 4>, grid, dim3(128), 0, s, p)
                      : launch(pattn::k_attn_join<T, D, 8>, grid, dim3(128), 0, s, p);
}

// ------------------------------------------------------------------ sampling
template <typename T, int C>
cudaError_t launch_sample(const sample::Params& p, int rows, cudaStream_t s) {
  static std::atomic<int> done[kMaxDevices];
  const size_t bytes = sizeof(sample::Smem) + (p.resident ? (size_t)p.slice * 4 : 0);
  cudaError_t ce = allow_smem(sample::k_sample<T, C>, done, sizeof(sample::Smem) + sample::kResident * 4);
  if (ce != cudaSuccess) return ce;
  return launch_cluster(C, sample::k_sample<T, C>, dim3((unsigned)rows * C), dim3(sample::kThreads), bytes, s, p);
}
template <typename T>
cudaError_t launch_sample(const sample::Params& p, int rows, int cluster, cudaStream_t s) {
  return cluster == 1 ? launch_sample<T, 1>(p, rows, s) : cluster == 2 ? launch_sample<T, 2>(p, rows, s)
         : cluster == 4 ? launch_sample<T, 4>(p, rows, s) : launch_sample<T, 8>(p, rows, s);
}

}  // namespace

extern "C" int vx_rope_append_kv(const vx_rope_append_args* ap, void* stream, char* err, size_t err_len) {
  const Err e{err, err_len};
  if (!ap) return e.fail(VX_E_INVALID, "arguments are null");
  const vx_rope_append_args& a = *ap;
  const vx_kv_pages& c = a.cache;
  int rc = check_cache(c, e);
  if (rc) return rc;
  if (a.dtype < 0 || a.dtype > 2) return e.fail(VX_E_INVALID, "dtype %d (0 F16, 1 BF16, 2 F32)", a.dtype);
  if (c.head_dim < 16 || c.head_dim > 512 || c.head_dim % 16)
    return e.fail(VX_E_RANGE, "head_dim %d must be a multiple of 16 in [16, 512]", c.head_dim);
  if (a.rot_dim < 0 || a.rot_dim > c.head_dim || a.rot_dim % 16)
    return e.fail(VX_E_RANGE, "rot_dim %d must be a multiple of 16 up to head_dim %d", a.rot_dim, c.head_dim);
  if (a.n_tokens < 0 || a.n_heads < 0 || a.n_seqs < 0 || a.max_pages < 0)
    return e.fail(VX_E_RANGE, "%d tokens, %d heads, %d sequences of %d pages", a.n_tokens, a.n_heads, a.n_seqs, a.max_pages);
  if ((int64_t)(a.n_heads + 2LL * c.n_kv_heads) * (c.head_dim / 16) > 0x7fffffff)
    return e.fail(VX_E_RANGE, "%d heads of %d values are too many", a.n_heads, c.head_dim);
  if (a.n_tokens == 0) return e.ok();
  if (!a.k || !a.v || !a.page_table || !a.seq_ids || !a.positions || (a.n_heads && (!a.q || !a.q_out)) || (a.rot_dim && !a.rope_freq))
    return e.fail(VX_E_INVALID, "q, k, v, q_out, page_table, seq_ids, positions and rope_freq must be device pointers");
  if (!aligned(a.q) || !aligned(a.k) || !aligned(a.v) || !aligned(a.q_out) || !row_strides(a.dtype, a.q_token_stride, a.q_head_stride) ||
      !row_strides(a.dtype, a.k_token_stride, a.k_head_stride) || !row_strides(a.dtype, a.v_token_stride, a.v_head_stride) ||
      !row_strides(0, a.q_out_token_stride, a.q_out_head_stride))
    return e.fail(VX_E_INVALID, "rows of q, k, v and q_out must start on 16-byte boundaries");
  append::Params p{};
  p.q = a.q; p.k = a.k; p.v = a.v; p.q_out = a.q_out; p.k_pages = c.k; p.v_pages = c.v;
  p.q_tok = a.q_token_stride; p.q_head = a.q_head_stride; p.k_tok = a.k_token_stride; p.k_head = a.k_head_stride;
  p.v_tok = a.v_token_stride; p.v_head = a.v_head_stride; p.qo_tok = a.q_out_token_stride; p.qo_head = a.q_out_head_stride;
  p.kp_page = c.k_page_stride; p.kp_head = c.k_head_stride; p.kp_slot = c.k_slot_stride;
  p.vp_page = c.v_page_stride; p.vp_head = c.v_head_stride; p.vp_slot = c.v_slot_stride;
  p.page_table = a.page_table; p.seq_ids = a.seq_ids; p.positions = a.positions; p.rope_positions = a.rope_positions; p.freq = a.rope_freq; p.status = a.status;
  p.table_stride = a.table_stride; p.n_tokens = a.n_tokens; p.n_heads = a.n_heads; p.n_kv = c.n_kv_heads;
  p.head_dim = c.head_dim; p.rot_dim = a.rot_dim; p.page_size = c.page_size; p.n_pages = c.n_pages; p.n_seqs = a.n_seqs;
  p.max_pages = a.max_pages;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t ce;
  if (c.dtype == 0)
    ce = a.dtype == 0 ? launch_append<__half, __half>(p, a.interleaved, s)
         : a.dtype == 1 ? launch_append<__nv_bfloat16, __half>(p, a.interleaved, s) : launch_append<float, __half>(p, a.interleaved, s);
  else
    ce = a.dtype == 0 ? launch_append<__half, __nv_bfloat16>(p, a.interleaved, s)
         : a.dtype == 1 ? launch_append<__nv_bfloat16, __nv_bfloat16>(p, a.interleaved, s)
                        : launch_append<float, __nv_bfloat16>(p, a.interleaved, s);
  return ce == cudaSuccess ? e.ok() : launch_error(e, ce);
}

extern "C" int64_t vx_shared_prefix_attention_workspace(const vx_shared_prefix_args* a) {
  Plan pl{};
  const Err e{nullptr, 0};
  return a && check_attention(*a, e) == VX_OK && plan_attention(*a, pl, e) == VX_OK ? pl.bytes : 0;
}

extern "C" int vx_shared_prefix_attention(const vx_shared_prefix_args* ap, void* stream, char* err, size_t err_len) {
  const Err e{err, err_len};
  if (!ap) return e.fail(VX_E_INVALID, "arguments are null");
  const vx_shared_prefix_args& a = *ap;
  const vx_kv_pages& c = a.cache;
  int rc = check_attention(a, e);
  if (rc) return rc;
  if (a.n_tokens == 0 || a.n_seqs == 0) return e.ok();
  if (!a.q || !a.out || !a.suffix_lens || (a.max_pages && !a.page_table) || (a.prefix_len && !a.prefix_pages))
    return e.fail(VX_E_INVALID, "q, out, suffix_lens, page_table and prefix_pages must be device pointers");
  if (!aligned(a.q) || !aligned(a.out) || !row_strides(0, a.q_token_stride, a.q_head_stride) ||
      !row_strides(0, a.out_token_stride, a.out_head_stride))
    return e.fail(VX_E_INVALID, "rows of q and out must start on 16-byte boundaries");
  if (a.out == a.q) return e.fail(VX_E_INVALID, "out must not overlap q");
  Plan pl{};
  rc = plan_attention(a, pl, e);
  if (rc) return rc;
  if (pl.bytes && (!a.workspace || (reinterpret_cast<uintptr_t>(a.workspace) & 255) || a.workspace_bytes < pl.bytes))
    return e.fail(VX_E_INVALID, "workspace: %lld bytes, 256-byte aligned, are needed", (long long)pl.bytes);
  pattn::Params p{};
  p.q = a.q; p.out = a.out;
  p.q_tok = a.q_token_stride; p.q_head = a.q_head_stride; p.o_tok = a.out_token_stride; p.o_head = a.out_head_stride;
  p.k = pattn::Pages{c.k, c.k_page_stride, c.k_head_stride, c.k_slot_stride};
  p.v = pattn::Pages{c.v, c.v_page_stride, c.v_head_stride, c.v_slot_stride};
  p.prefix_pages = a.prefix_pages; p.page_table = a.page_table; p.suffix_lens = a.suffix_lens; p.cu_q = a.cu_q;
  p.table_stride = a.table_stride; p.status = a.status;
  float* ws = (float*)a.workspace;   // f32 rows first, so that they stay 16-byte aligned
  p.tile_o = ws;
  p.row_o = ws + pl.tile_rows * c.head_dim;
  p.tile_ml = (float2*)(ws + (pl.tile_rows + pl.row_rows) * c.head_dim);
  p.row_ml = p.tile_ml + pl.tile_rows;
  p.row_parts = (int2*)(p.row_ml + pl.row_rows);
  p.tile_parts = pl.shared_parts + pl.own_parts;
  p.span = pl.join && a.cu_q ? p.row_parts + (pl.nt ? (int64_t)a.n_tokens * a.n_heads : 0) : nullptr;
  p.rows_run = 8 * pl.nt;
  p.own_only = pl.shared_pairs > 0;
  p.min_blocks = 2;
  p.direct = !pl.join;
  p.n_tokens = a.n_tokens; p.n_seqs = a.n_seqs; p.n_heads = a.n_heads; p.n_kv = c.n_kv_heads; p.group = a.n_heads / c.n_kv_heads;
  p.prefix_len = a.prefix_len; p.page_size = c.page_size; p.n_pages = c.n_pages; p.max_pages = a.max_pages;
  p.scale_log2 = a.scale * pattn::kLog2e;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t ce;
  if (c.dtype == 0) ce = c.head_dim == 64 ? launch_attention<__half, 64>(p, c, pl, s) : launch_attention<__half, 128>(p, c, pl, s);
  else ce = c.head_dim == 64 ? launch_attention<__nv_bfloat16, 64>(p, c, pl, s) : launch_attention<__nv_bfloat16, 128>(p, c, pl, s);
  return ce == cudaSuccess ? e.ok() : launch_error(e, ce);
}

extern "C" int vx_sample_logits(const vx_sample_args* ap, void* stream, char* err, size_t err_len) {
  const Err e{err, err_len};
  if (!ap) return e.fail(VX_E_INVALID, "arguments are null");
  const vx_sample_args& a = *ap;
  constexpr int most = sample::kMaxCols;
  if (a.dtype < 0 || a.dtype > 2) return e.fail(VX_E_INVALID, "dtype %d (0 F16, 1 BF16, 2 F32)", a.dtype);
  if (a.n_rows < 0 || a.n_cols < 1 || a.n_cols > most || a.row_stride < 0)
    return e.fail(VX_E_RANGE, "%d rows of %d logits (1 to %d), stride %lld", a.n_rows, a.n_cols, most, (long long)a.row_stride);
  if (!a.temperature && !(a.temperature_all >= 0.f && a.temperature_all <= 3e38f))
    return e.fail(VX_E_RANGE, "temperature %g must be 0 or more", (double)a.temperature_all);
  if (!a.top_p && !(a.top_p_all >= 0.f)) return e.fail(VX_E_RANGE, "top_p %g must be 0 or more", (double)a.top_p_all);
  if (!a.min_p && !(a.min_p_all >= 0.f && a.min_p_all <= 1.f))
    return e.fail(VX_E_RANGE, "min_p %g must be in [0, 1]", (double)a.min_p_all);
  if (a.n_rows == 0) return e.ok();
  if (!a.logits || !a.u || !a.out) return e.fail(VX_E_INVALID, "logits, u and out must be device pointers");
  if (reinterpret_cast<uintptr_t>(a.logits) % elem_size(a.dtype)) return e.fail(VX_E_INVALID, "logits must be aligned to their type");
  const int sms = sm_count();
  if (!sms) return e.fail(VX_E_CUDA, "no current CUDA device");
  // CTAs a row: more of them while all rows together give an SM less than one and a half (two fit),
  // none with fewer than 16384 logits.  One B200: 64 rows of 131072 bf16 logits with 2, 4, 8 CTAs a row
  // 47, 34, 43 us; 200 rows of f32 with 1, 2, 4 159, 142, 160 us; one row with 1, 4, 8 92, 34, 23 us; 64
  // rows of 8320 with 1, 2 CTAs 10, 12 us (top-k 64), 23, 26 us (top-p alone)
  int cluster = 1;
  while (cluster < sample::kMaxCluster && 2ll * a.n_rows * cluster < 3ll * sms && a.n_cols > 16384 * cluster) cluster *= 2;
  if ((long long)a.n_rows * cluster > 0x7fffffff) return e.fail(VX_E_RANGE, "%d rows are too many for one call", a.n_rows);
  sample::Params p{};
  p.logits = a.logits; p.stride = a.row_stride; p.u = a.u;
  p.temperature = a.temperature; p.top_p = a.top_p; p.min_p = a.min_p; p.top_k = a.top_k;
  p.temperature1 = a.temperature_all; p.top_p1 = a.top_p_all; p.min_p1 = a.min_p_all; p.top_k1 = a.top_k_all;
  p.out = a.out; p.n = a.n_cols;
  p.slice = ((a.n_cols + cluster - 1) / cluster + 7) & ~7;
  p.resident = p.slice <= sample::kResident;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t ce = a.dtype == 0 ? launch_sample<__half>(p, a.n_rows, cluster, s)
                         : a.dtype == 1 ? launch_sample<__nv_bfloat16>(p, a.n_rows, cluster, s) : launch_sample<float>(p, a.n_rows, cluster, s);
  return ce == cudaSuccess ? e.ok() : launch_error(e, ce);
}
