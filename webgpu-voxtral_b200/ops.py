"""Serving operators on the caller's torch tensors: one step of a batch over a paged K/V cache.

    q = rope_append_kv(q, k, v, k_pages, v_pages, page_table, seq_ids, own_positions, rope_freq,
                       rope_positions=own_positions + prefix_len)
    o = shared_prefix_attention(q, k_pages, v_pages, prefix_pages, prefix_len, page_table, suffix_lens)
    t = sample_logits(logits, u, temperature=0.8, top_k=50, top_p=0.95, min_p=0.02)

They bind vx_rope_append_kv, vx_shared_prefix_attention and vx_sample_logits of
include/voxtral_b200.h, which states what each computes.  Work goes to torch's current stream of
the tensors' device, nothing waits, and the calls may be captured into a CUDA graph.  Outputs and
workspace come from torch's allocator unless they are given.  Refused arguments raise VoxtralError;
what only the device can see (a page or an offset out of range) is reported in `status`, an int32
tensor of one element that the caller sets to 0.  The operators compute no gradients.

Page pools are [n_pages, n_kv_heads, page_size, head_dim] tensors of any strides with a contiguous
last dimension: a token-major pool [n_pages, page_size, n_kv_heads, head_dim] is passed as its
transpose(1, 2).
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
import threading

import torch
from torch.autograd import forward_ad

from .engine import VX_OK, VoxtralError, load_library

_DTYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_HALF = (torch.float16, torch.bfloat16)
_INT = torch.int32
_CACHE = "2P6q6i"                                # vx_kv_pages
_APPEND = struct.Struct("@" + _CACHE + "4P8q6Pq8i")   # vx_rope_append_args
_PREFIX = struct.Struct("@" + _CACHE + "2P4q6P2q5if")  # vx_shared_prefix_args
_SAMPLE = struct.Struct("@7Pq3f5i")              # vx_sample_args
_ERR = 256
_local = threading.local()


def _refuse(message: str):
    raise VoxtralError(-1, message)


@functools.lru_cache(maxsize=None)
def _library():
    L = load_library()
    for name in ("vx_rope_append_kv", "vx_shared_prefix_attention", "vx_sample_logits"):
        fn = getattr(L, name)
        fn.restype = ctypes.c_int
        fn.argtypes = [ctypes.c_char_p, ctypes.c_void_p, ctypes.c_char_p, ctypes.c_size_t]
    L.vx_shared_prefix_attention_workspace.restype = ctypes.c_int64
    L.vx_shared_prefix_attention_workspace.argtypes = [ctypes.c_char_p]
    return L


def _call(fn, args: bytes, device: int):
    """fn on torch's current stream of the device, which is made current for the call."""
    err = getattr(_local, "err", None)
    if err is None:
        err = _local.err = ctypes.create_string_buffer(_ERR)
    if device == torch.cuda.current_device():
        rc = fn(args, torch._C._cuda_getCurrentRawStream(device), err, _ERR)
    else:
        with torch.cuda.device(device):
            rc = fn(args, torch._C._cuda_getCurrentRawStream(device), err, _ERR)
    if rc != VX_OK:
        raise VoxtralError(rc, err.value.decode())


def _misplaced(names: str, *tensors):
    """Says which of the tensors is not where the first one is."""
    device, first = tensors[0].get_device(), names.split()[0]
    for name, t in zip(names.split(), tensors):
        if t is not None and (t.get_device() != device or device < 0):
            _refuse(f"{name} must be on a CUDA device, not {t.device}" if device < 0 else f"{name} is on {t.device}, {first} on cuda:{device}")
    _refuse("tensors must be on one CUDA device")


def _rows(name, t, dims, dtypes):
    """Shape and strides of a tensor of rows."""
    shape, stride = t.shape, t.stride()
    if len(shape) != dims or t.dtype not in dtypes or stride[-1] != 1 or t.requires_grad:
        if len(shape) != dims:
            _refuse(f"{name} must have {dims} dimensions, not {len(shape)}")
        if t.dtype not in dtypes:
            _refuse(f"{name} must be one of {', '.join(str(d) for d in dtypes)}, not {t.dtype}")
        if stride[-1] != 1 and shape[-1] > 1:
            _refuse(f"{name}: the last dimension must be contiguous")
        if t.requires_grad and torch.is_grad_enabled():
            _refuse(f"{name} requires a gradient, which this operator does not compute")
    return shape, stride


def _no_gradient(names: str, *tensors):
    """Refuses tangents, and gradients of what _rows has not looked at: the operators compute neither."""
    for i, t in enumerate(tensors):
        if t is None or not t.is_floating_point():
            continue
        if t.requires_grad and torch.is_grad_enabled():
            _refuse(f"{names.split()[i]} requires a gradient, which this operator does not compute")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            _refuse(f"{names.split()[i]} has a tangent, which this operator does not carry on")


def _whole(name, v):
    """A whole number that fits 32 bits."""
    try:
        n = int(v)
        if n == v and -2**31 <= n < 2**31:
            return n
    except (TypeError, ValueError, OverflowError):
        pass
    _refuse(f"{name} {v} must be a whole number of 32 bits")


def _real(name, v):
    try:
        return float(v)
    except (TypeError, ValueError, OverflowError):
        _refuse(f"{name} {v} must be a number")


def _vector(name, t, dtype, n=None):
    shape = t.shape
    if len(shape) != 1 or t.dtype is not dtype or not t.is_contiguous():
        _refuse(f"{name} must be a contiguous {dtype} tensor of one dimension, not {t.dtype} {tuple(shape)}")
    if n is not None and shape[0] != n:
        _refuse(f"{name} must have {n} elements, not {shape[0]}")


def _cache(k_pages, v_pages):
    shape, ks = _rows("k_pages", k_pages, 4, _HALF)
    shape_v, vs = _rows("v_pages", v_pages, 4, (k_pages.dtype,))
    if shape != shape_v:
        _refuse(f"k_pages {tuple(shape)} and v_pages {tuple(shape_v)} must have one shape")
    return (k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], *shape, _DTYPE[k_pages.dtype], 0)


def _table(page_table):
    """Rows, columns and row stride of a page table."""
    shape, stride = page_table.shape, page_table.stride()
    if len(shape) != 2 or page_table.dtype is not _INT or (shape[1] > 1 and stride[1] != 1):
        _refuse("page_table must be an int32 tensor [n_seqs, pages] with contiguous rows")
    return shape[0], shape[1], stride[0]


def _status(status):
    if status is None:
        return 0
    if status.dtype is not _INT or status.numel() != 1:
        _refuse("status must be an int32 tensor of one element")
    return status.data_ptr()


def rope_append_kv(q, k, v, k_pages, v_pages, page_table, seq_ids, positions, rope_freq, *, interleaved: bool = True,
                   rope_positions=None, q_out=None, status=None):
    """Rotates q and k of a ragged batch of tokens and appends k and v to a paged cache.

    q [n_tokens, n_heads, head_dim] (or None), k and v [n_tokens, n_kv_heads, head_dim]: f16, bf16
    or f32, one type.  Token t of sequence seq_ids[t] goes to position positions[t] (int32; negative:
    padding, of which nothing is written).  rope_freq: f32 [rot_dim / 2], the angle of pair i at
    position p is p * rope_freq[i]; pairs are neighbours (interleaved) or the two halves.
    rope_positions (int32): the positions to rotate by where they are not those in the cache, as with
    page tables that begin after a shared prefix.
    Returns the rotated q in the cache's type (q_out, if given; it may be q itself)."""
    shape, ks = _rows("k", k, 3, _DTYPE)
    shape_v, vs = _rows("v", v, 3, (k.dtype,))
    cache = _cache(k_pages, v_pages)
    n, kv, d = shape
    if shape_v != shape or kv != cache[9] or d != cache[11]:
        _refuse(f"k {tuple(shape)} and v {tuple(shape_v)} do not fit a cache of {cache[9]} heads of {cache[11]}")
    seqs, pages, table_stride = _table(page_table)
    _vector("seq_ids", seq_ids, _INT, n)
    _vector("positions", positions, _INT, n)
    if rope_positions is not None:
        _vector("rope_positions", rope_positions, _INT, n)
    _vector("rope_freq", rope_freq, torch.float32)
    if rope_freq.requires_grad or forward_ad._current_level >= 0:
        _no_gradient("k v q rope_freq k_pages v_pages q_out", k, v, q, rope_freq, k_pages, v_pages, q_out)
    heads = q_ptr = out_ptr = 0
    qs = os = (0, 0)
    if q is not None:
        shape_q, qs = _rows("q", q, 3, (k.dtype,))
        if shape_q[0] != n or shape_q[2] != d:
            _refuse(f"q {tuple(shape_q)} does not fit k {tuple(shape)}")
        if q_out is None:
            q_out = k_pages.new_empty(shape_q)
            os = q_out.stride()
        else:
            shape_o, os = _rows("q_out", q_out, 3, (k_pages.dtype,))
            if shape_o != shape_q:
                _refuse(f"q_out {tuple(shape_o)} must have q's shape {tuple(shape_q)}")
        heads, q_ptr, out_ptr = shape_q[1], q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        _refuse("q_out without q")
    device = k.get_device()
    if not (0 <= device == v.get_device() == k_pages.get_device() == v_pages.get_device() == page_table.get_device()
            == seq_ids.get_device() == positions.get_device() == rope_freq.get_device()
            and (q is None or q.get_device() == device == q_out.get_device()) and (status is None or status.get_device() == device)
            and (rope_positions is None or rope_positions.get_device() == device)):
        _misplaced("k q v k_pages v_pages page_table seq_ids positions rope_positions rope_freq q_out status", k, q, v, k_pages, v_pages,
                   page_table, seq_ids, positions, rope_positions, rope_freq, q_out, status)
    _call(_library().vx_rope_append_kv,
          _APPEND.pack(*cache, q_ptr, k.data_ptr(), v.data_ptr(), out_ptr, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1],
                       page_table.data_ptr(), seq_ids.data_ptr(), positions.data_ptr(), 0 if rope_positions is None else rope_positions.data_ptr(), rope_freq.data_ptr(), _status(status), table_stride,
                       _DTYPE[k.dtype], n, heads, seqs, pages, 2 * rope_freq.shape[0], 1 if interleaved else 0, 0), device)
    return q_out


def shared_prefix_attention(q, k_pages, v_pages, prefix_pages, prefix_len: int, page_table, suffix_lens, *, cu_q=None, scale=None,
                            out=None, workspace=None, status=None):
    """Attention over a paged cache for sequences that share their first prefix_len keys.

    q [n_tokens, n_heads, head_dim] in the cache's type.  Sequence b holds the prefix (prefix_pages,
    int32) and suffix_lens[b] keys of its own (row b of page_table), those of its query tokens among
    them; its query tokens are rows cu_q[b]:cu_q[b + 1] (int32, n_seqs + 1 of them), without cu_q
    row b.  The last query token sees every key of its sequence, each one before it one key less.
    scale defaults to 1 / sqrt(head_dim).  Returns out, shaped as q, of which it must share no memory; rows past cu_q's last are not
    written, a row that sees no key is 0.  workspace: a uint8 tensor of at least
    shared_prefix_attention_workspace bytes that no other call uses at the same time."""
    cache, sizes, pointers, device, out = _prefix_args(q, k_pages, v_pages, prefix_pages, prefix_len, page_table, suffix_lens, cu_q, out, status)
    need = _workspace_bytes(sizes, device)
    held = ptr = 0
    if workspace is not None:
        if workspace.dtype is not torch.uint8 or not workspace.is_contiguous() or workspace.get_device() != device:
            _refuse(f"workspace must be a contiguous uint8 tensor on cuda:{device}")
        ptr, held = workspace.data_ptr(), workspace.numel()
    elif need:
        workspace = q.new_empty(need >> 1)       # 2-byte elements; need is a multiple of 4
        ptr, held = workspace.data_ptr(), need
    _call(_library().vx_shared_prefix_attention,
          _PREFIX.pack(*cache, *pointers[:11], ptr, held, pointers[11], *sizes[6:], 1.0 / math.sqrt(sizes[3]) if scale is None else _real("scale", scale)),
          device)
    return out


def shared_prefix_attention_workspace(q, k_pages, v_pages, prefix_pages, prefix_len: int, page_table, suffix_lens, *, cu_q=None) -> int:
    """Bytes of workspace that shared_prefix_attention needs for these arguments.  They depend on
    shapes, prefix_len and whether cu_q is given, not on the values."""
    _, sizes, _, device, _ = _prefix_args(q, k_pages, v_pages, prefix_pages, prefix_len, page_table, suffix_lens, cu_q, q, None)
    return _workspace_bytes(sizes, device)


def _prefix_args(q, k_pages, v_pages, prefix_pages, prefix_len, page_table, suffix_lens, cu_q, out, status):
    """(cache, sizes, pointers and strides from q to status and then the table's stride, device, out)"""
    cache = _cache(k_pages, v_pages)
    shape, qs = _rows("q", q, 3, (k_pages.dtype,))
    if shape[2] != cache[11]:
        _refuse(f"q {tuple(shape)} does not fit a cache with head_dim {cache[11]}")
    if out is None:
        out = q.new_empty(shape)
        os = out.stride()
    else:
        shape_o, os = _rows("out", out, 3, (k_pages.dtype,))
        if shape_o != shape:
            _refuse(f"out {tuple(shape_o)} must have q's shape {tuple(shape)}")
    seqs, pages, table_stride = _table(page_table)
    _vector("suffix_lens", suffix_lens, _INT, seqs)
    _vector("prefix_pages", prefix_pages, _INT)
    prefix_len = _whole("prefix_len", prefix_len)
    if prefix_len < 0 or prefix_pages.shape[0] * cache[10] < prefix_len:
        _refuse(f"prefix_len {prefix_len} does not fit {prefix_pages.shape[0]} pages of {cache[10]}")
    if cu_q is not None:
        _vector("cu_q", cu_q, _INT, seqs + 1)
    if forward_ad._current_level >= 0:
        _no_gradient("q k_pages v_pages out", q, k_pages, v_pages, out)
    device = q.get_device()
    if not (0 <= device == k_pages.get_device() == v_pages.get_device() == prefix_pages.get_device() == page_table.get_device()
            == suffix_lens.get_device() == out.get_device() and (cu_q is None or cu_q.get_device() == device)
            and (status is None or status.get_device() == device)):
        _misplaced("q k_pages v_pages prefix_pages page_table suffix_lens cu_q out status", q, k_pages, v_pages, prefix_pages,
                   page_table, suffix_lens, cu_q, out, status)
    sizes = (*cache[8:13], cu_q is not None, shape[0], seqs, shape[1], prefix_len, pages)
    pointers = (q.data_ptr(), out.data_ptr(), qs[0], qs[1], os[0], os[1], prefix_pages.data_ptr(), page_table.data_ptr(),
                suffix_lens.data_ptr(), 0 if cu_q is None else cu_q.data_ptr(), _status(status), table_stride)
    return cache, sizes, pointers, device, out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(sizes, device):
    """The library's answer for these sizes (n_pages, kv heads, page, head_dim, dtype, ragged, tokens, sequences,
    heads, prefix, pages); only sizes enter it."""
    args = _PREFIX.pack(256, 256, *[sizes[3]] * 6, *sizes[:5], 0, *[0] * 9, 256 if sizes[5] else 0, *[0] * 4, *sizes[6:], 1.0)
    with torch.cuda.device(device):
        return _library().vx_shared_prefix_attention_workspace(args)


def sample_logits(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
    """Draws one token from each row of logits [n_rows, n_cols] (f16, bf16 or f32).

    u: float64 [n_rows] in [0, 1).  In descending order of the logits (equal ones in index order)
    min_p drops what is less likely than min_p times the first, top_k keeps that many (0: all), top_p
    the shortest run that holds that share of the remaining mass; the token is the first whose
    running mass reaches u times the kept mass.  temperature 0 takes the first.  Each setting is a
    tensor by row (f32; top_k int32), or a number, which counts as such a tensor of that value.  Returns int32 [n_rows]; -1 for a row whose
    logits are all -inf or NaN."""
    shape, stride = _rows("logits", logits, 2, _DTYPE)
    rows, cols = shape
    if u.dtype is not torch.float64 or u.shape != (rows,) or not u.is_contiguous():
        _refuse(f"u must be a contiguous float64 tensor of {rows} elements, not {u.dtype} {tuple(u.shape)}")
    tensors, each, one, graded = [logits, u], [0, 0, 0, 0], [temperature, top_p, min_p, top_k], u.requires_grad
    for i in range(4):
        v = one[i]
        if isinstance(v, torch.Tensor):
            kind = torch.float32 if i < 3 else _INT
            if v.dtype is not kind or v.shape != (rows,) or not v.is_contiguous():
                _refuse(f"{('temperature', 'top_p', 'min_p', 'top_k')[i]} must be a number or a contiguous {kind} tensor of {rows} elements, "
                        f"not {v.dtype} {tuple(v.shape)}")
            tensors.append(v)
            graded = graded or v.requires_grad
            each[i], one[i] = v.data_ptr(), 0
        elif type(v) is not (float if i < 3 else int):
            one[i] = _real(("temperature", "top_p", "min_p")[i], v) if i < 3 else _whole("top_k", v)
    if graded or forward_ad._current_level >= 0:
        _no_gradient("logits u setting setting setting setting", logits, u, *tensors[2:])
    if not -2**31 <= one[3] < 2**31:
        _refuse(f"top_k {one[3]} must be a whole number of 32 bits")
    if out is None:
        out = torch.empty(rows, dtype=_INT, device=logits.device)
    else:
        _vector("out", out, _INT, rows)
        tensors.append(out)
    device = logits.get_device()
    if device < 0 or any(t.get_device() != device for t in tensors):
        _misplaced("logits u setting setting setting setting out", *tensors)
    _call(_library().vx_sample_logits,
          _SAMPLE.pack(logits.data_ptr(), u.data_ptr(), *each, out.data_ptr(), stride[0], one[0], one[1], one[2], one[3],
                       _DTYPE[logits.dtype], rows, cols, 0), device)
    return out
