"""Serving operators on the caller's torch tensors: one step of a batch over a paged K/V cache.

    q = rope_append_kv(q, k, v, k_pages, v_pages, page_table, seq_ids, positions, rope_freq)
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
import math
import struct

import torch

from .engine import VX_OK, VoxtralError, load_library

_DTYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_CACHE = "2P6q6i"                                # vx_kv_pages
_APPEND = struct.Struct("@" + _CACHE + "4P8q5Pq8i")   # vx_rope_append_args
_PREFIX = struct.Struct("@" + _CACHE + "2P4q6P2q5if")  # vx_shared_prefix_args
_SAMPLE = struct.Struct("@7Pq3d6i")              # vx_sample_args
_ERR = 256


def _refuse(message: str):
    raise VoxtralError(-1, message)


def _library():
    L = load_library()
    if not hasattr(L, "_ops_bound"):
        for name in ("vx_rope_append_kv", "vx_shared_prefix_attention", "vx_sample_logits"):
            fn = getattr(L, name)
            fn.restype = ctypes.c_int
            fn.argtypes = [ctypes.c_char_p, ctypes.c_void_p, ctypes.c_char_p, ctypes.c_size_t]
        L.vx_shared_prefix_attention_workspace.restype = ctypes.c_int64
        L.vx_shared_prefix_attention_workspace.argtypes = [ctypes.c_char_p]
        L._ops_bound = True
    return L


def _call(fn, args: bytes, device):
    err = ctypes.create_string_buffer(_ERR)
    rc = fn(args, torch.cuda.current_stream(device).cuda_stream, err, _ERR)
    if rc != VX_OK:
        raise VoxtralError(rc, err.value.decode())


def _on(device):
    """The device made current for the call where it is not."""
    return torch.cuda.device(device)


def _same_place(device, **tensors):
    if device.type != "cuda":
        _refuse(f"tensors must be on a CUDA device, not {device}")
    for name, t in tensors.items():
        if t is not None and t.device != device:
            _refuse(f"{name} is on {t.device}, other arguments on {device}")


def _rows(name, t, dims, *dtypes):
    if t.dim() != dims:
        _refuse(f"{name} must have {dims} dimensions, not {t.dim()}")
    if t.dtype not in dtypes:
        _refuse(f"{name} must be one of {', '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        _refuse(f"{name}: the last dimension must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name} requires a gradient, which this operator does not compute")


def _ints(name, t, n=None):
    if t.dim() != 1 or t.dtype != torch.int32 or not t.is_contiguous():
        _refuse(f"{name} must be a contiguous int32 tensor of one dimension")
    if n is not None and t.shape[0] != n:
        _refuse(f"{name} must have {n} elements, not {t.shape[0]}")


def _cache(k_pages, v_pages):
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        _rows(name, t, 4, torch.float16, torch.bfloat16)
    if k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        _refuse("k_pages and v_pages must have one shape and type")
    n, kv, page, d = k_pages.shape
    ks, vs = k_pages.stride(), v_pages.stride()
    return (k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], n, kv, page, d, _DTYPE[k_pages.dtype], 0)


def _table(page_table):
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        _refuse("page_table must be an int32 tensor [n_seqs, pages] with contiguous rows")


def _status(status):
    if status is None:
        return 0
    if status.dtype != torch.int32 or status.numel() != 1:
        _refuse("status must be an int32 tensor of one element")
    return status.data_ptr()


def rope_append_kv(q, k, v, k_pages, v_pages, page_table, seq_ids, positions, rope_freq, *, interleaved: bool = True,
                   q_out=None, status=None):
    """Rotates q and k of a ragged batch of tokens and appends k and v to a paged cache.

    q [n_tokens, n_heads, head_dim] (or None), k and v [n_tokens, n_kv_heads, head_dim]: f16, bf16
    or f32, one type.  Token t of sequence seq_ids[t] goes to position positions[t] (int32; negative:
    padding, of which nothing is written).  rope_freq: f32 [rot_dim / 2], the angle of pair i at
    position p is p * rope_freq[i]; pairs are neighbours (interleaved) or the two halves.
    Returns the rotated q in the cache's type (q_out, if given; it may be q itself)."""
    _rows("k", k, 3, *_DTYPE)
    _rows("v", v, 3, k.dtype)
    cache = _cache(k_pages, v_pages)
    n, kv, d = k.shape
    if v.shape != k.shape or kv != cache[9] or d != cache[11]:
        _refuse(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit a cache of {cache[9]} heads of {cache[11]}")
    _table(page_table)
    _ints("seq_ids", seq_ids, n)
    _ints("positions", positions, n)
    if rope_freq.dtype != torch.float32 or rope_freq.dim() != 1 or not rope_freq.is_contiguous():
        _refuse("rope_freq must be a contiguous f32 tensor of one dimension")
    heads, qs, os = 0, (0, 0), (0, 0)
    if q is not None:
        _rows("q", q, 3, k.dtype)
        if q.shape[0] != n or q.shape[2] != d:
            _refuse(f"q {tuple(q.shape)} does not fit k {tuple(k.shape)}")
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=k_pages.dtype, device=q.device)
        _rows("q_out", q_out, 3, k_pages.dtype)
        if q_out.shape != q.shape:
            _refuse(f"q_out {tuple(q_out.shape)} must have q's shape {tuple(q.shape)}")
        heads, qs, os = q.shape[1], q.stride(), q_out.stride()
    elif q_out is not None:
        _refuse("q_out without q")
    device = k.device
    _same_place(device, q=q, v=v, k_pages=k_pages, v_pages=v_pages, page_table=page_table, seq_ids=seq_ids, positions=positions,
                rope_freq=rope_freq, q_out=q_out, status=status)
    ks, vs = k.stride(), v.stride()
    args = _APPEND.pack(*cache, q.data_ptr() if heads else 0, k.data_ptr(), v.data_ptr(), q_out.data_ptr() if heads else 0,
                        qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1], page_table.data_ptr(), seq_ids.data_ptr(),
                        positions.data_ptr(), rope_freq.data_ptr(), _status(status), page_table.stride(0), _DTYPE[k.dtype], n, heads,
                        page_table.shape[0], page_table.shape[1], 2 * rope_freq.shape[0], int(bool(interleaved)), 0)
    fn = _library().vx_rope_append_kv
    if device.index == torch.cuda.current_device():
        _call(fn, args, device)
    else:
        with _on(device):
            _call(fn, args, device)
    return q_out


def shared_prefix_attention(q, k_pages, v_pages, prefix_pages, prefix_len: int, page_table, suffix_lens, *, cu_q=None, scale=None,
                            out=None, workspace=None, status=None):
    """Attention over a paged cache for sequences that share their first prefix_len keys.

    q [n_tokens, n_heads, head_dim] in the cache's type.  Sequence b holds the prefix (prefix_pages,
    int32) and suffix_lens[b] keys of its own (row b of page_table), those of its query tokens among
    them; its query tokens are rows cu_q[b]:cu_q[b + 1] (int32, n_seqs + 1 of them), without cu_q
    row b.  The last query token sees every key of its sequence, each one before it one key less.
    scale defaults to 1 / sqrt(head_dim).  Returns out, shaped as q; rows past cu_q's last are not
    written, a row that sees no key is 0.  workspace: a uint8 tensor of at least
    shared_prefix_attention_workspace bytes that no other call uses at the same time."""
    args, device, out = _prefix_args(q, k_pages, v_pages, prefix_pages, prefix_len, page_table, suffix_lens, cu_q, scale, out, status)
    if device.index == torch.cuda.current_device():
        _prefix_call(args, device, workspace)
    else:
        with _on(device):
            _prefix_call(args, device, workspace)
    return out


def shared_prefix_attention_workspace(q, k_pages, v_pages, prefix_pages, prefix_len: int, page_table, suffix_lens, *, cu_q=None) -> int:
    """Bytes of workspace that shared_prefix_attention needs for these arguments.  They depend on
    shapes, prefix_len and whether cu_q is given, not on the values."""
    args, device, _ = _prefix_args(q, k_pages, v_pages, prefix_pages, prefix_len, page_table, suffix_lens, cu_q, None, q, None)
    with _on(device):
        return _library().vx_shared_prefix_attention_workspace(_PREFIX.pack(*args))


def _prefix_args(q, k_pages, v_pages, prefix_pages, prefix_len, page_table, suffix_lens, cu_q, scale, out, status):
    cache = _cache(k_pages, v_pages)
    _rows("q", q, 3, k_pages.dtype)
    if q.shape[2] != cache[11]:
        _refuse(f"q {tuple(q.shape)} does not fit a cache with head_dim {cache[11]}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _rows("out", out, 3, q.dtype)
    if out.shape != q.shape:
        _refuse(f"out {tuple(out.shape)} must have q's shape {tuple(q.shape)}")
    _table(page_table)
    seqs = page_table.shape[0]
    _ints("suffix_lens", suffix_lens, seqs)
    _ints("prefix_pages", prefix_pages)
    if prefix_len < 0 or prefix_pages.shape[0] * cache[10] < prefix_len:
        _refuse(f"prefix_len {prefix_len} does not fit {prefix_pages.shape[0]} pages of {cache[10]}")
    if cu_q is not None:
        _ints("cu_q", cu_q, seqs + 1)
    device = q.device
    _same_place(device, k_pages=k_pages, v_pages=v_pages, prefix_pages=prefix_pages, page_table=page_table, suffix_lens=suffix_lens,
                cu_q=cu_q, out=out, status=status)
    qs, os = q.stride(), out.stride()
    args = [*cache, q.data_ptr(), out.data_ptr(), qs[0], qs[1], os[0], os[1], prefix_pages.data_ptr(), page_table.data_ptr(),
            suffix_lens.data_ptr(), 0 if cu_q is None else cu_q.data_ptr(), _status(status), 0, 0, page_table.stride(0), q.shape[0], seqs,
            q.shape[1], prefix_len, page_table.shape[1], 1.0 / math.sqrt(q.shape[2]) if scale is None else scale]
    return args, device, out


_WORKSPACE = 25   # place of the workspace pointer in vx_shared_prefix_args; its size comes next


def _prefix_call(args, device, workspace):
    L = _library()
    if workspace is None:
        need = L.vx_shared_prefix_attention_workspace(_PREFIX.pack(*args))
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.device != device:
        _refuse(f"workspace must be a contiguous uint8 tensor on {device}")
    if workspace is not None:
        args[_WORKSPACE] = workspace.data_ptr()
        args[_WORKSPACE + 1] = workspace.numel()
    _call(L.vx_shared_prefix_attention, _PREFIX.pack(*args), device)


def sample_logits(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
    """Draws one token from each row of logits [n_rows, n_cols] (f16, bf16 or f32).

    u: float64 [n_rows] in [0, 1).  In descending order of the logits (equal ones in index order)
    min_p drops what is less likely than min_p times the first, top_k keeps that many (0: all), top_p
    the shortest run that holds that share of the remaining mass; the token is the first whose
    running mass reaches u times the kept mass.  temperature 0 takes the first.  Each setting is a
    number, or a tensor by row (f32; top_k int32).  Returns int32 [n_rows]; -1 for a row whose
    logits are all -inf or NaN."""
    _rows("logits", logits, 2, *_DTYPE)
    rows = logits.shape[0]
    if u.dim() != 1 or u.dtype != torch.float64 or not u.is_contiguous() or u.shape[0] != rows:
        _refuse(f"u must be a contiguous float64 tensor of {rows} elements")
    device = logits.device
    each, one = [], []
    for name, v, kind in (("temperature", temperature, torch.float32), ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32),
                          ("top_k", top_k, torch.int32)):
        if isinstance(v, torch.Tensor):
            if v.dtype != kind or v.dim() != 1 or not v.is_contiguous() or v.shape[0] != rows or v.device != device:
                _refuse(f"{name} must be a number or a contiguous {kind} tensor of {rows} elements on {device}")
            each.append(v.data_ptr())
            one.append(0)
        else:
            each.append(0)
            one.append(v)
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=device)
    _ints("out", out, rows)
    _same_place(device, u=u, out=out)
    if not -2**31 <= one[3] < 2**31:
        _refuse(f"top_k {one[3]} does not fit 32 bits")
    args = _SAMPLE.pack(logits.data_ptr(), u.data_ptr(), *each, out.data_ptr(), logits.stride(0), one[0], one[1], one[2], int(one[3]),
                        _DTYPE[logits.dtype], rows, logits.shape[1], 0, 0)
    fn = _library().vx_sample_logits
    if device.index == torch.cuda.current_device():
        _call(fn, args, device)
    else:
        with _on(device):
            _call(fn, args, device)
    return out
