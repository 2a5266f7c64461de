"""What the serving operators refuse, on the CPU: the Python checks with CPU tensors and the C ABI's
with arguments that it must turn down before any launch."""
import ctypes
import struct

import pytest

torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops(vx):
    import importlib
    return importlib.import_module("webgpu-voxtral_b200.ops")


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


def test_argument_structs_have_the_header_s_sizes(ops, tmp_path, vx):
    import os
    import subprocess
    src = tmp_path / "s.c"
    src.write_text('#include "voxtral_b200.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu %zu %zu", sizeof(vx_rope_append_args), '
                   'sizeof(vx_shared_prefix_args), sizeof(vx_sample_args), offsetof(vx_shared_prefix_args, workspace)); return 0; }')
    inc = os.path.join(os.path.dirname(os.path.dirname(vx.library_path())), "include")
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(tmp_path / "s")], check=True)
    want = [int(x) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout.split()]
    assert [ops._APPEND.size, ops._PREFIX.size, ops._SAMPLE.size] == want[:3]
    assert struct.calcsize("@" + ops._CACHE + "2P4q5P") == want[3]


def _append(**kw):
    a = dict(q=torch.zeros(3, 4, 64, dtype=F16), k=torch.zeros(3, 2, 64, dtype=F16), v=torch.zeros(3, 2, 64, dtype=F16),
             k_pages=torch.zeros(5, 2, 16, 64, dtype=F16), v_pages=torch.zeros(5, 2, 16, 64, dtype=F16), page_table=ints([[0, 1]]),
             seq_ids=ints([0, 0, 0]), positions=ints([0, 1, 2]), rope_freq=torch.zeros(32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,word", [
    ({}, "CUDA device"),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.float64)), "k must be one of"),
    (dict(v=torch.zeros(3, 2, 64, dtype=BF16)), "v must be one of"),
    (dict(q=torch.zeros(4, 4, 64, dtype=F16)), "does not fit k"),
    (dict(k_pages=torch.zeros(5, 2, 16, 64, dtype=F32)), "k_pages must be one of"),
    (dict(v_pages=torch.zeros(6, 2, 16, 64, dtype=F16)), "one shape"),
    (dict(k_pages=torch.zeros(5, 3, 16, 64, dtype=F16), v_pages=torch.zeros(5, 3, 16, 64, dtype=F16)), "do not fit a cache"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "positions must be"),
    (dict(seq_ids=ints([0, 0])), "seq_ids must have 3"),
    (dict(rope_positions=ints([0, 0])), "rope_positions must have 3"),
    (dict(page_table=ints([0, 1])), "page_table must be"),
    (dict(q_out=torch.zeros(3, 4, 64, dtype=BF16)), "q_out must be one of"),
    (dict(k=torch.zeros(3, 64, 2, dtype=F16).transpose(1, 2)), "last dimension"),
    (dict(q=torch.zeros(3, 4, 64, dtype=F16, requires_grad=True)), "requires a gradient"),
])
def test_append_refuses(vx, kw, word):
    with pytest.raises(vx.VoxtralError, match=word):
        vx.rope_append_kv(**_append(**kw))


def _attend(**kw):
    a = dict(q=torch.zeros(2, 4, 64, dtype=F16), k_pages=torch.zeros(5, 2, 16, 64, dtype=F16), v_pages=torch.zeros(5, 2, 16, 64, dtype=F16),
             prefix_pages=ints([0, 1]), prefix_len=30, page_table=ints([[2], [3]]), suffix_lens=ints([1, 2]))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,word", [
    ({}, "CUDA device"),
    (dict(q=torch.zeros(2, 4, 64, dtype=BF16)), "q must be one of"),
    (dict(q=torch.zeros(2, 4, 128, dtype=F16)), "head_dim 64"),
    (dict(prefix_len=33), "does not fit 2 pages"),
    (dict(prefix_len=-1), "does not fit"),
    (dict(suffix_lens=ints([1])), "suffix_lens must have 2"),
    (dict(cu_q=ints([0, 1])), "cu_q must have 3"),
    (dict(out=torch.zeros(2, 4, 64, dtype=F32)), "out must be one of"),
    (dict(out=torch.zeros(3, 4, 64, dtype=F16)), "q's shape"),
    (dict(q=torch.zeros(2, 4, 64, dtype=F16, requires_grad=True)), "requires a gradient"),
])
def test_attend_refuses(vx, kw, word):
    with pytest.raises(vx.VoxtralError, match=word):
        vx.shared_prefix_attention(**_attend(**kw))


@pytest.mark.parametrize("kw,word", [
    ({}, "CUDA device"),
    (dict(logits=torch.zeros(2, 9, dtype=torch.float64)), "logits must be one of"),
    (dict(logits=torch.zeros(9)), "2 dimensions"),
    (dict(u=torch.zeros(2)), "u must be"),
    (dict(u=torch.zeros(3, dtype=torch.float64)), "u must be"),
    (dict(top_k=torch.zeros(2)), "top_k must be"),
    (dict(temperature=torch.zeros(3)), "temperature must be"),
    (dict(top_k=2**40), "CUDA device|32 bits"),
    (dict(out=torch.zeros(2)), "out must be"),
])
def test_sample_refuses(vx, kw, word):
    a = dict(logits=torch.zeros(2, 9), u=torch.zeros(2, dtype=torch.float64))
    a.update(kw)
    with pytest.raises(vx.VoxtralError, match=word):
        vx.sample_logits(a.pop("logits"), a.pop("u"), **a)


# ---- the C ABI: made-up addresses, so a call that is not refused would fail at the launch only
P = 1 << 20


def _c(ops, fn, args):
    err = ctypes.create_string_buffer(256)
    rc = getattr(ops._library(), fn)(args, None, err, 256)
    return rc, err.value.decode()


def _cache(**kw):
    c = dict(k=P, v=P, kp=2048, kh=1024, ks=64, vp=2048, vh=1024, vs=64, n=5, kv=2, page=16, d=64, dtype=0)
    c.update(kw)
    return [*c.values(), 0]


@pytest.mark.parametrize("cache,change,code,word", [
    (dict(k=0), {}, -1, "k and v"),
    (dict(dtype=2), {}, -1, "dtype 2"),
    (dict(n=0), {}, -4, "0 pages"),
    (dict(k=P + 8), {}, -1, "16-byte"),
    (dict(vs=60), {}, -1, "16-byte"),
    (dict(kh=-1024), {}, -1, "negative"),
    (dict(d=72), {}, -4, "head_dim 72"),
    (dict(d=528), {}, -4, "head_dim 528"),
    ({}, dict(rot=80), -4, "rot_dim"),
    ({}, dict(rot=24), -4, "rot_dim"),
    ({}, dict(dtype=3), -1, "dtype 3"),
    ({}, dict(n_tokens=-1), -4, "-1 tokens"),
    ({}, dict(k=0), -1, "device pointers"),
    ({}, dict(freq=0), -1, "device pointers"),
    ({}, dict(q=P + 2), -1, "16-byte"),
    ({}, dict(qs=68), -1, "16-byte"),
    ({}, dict(n_tokens=0), 0, ""),
])
def test_append_c_refuses(ops, cache, change, code, word):
    a = dict(q=P, k=P, v=P, q_out=P, qs=256, qh=64, kst=128, kh=64, vst=128, vh=64, os=256, oh=64, table=P, seq=P, pos=P, rpos=0, freq=P, status=0,
             tstride=4, dtype=0, n_tokens=3, heads=4, n_seqs=1, max_pages=2, rot=64, inter=1, reserved=0)
    a.update(change)
    rc, msg = _c(ops, "vx_rope_append_kv", ops._APPEND.pack(*_cache(**cache), *a.values()))
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("cache,change,code,word", [
    (dict(d=96), {}, -4, "head_dim 96"),
    (dict(page=8), {}, -4, "page_size 8"),
    (dict(page=48), {}, -4, "page_size 48"),
    (dict(page=512), {}, -4, "page_size 512"),
    ({}, dict(heads=5), -4, "multiple"),
    ({}, dict(heads=0), -4, "multiple"),
    ({}, dict(prefix=-1), -4, "prefix_len"),
    ({}, dict(prefix=2**30 + 1), -4, "prefix_len"),
    ({}, dict(pages=2**29), -4, "own keys"),
    ({}, dict(scale=0.0), -4, "scale"),
    ({}, dict(scale=float("nan")), -4, "scale"),
    ({}, dict(scale=float("inf")), -4, "scale"),
    ({}, dict(n_tokens=3), -1, "cu_q is needed"),
    ({}, dict(q=0), -1, "device pointers"),
    ({}, dict(ppages=0), -1, "device pointers"),
    ({}, dict(out=P + 8), -1, "16-byte"),
    ({}, dict(oh=68), -1, "16-byte"),
    ({}, dict(n_tokens=0, seqs=0), 0, ""),
])
def test_attend_c_refuses(ops, cache, change, code, word):
    a = dict(q=P, out=P, qs=256, qh=64, os=256, oh=64, ppages=P, table=P, suffix=P, cu=0, status=0, ws=0, wsb=0, tstride=1, n_tokens=2, seqs=2,
             heads=4, prefix=30, pages=1, scale=0.125)
    a.update(change)
    args = ops._PREFIX.pack(*_cache(**cache), *a.values())
    rc, msg = _c(ops, "vx_shared_prefix_attention", args)
    assert rc == code and word in msg, (rc, msg)
    if code:
        assert ops._library().vx_shared_prefix_attention_workspace(args) in (0, ) or word in ("device pointers", "16-byte")


@pytest.mark.parametrize("change,code,word", [
    (dict(dtype=7), -1, "dtype 7"),
    (dict(n=0), -4, "0 logits"),
    (dict(n=262145), -4, "262145"),
    (dict(stride=-1), -4, "stride -1"),
    (dict(t=-0.5), -4, "temperature"),
    (dict(t=float("nan")), -4, "temperature"),
    (dict(top_p=-0.1), -4, "top_p"),
    (dict(top_p=float("nan")), -4, "top_p"),
    (dict(min_p=1.5), -4, "min_p"),
    (dict(logits=0), -1, "device pointers"),
    (dict(logits=P + 1), -1, "aligned"),
    (dict(rows=0), 0, ""),
])
def test_sample_c_refuses(ops, change, code, word):
    a = dict(logits=P, u=P, tp=0, topp=0, minp=0, topk=0, out=P, stride=9, t=1.0, top_p=1.0, min_p=0.0, k=0, dtype=0, rows=2, n=9, reserved=0)
    a.update(change)
    rc, msg = _c(ops, "vx_sample_logits", ops._SAMPLE.pack(*a.values()))
    assert rc == code and word in msg, (rc, msg)


def test_null_arguments(ops):
    for fn in ("vx_rope_append_kv", "vx_shared_prefix_attention", "vx_sample_logits"):
        rc, msg = _c(ops, fn, None)
        assert rc == -1 and "null" in msg
    assert ops._library().vx_shared_prefix_attention_workspace(None) == 0
