"""The ends of what the serving operators take, on the CPU: gradients and tangents, numbers that do not fit,
sizes whose sums would not fit 32 bits."""
import pytest

from test_ops_refusals import F16, P, _append, _attend, _c, _cache, ops  # noqa: F401

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("call,name", [("rope_append_kv", n) for n in ("q", "k", "v", "rope_freq", "k_pages")]
                         + [("shared_prefix_attention", n) for n in ("q", "k_pages", "v_pages")])
def test_tangents_are_refused(vx, call, name):
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        a = _append() if call == "rope_append_kv" else _attend()
        a[name] = fwd.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(vx.VoxtralError, match=f"{name} has a tangent"):
            getattr(vx, call)(**a)
        del a[name]


@pytest.mark.parametrize("name", ["logits", "u", "temperature", "top_p", "min_p"])
def test_sample_refuses_tangents_and_gradients(vx, name):
    import torch.autograd.forward_ad as fwd
    a = dict(logits=torch.zeros(2, 9), u=torch.zeros(2, dtype=torch.float64), temperature=torch.ones(2), top_p=torch.ones(2), min_p=torch.ones(2))
    with fwd.dual_level():
        b = dict(a)
        b[name] = fwd.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(vx.VoxtralError, match="has a tangent"):
            vx.sample_logits(b.pop("logits"), b.pop("u"), **b)
    a[name] = a[name].clone().requires_grad_()
    with pytest.raises(vx.VoxtralError, match="requires a gradient"):
        vx.sample_logits(a["logits"], a["u"], **{k: v for k, v in a.items() if k not in ("logits", "u")})
    with torch.no_grad(), pytest.raises(vx.VoxtralError, match="CUDA device"):
        vx.sample_logits(a["logits"], a["u"], **{k: v for k, v in a.items() if k not in ("logits", "u")})


def test_append_refuses_gradients_of_frequencies(vx):
    freq = torch.zeros(32, requires_grad=True)
    with pytest.raises(vx.VoxtralError, match="rope_freq requires a gradient"):
        vx.rope_append_kv(**_append(rope_freq=freq))
    with torch.no_grad(), pytest.raises(vx.VoxtralError, match="CUDA device"):
        vx.rope_append_kv(**_append(rope_freq=freq))


@pytest.mark.parametrize("kw,word", [(dict(top_k=2.5), "top_k 2.5"), (dict(top_k=float("nan")), "top_k nan"), (dict(top_k=None), "top_k None"),
                                     (dict(top_k=2**31), "32 bits"), (dict(temperature="warm"), "temperature warm"),
                                     (dict(min_p=None), "min_p None"), (dict(top_p=10**400), "top_p 1000"), (dict(top_k=50.0), "CUDA device")])
def test_sample_refuses_numbers(vx, kw, word):
    with pytest.raises(vx.VoxtralError, match=word):
        vx.sample_logits(torch.zeros(2, 9), torch.zeros(2, dtype=torch.float64), **kw)


@pytest.mark.parametrize("value,word", [(30.5, "prefix_len 30.5"), (None, "prefix_len None"), (2**31, "prefix_len 2147483648"),
                                        (float("inf"), "prefix_len inf"), (30.0, "CUDA device"), (torch.tensor(30), "CUDA device")])
def test_attend_refuses_prefix_lengths(vx, value, word):
    with pytest.raises(vx.VoxtralError, match=word):
        vx.shared_prefix_attention(**_attend(prefix_len=value))


@pytest.mark.parametrize("prefix,pages,code,word", [(2**30, 2**26, -4, "together"), (2**30, 2**26 - 15, -4, "together"),
                                                    (2**30, 2**26 - 16, -2, "CUDA"), (1, 2**26, -2, "CUDA")])
def test_attend_positions_fit_32_bits(ops, prefix, pages, code, word):
    """2^30 prefix keys and 2^30 own ones have a last position that no int holds (pages may repeat, so no
    such memory is needed).  The calls that fit get as far as looking for a device."""
    if torch.cuda.is_available():
        pytest.skip("made-up addresses")
    a = dict(q=P, out=2 * P, qs=256, qh=64, os=256, oh=64, ppages=P, table=P, suffix=P, cu=0, status=0, ws=0, wsb=0, tstride=1, n_tokens=2, seqs=2,
             heads=4, prefix=prefix, pages=pages, scale=0.125)
    rc, msg = _c(ops, "vx_shared_prefix_attention", ops._PREFIX.pack(*_cache(), *a.values()))
    assert rc == code and word in msg, (rc, msg)


def test_attend_refuses_its_queries_as_output(ops):
    """Some rows' results would be written while other warps still read their queries."""
    a = dict(q=P, out=P, qs=256, qh=64, os=256, oh=64, ppages=P, table=P, suffix=P, cu=0, status=0, ws=0, wsb=0, tstride=1, n_tokens=2, seqs=2,
             heads=4, prefix=30, pages=1, scale=0.125)
    rc, msg = _c(ops, "vx_shared_prefix_attention", ops._PREFIX.pack(*_cache(), *a.values()))
    assert rc == -1 and "overlap" in msg, (rc, msg)
