"""The serving operators at the edges of what their documentation allows, and just past them: malformed
offsets, lengths past a page table, settings at the ends of their range, page tables wider than needed.

Tolerances and plain float64 forms are those of test_gpu_ops.py unless a test says otherwise."""
import math

import numpy as np
import pytest

from test_gpu_ops import BAD_INDEX, BF16, F16, F32, attend_inputs, attend_reference, check_sample, ints, rand

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

MARGIN = 1 << 16


def attend_in_margins(vx, *args, fill=0, **kw):
    """shared_prefix_attention with a workspace of the least size between bytes that have to stay as they are."""
    need = vx.shared_prefix_attention_workspace(*args, **{k: v for k, v in kw.items() if k == "cu_q"})
    ws = torch.full((need + 2 * MARGIN,), 0xA5, dtype=torch.uint8, device="cuda")
    ws[MARGIN:MARGIN + need] = fill
    out = vx.shared_prefix_attention(*args, workspace=ws[MARGIN:MARGIN + need], **kw)
    assert bool((ws[:MARGIN] == 0xA5).all()) and bool((ws[MARGIN + need:] == 0xA5).all())
    return out


OFFSETS = [  # (query tokens, own keys) of each sequence's cache, offsets, sequences in front of the bad one, prefix, dtype
    ([(64, 70)] + [(0, 9)] * 63, [0, 64] * 32 + [0], 1, 0, F16),              # every second sequence decreases: by rows
    ([(64, 70)] + [(0, 9)] * 63, [0, 64] * 32 + [0], 1, 2000, BF16),          # ... with the prefix by tiles
    ([(100, 120), (0, 40), (0, 40), (100, 100)], [0, 100, 50, 200, 200], 1, 0, F16),    # whole sequences by tiles
    ([(100, 120), (0, 40), (0, 40), (100, 100)], [0, 100, 50, 200, 200], 1, 700, BF16),
    ([(3, 5), (4, 9), (0, 30)], [2, 5, 9, 4], 2, 40, F16),                    # the last one goes down
    ([(3, 5), (4, 9), (0, 30)], [0, 3, 7, 900], 2, 40, F16),                  # past the batch
    ([(3, 5), (4, 9), (0, 30)], [0, 3, 900, 7], 1, 40, BF16),
    ([(3, 5), (4, 9), (2, 30)], [-1, 3, 6, 8], 0, 40, F16),                   # before it
    ([(3, 5), (4, 9), (2, 30)], [-2**31, 2**31 - 1, 0, 3], 0, 40, F16),
    ([(100, 0), (80, 0), (60, 0)], [0, 100, 180, 90], 2, 700, F16),           # the prefix alone
]


@pytest.mark.parametrize("case", range(len(OFFSETS)))
def test_attend_offsets_out_of_order(vx, case):
    """The sequences in front of the first bad offset are computed, the others refused; nothing is
    written outside the workspace, nor into the refused ones' rows, whatever the workspace holds."""
    lens, cu, held, prefix, dtype = OFFSETS[case]
    q, kp, vp, ppages, table, suffix, _ = attend_inputs(lens, prefix, 32, 8, 128, 16, dtype, False, seed=case)
    n = max([200 if len(lens) == 4 else 64 if len(lens) == 64 else 9] + cu[:held + 1])
    first = max(cu[0], 0)
    q = torch.cat((q, q[:1].expand(max(0, n + 2 - len(q)), -1, -1)))[:n + 2]
    if not any(s for _, s in lens):
        table = table[:, :0]
    out, st = torch.full_like(q, 7.0), ints([0])
    attend_in_margins(vx, q[:n], kp, vp, ppages, prefix, table, suffix, cu_q=ints(cu), out=out[:n], status=st)
    assert int(st) == BAD_INDEX
    want, tol = attend_reference(q[first:], kp, vp, ppages, prefix, table, lens[:held], 128 ** -0.5) if held else (q[:0], q[:0])
    end = first + len(want)
    assert end == (cu[held] if held else first)
    off = (out[first:end].double() - want).abs() - tol
    assert held == 0 or float(off.max()) <= 0
    assert bool((out[:first] == 7.0).all()) and bool((out[end:] == 7.0).all())     # no sequence's rows, and refused ones'


@pytest.mark.parametrize("seqs,each", [(2, 1), (64, 1), (700, 1), (5, 30), (3, 130)])
@pytest.mark.parametrize("prefix", [90, 2500])
def test_attend_lengths_past_a_table_of_no_columns(vx, seqs, each, prefix):
    """Own keys that no page holds are reported and left out, whichever kernels take the prefix."""
    lens = [(each, 0)] * seqs
    q, kp, vp, ppages, table, suffix, cu = attend_inputs(lens, prefix, 16, 4, 64, 16, BF16, False, seed=seqs)
    q, kw = q[:seqs * each], {} if each == 1 else {"cu_q": cu}
    want, tol = attend_reference(q, kp, vp, ppages, prefix, table, lens, 64 ** -0.5)
    for bad in (None, seqs - 1, 0):
        s, st = suffix.clone(), ints([0])
        if bad is not None:
            s[bad] = 3
        got = vx.shared_prefix_attention(q, kp, vp, ppages, prefix, table[:, :0], s, status=st, **kw)
        assert int(st) == (0 if bad is None else BAD_INDEX)
        assert float(((got.double() - want).abs() - tol).max()) <= 0

@pytest.mark.parametrize("cols", [128, 512, 2048])
def test_attend_wide_page_tables(vx, cols):
    """A table as wide as the longest context that a server allows, of which short answers use little: the
    results, and (the workspace holds a partial for each key range) about as many ranges as with a table
    cut to length."""
    lens, prefix = [(1, 1 + 7 * i % 300) for i in range(64)], 32768
    q, kp, vp, ppages, table, suffix, _ = attend_inputs(lens, prefix, 32, 8, 128, 64, F16, False, seed=cols)
    wide = torch.full((64, cols), -1, dtype=torch.int32, device="cuda")        # the rest is no page
    wide[:, :table.shape[1]] = table
    st = ints([0])
    got = vx.shared_prefix_attention(q[:64], kp, vp, ppages, prefix, wide, suffix, status=st)
    want, tol = attend_reference(q[:64], kp, vp, ppages, prefix, table, lens, 128 ** -0.5)
    assert int(st) == 0 and float(((got.double() - want).abs() - tol).max()) <= 0
    need = [vx.shared_prefix_attention_workspace(q[:64], kp, vp, ppages, prefix, t, suffix) for t in (table, wide)]
    assert need[1] >= 0.75 * need[0]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("path", ["rows", "shared", "own"])
@pytest.mark.parametrize("e", [26.0, 26.3])
def test_attend_long_tails(vx, dtype, path, e):
    """2^20 equal keys, each at 2^-e of one strong key: by themselves below the steps of an f16 weight,
    together 1.5 % of the result.  The strong key's value is 0, the others' 1: o = n w / (1 + n w).  The
    batches are wide enough for each row to take (nearly) all keys in one range, the strong one among them.

    A weight is off by 2^-32 of the largest (f16) and by half a step of its type; a score by (d + 2) 2^-23 of itself, the
    exponential by 2^-22; the sums of weights and of products, 16 keys at a time, by 2^16 2^-23 each."""
    n, page, d = 1 << 20, 256, 64
    kp, vp = torch.zeros((n // page + 1, 1, page, d), dtype=dtype, device="cuda"), torch.ones((n // page + 1, 1, page, d), dtype=dtype, device="cuda")
    kp[7, 0, 11, 0], vp[7, 0, 11] = 4.0, 0.0
    pages = torch.arange(n // page + 1, dtype=torch.int32, device="cuda")
    seqs, each, heads = {"rows": (2072, 1, 1), "shared": (592, 1, 64), "own": (148, 64, 1)}[path]
    q = torch.zeros((seqs * each, heads, d), dtype=dtype, device="cuda")
    q[..., 0] = 8.0
    scale = float(np.float32(e * math.log(2) / 32.0))
    keys = torch.full((seqs,), n + 1, dtype=torch.int32, device="cuda")
    if path == "shared":
        o = vx.shared_prefix_attention(q, kp, vp, pages, n + 1, torch.zeros((seqs, 0), dtype=torch.int32, device="cuda"), keys * 0, scale=scale)
    else:
        cu = torch.arange(0, seqs * each + 1, each, dtype=torch.int32, device="cuda") if path == "own" else None
        o = vx.shared_prefix_attention(q, kp, vp, pages[:0], 0, pages[None].expand(seqs, -1), keys, cu_q=cu, scale=scale)
    u = torch.finfo(dtype).eps / 2
    for i in {0, each - 1}:                                                    # query i of each sequence
        nw = (n - (each - 1 - i)) * math.exp(-32.0 * scale)
        want = nw / (1 + nw)
        tol = n * 2.0 ** -32 * (dtype == F16) + want * (2 * u + 2 * (d + 2) * 2.0 ** -23 * 32 * scale + 2 * 2.0 ** -22 + 2 * 2.0 ** -7)
        assert float((o[i::each].double() - want).abs().max()) <= tol


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("each,own,prefix", [(1, 37, 700), (1, 90, 0), (70, 130, 0), (20, 33, 3000)])
def test_append_and_attend_in_one_layer_of_a_cache(vx, dtype, each, own, prefix):
    """K and V as views of one allocation [page][layer][K or V][head][slot][64]: pages lie far apart, and all
    other layers stay as they are."""
    seqs, heads, kv, d, page, layers, layer = 4, 8, 2, 64, 16, 3, 1
    shared, held = -(-prefix // page), -(-own // page)
    order = np.random.default_rng(own).permutation(shared + seqs * held + 2).astype(np.int32)
    buf = torch.full((len(order), layers, 2, kv, page, d), math.nan, dtype=dtype, device="cuda")
    kp, vp = buf[:, layer, 0], buf[:, layer, 1]
    ppages = torch.from_numpy(order[:shared]).cuda()
    table = torch.from_numpy(order[shared:shared + seqs * held].reshape(seqs, held)).cuda()
    # every key of the prefix and of the sequences goes in through the append, its rotation left out
    k, v = rand(prefix + seqs * own, kv, d, dtype=dtype, seed=1), rand(prefix + seqs * own, kv, d, dtype=dtype, seed=2)
    rows = [[0] * prefix, [b for b in range(seqs) for _ in range(own)]]
    where = [list(range(prefix)), list(range(own)) * seqs]
    for at, tab, seq, pos in ((0, ppages[None], rows[0], where[0]), (prefix, table, rows[1], where[1])):
        st = ints([0])
        vx.rope_append_kv(None, k[at:at + len(seq)], v[at:at + len(seq)], kp, vp, tab, ints(seq), ints(pos),
                          torch.zeros(0, device="cuda"), status=st)
        assert int(st) == 0
    assert torch.equal(kp[order[shared], :, 0], k[prefix])
    lens = [(each, own)] * seqs
    q = rand(seqs * each, heads, d, dtype=dtype, seed=3)
    kw = {} if each == 1 else {"cu_q": ints([each * b for b in range(seqs + 1)])}
    got = vx.shared_prefix_attention(q, kp, vp, ppages, prefix, table, ints([own] * seqs), **kw)
    want, tol = attend_reference(q, kp, vp, ppages, prefix, table, lens, d ** -0.5)
    assert float(((got.double() - want).abs() - tol).max()) <= 0
    buf[:, layer] = math.nan
    assert bool(torch.isnan(buf).all())


def test_attend_one_chunk_among_single_tokens(vx):
    lens = [(512, 600)] + [(1, 1 + 17 * b % 300) for b in range(40)]
    for prefix, dtype in ((0, F16), (1500, BF16)):
        q, kp, vp, ppages, table, suffix, cu = attend_inputs(lens, prefix, 16, 4, 64, 16, dtype, False, seed=prefix)
        got = vx.shared_prefix_attention(q[:552], kp, vp, ppages, prefix, table, suffix, cu_q=cu)
        want, tol = attend_reference(q[:552], kp, vp, ppages, prefix, table, lens, 64 ** -0.5)
        assert float(((got.double() - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("seqs,prefix,each", [(3, 50, 1), (64, 2000, 1), (3, 200, 90)])
def test_attend_over_broadcast_heads(vx, seqs, prefix, each):
    """One K/V head expanded to four (a head stride of 0) gives what four copies of it give."""
    lens = [(each, each + 9 * b % 70) for b in range(seqs)]
    q, kp, vp, ppages, table, suffix, cu = attend_inputs(lens, prefix, 8, 1, 64, 16, F16, False, seed=seqs)
    q, kw = q[:seqs * each], {} if each == 1 else {"cu_q": cu}
    wide = [x.expand(-1, 4, -1, -1) for x in (kp, vp)]
    got = vx.shared_prefix_attention(q, *wide, ppages, prefix, table, suffix, **kw)
    want = vx.shared_prefix_attention(q, *(x.contiguous() for x in wide), ppages, prefix, table, suffix, **kw)
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------- sampling
@pytest.mark.parametrize("temperature", [1.4e-45, 1e-41, 1.2e-38, 1e-37, 1.9e-37, 1e-36, 1e-30, 1e-20])
@pytest.mark.parametrize("n", [2, 600, 40000])
def test_sample_lowest_temperatures(vx, temperature, n):
    """Logits a few temperatures apart, where dividing by so small a number overflows, and far apart."""
    rng = np.random.default_rng(n)
    t = float(np.float32(temperature))
    x = -(rand(6, n, seed=n).abs().double() * 12 * t).float()
    x[3:5] = -torch.round(rand(2, n, seed=n + 1).abs() * 3) * t                # many equal ones
    x[5] = rand(1, n, seed=n + 2)[0]
    x[:, n // 2] = 0.0
    for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.0), (5, 1.0, 0.0), (0, 0.8, 0.3), (0, 1.0, 1.0), (1000, 0.97, 0.001)):
        u = rng.random(6) * 0.9999 + 0.00003
        check_sample(vx, x, u, temperature, k, p, m)
        by_row = [torch.full((6,), v, device="cuda") for v in (temperature, p, m)]
        check_sample(vx, x, u, by_row[0], k, by_row[1], by_row[2])
    check_sample(vx, x.to(BF16), rng.random(6) * 0.9999 + 0.00003, temperature, 0, 0.9, 0.0)


def test_sample_low_temperatures_by_row(vx):
    rng = np.random.default_rng(1)
    t = torch.tensor([1e-45, 1e-38, 1e-37, 1e-30, 1e-4, 1.0, 0.0, 3e38], device="cuda", dtype=F32)
    for n in (700, 30000):
        check_sample(vx, rand(8, n, seed=n), rng.random(8), t, 0, 0.95, 0.0)
        check_sample(vx, rand(8, n, seed=n) * t[:, None].clamp(max=1.0), rng.random(8), t.clamp(max=1e30), 0, 0.95, 0.0)


@pytest.mark.parametrize("seqs,heads", [(1, 8), (70, 8), (3, 520)])
def test_sample_right_behind_the_kernel_that_writes_its_logits(vx, seqs, heads):
    """Attention lets the next kernel start before it is done; the draw must see what it wrote.  The same
    buffers again and again with other contents, so that anything old shows."""
    q, kp, vp, ppages, table, suffix, _ = attend_inputs([(1, 1 + b % 40) for b in range(seqs)], 300, heads, 8, 128, 16, F16, False, seed=seqs)
    q, u = q[:seqs], torch.full((seqs,), 0.5, dtype=torch.float64, device="cuda")
    out = torch.empty_like(q)
    args = [(q * (1 + 0.1 * i)).contiguous() for i in range(8)]
    got, want = [], []
    for x in args:
        vx.shared_prefix_attention(x, kp, vp, ppages, 300, table, suffix, out=out)
        got.append(vx.sample_logits(out.flatten(1), u, temperature=0.01, top_p=0.9))
        want.append(out.clone())
    torch.cuda.synchronize()
    for g, o in zip(got, want):
        assert torch.equal(g, vx.sample_logits(o.flatten(1), u, temperature=0.01, top_p=0.9))
