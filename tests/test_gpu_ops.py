"""The serving operators on torch tensors (rope_append_kv, shared_prefix_attention, sample_logits)
against plain float64 implementations.

Tolerances.  u = finfo(type).eps / 2 is half a step of the output type.
- append: the value is rounded once (u |y|, or half the smallest step of f16), after a rotation in
  f32 whose cosine, sine, two products and sum are each off by at most 2^-23 or so of |a| + |b|:
  4 * 2^-23 (|a| + |b|) covers them with the angle's own 2^-24 of a turn.
- attention: with A = sum_p w_p |v_p| / l the weights' rounding gives u A, the output's u |o|.  A
  score is a dot product of D exact products added in f32, off by less than (D + 2) 2^-23 sum |q k|
  scale, the exponential adds 2^-22, and an error d of every score moves o by at most 2 d A; sums of n
  weights add n 2^-24 A.  f16 weights below 2^-14 are off by up to 2^-25 each: n 2^-25 max|v| / l, with
  l counted in the largest weight.
- sampling: indices are equal; every draw is required to lie further from the boundaries that decide
  it than the arithmetic of either side is off.  The operator's masses are whole multiples of 2^-44,
  each off by half of one, of weights that are off by a few units of the last place (2^-45 of themselves
  with the division by the temperature); the float64 running sums here are off by 2^-53 of the total a
  token.  So with n tokens, all as shares of the total mass M (in largest weights):
  - S_j >= p S_n (top-p): off by at most n 2^-45 / M for each of S_j and p S_n, n 2^-53 and 2^-45;
  - S_j >= u S_l (the draw, l the last kept token) says S_l - S_j <= (1 - u) S_l, and the tokens up to
    j cancel on the left: (l - j + 1) (2^-45 / M + 2^-53) there, and (1 - u) times n 2^-45 / M + n 2^-53 + 2^-45
    on the right, 2^-52 for u itself.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
BAD_INDEX = 5


def rand(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def pool(n, kv, page, d, dtype, token_major=False, fill=math.nan):
    shape = (n, page, kv, d) if token_major else (n, kv, page, d)
    p = torch.full(shape, fill, dtype=dtype, device="cuda")
    return p.transpose(1, 2) if token_major else p


def freqs(rot):
    return (1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / max(rot, 1))).float()


# ------------------------------------------------------------------------------- append
def rotated(x, pos, freq, interleaved):
    """(float64 rotation, |a| + |b| of each value's pair)"""
    x = x.double()
    rot = 2 * len(freq)
    y, mag = x.clone(), torch.zeros_like(x)
    i = torch.arange(len(freq), device="cuda")
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + len(freq))
    ang = (pos.double()[:, None] * freq.double())[:, None]
    y[..., a] = x[..., a] * ang.cos() - x[..., b] * ang.sin()
    y[..., b] = x[..., a] * ang.sin() + x[..., b] * ang.cos()
    mag[..., a] = mag[..., b] = x[..., a].abs() + x[..., b].abs()
    assert rot <= x.shape[-1]
    return y, mag


def check_rounded(got, want, mag):
    u = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == F16 else 0.0
    tol = u * want.abs() + 4 * 2.0 ** -23 * mag * (1 + u) + tiny
    assert torch.all((got.double() - want).abs() <= tol), float(((got.double() - want).abs() - tol).max())


APPEND = [  # io, cache, interleaved, heads, kv, dim, rot, page, token_major, lengths, starts
    (F32, F16, True, 32, 8, 128, 128, 64, False, [1], [617]),
    (F16, F16, False, 8, 8, 64, 64, 16, True, [5, 1, 33], [0, 1048575, 15]),
    (BF16, BF16, True, 12, 4, 128, 64, 32, False, [2, 70], [31, 199999]),
    (BF16, F16, False, 7, 1, 48, 32, 16, True, [17], [16]),
    (F16, BF16, True, 3, 3, 256, 0, 128, False, [3, 130], [127, 1]),
    (F32, BF16, False, 40, 2, 512, 512, 1, False, [2, 3], [7, 0]),
    (F16, F16, True, 0, 5, 80, 80, 24, False, [50], [23]),
]


@pytest.mark.parametrize("io,cache,inter,heads,kv,dim,rot,page,tm,lens,starts", APPEND)
def test_append(vx, io, cache, inter, heads, kv, dim, rot, page, tm, lens, starts):
    seq = sum(([b] * n for b, n in enumerate(lens)), []) + [0]
    pos = sum(([s + i for i in range(n)] for s, n in zip(starts, lens)), []) + [-1]      # the last row is padding
    n = len(pos)
    used = [list(range(s // page, (s + k - 1) // page + 1)) for s, k in zip(starts, lens)]
    total = sum(map(len, used)) + 2
    order = np.random.default_rng(n).permutation(total)
    table = np.zeros((len(lens), max(u[-1] for u in used) + 1), np.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, u] = order[at:at + len(u)]
        at += len(u)
    qkv = rand(n, (heads + 2 * kv) * dim, dtype=io, seed=n)                  # rows as a fused projection leaves them
    q, k, v = (qkv[:, a * dim:b * dim].view(n, b - a, dim) for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    kp, vp = pool(total, kv, page, dim, cache, tm, fill=7.0), pool(total, kv, page, dim, cache, tm, fill=7.0)
    out = torch.full((n, heads, dim), 7.0, dtype=cache, device="cuda")
    st = ints([0])
    tab, seqs, posn, fr = torch.from_numpy(table).cuda(), ints(seq), ints(pos), freqs(rot)
    r = vx.rope_append_kv(q if heads else None, k, v, kp, vp, tab, seqs, posn, fr, interleaved=inter, q_out=out if heads else None, status=st)
    assert int(st) == 0 and (r is out if heads else r is None)
    live = posn >= 0
    page_of = tab[seqs[live].long(), (posn[live] // page).long()].long()
    slot = (posn[live] % page).long()
    y, mag = rotated(k[live], posn[live], fr, inter)
    check_rounded(kp[page_of, :, slot], y, mag)
    check_rounded(vp[page_of, :, slot], v[live].double(), torch.zeros_like(mag))
    if heads:
        y, mag = rotated(q[live], posn[live], fr, inter)
        check_rounded(out[live], y, mag)
        assert torch.all(out[~live] == 7.0)                                  # padding: left as it was
    kp[page_of, :, slot] = 7.0
    vp[page_of, :, slot] = 7.0
    assert torch.all(kp == 7.0) and torch.all(vp == 7.0)                     # nothing else is written


def test_append_rotates_by_other_positions(vx):
    kp, vp = pool(2, 2, 16, 64, BF16, fill=7.0), pool(2, 2, 16, 64, BF16, fill=7.0)
    q, k, v = rand(3, 4, 64, dtype=BF16, seed=1), rand(3, 2, 64, dtype=BF16, seed=2), rand(3, 2, 64, dtype=BF16, seed=3)
    turn = ints([700, -5, 10_000_000])
    out = vx.rope_append_kv(q, k, v, kp, vp, ints([[1]]), ints([0, 0, 0]), ints([0, 15, 7]), freqs(64), rope_positions=turn)
    for x, got in ((q, out), (k, kp[1][:, [0, 15, 7]].transpose(0, 1))):
        y, mag = rotated(x, turn, freqs(64), True)
        check_rounded(got, y, mag)


def test_append_in_place_and_bad_indices(vx):
    kp, vp = pool(3, 2, 16, 64, F16, fill=7.0), pool(3, 2, 16, 64, F16, fill=7.0)
    q, k, v = rand(5, 4, 64, dtype=F16, seed=1), rand(5, 2, 64, dtype=F16, seed=2), rand(5, 2, 64, dtype=F16, seed=3)
    before = q.clone()
    # sequence 0 has page 2; then a page past the pool, a position past the table, sequences that do not exist
    table, st = ints([[2, 3], [-1, 0]]), ints([0])
    vx.rope_append_kv(q, k, v, kp, vp, table, ints([0, 0, 0, 2, -1]), ints([3, 16, 32, 0, 0]), freqs(64), q_out=q, status=st)
    assert int(st) == BAD_INDEX
    y, mag = rotated(before[:1], ints([3]), freqs(64), True)
    check_rounded(q[:1], y, mag)
    assert torch.equal(q[1:], before[1:])
    y, mag = rotated(k[:1], ints([3]), freqs(64), True)
    check_rounded(kp[2, :, 3][None], y, mag)
    kp[2, :, 3] = 7.0
    assert torch.all(kp == 7.0)


def test_append_nothing(vx):
    e = torch.empty((0, 2, 64), dtype=F16, device="cuda")
    kp, vp = pool(1, 2, 16, 64, F16), pool(1, 2, 16, 64, F16)
    assert vx.rope_append_kv(e, e, e, kp, vp, ints([[0]]), ints([]), ints([]), freqs(64)).shape == e.shape


# ------------------------------------------------------------------------------- attention
def attend_inputs(lens, prefix, heads, kv, d, page, dtype, token_major, seed=0, peaky=1.0):
    """lens: (query tokens, own keys) by sequence.  Slots that hold no key are NaN."""
    held = [-(-s // page) for _, s in lens]
    shared = -(-prefix // page)
    total = shared + sum(held) + 1
    order = np.random.default_rng(seed + 1).permutation(total).astype(np.int32)
    kp, vp = pool(total, kv, page, d, dtype, token_major), pool(total, kv, page, d, dtype, token_major)
    table = np.full((len(lens), max(held + [1])), 0, np.int32)
    at = shared
    keys = []
    for b, ((_, s), h) in enumerate(zip(lens, held)):
        table[b, :h] = order[at:at + h]
        keys.append((order[at:at + h], s))
        at += h
    for i, (pages, s) in enumerate([(order[:shared], prefix)] + keys):
        if s:
            p = torch.from_numpy(pages.astype(np.int64)).cuda()
            for w, x in ((0, kp), (1, vp)):
                full = torch.full((len(pages) * page, kv, d), math.nan, dtype=dtype, device="cuda")
                full[:s] = rand(s, kv, d, dtype=dtype, seed=seed * 1000 + 2 * i + w)
                x[p] = full.view(len(pages), page, kv, d).transpose(1, 2)
    t = sum(n for n, _ in lens)
    q = rand(t + 2, heads, d, dtype=dtype, seed=seed + 77, scale=peaky)      # two rows behind the last sequence
    cu = ints(np.concatenate([[0], np.cumsum([n for n, _ in lens])]).tolist())
    return q, kp, vp, torch.from_numpy(order[:shared]).cuda(), torch.from_numpy(table).cuda(), ints([s for _, s in lens]), cu


def attend_reference(q, kp, vp, ppages, prefix, table, lens, scale):
    """(float64 output, tolerance) of the rows of the sequences."""
    heads, d = q.shape[1:]
    kv = kp.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    outs, tols = [], []
    t = 0
    for b, (n, s) in enumerate(lens):
        pages = torch.cat((ppages.long(), table[b, :-(-s // kp.shape[2])].long()))
        k, v = (torch.cat((x[ppages.long()].transpose(0, 1).flatten(1, 2)[:, :prefix],
                           x[pages[len(ppages):]].transpose(0, 1).flatten(1, 2)[:, :s]), 1).double() for x in (kp, vp))
        x = q[t:t + n].double().unflatten(1, (kv, heads // kv))
        t += n
        sc = torch.einsum("ikgd,kpd->ikgp", x, k) * scale
        off = (d + 2) * 2.0 ** -23 * scale * torch.einsum("ikgd,kpd->ikgp", x.abs(), k.abs())
        seen = torch.arange(prefix + s, device="cuda") <= prefix + s - n + torch.arange(n, device="cuda")[:, None]
        seen = seen[:, None, None]
        sc, off = torch.where(seen, sc, -math.inf), torch.where(seen, off, 0.0)
        m = sc.amax(-1, keepdim=True) if prefix + s else torch.zeros(*sc.shape[:-1], 1, device="cuda").double()
        w = torch.where(seen, (sc - m).exp(), 0.0)
        total = w.sum(-1, keepdim=True).clamp_min(1e-300)
        some = seen.any(-1, keepdim=True)
        o = torch.where(some, torch.einsum("ikgp,kpd->ikgd", w, v) / total, 0.0)
        a = torch.einsum("ikgp,kpd->ikgd", w, v.abs()) / total
        count = prefix + s
        delta = (off.amax(-1, keepdim=True) if count else torch.zeros_like(total)) + 2.0 ** -22
        tol = u * (a + o.abs()) + 2 * delta * a + 2 * count * 2.0 ** -24 * a + 1e-30
        if q.dtype == F16 and count:
            tol += count * 2.0 ** -25 * v.abs().amax() / total.clamp_min(1.0) + 2.0 ** -25
        outs.append(torch.where(some, o, 0.0).reshape(n, heads, d))
        tols.append(torch.where(some, tol, 1e-30).reshape(n, heads, d))
    return torch.cat(outs), torch.cat(tols)


def check_attend(vx, lens, prefix, heads, kv, d, page, dtype, token_major=False, scale=None, seed=0, peaky=1.0, ragged=None):
    q, kp, vp, ppages, table, suffix, cu = attend_inputs(lens, prefix, heads, kv, d, page, dtype, token_major, seed, peaky)
    t = sum(n for n, _ in lens)
    ragged = any(n != 1 for n, _ in lens) if ragged is None else ragged
    out, st = torch.full_like(q, 7.0), ints([0])
    if ragged:
        vx.shared_prefix_attention(q, kp, vp, ppages, prefix, table, suffix, cu_q=cu, scale=scale, out=out, status=st)
    else:
        vx.shared_prefix_attention(q[:t], kp, vp, ppages, prefix, table, suffix, scale=scale, out=out[:t], status=st)
    assert int(st) == 0
    want, tol = attend_reference(q[:t], kp, vp, ppages, prefix, table, lens, scale or d ** -0.5)
    diff = (out[:t].double() - want).abs()
    assert torch.all(diff <= tol), (float((diff - tol).max()), float(diff.max()))
    assert torch.all(out[t:] == 7.0)                                         # rows of no sequence are left as they were
    return out


ATTEND = [  # lens, prefix, heads, kv, dim, page, type, token_major
    ([(1, 0)], 1, 4, 1, 128, 64, F16, False),
    ([(1, 1)], 0, 1, 1, 64, 16, BF16, False),
    ([(1, 0), (1, 7)], 0, 8, 2, 128, 16, F16, True),                          # a sequence without any key
    ([(1, 40), (1, 0), (1, 17), (1, 1)], 617, 32, 8, 128, 64, F16, False),
    ([(1, 3), (1, 500)], 127, 12, 4, 64, 32, BF16, True),
    ([(1, 129)] * 33, 128, 5, 5, 128, 128, F16, False),                       # one query head a K/V head
    ([(1, 20), (1, 65)], 130, 9, 1, 128, 256, BF16, False),                   # 9 query heads a K/V head
    ([(1, 2)], 1000, 40, 2, 64, 16, F16, True),                               # 20
    ([(1, 300)], 257, 48, 1, 128, 32, F16, False),                            # 48
    ([(1, 1 + 37 * i % 90) for i in range(70)], 1300, 16, 4, 64, 64, F16, False),
    ([(1, 9)] * 5, 9001, 8, 2, 128, 16, BF16, True),
    ([(3, 3), (1, 9), (0, 4), (16, 20), (7, 100)], 33, 8, 2, 128, 16, F16, True),
    ([(5, 2), (4, 0)], 3, 4, 2, 64, 16, F16, False),                          # queries that stand inside the prefix
    ([(6, 2), (1, 0)], 1, 4, 2, 128, 16, BF16, False),                        # queries before any key
    ([(150, 163), (2, 2), (131, 131)], 129, 8, 2, 128, 64, BF16, False),
    ([(64, 70)], 2500, 4, 1, 64, 32, F16, True),
    ([(33, 290), (0, 0), (1, 1), (260, 260)], 0, 6, 3, 128, 16, F16, False),
    ([(600, 600)], 64, 7, 7, 64, 64, BF16, False),
    ([(40, 47), (90, 95)], 515, 40, 2, 128, 128, F16, False),
    # ragged rows that take a long prefix together, then their own keys by rows or by tiles
    ([(1 + 7 * i % 41, 1 + 7 * i % 41 + 13 * i % 50) for i in range(14)], 3001, 32, 8, 128, 64, F16, False),
    ([(1 + 5 * i % 30, 3 * i % 17) for i in range(30)], 2600, 24, 8, 64, 16, BF16, True),   # some stand inside the prefix
    ([(90, 101), (70, 70), (0, 3), (83, 200), (100, 50)], 2300, 32, 8, 128, 32, BF16, False),
    ([(3, 0), (64, 0), (1, 0), (20, 0)], 4000, 32, 8, 128, 128, F16, False),               # no own keys at all
    ([(1, 1 + i % 3) for i in range(400)], 0, 8, 8, 128, 16, F16, False),                    # many short sequences
    ([(1, 0 if i % 7 else 40) for i in range(500)], 300, 16, 4, 64, 16, BF16, False),
]


@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attend(vx, case):
    check_attend(vx, *ATTEND[case], seed=case)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("peaky", [0.0, 12.0])
def test_attend_flat_and_peaked(vx, dtype, peaky):
    """Equal weights everywhere, and rows in which a few keys hold everything, whose running maximum
    keeps growing."""
    check_attend(vx, [(1, 77), (1, 0), (1, 300)], 1111, 16, 4, 128, 64, dtype, seed=3, peaky=peaky)
    check_attend(vx, [(70, 90), (45, 45)], 400, 16, 4, 128, 64, dtype, seed=4, peaky=peaky)


def test_attend_one_token_with_and_without_offsets(vx):
    lens = [(1, 5), (1, 64), (1, 0)]
    a = check_attend(vx, lens, 200, 8, 2, 128, 64, F16, seed=5, ragged=False)
    b = check_attend(vx, lens, 200, 8, 2, 128, 64, F16, seed=5, ragged=True)
    assert (a[:3].float() - b[:3].float()).abs().max() < 2e-3                 # each is within its bound of the same values


def test_attend_scale_and_strides(vx):
    check_attend(vx, [(1, 30), (1, 3)], 50, 8, 2, 64, 16, F16, seed=6, scale=0.31)
    q, kp, vp, ppages, table, suffix, _ = attend_inputs([(1, 30), (1, 3)], 50, 8, 2, 64, 16, F16, False, seed=6)
    want = vx.shared_prefix_attention(q[:2], kp, vp, ppages, 50, table, suffix)
    wide = torch.zeros((2, 3, 8, 72), dtype=F16, device="cuda")
    wide[:, 1, :, :64] = q[:2]
    out = torch.full((2, 8, 128), 7.0, dtype=F16, device="cuda")
    big = torch.zeros((2, 9), dtype=torch.int32, device="cuda")
    big[:, 3:3 + table.shape[1]] = table
    r = vx.shared_prefix_attention(wide[:, 1, :, :64], kp, vp, ppages, 50, big[:, 3:3 + table.shape[1]], suffix, out=out[:, :, 64:])
    assert torch.equal(r, want) and torch.all(out[:, :, :64] == 7.0)


def test_attend_bad_pages_and_offsets(vx):
    """What only the device sees is reported; nothing is read out of range and no other row changes."""
    lens = [(1, 30), (1, 20), (1, 10)]
    q, kp, vp, ppages, table, suffix, cu = attend_inputs(lens, 100, 8, 2, 128, 16, F16, False, seed=8)
    good = vx.shared_prefix_attention(q[:3], kp, vp, ppages, 100, table, suffix)
    for entry in (-1, kp.shape[0], 2**31 - 1):
        bad, st = table.clone(), ints([0])
        bad[1, 1] = entry
        r = vx.shared_prefix_attention(q[:3], kp, vp, ppages, 100, bad, suffix, status=st)
        assert int(st) == BAD_INDEX
        assert torch.equal(r[0], good[0]) and torch.equal(r[2], good[2]) and bool(torch.isfinite(r[1]).all())
    st = ints([0])
    more = suffix.clone()
    more[2] = 10**9                                                           # more keys than the table's row holds
    r = vx.shared_prefix_attention(q[:3], kp, vp, ppages, 100, table, more, status=st)
    assert int(st) == BAD_INDEX and torch.equal(r[:2], good[:2])
    st = ints([0])
    broken = ppages.clone()
    broken[2] = -5
    assert bool(torch.isfinite(vx.shared_prefix_attention(q[:3], kp, vp, broken, 100, table, suffix, status=st)).all())
    assert int(st) == BAD_INDEX
    st = ints([0])
    vx.shared_prefix_attention(q[:3], kp, vp, ppages, 100, table, suffix, cu_q=ints([0, 1, 2, 900]), status=st)
    assert int(st) == BAD_INDEX


def test_attend_nothing(vx):
    q, kp, vp, ppages, table, suffix, _ = attend_inputs([(1, 3)], 20, 4, 2, 64, 16, F16, False)
    assert vx.shared_prefix_attention(q[:0], kp, vp, ppages, 20, table[:0], suffix[:0]).shape == (0, 4, 64)


def test_attend_is_the_same_every_time(vx):
    q, kp, vp, ppages, table, suffix, _ = attend_inputs([(1, 9 * i) for i in range(40)], 3000, 16, 4, 128, 64, BF16, False, seed=9)
    a = vx.shared_prefix_attention(q[:40], kp, vp, ppages, 3000, table, suffix)
    for _ in range(5):
        assert torch.equal(a, vx.shared_prefix_attention(q[:40], kp, vp, ppages, 3000, table, suffix))


# ------------------------------------------------------------------------------- sampling
def sample_reference(row, u, temperature, top_k, top_p, min_p):
    """(index, slack): slack is the least distance, in shares of the mass, of a running sum from a
    boundary that decided the index, less what the arithmetic may be off there."""
    x = np.where(np.isnan(row), -np.inf, row.astype(np.float64)) + 0.0
    if not np.any(x > -np.inf):
        return -1, 1.0
    if temperature <= 0:
        return int(np.argmax(x)), 1.0
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temperature))
    slack = float(np.min(np.abs(w - min_p))) - 2.0 ** -45 if 0 < min_p < 1 else 1.0
    w = w[w >= max(min_p, 1e-300)]
    w = w[:top_k] if top_k > 0 else w
    n, sums = len(w), np.cumsum(w)
    unit = 2.0 ** -45 / sums[-1] + 2.0 ** -53
    last = n - 1
    if 0 < top_p < 1:
        goal = top_p * sums[-1]
        last = min(int(np.searchsorted(sums, goal)), last)
        off = np.abs(sums[max(0, last - 1):last + 1] - goal) / sums[-1]
        slack = min(slack, float(np.min(off)) - 2 * n * unit - 2.0 ** -45)
    elif top_p <= 0:
        last = 0
    goal = u * sums[last]
    at = min(int(np.searchsorted(sums, goal)), last)
    for i in (at - 1, at):
        if 0 <= i < last:
            allowed = (last - i + 1) * unit + (1 - u) * (n * unit + 2.0 ** -45) + 2.0 ** -52
            slack = min(slack, abs(sums[i] - goal) / sums[-1] - allowed)
    # weights that are all 1 have exact sums on both sides, and p S rounds alike at either scale (a
    # power of two apart), so a draw may land on a boundary
    return int(order[at]), 1.0 if np.all(w == 1.0) else slack


def check_sample(vx, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    got = vx.sample_logits(logits, torch.from_numpy(u).cuda(), temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p).cpu().numpy()
    host = logits.double().cpu().numpy()
    # a number counts as an f32 array of that value
    each = [v.cpu().numpy() if torch.is_tensor(v) else [np.float32(v)] * len(u) for v in (temperature, top_k, top_p, min_p)]
    for r in range(len(u)):
        want, slack = sample_reference(host[r], u[r], float(each[0][r]), int(each[1][r]), float(each[2][r]), float(each[3][r]))
        assert slack > 0 or u[r] == 0, r
        assert got[r] == want, (r, got[r], want)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 0, 0.9, 0.0), (0.7, 40, 1.0, 0.0), (1.3, 0, 1.0, 0.05), (0.9, 1000, 0.95, 0.001), (1.0, 1, 0.5, 0.0),
            (0.5, 5000, 0.999, 0.0), (0.0, 0, 0.9, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (5.0, 0, 0.7, 0.0)]


@pytest.mark.parametrize("n", [1, 2, 31, 1000, 8320, 32768, 32769, 70001, 131072, 262144])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_sample_sizes_and_settings(vx, n, dtype):
    rng = np.random.default_rng(n)
    for i, (t, k, p, m) in enumerate(SETTINGS if n <= 40000 or dtype != F16 else SETTINGS[:3]):
        u = np.concatenate([[0.0, 1.0 - 2.0 ** -53], rng.random(3)])
        check_sample(vx, rand(5, n, dtype=dtype, seed=n + i, scale=2.5), u, t, k, p, m)


def test_sample_wide_and_narrow_batches(vx):
    rng = np.random.default_rng(3)
    for rows, n in ((150, 20000), (40, 70001), (300, 1000)):
        check_sample(vx, rand(rows, n, seed=rows, scale=1.0), rng.random(rows), 0.9, 0, 0.9, 0.0)


def test_sample_settings_by_row(vx):
    rng = np.random.default_rng(4)
    n = len(SETTINGS)
    cols = [torch.tensor([s[i] for s in SETTINGS], device="cuda") for i in range(4)]
    check_sample(vx, rand(n, 9000, seed=5, scale=2.0), rng.random(n), cols[0], cols[1].int(), cols[2], cols[3])


@pytest.mark.parametrize("n", [5000, 50000])
def test_sample_ties(vx, n):
    """Runs of equal logits longer than any list: the order inside one is the index order."""
    rng = np.random.default_rng(n)
    flat = torch.zeros((6, n), device="cuda")
    flat[3:] = torch.round(rand(3, n, seed=6))
    flat[1, ::2] = -0.0                                                        # -0 and 0 are one value
    flat[2, : n // 2] = -math.inf
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, n // 2 + 7, 1.0, 0.0), (1.0, 0, 0.61803, 0.0), (0.8, 2100, 0.9, 0.01)):
        check_sample(vx, flat, rng.random(6) * 0.9999 + 0.00003, t, k, p, m)
    near = (1.0 + 1e-6 * rand(4, n, seed=7)).float()                           # many values inside one bin
    check_sample(vx, near, rng.random(4), 1.0, 0, 0.7, 0.0)
    check_sample(vx, 1e-30 * rand(4, n, seed=8), rng.random(4), 1.0, n // 3, 0.7, 0.0)


def test_sample_infinities_and_nan(vx):
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf] * 6, [nan] * 6, [nan, -inf, 3.0, nan, -inf, -inf], [inf, 1.0, inf, 2.0, -inf, nan],
                      [-3.4e38, 3.4e38, 0, 0, 0, 0], [-3.4e38] * 6], device="cuda")
    u = np.array([0.3, 0.3, 0.9, 0.7, 0.99, 0.4])
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.5, 3, 0.9, 0.1), (0.0, 0, 1.0, 0.0)):
        got = vx.sample_logits(x, torch.from_numpy(u).cuda(), temperature=t, top_k=k, top_p=p, min_p=m).tolist()
        assert got[:2] == [-1, -1] and got[2] == 2 and got[4] == 1
        assert got[3] == (0 if t == 0 else 2) and got[5] == (0 if t == 0 else 2 if k == 0 else 1)


def test_sample_strides_and_out(vx):
    big = rand(4, 3, 777, seed=9)
    u = torch.rand(4, dtype=torch.float64, device="cuda")
    out = torch.full((4,), -9, dtype=torch.int32, device="cuda")
    r = vx.sample_logits(big[:, 1, 5:700], u, top_p=0.9, out=out)
    assert r is out and torch.equal(out, vx.sample_logits(big[:, 1, 5:700].contiguous(), u, top_p=0.9))
    one = vx.sample_logits(big[:1, 0].expand(4, 777), u, top_p=0.9)            # one row, four draws
    assert torch.equal(one, vx.sample_logits(big[:1, 0].repeat(4, 1), u, top_p=0.9))
    assert vx.sample_logits(big[0, :0], u[:0]).shape == (0,)


def test_sample_numbers_are_arrays_of_one_value(vx):
    x, u = rand(64, 131072, seed=12, scale=1.5), torch.rand(64, dtype=torch.float64, device="cuda")
    full = [torch.full((64,), v, device="cuda") for v in (0.8, 0.95, 0.001)]
    a = vx.sample_logits(x, u, temperature=0.8, top_p=0.95, min_p=0.001)
    assert torch.equal(a, vx.sample_logits(x, u, temperature=full[0], top_p=full[1], min_p=full[2]))


def test_sample_follows_the_distribution(vx):
    """20000 draws of one row: counts within 6 standard deviations of the kept masses."""
    x = torch.tensor([1.0, 0.5, 2.0, -1.0, 0.0, -30.0], device="cuda")
    n = 20000
    u = torch.rand(n, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    got = torch.bincount(vx.sample_logits(x.expand(n, 6), u, min_p=0.06).long(), minlength=6).cpu().numpy()
    w = np.exp(x.double().cpu().numpy() - 2.0)
    w[w < 0.06] = 0
    w /= w.sum()
    assert np.all(np.abs(got - n * w) <= 6 * np.sqrt(n * w * (1 - w)) + 1e-9)


# ------------------------------------------------------------------------------- together
class Step:
    """A decode step of a small batch over shared pages: append, attend, project, draw."""

    def __init__(self, vx, seqs=6, prefix=83, heads=8, kv=2, d=64, page=16, vocab=5000, dtype=F16):
        self.vx, self.prefix, self.heads, self.kv, self.d, self.page, self.dtype = vx, prefix, heads, kv, d, page, dtype
        shared = -(-prefix // page)
        self.kp, self.vp = pool(shared + seqs * 4, kv, page, d, dtype), pool(shared + seqs * 4, kv, page, d, dtype)
        self.ppages = ints(list(range(shared)))
        self.table = ints([[shared + 4 * b + i for i in range(4)] for b in range(seqs)])
        self.freq, self.seq, self.u = freqs(d), ints(list(range(seqs))), torch.zeros(seqs, dtype=torch.float64, device="cuda")
        self.lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.pos = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.qkv = torch.zeros((seqs, heads + 2 * kv, d), dtype=dtype, device="cuda")
        self.w = rand(heads * d, vocab, dtype=dtype, seed=11, scale=0.2)
        # the shared prompt: its own "sequence" of the prefix pages
        k, v = rand(prefix, kv, d, dtype=dtype, seed=12), rand(prefix, kv, d, dtype=dtype, seed=13)
        vx.rope_append_kv(None, k, v, self.kp, self.vp, self.ppages[None], ints([0] * prefix), ints(list(range(prefix))), self.freq)

    def fill(self, n, seed):
        self.lens.fill_(n + 1)
        self.pos.fill_(n)                       # own keys count from the first own page
        self.qkv.copy_(rand(*self.qkv.shape, dtype=self.dtype, seed=seed))
        self.u.copy_(torch.rand(len(self.u), dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)))

    def run(self):
        h, kv = self.heads, self.kv
        q, k, v = self.qkv[:, :h], self.qkv[:, h:h + kv], self.qkv[:, h + kv:]
        q = self.vx.rope_append_kv(q, k, v, self.kp, self.vp, self.table, self.seq, self.pos, self.freq,
                                   rope_positions=self.pos + self.prefix)
        o = self.vx.shared_prefix_attention(q, self.kp, self.vp, self.ppages, self.prefix, self.table, self.lens)
        logits = o.flatten(1) @ self.w
        return q, o, logits, self.vx.sample_logits(logits, self.u, temperature=0.9, top_k=300, top_p=0.97)

    def check(self, q, o, logits, tok):
        lens = [(1, int(n)) for n in self.lens]
        want, tol = attend_reference(q, self.kp, self.vp, self.ppages, self.prefix, self.table, lens, self.d ** -0.5)
        assert torch.all((o.double() - want).abs() <= tol)
        for r in range(len(lens)):
            idx, slack = sample_reference(logits[r].double().cpu().numpy(), float(self.u[r]), float(np.float32(0.9)), 300, float(np.float32(0.97)), 0.0)
            assert slack > 0 and int(tok[r]) == idx


def test_serving_steps(vx):
    s = Step(vx)
    for n in range(20):
        s.fill(n, 100 + n)
        s.check(*s.run())


def test_serving_step_captured_and_replayed(vx):
    """The step as one CUDA graph, replayed with other contents; a second graph of the same step
    and an eager step in between share nothing with it."""
    s, other = Step(vx), Step(vx, seqs=3, prefix=700, dtype=BF16)
    side = torch.cuda.Stream()
    graphs = []
    for x in (s, other):
        x.fill(0, 1)
        x.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            r = x.run()
        graphs.append((g, r))
    for n in range(8):
        for x, (g, r) in zip((s, other), graphs):
            x.fill(n, 200 + n)
            g.replay()
            x.check(*r)
        tok = graphs[0][1][3].clone()
        assert torch.equal(s.run()[3], tok)


def test_operators_on_several_streams(vx):
    steps = [Step(vx, seqs=4 + i, prefix=50 + 300 * i) for i in range(3)]
    streams = [torch.cuda.Stream() for _ in steps]
    for n in range(6):
        for i, x in enumerate(steps):
            x.fill(n, 300 + 10 * n + i)
        torch.cuda.synchronize()
        res = []
        for x, st in zip(steps, streams):
            with torch.cuda.stream(st):
                res.append(x.run())
        torch.cuda.synchronize()
        for x, r in zip(steps, res):
            x.check(*r)


def test_operators_captured_as_their_first_call(vx):
    """In a fresh process nothing has been set up yet when the capture begins."""
    import os
    import subprocess
    import sys
    code = """
import importlib, torch
vx = importlib.import_module("webgpu-voxtral_b200")
c = dict(device="cuda")
kp, vp = torch.zeros(90, 8, 64, 128, dtype=torch.float16, **c), torch.randn(90, 8, 64, 128, **c).half()
q, k = torch.randn(64, 32, 128, **c).half(), torch.randn(64, 8, 128, **c).half()
i32 = lambda v: torch.tensor(v, dtype=torch.int32, **c)
pp, table, pos, seq = i32(list(range(20))), i32([[20 + b] for b in range(64)]), i32([0] * 64), i32(list(range(64)))
fr, u = torch.ones(64, **c), torch.full((64,), 0.5, dtype=torch.float64, **c)
w = torch.randn(4096, 40000, **c).half()
def step():
    r = vx.rope_append_kv(q, k, k, kp, vp, table, seq, pos, fr)
    o = vx.shared_prefix_attention(r, kp, vp, pp, 1280, table, pos + 1)
    x = vx.shared_prefix_attention(r, kp, vp, pp, 1280, table, pos + 1, cu_q=i64)
    return r, o, x, vx.sample_logits(o.flatten(1) @ w, u, top_p=0.9)
i64 = i32(list(range(65)))
torch.zeros(1, **c) @ torch.zeros(1, **c)
g = torch.cuda.CUDAGraph()
s = torch.cuda.Stream()
with torch.cuda.stream(s):
    torch.zeros(64, 4096, **c).half() @ w       # the library's own workspace
torch.cuda.synchronize()
with torch.cuda.graph(g, stream=s):
    a = step()
g.replay()
torch.cuda.synchronize()
b = step()
assert all(torch.equal(x, y) for x, y in zip(a[:2], b[:2])) and (a[1].float() - a[2].float()).abs().max() < 2e-2
print("same")
"""
    root = os.path.dirname(os.path.dirname(vx.library_path()))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_attend_without_own_pages(vx):
    """A page table of no columns: the prefix alone, through each kernel that may take it."""
    for seqs, prefix in ((2, 100), (64, 2000)):
        q, kp, vp, ppages, table, suffix, cu = attend_inputs([(1, 0)] * seqs, prefix, 32, 8, 128, 64, F16, False, seed=seqs)
        want, tol = attend_reference(q[:seqs], kp, vp, ppages, prefix, table, [(1, 0)] * seqs, 128 ** -0.5)
        for kw in ({}, {"cu_q": cu}):
            got = vx.shared_prefix_attention(q[:seqs], kp, vp, ppages, prefix, table[:, :0], suffix, **kw)
            assert torch.all((got.double() - want).abs() <= tol)


def test_attend_workspace(vx):
    q, kp, vp, ppages, table, suffix, _ = attend_inputs([(1, 30), (1, 3)], 500, 8, 2, 64, 16, F16, False, seed=6)
    need = vx.shared_prefix_attention_workspace(q[:2], kp, vp, ppages, 500, table, suffix)
    want = vx.shared_prefix_attention(q[:2], kp, vp, ppages, 500, table, suffix)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")               # NaN in every float
    assert torch.equal(want, vx.shared_prefix_attention(q[:2], kp, vp, ppages, 500, table, suffix, workspace=ws))
    with pytest.raises(vx.VoxtralError, match="workspace"):
        vx.shared_prefix_attention(q[:2], kp, vp, ppages, 500, table, suffix, workspace=ws[:need - 1])
    with pytest.raises(vx.VoxtralError, match="workspace"):
        vx.shared_prefix_attention(q[:2], kp, vp, ppages, 500, table, suffix, workspace=torch.empty(need + 64, dtype=torch.uint8, device="cuda")[1:])
