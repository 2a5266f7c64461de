"""The serving operators on the caller's device memory, as workloads: one decode or prefill step
of a batch that decodes over a paged K/V cache.

- append: rotary positions on q and k, and k / v appended to a paged cache (rope_append_kv);
- attend: attention of a batch whose sequences share a long prefix (shared_prefix_attention);
- sample: min-p, top-k, top-p and a draw from given random numbers (sample_logits).

`run` computes them from elementary torch operations where `own` is false, and through the
package's entry points where it is true; `exact` computes them again in 64 bits.
"""
import importlib
import math
import random

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_THETA = 1e6     # rope base of the package's backbone
_vx = None


def _package():
    global _vx
    if _vx is None:
        _vx = importlib.import_module("webgpu-voxtral_b200")
    return _vx


# ------------------------------------------------------------------------------------ cases
def _append(name, **kw):
    c = {"op": "append", "batch": 1, "new_min": 1, "new_max": 1, "context": 2048, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "io": "f16", "cache": "f16", "interleaved": True, "token_major": False, "padding": 0}
    return dict(c, name=name, **kw) if name else dict(c, **kw)


def _attend(name, **kw):
    c = {"op": "attend", "batch": 1, "q_min": 1, "q_max": 1, "prefix": 617, "suffix_min": 0, "suffix_max": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "f16", "token_major": False}
    return dict(c, name=name, **kw) if name else dict(c, **kw)


def _sample(name, **kw):
    c = {"op": "sample", "rows": 1, "vocab": 8320, "type": "f32", "spread": 2.5, "masked": 0, "temperature": 0.8, "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "by_row": False}
    return dict(c, name=name, **kw) if name else dict(c, **kw)


def listed():
    return [
        # one utterance's next frame: one token, f32 activations, f16 cache (the smallest call)
        _append("append one token", io="f32"),
        # 64 utterances in lockstep, each at its own position; the batch is padded to 72 rows
        _append("append batch 64", batch=64, context=2117, io="bf16", cache="bf16", padding=8),
        # prompts of many lengths prefilled together, K/V in a token-major cache of small pages
        _append("append ragged prefill", batch=24, new_min=17, new_max=1200, context=32768, io="f16", page=16, token_major=True,
                interleaved=False),
        # four utterances just after a 617-position prompt that they share
        _attend("attend batch 4", batch=4, suffix_max=40),
        # 64 utterances of one voice, each up to 1500 frames past the 617 shared positions
        _attend("attend batch 64", batch=64, suffix_min=1, suffix_max=1500, type="bf16"),
        # the long-context form: 32768 shared positions, short answers
        _attend("attend long prefix", batch=64, prefix=32768, suffix_min=1, suffix_max=300),
        # a wide batch over a long prefix, more query heads per K/V head, smaller pages
        _attend("attend wide batch", batch=250, prefix=8191, suffix_min=0, suffix_max=200, heads=56, kv_heads=7, dim=64, page=32,
                type="bf16"),
        # ragged text chunks prefilled behind the shared prompt
        _attend("attend ragged chunks", batch=16, q_min=1, q_max=150, prefix=2049, suffix_min=0, suffix_max=260, page=16,
                token_major=True),
        # the semantic code of one frame: 8320 logits, ids 0 and from 8194 on masked
        _sample("sample one frame", masked=126, spread=1.0),
        # the same for 64 utterances, each with its own settings
        _sample("sample batch 64", rows=64, masked=126, by_row=True, top_k=64, min_p=0.02),
        # text tokens of a large vocabulary, bf16 logits (many ties), all filters
        _sample("sample vocabulary", rows=64, vocab=131072, type="bf16", top_k=50, top_p=0.95, min_p=0.01),
        # a wide batch with the nucleus alone, over a flat distribution
        _sample("sample wide batch", rows=200, vocab=131072, spread=1.5, top_p=0.95, temperature=1.0),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        a = most.setdefault(c["op"], [0, 0])
        a[0], a[1] = max(a[0], w["bytes"]), max(a[1], w["flops"])
    while True:
        op = rng.choice(["append", "attend", "sample"])
        if op == "sample":
            c = _sample(None, rows=_log(rng, 1, 256), vocab=_log(rng, 200, 131072), type=rng.choice(["f32", "f16", "bf16"]),
                        spread=rng.choice([1.0, 2.0, 4.0]), temperature=round(rng.uniform(0.3, 1.6), 3), top_k=rng.choice([0, 0, _log(rng, 1, 2000)]),
                        top_p=rng.choice([1.0, round(rng.uniform(0.1, 0.999), 4)]), min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.2), 4)]),
                        by_row=rng.random() < 0.3)
        else:
            kv = rng.choice([1, 2, 3, 4, 8])
            dim = rng.choice([64, 128])
            heads = kv * rng.choice([1, 2, 4, 6, 8])
            page = rng.choice([16, 32, 64, 128])
            if op == "append":
                new = _log(rng, 1, 700)
                c = _append(None, batch=_log(rng, 1, 200), new_min=rng.randint(1, new), new_max=new, context=_log(rng, 1, 200000),
                            heads=heads, kv_heads=kv, dim=dim, page=page, io=rng.choice(["f16", "bf16", "f32"]),
                            cache=rng.choice(["f16", "bf16"]), interleaved=rng.random() < 0.5, token_major=rng.random() < 0.4,
                            padding=rng.choice([0, rng.randint(1, 9)]))
            else:
                q = rng.choice([1, 1, 1, _log(rng, 2, 160)])
                suffix = _log(rng, 1, 2500)
                c = _attend(None, batch=_log(rng, 1, 256), q_min=rng.randint(1, q), q_max=q, prefix=rng.choice([0, _log(rng, 1, 33000)]),
                            suffix_min=rng.randint(0, suffix), suffix_max=suffix, heads=heads, kv_heads=kv, dim=dim, page=page,
                            type=rng.choice(["f16", "bf16"]), token_major=rng.random() < 0.4)
        w = work(c)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1] and _scores(c) <= 300e6:
            return c


def _scores(c):
    """Attention weights of the case over padded rows (what the plain form holds at once)."""
    if c["op"] != "attend":
        return 0
    return c["batch"] * c["q_max"] * c["heads"] * (c["prefix"] + c["suffix_max"] + c["q_max"])


def _spread(c, lo, hi, salt):
    """One length per sequence in [lo, hi], both ends among them, the same for every seed."""
    r = random.Random("%s %d %d %d %d" % (salt, c["batch"], lo, hi, c["page"]))
    got = [_log(r, lo + 1, hi + 1) - 1 for _ in range(c["batch"])]
    got[0] = hi
    if len(got) > 1:
        got[-1] = lo
    return got


def _lengths(c):
    """attend: (query tokens, keys past the prefix) of each sequence, its query tokens' own keys among them."""
    n = _spread(c, c["q_min"], c["q_max"], "q")
    return n, [a + b for a, b in zip(n, _spread(c, c["suffix_min"], c["suffix_max"], "s"))]


def work(case):
    c, size = case, {"f16": 2, "bf16": 2, "f32": 4}
    if c["op"] == "append":
        n = sum(_spread(c, c["new_min"], c["new_max"], "n"))
        values = n * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": values * size[c["io"]] + values * 2 + (n + c["padding"]) * 8, "flops": 3 * n * (c["heads"] + c["kv_heads"]) * c["dim"]}
    if c["op"] == "attend":
        nq, ns = _lengths(c)
        kv = (c["prefix"] + sum(ns)) * c["kv_heads"] * c["dim"] * 2 * 2
        pairs = sum(a * (c["prefix"] + s - a) + a * (a + 1) // 2 for a, s in zip(nq, ns))
        return {"bytes": kv + 2 * sum(nq) * c["heads"] * c["dim"] * 2, "flops": 4 * pairs * c["heads"] * c["dim"]}
    return {"bytes": c["rows"] * (c["vocab"] * size[c["type"]] + 12), "flops": 3 * c["rows"] * c["vocab"]}


# ------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)


def _pool(c, n, dtype):
    """Pages [n, kv_heads, page, dim]; token-major pools keep a token's heads next to each other."""
    shape = (n, c["page"], c["kv_heads"], c["dim"]) if c["token_major"] else (n, c["kv_heads"], c["page"], c["dim"])
    p = torch.zeros(shape, dtype=dtype, device="cuda")
    return p.transpose(1, 2) if c["token_major"] else p


def prepare(case, seed):
    return {"append": _prepare_append, "attend": _prepare_attend, "sample": _prepare_sample}[case["op"]](case, seed)


def _prepare_append(c, seed):
    g, r = _gen(seed), random.Random(seed)
    new = _spread(c, c["new_min"], c["new_max"], "n")
    start = [r.randint(0, c["context"]) for _ in new]
    start[0] = c["context"]
    wide = (max(s + n for s, n in zip(start, new)) + c["page"] - 1) // c["page"]
    used = [range(s // c["page"], (s + n - 1) // c["page"] + 1) for s, n in zip(start, new)]
    total = sum((n - 1) // c["page"] + 2 for n in new) + 1     # the same for every seed
    order = list(range(total))
    r.shuffle(order)
    at, table = 0, torch.zeros((c["batch"], wide), dtype=torch.int32)
    for b, u in enumerate(used):
        table[b, u.start:u.stop] = torch.tensor(order[at:at + len(u)], dtype=torch.int32)
        at += len(u)
    seq = [b for b, n in enumerate(new) for _ in range(n)] + [0] * c["padding"]
    pos = [s + i for s, n in zip(start, new) for i in range(n)] + [-1] * c["padding"]
    t, h, kv, d = len(seq), c["heads"], c["kv_heads"], c["dim"]
    qkv = torch.randn((t, (h + 2 * kv) * d), generator=g, device="cuda").to(_TYPES[c["io"]])
    freq = (_THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)).float()
    return {"op": "append", "interleaved": c["interleaved"], "q": qkv[:, :h * d].view(t, h, d), "k": qkv[:, h * d:(h + kv) * d].view(t, kv, d),
            "v": qkv[:, (h + kv) * d:].view(t, kv, d), "k_pages": _pool(c, total, _TYPES[c["cache"]]), "v_pages": _pool(c, total, _TYPES[c["cache"]]),
            "table": table.cuda(), "seq": torch.tensor(seq, dtype=torch.int32).cuda(), "pos": torch.tensor(pos, dtype=torch.int32).cuda(), "freq": freq,
            "q_out": torch.zeros((t, h, d), dtype=_TYPES[c["cache"]], device="cuda")}


def _prepare_attend(c, seed):
    g, r = _gen(seed), random.Random(seed)
    nq, ns = _lengths(c)
    t, h, kv, d, page = sum(nq), c["heads"], c["kv_heads"], c["dim"], c["page"]
    shared, wide = -(-c["prefix"] // page), max(1, -(-max(ns) // page))
    held = [-(-s // page) for s in ns]
    total = shared + sum(held) + 2
    order = list(range(total))
    r.shuffle(order)
    at, table = shared, torch.zeros((c["batch"], wide), dtype=torch.int32)
    for b, n in enumerate(held):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    k, v = _pool(c, total, _TYPES[c["type"]]), _pool(c, total, _TYPES[c["type"]])
    k.normal_(generator=g)
    v.normal_(generator=g)
    qkv = torch.randn((t, (h + 2 * kv) * d), generator=g, device="cuda").mul_(1.5).to(_TYPES[c["type"]])
    cu = torch.tensor([0] + nq, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    return {"op": "attend", "q": qkv[:, :h * d].view(t, h, d), "k_pages": k, "v_pages": v, "prefix": c["prefix"],
            "prefix_pages": torch.tensor(order[:shared], dtype=torch.int32).cuda(), "table": table.cuda(),
            "suffix": torch.tensor(ns, dtype=torch.int32).cuda(), "cu": cu, "one": c["q_max"] == 1, "widest": max(nq), "longest": max(ns)}


def _prepare_sample(c, seed):
    g = _gen(seed)
    x = torch.randn((c["rows"], c["vocab"]), generator=g, device="cuda") * c["spread"]
    x += 3 * c["spread"] * (torch.rand(x.shape, generator=g, device="cuda") < 4 / c["vocab"])   # a few likely ones
    x = x.to(_TYPES[c["type"]])
    if c["masked"]:
        x[:, 0] = -math.inf
        x[:, c["vocab"] - c["masked"]:] = -math.inf
    s = {"op": "sample", "logits": x, "u": torch.rand(c["rows"], generator=g, device="cuda", dtype=torch.float64)}
    for k in ("temperature", "top_k", "top_p", "min_p"):
        s[k] = c[k]
    if c["by_row"]:
        one = torch.rand((4, c["rows"]), generator=g, device="cuda")
        s["temperature"] = 0.5 + one[0]
        s["top_k"] = (one[1] * 2 * c["top_k"]).int()      # 0: no such filter in that row
        s["top_p"] = 0.5 + 0.5 * one[2]
        s["min_p"] = 0.1 * one[3] * (c["min_p"] > 0)
    return s


# ------------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    if s["op"] == "append":
        if own:
            _package().rope_append_kv(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["seq"], s["pos"], s["freq"],
                                      interleaved=s["interleaved"], q_out=s["q_out"])
        else:
            _plain_append(s)
        return s["q_out"], s["k_pages"], s["v_pages"]
    if s["op"] == "attend":
        if own:
            return _package().shared_prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["prefix_pages"], s["prefix"], s["table"],
                                                      s["suffix"], cu_q=None if s["one"] else s["cu"])
        return _plain_attend(s)
    if own:
        return _package().sample_logits(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return _plain_sample(s)


def _plain_append(s):
    live = (s["pos"] >= 0).nonzero()[:, 0]
    pos, seq, page = s["pos"][live].long(), s["seq"][live].long(), s["k_pages"].shape[2]
    angle = pos[:, None].double() * s["freq"].double()          # 64 bits: far positions lose the angle in 32
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x):
        x = x[live].float()
        if s["interleaved"]:
            a, b = x[..., 0::2], x[..., 1::2]
            return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)

    at, slot = s["table"][seq, pos // page].long(), pos % page
    s["q_out"][live] = turn(s["q"]).to(s["q_out"].dtype)
    s["k_pages"][at, :, slot] = turn(s["k"]).to(s["k_pages"].dtype)
    s["v_pages"][at, :, slot] = s["v"][live].float().to(s["v_pages"].dtype)


def _plain_attend(s):
    q, cu, suffix, prefix = s["q"], s["cu"].long(), s["suffix"].long(), s["prefix"]
    t, h, d = q.shape
    batch, kv, most, far = len(suffix), s["k_pages"].shape[1], s["widest"], s["longest"]
    tok = torch.arange(t, device=q.device)
    b = torch.searchsorted(cu, tok, right=True) - 1
    j = tok - cu[b]
    rows = q.new_zeros((batch, most, h, d), dtype=torch.float32)
    rows[b, j] = q.float()
    rows = rows.view(batch, most, kv, h // kv, d).permute(2, 0, 3, 1, 4) / math.sqrt(d)      # [kv, batch, group, query, d]

    def shared(p):
        return p[s["prefix_pages"].long()].transpose(0, 1).flatten(1, 2)[:, :prefix].float()

    def each(p):
        return p[s["table"].long()].transpose(1, 2).flatten(2, 3)[:, :, :far].float()

    left = rows.reshape(kv, -1, d) @ shared(s["k_pages"]).transpose(1, 2)
    right = rows.transpose(0, 1).reshape(batch, kv, -1, d) @ each(s["k_pages"]).transpose(2, 3)
    left, right = left.view(*rows.shape[:4], prefix), right.view(batch, kv, h // kv, most, far).transpose(0, 1)
    # query i of a sequence stands at position (all its keys) - (its queries) + i
    seen = (prefix + suffix - (cu[1:] - cu[:-1]))[:, None] + torch.arange(most, device=q.device) + 1
    key = torch.arange(prefix + far, device=q.device)
    score = torch.cat((left, right), -1).masked_fill_(~(key < seen[..., None])[:, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    score = score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score[..., :prefix].flatten(1, 3) @ shared(s["v_pages"])).view(rows.shape)
    out += (score[..., prefix:].transpose(0, 1).reshape(batch, kv, -1, far) @ each(s["v_pages"])).view(batch, kv, h // kv, most, d).transpose(0, 1)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(1, 3, 0, 2, 4).reshape(batch, most, h, d)[b, j].to(q.dtype)


def _plain_sample(s):
    x = s["logits"].double()         # 64 bits: running sums next to a border decide whole numbers
    rows, n = x.shape

    def by_row(v):
        return torch.as_tensor(v, device=x.device).double().expand(rows)[:, None]

    order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = ((order.values - order.values[:, :1]) / by_row(s["temperature"])).exp()
    w = torch.where(w >= by_row(s["min_p"]), w, 0.0)
    k = by_row(s["top_k"])
    place = torch.arange(n, device=x.device)
    w = torch.where((k <= 0) | (place < k), w, 0.0)
    run_ = w.cumsum(-1)
    kept = (run_ - w < by_row(s["top_p"]) * run_[:, -1:]) & (w > 0)
    mass = torch.where(kept, run_, 0.0).amax(-1, keepdim=True)
    pick = (run_ < s["u"][:, None] * mass).sum(-1).clamp_max(n - 1)
    return order.indices.gather(-1, pick[:, None])[:, 0].int()


# ------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s)


def _exact_append(s):
    page = s["k_pages"].shape[2]
    q_out, k_pages, v_pages = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("q_out", "k_pages", "v_pages"))
    d = s["q"].shape[-1]
    half = torch.arange(d // 2, device="cuda")
    first = 2 * half if s["interleaved"] else half
    second = first + (1 if s["interleaved"] else d // 2)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double()[:, None] * s["freq"].double())[:, None]

    def rotated(x):
        z = torch.complex(x[..., first].double(), x[..., second].double()) * turn
        y = torch.empty(x.shape, dtype=torch.float64, device="cuda")
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = rotated(s["q"]), rotated(s["k"])
    for i, (b, p) in enumerate(zip(s["seq"].tolist(), s["pos"].tolist())) if len(s["pos"]) <= 256 else ():
        if p >= 0:
            q_out[i] = q[i]
            k_pages[s["table"][b, p // page], :, p % page] = k[i]
            v_pages[s["table"][b, p // page], :, p % page] = s["v"][i].double()
    if len(s["pos"]) > 256:
        ok = s["pos"] >= 0
        row = s["table"][s["seq"][ok].long(), (s["pos"][ok] // page).long()].long() * page + (s["pos"][ok] % page).long()
        q_out[ok] = q[ok]
        for pool, new in ((k_pages, k), (v_pages, s["v"].double())):
            flat = torch.zeros((pool.shape[0] * page, *new.shape[1:]), dtype=torch.float64, device="cuda")
            flat[row] = new[ok]
            pool.copy_(flat.view(pool.shape[0], page, *new.shape[1:]).transpose(1, 2))
    return q_out, k_pages, v_pages


def _exact_attend(s):
    q, prefix = s["q"].double(), s["prefix"]
    t, h, d = q.shape
    kv = s["k_pages"].shape[1]
    out = torch.zeros((t, h, d), dtype=torch.float64, device="cuda")
    lead = [p[s["prefix_pages"].long()].permute(1, 0, 2, 3).flatten(1, 2)[:, :prefix].double() for p in (s["k_pages"], s["v_pages"])]
    cu = s["cu"].tolist()
    for b, n in enumerate(s["suffix"].tolist()):
        held = -(-n // s["k_pages"].shape[2])
        k, v = (torch.cat((a, p[s["table"][b, :held].long()].permute(1, 0, 2, 3).flatten(1, 2)[:, :n].double()), 1)
                for a, p in zip(lead, (s["k_pages"], s["v_pages"])))
        x = q[cu[b]:cu[b + 1]].unflatten(1, (kv, h // kv))                       # [query, kv, group, d]
        score = torch.einsum("ikgd,kpd->kgip", x, k) / math.sqrt(d)
        last = prefix + n - x.shape[0] + torch.arange(x.shape[0], device="cuda")
        score = torch.where(torch.arange(prefix + n, device="cuda") <= last[:, None], score, -math.inf)
        y = torch.einsum("kgip,kpd->ikgd", torch.softmax(score, -1), v)
        out[cu[b]:cu[b + 1]] = torch.nan_to_num(y).reshape(x.shape[0], h, d)
    return out


def _exact_sample(s):
    import numpy as np

    x, u = s["logits"].double().cpu().numpy(), s["u"].cpu().numpy()
    if x.size > 4_000_000:
        return None
    want = []
    for i, row in enumerate(x):
        t, k, p, m = (float(v[i]) if torch.is_tensor(v) else v for v in (s["temperature"], s["top_k"], s["top_p"], s["min_p"]))
        order = np.argsort(-row, kind="stable")
        w = np.exp((row[order] - row[order[0]]) / t)
        w = w[w >= max(m, 1e-300)]
        w = w[:int(k)] if k > 0 else w
        sums = np.cumsum(w)
        last = min(int(np.searchsorted(sums, p * sums[-1], side="left")), len(w) - 1)
        want.append(int(order[min(int(np.searchsorted(sums, u[i] * sums[last], side="left")), last)]))
    return torch.tensor(want, dtype=torch.int32)
