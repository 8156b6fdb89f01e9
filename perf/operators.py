"""Timed cases of the operators around a cache that several continuations share: attention of a chunk of new tokens
over the paged cache, norms of queries and keys per head (with the position rotation for rows that are trained, into the
cache's pages for rows that are served), and copies of pages (forks of a prompt, compaction of a pool).

``listed`` names the cases, ``draw`` makes more of the same ranges, ``prepare`` makes what a program has in hand before
the call, ``run`` is one call, in plain torch operations or - with ``own`` - through the package's entry points,
``work`` the bytes and operations it cannot do without, ``exact`` the result from the definition in 64 bits."""
from __future__ import annotations

import math
import random

import torch

own = False

D = 128                 # head dimension
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # Two short conversations take a few new tokens each: nothing but latency.
        dict(name="extend_small", kind="extend", requests=2, new_lo=3, new_hi=4, ctx_lo=100, ctx_hi=300, kv_heads=8,
             group=4, page=16, dtype="bf16", len_seed=11),
        # A batch whose last few tokens, drafted ahead, are verified in one step.
        dict(name="extend_draft", kind="extend", requests=32, new_lo=4, new_hi=8, ctx_lo=512, ctx_hi=4096, kv_heads=8,
             group=4, page=16, dtype="bf16", len_seed=12),
        # One very long document, a short question behind it.
        dict(name="extend_long", kind="extend", requests=1, new_lo=17, new_hi=17, ctx_lo=65551, ctx_hi=65551, kv_heads=8,
             group=4, page=16, dtype="fp16", len_seed=13),
        # The next turn of sixteen conversations, one kv head per query head.
        dict(name="extend_turn", kind="extend", requests=16, new_lo=20, new_hi=120, ctx_lo=700, ctx_hi=4000, kv_heads=32,
             group=1, page=32, dtype="bf16", len_seed=14),
        # Long prompts taken in pieces of some hundred tokens.
        dict(name="extend_chunk", kind="extend", requests=4, new_lo=400, new_hi=512, ctx_lo=4096, ctx_hi=12288, kv_heads=8,
             group=4, page=16, dtype="bf16", len_seed=15),
        # A decode step's new tokens on their way into the cache: one per request, slices of one fused projection.
        dict(name="norm_append_decode", kind="append", requests=64, new_lo=1, new_hi=1, ctx_lo=1, ctx_hi=150, kv_heads=8,
             group=4, page=16, dtype="bf16", len_seed=16),
        # Prompts on their way into the cache.
        dict(name="norm_append_prompts", kind="append", requests=12, new_lo=30, new_hi=1500, ctx_lo=0, ctx_hi=100,
             kv_heads=8, group=4, page=16, dtype="fp16", len_seed=17),
        # The rows that are trained, forward and backward: a long batch, and a short one far into a long text whose
        # heads carry no norm.
        dict(name="norm_rope_train", kind="train", tokens=8192, first=0, norm=True, kv_heads=8, group=4, dtype="bf16"),
        dict(name="rope_train_small", kind="train", tokens=181, first=100003, norm=False, kv_heads=32, group=1,
             dtype="fp16"),
        # Every prompt of a batch continued four ways: the filled part of its last page is copied to each.
        dict(name="fork_tails", kind="copy", sources=24, copies=4, layers=32, kv_heads=8, page=16, full=False,
             dtype="bf16", len_seed=18),
        # A fragmented pool drawn together: whole pages move.
        dict(name="compact_pages", kind="copy", sources=280, copies=1, layers=32, kv_heads=8, page=16, full=True,
             dtype="bf16", len_seed=19),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["extend", "extend", "extend", "append", "train", "copy"])
    dtype = rng.choice(["bf16", "fp16"])
    seed = rng.randrange(1 << 20)
    heads = rng.choice([(8, 4), (32, 1), (2, 8), (16, 1), (4, 2), (8, 8), (1, 8)])
    base = dict(kind=kind, kv_heads=heads[0], group=heads[1], dtype=dtype, len_seed=seed)
    if kind == "extend":
        hi = min(_log(rng, 16, 65536), 1200000 // heads[0])
        new = min(_log(rng, 1, 512), hi, max(1, int(4.0e8 / (hi * heads[0] * heads[1]))))
        requests = min(_log(rng, 1, 64), max(1, 1200000 // (heads[0] * hi)),
                       max(1, int(4.0e8 / (hi * new * heads[0] * heads[1]))))
        return dict(base, requests=requests, new_lo=max(1, new // rng.randint(1, 8)), new_hi=new,
                    ctx_lo=max(1, hi // rng.randint(1, 16)), ctx_hi=hi, page=rng.choice([8, 16, 32, 64]))
    if kind == "append":
        new = rng.choice([1, _log(rng, 2, 1500)])
        return dict(base, requests=min(_log(rng, 1, 200), max(1, 16000 // new)), new_lo=max(1, new // rng.randint(1, 8)),
                    new_hi=new, ctx_lo=0, ctx_hi=_log(rng, 1, 200), page=rng.choice([8, 16, 32, 64]))
    if kind == "train":
        return dict(kind=kind, kv_heads=heads[0], group=heads[1], dtype=dtype, tokens=_log(rng, 1, 8192),
                    first=rng.choice([0, _log(rng, 1, 200000)]), norm=rng.random() < 0.7)
    full = rng.random() < 0.5
    layers, page = rng.choice([2, 16, 32]), rng.choice([8, 16, 32])
    entry = 4 * layers * heads[0] * D   # bytes of one position
    copies = 1 if full else rng.randint(1, 8)
    sources = min(_log(rng, 1, 280), max(1, int(5.0e8 / (entry * page * copies))))
    return dict(kind=kind, sources=sources, copies=copies, layers=layers, kv_heads=heads[0], page=page, full=full,
                dtype=dtype, len_seed=seed)


# ---------------------------------------------------------------------------
# what a case is made of
# ---------------------------------------------------------------------------

BASE = 10000.0
EPS = 1e-6
LAYERS, LAYER = 2, 1    # of the caches of the attention and append cases


def _lengths(c):
    """New tokens and total length (new ones included) of every request."""
    r = random.Random(c["len_seed"])
    new, total = [], []
    for _ in range(c["requests"]):
        n = r.randint(c["new_lo"], c["new_hi"])
        new.append(n)
        total.append(max(n, 1) + r.randint(c["ctx_lo"], c["ctx_hi"]))
    return new, total


def _page_table(total, page):
    """The requests take pages in turn, as conversations that grow side by side do: for every request the places of
    its pages in the pool."""
    left = [-(-t // page) for t in total]
    table, nxt = [[] for _ in total], 0
    while any(left):
        for b in range(len(total)):
            if left[b]:
                table[b].append(nxt)
                left[b] -= 1
                nxt += 1
    return table, nxt


def _entries(c):
    """Positions to copy of every source page."""
    r = random.Random(c["len_seed"])
    return [c["page"] if c["full"] else r.randint(1, c["page"] - 1) for _ in range(c["sources"])]


class _Maker:
    """Seeded tensors of one case."""

    def __init__(self, c, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.g = torch.Generator(device=self.dev).manual_seed(seed)
        self.dtype = DTYPES[c["dtype"]]

    def normal(self, shape, scale=1.0):
        return (torch.randn(shape, generator=self.g, device=self.dev) * scale).to(self.dtype)

    def weight(self):
        return (1.0 + 0.3 * torch.randn(D, generator=self.g, device=self.dev)).to(self.dtype)

    def ints(self, v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=self.dev)


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _inputs(c, seed):
    m = _Maker(c, seed)
    kind = c["kind"]
    d = dict(case=c, kind=kind)
    N = c["kv_heads"]
    if kind in ("extend", "append"):
        Nq = N * c["group"]
        new, total = _lengths(c)
        table, pages = _page_table(total, c["page"])
        d.update(new=new, total=total, table=table, starts=_starts(new))
        # the pool of pages; keys and values of a trained model are of order one
        d["pool"] = m.normal((pages, LAYERS, 2, N, c["page"], D))
        if kind == "extend":
            d["q"] = m.normal((sum(new), Nq, D))
        else:
            qkv = m.normal((sum(new), Nq + 2 * N, D), 1.7)
            d["q"], d["k"], d["v"] = qkv[:, :Nq], qkv[:, Nq:Nq + N], qkv[:, Nq + N:]
            d["wq"], d["wk"] = m.weight(), m.weight()
    elif kind == "train":
        T, Nq = c["tokens"], N * c["group"]
        qkv = m.normal((T, Nq + 2 * N, D), 1.7)
        d["q"], d["k"] = qkv[:, :Nq], qkv[:, Nq:Nq + N]
        d["gq"], d["gk"] = m.normal((T, Nq, D)), m.normal((T, N, D))
        d["positions"] = torch.arange(c["first"], c["first"] + T, device=m.dev)
        d["wq"], d["wk"] = (m.weight(), m.weight()) if c["norm"] else (None, None)
    else:
        src = [s for s in range(c["sources"]) for _ in range(c["copies"])]
        ent = _entries(c)
        d["src"], d["entries"] = src, [ent[s] for s in src]
        shape = (c["layers"], 2, N, c["page"], D)
        d["from"] = m.normal((c["sources"],) + shape)
        d["to"] = m.normal((len(src),) + shape)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    dev = (d["from"] if d["kind"] == "copy" else d["q"]).device
    if d["kind"] in ("extend", "append"):
        if own:
            from loquetier_b200 import kvcache
            pool = kvcache.KvPool(LAYERS, case["kv_heads"], D, case["page"], d["pool"].dtype, dev,
                                  pages_per_slab=d["pool"].size(0))
            caches = [kvcache.KvCache(pool, 0) for _ in d["total"]]
            left = list(d["total"])
            while any(left):
                for b, cache in enumerate(caches):
                    n = min(left[b], case["page"])
                    if n:
                        cache.extend(n)
                        left[b] -= n
            slab = caches[0].pages[0]._base
            slab.copy_(d["pool"])
            d["pool"] = slab
            d["caches"], d["kv"] = caches, kvcache.BatchedKvCache(caches)
        d["indptr"] = torch.tensor(d["starts"], dtype=torch.int32, device=dev)
        d["rows"] = [torch.tensor(t, dtype=torch.int64, device=dev) for t in d["table"]]
        if d["kind"] == "append":   # where the new tokens go: page and place of each
            P = case["page"]
            at = [(t[p // P], p % P) for n, L, t in zip(d["new"], d["total"], d["table"]) for p in range(L - n, L)]
            d["at_page"] = torch.tensor([a for a, _ in at], device=dev)
            d["at_entry"] = torch.tensor([e for _, e in at], device=dev)
    elif d["kind"] == "train":
        for name in ("q", "k", "wq", "wk"):
            if d[name] is not None:
                d[name].requires_grad_(own)
    else:
        if own:
            from loquetier_b200 import kvcache
            n = d["from"].size(0) + d["to"].size(0)
            pool = kvcache.KvPool(case["layers"], case["kv_heads"], D, case["page"], d["from"].dtype, dev, pages_per_slab=n)
            pages = [pool.alloc_page() for _ in range(n)]
            slab = pages[0]._base
            slab[:d["from"].size(0)].copy_(d["from"])
            slab[d["from"].size(0):].copy_(d["to"])
            ptrs = torch.tensor([p.data_ptr() for p in pages], dtype=torch.int64, device=dev)
            d["pool"] = pool
            d["to"] = slab[d["from"].size(0):]
            d["to_ptrs"] = ptrs[d["from"].size(0):].contiguous()
            d["from_ptrs"] = ptrs[:d["from"].size(0)][torch.tensor(d["src"], device=dev)].contiguous()
            del d["from"]
        d["src"] = torch.tensor(d["src"], device=dev)
        d["entries"] = None if case["full"] else torch.tensor(d["entries"], dtype=torch.int32, device=dev)
    return d


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _cos_sin(pos):
    """cos and sin [T, 64] of the rotation at integer positions; the angles in 64 bits, as far positions need."""
    freq = BASE ** (-torch.arange(D // 2, device=pos.device, dtype=torch.float64) * 2.0 / D)
    ang = pos.to(torch.float64)[:, None] * freq
    return ang.cos().float(), ang.sin().float()


def _rotate(x, cos, sin):
    """x [T, N, D] turned by [T, 64]; (cos, -sin) turns back."""
    a, b = x[..., :D // 2], x[..., D // 2:]
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _normalise(x, w):
    s = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * s * w, s


def _plain_extend(d):
    c = d["case"]
    N, G = c["kv_heads"], c["group"]
    out = torch.empty_like(d["q"])
    for b, rows in enumerate(d["rows"]):
        n, L, t0 = d["new"][b], d["total"][b], d["starts"][b]
        kv = d["pool"][:, LAYER].index_select(0, rows).float()                       # [pages, 2, N, P, D]
        kv = kv.permute(1, 0, 3, 2, 4).reshape(2, -1, N, D)[:, :L]
        cos, sin = _cos_sin(torch.arange(L, device=rows.device))
        k = _rotate(kv[0], cos, sin)
        q = _rotate(d["q"][t0:t0 + n].float(), cos[L - n:], sin[L - n:])
        hidden = torch.arange(L, device=rows.device)[None, :] > torch.arange(L - n, L, device=rows.device)[:, None]
        for h in range(N):   # one kv head at a time: the scores of all would not fit beside long caches
            s = q[:, h * G:(h + 1) * G].transpose(0, 1) @ k[:, h].t() / math.sqrt(D)     # [G, n, L]
            s = s.masked_fill(hidden, float("-inf"))
            e = torch.exp(s - s.max(-1, keepdim=True).values)
            o = (e @ kv[1, :, h]) / e.sum(-1, keepdim=True)
            out[t0:t0 + n, h * G:(h + 1) * G] = o.transpose(0, 1).to(out.dtype)
    return out


def _plain_append(d):
    q = _normalise(d["q"].float(), d["wq"].float())[0].to(d["q"].dtype)
    k = _normalise(d["k"].float(), d["wk"].float())[0].to(d["k"].dtype)
    d["pool"][d["at_page"], LAYER, 0, :, d["at_entry"]] = k
    d["pool"][d["at_page"], LAYER, 1, :, d["at_entry"]] = d["v"]
    return [q, d["pool"]]


def _plain_train(d):
    cos, sin = _cos_sin(d["positions"])
    outs, grads, wgrads = [], [], []
    for x, w, g in ((d["q"], d["wq"], d["gq"]), (d["k"], d["wk"], d["gk"])):
        xf = x.float()
        dn = _rotate(g.float(), cos, -sin)
        if w is None:
            y, dx = _rotate(xf, cos, sin), dn
        else:
            n, s = _normalise(xf, w.float())
            y = _rotate(n, cos, sin)
            dw = (xf * s * dn).sum((0, 1), dtype=torch.float64)
            wdn = dn * w.float()
            dx = s * (wdn - xf * (s * s) * (wdn * xf).mean(-1, keepdim=True))
            wgrads.append(dw.to(w.dtype))
        outs.append(y.to(x.dtype))
        grads.append(dx.to(x.dtype))
    return outs + grads + wgrads


def _plain_copy(d):
    new = d["from"].index_select(0, d["src"])
    if d["entries"] is not None:
        P = new.size(4)
        keep = torch.arange(P, device=new.device)[None, :] < d["entries"][:, None]
        new = torch.where(keep[:, None, None, None, :, None], new, d["to"])
    d["to"].copy_(new)
    return d["to"]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    d, kind = state, state["kind"]
    if not own:
        return {"extend": _plain_extend, "append": _plain_append, "train": _plain_train, "copy": _plain_copy}[kind](d)
    from loquetier_b200 import kernel_utils, kvcache
    if kind == "extend":
        return kvcache.batch_extend(d["q"], d["indptr"], d["kv"], BASE, LAYER)
    if kind == "append":
        q = kvcache.norm_append_kv(d["kv"], d["q"], d["k"], d["v"], d["wq"], d["wk"], EPS, LAYER,
                                   None if d["case"]["new_hi"] == 1 else d["indptr"])
        return [q, d["pool"]]
    if kind == "train":
        wrt = [d[n] for n in ("q", "k", "wq", "wk") if d[n] is not None]
        yq, yk = kernel_utils.qk_norm_rope.apply(d["q"], d["k"], d["wq"], d["wk"], d["positions"], BASE, EPS)
        return [yq.detach(), yk.detach(), *torch.autograd.grad((yq, yk), wrt, (d["gq"], d["gk"]))]
    kvcache.copy_pages(d["pool"], d["to_ptrs"], d["from_ptrs"], d["entries"])
    return d["to"]


def work(case):
    c = case
    if c["kind"] in ("extend", "append"):
        N, Nq = c["kv_heads"], c["kv_heads"] * c["group"]
        new, total = _lengths(c)
        if c["kind"] == "extend":
            seen = sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(new, total))
            return {"bytes": 4 * D * N * sum(total) + 4 * D * Nq * sum(new), "flops": 4 * D * Nq * seen}
        return {"bytes": 4 * D * (Nq + 2 * N) * sum(new), "flops": 5 * D * (Nq + N) * sum(new)}
    if c["kind"] == "train":
        el = c["tokens"] * c["kv_heads"] * (c["group"] + 1) * D
        return {"bytes": 8 * el, "flops": (22 if c["norm"] else 6) * el}
    entry = 4 * c["layers"] * c["kv_heads"] * D
    filled = sum(_entries(c))
    return {"bytes": entry * filled * (1 + c["copies"]), "flops": 0}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _phase(pos):
    """exp(i p theta_j) as complex numbers [T, 64]."""
    j = torch.arange(D // 2, dtype=torch.float64, device=pos.device)
    ang = torch.outer(pos.double(), torch.exp(-math.log(BASE) * j / (D // 2)))
    return torch.complex(torch.cos(ang), torch.sin(ang))


def _turn(x, phase):
    """The rotation as a product of complex numbers: dimensions j and j + 64 are the two parts of one."""
    z = torch.complex(x[..., :D // 2].double().contiguous(), x[..., D // 2:].double().contiguous()) * phase[:, None, :]
    return torch.cat([z.real, z.imag], dim=-1)


def exact(case, seed):
    d = _inputs(case, seed)
    kind = d["kind"]
    if kind == "extend":
        N, G, P = case["kv_heads"], case["group"], case["page"]
        out = torch.zeros(d["q"].shape, dtype=torch.float64, device=d["q"].device)
        for b, pages in enumerate(d["table"]):
            n, L, t0 = d["new"][b], d["total"][b], d["starts"][b]
            pos = torch.arange(L, device=out.device)
            phase = _phase(pos)
            qr = _turn(d["q"][t0:t0 + n], phase[L - n:]).unflatten(1, (N, G))
            for h in range(N):
                flat = d["pool"][torch.tensor(pages, device=out.device), LAYER, :, h].double()     # [pages, 2, P, D]
                keys, values = (flat[:, i].reshape(-1, D)[:L] for i in (0, 1))
                score = torch.einsum("ngd,ld->ngl", qr[:, h], _turn(keys[:, None], phase)[:, 0]) * D ** -0.5
                score += torch.where(pos[None, :] <= pos[L - n:, None], 0.0, -math.inf)[:, None, :]
                weight = torch.exp(score - torch.logsumexp(score, dim=-1, keepdim=True))
                out[t0:t0 + n, h * G:(h + 1) * G] = torch.einsum("ngl,ld->ngd", weight, values)
        return out
    if kind == "append":
        unit = [x.double() / ((x.double() ** 2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
                for x, w in ((d["q"], d["wq"]), (d["k"], d["wk"]))]
        pool = d["pool"].double()
        t = 0
        for n, L, pages in zip(d["new"], d["total"], d["table"]):
            p = torch.arange(L - n, L)
            slot, place = torch.tensor(pages)[p // case["page"]].to(pool.device), (p % case["page"]).to(pool.device)
            pool[slot, LAYER, 0, :, place] = unit[1][t:t + n]
            pool[slot, LAYER, 1, :, place] = d["v"][t:t + n].double()
            t += n
        return [unit[0], pool]
    if kind == "train":
        phase = _phase(d["positions"])
        ys, dxs, dws = [], [], []
        for x, w, g in ((d["q"], d["wq"], d["gq"]), (d["k"], d["wk"], d["gk"])):
            x64, dn = x.double(), _turn(g, phase.conj())
            if w is None:
                ys.append(_turn(x64, phase))
                dxs.append(dn)
                continue
            r = ((x64 ** 2).sum(-1, keepdim=True) / D + EPS).sqrt()
            u, w64 = x64 / r, w.double()
            ys.append(_turn(u * w64, phase))
            dws.append((u * dn).sum((0, 1)))
            dxs.append((dn * w64 - u * (dn * w64 * u).sum(-1, keepdim=True) / D) / r)
        return ys + dxs + dws
    out = d["to"].double()
    for i, (s, e) in enumerate(zip(d["src"], d["entries"])):
        out[i, :, :, :, :e] = d["from"][s, :, :, :, :e].double()
    return out
