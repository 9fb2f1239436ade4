"""The measured calls of beam search and tree speculation over a paged key/value cache: the
selection over beams and vocabulary, attention of drafted nodes over the cache, the commit of the
accepted ones, the writing of new rows, and the forking of page tables.

`run` computes a case in its plain form, in elementary torch operations, or (`own`) through the
framework's entry points.  Both take the same state.  The cache's layout is the framework's: keys
[layers, pages, kv_heads, page, D], values [layers, pages, kv_heads, page / 8, D, 8].

Lengths, tree shapes and accepted counts follow from the case; the seed decides which sequence
has which, the values, the page tables' order and the tokens.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ITEM = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------ the cases

def _beam(name, G, W, V, n_out, dtype, hist):
    return {"name": name, "kind": "beam", "G": G, "W": W, "V": V, "n_out": n_out, "dtype": dtype, "hist": hist}


def _attn(name, B, T, Hq, Hkv, D, lo, hi, page, dtype, lse=False):
    return {"name": name, "kind": "attn", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "lo": lo, "hi": hi, "page": page,
            "dtype": dtype, "lse": lse}


def _append(name, L, B, T, Hkv, D, lo, hi, page, dtype, least):
    return {"name": name, "kind": "append", "L": L, "B": B, "T": T, "Hkv": Hkv, "D": D, "lo": lo, "hi": hi, "page": page,
            "dtype": dtype, "least": least}


def _commit(name, L, B, T, Hkv, D, lo, hi, page, dtype, most):
    return {"name": name, "kind": "commit", "L": L, "B": B, "T": T, "Hkv": Hkv, "D": D, "lo": lo, "hi": hi, "page": page,
            "dtype": dtype, "most": most}


def _fork(name, L, R, Hkv, D, lo, hi, page, dtype, room, width):
    return {"name": name, "kind": "fork", "L": L, "R": R, "Hkv": Hkv, "D": D, "lo": lo, "hi": hi, "page": page,
            "dtype": dtype, "room": room, "width": width}


def listed():
    return [
        # one request decoded with four beams, a 32k vocabulary: the smallest selection
        _beam("beam_one", 1, 4, 32000, 4, "fp32", 64),
        # a batch of 32 requests with eight beams each over a large vocabulary
        _beam("beam_batch", 32, 8, 128256, 8, "bf16", 512),
        # a single decoded token of a small model with a short context: latency
        _attn("attn_step", 1, 1, 8, 2, 64, 217, 217, 16, "fp16"),
        # a serving batch of mixed contexts, eight drafted nodes per sequence
        _attn("attn_batch", 32, 8, 32, 8, 128, 100, 4096, 64, "bf16"),
        # large drafted trees, eight query heads to a key head: the most arithmetic
        _attn("attn_wide", 16, 63, 32, 4, 128, 2000, 6000, 64, "bf16", lse=True),
        # one user with a very long context and a small tree
        _attn("attn_long", 1, 5, 32, 8, 128, 131000, 131000, 128, "bf16"),
        # a decode step's new rows of every layer
        _append("append_step", 16, 8, 1, 8, 128, 50, 2000, 64, "bf16", 1),
        # prompts of different lengths written into fresh pages
        _append("append_prompt", 16, 6, 2048, 8, 128, 0, 0, 64, "bf16", 300),
        # one user's tree: the accepted path found and written
        _commit("commit_one", 16, 1, 25, 8, 128, 1500, 1500, 64, "bf16", 5),
        # a batch of large trees
        _commit("commit_batch", 32, 64, 63, 8, 128, 100, 3000, 64, "bf16", 8),
        # four beams of one request reordered
        _fork("fork_one", 16, 4, 8, 128, 530, 530, 64, "bf16", 1, 4),
        # 16 requests of eight beams each reordered, every layer's partial pages copied
        _fork("fork_batch", 16, 128, 8, 128, 100, 900, 64, "bf16", 1, 8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["beam", "beam", "attn", "attn", "attn", "append", "commit", "fork"])
    if kind == "beam":
        V = _log_int(rng, 300, 151936)
        if rng.random() < 0.5:
            V = max(320, V // 64 * 64)
        dtype = rng.choice(["fp32", "bf16"])
        W = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
        G = _log_int(rng, 1, max(1, min(256, int(60e6 / (W * V * ITEM[dtype])))))
        c = _beam("", G, W, V, rng.choice([W, 2 * W]), dtype, rng.choice([0, _log_int(rng, 4, 1000)]))
    else:
        Hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 64, 96, 128, 128, 128, 256])
        page, dtype = rng.choice([16, 32, 64, 64, 128]), rng.choice(["bf16", "bf16", "fp16"])
        row = Hkv * D * 4  # bytes of a token's keys and values
        L = rng.choice([1, 4, 16])
        if kind == "attn":
            T = rng.choice([1, 1, rng.randint(2, 8), rng.randint(9, 64)])
            group = rng.choice([1, 2, 4, 4, 7, 8])
            hi = _log_int(rng, 1, 60000)
            most = min(250e6 / (hi * row), 30e9 / (4.0 * hi * T * Hkv * group * D))
            B = _log_int(rng, 1, max(1, min(64, int(most))))
            while B * hi * row > 400e6 or 4.0 * B * hi * T * Hkv * group * D > 55e9:
                hi = hi // 2 + 1
            lo = rng.choice([hi, hi // 3, 0])
            c = _attn("", B, T, Hkv * group, Hkv, D, lo, hi, page, dtype, lse=rng.random() < 0.3)
        elif kind == "append":
            T = rng.choice([1, rng.randint(2, 40), _log_int(rng, 40, 3000)])
            B = _log_int(rng, 1, max(1, min(64, int(150e6 / (L * T * row)))))
            lo = rng.choice([0, rng.randint(1, 500)])
            c = _append("", L, B, T, Hkv, D, lo, lo + rng.choice([0, 300]), page, dtype, rng.randint(1, T))
        elif kind == "commit":
            T = rng.randint(2, 64)
            B = _log_int(rng, 1, 64)
            lo = rng.choice([0, rng.randint(1, 500)])
            c = _commit("", L, B, T, Hkv, D, lo, lo + rng.choice([0, 700]), page, dtype, rng.randint(1, min(T - 1, 10)))
        else:
            width = rng.choice([1, 2, 4, 8, 16])
            R = width * _log_int(rng, 1, max(1, min(128 // width, int(200e6 / (width * L * page * row)))))
            lo = rng.randint(1, 600)
            c = _fork("", L, R, Hkv, D, lo, lo + rng.choice([0, 200]), page, dtype, rng.choice([0, 1, 1, 24]), width)
    del c["name"]
    return c


# ------------------------------------------------------------------ what a case fixes

def _spread(n, lo, hi):
    """n whole numbers from lo to hi, evenly spread (the seed shuffles them over the sequences)."""
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)] if n > 1 else [hi]


def _lens(c):
    return _spread(c["R"] // c["width"] if c["kind"] == "fork" else c["B"], c["lo"], c["hi"])


def _counts(c):
    """Rows written per sequence: the new tokens of an append, the root and the accepted nodes of a commit."""
    if c["kind"] == "append":
        return _spread(c["B"], c["least"], c["T"])
    return [1 + a for a in _spread(c["B"], 0 if c["B"] > 1 else c["most"], c["most"])]


def _copied(c):
    """Tokens of copied partial pages: every beam but the two parents of a request takes a copy."""
    return sum((n % c["page"] + 7) // 8 * 8 * max(c["width"] - 2, 0) for n in _lens(c))


def work(case):
    c = case
    if c["kind"] == "beam":
        n, rows = c["G"] * c["W"] * c["V"], c["G"] * c["n_out"]
        return {"bytes": n * ITEM[c["dtype"]] + rows * 12 + 8 * rows * c["hist"], "flops": 4 * n}
    row = 2 * c["Hkv"] * c["D"] * ITEM[c["dtype"]]
    if c["kind"] == "attn":
        lens, T = _lens(c), c["T"]
        q = 2 * c["B"] * T * c["Hq"] * c["D"] * ITEM[c["dtype"]]
        flops = 4.0 * sum((n + (T + 1) / 2) * T for n in lens) * c["Hq"] * c["D"]
        return {"bytes": (sum(lens) + c["B"] * T) * row + q, "flops": flops}
    if c["kind"] in ("append", "commit"):
        return {"bytes": 2 * sum(_counts(c)) * row * c["L"] + 64 * c["B"], "flops": 0}
    pages = sum((n + c["page"] - 1) // c["page"] for n in _lens(c)) * c["width"]
    return {"bytes": 2 * _copied(c) * row * c["L"] + 8 * pages + 8 * c["R"], "flops": 0}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape, dtype):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=g)


def _shuffled(g, values):
    v = torch.tensor(values, dtype=torch.int32, device=DEV)
    return v[torch.randperm(len(values), generator=g, device=DEV)].contiguous()


def _cache(g, c, L, pages):
    """A pool whose pages hold earlier requests' rows (also past a sequence's end)."""
    k = _normal(g, L, pages, c["Hkv"], c["page"], c["D"], dtype=DTYPES[c["dtype"]])
    return k, _normal(g, L, pages, c["Hkv"], c["page"] // 8, c["D"], 8, dtype=DTYPES[c["dtype"]])


def _tables(g, c, tokens):
    """Page tables of sequences that have room for `tokens` each, pages in random order, a few to spare."""
    P = max(1, max((n + c["page"] - 1) // c["page"] for n in tokens))
    pages = len(tokens) * P + 3
    t = torch.randperm(pages, generator=g, device=DEV)[: len(tokens) * P].to(torch.int32)
    return t.view(len(tokens), P).contiguous(), pages


def _tree(g, B, T, deep):
    """Drafted trees [B, T]: node 0 is the root, deep[b] nodes of row b lie on one path, the parents of the others are
    random earlier nodes; the tokens of a tree differ; the ids sampled at the path's nodes follow it to its end."""
    nodes = torch.arange(T, device=DEV).expand(B, T)
    key = torch.rand(B, T, generator=g, device=DEV)
    key[:, 0] = -1.0
    on = key.argsort(1).argsort(1) <= deep[:, None]
    before = torch.where(on, nodes, 0).cummax(1).values.roll(1, 1)  # the last path node ahead of each node
    other = (torch.rand(B, T, generator=g, device=DEV) * nodes).long()
    parents = torch.where(on, before, other)
    parents[:, 0] = -1
    draft = torch.rand(B, 4096, generator=g, device=DEV).argsort(1)[:, :T].contiguous()
    after = torch.where(on, nodes, T).flip(1).cummin(1).values.flip(1).roll(-1, 1)  # the next path node
    after[:, -1] = T
    wrong = 5000 + (torch.rand(B, T, generator=g, device=DEV) * 100).long()
    follow = torch.where(after < T, draft.gather(1, after.clamp(max=T - 1)), wrong)
    elsewhere = draft.gather(1, (torch.rand(B, T, generator=g, device=DEV) * T).long())
    sampled = torch.where(on, follow, elsewhere)
    i32 = torch.int32
    return parents.to(i32).contiguous(), draft.to(i32), sampled.to(i32).contiguous()


def prepare(case, seed):
    c, g = case, _gen(seed)
    i32 = torch.int32
    s = {"case": c}
    if c["kind"] == "beam":
        G, W, V, H, n = c["G"], c["W"], c["V"], c["hist"], c["n_out"]
        x = torch.randn(G * W, V, generator=g, device=DEV) * 3.0
        x.scatter_(1, torch.randint(0, V, (G * W, 8), generator=g, device=DEV), 12.0)
        x.scatter_(1, torch.randint(0, V, (G * W, 16), generator=g, device=DEV), -math.inf)  # forbidden ids
        s["logits"] = x.to(DTYPES[c["dtype"]])
        scores = (-40 * torch.rand(G, 1, generator=g, device=DEV) - torch.rand(G, W, generator=g, device=DEV).cumsum(1))
        if W > 2:  # a beam in eight has ended
            scores[:, W - 1] = torch.where(torch.rand(G, generator=g, device=DEV) < 0.125, -math.inf, scores[:, W - 1])
        s["scores"] = scores.view(-1).contiguous()
        s["out"] = {"scores": torch.empty(G * n, device=DEV), "parents": torch.empty(G * n, dtype=i32, device=DEV),
                    "tokens": torch.empty(G * n, dtype=i32, device=DEV)}
        if H:
            s["hist"] = torch.randint(0, V, (G * W, H), generator=g, device=DEV).to(i32)
            s["hist_len"] = torch.randint(0, H + 1, (G, 1), generator=g, device=DEV).to(i32).expand(G, W).reshape(-1).contiguous()
            s["out"] |= {"hist": torch.empty(G * n, H, dtype=i32, device=DEV), "hist_len": torch.empty(G * n, dtype=i32, device=DEV)}
        return s
    lens = _lens(c)
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "attn":
        B, T = c["B"], c["T"]
        s["lens"] = _shuffled(g, lens)
        s["tables"], pages = _tables(g, c, [max(lens)] * B)
        k, v = _cache(g, c, 1, pages)
        s["k"], s["v"] = k[0], v[0]
        s["q"] = _normal(g, B, T, c["Hq"], c["D"], dtype=dt) * 2  # sharper than uniform, as trained heads are
        s["k_new"] = _normal(g, B, T, c["Hkv"], c["D"], dtype=dt)
        s["v_new"] = _normal(g, B, T, c["Hkv"], c["D"], dtype=dt)
        deep = torch.full((B,), min(T - 1, 6), dtype=torch.long, device=DEV)
        s["parents"] = _tree(g, B, T, deep)[0]
        s["max_len"] = max(lens)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(B, T, c["Hq"], device=DEV) if c["lse"] else None
        return s
    if c["kind"] == "fork":
        R, w = c["R"], c["width"]
        P = (c["hi"] + c["room"] + 1 + c["page"] - 1) // c["page"] + 1
        pages = 2 * R * P + 3  # a request's beams each hold their pages, and there is room for the next step's
        lens_r = _shuffled(g, lens).repeat_interleave(w)
        t = torch.randperm(pages, generator=g, device=DEV)[: R * P].to(torch.int32).view(R, P)
        full = (lens_r // c["page"])[:, None]
        slot = torch.arange(P, device=DEV)[None]
        t = torch.where(slot < full, t.view(-1, w, P)[:, :1].expand(-1, w, P).reshape(R, P), t)  # full pages are shared
        s["tables"] = torch.where(slot < (lens_r[:, None] + c["page"] - 1) // c["page"], t, -1).to(i32).contiguous()
        s["lens"] = lens_r.contiguous()
        # two beams of a request go on, the first of them with one child fewer than the rest
        first = torch.randint(0, w, (R // w, 1), generator=g, device=DEV)
        second = (first + 1) % w
        to = torch.arange(w, device=DEV)[None].expand(R // w, w)
        par = torch.where(to < (w + 1) // 2, first, second) + w * torch.arange(R // w, device=DEV)[:, None]
        s["parents"] = par.reshape(-1).to(i32).contiguous()
        s["k"], s["v"] = _cache(g, c, c["L"], pages)
        s["out"] = {"tables": torch.empty_like(s["tables"]), "lens": torch.empty_like(s["lens"])}
        return s
    B, T = c["B"], c["T"]
    s["lens"] = _shuffled(g, lens)
    s["counts"] = _shuffled(g, _counts(c))
    s["tables"], pages = _tables(g, c, [max(lens) + T] * B)
    s["k"], s["v"] = _cache(g, c, c["L"], pages)
    s["k_new"] = _normal(g, c["L"], B, T, c["Hkv"], c["D"], dtype=dt)
    s["v_new"] = _normal(g, c["L"], B, T, c["Hkv"], c["D"], dtype=dt)
    s["out"] = {"lens": torch.empty_like(s["lens"])}
    if c["kind"] == "commit":
        s["parents"], s["draft"], s["sampled"] = _tree(g, B, T, s["counts"].long() - 1)
        s["out"] |= {"n_acc": torch.empty(B, dtype=i32, device=DEV), "tokens": torch.empty(B, T, dtype=i32, device=DEV),
                     "path": torch.empty(B, T, dtype=i32, device=DEV)}
    return s


# ------------------------------------------------------------------ plain forms

def _plain_beam(s):
    c = s["case"]
    G, W, V, H, n = c["G"], c["W"], c["V"], c["hist"], c["n_out"]
    # in 64 bits: candidates of different beams lie next to each other, and their order is the answer
    x = s["logits"].double()
    m = x.amax(1, keepdim=True)
    lse = m + (x - m).exp().sum(1, keepdim=True).log()
    total = (s["scores"].double()[:, None] + (x - lse)).view(G, W * V)
    best, at = total.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    parents = (at // V + W * torch.arange(G, device=DEV)[:, None]).view(-1)
    tokens = (at % V).view(-1)
    out = {"scores": best.reshape(-1).float(), "parents": parents.int(), "tokens": tokens.int()}
    if H:
        have = s["hist_len"].long()[parents]
        drop = (have == H).long()
        slot = torch.arange(H, device=DEV)[None]
        moved = s["hist"].long()[parents].gather(1, (slot + drop[:, None]).clamp(max=H - 1))
        kept = (have - drop)[:, None]
        out["hist"] = torch.where(slot < kept, moved, torch.where(slot == kept, tokens[:, None], -1)).int()
        out["hist_len"] = (kept[:, 0] + 1).int()
    return out


def _ancestors(parents):
    """[B, T, T]: whether node j is node i or an ancestor of it ((I + parent)^(T - 1) has a path's binomial there)."""
    B, T = parents.shape
    step = (torch.arange(T, device=DEV)[None, None] == parents[:, :, None]).float()
    return torch.linalg.matrix_power(step + torch.eye(T, device=DEV), max(T - 1, 1)) > 0


def _rows(cache, tables, page):
    """Keys of each sequence's pages in order: [B, kv_heads, tokens, D]."""
    B, P = tables.shape
    r = cache[tables.clamp(min=0).long()]
    return r.permute(0, 2, 1, 3, 4).reshape(B, cache.shape[1], P * page, cache.shape[3]).float()


def _plain_attn(s):
    c = s["case"]
    B, T, Hq, Hkv, D, page = (c[x] for x in ("B", "T", "Hq", "Hkv", "D", "page"))
    v_rows = s["v"].permute(0, 1, 2, 4, 3).reshape(s["v"].shape[0], Hkv, page, D)
    k = torch.cat([_rows(s["k"], s["tables"], page), s["k_new"].float().transpose(1, 2)], 2)
    v = torch.cat([_rows(v_rows, s["tables"], page), s["v_new"].float().transpose(1, 2)], 2)
    S = k.shape[2] - T
    q = s["q"].float().view(B, T, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(B, Hkv, -1, T, S + T) / math.sqrt(D)
    seen = torch.cat([(torch.arange(S, device=DEV)[None] < s["lens"][:, None])[:, None].expand(B, T, S), _ancestors(s["parents"])], 2)
    x = torch.where(seen[:, None, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = (x - m).exp()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul((p / total).view(B, Hkv, -1, S + T), v).view(B, Hkv, -1, T, D)
    out = {"out": o.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(s["q"].dtype)}
    if c["lse"]:
        out["lse"] = (m + total.log())[..., 0].permute(0, 3, 1, 2).reshape(B, T, Hq)
    return out


def _plain_write(s, node, count):
    """Rows node[b, i], i < count[b], to positions lens[b] + i."""
    page = s["case"]["page"]
    i = torch.minimum(torch.arange(node.shape[1], device=DEV)[None], count[:, None] - 1)  # past the count: its last row again
    node = node.gather(1, i)
    at = s["lens"].long()[:, None] + i
    pages = s["tables"].long().gather(1, at // page)
    b = torch.arange(node.shape[0], device=DEV)[:, None]
    slot = at % page
    s["k"][:, pages, :, slot] = s["k_new"][:, b, node].transpose(0, 1).transpose(1, 2)
    s["v"][:, pages, :, slot // 8, :, slot % 8] = s["v_new"][:, b, node].transpose(0, 1).transpose(1, 2)
    return {"k": s["k"], "v": s["v"], "lens": (s["lens"] + count).int()}


def _plain_append(s):
    c = s["case"]
    node = torch.arange(c["T"], device=DEV)[None].expand(c["B"], c["T"])
    return _plain_write(s, node, s["counts"].long())


def _plain_commit(s):
    T = s["case"]["T"]
    nodes = torch.arange(T, device=DEV)[None]
    parents, draft, sampled = s["parents"].long(), s["draft"].long(), s["sampled"].long()
    fits = (draft == sampled.gather(1, parents.clamp(min=0))) & (parents >= 0)
    # an earlier child of the same parent that fits too goes first
    earlier = (parents[:, :, None] == parents[:, None]) & fits[:, None] & (nodes[:, None] < nodes[:, :, None])
    fits = (fits & ~earlier.any(2)) | (nodes == 0)
    line = _ancestors(s["parents"])
    taken = ~(line & ~fits[:, None]).any(2) & line[:, :, 0]
    count = taken.sum(1)
    order = torch.where(taken, nodes, T).sort(1).values
    last = order.gather(1, count[:, None] - 1)
    path = torch.where(order < T, order, -1)
    token = draft.gather(1, path.clamp(min=0)).roll(-1, 1)
    token = torch.where(nodes < count[:, None] - 1, token, torch.where(nodes == count[:, None] - 1, sampled.gather(1, last), -1))
    out = _plain_write(s, path.clamp(min=0), count)
    return out | {"n_acc": (count - 1).int(), "tokens": token.int(), "path": path.int()}


def _plain_fork(s):
    c = s["case"]
    page, room = c["page"], c["room"]
    N, (R, P) = s["k"].shape[1], s["tables"].shape
    parents = s["parents"].long()
    lens = s["lens"].long()[parents][:, None]
    t = s["tables"].long()[parents]
    slot, flat = torch.arange(P, device=DEV)[None], torch.arange(R * P, device=DEV).view(R, P)
    shared = slot < lens // page
    mine = ~shared & (slot < (lens + room + page - 1) // page)
    named = mine & (t >= 0)
    # a page's owner: -1 where a row shares it, else the first row that would write to it
    owner = torch.full((N + 1,), R * P, device=DEV)
    owner.scatter_reduce_(0, torch.where(shared, t, torch.where(named, t, N)).view(-1),
                          torch.where(shared, -1, flat).view(-1), "amin")
    kept = named & (owner[t.clamp(min=0)] == flat)
    needs = mine & ~kept
    free = (owner[:N] < R * P).int().sort(stable=True).indices  # the free pages first, in order
    fresh = free[(needs.view(-1).long().cumsum(0) - 1).clamp(min=0)].view(R, P)
    tables = torch.where(shared | kept, t, torch.where(needs, fresh, -1))
    copied = needs & (slot * page < lens)
    # every row copies one page; a row without a copy takes its page's own rows
    at = (lens[:, 0] // page).clamp(max=P - 1)[:, None]
    to = tables.gather(1, at).clamp(min=0)[:, 0]
    source = torch.where(copied.gather(1, at), t.gather(1, at), to[:, None])[:, 0]
    upto = (lens % page + 7) // 8 * 8
    token = torch.arange(page, device=DEV)[None]
    take = (token < upto) & copied.gather(1, at)
    k, v = s["k"], s["v"]
    k[:, to] = torch.where(take[None, :, None, :, None], k[:, source], k[:, to])
    v[:, to] = torch.where(take[None, :, None, ::8, None, None], v[:, source], v[:, to])
    return {"k": k, "v": v, "tables": tables.int(), "lens": lens[:, 0].int()}


PLAIN = {"beam": _plain_beam, "attn": _plain_attn, "append": _plain_append, "commit": _plain_commit, "fork": _plain_fork}


# ------------------------------------------------------------------ the framework's calls

@functools.lru_cache(maxsize=None)
def _sampler():
    """The process's handle, as a server keeps one."""
    import tinygpt_amd as tg

    return tg.Sampler(device=0, max_batch=4096, max_vocab=152064, max_hist=1024)


def _own_beam(s):
    o = s["out"]
    _sampler().beam_select(s["logits"], s["scores"], s["case"]["W"], s["case"]["n_out"], hist=s.get("hist"),
                           hist_len=s.get("hist_len"), out=o)
    return o


def _own_attn(s):
    _sampler().tree_attention(s["q"], s["k_new"], s["v_new"], s["k"], s["v"], s["tables"], s["lens"], parents=s["parents"],
                              max_len=s["max_len"], out=s["out"], lse=s["lse"])
    return {"out": s["out"]} | ({"lse": s["lse"]} if s["lse"] is not None else {})


def _own_append(s):
    o = s["out"]
    _sampler().kv_append(s["k_new"], s["v_new"], s["k"], s["v"], s["tables"], s["lens"], counts=s["counts"], lens_out=o["lens"])
    return {"k": s["k"], "v": s["v"], "lens": o["lens"]}


def _own_commit(s):
    o = s["out"]
    _sampler().tree_commit(s["k_new"], s["v_new"], s["k"], s["v"], s["tables"], s["lens"], s["parents"], s["draft"],
                           s["sampled"], out=o)
    return {"k": s["k"], "v": s["v"]} | o


def _own_fork(s):
    o = s["out"]
    _sampler().kv_fork(s["k"], s["v"], s["tables"], s["lens"], s["parents"], room=s["case"]["room"], tables_out=o["tables"],
                       lens_out=o["lens"])
    return {"k": s["k"], "v": s["v"]} | o


OWN = {"beam": _own_beam, "attn": _own_attn, "append": _own_append, "commit": _own_commit, "fork": _own_fork}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ------------------------------------------------------------------ the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "beam":
        return _exact_beam(s)
    return _exact_attn(s) if case["kind"] == "attn" else _exact_cache(s)


def _exact_beam(s):
    c = s["case"]
    W, n = c["W"], c["n_out"]
    scores = []
    for g in range(c["G"]):
        rows = s["logits"][g * W:(g + 1) * W].double()
        total = torch.log_softmax(rows, 1) + s["scores"][g * W:(g + 1) * W, None].double()
        scores.append(total.flatten().topk(n).values)
    return {"scores": torch.cat(scores)}


def _exact_attn(s):
    c = s["case"]
    B, T, Hq, Hkv, D, page = (c[x] for x in ("B", "T", "Hq", "Hkv", "D", "page"))
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=DEV)
    lse = torch.zeros(B, T, Hq, dtype=torch.float64, device=DEV)
    parents = s["parents"].tolist()
    for b in range(B):
        n = int(s["lens"][b])
        pages = s["tables"][b, : (n + page - 1) // page].long()
        line = torch.zeros(T, T, dtype=torch.bool)
        for i in range(T):
            j = i
            while j >= 0:
                line[i, j] = True
                j = parents[b][j]
        bar = torch.cat([torch.ones(T, n, dtype=torch.bool), line], 1).to(DEV)
        for h in range(Hkv):
            k = torch.cat([s["k"][pages, h].reshape(-1, D)[:n], s["k_new"][b, :, h]]).double()
            v = torch.cat([s["v"][pages, h].transpose(2, 3).reshape(-1, D)[:n], s["v_new"][b, :, h]]).double()
            kT = k.t().contiguous()
            for i in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                x = (s["q"][b, :, i].double() @ kT / math.sqrt(D)).masked_fill(~bar, -math.inf)
                out[b, :, i] = torch.softmax(x, 1) @ v
                lse[b, :, i] = torch.logsumexp(x, 1)
    return {"out": out} | ({"lse": lse} if c["lse"] else {})


def _exact_cache(s):
    """Moved rows have their values: sequence by sequence, layer by layer, on the cache itself."""
    c = s["case"]
    page = c["page"]
    lens, tables = s["lens"].tolist(), s["tables"].tolist()
    k, v = s["k"], s["v"]
    if c["kind"] == "fork":
        return _exact_fork(s, lens, tables)
    for b in range(c["B"]):
        if c["kind"] == "append":
            nodes = list(range(int(s["counts"][b])))
        else:
            parents, draft, sampled = (s[x][b].tolist() for x in ("parents", "draft", "sampled"))
            nodes = [0]
            while True:
                more = [j for j in range(1, c["T"]) if parents[j] == nodes[-1] and draft[j] == sampled[nodes[-1]]]
                if not more:
                    break
                nodes.append(more[0])
        for first in range(0, len(nodes)):
            at = lens[b] + first
            to = tables[b][at // page]
            k[:, to, :, at % page] = s["k_new"][:, b, nodes[first]]
            v[:, to, :, at % page // 8, :, at % 8] = s["v_new"][:, b, nodes[first]]
    return {"k": k, "v": v}


def _exact_fork(s, lens, tables):
    c = s["case"]
    page, k, v = c["page"], s["k"], s["v"]
    parents = s["parents"].tolist()
    used, want, wrote = set(), [], set()
    for p in parents:
        used.update(tables[p][: lens[p] // page])
    for p in parents:
        for i in range(lens[p] // page, (lens[p] + c["room"] + page - 1) // page):
            e = tables[p][i]
            if e >= 0 and e not in used and e not in wrote:
                wrote.add(e)
            else:
                want.append((e, (lens[p] - i * page + 7) // 8 if lens[p] > i * page else 0))
    free = [n for n in range(k.shape[1]) if n not in used and n not in wrote]
    for (e, blocks), to in zip(want, free):
        if blocks:
            k[:, to, :, : 8 * blocks] = k[:, e, :, : 8 * blocks].clone()
            v[:, to, :, :blocks] = v[:, e, :, :blocks].clone()
    return {"k": k, "v": v}
