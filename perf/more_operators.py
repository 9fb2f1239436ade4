"""The measured calls of a paged key/value cache held in 8 bits, and of the position rotation: attention of
drafted nodes over that cache, the writing of new rows (rotated on the way), the rotation of a step's queries and
keys, the commit of accepted nodes, and the forking of page tables.

`run` computes a case in its plain form, in elementary torch operations, or (`own`) through the framework's entry
points.  Both take the same state.  The 8-bit cache: keys [layers, pages, kv_heads, page, D] and values [layers,
pages, kv_heads, page / 16, D, 16] in e4m3, scales [layers, pages, kv_heads, page / 16, 2] in e8m0 (powers of two):
one of the keys and one of the values of each block of 16 tokens of a head.  A block that is written has the smallest
scale with which its largest magnitude stays within 448, but none below that of the tokens it holds already; those are
rounded again where the scale grows.  The 16-bit cache: values [layers, pages, kv_heads, page / 8, D, 8].

Lengths, tree shapes and accepted counts follow from the case; the seed decides which sequence has which, the values,
the page tables' order and the tokens.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
FLOOR = {"bf16": -100, "fp16": -15}  # the smallest exponent of a block's scale
E4M3, E8M0, U8, I32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.uint8, torch.int32
BLOCK = 16


# ------------------------------------------------------------------ the cases

def _attn(name, B, T, Hq, Hkv, D, lo, hi, page, dtype, lse=False):
    return {"name": name, "kind": "attn", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "lo": lo, "hi": hi, "page": page,
            "dtype": dtype, "lse": lse}


def _append(name, L, B, T, Hkv, D, lo, hi, page, dtype, least, e8, dims, pairs):
    """dims: how many of a key's D dimensions are rotated (0: none); pairs: neighbours, else halves."""
    return {"name": name, "kind": "append", "L": L, "B": B, "T": T, "Hkv": Hkv, "D": D, "lo": lo, "hi": hi, "page": page,
            "dtype": dtype, "least": least, "e8": e8, "dims": dims, "pairs": pairs}


def _rotate(name, B, T, Hq, Hkv, D, lo, hi, dtype, dims, pairs, tree):
    return {"name": name, "kind": "rotate", "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "lo": lo, "hi": hi, "dtype": dtype,
            "dims": dims, "pairs": pairs, "tree": tree}


def _commit(name, L, B, T, Hkv, D, lo, hi, page, dtype, most):
    return {"name": name, "kind": "commit", "L": L, "B": B, "T": T, "Hkv": Hkv, "D": D, "lo": lo, "hi": hi, "page": page,
            "dtype": dtype, "most": most, "e8": True}


def _fork(name, L, R, Hkv, D, lo, hi, page, room, width):
    return {"name": name, "kind": "fork", "L": L, "R": R, "Hkv": Hkv, "D": D, "lo": lo, "hi": hi, "page": page, "dtype": "bf16",
            "room": room, "width": width}


def listed():
    return [
        # a single decoded token of a small model with a short context: latency
        _attn("attn8_step", 1, 1, 8, 2, 64, 217, 217, 16, "fp16"),
        # a serving batch of mixed contexts, eight drafted nodes per sequence
        _attn("attn8_batch", 32, 8, 32, 8, 128, 100, 4096, 64, "bf16"),
        # large drafted trees, eight query heads to a key head: the most arithmetic
        _attn("attn8_wide", 16, 63, 32, 4, 128, 2000, 6000, 64, "bf16", lse=True),
        # one user with a very long context and a small tree
        _attn("attn8_long", 1, 5, 32, 8, 128, 131000, 131000, 128, "bf16"),
        # a decode step's new rows of every layer, rotated and encoded into blocks that are filled in part
        _append("append8_step", 16, 8, 1, 8, 128, 50, 2000, 64, "bf16", 1, True, 128, False),
        # prompts of different lengths rotated and encoded into fresh pages
        _append("append8_prompt", 16, 6, 2048, 8, 128, 0, 0, 64, "bf16", 300, True, 128, False),
        # a decode step's queries and keys, half of each head rotated by neighbours
        _rotate("rotate_step", 8, 1, 32, 8, 128, 50, 2000, "fp16", 64, True, False),
        # the nodes of a batch of large drafted trees at their depths
        _rotate("rotate_tree", 64, 63, 32, 8, 128, 100, 30000, "bf16", 128, False, True),
        # one user's tree: the accepted path found, encoded and written
        _commit("commit8_one", 16, 1, 25, 8, 128, 1500, 1500, 64, "bf16", 5),
        # a batch of large trees
        _commit("commit8_batch", 32, 64, 63, 8, 128, 100, 2900, 64, "bf16", 8),
        # four beams of one request reordered
        _fork("fork8_one", 16, 4, 8, 128, 530, 530, 64, 1, 4),
        # 16 requests of eight beams each reordered, every layer's partial pages copied
        _fork("fork8_batch", 16, 128, 8, 128, 100, 900, 64, 1, 8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "append", "append", "rotate", "commit", "fork"])
    Hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 64, 96, 128, 128, 128, 256])
    page, dtype = rng.choice([16, 32, 64, 64, 128]), rng.choice(["bf16", "bf16", "fp16"])
    row = Hkv * D * 2  # bytes of a token's keys and values
    L, group = rng.choice([1, 4, 16]), rng.choice([1, 2, 4, 4, 7, 8])
    dims, pairs = rng.choice([D, D, D // 2, 32]), rng.random() < 0.4
    if kind == "attn":
        T = rng.choice([1, 1, rng.randint(2, 8), rng.randint(9, 64)])
        hi = _log_int(rng, 1, 100000)
        most = min(250e6 / (hi * row), 30e9 / (4.0 * hi * T * Hkv * group * D))
        B = _log_int(rng, 1, max(1, min(64, int(most))))
        while B * hi * row > 250e6 or 4.0 * B * hi * T * Hkv * group * D > 55e9:
            hi = hi // 2 + 1
        lo = rng.choice([hi, hi // 3, 0])
        c = _attn("", B, T, Hkv * group, Hkv, D, lo, hi, page, dtype, lse=rng.random() < 0.3)
    elif kind == "append":
        e8 = rng.random() < 0.6
        T = rng.choice([1, rng.randint(2, 40), _log_int(rng, 40, 2500)])
        B = _log_int(rng, 1, max(1, min(64, int(75e6 / (L * T * row)))))
        lo = rng.choice([0, rng.randint(1, 500), rng.randint(1, 500)])
        c = _append("", L, B, T, Hkv, D, lo, lo + rng.choice([0, 300]), page, dtype, rng.randint(1, T), e8,
                    rng.choice([dims, dims, 0]) if e8 else dims, pairs)
    elif kind == "rotate":
        tree = rng.random() < 0.5
        T = rng.randint(2, 64) if tree else rng.choice([1, _log_int(rng, 2, 2000)])
        B = _log_int(rng, 1, max(1, min(64, int(30e6 / (T * Hkv * (group + 1) * D * 2)))))
        lo = rng.choice([0, _log_int(rng, 1, 100000)])
        c = _rotate("", B, T, Hkv * group, Hkv, D, lo, lo + rng.choice([0, 3000]), dtype, dims, pairs, tree)
    elif kind == "commit":
        T = rng.randint(2, 64)
        B = _log_int(rng, 1, 64)
        lo = rng.choice([0, rng.randint(1, 500)])
        c = _commit("", L, B, T, Hkv, D, lo, lo + rng.choice([0, 700]), page, dtype, rng.randint(1, min(T - 1, 20)))
    else:
        width = rng.choice([1, 2, 4, 8, 16])
        R = width * _log_int(rng, 1, max(1, min(128 // width, int(200e6 / (width * L * page * row)))))
        lo = rng.randint(1, 600)
        c = _fork("", L, R, Hkv, D, lo, lo + rng.choice([0, 200]), page, rng.choice([0, 1, 1, 24]), width)
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


def work(case):
    c = case
    D, Hkv = c["D"], c["Hkv"]
    if c["kind"] == "rotate":
        n = c["B"] * c["T"] * (c["Hq"] + Hkv)
        return {"bytes": 4 * n * D, "flops": 3 * n * c["dims"]}
    row, scales = 2 * Hkv * D, 2 * Hkv / BLOCK  # bytes of a token in 8 bits, and its share of its block's scales
    if c["kind"] == "attn":
        lens, T = _lens(c), c["T"]
        q = 4 * c["B"] * T * c["Hq"] * D
        flops = 4.0 * sum((n + (T + 1) / 2) * T for n in lens) * c["Hq"] * D
        return {"bytes": int(sum(lens) * (row + scales)) + 2 * c["B"] * T * row + q, "flops": flops}
    if c["kind"] in ("append", "commit"):
        out = row + scales if c["e8"] else 2 * row
        n = sum(_counts(c)) * c["L"]
        return {"bytes": int(n * (2 * row + out)) + 64 * c["B"], "flops": 3 * n * Hkv * c.get("dims", 0)}
    copied = sum((n % c["page"] + BLOCK - 1) // BLOCK * BLOCK * max(c["width"] - 2, 0) for n in _lens(c))
    pages = sum((n + c["page"] - 1) // c["page"] for n in _lens(c)) * c["width"]
    return {"bytes": int(2 * copied * (row + scales) * c["L"]) + 8 * pages + 8 * c["R"], "flops": 0}


# ------------------------------------------------------------------ the 8-bit blocks

def _need(most, dtype):
    """Exponent of the smallest scale for a block's largest magnitude (448 = 0.875 * 2^9)."""
    m, x = torch.frexp(most)
    e = torch.where(m > 0.875, x - 8, x - 9)
    return torch.where(most > 0, e, FLOOR[dtype]).clamp(min=FLOOR[dtype])


def _encode(x, e):
    """Blocks x [..., 16, D] with exponents e [...], in e4m3."""
    return torch.ldexp(x, -e[..., None, None]).to(E4M3)


def _scale(e):
    return (e + 127).to(U8)


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=g)


def _shuffled(g, values):
    v = torch.tensor(values, dtype=I32, device=DEV)
    return v[torch.randperm(len(values), generator=g, device=DEV)].contiguous()


def _tables(g, c, tokens):
    """Page tables of sequences that have room for `tokens` each, pages in random order, a few to spare."""
    P = max(1, max((n + c["page"] - 1) // c["page"] for n in tokens))
    pages = len(tokens) * P + 3
    t = torch.randperm(pages, generator=g, device=DEV)[: len(tokens) * P].to(I32)
    return t.view(len(tokens), P).contiguous(), pages


def _channels(g, D):
    """Magnitudes of a key's dimensions: a few are several times the others, as trained keys' are."""
    return torch.exp(0.7 * _normal(g, D))


def _cache8(g, c, L, pages):
    """A pool whose pages hold earlier requests' rows (also past a sequence's end)."""
    H, page, D = c["Hkv"], c["page"], c["D"]
    k = torch.empty(L, pages, H, page, D, dtype=E4M3, device=DEV)
    v = torch.empty(L, pages, H, page // BLOCK, D, BLOCK, dtype=E4M3, device=DEV)
    s = torch.empty(L, pages, H, page // BLOCK, 2, dtype=U8, device=DEV)
    part = max(1, (1 << 25) // (H * page * D))  # pages a go
    for layer in range(L):
        wide = _channels(g, D)
        for p in range(0, pages, part):
            n = min(part, pages - p)
            x = _normal(g, n, H, page // BLOCK, BLOCK, D) * wide
            e = _need(x.abs().amax((-1, -2)), c["dtype"])
            k[layer, p:p + n] = _encode(x, e).view(n, H, page, D)
            s[layer, p:p + n, ..., 0] = _scale(e)
            x = _normal(g, n, H, page // BLOCK, BLOCK, D)
            e = _need(x.abs().amax((-1, -2)), c["dtype"])
            v[layer, p:p + n] = _encode(x, e).transpose(-1, -2)
            s[layer, p:p + n, ..., 1] = _scale(e)
    return k, v, s.view(E8M0)


def _cache16(g, c, L, pages):
    dt = DTYPES[c["dtype"]]
    k = _normal(g, L, pages, c["Hkv"], c["page"], c["D"], dtype=dt)
    return k, _normal(g, L, pages, c["Hkv"], c["page"] // 8, c["D"], 8, dtype=dt)


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
    return parents.to(I32).contiguous(), draft.to(I32), sampled.to(I32).contiguous()


def _frequencies(c):
    """10000^(-2 j / dims), the angle of pair j per position."""
    n = c["dims"] // 2
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64, device=DEV) / max(n, 1))).float() if n else None


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    dt, lens = DTYPES[c["dtype"]], _lens(c)
    if c["kind"] == "fork":
        return _prepare_fork(s, c, g, lens)
    B, T, Hkv, D = c["B"], c["T"], c["Hkv"], c["D"]
    s["lens"] = _shuffled(g, lens)
    if c["kind"] == "attn":
        s["tables"], pages = _tables(g, c, [max(lens)] * B)
        k, v, scales = _cache8(g, c, 1, pages)
        s["k"], s["v"], s["scales"] = k[0], v[0], scales[0]
        s["q"] = _normal(g, B, T, c["Hq"], D, dtype=dt) * 1.5  # sharper than uniform, as trained heads are
        s["k_new"] = _normal(g, B, T, Hkv, D, dtype=dt)
        s["v_new"] = _normal(g, B, T, Hkv, D, dtype=dt)
        s["parents"] = _tree(g, B, T, torch.full((B,), min(T - 1, 6), dtype=torch.long, device=DEV))[0]
        s["max_len"] = max(lens)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(B, T, c["Hq"], device=DEV) if c["lse"] else None
        return s
    s["freq"] = _frequencies(c) if c.get("dims") else None
    if c["kind"] == "rotate":
        s["q"], s["k_new"] = _normal(g, B, T, c["Hq"], D, dtype=dt), _normal(g, B, T, Hkv, D, dtype=dt)
        s["parents"] = _tree(g, B, T, torch.full((B,), min(T - 1, 6), dtype=torch.long, device=DEV))[0] if c["tree"] else None
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k_new"])
        return s
    s["counts"] = _shuffled(g, _counts(c))
    s["tables"], pages = _tables(g, c, [max(lens) + T] * B)
    if c["e8"]:
        s["k"], s["v"], s["scales"] = _cache8(g, c, c["L"], pages)
    else:
        s["k"], s["v"] = _cache16(g, c, c["L"], pages)
    s["k_new"] = _normal(g, c["L"], B, T, Hkv, D, dtype=dt).mul_(_channels(g, D).to(dt))
    s["v_new"] = _normal(g, c["L"], B, T, Hkv, D, dtype=dt)
    s["out"] = {"lens": torch.empty_like(s["lens"])}
    if c["kind"] == "commit":
        s["parents"], s["draft"], s["sampled"] = _tree(g, B, T, s["counts"].long() - 1)
        s["out"] |= {"n_acc": torch.empty(B, dtype=I32, device=DEV), "tokens": torch.empty(B, T, dtype=I32, device=DEV),
                     "path": torch.empty(B, T, dtype=I32, device=DEV)}
    return s


def _prepare_fork(s, c, g, lens):
    R, w = c["R"], c["width"]
    P = (c["hi"] + c["room"] + 1 + c["page"] - 1) // c["page"] + 1
    pages = 2 * R * P + 3  # a request's beams each hold their pages, and there is room for the next step's
    lens_r = _shuffled(g, lens).repeat_interleave(w)
    t = torch.randperm(pages, generator=g, device=DEV)[: R * P].to(I32).view(R, P)
    full = (lens_r // c["page"])[:, None]
    slot = torch.arange(P, device=DEV)[None]
    t = torch.where(slot < full, t.view(-1, w, P)[:, :1].expand(-1, w, P).reshape(R, P), t)  # full pages are shared
    s["tables"] = torch.where(slot < (lens_r[:, None] + c["page"] - 1) // c["page"], t, -1).to(I32).contiguous()
    s["lens"] = lens_r.contiguous()
    # two beams of a request go on, the first of them with one child fewer than the rest
    first = torch.randint(0, w, (R // w, 1), generator=g, device=DEV)
    second = (first + 1) % w
    to = torch.arange(w, device=DEV)[None].expand(R // w, w)
    par = torch.where(to < (w + 1) // 2, first, second) + w * torch.arange(R // w, device=DEV)[:, None]
    s["parents"] = par.reshape(-1).to(I32).contiguous()
    s["k"], s["v"], s["scales"] = _cache8(g, c, c["L"], pages)
    s["out"] = {"tables": torch.empty_like(s["tables"]), "lens": torch.empty_like(s["lens"])}
    return s


# ------------------------------------------------------------------ plain forms

def _ancestors(parents):
    """[B, T, T]: whether node j is node i or an ancestor of it ((I + parent)^(T - 1) has a path's binomial there)."""
    B, T = parents.shape
    step = (torch.arange(T, device=DEV)[None, None] == parents[:, :, None]).float()
    return torch.linalg.matrix_power(step + torch.eye(T, device=DEV), max(T - 1, 1)) > 0


def _decoded(codes, scales, which):
    """Blocks [..., 16, D] of codes with their scales [..., 2], as numbers."""
    return codes.view(E4M3).float() * scales.view(E8M0).float()[..., which, None, None]


def _plain_attn(s):
    c = s["case"]
    B, T, Hq, Hkv, D, page = (c[x] for x in ("B", "T", "Hq", "Hkv", "D", "page"))
    at = s["tables"].long()
    S = at.shape[1] * page
    scales = s["scales"].view(U8)[at]                                     # [B, slots, heads, blocks, 2]
    k = _decoded(s["k"].view(U8)[at].unflatten(3, (-1, BLOCK)), scales, 0)  # [B, slots, heads, blocks, 16, D]
    v = _decoded(s["v"].view(U8)[at].transpose(-1, -2), scales, 1)
    k, v = (x.permute(0, 2, 1, 3, 4, 5).reshape(B, Hkv, S, D) for x in (k, v))
    k = torch.cat([k, s["k_new"].float().transpose(1, 2)], 2)
    v = torch.cat([v, s["v_new"].float().transpose(1, 2)], 2)
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


def _rotated(x, position, freq, pairs):
    """Rows x [..., D] in 32 bits, turned by position * freq; position: x's dimensions but the last, or 1 where it is shared."""
    n = freq.shape[0]
    angle = position.double()[..., None] * freq.double()  # (a far position's angle needs more than 32 bits)
    co, si = angle.cos().float(), angle.sin().float()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if pairs else (x[..., :n], x[..., n:2 * n])
    both = [a * co - b * si, b * co + a * si]
    turned = torch.stack(both, -1).flatten(-2) if pairs else torch.cat(both, -1)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _plain_rotate(s):
    c = s["case"]
    T = c["T"]
    depth = _ancestors(s["parents"]).sum(2) - 1 if s["parents"] is not None else torch.arange(T, device=DEV)[None]
    at = (s["lens"].long()[:, None] + depth)[..., None]
    q, k = (_rotated(x.float(), at, s["freq"], c["pairs"]).to(x.dtype) for x in (s["q"], s["k_new"]))
    return {"q": q, "k": k}


def _plain_write16(s, node, count):
    """Rows node[b, i], i < count[b], to positions lens[b] + i."""
    c = s["case"]
    page = c["page"]
    i = torch.minimum(torch.arange(node.shape[1], device=DEV)[None], count[:, None] - 1)  # past the count: its last row again
    node = node.gather(1, i)
    at = s["lens"].long()[:, None] + i
    pages = s["tables"].long().gather(1, at // page)
    b = torch.arange(node.shape[0], device=DEV)[:, None]
    slot = at % page
    new = s["k_new"][:, b, node]
    new = _rotated(new.float(), at[None, ..., None], s["freq"], c["pairs"]).to(new.dtype)
    s["k"][:, pages, :, slot] = new.transpose(0, 1).transpose(1, 2)
    s["v"][:, pages, :, slot // 8, :, slot % 8] = s["v_new"][:, b, node].transpose(0, 1).transpose(1, 2)
    return {"k": s["k"], "v": s["v"], "lens": (s["lens"] + count).int()}


def _plain_write8(s, node, count):
    """The same, block by block of 16 tokens."""
    c = s["case"]
    page, B = c["page"], node.shape[0]
    start, end = s["lens"].long()[:, None], (s["lens"] + count).long()[:, None]
    n = node.shape[1] // BLOCK + 2
    blk = torch.minimum(start // BLOCK + torch.arange(n, device=DEV), (end - 1) // BLOCK)  # past the end: the last block again
    at = blk[..., None] * BLOCK + torch.arange(BLOCK, device=DEV)                          # [B, n, 16]
    fresh = (at >= start[..., None]) & (at < end[..., None])
    held = at < start[..., None]
    pages, inner = s["tables"].long().gather(1, blk * BLOCK // page), blk % (page // BLOCK)
    i = (at - start[..., None]).clamp(min=0, max=node.shape[1] - 1).view(B, -1)
    rows = node.gather(1, i).view(B, n, BLOCK)
    b = torch.arange(B, device=DEV)[:, None, None]
    L, N, H, _, D = s["k"].shape
    scales = s["scales"].view(U8)
    old = scales[:, pages, :, inner]  # [B, n, L, heads, 2]
    kb, vb = s["k"].view(U8).view(L, N, H, -1, BLOCK, D), s["v"].view(U8)
    for which, pool, new in ((0, kb, s["k_new"]), (1, vb, s["v_new"])):
        x = new[:, b, rows].float()  # [L, B, n, 16, heads, D]
        if which == 0 and s.get("freq") is not None:
            x = _rotated(x, at[None, ..., None], s["freq"], c["pairs"])
        x = x.permute(1, 2, 0, 4, 3, 5)  # [B, n, L, heads, 16, D]
        codes = pool[:, pages, :, inner]
        codes = codes.transpose(-1, -2) if which else codes
        f, h = fresh[:, :, None, None, :, None], held[:, :, None, None, :, None]
        e = _need(torch.where(f, x, 0).abs().amax((-1, -2)), c["dtype"])
        before = old[..., which].int() - 127
        e = torch.where(held.any(2)[:, :, None, None], torch.maximum(e, before), e)
        x = _encode(torch.where(f, x, torch.where(h, _decoded(codes, old, which), 0)), e).view(U8)
        x = torch.where(f | h, x, codes)  # what lies behind the last token stays
        pool[:, pages, :, inner] = x.transpose(-1, -2) if which else x
        scales[:, pages, :, inner, which] = _scale(e)
    return {"k": s["k"], "v": s["v"], "scales": s["scales"], "lens": (s["lens"] + count).int()}


def _plain_append(s):
    c = s["case"]
    node = torch.arange(c["T"], device=DEV)[None].expand(c["B"], c["T"])
    return (_plain_write8 if c["e8"] else _plain_write16)(s, node, s["counts"].long())


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
    out = _plain_write8(s, path.clamp(min=0), count)
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
    upto = (lens % page + BLOCK - 1) // BLOCK  # blocks
    block = torch.arange(page // BLOCK, device=DEV)[None]
    take = ((block < upto) & copied.gather(1, at))[None, :, None, :, None]
    L, _, H, _, D = s["k"].shape
    for x in (s["k"].view(U8).view(L, N, H, -1, BLOCK * D), s["v"].view(U8).view(L, N, H, -1, BLOCK * D), s["scales"].view(U8)):
        x[:, to] = torch.where(take, x[:, source], x[:, to])
    return {"k": s["k"], "v": s["v"], "scales": s["scales"], "tables": tables.int(), "lens": lens[:, 0].int()}


PLAIN = {"attn": _plain_attn, "append": _plain_append, "rotate": _plain_rotate, "commit": _plain_commit, "fork": _plain_fork}


# ------------------------------------------------------------------ the framework's calls

@functools.lru_cache(maxsize=None)
def _sampler():
    """The process's handle, as a server keeps one."""
    import tinygpt_amd as tg

    return tg.Sampler(device=0, max_batch=4096, max_vocab=152064, max_hist=1024)


def _own_attn(s):
    _sampler().tree_attention(s["q"], s["k_new"], s["v_new"], s["k"], s["v"], s["tables"], s["lens"], parents=s["parents"],
                              max_len=s["max_len"], out=s["out"], lse=s["lse"], scales=s["scales"])
    return {"out": s["out"]} | ({"lse": s["lse"]} if s["lse"] is not None else {})


def _own_append(s):
    o, c = s["out"], s["case"]
    _sampler().kv_append(s["k_new"], s["v_new"], s["k"], s["v"], s["tables"], s["lens"], counts=s["counts"], lens_out=o["lens"],
                         scales=s.get("scales"), rotary=s["freq"], pairs=c["pairs"])
    return {"k": s["k"], "v": s["v"], "lens": o["lens"]} | ({"scales": s["scales"]} if c["e8"] else {})


def _own_rotate(s):
    _sampler().rotate(s["q"], s["k_new"], s["lens"], s["freq"], pairs=s["case"]["pairs"], parents=s["parents"],
                      q_out=s["q_out"], k_out=s["k_out"])
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_commit(s):
    o = s["out"]
    _sampler().tree_commit(s["k_new"], s["v_new"], s["k"], s["v"], s["tables"], s["lens"], s["parents"], s["draft"],
                           s["sampled"], out=o, scales=s["scales"])
    return {"k": s["k"], "v": s["v"], "scales": s["scales"]} | o


def _own_fork(s):
    o = s["out"]
    _sampler().kv_fork(s["k"], s["v"], s["tables"], s["lens"], s["parents"], room=s["case"]["room"], tables_out=o["tables"],
                       lens_out=o["lens"], scales=s["scales"])
    return {"k": s["k"], "v": s["v"], "scales": s["scales"]} | o


OWN = {"attn": _own_attn, "append": _own_append, "rotate": _own_rotate, "commit": _own_commit, "fork": _own_fork}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ------------------------------------------------------------------ the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "append": _exact_write, "rotate": _exact_rotate, "commit": _exact_write,
            "fork": lambda s: None}[case["kind"]](s)  # (a fork computes no numbers)


def _exact_line(parents):
    """bool [T, T]: the nodes from each node up to its root."""
    line = torch.zeros(len(parents), len(parents), dtype=torch.bool)
    for i in range(len(parents)):
        j = i
        while j >= 0:
            line[i, j] = True
            j = parents[j]
    return line


def _exact_attn(s):
    c = s["case"]
    B, T, Hq, Hkv, D, page = (c[x] for x in ("B", "T", "Hq", "Hkv", "D", "page"))
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=DEV)
    lse = torch.zeros(B, T, Hq, dtype=torch.float64, device=DEV)
    parents = s["parents"].tolist()
    for b in range(B):
        n = int(s["lens"][b])
        pages = s["tables"][b, : (n + page - 1) // page].long()
        bar = torch.cat([torch.ones(T, n, dtype=torch.bool), _exact_line(parents[b])], 1).to(DEV)
        for h in range(Hkv):
            scale = s["scales"].view(U8)[pages, h].view(E8M0).double().reshape(-1, 2).repeat_interleave(BLOCK, 0)
            k = s["k"].view(U8)[pages, h].view(E4M3).double().reshape(-1, D) * scale[:, :1]
            v = s["v"].view(U8)[pages, h].view(E4M3).double().transpose(2, 3).reshape(-1, D) * scale[:, 1:]
            kT = torch.cat([k[:n], s["k_new"][b, :, h].double()]).t().contiguous()
            v = torch.cat([v[:n], s["v_new"][b, :, h].double()])
            for i in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                x = (s["q"][b, :, i].double() @ kT / math.sqrt(D)).masked_fill(~bar, -math.inf)
                out[b, :, i] = torch.softmax(x, 1) @ v
                lse[b, :, i] = torch.logsumexp(x, 1)
    return {"out": out} | ({"lse": lse} if c["lse"] else {})


def _exact_turn(x, angle, pairs):
    """Rows x [..., D] as complex numbers times e^(i angle), angle [..., n]."""
    n = angle.shape[-1]
    y = x.clone()
    z = (torch.complex(x[..., 0:2 * n:2].contiguous(), x[..., 1:2 * n:2].contiguous()) if pairs
         else torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous()))
    z = z * torch.exp(torch.complex(torch.zeros_like(angle), angle))
    if pairs:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = z.real, z.imag
    else:
        y[..., :n], y[..., n:2 * n] = z.real, z.imag
    return y


def _exact_rotate(s):
    c = s["case"]
    q, k = torch.empty_like(s["q"], dtype=torch.float64), torch.empty_like(s["k_new"], dtype=torch.float64)
    for b in range(c["B"]):
        depth = _exact_line(s["parents"][b].tolist()).sum(1) - 1 if c["tree"] else torch.arange(c["T"])
        angle = ((int(s["lens"][b]) + depth).double().to(DEV)[:, None] * s["freq"].double())[:, None]
        q[b] = _exact_turn(s["q"][b].double(), angle, c["pairs"])
        k[b] = _exact_turn(s["k_new"][b].double(), angle, c["pairs"])
    return {"q": q, "k": k}


def _exact_nodes(s, b):
    c = s["case"]
    if c["kind"] == "append":
        return list(range(int(s["counts"][b])))
    parents, draft, sampled = (s[x][b].tolist() for x in ("parents", "draft", "sampled"))
    nodes = [0]
    while True:
        more = [j for j in range(1, c["T"]) if parents[j] == nodes[-1] and draft[j] == sampled[nodes[-1]]]
        if not more:
            return nodes
        nodes.append(more[0])


def _exact_write(s):
    """The cache's numbers over their blocks' scales, not rounded; sequence by sequence, block by block, a layer at a time."""
    c = s["case"]
    if c["L"] * sum(_counts(c)) * c["Hkv"] * c["D"] > 2e8 or c["L"] * sum(_counts(c)) > 8000 * BLOCK:
        return None
    page, freq = c["page"], s.get("freq")
    lens, tables = s["lens"].tolist(), s["tables"].tolist()
    k, v = s["k"].double(), s["v"].double()
    scales = s["scales"].double() if c["e8"] else None
    for b in range(c["B"]):
        nodes = torch.tensor(_exact_nodes(s, b), device=DEV)
        n0, n1 = lens[b], lens[b] + len(nodes)
        at = torch.arange(n0, n1, device=DEV)
        kn, vn = s["k_new"][:, b, nodes].double(), s["v_new"][:, b, nodes].double()  # [L, rows, heads, D]
        if freq is not None:
            kn = _exact_turn(kn, (at.double()[:, None] * freq.double())[None, :, None], c["pairs"])
        size = BLOCK if c["e8"] else 8
        for blk in range(n0 // size, (n1 - 1) // size + 1):
            lo, hi = max(blk * size, n0), min((blk + 1) * size, n1)
            p, first, held = tables[b][blk * size // page], blk * size % page, max(n0 - blk * size, 0)
            x, y = (z[:, lo - n0:hi - n0].transpose(1, 2) for z in (kn, vn))  # [L, heads, tokens, D]
            kd, vd = k[:, p, :, first:first + size], v[:, p, :, first // size].transpose(2, 3)
            if c["e8"]:
                for which, z, d in ((0, x, kd), (1, y, vd)):
                    most = z.abs().amax((2, 3))
                    e = torch.ceil(torch.log2(most / 448)).clamp(min=FLOOR[c["dtype"]])
                    now = torch.exp2(e)
                    if held:
                        before = scales[:, p, :, first // size, which]
                        now = torch.maximum(now, before)
                        d[:, :, :held] *= (before / now)[..., None, None]
                    d[:, :, lo - blk * size:hi - blk * size] = z / now[..., None, None]
                    scales[:, p, :, first // size, which] = now
            else:
                kd[:, :, lo - blk * size:hi - blk * size] = x
                vd[:, :, lo - blk * size:hi - blk * size] = y
    return {"k": k, "v": v} | ({"scales": scales} if c["e8"] else {})
