"""Extreme inputs of the beam, tree-attention and cache tests, and what is
expected of them (shared by the CPU simulation's tests and the GPU's)."""
from __future__ import annotations

import math

import torch

import kv_cases as C

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ beams

# (type, value of a masked id: a large finite number, as grammars and padded vocabularies write it)
MASKS = [(dt, v) for dt in (F32, BF16)
         for v in (-1e4, -1e9, -1e10, -1e12, -1e30, -1e38, -2.4e38, torch.finfo(dt).min)]


def mask_name(case):
    return f"{str(case[0])[6:]}{case[1]:.3g}"


def masked_logits(dt, value, V):
    """Requests of three beams: a few ids allowed in each row; all but the last ids masked in one, all ids in another;
    a padded vocabulary; a whole request at the mask's value, one with a single larger id in it."""
    g = gen(abs(int(value)) % 1000 + V)
    x = torch.randn(4 * 3, V, generator=g) * 3
    mask = torch.ones(12, V, dtype=torch.bool)
    for r in range(3):
        mask[r, torch.randperm(V, generator=g)[:40]] = False
    mask[3, -5:] = False       # one live thread in a chunk, and one chunk alone of a row
    mask[5, :7] = False        # (row 4: masked whole, beside rows that are not)
    mask[6:9, : V - V // 4] = False
    x = torch.where(mask, torch.tensor(value), x).to(dt)
    x[11, V // 2] = x[11, 0].double() * (1 - 2.0**-6)
    scores = -3 * torch.rand(12, generator=g).cumsum(0)
    return x, scores


def large_logits(dt, V):
    """Two beams each: rows around one large value, a few steps of the type apart, and rows with one huge id."""
    g = gen(V)
    rows = []
    for at in (1e6, 2.0**22 - 3, 2.0**22 + 3, 1e7, 1e9, 1e10, 1e20, 3e38):
        for sign in (-1, 1):
            step = at * torch.finfo(dt).eps
            rows.append(sign * at + torch.randint(-4, 4, (V,), generator=g).double() * max(step, 1.0))
            one = torch.randn(V, generator=g).double()
            one[int(torch.randint(0, V, (1,), generator=g))] = sign * at
            rows.append(one)
    x = torch.stack(rows).to(dt)
    assert torch.isfinite(x).all()
    return x, -3 * torch.rand(len(rows), generator=g)


def check_beam(got, want, x):
    # a total's one 32-bit rounding, the logsumexp's sum of 32-bit exponentials (relative 2^-21 at most), and the
    # 64-bit roundings of a logsumexp as large as the row's logits and of the difference from it, on both sides
    w = want["scores"]
    top = x.double().amax(1)[want["parents"].long().clamp(min=0)].abs()
    assert torch.equal(got["parents"], want["parents"]) and torch.equal(got["tokens"], want["tokens"])
    fin = torch.isfinite(w)
    assert torch.equal(fin, torch.isfinite(got["scores"]))
    err = (got["scores"].double() - w).abs()
    assert (err <= w.abs() * 2**-24 + 2**-21 + 4 * top * 2**-53)[fin].all(), float(err[fin].max())


# ------------------------------------------------------------------ forks

def fork(k, v, tabs, lens, parents, room):
    """Forks in plain form: pages are given to rows in order, to a row all that it needs or none.  A row with tokens in
    a slot that names no page of the pool is given none and fails; a length that is none stays a failure."""
    k, v = k.clone(), v.clone()
    R, P = tabs.shape
    N, page = k.shape[1], k.shape[3]
    to, out = torch.full((R, P), -1, dtype=torch.int32), torch.zeros(R, dtype=torch.int32)
    rows = []
    for r in range(R):
        p = int(parents[r])
        n = int(lens[p]) if 0 <= p < R else -1
        rows.append((tabs[p].tolist(), n, n // page, min((n + room + page - 1) // page, P)) if 0 <= n <= P * page else None)
    shared = {x for row in rows if row for x in row[0][:row[2]]}
    writer = {}
    for r, row in enumerate(rows):
        for i in range(row[2], row[3]) if row else ():
            if 0 <= row[0][i] < N and row[0][i] not in shared:
                writer.setdefault(row[0][i], (r, i))
    free = [x for x in range(N) if x not in shared and x not in writer]
    for r, row in enumerate(rows):
        if row is None:
            out[r] = -1 if 0 <= int(parents[r]) < R else 0
            continue
        t, n, full, end = row
        to[r, :full] = torch.tensor(t[:full], dtype=torch.int32)
        fresh = [i for i in range(full, end) if writer.get(t[i]) != (r, i)]
        bad = any(not 0 <= x < N for x in t[: (n + page - 1) // page])
        fits = len(fresh) <= len(free) and not bad
        for i in range(full, end):
            if i not in fresh:
                to[r, i] = t[i]
            elif fits:
                to[r, i] = new = free.pop(0)
                if n > i * page:
                    blocks = (min(max(n - i * page, 0), page) + 7) // 8
                    k[:, new, :, : blocks * 8] = k[:, t[i], :, : blocks * 8].clone()
                    v[:, new, :, :blocks] = v[:, t[i], :, :blocks].clone()
        out[r] = n if fits and n + room <= P * page else -1
    return k, v, to, out


def fork_case(tabs, lens, parents, pages, L=1, H=1, page=8, D=16, dt=BF16, seed=0):
    g = gen(seed)
    k = torch.randn(L, pages, H, page, D, generator=g).to(dt)
    v = torch.randn(L, pages, H, page // 8, D, 8, generator=g).to(dt)
    return k, v, *(torch.tensor(x, dtype=torch.int32) for x in (tabs, lens, parents))


# (the case, room, the expected tables and lengths): pools that run out
SHORT_POOLS = {
    # rows 1 and 3 find no page; row 2 keeps its own
    "kept": (fork_case([[0, 1], [0, 1], [2, 3], [2, 3]], [12] * 4, [0, 0, 2, 2], 4), 1,
             [[0, 1], [0, -1], [2, 3], [2, -1]], [12, -1, 12, -1]),
    # row 1 would take two pages of the one there is: row 3 gets it, and row 2, whose page no one writes to, needs none
    "smaller": (fork_case([[0, 1, 2], [0, 1, 2], [3, 4, -1], [3, 4, -1]], [12, 12, 12, 12], [0, 0, 2, 2], 6), 9,
                [[0, 1, 2], [0, -1, -1], [3, 4, 5], [3, -1, -1]], [12, -1, 12, -1]),
    # row 0 would take two of the one free page, row 2 takes it
    "later": (fork_case([[0, -1, -1], [2, 3, -1], [2, 3, -1]], [8, 12, 12], [0, 1, 1], 4), 9,
              [[0, -1, -1], [2, 3, 1], [2, -1, -1]], [-1, 12, -1]),
    # nothing to copy and no page for the room
    "no room": (fork_case([[0], [1]], [8, 8], [0, 1], 2), 0, [[0], [1]], [8, 8]),
}


# (the case, room, the expected tables and lengths): slots that hold tokens and name no page of the pool
BAD_ENTRIES = {
    # a partly filled page: the row's parent would give NaN and not be appended to, and the row must not look sound
    "partial": (fork_case([[0, 99, -1], [1, 2, -1]], [12, 12], [0, 1], 8), 5, [[0, -1, -1], [1, 2, 3]], [-1, 12]),
    "no page": (fork_case([[0, -1, -1]], [12], [0], 8), 1, [[0, -1, -1]], [-1]),
    "below 0": (fork_case([[0, -7, -1]], [9], [0], 8), 1, [[0, -1, -1]], [-1]),
    "full": (fork_case([[8, 5, -1], [0, 1, -1]], [12, 12], [0, 1], 8), 9, [[8, 5, -1], [0, 1, 2]], [-1, 12]),
    # rows of one bad parent take none of the two free pages
    "children": (fork_case([[0, 77], [1, 2], [1, 2], [3, 4]], [12, 12, 12, 12], [0, 0, 1, 1], 4), 1,
                 [[0, -1], [0, -1], [1, 2], [1, 3]], [-1, -1, 12, 12]),
    # an entry that holds no tokens is not looked at
    "unused": (fork_case([[0, 99], [1, -5]], [8, 8], [0, 1], 8), 3, [[0, 2], [1, 3]], [8, 8]),
}


# (the case, room, the expected tables and lengths): lengths that are none, as an append, a commit or a fork before
# returns them for rows that did not fit; the pages of such rows are free
FAILED_LENGTHS = {
    "failed": (fork_case([[0, 1], [2, 3], [4, 5]], [12, -1, 12], [1, 0, 1], 6), 1, [[-1, -1], [0, 1], [-1, -1]], [-1, 12, -1]),
    "past the table": (fork_case([[0, 1], [2, 3]], [17, 16], [0, 1], 4), 0, [[-1, -1], [2, 3]], [-1, 16]),
    "dead parents": (fork_case([[0, 1], [2, 3]], [-1, 9], [-1, 2], 4), 1, [[-1, -1], [-1, -1]], [0, 0]),
    "pages go on": (fork_case([[0, 1], [2, 3], [2, 3]], [-1, 12, 12], [0, 1, 1], 4), 1,
                    [[-1, -1], [2, 3], [2, 0]], [-1, 12, 12]),
}


def many_short_rows(R=1100, seed=3):
    """More rows than the planning workgroup has threads, in requests of four, and fewer pages than they need."""
    g = gen(seed)
    need = R // 4 * 4
    lens = torch.randint(1, 24, (R // 4,), generator=g).repeat_interleave(4)
    tabs = torch.full((need, 4), -1, dtype=torch.int32)
    at = 0
    for r in range(0, need, 4):
        n = (int(lens[r]) + 7) // 8
        tabs[r:r + 4, :n] = torch.arange(at, at + n, dtype=torch.int32)
        at += n
    parents = torch.arange(need) // 4 * 4 + torch.randint(0, 4, (need,), generator=g)
    return *fork_case(tabs.tolist(), lens.tolist(), parents.tolist(), at + R // 2, page=8, D=8), 9


# ------------------------------------------------------------------ attention

def failed_attention(T, dt=BF16):
    """Inputs of five sequences, the second and the last of which failed before (length -1)."""
    from test_kv_sim import attn_inputs

    q, kn, vn, k, v, tabs, lens, par = attn_inputs(17, 5, T, 2, 1, 64, [40, 12, 0, 33, 20], 16, dt, slots=40)
    lens[1], lens[4] = -1, -1
    return q, kn, vn, k, v, tabs, lens, par


def attention(args, scale=None):
    """The plain form; NaN for a sequence of the length -1."""
    q, kn, vn, k, v, tabs, lens, par = args
    out, lse = C.attention(q, kn, vn, k, v, tabs, lens.clamp(min=0), par, q.shape[-1] ** -0.5 if scale is None else scale)
    out[lens == -1], lse[lens == -1] = math.nan, math.nan
    return out, lse


# shapes (T, q heads, kv heads, D, lens, page, type): both kernels, every count of waves and every kind of share
UNSEEN = [(2, 1, 1, 64, [5, 0], 16, BF16), (8, 4, 2, 128, [70, 33], 16, F16), (16, 2, 1, 96, [40], 8, BF16),
          (20, 2, 1, 64, [9], 16, BF16), (9, 4, 1, 96, [70], 16, F16), (64, 1, 1, 128, [30], 32, BF16),
          (33, 8, 1, 64, [20], 16, F16), (20, 2, 1, 256, [40], 16, BF16), (6, 2, 1, 256, [33], 16, F16)]


def unseen_garbage(T, Hq, Hkv, D, lens, page, dt, chain=False, slots=None):
    """Drafted rows as a padded batch of trees holds them: nodes that others do not see with keys and values of NaN and
    infinities (whole rows and single elements), and one of each among the values of nodes that others do see."""
    from test_kv_sim import attn_inputs

    q, kn, vn, k, v, tabs, lens, par = attn_inputs(T * D + 1, len(lens), T, Hq, Hkv, D, lens, page, dt, slots=slots)
    par[:, T - 1] = 0  # leaves: the last nodes
    vn[:, T - 1] = math.nan
    kn[:, T - 1, :, ::3] = math.inf
    if T > 4:
        par[par == T - 2] = 0
        vn[:, T - 2, :, 1::2] = math.inf
        vn[:, T - 2, :, 2] = -math.inf
        kn[:, T - 2] = math.nan
        vn[:, 1, 0, 5] = math.nan
        vn[:, 2, 0, 7] = -math.inf
    return q, kn, vn, k, v, tabs, lens, None if chain else par


def check_unseen(out, lse, args, check):
    """Values that are no numbers reach the elements of the rows that see them, and nothing else."""
    want, want_lse = attention(args)
    huge = torch.isinf(want)
    assert torch.equal(huge, torch.isinf(out)) and torch.equal(want[huge] > 0, out[huge] > 0)
    # (check takes no infinities)
    vn, v = args[2].double(), args[4].double()
    vmax = max(float(x[torch.isfinite(x)].abs().max()) for x in (vn, v))
    check(out.masked_fill(huge, 0), lse, want.masked_fill(huge, 0), want_lse, vmax, out.dtype)


def faint_tail(D, dt, n, page=32, T=1, Hq=1):
    """One token in 32 far ahead of the others, whose weights are 2^-25.5 of its: it has the values 0 and they 1000, so
    that the result is what they hold."""
    N = (n + page - 1) // page
    k = torch.zeros(N, 1, page, D, dtype=dt)
    v = torch.full((N, 1, page // 8, D, 8), 1000.0).to(dt)
    k[:, 0, 3] = 0.25
    v[:, 0, 0, :, 3] = 0.0
    q = torch.full((1, T, Hq, D), 4.0).to(dt)  # (products of D with it, and of 0)
    kn, vn = torch.zeros(1, T, 1, D, dtype=dt), torch.full((1, T, 1, D), 1000.0).to(dt)
    table = torch.arange(N, dtype=torch.int32)[None]
    return (q, kn, vn, k, v, table, torch.tensor([n], dtype=torch.int32), None), 25.5 * math.log(2) / D


def check_faint_tail(out, lse, args, scale):
    """Half a step of each weight and of the result, and where weights are below the type's least normal number half a
    step there, for weights held up to 2^9 of the largest: of tokens of 1000 over those ahead."""
    want, want_lse = attention(args, scale)
    half = torch.finfo(out.dtype).eps / 2
    least = torch.finfo(out.dtype).tiny * half * 2.0**-9
    tokens = int(args[6][0]) + out.shape[1]
    bound = (2 * half + 2**-16) * want + least * 1000 * tokens / (int(args[6][0]) // 32)
    assert ((out.double() - want).abs() <= bound).all(), (out.flatten()[0], want.flatten()[0])
    assert ((lse.double() - want_lse).abs() <= 2**-18 * (1 + want_lse.abs())).all()


def named_tokens(B, T, G, Hkv, D, lens, page, dt, seed=0):
    """A cache whose tokens have random keys and values of +-1: a query that is a token's key takes that token's value
    alone.  Returns the pools, tables, lengths, the tokens' keys and values [B][Hkv, len, D], and drafted rows of 0."""
    g = gen(seed)
    P = max(1, max((n + page - 1) // page for n in lens))
    tabs = torch.randperm(B * P + 2, generator=g)[: B * P].view(B, P).to(torch.int32)
    k = torch.zeros(B * P + 2, Hkv, page, D, dtype=dt)
    v = torch.zeros(B * P + 2, Hkv, page // 8, D, 8, dtype=dt)
    keys, values = [], []
    for b in range(B):
        n = P * page
        x, y = (torch.randint(0, 2, (Hkv, n, D), generator=g).mul(2).sub(1).to(dt) for _ in range(2))
        for i in range(P):
            k[tabs[b, i]] = x[:, i * page:(i + 1) * page]
            v[tabs[b, i]] = y[:, i * page:(i + 1) * page].view(Hkv, page // 8, 8, D).transpose(2, 3)
        keys.append(x)
        values.append(y)
    rows = torch.zeros(B, T, Hkv, D, dtype=dt)
    return k, v, tabs, torch.tensor(lens, dtype=torch.int32), keys, values, rows


def queries(keys, lens, T, G, first, step):
    """Row i of a key head asks for token (first + step i) % len of its sequence: queries [B, T, Hkv G, D] and the tokens
    [B, T, Hkv G]."""
    B, (Hkv, _, D) = len(keys), keys[0].shape
    t = torch.arange(T)[:, None, None] * G + torch.arange(G)[None, None] + 7 * torch.arange(Hkv)[None, :, None]
    q, at = torch.zeros(B, T, Hkv, G, D, dtype=keys[0].dtype), []
    for b in range(B):
        tok = (first + step * t) % int(lens[b])
        for h in range(Hkv):
            q[b, :, h] = keys[b][h, tok[:, h]]
        at.append(tok)
    return q.view(B, T, Hkv * G, D), torch.stack(at)


def check_named(out, at, values):
    # the others' weights: a product at most 3/4 D of a token's own D at these sizes, so e^(-D / 4 scale) each
    B, T, Hkv, G = at.shape
    out = out.view(B, T, Hkv, G, -1)
    for b in range(B):
        for h in range(Hkv):
            assert ((out[b, :, h].double() - values[b][h, at[b, :, h]].double()).abs() < 2**-7).all(), (b, h)


def one_value(T, G, D, dt, n=160, page=32):
    """Every value is one number of the type, just below 2: whatever the weights are, so is every result.  One token
    comes late and lies up to 2^5.9 above the first, by a different factor in every row, and the others 2^30 below."""
    N = n // page
    c = 2 - 2 * torch.finfo(dt).eps
    k = torch.zeros(N, 1, page, D, dtype=dt)
    k[..., 1] = -30
    k[0, 0, 1] = 0
    k[N - 1, 0, 2] = 0
    k[N - 1, 0, 2, 0] = 1
    v = torch.full((N, 1, page // 8, D, 8), c).to(dt)
    q = torch.zeros(1, T, G, D, dtype=dt)
    q[..., 0] = (5.9 * (torch.arange(T * G) + 1) / (T * G)).view(1, T, G)
    q[..., 1] = 1
    kn, vn = torch.zeros(1, T, 1, D, dtype=dt), torch.full((1, T, 1, D), c).to(dt)
    kn[..., 1] = -30
    table = torch.arange(N, dtype=torch.int32)[None]
    return (q, kn, vn, k, v, table, torch.tensor([n], dtype=torch.int32), None), math.log(2), c
