"""Inputs and plain 64-bit forms for the 8-bit cache and the position rotation,
and one way to make each call on the simulation (CPU)."""
from __future__ import annotations

import math

import torch

import kv_cases as C

BF16, F16 = torch.bfloat16, torch.float16
E4M3, E8M0, U8, I32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.uint8, torch.int32
FLOOR = {BF16: -100, F16: -15}
CAP = {BF16: 1.875 * 2.0**127, F16: 61440.0}
BLOCK = 16


# ------------------------------------------------------------------ blocks

def numbers(codes, scale_bytes):
    """float64 of e4m3 codes and scale bytes (broadcast): 255 is NaN."""
    s = torch.where(scale_bytes == 255, math.nan, torch.exp2(scale_bytes.double() - 127))
    return codes.view(E4M3).double() * s


def need(x, dt):
    """Exponent of the smallest scale of a block's new numbers (any shape), from its definition."""
    x = x[torch.isfinite(x)].abs().clamp(max=CAP[dt])
    e = FLOOR[dt]
    if x.numel():
        while float(x.max()) > 448.0 * 2.0**e:
            e += 1
    return e


def encode(x, e, dt=None):
    """float64 numbers to codes of the scale 2^e (dt: new numbers, with their type's cap)."""
    if dt is not None:
        x = torch.where(torch.isfinite(x), x.clamp(-CAP[dt], CAP[dt]), math.nan)
    y = x * 2.0**-e
    # to the nearest by the grid of a number's own exponent, ties to even
    q = torch.exp2((torch.frexp(y.abs()).exponent - 4).clamp(min=-9).double())
    y = (y / q).round() * q
    return y.float().to(E4M3).view(U8)


def block(pools, layer, pg, h, i):
    """(keys [16, D], values [16, D], scales [2]) of block i of a page: views of the pools' bytes."""
    k, v, s = pools
    return k[layer, pg, h, i * BLOCK:(i + 1) * BLOCK], v[layer, pg, h, i].t(), s[layer, pg, h, i]


def pools(g, L, N, H, page, D, dt, spread=1.0):
    """Encoded random pools, as bytes."""
    k = torch.empty(L, N, H, page, D, dtype=U8)
    v = torch.empty(L, N, H, page // BLOCK, D, BLOCK, dtype=U8)
    s = torch.empty(L, N, H, page // BLOCK, 2, dtype=U8)
    x = torch.randn(2, L, N, H, page // BLOCK, BLOCK, D, generator=g).double()
    x = (x * torch.exp2(spread * torch.randn(2, L, N, H, page // BLOCK, 1, 1, generator=g).double())).to(dt).double()
    most = x.abs().amax((-1, -2)).clamp(max=CAP[dt])
    e = torch.ceil(torch.log2(most / 448)).clamp(min=FLOOR[dt])
    codes = torch.empty(x.shape, dtype=U8)
    for c in range(2):
        y = x[c] * torch.exp2(-e[c])[..., None, None]
        q = torch.exp2((torch.frexp(y.abs()).exponent - 4).clamp(min=-9).double())
        codes[c] = ((y / q).round() * q).float().to(E4M3).view(U8)
        s[..., c] = (e[c] + 127).to(U8)
    k[:] = codes[0].reshape(k.shape)
    v[:] = codes[1].transpose(-1, -2)
    return k, v, s


def as_tensors(p):
    return p[0].view(E4M3), p[1].view(E4M3), p[2].view(E8M0)


def same(a, b):
    """Codes are alike where they are the same number or both NaN."""
    nan_a, nan_b = (a & 0x7F) == 0x7F, (b & 0x7F) == 0x7F
    return torch.equal(nan_a, nan_b) and torch.equal(torch.where(nan_a, 0, a), torch.where(nan_b, 0, b))


# ------------------------------------------------------------------ plain forms

def turned(x, position, freq, pairs):
    """One row's heads x [..., D] in float64, turned."""
    y = x.clone()
    for j, f in enumerate(freq.tolist()):
        a, b = (2 * j, 2 * j + 1) if pairs else (j, j + len(freq))
        c, s = math.cos(position * f), math.sin(position * f)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def write(k_new, v_new, p, tabs, lens, nodes, dt, freq=None, pairs=False):
    """nodes: per sequence the rows written (None: the sequence fails).  Returns the pools' bytes, the lengths, and the
    float64 numbers written: {(layer, page, head, block, which): (first, [tokens, D])}."""
    p = [x.clone() for x in p]
    L, _, _, H, D = k_new.shape
    page = p[0].shape[3]
    out, put = lens.clone(), {}
    for b, rows in enumerate(nodes):
        if rows is None:
            out[b] = -1
            continue
        n0, n1 = int(lens[b]), int(lens[b]) + len(rows)
        out[b] = n1
        for blk in range(n0 // BLOCK, (n1 - 1) // BLOCK + 1 if rows else 0):
            lo, hi = max(n0 - blk * BLOCK, 0), min(n1 - blk * BLOCK, BLOCK)
            pg = int(tabs[b, blk * BLOCK // page])
            idx = torch.tensor(rows[blk * BLOCK + lo - n0:blk * BLOCK + hi - n0])
            for layer in range(L):
                kx, vx = k_new[layer, b, idx].double(), v_new[layer, b, idx].double()  # [tokens, H, D]
                if freq is not None:
                    kx = torch.stack([turned(kx[i], blk * BLOCK + lo + i, freq, pairs) for i in range(len(idx))])
                for h in range(H):
                    kc, vc, s = block(p, layer, pg, h, blk * BLOCK % page // BLOCK)
                    for which, x, codes in ((0, kx[:, h], kc), (1, vx[:, h], vc)):
                        e = need(x, dt)
                        if lo:
                            old = int(s[which]) - 127
                            if old > e:
                                e = old
                            elif e > old:
                                codes[:lo] = encode(numbers(codes[:lo].contiguous(), torch.tensor(old + 127)), e)
                        codes[lo:hi] = encode(x, e, dt)
                        s[which] = e + 127
                        put[layer, pg, h, blk * BLOCK % page // BLOCK, which] = (lo, x)
    return p, out, put


def fits(tabs, lens, counts, T, page, N):
    return [C._fits(tabs[b].tolist(), int(lens[b]), int(counts[b]), T, page, N) for b in range(len(lens))]


def append(k_new, v_new, p, tabs, lens, counts, dt, freq=None, pairs=False):
    T = k_new.shape[2]
    c = torch.full_like(lens, T) if counts is None else counts
    ok = fits(tabs, lens, c, T, p[0].shape[3], p[0].shape[1])
    return write(k_new, v_new, p, tabs, lens, [list(range(int(n))) if f else None for n, f in zip(c, ok)], dt, freq, pairs)


def commit(k_new, v_new, p, tabs, lens, parents, draft, sampled, dt):
    B, T = parents.shape
    o = dict(n_acc=torch.zeros(B, dtype=I32), tokens=torch.full((B, T), -1, dtype=I32), path=torch.full((B, T), -1, dtype=I32))
    nodes = []
    for b in range(B):
        at = [0]
        while True:
            more = [j for j in range(at[-1] + 1, T) if parents[b, j] == at[-1] and draft[b, j] == sampled[b, at[-1]]]
            if not more:
                break
            at.append(more[0])
        c = len(at)
        o["n_acc"][b] = c - 1
        o["path"][b, :c] = torch.tensor(at, dtype=I32)
        o["tokens"][b, :c] = torch.tensor([int(draft[b, j]) for j in at[1:]] + [int(sampled[b, at[-1]])], dtype=I32)
        nodes.append(at)
    ok = fits(tabs, lens, torch.tensor([len(x) for x in nodes]), T, p[0].shape[3], p[0].shape[1])
    q, lens_out, _ = write(k_new, v_new, p, tabs, lens, [x if f else None for x, f in zip(nodes, ok)], dt)
    return q, o | dict(lens=lens_out)


def fork(p, tabs, lens, parents, room):
    """The 16-bit form's tables and lengths; a row that got another page than its parent's has copies of whole blocks."""
    import kv_edges as E

    N, page = p[0].shape[1], p[0].shape[3]
    k, v = torch.zeros(1, N, 1, page, 8), torch.zeros(1, N, 1, page // 8, 8, 8)
    _, _, to, out = E.fork(k, v, tabs, lens, parents, room)
    q = [x.clone() for x in p]
    for r in range(len(parents)):
        par = int(parents[r])
        n = int(lens[par]) if 0 <= par < len(parents) else -1
        if n <= 0 or n > tabs.shape[1] * page or n % page == 0:
            continue
        a, z = int(tabs[par, n // page]), int(to[r, n // page])
        if z >= 0 and a != z:
            nb = (n % page + BLOCK - 1) // BLOCK
            q[0][:, z, :, :nb * BLOCK] = p[0][:, a, :, :nb * BLOCK]
            q[1][:, z, :, :nb], q[2][:, z, :, :nb] = p[1][:, a, :, :nb], p[2][:, a, :, :nb]
    return q, to, out


def decoded(p):
    """The layer's pools as a 16-bit cache of the type float64: keys [N, H, page, D], values [N, H, page / 8, D, 8]."""
    k, v, s = p
    N, H, page, D = k.shape
    kd = numbers(k.unflatten(2, (-1, BLOCK)), s[..., 0, None, None]).reshape(N, H, page, D)
    vd = numbers(v, s[..., 1, None, None]).transpose(-1, -2).reshape(N, H, page // 8, 8, D).transpose(-1, -2).contiguous()
    return kd, vd


def rotate(x, lens, parents, freq, pairs):
    """Rows x [B, T, heads, D] at their positions, float64."""
    B, T = x.shape[:2]
    y = torch.empty(x.shape, dtype=torch.float64)
    for b in range(B):
        for t in range(T):
            d = t if parents is None else int(C.ancestor_mask(parents[b].tolist())[t].sum()) - 1
            y[b, t] = turned(x[b, t].double(), max(int(lens[b]), 0) + d, freq, pairs)
    return y


# ------------------------------------------------------------------ what a rotated row may be off by

# A turned number is two products of 32 bits and their sum, of a cosine and a sine off by 2^-24 (their rounding to 32
# bits, and less than that by their polynomials): below 2^-22 of the pair's larger magnitude, times two.
TURN = 2.0**-21


def pair_size(x, n, pairs):
    """Of each number the sum of its pair's magnitudes (0 where a row does not turn); x [..., D], n pairs."""
    y = torch.zeros_like(x)
    if n:
        a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if pairs else (x[..., :n], x[..., n:2 * n])
        m = a.abs() + b.abs()
        if pairs:
            y[..., 0:2 * n:2], y[..., 1:2 * n:2] = m, m
        else:
            y[..., :n], y[..., n:2 * n] = m, m
    return y


def check_turned16(got, want, n, pairs):
    """16-bit rows: half a step of the result, and the turn's own error."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * half  # half a step below the normal numbers
    slack = TURN * pair_size(want, n, pairs)
    assert ((got.double() - want).abs() <= half * (want.abs() + slack) + slack + tiny).all()


def check_written(before, got, want, put, dt, n=0, pairs=False):
    """Pools after a write: bytes equal to the plain form's, but where keys turn (n pairs): there the numbers are
    within a rounding of the exact ones, and a scale may differ where the largest magnitude lies at its border."""
    if n == 0:
        assert same(got[0], want[0]) and same(got[1], want[1]) and torch.equal(got[2], want[2])
        return
    assert same(got[1], want[1]) and torch.equal(got[2][..., 1], want[2][..., 1])
    rest = torch.ones(got[2].shape[:-1], dtype=torch.bool)
    for (layer, pg, h, i, which), (lo, x) in put.items():
        if which:
            continue
        rest[layer, pg, h, i] = False
        gk, gs = got[0][layer, pg, h, i * BLOCK:(i + 1) * BLOCK], int(got[2][layer, pg, h, i, 0])
        wk, ws = want[0][layer, pg, h, i * BLOCK:(i + 1) * BLOCK], int(want[2][layer, pg, h, i, 0])
        hi = lo + len(x)
        assert torch.equal(gk[hi:], wk[hi:])  # behind the last token
        if gs != ws:
            m = float(x[torch.isfinite(x)].abs().max())
            assert need(torch.tensor([m * (1 + 2 * TURN)], dtype=torch.float64), dt) != need(
                torch.tensor([m * (1 - 2 * TURN)], dtype=torch.float64), dt), (m, gs, ws)
        else:
            assert same(gk[:lo], wk[:lo])
        slack = TURN * pair_size(x, n, pairs)
        err = (numbers(gk[lo:hi].contiguous(), torch.tensor(gs)) - x).abs()
        assert (err <= 2.0**-4 * (x.abs() + slack) + slack + 2.0**(gs - 127 - 10)).all(), float(err.max())
    gk, wk = (y[0].unflatten(3, (-1, BLOCK)) for y in (got, want))
    assert torch.equal(gk[rest], wk[rest]) and torch.equal(got[2][rest], want[2][rest])


# ------------------------------------------------------------------ calls on the simulation

def cache_meta(p, dt):
    k, v, s = p
    L, N, H, page, D = k.shape
    return dict(layers=L, pages=N, kv_heads=H, page=page, D=D, dtype=C.CODE[dt], k_layer=k.stride(0) if L > 1 else 0,
                k_page=k.stride(1), v_layer=v.stride(0) if L > 1 else 0, v_page=v.stride(1),
                s_layer=s.stride(0) if L > 1 else 0, s_page=s.stride(1))


def rot_meta(freq, pairs):
    return dict(dims=0 if freq is None else 2 * len(freq), pairs=int(pairs))


def sim_attention(sim, q, k_new, v_new, p, tabs, lens, parents, scale=None, max_len=None, want_lse=True, **kw):
    B, T, Hq, D = q.shape
    meta = cache_meta([x[None] for x in p], q.dtype) | C._rows_meta(k_new[None], v_new[None]) | C._strides(q, ("qs", "qt", "qh"))
    o = dict(o_out=torch.zeros(B, T, Hq, D, dtype=q.dtype), o_lse=torch.zeros(B, T, Hq) if want_lse else None)
    rc, out = sim.call("attn8", dict(q=q, k_new=k_new, v_new=v_new, k=p[0], v=p[1], scales=p[2], tables=tabs, lens=lens,
                                     parents=parents, **o), B=B, P=tabs.shape[1], T=T, Hq=Hq,
                       scale=D ** -0.5 if scale is None else scale,
                       max_len=tabs.shape[1] * p[0].shape[2] if max_len is None else max_len, **meta, **kw)
    return rc, out["o_out"], out.get("o_lse")


def sim_append(sim, k_new, v_new, p, tabs, lens, counts, freq=None, pairs=False, **kw):
    rc, o = sim.call("append8", dict(k_new=k_new, v_new=v_new, k=p[0], v=p[1], scales=p[2], tables=tabs, lens=lens, counts=counts,
                                     freq=freq, o_lens=torch.zeros_like(lens)), B=tabs.shape[0], P=tabs.shape[1], T=k_new.shape[2],
                     **cache_meta(p, k_new.dtype), **C._rows_meta(k_new, v_new), **rot_meta(freq, pairs), **kw)
    return rc, [o["k"], o["v"], o["scales"]], o["o_lens"]


def sim_append_rotated(sim, k_new, v_new, k, v, tabs, lens, counts, freq, pairs, **kw):
    rc, o = sim.call("append_rotated", dict(k_new=k_new, v_new=v_new, k=k, v=v, tables=tabs, lens=lens, counts=counts, freq=freq,
                                            o_lens=torch.zeros_like(lens)), B=tabs.shape[0], P=tabs.shape[1], T=k_new.shape[2],
                     **C._cache_meta(k, v), **C._rows_meta(k_new, v_new), **rot_meta(freq, pairs), **kw)
    return rc, o["k"], o["v"], o["o_lens"]


def sim_commit(sim, k_new, v_new, p, tabs, lens, parents, draft, sampled, **kw):
    B, T = parents.shape
    rc, o = sim.call("commit8", dict(k_new=k_new, v_new=v_new, k=p[0], v=p[1], scales=p[2], tables=tabs, lens=lens, parents=parents,
                                     draft=draft, sampled=sampled, o_n_acc=torch.zeros(B, dtype=I32),
                                     o_tokens=torch.zeros(B, T, dtype=I32), o_path=torch.zeros(B, T, dtype=I32),
                                     o_lens=torch.zeros(B, dtype=I32)), B=B, P=tabs.shape[1], T=T,
                     **cache_meta(p, k_new.dtype), **C._rows_meta(k_new, v_new), **kw)
    return rc, [o["k"], o["v"], o["scales"]], {x: o["o_" + x] for x in ("n_acc", "tokens", "path", "lens")}


def sim_fork(sim, p, tabs, lens, parents, room, **kw):
    rc, o = sim.call("fork8", dict(k=p[0], v=p[1], scales=p[2], tables=tabs, lens=lens, parents=parents,
                                   o_tables=torch.zeros_like(tabs), o_lens=torch.zeros_like(lens)), B=tabs.shape[0],
                     P=tabs.shape[1], room=room, **cache_meta(p, BF16), **kw)
    return rc, [o["k"], o["v"], o["scales"]], o["o_tables"], o["o_lens"]


def _copy(t):
    """A copy of the same strides."""
    n = 1 + sum((a - 1) * b for a, b in zip(t.shape, t.stride()))
    return torch.as_strided(torch.as_strided(t, (n,), (1,)).clone(), t.shape, t.stride())


def sim_rotate(sim, q, k_new, lens, parents, freq, pairs, here=False, **kw):
    """here: in place."""
    B, T, Hq, D = q.shape
    oq = _copy(q) if here else torch.zeros(q.shape, dtype=q.dtype)
    ok = None if k_new is None else _copy(k_new) if here else torch.zeros(k_new.shape, dtype=q.dtype)
    meta = C._strides(q, ("qs", "qt", "qh")) | C._strides(oq, ("oqs", "oqt", "oqh")) | dict(Hk=0)
    if k_new is not None:
        meta |= C._strides(k_new, ("ks", "kt", "kh")) | C._strides(ok, ("oks", "okt", "okh")) | dict(Hk=k_new.shape[2])
    rc, o = sim.call("rotate", dict(q=q, k_new=k_new, o_q=oq, o_k=ok, lens=lens, parents=parents, freq=freq), B=B, T=T, Hq=Hq, D=D,
                     dtype=C.CODE[q.dtype], here=int(here), **meta, **rot_meta(freq, pairs), **kw)
    return rc, o["o_q"], o.get("o_k")
