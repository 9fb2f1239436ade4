"""Inputs and plain 64-bit forms for the beam, tree-attention and cache tests,
and one way to make each call on the simulation (CPU) or through the sampler
(GPU)."""
from __future__ import annotations

import math

import torch

CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


# ------------------------------------------------------------------ inputs

def pools(g, L, N, H, page, D, dt, scale=1.0):
    k = (torch.randn(L, N, H, page, D, generator=g) * scale).to(dt)
    v = torch.randn(L, N, H, page // 8, D, 8, generator=g).to(dt)
    return k, v


def tables(g, B, P, spare=2):
    N = B * P + spare
    return torch.randperm(N, generator=g)[: B * P].view(B, P).to(torch.int32), N


def tree(g, B, T):
    """Random parents (an earlier node each), node 0 the root."""
    par = (torch.rand(B, T, generator=g) * torch.arange(T)).long()
    par[:, 0] = -1
    return par.to(torch.int32)


def ancestor_mask(parents):
    """bool [T, T] of one tree: j is i or an ancestor of i (parents that are no earlier node make roots)."""
    T = len(parents)
    m = torch.zeros(T, T, dtype=torch.bool)
    for i in range(T):
        j = i
        while j >= 0:
            m[i, j] = True
            j = parents[j] if parents[j] < j else -1
    return m


# ------------------------------------------------------------------ plain forms

def beam(logits, scores, W, n, hist=None, hist_len=None):
    x = logits.double()
    rows, V = x.shape
    G = rows // W
    out = dict(scores=torch.full((G * n,), -math.inf, dtype=torch.float64), parents=torch.full((G * n,), -1, dtype=torch.int32),
               tokens=torch.full((G * n,), -1, dtype=torch.int32))
    if hist is not None:
        H = hist.shape[1]
        out["hist"] = torch.full((G * n, H), -1, dtype=torch.int32)
        out["hist_len"] = torch.zeros(G * n, dtype=torch.int32)
    for r in range(G):
        cand = []
        for w in range(W):
            row = x[r * W + w]
            s = float(scores[r * W + w])
            ok = ~torch.isnan(row) & (row > -math.inf)
            if not math.isfinite(s) or not ok.any() or torch.isinf(row[ok]).any():
                continue
            total = s + (row - torch.logsumexp(row[ok], 0))
            keep = torch.nonzero(ok)[:, 0]
            order = sorted(keep.tolist(), key=lambda v: (-float(row[v]), v))[:n]
            cand += [(-float(total[v]), w, i, v) for i, v in enumerate(order)]
        cand.sort()
        for i, (neg, w, _, v) in enumerate(cand[:n]):
            at, p = r * n + i, r * W + w
            out["scores"][at], out["parents"][at], out["tokens"][at] = -neg, p, v
            if hist is not None:
                have = min(max(int(hist_len[p]), 0), H)
                h = (hist[p, :have].tolist() + [v])[-H:]
                out["hist"][at, : len(h)] = torch.tensor(h, dtype=torch.int32)
                out["hist_len"][at] = len(h)
    return out


def attention(q, k_new, v_new, k, v, tabs, lens, parents, scale):
    """q [B, T, Hq, D], one layer's pools; float64 out and lse.  NaN for a sequence with a page outside the pool."""
    B, T, Hq, D = q.shape
    N, H, page, _ = k.shape
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    lse = torch.zeros(B, T, Hq, dtype=torch.float64)
    for b in range(B):
        n = min(max(int(lens[b]), 0), tabs.shape[1] * page)
        pg = tabs[b, : (n + page - 1) // page].long()
        if ((pg < 0) | (pg >= N)).any():
            out[b], lse[b] = math.nan, math.nan
            continue
        par = parents[b].tolist() if parents is not None else list(range(-1, T - 1))
        bar = torch.cat([torch.ones(T, n, dtype=torch.bool), ancestor_mask(par)], 1)
        for h in range(H):
            kk = torch.cat([k[pg, h].reshape(-1, D)[:n], k_new[b, :, h]]).double()
            vv = torch.cat([v[pg, h].transpose(2, 3).reshape(-1, D)[:n], v_new[b, :, h]]).double()
            for i in range(h * (Hq // H), (h + 1) * (Hq // H)):
                x = (q[b, :, i].double() @ kk.T * scale).masked_fill(~bar, -math.inf)
                w = torch.softmax(x, 1).masked_fill(~bar, 0.0)
                for t in range(T):  # (values of masked tokens are not used, whatever they are)
                    out[b, t, i] = w[t, bar[t]] @ vv[bar[t]]
                lse[b, :, i] = torch.logsumexp(x, 1)
    return out, lse


def _put(k, v, k_new, v_new, b, node, page_id, slot):
    k[:, page_id, :, slot] = k_new[:, b, node]
    v[:, page_id, :, slot // 8, :, slot % 8] = v_new[:, b, node]


def _fits(tabs_b, n0, count, T, page, N):
    if not 0 <= count <= T or n0 < 0 or n0 + count > len(tabs_b) * page:
        return False
    return all(0 <= tabs_b[p // page] < N for p in range(n0, n0 + count))


def append(k_new, v_new, k, v, tabs, lens, counts):
    k, v = k.clone(), v.clone()
    _, B, T = k_new.shape[:3]
    N, page = k.shape[1], k.shape[3]
    out = lens.clone()
    for b in range(B):
        c, n0, t = T if counts is None else int(counts[b]), int(lens[b]), tabs[b].tolist()
        if not _fits(t, n0, c, T, page, N):
            out[b] = -1
            continue
        for i in range(c):
            _put(k, v, k_new, v_new, b, i, t[(n0 + i) // page], (n0 + i) % page)
        out[b] = n0 + c
    return k, v, out


def commit(k_new, v_new, k, v, tabs, lens, parents, draft, sampled):
    k, v = k.clone(), v.clone()
    _, B, T = k_new.shape[:3]
    N, page = k.shape[1], k.shape[3]
    o = dict(n_acc=torch.zeros(B, dtype=torch.int32), tokens=torch.full((B, T), -1, dtype=torch.int32),
             path=torch.full((B, T), -1, dtype=torch.int32), lens=lens.clone())
    for b in range(B):
        nodes = [0]
        while True:
            more = [j for j in range(nodes[-1] + 1, T) if parents[b, j] == nodes[-1] and draft[b, j] == sampled[b, nodes[-1]]]
            if not more:
                break
            nodes.append(more[0])
        c, n0, t = len(nodes), int(lens[b]), tabs[b].tolist()
        o["n_acc"][b] = c - 1
        o["path"][b, :c] = torch.tensor(nodes, dtype=torch.int32)
        o["tokens"][b, : c] = torch.tensor([int(draft[b, j]) for j in nodes[1:]] + [int(sampled[b, nodes[-1]])], dtype=torch.int32)
        if not _fits(t, n0, c, T, page, N):
            o["lens"][b] = -1
            continue
        for i, node in enumerate(nodes):
            _put(k, v, k_new, v_new, b, node, t[(n0 + i) // page], (n0 + i) % page)
        o["lens"][b] = n0 + c
    return k, v, o


def fork(k, v, tabs, lens, parents, room):
    k, v = k.clone(), v.clone()
    R, P = tabs.shape
    N, page = k.shape[1], k.shape[3]
    cap = P * page
    to, out = torch.full((R, P), -1, dtype=torch.int32), torch.zeros(R, dtype=torch.int32)
    rows = []
    for r in range(R):
        p = int(parents[r])
        n = int(lens[p]) if 0 <= p < R else -1
        if n < 0 or n > cap:
            rows.append(None)
            continue
        rows.append((tabs[p].tolist(), n, n // page, min((n + room + page - 1) // page, P)))
    shared, first = set(), {}
    for row in rows:
        if row:
            shared.update(x for x in row[0][: row[2]] if 0 <= x < N)
    for r, row in enumerate(rows):
        if row:
            for i in range(row[2], row[3]):
                x = row[0][i]
                if 0 <= x < N and x not in shared:
                    first.setdefault(x, (r, i))
    free = [x for x in range(N) if x not in shared and x not in first]
    at = 0
    for r, row in enumerate(rows):
        if row is None:
            continue
        t, n, full, end = row
        to[r, :full] = torch.tensor(t[:full], dtype=torch.int32)
        need = [i for i in range(full, end) if not (0 <= t[i] < N and first.get(t[i]) == (r, i))]
        fits = at + len(need) <= len(free)
        for i in range(full, end):
            if i not in need:
                to[r, i] = t[i]
                continue
            if fits:
                to[r, i] = free[at]
                held = min(n - i * page, page)
                if held > 0 and 0 <= t[i] < N:
                    nb = (held + 7) // 8
                    k[:, free[at], :, : nb * 8] = k[:, t[i], :, : nb * 8].clone()
                    v[:, free[at], :, :nb] = v[:, t[i], :, :nb].clone()
                at += 1
        if not fits:
            at += len(need)
        out[r] = n if fits and n + room <= cap else -1
    return k, v, to, out


# ------------------------------------------------------------------ calls on the simulation

def _strides(t, names):
    return dict(zip(names, t.stride()))


def _cache_meta(k, v):
    L, N, H, page, D = k.shape
    return dict(layers=L, pages=N, kv_heads=H, page=page, D=D, dtype=CODE[k.dtype], k_layer=k.stride(0) if L > 1 else 0,
                k_page=k.stride(1), v_layer=v.stride(0) if L > 1 else 0, v_page=v.stride(1))


def _rows_meta(k_new, v_new):
    return _strides(k_new, ("kl", "ks", "kt", "kh")) | _strides(v_new, ("vl", "vs", "vt", "vh"))


def sim_beam(sim, logits, scores, W, n, hist=None, hist_len=None, V=None, **kw):
    rows = logits.shape[0]
    V = logits.shape[1] if V is None else V
    G, i32 = rows // W, torch.int32
    o = dict(o_scores=torch.zeros(G * n), o_parents=torch.zeros(G * n, dtype=i32), o_tokens=torch.zeros(G * n, dtype=i32))
    if hist is not None:
        o |= dict(o_hist=torch.zeros(G * n, hist.shape[1], dtype=i32), o_hist_len=torch.zeros(G * n, dtype=i32))
    rc, out = sim.call("beam", dict(logits=logits, scores=scores, hist=hist, hist_len=hist_len, **o), G=G, W=W, V=V, n=n,
                       stride=logits.stride(0), dtype=CODE[logits.dtype], H=0 if hist is None else hist.shape[1], **kw)
    return rc, {k[2:]: x for k, x in out.items()}


def sim_attention(sim, q, k_new, v_new, k, v, tabs, lens, parents, scale=None, max_len=None, want_lse=True, **kw):
    B, T, Hq, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    meta = _cache_meta(k[None], v[None]) | _rows_meta(k_new[None], v_new[None]) | _strides(q, ("qs", "qt", "qh"))
    o = dict(o_out=torch.zeros(B, T, Hq, D, dtype=q.dtype), o_lse=torch.zeros(B, T, Hq) if want_lse else None)
    rc, out = sim.call("attn", dict(q=q, k_new=k_new, v_new=v_new, k=k, v=v, tables=tabs, lens=lens, parents=parents, **o), B=B,
                       P=tabs.shape[1], T=T, Hq=Hq, scale=scale,
                       max_len=tabs.shape[1] * k.shape[2] if max_len is None else max_len, **meta, **kw)
    return rc, out["o_out"], out.get("o_lse")


def sim_append(sim, k_new, v_new, k, v, tabs, lens, counts, **kw):
    rc, o = sim.call("append", dict(k_new=k_new, v_new=v_new, k=k, v=v, tables=tabs, lens=lens, counts=counts,
                                    o_lens=torch.zeros_like(lens)), B=tabs.shape[0], P=tabs.shape[1], T=k_new.shape[2],
                     **_cache_meta(k, v), **_rows_meta(k_new, v_new), **kw)
    return rc, o["k"], o["v"], o["o_lens"]


def sim_commit(sim, k_new, v_new, k, v, tabs, lens, parents, draft, sampled, **kw):
    B, T = parents.shape
    i32 = torch.int32
    rc, o = sim.call("commit", dict(k_new=k_new, v_new=v_new, k=k, v=v, tables=tabs, lens=lens, parents=parents, draft=draft,
                                    sampled=sampled, o_n_acc=torch.zeros(B, dtype=i32), o_tokens=torch.zeros(B, T, dtype=i32),
                                    o_path=torch.zeros(B, T, dtype=i32), o_lens=torch.zeros(B, dtype=i32)),
                     B=B, P=tabs.shape[1], T=T, **_cache_meta(k, v), **_rows_meta(k_new, v_new), **kw)
    return rc, o["k"], o["v"], {x: o["o_" + x] for x in ("n_acc", "tokens", "path", "lens")}


def sim_fork(sim, k, v, tabs, lens, parents, room, **kw):
    rc, o = sim.call("fork", dict(k=k, v=v, tables=tabs, lens=lens, parents=parents, o_tables=torch.zeros_like(tabs),
                                  o_lens=torch.zeros_like(lens)), B=tabs.shape[0], P=tabs.shape[1], room=room,
                     **_cache_meta(k, v), **kw)
    return rc, o["k"], o["v"], o["o_tables"], o["o_lens"]
