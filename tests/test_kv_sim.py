"""The beam, tree-attention and cache kernels on the CPU simulation under
AddressSanitizer, against plain forms in 64 bits: odd sizes, strides, empty
and single-token sequences, garbage past a sequence's end, bad pages."""
import importlib.util
import math
import os

import pytest
import torch

import kv_cases as C

HERE = os.path.dirname(os.path.abspath(__file__))
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def sim():
    spec = importlib.util.spec_from_file_location("kv_sim", os.path.join(HERE, "kv_sim", "sim.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.build()
    return m


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ beams

def beam_inputs(g, G, W, V, dt, H=0, spread=3.0, pad=0):
    x = torch.randn(G * W, V + pad, generator=g) * spread
    x = x.to(dt)
    scores = -10 * torch.rand(G * W, generator=g)
    if not H:
        return x, scores, None, None
    hist = torch.randint(0, V, (G * W, H), generator=g).to(torch.int32)
    hl = torch.randint(0, H + 1, (G * W,), generator=g).to(torch.int32)
    return x, scores, hist, hl


def check_beam(rc, got, want):
    assert rc == 0
    for k in want:
        if k == "scores":
            # a total of one 32-bit rounding, and of the logsumexp's sum of 32-bit exponentials (relative 2^-21 at most)
            w = want[k]
            fin = torch.isfinite(w)
            assert torch.equal(fin, torch.isfinite(got[k]))
            assert ((got[k].double() - w).abs()[fin] <= w.abs()[fin] * 2**-24 + 2**-21).all()
        else:
            assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("G,W,V,n,dt,H", [
    (1, 1, 1, 1, F32, 0), (2, 3, 37, 5, BF16, 4), (1, 4, 2500, 8, F32, 1), (1, 2, 4999, 64, BF16, 0), (1, 5, 300, 10, F32, 7),
    (1, 1, 16500, 2, F32, 0)])
def test_beam(sim, G, W, V, n, dt, H):
    x, scores, hist, hl = beam_inputs(gen(V + n), G, W, V, dt, H, pad=3)
    rc, got = C.sim_beam(sim, x, scores, W, n, hist, hl, V=V)
    check_beam(rc, got, C.beam(x[:, :V], scores, W, n, hist, hl))


def test_beam_equal_logits_ended_beams_and_rows_that_give_nothing(sim):
    g = gen(5)
    x, scores, hist, hl = beam_inputs(g, 5, 3, 2100, F32, 2)
    x[0] = 1.5                      # more equal logits than the candidate buffer holds
    x[1] = x[0]                     # and an equal beam of equal score
    scores[1] = scores[0]
    scores[2] = -math.inf           # ended
    x[3, 7], x[4, :] = math.nan, math.nan
    x[5, 11] = math.inf
    x[6:9] = -math.inf              # a request with one id in all
    x[7, 2099] = -3.0
    scores[9:12] = -math.inf        # and one with nothing
    x[12:15, 5:] = -math.inf
    x[12:15, :5] = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 0.0])
    scores[12:15] = -1.0
    rc, got = C.sim_beam(sim, x, scores, 3, 6, hist, hl)
    check_beam(rc, got, C.beam(x, scores, 3, 6, hist, hl))


# ------------------------------------------------------------------ attention

def attn_inputs(seed, B, T, Hq, Hkv, D, lens, page, dt, strided=False, slots=None):
    g = gen(seed)
    P = slots or max(1, max((n + page - 1) // page for n in lens))
    tabs, N = C.tables(g, B, P)
    k, v = C.pools(g, 1, N, Hkv, page, D, dt)
    k, v = k[0], v[0]
    q = (torch.randn(B, T, Hq, D, generator=g) * 2).to(dt)
    kn, vn = (torch.randn(B, T, Hkv, D, generator=g).to(dt) for _ in range(2))
    if strided:  # slices of one projection, at any alignment
        w = torch.randn(B, T, (Hq + 2 * Hkv) * D + 3, generator=g).to(dt)
        w[..., 1:1 + Hq * D] = q.view(B, T, -1)
        w[..., 1 + Hq * D: 1 + (Hq + Hkv) * D] = kn.view(B, T, -1)
        w[..., 1 + (Hq + Hkv) * D: 1 + (Hq + 2 * Hkv) * D] = vn.view(B, T, -1)
        q = w[..., 1:1 + Hq * D].unflatten(-1, (Hq, D))
        kn = w[..., 1 + Hq * D: 1 + (Hq + Hkv) * D].unflatten(-1, (Hkv, D))
        vn = w[..., 1 + (Hq + Hkv) * D: 1 + (Hq + 2 * Hkv) * D].unflatten(-1, (Hkv, D))
    lens = torch.tensor(lens, dtype=torch.int32)
    parents = C.tree(g, B, T)
    # past a sequence's end: NaN, infinities; slots past it: no page
    for b in range(B):
        n = int(lens[b])
        for i in range(P):
            p = int(tabs[b, i])
            held = min(max(n - i * page, 0), page)
            k[p, :, held:] = math.nan
            x = v[p].transpose(2, 3).reshape(Hkv, page, D).clone()
            x[:, held:] = math.inf
            v[p] = x.view(Hkv, page // 8, 8, D).transpose(2, 3)
            if held == 0:
                tabs[b, i] = -1 if i % 2 else N + 5
    return q, kn, vn, k, v, tabs, lens, parents


def check_attn(out, lse, want, want_lse, vmax, dt):
    # P and the output are rounded to 16 bits (half a step each, of weights that sum to 1 and of the result), the
    # products and sums are of 32 bits: D + len terms, far below
    half = torch.finfo(dt).eps / 2
    nan = torch.isnan(want)
    assert torch.equal(nan, torch.isnan(out))
    err = (out.double() - want).abs()[~nan]
    assert (err <= half * want.abs()[~nan] + (half + 2**-18) * vmax).all(), float(err.max())
    if lse is not None:
        assert torch.equal(torch.isnan(want_lse), torch.isnan(lse))
        ok = ~torch.isnan(want_lse)
        assert ((lse.double() - want_lse).abs()[ok] <= 2**-18 * (1 + want_lse.abs()[ok])).all()


def run_attn(sim, args, scale=None, parents=True, **kw):
    q, kn, vn, k, v, tabs, lens, par = args
    par = par if parents else None
    rc, out, lse = C.sim_attention(sim, q, kn, vn, k, v, tabs, lens, par, scale, **kw)
    assert rc == 0
    want, want_lse = C.attention(q, kn, vn, k, v, tabs, lens, par, q.shape[-1] ** -0.5 if scale is None else scale)
    vmax = max(float(vn.double().abs().max()), float(v.double()[torch.isfinite(v.double())].abs().max()))
    check_attn(out, lse, want, want_lse, vmax, q.dtype)


@pytest.mark.parametrize("T,Hq,Hkv,D,lens,page,dt,cu", [
    (1, 1, 1, 64, [0], 8, BF16, 4),
    (1, 8, 2, 64, [1, 33, 70], 16, F16, 4),
    (3, 7, 1, 96, [31, 0, 64], 8, BF16, 4),
    (2, 4, 2, 128, [300, 5], 64, BF16, 2),
    (9, 6, 2, 64, [130], 32, F16, 4),
    (1, 2, 1, 256, [90], 128, BF16, 4),
    (32, 1, 1, 64, [40], 16, BF16, 4),
])
def test_attention_few_rows(sim, T, Hq, Hkv, D, lens, page, dt, cu):
    run_attn(sim, attn_inputs(T * D + len(lens), len(lens), T, Hq, Hkv, D, lens, page, dt), num_cu=cu)


@pytest.mark.parametrize("T,Hq,Hkv,D,lens,page,dt", [
    (33, 1, 1, 64, [70], 16, F16),
    (9, 8, 2, 128, [65, 0], 64, BF16),
    (64, 2, 1, 96, [100], 8, BF16),
    (40, 4, 1, 64, [1], 32, BF16),
    (20, 2, 1, 256, [66], 32, F16),
])
def test_attention_many_rows(sim, T, Hq, Hkv, D, lens, page, dt):
    run_attn(sim, attn_inputs(T * D, len(lens), T, Hq, Hkv, D, lens, page, dt), num_cu=2)


@pytest.mark.parametrize("T,Hq,Hkv,lens,max_len,cu", [
    (1, 2, 2, [900, 3, 611], None, 3),   # shares that start and end inside sequences
    (2, 4, 1, [640], None, 7),
    (40, 1, 1, [900], None, 2),          # the same with tiles in LDS
    (33, 8, 1, [700], None, 16),         # and two groups of rows, eight workers each
    (1, 2, 1, [500], 20, 3),             # a bound of the lengths that is too low changes nothing
])
def test_attention_split(sim, T, Hq, Hkv, lens, max_len, cu):
    args = attn_inputs(sum(lens) + T, len(lens), T, Hq, Hkv, 64, lens, 32, BF16)
    run_attn(sim, args, num_cu=cu, max_len=max_len)


def test_attention_strided_rows_chain_and_scale(sim):
    args = attn_inputs(3, 2, 5, 4, 2, 64, [17, 40], 16, BF16, strided=True)
    run_attn(sim, args, parents=False, scale=0.3, want_lse=False)
    args = attn_inputs(4, 1, 35, 2, 2, 64, [17], 16, F16, strided=True)
    run_attn(sim, args, parents=False, scale=0.3)


@pytest.mark.parametrize("T", [2, 40])
def test_attention_bad_pages_lengths_and_parents(sim, T):
    q, kn, vn, k, v, tabs, lens, par = attn_inputs(11, 4, T, 1, 1, 64, [40, 40, 40, 40], 16, BF16)
    tabs[1, 1] = k.shape[0]
    lens[2], lens[3] = -5, 3 * 16 + 9      # below 0: none; past the table: all of it
    p = int(tabs[3, 2])
    k[p], v[p] = 0.5, 0.25
    par[0, 1] = T - 1 if T > 2 else 1      # no earlier node: a root
    run_attn(sim, (q, kn, vn, k, v, tabs, lens, par))


def test_attention_sharp_scores(sim):
    """Scores whose maximum grows from tile to tile, by more and by less than the slack, and one key far ahead."""
    q, kn, vn, k, v, tabs, lens, par = attn_inputs(12, 1, 2, 2, 1, 64, [400], 16, F16)
    for i in range(25):
        k[int(tabs[0, i])] *= 0.25 * (1 + i)
    k[int(tabs[0, 24]), 0, 3] *= 4
    run_attn(sim, (q, kn, vn, k, v, tabs, lens, par), num_cu=2)
    k2 = k.clone()
    for i in range(25):
        k2[int(tabs[0, i])] = k[int(tabs[0, 24 - i])]
    run_attn(sim, (q, kn, vn, k2, v, tabs, lens, par), num_cu=2)


# ------------------------------------------------------------------ the cache

def write_inputs(seed, L, B, T, H, D, page, P, dt, strided=False):
    g = gen(seed)
    tabs, N = C.tables(g, B, P)
    k, v = C.pools(g, L, N, H, page, D, dt)
    kn, vn = (torch.randn(L, B, T, H, D, generator=g).to(dt) for _ in range(2))
    if strided:
        w = torch.randn(L, B, T, 2 * H * D + 5, generator=g).to(dt)
        kn, vn = w[..., 1:1 + H * D].unflatten(-1, (H, D)), w[..., 1 + H * D:1 + 2 * H * D].unflatten(-1, (H, D))
    return kn, vn, k, v, tabs


@pytest.mark.parametrize("L,B,T,H,D,page,dt,strided", [
    (1, 1, 1, 1, 8, 8, BF16, False), (2, 3, 1, 2, 64, 16, F16, False), (2, 4, 21, 3, 24, 8, BF16, True), (1, 3, 40, 8, 128, 64, BF16, False)])
def test_append(sim, L, B, T, H, D, page, dt, strided):
    P = (T + 30 + page - 1) // page
    kn, vn, k, v, tabs = write_inputs(T + D, L, B, T, H, D, page, P, dt, strided)
    g = gen(T)
    lens = torch.randint(0, 29, (B,), generator=g).to(torch.int32)
    counts = torch.randint(0, T + 1, (B,), generator=g).to(torch.int32)
    for c in (counts, None):
        rc, k1, v1, l1 = C.sim_append(sim, kn, vn, k, v, tabs, lens, c)
        k2, v2, l2 = C.append(kn, vn, k, v, tabs, lens, c)
        assert rc == 0 and torch.equal(k1, k2) and torch.equal(v1, v2) and torch.equal(l1, l2)


def test_append_rows_that_do_not_fit(sim):
    kn, vn, k, v, tabs = write_inputs(7, 2, 6, 10, 1, 16, 8, 4, BF16)
    tabs[2, 1], tabs[3, 3] = -1, k.shape[1]
    lens = torch.tensor([30, 5, 3, 9, -1, 0], dtype=torch.int32)
    counts = torch.tensor([3, 11, 8, 10, 1, -2], dtype=torch.int32)  # past the table, past T, a bad page; fits; bad length, bad count
    rc, k1, v1, l1 = C.sim_append(sim, kn, vn, k, v, tabs, lens, counts)
    k2, v2, l2 = C.append(kn, vn, k, v, tabs, lens, counts)
    assert l2.tolist() == [-1, -1, -1, 19, -1, -1]
    assert rc == 0 and torch.equal(k1, k2) and torch.equal(v1, v2) and torch.equal(l1, l2)


def commit_ids(g, B, T, ids=3):
    """Few ids, so that paths fit by chance and siblings hold equal tokens."""
    return (torch.randint(0, ids, (B, T), generator=g).to(torch.int32) for _ in range(2))


@pytest.mark.parametrize("L,B,T,H,D,page,dt", [(1, 2, 1, 1, 8, 8, BF16), (2, 5, 9, 2, 64, 16, F16), (1, 3, 64, 2, 128, 32, BF16)])
def test_commit(sim, L, B, T, H, D, page, dt):
    P = (T + 30 + page - 1) // page
    kn, vn, k, v, tabs = write_inputs(T + D, L, B, T, H, D, page, P, dt)
    g = gen(T)
    lens = torch.randint(0, 29, (B,), generator=g).to(torch.int32)
    if B > 2:
        lens[0] = P * page  # no room for the root
    parents = C.tree(g, B, T)
    draft, sampled = commit_ids(g, B, T)
    if T == 64:  # a path through every node
        parents[1] = torch.arange(-1, T - 1)
        draft[1], sampled[1] = 1, 1
    rc, k1, v1, o1 = C.sim_commit(sim, kn, vn, k, v, tabs, lens, parents, draft, sampled)
    k2, v2, o2 = C.commit(kn, vn, k, v, tabs, lens, parents, draft, sampled)
    assert rc == 0 and torch.equal(k1, k2) and torch.equal(v1, v2)
    for x in o2:
        assert torch.equal(o1[x], o2[x]), x


def fork_inputs(seed, L, R, H, D, page, P, dt, most, width=4):
    """Rows as an earlier fork leaves them: requests of `width` beams share their full pages."""
    g = gen(seed)
    tabs, N = C.tables(g, R, P, spare=R + 2)
    lens = torch.randint(0, most + 1, (R // width,), generator=g).to(torch.int32).repeat_interleave(width)
    for r in range(R):
        full = int(lens[r]) // page
        tabs[r, :full] = tabs[r // width * width, :full]
        tabs[r, (int(lens[r]) + page - 1) // page:] = -1
    k, v = C.pools(g, L, N, H, page, D, dt)
    parents = (torch.rand(R, generator=g) * width).int() + torch.arange(R) // width * width
    return k, v, tabs, lens, parents.to(torch.int32)


def check_fork(sim, k, v, tabs, lens, parents, room):
    rc, k1, v1, t1, l1 = C.sim_fork(sim, k, v, tabs, lens, parents, room)
    k2, v2, t2, l2 = C.fork(k, v, tabs, lens, parents, room)
    assert rc == 0 and torch.equal(t1, t2) and torch.equal(l1, l2) and torch.equal(k1, k2) and torch.equal(v1, v2)
    return l2


@pytest.mark.parametrize("L,R,H,D,page,P,dt,most,width,room", [
    (1, 1, 1, 8, 8, 2, BF16, 9, 1, 1), (2, 8, 2, 64, 16, 4, F16, 50, 4, 1), (1, 6, 1, 16, 8, 6, BF16, 30, 3, 17), (1, 8, 1, 8, 8, 4, BF16, 24, 8, 0)])
def test_fork(sim, L, R, H, D, page, P, dt, most, width, room):
    for seed in range(3):
        check_fork(sim, *fork_inputs(seed, L, R, H, D, page, P, dt, most, width), room)


def test_fork_dead_parents_full_pool_and_bad_entries(sim):
    k, v, tabs, lens, parents = fork_inputs(3, 1, 8, 1, 16, 8, 4, BF16, 25)
    parents[1], parents[6] = -1, 8
    check_fork(sim, k, v, tabs, lens, parents, 1)
    tabs[2, 0] = k.shape[1] + 3  # an entry that is no page is carried, never followed
    lens[3] = 33                 # a length past the table
    check_fork(sim, k, v, tabs, lens, parents, 1)
    k, v, tabs, lens, _ = fork_inputs(4, 1, 4, 1, 16, 8, 3, BF16, 18)
    lens[:] = 17
    tabs = torch.arange(12, dtype=torch.int32).view(4, 3)
    tabs[1:, :2] = tabs[0, :2]
    parents = torch.tensor([2, 2, 2, 2], dtype=torch.int32)
    small = k[:, :12].contiguous(), v[:, :12].contiguous()
    assert check_fork(sim, *small, tabs, lens, parents, 1).tolist() == [17] * 4
    # a pool with two pages to spare for three copies; a table with no slot for the room
    assert check_fork(sim, k[:, :12].contiguous(), v[:, :12].contiguous(), tabs, lens, parents, 9).tolist() == [-1] * 4


# ------------------------------------------------------------------ refusals

def test_refusals(sim):
    g = gen(1)
    x, s, _, _ = beam_inputs(g, 1, 2, 40, F32)
    assert C.sim_beam(sim, x, s, 2, 65)[0] == -1
    assert C.sim_beam(sim, x[:, :1].contiguous(), s, 2, 3)[0] == -1      # more than there are candidates
    assert C.sim_beam(sim, x, s, 2, 3, ws_words=4)[0] == -5
    a = attn_inputs(1, 1, 2, 2, 1, 64, [9], 16, BF16)
    q, kn, vn, k, v, tabs, lens, par = a
    assert C.sim_attention(sim, *a, scale=-1.0)[0] == -1
    assert C.sim_attention(sim, *a, scale=math.nan)[0] == -1
    assert C.sim_attention(sim, *attn_inputs(1, 1, 2, 2, 1, 32, [9], 16, BF16))[0] == -1    # head_dim
    assert C.sim_attention(sim, *attn_inputs(1, 1, 2, 3, 2, 64, [9], 16, BF16))[0] == -1    # heads
    assert C.sim_attention(sim, *attn_inputs(1, 1, 65, 1, 1, 64, [9], 16, BF16))[0] == -1   # nodes
    assert C.sim_attention(sim, *attn_inputs(1, 1, 1, 1, 1, 64, [9], 24, BF16))[0] == -1    # page size
    kn, vn, k, v, tabs = write_inputs(1, 1, 1, 2, 1, 16, 8, 2, BF16)
    lens = torch.zeros(1, dtype=torch.int32)
    assert C.sim_append(sim, kn, vn, k.float(), v.float(), tabs, lens, None)[0] == -1       # dtype
    assert C.sim_fork(sim, k, v, tabs, lens, lens, -1)[0] == -1
    assert C.sim_fork(sim, k, v, tabs, lens, lens, 1, ws_words=1)[0] == -5
