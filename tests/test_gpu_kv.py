"""GPU: beam selection, tree attention and the paged cache through the public
entry points (`Sampler`), against plain forms in 64 bits on the CPU."""
import math

import pytest
import torch

import gpu_harness as H
import kv_cases as C
from test_kv_sim import (BF16, F16, F32, attn_inputs, beam_inputs, check_attn, check_beam, commit_ids, fork_inputs, gen,
                         write_inputs)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dev(t):
    """On the GPU with the same strides."""
    if t is None:
        return None
    n = 1 + sum((s - 1) * st for s, st in zip(t.shape, t.stride())) if t.numel() else 0
    flat = torch.as_strided(t, (n,), (1,)).to(DEV)
    return torch.as_strided(flat, t.shape, t.stride())


def cpu(x):
    return {k: t.cpu() for k, t in x.items()}


# ------------------------------------------------------------------ beams

@pytest.mark.parametrize("G,W,V,n,dt,hist", [
    (1, 1, 1, 1, F32, 0), (3, 3, 37, 5, BF16, 4), (1, 4, 32000, 4, F32, 64), (2, 16, 9001, 32, BF16, 5), (4, 8, 50257, 16, BF16, 0),
    (1, 64, 3000, 64, F32, 0), (5, 2, 128256, 4, F32, 9), (33, 5, 301, 10, F32, 1)])
def test_beam(sampler, G, W, V, n, dt, hist):
    H.log(f"beam G={G} W={W} V={V} n={n}")
    x, scores, hs, hl = beam_inputs(gen(V + n), G, W, V, dt, hist, pad=5)
    got = sampler.beam_select(dev(x), scores.to(DEV), W, n, hist=dev(hs), hist_len=dev(hl), vocab=V)
    torch.cuda.synchronize()
    check_beam(0, cpu(got), C.beam(x[:, :V], scores, W, n, hs, hl))


def test_beam_equal_logits_ended_beams_and_rows_that_give_nothing(sampler):
    H.log("beam special rows")
    x, scores, hs, hl = beam_inputs(gen(5), 5, 3, 9100, F32, 2)
    x[0] = 1.5
    x[1] = x[0]
    scores[1] = scores[0]
    scores[2] = -math.inf
    x[3, 7], x[4, :] = math.nan, math.nan
    x[5, 11] = math.inf
    x[6:9] = -math.inf
    x[7, 9099] = -3.0
    scores[9:12] = -math.inf
    x[12:15, 5:] = -math.inf
    x[12:15, :5] = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 0.0])
    scores[12:15] = -1.0
    got = sampler.beam_select(dev(x), scores.to(DEV), 3, 6, hist=dev(hs), hist_len=dev(hl))
    torch.cuda.synchronize()
    check_beam(0, cpu(got), C.beam(x, scores, 3, 6, hs, hl))


# ------------------------------------------------------------------ attention

def run_attn(sampler, args, scale=None, parents=True, lse=True, max_len=None):
    q, kn, vn, k, v, tabs, lens, par = args
    par = par if parents else None
    B, T, Hq, D = q.shape
    H.log(f"attention B={B} T={T} Hq={Hq} Hkv={kn.shape[2]} D={D} lens={lens.tolist()[:4]} page={k.shape[2]} {q.dtype}")
    lse_t = torch.empty(B, T, Hq, device=DEV) if lse else None
    out = sampler.tree_attention(dev(q), dev(kn), dev(vn), dev(k), dev(v), dev(tabs), dev(lens), parents=dev(par),
                                 max_len=max_len, scale=scale, lse=lse_t)
    torch.cuda.synchronize()
    want, want_lse = C.attention(q, kn, vn, k, v, tabs, lens, par, D ** -0.5 if scale is None else scale)
    vmax = max(float(vn.double().abs().max()), float(v.double()[torch.isfinite(v.double())].abs().max()))
    check_attn(out.cpu(), None if lse_t is None else lse_t.cpu(), want, want_lse, vmax, q.dtype)


SHAPES = [(1, 1, 1), (1, 8, 2), (5, 7, 1), (8, 8, 2), (16, 2, 1), (33, 3, 3), (20, 8, 2), (64, 4, 1), (63, 8, 1)]


@pytest.mark.parametrize("T,Hq,Hkv", SHAPES)
@pytest.mark.parametrize("D,page,dt", [(64, 16, F16), (96, 8, BF16), (128, 64, BF16), (256, 128, F16)])
def test_attention(sampler, T, Hq, Hkv, D, page, dt):
    run_attn(sampler, attn_inputs(T * D + Hq, 4, T, Hq, Hkv, D, [0, 1, 77, 513], page, dt))


@pytest.mark.parametrize("T,Hq,Hkv,lens,page", [(1, 4, 1, [9000], 64), (5, 8, 2, [5000, 0, 17, 2049], 16), (63, 8, 1, [3001], 32),
                                                (40, 2, 1, [2500, 64, 63], 64)])
def test_attention_long(sampler, T, Hq, Hkv, lens, page):
    args = attn_inputs(sum(lens), len(lens), T, Hq, Hkv, 128, lens, page, BF16)
    run_attn(sampler, args)
    run_attn(sampler, args, lse=False, max_len=0)  # a bound that is too low changes nothing


def test_attention_strided_rows_chain_and_scale(sampler):
    for T, Hq, dt in ((5, 4, BF16), (35, 2, F16)):
        run_attn(sampler, attn_inputs(3, 2, T, Hq, 2, 64, [17, 40], 16, dt, strided=True), parents=False, scale=0.3)


def test_attention_of_a_strided_pool(sampler):
    """Keys and values of one allocation, page by page, a layer in the middle."""
    q, kn, vn, k, v, tabs, lens, par = attn_inputs(8, 2, 3, 4, 2, 64, [70, 33], 16, BF16)
    N, h, page, D = k.shape
    both = torch.zeros(N, 3, h * page * D, dtype=BF16)
    both[:, 1] = k.reshape(N, -1)
    both[:, 2] = v.reshape(N, -1)
    both = both.to(DEV)
    kd = both[:, 1].unflatten(-1, (h, page, D))
    vd = both[:, 2].unflatten(-1, (h, page // 8, D, 8))
    H.log("attention of a strided pool")
    out = sampler.tree_attention(dev(q), dev(kn), dev(vn), kd, vd, dev(tabs), dev(lens), parents=dev(par))
    ref = sampler.tree_attention(dev(q), dev(kn), dev(vn), dev(k), dev(v), dev(tabs), dev(lens), parents=dev(par))
    torch.cuda.synchronize()
    assert torch.equal(out, ref)


def test_attention_pages_past_32_bits(sampler):
    """Page offsets beyond 2^32 elements."""
    H.log("attention past 32-bit offsets")
    N, h, page, D = 1030, 8, 512, 1 << 7
    big = torch.empty(N * 8 * page * D * 2, dtype=BF16, device=DEV)  # 8.6 G elements
    k = big[: N * h * page * D * 2].view(N, 2, h, page, D)[:, 0]
    q, kn, vn, ks, vs, tabs, lens, par = attn_inputs(9, 1, 2, 8, 8, D, [700], page, BF16)
    pages = torch.tensor([[N - 1, N - 3]], dtype=torch.int32)
    k[N - 1], k[N - 3] = ks[int(tabs[0, 0])].to(DEV), ks[int(tabs[0, 1])].to(DEV)
    v = big[: N * h * page * D * 2].view(N, 2, h, page // 8, D, 8)[:, 1]
    v[N - 1], v[N - 3] = vs[int(tabs[0, 0])].to(DEV), vs[int(tabs[0, 1])].to(DEV)
    out = sampler.tree_attention(dev(q), dev(kn), dev(vn), k, v, dev(pages), dev(lens), parents=dev(par))
    ref = sampler.tree_attention(dev(q), dev(kn), dev(vn), dev(ks), dev(vs), dev(tabs), dev(lens), parents=dev(par))
    torch.cuda.synchronize()
    assert torch.equal(out, ref)


def test_attention_bad_pages_lengths_and_parents(sampler):
    for T in (2, 40):
        q, kn, vn, k, v, tabs, lens, par = attn_inputs(11, 4, T, 1, 1, 64, [40, 40, 40, 40], 16, BF16)
        tabs[1, 1] = k.shape[0]
        lens[2], lens[3] = -5, 3 * 16 + 9
        p = int(tabs[3, 2])
        k[p], v[p] = 0.5, 0.25
        par[0, 1] = T - 1 if T > 2 else 1
        run_attn(sampler, (q, kn, vn, k, v, tabs, lens, par))


# ------------------------------------------------------------------ the cache

@pytest.mark.parametrize("L,B,T,h,D,page,dt,strided", [
    (1, 1, 1, 1, 8, 8, BF16, False), (3, 9, 1, 8, 128, 64, F16, False), (2, 4, 21, 3, 24, 8, BF16, True), (2, 3, 300, 4, 96, 32, BF16, False)])
def test_append(sampler, L, B, T, h, D, page, dt, strided):
    H.log(f"append L={L} B={B} T={T} D={D}")
    P = (T + 30 + page - 1) // page
    kn, vn, k, v, tabs = write_inputs(T + D, L, B, T, h, D, page, P, dt, strided)
    lens = torch.randint(0, 29, (B,), generator=gen(T)).to(torch.int32)
    counts = torch.randint(0, T + 1, (B,), generator=gen(T + 1)).to(torch.int32)
    counts[0] = T
    if B > 2:
        tabs[2, 0] = k.shape[1]  # (a page outside the pool: where rows go there, nothing of the sequence is written)
        lens[2] = 0
    for c in (counts, None):
        kd, vd = dev(k), dev(v)
        l1 = sampler.kv_append(dev(kn), dev(vn), kd, vd, dev(tabs), dev(lens), counts=dev(c))
        torch.cuda.synchronize()
        k2, v2, l2 = C.append(kn, vn, k, v, tabs, lens, c)
        assert torch.equal(kd.cpu(), k2) and torch.equal(vd.cpu(), v2) and torch.equal(l1.cpu(), l2)


@pytest.mark.parametrize("L,B,T,h,D,page,dt", [(1, 2, 1, 1, 8, 8, BF16), (3, 17, 9, 2, 64, 16, F16), (2, 5, 64, 8, 128, 32, BF16)])
def test_commit(sampler, L, B, T, h, D, page, dt):
    H.log(f"commit L={L} B={B} T={T}")
    P = (T + 30 + page - 1) // page
    kn, vn, k, v, tabs = write_inputs(T + D, L, B, T, h, D, page, P, dt)
    g = gen(T)
    lens = torch.randint(0, 29, (B,), generator=g).to(torch.int32)
    if B > 2:
        lens[0] = P * page
    parents = C.tree(g, B, T)
    draft, sampled = commit_ids(g, B, T)
    if T == 64:
        parents[1] = torch.arange(-1, T - 1)
        draft[1], sampled[1] = 1, 1
    kd, vd = dev(k), dev(v)
    o1 = sampler.tree_commit(dev(kn), dev(vn), kd, vd, dev(tabs), dev(lens), dev(parents), dev(draft), dev(sampled))
    torch.cuda.synchronize()
    k2, v2, o2 = C.commit(kn, vn, k, v, tabs, lens, parents, draft, sampled)
    assert torch.equal(kd.cpu(), k2) and torch.equal(vd.cpu(), v2)
    for x in o2:
        assert torch.equal(o1[x].cpu(), o2[x]), x


def run_fork(sampler, k, v, tabs, lens, parents, room):
    H.log(f"fork rows={tabs.shape[0]} pages={k.shape[1]} room={room}")
    kd, vd = dev(k), dev(v)
    t1, l1 = sampler.kv_fork(kd, vd, dev(tabs), dev(lens), dev(parents), room=room)
    torch.cuda.synchronize()
    k2, v2, t2, l2 = C.fork(k, v, tabs, lens, parents, room)
    assert torch.equal(t1.cpu(), t2) and torch.equal(l1.cpu(), l2) and torch.equal(kd.cpu(), k2) and torch.equal(vd.cpu(), v2)
    return l2


@pytest.mark.parametrize("L,R,h,D,page,P,dt,most,width,room", [
    (1, 1, 1, 8, 8, 2, BF16, 9, 1, 1), (2, 128, 2, 64, 16, 6, F16, 80, 8, 1), (1, 6, 1, 16, 8, 6, BF16, 30, 3, 17),
    (1, 1100, 1, 8, 8, 4, BF16, 24, 4, 1)])
def test_fork(sampler, L, R, h, D, page, P, dt, most, width, room):
    for seed in range(2):
        run_fork(sampler, *fork_inputs(seed, L, R, h, D, page, P, dt, most, width), room)


def test_fork_of_a_large_pool(sampler):
    """More pages than the planning kernel's LDS has owners for."""
    k, v, tabs, lens, parents = fork_inputs(5, 1, 16, 1, 8, 8, 6, BF16, 40, 4)
    more = 40000
    k = torch.cat([k, torch.zeros(1, more, 1, 8, 8, dtype=BF16)], 1)
    v = torch.cat([v, torch.zeros(1, more, 1, 1, 8, 8, dtype=BF16)], 1)
    run_fork(sampler, k, v, tabs, lens, parents, 1)


def test_fork_dead_parents_and_full_pool(sampler):
    k, v, tabs, lens, parents = fork_inputs(3, 1, 8, 1, 16, 8, 4, BF16, 25)
    parents[1], parents[6] = -1, 8
    tabs[2, 0] = k.shape[1] + 3
    lens[3] = 33
    run_fork(sampler, k, v, tabs, lens, parents, 1)
    k, v, _, lens, _ = fork_inputs(4, 1, 4, 1, 16, 8, 3, BF16, 18)
    lens[:] = 17
    tabs = torch.tensor([[0, 1, 2], [0, 1, 3], [0, 1, 4], [0, 1, 3]], dtype=torch.int32)
    parents = torch.tensor([2, 2, 2, 2], dtype=torch.int32)
    k, v = k[:, :5].contiguous(), v[:, :5].contiguous()  # page 4 stays with row 0; 2 and 3 are free, for three copies
    assert run_fork(sampler, k, v, tabs, lens, parents, 1).tolist() == [17, 17, 17, -1]


# ------------------------------------------------------------------ streams, graphs, refusals

def test_a_decode_step_on_a_stream_and_in_a_graph(sampler):
    """Attention, beam selection, fork and append captured together: every
    replay equals the eager calls on the same inputs."""
    H.log("decode step in a graph")
    g = gen(21)
    k, v, tabs, lens, _ = fork_inputs(6, 1, 8, 2, 64, 16, 12, BF16, 150, 4)
    q = torch.randn(8, 1, 8, 64, generator=g).to(BF16)
    kn, vn = (torch.randn(1, 8, 1, 2, 64, generator=g).to(BF16) for _ in range(2))
    x, scores, hs, hl = beam_inputs(g, 2, 4, 5000, F32, 6)
    ins = [dev(t) for t in (q, kn, vn, tabs, lens, x, scores, hs, hl)]
    kd, vd = dev(k), dev(v)

    def step(q, kn, vn, tabs, lens, x, scores, hs, hl):
        out = sampler.tree_attention(q, kn[0], vn[0], kd[0], vd[0], tabs, lens)
        o = sampler.beam_select(x, scores, 4, 4, hist=hs, hist_len=hl)
        t2, l2 = sampler.kv_fork(kd, vd, tabs, lens, o["parents"], room=1)
        l3 = sampler.kv_append(kn, vn, kd, vd, t2, l2)
        return [out, *o.values(), t2, l2, l3, kd, vd]

    def eager():
        kd.copy_(k), vd.copy_(v)
        r = [t.clone() for t in step(*ins)]
        torch.cuda.synchronize()
        return r

    side = torch.cuda.Stream()
    eager()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        got = step(*ins)
    torch.cuda.synchronize()
    for i in range(4):
        ins[0].copy_(torch.randn(8, 1, 8, 64, generator=g).to(BF16))
        ins[5].copy_(torch.randn(8, 5000, generator=g) * 3)
        want = eager()
        kd.copy_(k), vd.copy_(v)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


def test_a_given_stream(sampler):
    args = attn_inputs(31, 2, 4, 4, 2, 64, [300, 20], 16, BF16)
    H.log("attention on a given stream")
    d = [dev(t) for t in args]
    ref = sampler.tree_attention(*d[:7], parents=d[7])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    out = torch.zeros_like(ref)
    torch.cuda.synchronize()
    sampler.tree_attention(*d[:7], parents=d[7], out=out, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(out, ref)


def test_empty_batches(sampler):
    H.log("empty batches")
    z = torch.empty(0, dtype=torch.int32, device=DEV)
    k, v = (t.to(DEV) for t in C.pools(gen(1), 1, 3, 1, 8, 64, BF16))
    rows = torch.empty(1, 0, 2, 1, 64, dtype=BF16, device=DEV)
    tabs = torch.empty(0, 2, dtype=torch.int32, device=DEV)
    assert sampler.kv_append(rows, rows, k, v, tabs, z).numel() == 0
    assert sampler.kv_fork(k, v, tabs, z, z)[0].shape == (0, 2)
    q = torch.empty(0, 2, 1, 64, dtype=BF16, device=DEV)
    assert sampler.tree_attention(q, q, q, k[0], v[0], tabs, z).shape == (0, 2, 1, 64)
    assert sampler.beam_select(torch.empty(0, 9, device=DEV), torch.empty(0, device=DEV), 2, 2)["tokens"].numel() == 0


def test_refusals(sampler):
    H.log("refusals")
    import tinygpt_amd as tg

    q, kn, vn, k, v, tabs, lens, par = [dev(t) for t in attn_inputs(1, 2, 3, 4, 2, 64, [20, 9], 16, BF16)]
    good = dict(parents=par)

    def refused(err, *a, **kw):
        with pytest.raises(err):
            sampler.tree_attention(*a, **kw)

    refused(ValueError, q.float(), kn, vn, k, v, tabs, lens, **good)
    refused(TypeError, q.float(), kn.float(), vn.float(), k.float(), v.float(), tabs, lens, **good)
    refused(ValueError, q[:1], kn, vn, k, v, tabs, lens, **good)
    refused(ValueError, q, kn[:, :2], vn, k, v, tabs, lens, **good)
    refused(ValueError, q, kn, vn, k, k, tabs, lens, **good)
    refused(ValueError, q, kn, vn, k.transpose(1, 2), v, tabs, lens, **good)
    refused(ValueError, q, kn, vn, k, v, tabs.long(), lens, **good)
    refused(ValueError, q, kn, vn, k, v, tabs, lens[:1], **good)
    refused(ValueError, q, kn, vn, k, v, tabs, lens, parents=par[:, :2])
    refused(ValueError, q, kn, vn, k, v, tabs, lens.cpu(), **good)
    refused(ValueError, q[:, :, :3], kn, vn, k, v, tabs, lens, **good)
    refused(ValueError, q, kn, vn, k, v, tabs, lens, out=q, **good)
    refused(tg.TgsError, q, kn, vn, k, v, tabs, lens, scale=0.0, **good)
    x, s = torch.zeros(4, 50, device=DEV), torch.zeros(4, device=DEV)
    for err, a in ((ValueError, (x, s, 3, 2)), (ValueError, (x, s[:3], 2, 2)), (TypeError, (x.half(), s, 2, 2)),
                   (tg.TgsError, (x, s, 2, 65)), (tg.TgsError, (x, s, 2, 0))):
        with pytest.raises(err):
            sampler.beam_select(*a)
    with pytest.raises(ValueError):
        sampler.beam_select(x, s, 2, 2, hist=torch.zeros(4, 3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        sampler.kv_fork(k[None], v[None], tabs, lens, lens.clone(), tables_out=tabs)
    with pytest.raises(ValueError):
        sampler.kv_append(kn[None], vn[None], k[None], v[None], tabs, lens, lens_out=lens)


@pytest.mark.parametrize("name", ["scores", "parents", "tokens", "hist", "hist_len"])
def test_beam_outputs_that_are_inputs_are_refused(sampler, name):
    H.log(f"beam outputs that are inputs: {name}")
    ints = dict(dtype=torch.int32, device=DEV)
    x, s, hist, n = torch.zeros(4, 50, device=DEV), torch.zeros(4, device=DEV), torch.zeros(4, 1, **ints), torch.zeros(4, **ints)
    out = {"scores": torch.zeros(4, device=DEV), "parents": torch.zeros(4, **ints), "tokens": torch.zeros(4, **ints),
           "hist": torch.zeros(4, 1, **ints), "hist_len": torch.zeros(4, **ints)}
    out[name] = {"scores": s, "hist": hist}.get(name, n)
    with pytest.raises(ValueError):
        sampler.beam_select(x, s, 2, 2, hist=hist, hist_len=n, out=out)
