"""GPU: the 8-bit cache and the position rotation through the public entry
points (`Sampler`), against plain forms in 64 bits on the CPU."""
import pytest
import torch

import gpu_harness as H
import kv8_cases as K
import kv_cases as C
from test_gpu_kv import dev
from test_kv8_sim import FREQ, attn_inputs, border_rows, vmax_of, wanted, write_inputs
from test_kv_sim import check_attn, commit_ids, gen

pytestmark = pytest.mark.gpu
BF16, F16, I32, U8, DEV = torch.bfloat16, torch.float16, torch.int32, torch.uint8, "cuda:0"


def pools(p):
    """Byte pools on the GPU, and as the calls take them."""
    raw = [dev(x) for x in p]
    return raw, K.as_tensors(raw)


# ------------------------------------------------------------------ attention

def run_attn(sampler, args, scale=None, parents=True, lse=True, max_len=None):
    q, kn, vn, p, tabs, lens, par = args
    B, T, Hq, D = q.shape
    H.log(f"8-bit attention B={B} T={T} Hq={Hq} Hkv={kn.shape[2]} D={D} lens={lens.tolist()[:4]} page={p[0].shape[2]} {q.dtype}")
    lse_t = torch.empty(B, T, Hq, device=DEV) if lse else None
    _, (k, v, s) = pools(p)
    out = sampler.tree_attention(dev(q), dev(kn), dev(vn), k, v, dev(tabs), dev(lens), parents=dev(par) if parents else None,
                                 max_len=max_len, scale=scale, lse=lse_t, scales=s)
    torch.cuda.synchronize()
    want, want_lse = wanted(args, scale, parents)
    check_attn(out.cpu(), None if lse_t is None else lse_t.cpu(), want, want_lse, vmax_of(args), q.dtype)


SHAPES = [(1, 1, 1), (1, 8, 2), (5, 7, 1), (8, 8, 2), (16, 2, 1), (33, 3, 3), (20, 8, 2), (64, 4, 1), (63, 8, 1)]


@pytest.mark.parametrize("T,Hq,Hkv", SHAPES)
@pytest.mark.parametrize("D,page,dt", [(64, 16, F16), (96, 32, BF16), (128, 64, BF16), (256, 128, F16)])
def test_attention(sampler, T, Hq, Hkv, D, page, dt):
    run_attn(sampler, attn_inputs(T * D + Hq, 4, T, Hq, Hkv, D, [0, 1, 77, 513], page, dt))


@pytest.mark.parametrize("T,Hq,Hkv,lens,page", [(1, 4, 1, [9000], 64), (5, 8, 2, [5000, 0, 17, 2049], 16), (63, 8, 1, [3001], 32),
                                                (40, 2, 1, [2500, 64, 63], 64), (1, 2, 1, [12000], 1024)])
def test_attention_long(sampler, T, Hq, Hkv, lens, page):
    args = attn_inputs(sum(lens), len(lens), T, Hq, Hkv, 128, lens, page, BF16)
    run_attn(sampler, args)
    run_attn(sampler, args, lse=False, max_len=0)  # a bound that is too low changes nothing


def test_attention_strided_rows_chain_and_scale(sampler):
    for T, Hq, dt in ((5, 4, BF16), (35, 2, F16)):
        run_attn(sampler, attn_inputs(3, 2, T, Hq, 2, 64, [17, 40], 16, dt, strided=True), parents=False, scale=0.3)


def test_attention_many_sequences(sampler):
    """More sequences than a wave has lanes, most of them short."""
    lens = [int(x) for x in torch.randint(0, 90, (150,), generator=gen(2))]
    lens[77], lens[140] = 1500, 700
    run_attn(sampler, attn_inputs(5, 150, 2, 2, 1, 64, lens, 64, BF16))


def test_attention_of_a_strided_pool(sampler):
    """Keys, values and scales of one allocation, page by page."""
    q, kn, vn, p, tabs, lens, par = attn_inputs(8, 2, 3, 4, 2, 64, [70, 33], 16, BF16)
    N, h, page, D = p[0].shape
    whole, few = h * page * D, h * page // 8
    both = torch.zeros(N, 3 * whole + 16, dtype=U8)
    both[:, whole:2 * whole], both[:, 2 * whole:3 * whole] = p[0].reshape(N, -1), p[1].reshape(N, -1)
    both[:, 3 * whole:3 * whole + few] = p[2].reshape(N, -1)
    both = both.to(DEV)
    k = both[:, whole:2 * whole].unflatten(-1, (h, page, D)).view(K.E4M3)
    v = both[:, 2 * whole:3 * whole].unflatten(-1, (h, page // 16, D, 16)).view(K.E4M3)
    s = both[:, 3 * whole:3 * whole + few].unflatten(-1, (h, page // 16, 2)).view(K.E8M0)
    _, (k2, v2, s2) = pools(p)
    H.log("8-bit attention of a strided pool")
    rest = dict(parents=dev(par))
    out = sampler.tree_attention(dev(q), dev(kn), dev(vn), k, v, dev(tabs), dev(lens), scales=s, **rest)
    ref = sampler.tree_attention(dev(q), dev(kn), dev(vn), k2, v2, dev(tabs), dev(lens), scales=s2, **rest)
    torch.cuda.synchronize()
    assert torch.equal(out, ref)


def test_pages_past_32_bits(sampler):
    """Page offsets beyond 2^32 bytes: appended to and attended."""
    H.log("8-bit cache past 32-bit offsets")
    N, h, page, D = 9000, 8, 512, 128
    k = torch.empty(1, N, h, page, D, dtype=K.E4M3, device=DEV)
    v = torch.empty(1, N, h, page // 16, D, 16, dtype=K.E4M3, device=DEV)
    s = torch.empty(1, N, h, page // 16, 2, dtype=K.E8M0, device=DEV)
    q, kn, vn, p, tabs, lens, par = attn_inputs(9, 1, 2, 8, 8, D, [700], page, BF16)
    pages = torch.tensor([[N - 1, N - 3]], dtype=I32)
    raw, (ks, vs, ss) = pools([x[None] for x in p])
    for i in range(2):
        for a, b in ((k, ks), (v, vs), (s, ss)):
            a.view(U8)[:, int(pages[0, i])] = b.view(U8)[:, int(tabs[0, i])]
    rows = [torch.randn(1, 1, 40, h, D, generator=gen(i)).to(BF16).to(DEV) for i in (1, 2)]
    outs = []
    for kk, vv, sc, t in ((k, v, s, pages), (ks, vs, ss, tabs)):
        l = sampler.kv_append(*rows, kk, vv, dev(t), dev(lens), scales=sc, rotary=dev(FREQ[128]))
        outs.append(sampler.tree_attention(dev(q), dev(kn), dev(vn), kk[0], vv[0], dev(t), l, parents=dev(par), scales=sc[0]))
    torch.cuda.synchronize()
    assert torch.equal(*outs) and torch.isfinite(outs[0].float()).all()


def test_attention_bad_pages_lengths_and_nan_scales(sampler):
    for T in (2, 40):
        q, kn, vn, p, tabs, lens, par = attn_inputs(11, 5, T, 1, 1, 64, [40, 40, 40, 40, 40], 16, BF16)
        tabs[1, 1] = p[0].shape[0]
        lens[2], lens[4] = -5, -1
        p[2][int(tabs[3, 1]), 0, 0, T % 3 % 2] = 255
        H.log(f"8-bit attention: bad pages T={T}")
        _, (k, v, s) = pools(p)
        out = sampler.tree_attention(dev(q), dev(kn), dev(vn), k, v, dev(tabs), dev(lens), parents=dev(par), scales=s).cpu()
        assert torch.isnan(out[[1, 3, 4]].float()).all()
        want, _ = wanted((q, kn, vn, p, tabs, lens, par))
        check_attn(out[[0, 2]], None, want[[0, 2]], None, vmax_of((q, kn, vn, p, tabs, lens, par)), BF16)


# ------------------------------------------------------------------ writes

@pytest.mark.parametrize("L,B,T,h,D,page,dt,strided,dims,pairs", [
    (1, 1, 1, 1, 16, 16, BF16, False, 0, False), (3, 9, 1, 8, 128, 64, F16, False, 128, False),
    (2, 4, 21, 3, 48, 16, BF16, True, 32, True), (2, 3, 300, 4, 96, 32, BF16, False, 96, False),
    (1, 2, 130, 2, 256, 16, F16, False, 128, True), (1, 3, 77, 5, 112, 128, BF16, True, 0, False)])
def test_append(sampler, L, B, T, h, D, page, dt, strided, dims, pairs):
    H.log(f"8-bit append L={L} B={B} T={T} D={D} dims={dims}")
    P = (T + 30 + page - 1) // page
    kn, vn, p, tabs = write_inputs(T + D, L, B, T, h, D, page, P, dt, strided, spread=2.0)
    lens = torch.randint(0, 29, (B,), generator=gen(T)).to(I32)
    counts = torch.randint(0, T + 1, (B,), generator=gen(T + 1)).to(I32)
    counts[0] = T
    if B > 2:
        tabs[2, 0] = p[0].shape[1]  # (a page outside the pool: where rows go there, nothing of the sequence is written)
        lens[2] = 0
    freq = FREQ[dims] if dims else None
    for c in (counts, None):
        raw, (k, v, s) = pools(p)
        l1 = sampler.kv_append(dev(kn), dev(vn), k, v, dev(tabs), dev(lens), counts=dev(c), scales=s, rotary=dev(freq), pairs=pairs)
        torch.cuda.synchronize()
        want, l2, put = K.append(kn, vn, p, tabs, lens, c, dt, freq, pairs)
        assert torch.equal(l1.cpu(), l2)
        K.check_written(p, [x.cpu() for x in raw], want, put, dt, dims // 2, pairs)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_append_borders(sampler, dt):
    H.log(f"8-bit append at the borders {dt}")
    rows = border_rows(dt)
    n = len(rows)
    kn = rows[None, :, None, None, :].contiguous()
    vn = kn.flip(1).contiguous()
    g = gen(3)
    tabs, N = C.tables(g, n, 1)
    p = K.pools(g, 1, N, 1, 16, 16, dt)
    for held in (0, 3):
        lens = torch.full((n,), held, dtype=I32)
        raw, (k, v, s) = pools(p)
        sampler.kv_append(dev(kn), dev(vn), k, v, dev(tabs), dev(lens), scales=s)
        torch.cuda.synchronize()
        want, _, put = K.append(kn, vn, p, tabs, lens, None, dt)
        K.check_written(p, [x.cpu() for x in raw], want, put, dt)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_append_token_by_token(sampler, dt):
    H.log(f"8-bit append token by token {dt}")
    kn, vn, p, tabs = write_inputs(5, 1, 1, 24, 2, 64, 16, 2, dt)
    kn *= torch.exp2(torch.tensor([0, 1, 3, 2, 9, -4] * 4).float())[None, None, :, None, None].to(dt)
    raw, (k, v, s) = pools(p)
    want, wl, lens = p, torch.zeros(1, dtype=I32), torch.zeros(1, dtype=I32, device=DEV)
    t = dev(tabs)
    for i in range(24):
        rows = kn[:, :, i:i + 1].contiguous(), vn[:, :, i:i + 1].contiguous()
        lens = sampler.kv_append(dev(rows[0]), dev(rows[1]), k, v, t, lens, scales=s)
        want, wl, _ = K.append(*rows, want, tabs, wl, None, dt)
        torch.cuda.synchronize()
        assert torch.equal(lens.cpu(), wl)
        K.check_written(p, [x.cpu() for x in raw], want, {}, dt)


@pytest.mark.parametrize("L,B,T,h,D,page,dt,dims,pairs", [
    (1, 1, 1, 1, 16, 8, BF16, 16, False), (3, 9, 1, 8, 128, 64, F16, 64, True), (2, 4, 21, 3, 24, 8, BF16, 16, True),
    (2, 3, 300, 4, 96, 32, BF16, 96, False), (1, 2, 50, 2, 72, 16, F16, 64, False)])
def test_append_rotated(sampler, L, B, T, h, D, page, dt, dims, pairs):
    H.log(f"rotated append L={L} B={B} T={T} D={D} dims={dims}")
    g = gen(T + D)
    P = (T + 30 + page - 1) // page
    tabs, N = C.tables(g, B, P)
    k, v = C.pools(g, L, N, h, page, D, dt)
    kn, vn = (torch.randn(L, B, T, h, D, generator=g).to(dt) for _ in range(2))
    lens = torch.randint(0, 29, (B,), generator=g).to(I32)
    counts = torch.randint(0, T + 1, (B,), generator=g).to(I32)
    counts[0] = T
    kd, vd = dev(k), dev(v)
    l1 = sampler.kv_append(dev(kn), dev(vn), kd, vd, dev(tabs), dev(lens), counts=dev(counts), rotary=dev(FREQ[dims]), pairs=pairs)
    torch.cuda.synchronize()
    k2, v2, l2 = C.append(kn, vn, k, v, tabs, lens, counts)
    k1 = kd.cpu()
    assert torch.equal(vd.cpu(), v2) and torch.equal(l1.cpu(), l2)
    for b in range(B):
        for i in range(int(counts[b])):
            pos = int(lens[b]) + i
            pg, slot = int(tabs[b, pos // page]), pos % page
            K.check_turned16(k1[:, pg, :, slot], K.turned(kn[:, b, i].double(), pos, FREQ[dims], pairs), dims // 2, pairs)
            k2[:, pg, :, slot] = k1[:, pg, :, slot]
    assert torch.equal(k1, k2)


@pytest.mark.parametrize("L,B,T,h,D,page,dt", [(1, 2, 1, 1, 16, 16, BF16), (3, 17, 9, 2, 64, 16, F16), (2, 5, 64, 8, 128, 32, BF16)])
def test_commit(sampler, L, B, T, h, D, page, dt):
    H.log(f"8-bit commit L={L} B={B} T={T}")
    P = (T + 30 + page - 1) // page
    kn, vn, p, tabs = write_inputs(T + D, L, B, T, h, D, page, P, dt)
    g = gen(T)
    lens = torch.randint(0, 29, (B,), generator=g).to(I32)
    if B > 2:
        lens[0] = P * page
    parents = C.tree(g, B, T)
    draft, sampled = commit_ids(g, B, T)
    if T == 64:
        parents[1] = torch.arange(-1, T - 1)
        draft[1], sampled[1] = 1, 1
    raw, (k, v, s) = pools(p)
    o1 = sampler.tree_commit(dev(kn), dev(vn), k, v, dev(tabs), dev(lens), dev(parents), dev(draft), dev(sampled), scales=s)
    torch.cuda.synchronize()
    want, o2 = K.commit(kn, vn, p, tabs, lens, parents, draft, sampled, dt)
    K.check_written(p, [x.cpu() for x in raw], want, {}, dt)
    for x in o2:
        assert torch.equal(o1[x].cpu(), o2[x]), x


@pytest.mark.parametrize("L,R,h,D,page,P,most,width,room", [
    (1, 1, 1, 16, 16, 2, 9, 1, 1), (2, 128, 2, 64, 32, 6, 160, 8, 1), (1, 6, 1, 16, 16, 6, 60, 3, 17), (1, 1100, 1, 16, 16, 4, 48, 4, 1)])
def test_fork(sampler, L, R, h, D, page, P, most, width, room):
    for seed in range(2):
        H.log(f"8-bit fork rows={R} room={room}")
        g = gen(seed)
        tabs, N = C.tables(g, R, P, spare=R + 2)
        lens = torch.randint(0, most + 1, (R // width,), generator=g).to(I32).repeat_interleave(width)
        for r in range(R):
            tabs[r, :int(lens[r]) // page] = tabs[r // width * width, :int(lens[r]) // page]
            tabs[r, (int(lens[r]) + page - 1) // page:] = -1
        parents = ((torch.rand(R, generator=g) * width).int() + torch.arange(R) // width * width).to(I32)
        p = K.pools(g, L, N, h, page, D, BF16)
        raw, (k, v, s) = pools(p)
        t1, l1 = sampler.kv_fork(k, v, dev(tabs), dev(lens), dev(parents), room=room, scales=s)
        torch.cuda.synchronize()
        want, t2, l2 = K.fork(p, tabs, lens, parents, room)
        assert torch.equal(t1.cpu(), t2) and torch.equal(l1.cpu(), l2)
        assert all(torch.equal(x.cpu(), y) for x, y in zip(raw, want))


# ------------------------------------------------------------------ rotation

@pytest.mark.parametrize("B,T,Hq,Hk,D,dims,pairs,dt,tree,strided", [
    (1, 1, 1, 0, 16, 16, False, BF16, False, False), (3, 1, 4, 2, 64, 64, False, F16, False, False),
    (2, 9, 3, 1, 96, 96, True, BF16, True, True), (3, 64, 2, 1, 128, 64, False, BF16, True, False),
    (2, 700, 1, 1, 40, 32, True, F16, False, True), (1, 5, 2, 2, 256, 256, False, F16, True, False)])
def test_rotate(sampler, B, T, Hq, Hk, D, dims, pairs, dt, tree, strided):
    H.log(f"rotate B={B} T={T} Hq={Hq} Hk={Hk} D={D} dims={dims}")
    g = gen(T + D)
    q, k = torch.randn(B, T, Hq, D, generator=g).to(dt), torch.randn(B, T, max(Hk, 1), D, generator=g).to(dt)
    if strided:
        w = torch.randn(B, T, (Hq + Hk) * D + 7, generator=g).to(dt)
        q, k = w[..., 1:1 + Hq * D].unflatten(-1, (Hq, D)), w[..., 1 + Hq * D:1 + (Hq + Hk) * D].unflatten(-1, (Hk, D))
    k = k if Hk else None
    lens = torch.tensor([131071, 0, -1][:B], dtype=I32)
    parents = C.tree(g, B, T) if tree else None
    want = [None if x is None else K.rotate(x, lens, parents, FREQ[dims], pairs) for x in (q, k)]
    qd, kd = dev(q), dev(k)
    apart = sampler.rotate(qd, kd, dev(lens), dev(FREQ[dims]), pairs=pairs, parents=dev(parents))
    here = sampler.rotate(qd, kd, dev(lens), dev(FREQ[dims]), pairs=pairs, parents=dev(parents), q_out=qd, k_out=kd)
    torch.cuda.synchronize()
    for out in (apart, here):
        for o, w in zip(out, want):
            assert (o is None) == (w is None)
            if w is not None:
                K.check_turned16(o.cpu(), w, dims // 2, pairs)


# ------------------------------------------------------------------ together, streams, graphs, refusals

def test_a_decode_step_in_a_graph(sampler):
    """Rotation, attention over the 8-bit cache, a fork and an append captured together: every replay equals the eager
    calls on the same inputs."""
    H.log("8-bit decode step in a graph")
    g = gen(21)
    h, D, page, P, B = 2, 64, 16, 12, 8
    tabs, N = C.tables(g, B, P, spare=10)
    lens = torch.tensor([150, 3, 0, 47, 80, 16, 33, 121], dtype=I32)
    p = K.pools(g, 1, N, h, page, D, BF16)
    q = torch.randn(B, 1, 8, D, generator=g).to(BF16)
    kn, vn = (torch.randn(1, B, 1, h, D, generator=g).to(BF16) for _ in range(2))
    parents = torch.tensor([0, 0, 2, 4, 4, 5, 6, 6], dtype=I32)
    ins = [dev(t) for t in (q, kn, vn, tabs, lens, parents)]
    freq = FREQ[64].to(DEV)
    raw, (k, v, s) = pools(p)
    first = [x.clone() for x in raw]

    def step(q, kn, vn, tabs, lens, parents):
        qr, kr = sampler.rotate(q, kn[0], lens, freq)
        out = sampler.tree_attention(qr, kr, vn[0], k[0], v[0], tabs, lens, scales=s[0])
        t2, l2 = sampler.kv_fork(k, v, tabs, lens, parents, room=1, scales=s)
        l3 = sampler.kv_append(kn, vn, k, v, t2, l2, scales=s, rotary=freq)
        return [qr, kr, out, t2, l2, l3, *raw]

    def reset():
        for x, y in zip(raw, first):
            x.copy_(y)

    def eager():
        reset()
        r = [t.clone() for t in step(*ins)]
        torch.cuda.synchronize()
        return r

    eager()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(), capture_error_mode="thread_local"):
        got = step(*ins)
    torch.cuda.synchronize()
    for i in range(4):
        ins[0].copy_(torch.randn(B, 1, 8, D, generator=g).to(BF16))
        ins[1].copy_(torch.randn(1, B, 1, h, D, generator=g).to(BF16))
        want = eager()
        reset()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


def test_a_given_stream(sampler):
    q, kn, vn, p, tabs, lens, par = attn_inputs(31, 2, 4, 4, 2, 64, [300, 20], 16, BF16)
    H.log("8-bit attention on a given stream")
    _, (k, v, s) = pools(p)
    d = [dev(t) for t in (q, kn, vn)]
    rest = dict(parents=dev(par), scales=s)
    t, l = dev(tabs), dev(lens)
    ref = sampler.tree_attention(*d, k, v, t, l, **rest)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    out = torch.zeros_like(ref)
    torch.cuda.synchronize()
    sampler.tree_attention(*d, k, v, t, l, out=out, stream=stream.cuda_stream, **rest)
    stream.synchronize()
    assert torch.equal(out, ref)


def test_empty_batches(sampler):
    H.log("8-bit empty batches")
    z = torch.empty(0, dtype=I32, device=DEV)
    _, (k, v, s) = pools(K.pools(gen(1), 1, 3, 1, 16, 64, BF16))
    rows = torch.empty(1, 0, 2, 1, 64, dtype=BF16, device=DEV)
    tabs = torch.empty(0, 2, dtype=I32, device=DEV)
    f = FREQ[64].to(DEV)
    assert sampler.kv_append(rows, rows, k, v, tabs, z, scales=s, rotary=f).numel() == 0
    assert sampler.kv_fork(k, v, tabs, z, z, scales=s)[0].shape == (0, 2)
    q = torch.empty(0, 2, 1, 64, dtype=BF16, device=DEV)
    assert sampler.tree_attention(q, q, q, k[0], v[0], tabs, z, scales=s[0]).shape == (0, 2, 1, 64)
    assert sampler.rotate(q, q.clone(), z, f)[0].shape == (0, 2, 1, 64)
    t = torch.empty(0, 2, dtype=I32, device=DEV)
    assert sampler.tree_commit(rows, rows, k, v, tabs, z, t, t, t, scales=s)["lens"].numel() == 0


def test_refusals(sampler):
    H.log("8-bit refusals")
    import tinygpt_amd as tg

    q, kn, vn, p, tabs, lens, par = attn_inputs(1, 2, 3, 4, 2, 64, [20, 9], 16, BF16)
    q, kn, vn, tabs, lens, par = (dev(t) for t in (q, kn, vn, tabs, lens, par))
    _, (k, v, s) = pools(p)

    def refused(err, call, *a, **kw):
        with pytest.raises(err):
            call(*a, **kw)

    att = sampler.tree_attention
    refused(TypeError, att, q, kn, vn, k, v, tabs, lens)                                # codes without scales
    refused(TypeError, att, q, kn, vn, k, v, tabs, lens, scales=s.view(U8))
    refused(TypeError, att, q, kn, vn, k.view(U8), v.view(U8), tabs, lens, scales=s)
    refused(TypeError, att, q.float(), kn.float(), vn.float(), k, v, tabs, lens, scales=s)
    refused(ValueError, att, q, kn.half(), vn.half(), k, v, tabs, lens, scales=s)
    refused(ValueError, att, q, kn, vn, k, v, tabs, lens, scales=s[:-1])
    refused(ValueError, att, q, kn, vn, k, v, tabs, lens, scales=s.transpose(1, 2).contiguous().transpose(1, 2)[..., :1])
    refused(ValueError, att, q, kn, vn, k, v, tabs, lens, scales=s.cpu())
    refused(ValueError, att, q, kn, vn, k, v.transpose(-1, -2), tabs, lens, scales=s)
    refused(ValueError, att, q, kn, vn, k, v, tabs, lens, scales=s, out=q)
    f = FREQ[64].to(DEV)
    cache = (k[None], v[None], tabs, lens)
    rows = (kn[None], vn[None])
    refused(ValueError, sampler.kv_append, *rows, *cache, scales=s)                      # without layers
    refused(ValueError, sampler.kv_append, *rows, *cache, scales=s[None], lens_out=lens)
    refused(ValueError, sampler.kv_append, *rows, *cache, scales=s[None], rotary=f.double())
    refused(ValueError, sampler.kv_append, *rows, *cache, scales=s[None], rotary=f[None])
    refused(tg.TgsError, sampler.kv_append, *rows, *cache, scales=s[None], rotary=f[:7].contiguous())
    refused(tg.TgsError, sampler.kv_append, *rows, *cache, scales=s[None], rotary=FREQ[128].to(DEV))
    refused(ValueError, sampler.kv_fork, k[None], v[None], tabs, lens, lens.clone(), scales=s[None], tables_out=tabs)
    rot = sampler.rotate
    refused(ValueError, rot, q, kn, lens, None)
    refused(TypeError, rot, q.float(), kn.float(), lens, f)
    refused(ValueError, rot, q, kn.half(), lens, f)
    refused(ValueError, rot, q, kn, lens[:1], f)
    refused(ValueError, rot, q, kn, lens, f, parents=par[:, :2])
    refused(ValueError, rot, q, kn, lens, f, q_out=kn)
    refused(ValueError, rot, q[:, :, :2], kn, lens, f, q_out=kn)
    refused(ValueError, rot, q, kn, lens, f, q_out=q[:, :, :1].expand(2, 3, 4, 64))
    refused(tg.TgsError, rot, torch.zeros(2, 65, 1, 64, dtype=BF16, device=DEV), None, lens, f, parents=torch.zeros(2, 65, dtype=I32, device=DEV))
