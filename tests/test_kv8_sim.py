"""The 8-bit cache's and the rotation's kernels on the CPU simulation under
AddressSanitizer, against plain forms in 64 bits: odd sizes, strides, empty and
single-token sequences, blocks filled in part, garbage past a sequence's end, bad
pages, scales at their borders, refusals."""
import math

import pytest
import torch

import kv8_cases as K
import kv_cases as C
import kv_edges as E
from test_kv_sim import check_attn, commit_ids, gen, sim  # noqa: F401  (sim: a fixture)

BF16, F16, I32, U8 = torch.bfloat16, torch.float16, torch.int32, torch.uint8


# ------------------------------------------------------------------ attention

def attn_inputs(seed, B, T, Hq, Hkv, D, lens, page, dt, strided=False, spread=1.0):
    """Encoded pools with codes of NaN past a sequence's end, scales of NaN in blocks past it and slots without a page."""
    g = gen(seed)
    P = max(1, max((n + page - 1) // page for n in lens))
    tabs, N = C.tables(g, B, P)
    k, v, s = (x[0] for x in K.pools(g, 1, N, Hkv, page, D, dt, spread))
    q = (torch.randn(B, T, Hq, D, generator=g) * 2).to(dt)
    kn, vn = (torch.randn(B, T, Hkv, D, generator=g).to(dt) for _ in range(2))
    if strided:  # slices of one projection, at any alignment
        w = torch.randn(B, T, (Hq + 2 * Hkv) * D + 3, generator=g).to(dt)
        q = w[..., 1:1 + Hq * D].unflatten(-1, (Hq, D))
        kn = w[..., 1 + Hq * D: 1 + (Hq + Hkv) * D].unflatten(-1, (Hkv, D))
        vn = w[..., 1 + (Hq + Hkv) * D: 1 + (Hq + 2 * Hkv) * D].unflatten(-1, (Hkv, D))
    lens = torch.tensor(lens, dtype=I32)
    parents = C.tree(g, B, T)
    for b in range(B):
        n = int(lens[b])
        for i in range(P):
            p, held = int(tabs[b, i]), min(max(n - i * page, 0), page)
            k[p, :, held:] = 0x7F
            x = v[p].transpose(-1, -2).reshape(Hkv, page, D).clone()
            x[:, held:] = 0xFF
            v[p] = x.view(Hkv, page // K.BLOCK, K.BLOCK, D).transpose(-1, -2)
            s[p, :, (held + K.BLOCK - 1) // K.BLOCK:] = 255
            if held == 0:
                tabs[b, i] = -1 if i % 2 else N + 5
    return q, kn, vn, [k, v, s], tabs, lens, parents


def wanted(args, scale=None, parents=True):
    q, kn, vn, p, tabs, lens, par = args
    kd, vd = K.decoded(p)
    return C.attention(q, kn, vn, kd, vd, tabs, lens, par if parents else None, q.shape[-1] ** -0.5 if scale is None else scale)


def vmax_of(args):
    v = K.decoded(args[3])[1]
    return max(float(args[2].double().abs().max()), float(v[torch.isfinite(v)].abs().max()))


def run_attn(sim, args, scale=None, parents=True, **kw):  # noqa: F811
    q, kn, vn, p, tabs, lens, par = args
    rc, out, lse = K.sim_attention(sim, q, kn, vn, p, tabs, lens, par if parents else None, scale, **kw)
    assert rc == 0
    # (what the cache stands for is exact in the rows' type, so the bounds are those of a 16-bit cache)
    check_attn(out, lse, *wanted(args, scale, parents), vmax_of(args), q.dtype)


@pytest.mark.parametrize("T,Hq,Hkv,D,lens,page,dt,cu", [
    (1, 1, 1, 64, [0], 16, BF16, 4),
    (1, 8, 2, 64, [1, 33, 70], 16, F16, 4),
    (3, 7, 1, 96, [31, 0, 64], 32, BF16, 4),
    (2, 4, 2, 128, [300, 5], 64, BF16, 2),
    (9, 6, 2, 64, [130], 32, F16, 4),
    (1, 2, 1, 256, [90], 128, BF16, 4),
    (32, 1, 1, 64, [40], 16, BF16, 4),
    (11, 2, 1, 96, [65, 127], 16, F16, 4),
    (5, 4, 1, 256, [17], 16, F16, 4),
])
def test_attention_few_rows(sim, T, Hq, Hkv, D, lens, page, dt, cu):  # noqa: F811
    run_attn(sim, attn_inputs(T * D + len(lens), len(lens), T, Hq, Hkv, D, lens, page, dt), num_cu=cu)


@pytest.mark.parametrize("T,Hq,Hkv,D,lens,page,dt", [
    (33, 1, 1, 64, [70], 16, F16),
    (9, 8, 2, 128, [65, 0], 64, BF16),
    (64, 2, 1, 96, [100], 16, BF16),
    (40, 4, 1, 64, [1], 32, BF16),
    (20, 2, 1, 256, [66], 32, F16),
    (48, 4, 1, 96, [47], 16, F16),
])
def test_attention_many_rows(sim, T, Hq, Hkv, D, lens, page, dt):  # noqa: F811
    run_attn(sim, attn_inputs(T * D, len(lens), T, Hq, Hkv, D, lens, page, dt), num_cu=2)


@pytest.mark.parametrize("T,Hq,Hkv,lens,max_len,cu", [
    (1, 2, 2, [1700, 3, 611], None, 4),   # shares that start and end inside sequences
    (2, 4, 1, [1640], None, 7),
    (40, 1, 1, [900], None, 2),           # the same with tiles in LDS
    (33, 8, 1, [700], None, 16),          # and two groups of rows, eight workers each
    (1, 2, 1, [1000], 20, 3),             # a bound of the lengths that is too low changes nothing
])
def test_attention_split(sim, T, Hq, Hkv, lens, max_len, cu):  # noqa: F811
    run_attn(sim, attn_inputs(sum(lens) + T, len(lens), T, Hq, Hkv, 64, lens, 32, BF16), num_cu=cu, max_len=max_len)


def test_attention_strided_rows_chain_and_scale(sim):  # noqa: F811
    run_attn(sim, attn_inputs(3, 2, 5, 4, 2, 64, [17, 40], 16, BF16, strided=True), parents=False, scale=0.3, want_lse=False)
    run_attn(sim, attn_inputs(4, 1, 35, 2, 2, 64, [17], 16, F16, strided=True), parents=False, scale=0.3)


@pytest.mark.parametrize("T", [2, 40])
def test_attention_bad_pages_lengths_and_parents(sim, T):  # noqa: F811
    q, kn, vn, p, tabs, lens, par = attn_inputs(11, 5, T, 1, 1, 64, [40, 40, 40, 40, 40], 16, BF16)
    tabs[1, 1] = p[0].shape[0]
    lens[2], lens[3], lens[4] = -5, 3 * 16 + 9, -1   # below 0: none; past the table: all of it; failed: NaN
    last = int(tabs[3, 2])
    p[0][last], p[1][last], p[2][last] = 0x30, 0x28, 127
    par[0, 1] = T - 1 if T > 2 else 1                # no earlier node: a root
    rc, out, lse = K.sim_attention(sim, q, kn, vn, p, tabs, lens, par)
    assert rc == 0 and torch.isnan(out[4].float()).all() and torch.isnan(lse[4]).all()
    want, want_lse = wanted((q, kn, vn, p, tabs, lens, par))
    check_attn(out[:4], lse[:4], want[:4], want_lse[:4], vmax_of((q, kn, vn, p, tabs, lens, par)), BF16)


def test_attention_scales_of_nan(sim):  # noqa: F811
    """A block whose scale is NaN reaches every row, one of another sequence does not."""
    for T in (2, 40):
        q, kn, vn, p, tabs, lens, par = attn_inputs(17, 3, T, 1, 1, 64, [40, 40, 40], 16, F16)
        p[2][int(tabs[0, 1]), 0, 0, 0] = 255
        p[2][int(tabs[1, 2]), 0, 0, 1] = 255
        rc, out, _ = K.sim_attention(sim, q, kn, vn, p, tabs, lens, par)
        assert rc == 0 and torch.isnan(out[:2].float()).all() and torch.isfinite(out[2].float()).all()


@pytest.mark.parametrize("dt,spread", [(BF16, 12.0), (F16, 3.0)])
def test_attention_far_scales(sim, dt, spread):  # noqa: F811
    """Blocks whose scales lie far apart, up to the type's range and down to its floor; few rows and many."""
    for T in (2, 40):
        q, kn, vn, p, tabs, lens, par = attn_inputs(19, 1, T, 1, 1, 64, [77], 16, dt)
        pages = tabs[0].long()
        # values of block i: 2^(i spread) apart, keys small enough for scores that differ by less than a few units
        for i, pg in enumerate(pages.tolist()):
            p[2][pg, ..., 0] = 112
            p[2][pg, 0, :, 1] = 127 - int(spread) * i
        run_attn(sim, (q, kn, vn, p, tabs, lens, par))
    # the smallest scale: steps of 2^-24 in fp16, which its denormal numbers hold
    q, kn, vn, p, tabs, lens, par = attn_inputs(23, 1, 1, 1, 1, 64, [64], 16, dt)
    p[2][..., 1] = K.FLOOR[dt] + 127
    vn.zero_()
    rc, out, _ = K.sim_attention(sim, q, kn, vn, p, tabs, lens, par)
    want, _ = wanted((q, kn, vn, p, tabs, lens, par))
    # (half a step of the weights and of the result, and of fp16 half a step of its denormal numbers)
    step = torch.finfo(dt).eps
    assert rc == 0 and ((out.double() - want).abs() <= step * vmax_of((q, kn, vn, p, tabs, lens, par)) + (2.0**-25 if dt == F16 else 0)).all()


# ------------------------------------------------------------------ writes

def write_inputs(seed, L, B, T, H, D, page, P, dt, strided=False, spread=1.0):
    g = gen(seed)
    tabs, N = C.tables(g, B, P)
    p = K.pools(g, L, N, H, page, D, dt)
    kn, vn = (torch.randn(L, B, T, H, D, generator=g) * torch.exp2(spread * torch.randn(L, B, T, H, 1, generator=g)) for _ in range(2))
    kn, vn = kn.to(dt), vn.to(dt)
    if strided:
        w = torch.randn(L, B, T, 2 * H * D + 5, generator=g).to(dt)
        kn, vn = w[..., 1:1 + H * D].unflatten(-1, (H, D)), w[..., 1 + H * D:1 + 2 * H * D].unflatten(-1, (H, D))
    return kn, vn, p, tabs


FREQ = {n: (10000.0 ** (-torch.arange(n // 2).double() / (n // 2))).float() for n in (16, 32, 64, 96, 128, 256)}


@pytest.mark.parametrize("L,B,T,H,D,page,dt,strided,dims,pairs", [
    (1, 1, 1, 1, 16, 16, BF16, False, 0, False), (2, 3, 1, 2, 64, 16, F16, False, 64, False),
    (2, 4, 21, 3, 48, 16, BF16, True, 16, True), (1, 3, 40, 8, 128, 64, BF16, False, 128, False),
    (1, 2, 37, 1, 96, 32, F16, False, 96, True), (1, 2, 18, 2, 256, 16, BF16, False, 128, False),
    (1, 2, 20, 5, 80, 32, F16, True, 0, False), (1, 1, 33, 1, 256, 32, F16, False, 256, True),
    (1, 2, 19, 1, 112, 16, BF16, False, 32, False)])
def test_append(sim, L, B, T, H, D, page, dt, strided, dims, pairs):  # noqa: F811
    P = (T + 30 + page - 1) // page
    kn, vn, p, tabs = write_inputs(T + D, L, B, T, H, D, page, P, dt, strided)
    g = gen(T)
    lens = torch.randint(0, 29, (B,), generator=g).to(I32)
    counts = torch.randint(0, T + 1, (B,), generator=g).to(I32)
    freq = FREQ[dims] if dims else None
    for c in (counts, None):
        rc, q, l1 = K.sim_append(sim, kn, vn, p, tabs, lens, c, freq, pairs)
        want, l2, put = K.append(kn, vn, p, tabs, lens, c, dt, freq, pairs)
        assert rc == 0 and torch.equal(l1, l2)
        K.check_written(p, q, want, put, dt, dims // 2, pairs)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_append_token_by_token(sim, dt):  # noqa: F811
    """A block filled one row at a time, of rising and falling magnitudes: its scale grows, the earlier codes are rounded again."""
    kn, vn, p, tabs = write_inputs(5, 1, 1, 24, 1, 32, 16, 2, dt)
    kn *= torch.exp2(torch.tensor([0, 1, 3, 2, 9, -4] * 4).float())[None, None, :, None, None].to(dt)
    q, lens = p, torch.zeros(1, dtype=I32)
    want, wl = p, lens
    for t in range(24):
        rows = kn[:, :, t:t + 1].contiguous(), vn[:, :, t:t + 1].contiguous()
        rc, q, lens = K.sim_append(sim, *rows, q, tabs, lens, None)
        want, wl, put = K.append(*rows, want, tabs, wl, None, dt)
        assert rc == 0 and torch.equal(lens, wl)
        K.check_written(p, q, want, put, dt)


def border_rows(dt):
    """Rows [n, 16] whose blocks lie at the borders of scales, of the type's range and of what is finite."""
    tiny, big = torch.finfo(dt).tiny, torch.finfo(dt).max
    sub = tiny * torch.finfo(dt).eps
    f = 2.0**-16
    rows = [[0.0] * 16, [448.0 * f] * 16, [449.0 * f] * 16, [450.0 * f] * 16, [-448.0] * 16, [-452.0] * 16, [big, -big] * 8,
            [tiny, sub, -sub] * 5 + [0.0], [big, sub] * 8, [448.0 * 2.0**K.FLOOR[dt]] * 16,
            [math.inf, 1.0] * 8, [-math.inf] * 16, [math.nan, 2.0] * 8, [math.nan] * 16, [-0.0, 0.0] * 8,
            [float(x) for x in range(240, 272, 2)], [2.0**-k for k in range(16)], [61440.0, 61472.0, 63488.0, 65504.0] * 4]
    return torch.tensor(rows, dtype=torch.float64).to(dt)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_append_borders(sim, dt):  # noqa: F811
    """Each row alone in a block, and after others; codes that round to 448 and to the next scale."""
    rows = border_rows(dt)
    n = len(rows)
    kn = rows[None, :, None, None, :].contiguous()      # one token of n sequences, D = 16
    vn = kn.flip(1).contiguous()
    g = gen(3)
    tabs, N = C.tables(g, n, 1)
    p = K.pools(g, 1, N, 1, 16, 16, dt)
    for held in (0, 3):
        lens = torch.full((n,), held, dtype=I32)
        rc, q, l1 = K.sim_append(sim, kn, vn, p, tabs, lens, None)
        want, l2, put = K.append(kn, vn, p, tabs, lens, None, dt)
        assert rc == 0 and torch.equal(l1, l2)
        K.check_written(p, q, want, put, dt)
        # what is finite is finite in the type
        s = q[2][0, tabs[:, 0].long(), 0, 0]
        for i in range(n):
            x = K.numbers(q[0][0, int(tabs[i, 0]), 0, held], s[i, 0])
            fin = torch.isfinite(rows[i])
            assert torch.isfinite(x[fin].to(dt)).all() and torch.isnan(x[~fin]).all()
            assert torch.equal(x[fin].to(dt).double(), x[fin])


def test_append_to_a_block_of_foreign_scales(sim):  # noqa: F811
    """Held blocks whose scale another program wrote: NaN stays NaN, the extremes stay what they are."""
    kn, vn, p, tabs = write_inputs(6, 1, 6, 2, 1, 16, 16, 1, BF16)
    for b, byte in enumerate((255, 254, 0, 1, 26, 250)):
        p[2][0, int(tabs[b, 0])] = byte
    lens = torch.full((6,), 5, dtype=I32)
    rc, q, _ = K.sim_append(sim, kn, vn, p, tabs, lens, None)
    assert rc == 0
    for b, byte in enumerate((255, 254, 0, 1, 26, 250)):
        pg = int(tabs[b, 0])
        for which, x in ((0, kn), (1, vn)):
            s = int(q[2][0, pg, 0, 0, which])
            codes = K.block(q, 0, pg, 0, 0)[which]
            if byte == 255:
                assert s == 255
                continue
            e = max(K.need(x[0, b].double(), BF16) + 127, byte)
            assert s == e
            assert K.same(codes[5:7].contiguous(), K.encode(x[0, b, :, 0].double(), e - 127, BF16))
            old = K.numbers(K.block(p, 0, pg, 0, 0)[which][:5].contiguous(), torch.tensor(byte))
            assert K.same(codes[:5].contiguous(), K.encode(old, e - 127))


def test_append_rows_that_do_not_fit(sim):  # noqa: F811
    kn, vn, p, tabs = write_inputs(7, 2, 6, 10, 1, 16, 16, 4, BF16)
    tabs[2, 1], tabs[3, 3] = -1, p[0].shape[1]
    lens = torch.tensor([62, 5, 8, 9, -1, 0], dtype=I32)
    counts = torch.tensor([3, 11, 9, 10, 1, -2], dtype=I32)  # past the table, past T, a bad page; fits; bad length, bad count
    rc, q, l1 = K.sim_append(sim, kn, vn, p, tabs, lens, counts)
    want, l2, put = K.append(kn, vn, p, tabs, lens, counts, BF16)
    assert l2.tolist() == [-1, -1, -1, 19, -1, -1]
    assert rc == 0 and torch.equal(l1, l2)
    K.check_written(p, q, want, put, BF16)


@pytest.mark.parametrize("L,B,T,H,D,page,dt,dims,pairs", [
    (1, 1, 1, 1, 16, 8, BF16, 16, False), (2, 4, 21, 3, 24, 8, BF16, 16, True), (1, 3, 40, 8, 128, 64, BF16, 128, False),
    (1, 2, 9, 2, 72, 16, F16, 64, False), (1, 2, 12, 1, 96, 16, F16, 96, True)])
def test_append_rotated(sim, L, B, T, H, D, page, dt, dims, pairs):  # noqa: F811
    """16-bit caches: turned keys within a rounding, everything else as an append leaves it."""
    g = gen(T + D)
    P = (T + 30 + page - 1) // page
    tabs, N = C.tables(g, B, P)
    k, v = C.pools(g, L, N, H, page, D, dt)
    kn, vn = (torch.randn(L, B, T, H, D, generator=g).to(dt) for _ in range(2))
    if T > 10:
        w = torch.randn(L, B, T, H * D + 5, generator=g).to(dt)
        kn = w[..., 1:1 + H * D].unflatten(-1, (H, D))
    lens = torch.randint(0, 29, (B,), generator=g).to(I32)
    counts = torch.randint(0, T + 1, (B,), generator=g).to(I32)
    for c in (counts, None):
        rc, k1, v1, l1 = K.sim_append_rotated(sim, kn, vn, k, v, tabs, lens, c, FREQ[dims], pairs)
        k2, v2, l2 = C.append(kn, vn, k, v, tabs, lens, c)
        assert rc == 0 and torch.equal(v1, v2) and torch.equal(l1, l2)
        for b in range(B):
            n = T if c is None else int(c[b])
            for i in range(n):
                pos = int(lens[b]) + i
                pg, slot = int(tabs[b, pos // page]), pos % page
                want = K.turned(kn[:, b, i].double(), pos, FREQ[dims], pairs)
                K.check_turned16(k1[:, pg, :, slot], want, dims // 2, pairs)
                k2[:, pg, :, slot] = k1[:, pg, :, slot]
        assert torch.equal(k1, k2)


@pytest.mark.parametrize("L,B,T,H,D,page,dt", [(1, 2, 1, 1, 16, 16, BF16), (2, 5, 9, 2, 64, 16, F16), (1, 3, 64, 2, 128, 32, BF16)])
def test_commit(sim, L, B, T, H, D, page, dt):  # noqa: F811
    P = (T + 30 + page - 1) // page
    kn, vn, p, tabs = write_inputs(T + D, L, B, T, H, D, page, P, dt)
    g = gen(T)
    lens = torch.randint(0, 29, (B,), generator=g).to(I32)
    if B > 2:
        lens[0] = P * page  # no room for the root
    parents = C.tree(g, B, T)
    draft, sampled = commit_ids(g, B, T)
    if T == 64:  # a path through every node
        parents[1] = torch.arange(-1, T - 1)
        draft[1], sampled[1] = 1, 1
    rc, q, o1 = K.sim_commit(sim, kn, vn, p, tabs, lens, parents, draft, sampled)
    want, o2 = K.commit(kn, vn, p, tabs, lens, parents, draft, sampled, dt)
    assert rc == 0
    K.check_written(p, q, want, {}, dt)
    for x in o2:
        assert torch.equal(o1[x], o2[x]), x


# ------------------------------------------------------------------ forks

def check_fork(sim, p, tabs, lens, parents, room):  # noqa: F811
    rc, q, t1, l1 = K.sim_fork(sim, p, tabs, lens, parents, room)
    want, t2, l2 = K.fork(p, tabs, lens, parents, room)
    assert rc == 0 and torch.equal(t1, t2) and torch.equal(l1, l2)
    assert all(torch.equal(x, y) for x, y in zip(q, want))
    return l2


@pytest.mark.parametrize("L,R,H,D,page,P,most,width,room", [
    (1, 1, 1, 16, 16, 2, 9, 1, 1), (2, 8, 2, 64, 32, 4, 90, 4, 1), (1, 6, 1, 16, 16, 6, 50, 3, 17), (1, 8, 1, 48, 64, 4, 200, 8, 0)])
def test_fork(sim, L, R, H, D, page, P, most, width, room):  # noqa: F811
    for seed in range(3):
        g = gen(seed)
        tabs, N = C.tables(g, R, P, spare=R + 2)
        lens = torch.randint(0, most + 1, (R // width,), generator=g).to(I32).repeat_interleave(width)
        for r in range(R):
            tabs[r, :int(lens[r]) // page] = tabs[r // width * width, :int(lens[r]) // page]
            tabs[r, (int(lens[r]) + page - 1) // page:] = -1
        parents = ((torch.rand(R, generator=g) * width).int() + torch.arange(R) // width * width).to(I32)
        check_fork(sim, K.pools(g, L, N, H, page, D, BF16), tabs, lens, parents, room)


@pytest.mark.parametrize("cases", [E.SHORT_POOLS, E.BAD_ENTRIES, E.FAILED_LENGTHS])
@pytest.mark.parametrize("layers", [1, 4])
def test_fork_short_pools_bad_entries_and_failed_lengths(sim, cases, layers):  # noqa: F811
    """The 16-bit cache's cases with pages and lengths of twice the tokens."""
    for (k, _, tabs, lens, parents), room, *_ in cases.values():
        lens = torch.where(lens > 0, 2 * lens, lens)
        check_fork(sim, K.pools(gen(1), layers, k.shape[1], 1, 16, 16, BF16), tabs, lens, parents, 2 * room)


def test_fork_of_a_large_pool(sim):  # noqa: F811
    """More pages than the plan's lists in LDS hold."""
    tabs, lens = torch.tensor([[3, 4], [3, 5]], dtype=I32), torch.tensor([25, 25], dtype=I32)
    check_fork(sim, K.pools(gen(1), 1, 20000, 1, 16, 16, BF16), tabs, lens, torch.tensor([1, 1], dtype=I32), 1)


# ------------------------------------------------------------------ rotation

@pytest.mark.parametrize("B,T,Hq,Hk,D,dims,pairs,dt,tree,strided", [
    (1, 1, 1, 0, 16, 16, False, BF16, False, False), (3, 1, 4, 2, 64, 64, False, F16, False, False),
    (2, 9, 3, 1, 96, 96, True, BF16, True, True), (1, 64, 2, 1, 128, 64, False, BF16, True, False),
    (2, 70, 1, 1, 40, 32, True, F16, False, True), (1, 5, 2, 2, 256, 256, False, F16, True, False)])
def test_rotate(sim, B, T, Hq, Hk, D, dims, pairs, dt, tree, strided):  # noqa: F811
    g = gen(T + D)
    q, k = torch.randn(B, T, Hq, D, generator=g).to(dt), torch.randn(B, T, max(Hk, 1), D, generator=g).to(dt)
    if strided:
        w = torch.randn(B, T, (Hq + Hk) * D + 7, generator=g).to(dt)
        q, k = w[..., 1:1 + Hq * D].unflatten(-1, (Hq, D)), w[..., 1 + Hq * D:1 + (Hq + Hk) * D].unflatten(-1, (Hk, D))
    k = k if Hk else None
    lens = torch.tensor([131071, 0, -1][:B], dtype=I32)
    parents = C.tree(g, B, T) if tree else None
    if tree:
        parents[0, 1] = T - 1  # no earlier node: a root
    for cu in (1, 256):  # four tokens to a workgroup, and one
        for here in (False, True):
            rc, oq, ok = K.sim_rotate(sim, q, k, lens, parents, FREQ[dims], pairs, here=here, num_cu=cu)
            assert rc == 0
            for x, o in ((q, oq), (k, ok)):
                if x is not None:
                    K.check_turned16(o, K.rotate(x, lens, parents, FREQ[dims], pairs), dims // 2, pairs)


def test_rotate_far_positions_and_extreme_frequencies(sim):  # noqa: F811
    """Positions up to 2^31 - 1 at frequencies whose products lose 32-bit numbers' last angle bits; 0, large and negative ones."""
    freq = torch.tensor([1.0, 0.7391, -0.25, 0.0, 3.14159274, 1e-30, 1000.1, 1e-4])
    q = torch.randn(4, 1, 1, 16, generator=gen(1)).to(F16)
    lens = torch.tensor([2**31 - 1, 2**24 + 1, 1000003, 7], dtype=I32)
    rc, oq, _ = K.sim_rotate(sim, q, None, lens, None, freq, True)
    assert rc == 0
    want = K.rotate(q, lens, None, freq, True)
    # the angle's 64-bit product is off by 2^-53 of it, in turns: at 2^31 * 1000 / 2 pi turns below 2^-14 of one
    slack = 2.0**-12 * K.pair_size(want, 8, True)
    assert ((oq.double() - want).abs()[0] <= 2.0**-11 * want.abs()[0] + slack[0]).all()
    K.check_turned16(oq[1:], want[1:], 8, True)


def test_rotate_then_append_is_append_rotated(sim):  # noqa: F811
    """A chain turned ahead of an append and one turned on the way hold the same 16-bit numbers."""
    g = gen(8)
    kn, vn = (torch.randn(1, 2, 12, 2, 64, generator=g).to(BF16) for _ in range(2))
    tabs, N = C.tables(g, 2, 3)
    k, v = C.pools(g, 1, N, 2, 16, 64, BF16)
    lens = torch.tensor([7, 20], dtype=I32)
    rc, turned, _ = K.sim_rotate(sim, kn[0], None, lens, None, FREQ[64], False)
    rc1, k1, v1, _ = K.sim_append_rotated(sim, kn, vn, k, v, tabs, lens, None, FREQ[64], False)
    rc2, k2, v2, _ = C.sim_append(sim, turned[None].contiguous(), vn, k, v, tabs, lens, None)
    assert rc == rc1 == rc2 == 0 and torch.equal(k1, k2) and torch.equal(v1, v2)


# ------------------------------------------------------------------ refusals

def test_refusals(sim):  # noqa: F811
    a = attn_inputs(1, 1, 2, 2, 1, 64, [9], 16, BF16)
    q, kn, vn, p, tabs, lens, par = a
    assert K.sim_attention(sim, *a, scale=-1.0)[0] == -1
    assert K.sim_attention(sim, *attn_inputs(1, 1, 2, 2, 1, 32, [9], 16, BF16))[0] == -1   # head_dim
    assert K.sim_attention(sim, *attn_inputs(1, 1, 2, 3, 2, 64, [9], 16, BF16))[0] == -1   # heads
    assert K.sim_attention(sim, *attn_inputs(1, 1, 65, 1, 1, 64, [9], 16, BF16))[0] == -1  # nodes
    assert K.sim_attention(sim, q.float(), kn, vn, p, tabs, lens, par)[0] == -1            # type
    kn, vn, p, tabs = write_inputs(1, 1, 1, 2, 1, 16, 16, 2, BF16)
    lens = torch.zeros(1, dtype=I32)
    assert K.sim_append(sim, kn.float(), vn.float(), p, tabs, lens, None)[0] == -1         # type
    assert K.sim_append(sim, kn, vn, p, tabs, lens, None, torch.ones(16))[0] == -1         # more dims than a head has
    assert K.sim_append(sim, kn, vn, p, tabs, lens, None, torch.ones(4))[0] == -1          # no multiple of 16
    wide = write_inputs(1, 1, 1, 2, 1, 272, 16, 2, BF16)
    assert K.sim_append(sim, *wide, lens, None)[0] == -1                                   # head_dim
    assert K.sim_fork(sim, p, tabs, lens, lens, -1)[0] == -1
    assert K.sim_fork(sim, p, tabs, lens, lens, 1, ws_words=1)[0] == -5
    odd = [x.clone() for x in p]
    odd[0] = torch.zeros(1, p[0].shape[1], 16 * 16 + 8, dtype=U8)[..., :256].unflatten(-1, (1, 16, 16))
    assert K.sim_append(sim, kn, vn, odd, tabs, lens, None)[0] == -1                       # a page's stride
    q = torch.zeros(1, 65, 1, 16, dtype=BF16)
    par = torch.zeros(1, 65, dtype=I32)
    assert K.sim_rotate(sim, q, None, lens, par, torch.ones(8), False)[0] == -1            # nodes
    assert K.sim_rotate(sim, q, None, lens, None, torch.ones(16), False)[0] == -1          # dims
    assert K.sim_rotate(sim, q.expand(1, 65, 2, 16), None, lens, None, torch.ones(8), False, here=True)[0] == -1  # rows that share memory
    assert K.sim_rotate(sim, q.float(), None, lens, None, torch.ones(8), False)[0] == -1   # type
