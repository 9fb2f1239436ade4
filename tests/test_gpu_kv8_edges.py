"""GPU: the 8-bit cache where inputs are extreme, many layers share a workgroup, graphs
share the sampler's workspace, and calls run beside each other."""
import pytest
import torch

import gpu_harness as H
import kv8_cases as K
import kv_cases as C
from test_gpu_kv import dev
from test_gpu_kv8 import pools, run_attn
from test_kv8_edges import SHAPES, check_unseen, unseen_garbage, widened
from test_kv8_sim import FREQ, attn_inputs, write_inputs
from test_kv_sim import commit_ids, gen

pytestmark = pytest.mark.gpu
BF16, F16, I32, DEV = torch.bfloat16, torch.float16, torch.int32, "cuda:0"


@pytest.mark.parametrize("shape", [s[:-1] for s in SHAPES] + [(6, 8, 2, 64, [3000, 7, 900], 16), (40, 4, 1, 128, [6000, 0], 16)], ids=str)
def test_unseen_garbage(sampler, shape):
    for dt, chain in ((BF16, False), (F16, True), (F16, False)):
        args = unseen_garbage(*shape, dt, chain=chain)
        q, kn, vn, p, tabs, lens, par = args
        H.log(f"8-bit attention, garbage in unseen nodes {shape} {dt} chain={chain}")
        lse = torch.empty(q.shape[:3], device=DEV)
        _, (k, v, s) = pools(p)
        for more in (0, 6000):
            slots = dev(widened(args, more)[4])
            out = sampler.tree_attention(dev(q), dev(kn), dev(vn), k, v, slots, dev(lens), parents=dev(par), lse=lse, scales=s)
            torch.cuda.synchronize()
            check_unseen(out.cpu(), lse.cpu(), args)


@pytest.mark.parametrize("T,Hq,Hkv,D,lens,page,dt", [
    (1, 4, 2, 64, [1500, 0, 77, 1535], 16, F16), (5, 8, 2, 128, [1200, 130, 1536], 64, BF16), (3, 2, 1, 96, [1000, 1], 32, BF16),
    (20, 1, 1, 64, [933, 300], 16, F16), (2, 8, 1, 256, [460, 90], 64, BF16), (2, 20, 1, 96, [1500, 40], 16, F16)])
def test_shares_of_few_rows(sampler, T, Hq, Hkv, D, lens, page, dt):
    """Workers that share (sequence, key head)s, and the unshared form, of the same rows."""
    args = attn_inputs(T + D, len(lens), T, Hq, Hkv, D, lens, page, dt)
    for more in (0, 6000):
        run_attn(sampler, widened(args, more))


@pytest.mark.parametrize("dims,pairs", [(0, False), (16, True)])
def test_layers_that_share_a_workgroup(sampler, dims, pairs):
    """A batch so large that a workgroup takes several layers, whose count it does not divide."""
    L, B, T, h, D, page, dt = 37, 64, 17, 1, 16, 16, BF16
    H.log(f"8-bit append and commit, 37 layers, dims={dims}")
    kn, vn, p, tabs = write_inputs(7, L, B, T, h, D, page, 3, dt)
    lens = torch.randint(0, 29, (B,), generator=gen(7)).to(I32)
    freq = FREQ[dims] if dims else None
    raw, (k, v, s) = pools(p)
    l1 = sampler.kv_append(dev(kn), dev(vn), k, v, dev(tabs), dev(lens), scales=s, rotary=dev(freq), pairs=pairs)
    torch.cuda.synchronize()
    want, l2, put = K.append(kn, vn, p, tabs, lens, None, dt, freq, pairs)
    assert torch.equal(l1.cpu(), l2)
    K.check_written(p, [x.cpu() for x in raw], want, put, dt, dims // 2, pairs)
    if dims:
        return
    parents = C.tree(gen(8), B, T)
    draft, sampled = commit_ids(gen(9), B, T)
    raw, (k, v, s) = pools(p)
    o1 = sampler.tree_commit(dev(kn), dev(vn), k, v, dev(tabs), dev(lens), dev(parents), dev(draft), dev(sampled), scales=s)
    torch.cuda.synchronize()
    want, o2 = K.commit(kn, vn, p, tabs, lens, parents, draft, sampled, dt)
    K.check_written(p, [x.cpu() for x in raw], want, {}, dt)
    assert torch.equal(o1["lens"].cpu(), o2["lens"])


def graph_of(f):
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(), capture_error_mode="thread_local"):
        got = f()
    torch.cuda.synchronize()
    return graph, got


def test_two_graphs_share_the_workspace(sampler):
    """Attention split over workers, of an 8-bit and of a 16-bit cache, captured on one sampler and replayed in turn."""
    H.log("8-bit and 16-bit attention in two graphs")
    calls = []
    q, kn, vn, p, tabs, lens, par = attn_inputs(1, 3, 5, 8, 2, 64, [5000, 900, 3], 16, BF16)
    _, (k, v, s) = pools(p)
    d = [dev(x) for x in (q, kn, vn, tabs, lens, par)]
    calls.append((d[0], lambda: sampler.tree_attention(d[0], d[1], d[2], k, v, d[3], d[4], parents=d[5], scales=s)))
    g = gen(3)
    tabs16, N = C.tables(g, 2, 90)
    k16, v16 = (x[0].to(DEV) for x in C.pools(g, 1, N, 2, 32, 128, F16))
    e = [torch.randn(2, 40, n, 128, generator=g).to(F16).to(DEV) for n in (4, 2, 2)]
    t16, l16 = dev(tabs16), torch.tensor([2800, 70], dtype=I32, device=DEV)
    calls.append((e[0], lambda: sampler.tree_attention(*e, k16, v16, t16, l16)))
    graphs = [graph_of(f) for _, f in calls]
    for i in range(3):
        wants = []
        for x, f in calls:
            x.copy_(torch.randn(x.shape, generator=g).to(x.dtype))
            wants.append(f().clone())
        torch.cuda.synchronize()
        for j in (0, 1, 0) if i % 2 else (1, 0):
            graphs[j][0].replay()
            torch.cuda.synchronize()
            assert torch.equal(graphs[j][1], wants[j]), (i, j)


def test_a_commit_in_a_graph(sampler):
    """The accepted path's length changes from replay to replay."""
    H.log("8-bit commit in a graph")
    L, B, T, h, D, page = 2, 3, 40, 2, 64, 16
    kn, vn, p, tabs = write_inputs(3, L, B, T, h, D, page, 5, F16)
    lens = torch.tensor([0, 13, 31], dtype=I32)
    parents = torch.arange(-1, T - 1, dtype=I32).expand(B, T).contiguous()
    draft = torch.arange(T, dtype=I32).expand(B, T).contiguous()
    sampled = torch.zeros(B, T, dtype=I32)
    raw, (k, v, s) = pools(p)
    first = [x.clone() for x in raw]
    d = [dev(x) for x in (kn, vn, tabs, lens, parents, draft, sampled)]
    graph, got = graph_of(lambda: sampler.tree_commit(d[0], d[1], k, v, d[2], d[3], d[4], d[5], d[6], scales=s))
    for taken in ([1, 2, 40], [40, 17, 3], [16, 4, 33]):
        for b, n in enumerate(taken):
            sampled[b] = -7
            sampled[b, :n - 1] = draft[b, 1:n]
        d[6].copy_(sampled)
        for x, y in zip(raw, first):
            x.copy_(y)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, o2 = K.commit(kn, vn, p, tabs, lens, parents, draft, sampled, F16)
        K.check_written(p, [x.cpu() for x in raw], want, {}, F16)
        for x in o2:
            assert torch.equal(got[x].cpu(), o2[x]), x


def test_appends_beside_each_other(sampler):
    """Two streams write two halves of a batch to one cache (no page is of both)."""
    H.log("8-bit appends on two streams")
    L, B, T, h, D, page, dt = 2, 8, 50, 4, 128, 32, BF16
    kn, vn, p, tabs = write_inputs(11, L, B, T, h, D, page, 4, dt)
    lens = torch.randint(0, 40, (B,), generator=gen(5)).to(I32)
    raw, (k, v, s) = pools(p)
    d = [dev(x) for x in (kn, vn, tabs, lens)]
    torch.cuda.synchronize()
    outs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for st, part in zip(streams, (slice(0, 4), slice(4, 8))):
        with torch.cuda.stream(st):
            outs.append(sampler.kv_append(d[0][:, part], d[1][:, part], k, v, d[2][part], d[3][part], scales=s))
    torch.cuda.synchronize()
    want, l2, put = K.append(kn, vn, p, tabs, lens, None, dt)
    assert torch.equal(torch.cat(outs).cpu(), l2)
    K.check_written(p, [x.cpu() for x in raw], want, put, dt)


def test_rows_behind_the_batch_stay(sampler):
    """Outputs and pools of a padded batch: what belongs to no sequence of the call keeps its bytes."""
    H.log("8-bit calls of part of a batch")
    q, kn, vn, p, tabs, lens, par = attn_inputs(2, 3, 4, 4, 2, 64, [100, 20, 47], 16, BF16)
    _, (k, v, s) = pools(p)
    d = [dev(x) for x in (q, kn, vn, tabs, lens, par)]
    out = torch.full((5, 4, 4, 64), 7.0, dtype=BF16, device=DEV)
    lse = torch.full((5, 4, 4), 7.0, device=DEV)
    sampler.tree_attention(d[0], d[1], d[2], k, v, d[3], d[4], parents=d[5], out=out[:3], lse=lse[:3], scales=s)
    q_out = torch.full((5, 4, 4, 64), 7.0, dtype=BF16, device=DEV)
    sampler.rotate(d[0], None, d[4], FREQ[64].to(DEV), q_out=q_out[:3])
    torch.cuda.synchronize()
    for x in (out, lse, q_out):
        assert (x[3:] == 7).all() and torch.isfinite(x[:3].float()).all()
