"""GPU: the beam, tree-attention and cache calls where their inputs are extreme
(the CPU simulation's cases of test_kv_edges.py at larger sizes)."""
import pytest
import torch

import gpu_harness as H
import kv_cases as C
import kv_edges as E
from test_gpu_kv import attn_inputs, check_attn, cpu, dev, write_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# ------------------------------------------------------------------ beams

@pytest.mark.parametrize("case", E.MASKS, ids=E.mask_name)
def test_beam_finite_masks(sampler, case):
    H.log(f"beam finite masks {E.mask_name(case)}")
    x, scores = E.masked_logits(*case, V=32003)
    got = sampler.beam_select(dev(x), scores.to(DEV), 3, 5)
    torch.cuda.synchronize()
    E.check_beam(cpu(got), C.beam(x, scores, 3, 5), x)


@pytest.mark.parametrize("dt", [E.F32, E.BF16])
def test_beam_large_logits(sampler, dt):
    H.log(f"beam large logits {dt}")
    x, scores = E.large_logits(dt, V=20001)
    got = sampler.beam_select(dev(x), scores.to(DEV), 2, 6)
    torch.cuda.synchronize()
    E.check_beam(cpu(got), C.beam(x, scores, 2, 6), x)


# ------------------------------------------------------------------ forks

def run_fork(sampler, case, room):
    H.log(f"fork rows={case[2].shape[0]} pages={case[0].shape[1]} room={room}")
    k, v = dev(case[0]), dev(case[1])
    t1, l1 = sampler.kv_fork(k, v, *(dev(x) for x in case[2:]), room=room)
    torch.cuda.synchronize()
    k2, v2, t2, l2 = E.fork(*case, room)
    assert torch.equal(t1.cpu(), t2) and torch.equal(l1.cpu(), l2) and torch.equal(k.cpu(), k2) and torch.equal(v.cpu(), v2)
    return t1.tolist(), l1.tolist()


@pytest.mark.parametrize("name", list(E.SHORT_POOLS))
@pytest.mark.parametrize("layers", [1, 200])
def test_fork_short_pools(sampler, name, layers):
    (k, v, *rest), room, tabs, lens = E.SHORT_POOLS[name]
    case = (k.repeat(layers, 1, 1, 1, 1), v.repeat(layers, 1, 1, 1, 1, 1), *rest)
    assert run_fork(sampler, case, room) == (tabs, lens)


def test_fork_short_pool_of_many_rows(sampler):
    case = E.many_short_rows()
    _, lens = run_fork(sampler, case[:5], case[5])
    assert -1 in lens[:1024] and max(lens[lens.index(-1):1024]) > 0


@pytest.mark.parametrize("name", list(E.BAD_ENTRIES))
@pytest.mark.parametrize("spare", [0, 20000])
def test_fork_entries_outside_the_pool(sampler, name, spare):
    """Reported by the length -1 (spare: pages of no row, so many that the plan's lists lie in the workspace)."""
    (k, v, t, n, p), room, tabs, lens = E.BAD_ENTRIES[name]
    if spare:
        k = torch.cat([k, k.new_zeros(1, spare, *k.shape[2:])], 1)
        v = torch.cat([v, v.new_zeros(1, spare, *v.shape[2:])], 1)
        t = torch.where(t >= 8, t + spare, t)
        tabs = [[x + spare if x >= 8 else x for x in row] for row in tabs]
    case = (k, v, t, n, p)
    assert run_fork(sampler, case, room) == (tabs, lens)


@pytest.mark.parametrize("name", list(E.FAILED_LENGTHS))
def test_fork_failed_lengths(sampler, name):
    """A row that failed before does not become an empty one."""
    case, room, tabs, lens = E.FAILED_LENGTHS[name]
    assert run_fork(sampler, case, room) == (tabs, lens)


# ------------------------------------------------------------------ attention

def run_attn(sampler, args, max_len=None):
    q, kn, vn, k, v, tabs, lens, par = args
    B, T, Hq, D = q.shape
    H.log(f"attention B={B} T={T} Hq={Hq} Hkv={kn.shape[2]} D={D} lens={lens.tolist()[:4]} {q.dtype}")
    lse = torch.empty(B, T, Hq, device=DEV)
    out = sampler.tree_attention(*(dev(t) for t in args[:7]), parents=dev(par), max_len=max_len, lse=lse)
    torch.cuda.synchronize()
    want, want_lse = E.attention(args)
    finite = [x.double()[torch.isfinite(x.double())].abs().max() for x in (vn, v)]
    check_attn(out.cpu(), lse.cpu(), want, want_lse, float(max(finite)), q.dtype)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_attention_of_failed_sequences(sampler, T):
    run_attn(sampler, E.failed_attention(T))
    run_attn(sampler, E.failed_attention(T), max_len=4000)


@pytest.mark.parametrize("shape", [s[:-1] for s in E.UNSEEN] + [(6, 8, 2, 64, [3000, 7, 900], 16), (40, 4, 1, 128, [6000, 0], 16)], ids=str)
@pytest.mark.parametrize("chain", [False, True])
def test_attention_garbage_in_nodes_that_are_not_seen(sampler, shape, chain):
    for dt in (E.BF16, E.F16):
        args = E.unseen_garbage(*shape, dt, chain=chain)
        q, kn, vn, k, v, tabs, lens, par = args
        H.log(f"attention, garbage in unseen nodes {shape} {dt} chain={chain}")
        lse = torch.empty(q.shape[:3], device=DEV)
        out = sampler.tree_attention(*(dev(t) for t in args[:7]), parents=dev(par), lse=lse)
        torch.cuda.synchronize()
        E.check_unseen(out.cpu(), lse.cpu(), args, check_attn)


@pytest.mark.parametrize("T,D,n", [(1, 128, 40000), (3, 256, 330), (40, 64, 9000), (36, 128, 200)])
@pytest.mark.parametrize("dt", [E.BF16, E.F16])
def test_attention_faint_tail(sampler, T, D, n, dt):
    args, scale = E.faint_tail(D, dt, n, T=T)
    H.log(f"attention of a faint tail T={T} D={D} n={n} {dt}")
    lse = torch.empty(1, T, 1, device=DEV)
    out = sampler.tree_attention(*(dev(t) for t in args[:7]), scale=scale, lse=lse)
    torch.cuda.synchronize()
    E.check_faint_tail(out.cpu(), lse.cpu(), args, scale)


# ------------------------------------------------------------------ appends

def test_append_of_few_of_many_rows(sampler):
    """Rows of a shape whose blocks are more than a grid holds, of which the counts take a few."""
    H.log("append, 140 million rows of which 21")
    T = 140_000_000
    kn, vn, k, v, tabs = write_inputs(5, 1, 2, 1, 1, 8, 8, 3, E.BF16)
    lens = torch.tensor([3, 0], dtype=torch.int32)
    counts = torch.tensor([21, 0], dtype=torch.int32)
    kd, vd = dev(k), dev(v)
    rows = [dev(x).expand(1, 2, T, 1, 8) for x in (kn, vn)]
    l1 = sampler.kv_append(*rows, kd, vd, dev(tabs), dev(lens), counts=dev(counts))
    torch.cuda.synchronize()
    k2, v2, l2 = C.append(*(x.expand(1, 2, 21, 1, 8) for x in (kn, vn)), k, v, tabs, lens, counts)
    assert torch.equal(kd.cpu(), k2) and torch.equal(vd.cpu(), v2) and torch.equal(l1.cpu(), l2)


# ------------------------------------------------------------------ every token's value, many sequences

@pytest.mark.parametrize("T,G,Hkv,D,lens", [
    (1, 4, 2, 64, [5000, 64, 901]), (8, 4, 4, 128, [4096, 100, 2049, 1]), (5, 8, 2, 128, [9000, 5]), (63, 8, 1, 128, [6000, 2000]),
    (40, 2, 2, 64, [3000, 3]), (7, 4, 1, 256, [2500]), (30, 4, 1, 256, [2500, 70]), (48, 1, 2, 96, [1900, 333])])
@pytest.mark.parametrize("dt", [E.BF16, E.F16])
def test_attention_takes_each_tokens_value(sampler, T, G, Hkv, D, lens, dt):
    """Rows that ask for one token each, spread over every tile of the contexts."""
    k, v, tabs, n, keys, values, rows = E.named_tokens(len(lens), T, G, Hkv, D, lens, 64, dt)
    d = [dev(x) for x in (rows, rows, k, v, tabs, n)]
    step = max(1, -(-max(lens) // (T * G)))  # (the rows of a call spread over the longest context)
    for first in range(0, step, max(1, min(step // 3, 29))):
        H.log(f"attention of named tokens T={T} G={G} D={D} lens={lens} first={first} {dt}")
        q, at = E.queries(keys, n, T, G, first, step)
        out = sampler.tree_attention(dev(q), *d, scale=2.0)
        torch.cuda.synchronize()
        E.check_named(out.cpu(), at, values)


@pytest.mark.parametrize("B,T,Hq", [(130, 1, 1), (300, 5, 2), (70, 40, 1)])
def test_attention_of_many_sequences(sampler, B, T, Hq):
    lens = torch.randint(0, 90, (B,), generator=E.gen(B)).tolist()
    lens[B - 4] = 1500
    run_attn(sampler, attn_inputs(B, B, T, Hq, 1, 64, lens, 32, E.BF16))


@pytest.mark.parametrize("T,G,D,n", [(2, 8, 64, 160), (4, 8, 128, 160), (8, 8, 64, 160), (4, 32, 96, 160), (4, 8, 256, 160), (16, 8, 256, 320)])
@pytest.mark.parametrize("dt", [E.BF16, E.F16])
def test_attention_of_one_value(sampler, T, G, D, n, dt):
    args, scale, c = E.one_value(T, G, D, dt, n=n)
    H.log(f"attention of one value T={T} G={G} D={D} n={n} {dt}")
    lse = torch.empty(1, T, G, device=DEV)
    out = sampler.tree_attention(*(dev(t) for t in args[:7]), scale=scale, lse=lse)
    torch.cuda.synchronize()
    assert (out.cpu().double() == c).all(), out.cpu().double().sub(c).abs().max()
    want = E.attention(args, scale)[1]
    assert ((lse.cpu().double() - want).abs() <= 2**-18 * (1 + want.abs())).all()
