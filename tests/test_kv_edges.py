"""The beam, tree-attention and cache kernels on the CPU simulation where their
inputs are extreme: finite masks, garbage in rows that a tree does not see,
failed lengths, entries outside the pool."""
import math

import pytest
import torch

import kv_cases as C
import kv_edges as E
from test_kv_sim import BF16, F16, F32, attn_inputs, check_attn, sim, write_inputs  # noqa: F401  (sim: a fixture)


# ------------------------------------------------------------------ beams

@pytest.mark.parametrize("case", E.MASKS, ids=E.mask_name)
def test_beam_finite_masks(sim, case):  # noqa: F811
    x, scores = E.masked_logits(*case, V=2100)
    rc, got = C.sim_beam(sim, x, scores, 3, 5)
    assert rc == 0
    E.check_beam(got, C.beam(x, scores, 3, 5), x)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_beam_large_logits(sim, dt):  # noqa: F811
    x, scores = E.large_logits(dt, V=2100)
    rc, got = C.sim_beam(sim, x, scores, 2, 6)
    assert rc == 0
    E.check_beam(got, C.beam(x, scores, 2, 6), x)


# ------------------------------------------------------------------ forks

def run_fork(sim, case, room):  # noqa: F811
    """The simulation's tables and lengths; they and the pools are the plain form's."""
    rc, k1, v1, t1, l1 = C.sim_fork(sim, *case, room)
    k2, v2, t2, l2 = E.fork(*case, room)
    assert rc == 0 and torch.equal(t1, t2) and torch.equal(l1, l2) and torch.equal(k1, k2) and torch.equal(v1, v2)
    return t1.tolist(), l1.tolist()


@pytest.mark.parametrize("name", list(E.SHORT_POOLS))
@pytest.mark.parametrize("layers", [1, 4])
def test_fork_short_pools(sim, name, layers):  # noqa: F811
    """Rows that need no page, or no more than are left, go on when the pool has run out for others."""
    (k, v, *rest), room, tabs, lens = E.SHORT_POOLS[name]
    case = (k.repeat(layers, 1, 1, 1, 1), v.repeat(layers, 1, 1, 1, 1, 1), *rest)
    assert run_fork(sim, case, room) == (tabs, lens)


def test_fork_short_pool_of_many_rows(sim):  # noqa: F811
    case = E.many_short_rows()
    _, lens = run_fork(sim, case[:5], case[5])
    assert -1 in lens[:1024] and max(lens[lens.index(-1):1024]) > 0


@pytest.mark.parametrize("name", list(E.BAD_ENTRIES))
@pytest.mark.parametrize("spare", [0, 20000])
def test_fork_entries_outside_the_pool(sim, name, spare):  # noqa: F811
    """Reported by the length -1 (spare: pages of no row, so many that the plan's lists lie in the workspace)."""
    (k, v, t, n, p), room, tabs, lens = E.BAD_ENTRIES[name]
    if spare:
        k = torch.cat([k, k.new_zeros(1, spare, *k.shape[2:])], 1)
        v = torch.cat([v, v.new_zeros(1, spare, *v.shape[2:])], 1)
        t = torch.where(t >= 8, t + spare, t)
        tabs = [[x + spare if x >= 8 else x for x in row] for row in tabs]
    case = (k, v, t, n, p)
    assert run_fork(sim, case, room) == (tabs, lens)


@pytest.mark.parametrize("name", list(E.FAILED_LENGTHS))
def test_fork_failed_lengths(sim, name):  # noqa: F811
    """A row that failed before does not become an empty one."""
    case, room, tabs, lens = E.FAILED_LENGTHS[name]
    assert run_fork(sim, case, room) == (tabs, lens)


# ------------------------------------------------------------------ attention

def run_attn(sim, args, **kw):  # noqa: F811
    q, kn, vn, k, v, tabs, lens, par = args
    rc, out, lse = C.sim_attention(sim, *args, **kw)
    assert rc == 0
    want, want_lse = E.attention(args)
    finite = [x.double()[torch.isfinite(x.double())].abs().max() for x in (vn, v)]
    check_attn(out, lse, want, want_lse, float(max(finite)), q.dtype)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_attention_of_failed_sequences(sim, T):  # noqa: F811
    """The length -1, by which an append, a commit or a fork reports a failure, gives NaN and no context of length 0."""
    run_attn(sim, E.failed_attention(T))
    run_attn(sim, E.failed_attention(T), num_cu=8, max_len=4000)


@pytest.mark.parametrize("shape", E.UNSEEN, ids=str)
@pytest.mark.parametrize("chain", [False, True])
def test_attention_garbage_in_nodes_that_are_not_seen(sim, shape, chain):  # noqa: F811
    args = E.unseen_garbage(*shape, chain=chain)
    rc, out, lse = C.sim_attention(sim, *args)
    assert rc == 0
    E.check_unseen(out, lse, args, check_attn)


@pytest.mark.parametrize("shape", [(6, 2, 1, 64, [300, 7], 16, BF16), (40, 1, 1, 64, [600], 16, F16)], ids=str)
def test_attention_garbage_in_shares(sim, shape):  # noqa: F811
    """The same where the drafted nodes' part is joined with others."""
    args = E.unseen_garbage(*shape)
    rc, out, lse = C.sim_attention(sim, *args, num_cu=5)
    assert rc == 0
    E.check_unseen(out, lse, args, check_attn)


@pytest.mark.parametrize("T,D,n", [(1, 64, 600), (3, 256, 330), (40, 64, 700), (36, 128, 200)])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_attention_faint_tail(sim, T, D, n, dt):  # noqa: F811
    """Weights far below the largest: fp16 holds them as well as half a step."""
    args, scale = E.faint_tail(D, dt, n, T=T)
    rc, out, lse = C.sim_attention(sim, *args, scale=scale)
    assert rc == 0
    E.check_faint_tail(out, lse, args, scale)


# ------------------------------------------------------------------ appends

def test_append_of_few_of_many_rows(sim):  # noqa: F811
    """Rows of the largest shape, of which the counts take a few: the launch is sized by what the tables hold."""
    T = 2**31 - 1
    kn, vn, k, v, tabs = write_inputs(5, 1, 2, 1, 1, 8, 8, 3, BF16)
    lens, counts = torch.tensor([3, 0], dtype=torch.int32), torch.tensor([21, 0], dtype=torch.int32)
    rc, k1, v1, l1 = C.sim_append(sim, kn.expand(1, 2, T, 1, 8), vn.expand(1, 2, T, 1, 8), k, v, tabs, lens, counts)
    k2, v2, l2 = C.append(*(x.expand(1, 2, 21, 1, 8) for x in (kn, vn)), k, v, tabs, lens, counts)
    assert rc == 0 and torch.equal(k1, k2) and torch.equal(v1, v2) and torch.equal(l1, l2)


# ------------------------------------------------------------------ every token's value, many sequences

@pytest.mark.parametrize("T,G,D,lens", [(4, 2, 64, [300, 77]), (11, 3, 64, [290, 64])])
def test_attention_takes_each_tokens_value(sim, T, G, D, lens):  # noqa: F811
    k, v, tabs, n, keys, values, rows = E.named_tokens(2, T, G, 1, D, lens, 16, F16)
    for first, step in ((0, 9), (5, 31)):
        q, at = E.queries(keys, n, T, G, first, step)
        rc, out, _ = C.sim_attention(sim, q, rows, rows, k, v, tabs, n, None, 2.0, num_cu=3)
        assert rc == 0
        E.check_named(out, at, values)


def test_attention_of_many_sequences(sim):  # noqa: F811
    """More sequences than a wave has lanes, in shares that start anywhere among them."""
    lens = torch.randint(0, 60, (70,), generator=E.gen(2)).tolist()
    lens[66] = 290
    run_attn(sim, attn_inputs(70, 70, 1, 1, 1, 64, lens, 32, BF16), num_cu=9)


@pytest.mark.parametrize("T,G,D,n", [(2, 8, 64, 160), (4, 8, 128, 160), (8, 8, 64, 160), (4, 32, 96, 160), (16, 4, 64, 320)])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_attention_of_one_value(sim, T, G, D, n, dt):  # noqa: F811
    """Results are sums over the weights that the product has, so that their rounding does not show in equal values (a
    result before its rounding is off by a few steps of 32 bits, and the value is a number of the type)."""
    args, scale, c = E.one_value(T, G, D, dt, n=n)
    rc, out, lse = C.sim_attention(sim, *args, scale=scale)
    assert rc == 0
    assert (out.double() == c).all(), out.double().sub(c).abs().max()
    want = E.attention(args, scale)[1]
    assert ((lse.double() - want).abs() <= 2**-18 * (1 + want.abs())).all()
