"""The 8-bit cache's kernels on the CPU simulation where inputs are extreme: garbage in
drafted rows that a tree does not see, with both kernels and every kind of share."""
import math

import pytest
import torch

import kv8_cases as K
import kv_edges as E
from test_kv8_sim import attn_inputs, run_attn
from test_kv_sim import check_attn, sim  # noqa: F401  (sim: a fixture)

BF16, F16 = torch.bfloat16, torch.float16

# (T, q heads, kv heads, D, lens, page, type)
SHAPES = [(2, 1, 1, 64, [5, 0], 16, BF16), (8, 4, 2, 128, [70, 33], 16, F16), (16, 2, 1, 96, [40], 32, BF16),
          (20, 2, 1, 64, [200, 9], 16, BF16), (64, 1, 1, 128, [150], 32, BF16), (33, 8, 1, 64, [20], 16, F16),
          (6, 2, 1, 256, [133], 16, F16), (20, 2, 1, 256, [40], 16, BF16)]


def unseen_garbage(T, Hq, Hkv, D, lens, page, dt, chain=False):
    """The 16-bit case's drafted rows over an 8-bit cache."""
    q, kn, vn, _, _, _, _, par = E.unseen_garbage(T, Hq, Hkv, D, [0] * len(lens), page, dt, chain=chain)
    _, _, _, p, tabs, lens, _ = attn_inputs(T + D, len(lens), T, Hq, Hkv, D, lens, page, dt)
    return q, kn, vn, p, tabs, lens, par


def check_unseen(out, lse, args):
    q, kn, vn, p, tabs, lens, par = args
    E.check_unseen(out, lse, (q, kn, vn, *K.decoded(p), tabs, lens, par), check_attn)


@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_unseen_garbage(sim, shape, chain):  # noqa: F811
    args = unseen_garbage(*shape, chain=chain)
    q, kn, vn, p, tabs, lens, par = args
    for more in (0, 6000):
        wide = widened(args, more)[4]
        rc, out, lse = K.sim_attention(sim, q, kn, vn, p, wide, lens, par, None)
        assert rc == 0
        check_unseen(out, lse, args)


def widened(args, tokens):
    """The same sequences with slots for `tokens` tokens, the added ones without a page: work is shared by that bound."""
    q, kn, vn, p, tabs, lens, par = args
    page = p[0].shape[2]
    more = torch.full((tabs.shape[0], max(0, -(-tokens // page) - tabs.shape[1])), -1, dtype=tabs.dtype)
    return q, kn, vn, p, torch.cat([tabs, more], 1), lens, par


@pytest.mark.parametrize("T,Hq,Hkv,D,lens,page,dt,cu", [
    (1, 4, 2, 64, [300, 0, 77], 16, F16, 3), (5, 8, 2, 128, [200, 130], 64, BF16, 2), (3, 2, 1, 96, [500, 1], 32, BF16, 4),
    (20, 1, 1, 64, [333], 16, F16, 2), (2, 8, 1, 256, [260, 90], 64, BF16, 5)])
def test_shares_of_few_rows(sim, T, Hq, Hkv, D, lens, page, dt, cu):  # noqa: F811
    """Workers that share (sequence, key head)s, and the unshared form, of the same rows."""
    args = attn_inputs(T + D, len(lens), T, Hq, Hkv, D, lens, page, dt)
    for more in (0, 6000):
        run_attn(sim, widened(args, more), num_cu=cu)


def test_finite_scores_far_apart(sim):  # noqa: F811
    """Scores of +-300 between a cache's blocks: the later ones take the whole weight or none."""
    for T in (1, 40):
        q, kn, vn, p, tabs, lens, par = attn_inputs(T, 1, T, 1, 1, 64, [100], 16, BF16)
        q.fill_(1.0)
        kn.fill_(-300.0 / 8)
        for i in range(7):
            pg = int(tabs[0, i])
            p[0][pg, 0, :max(min(100 - 16 * i, 16), 0)] = 0x38 if i % 2 else 0xB8  # 1, -1
            p[2][pg, 0, 0, 0] = 127 + (5 if i == 3 else 2)
        rc, out, lse = K.sim_attention(sim, q, kn, vn, p, tabs, lens, par, None)
        v = K.decoded(p)[1][int(tabs[0, 3]), 0].transpose(-1, -2).reshape(16, 64)
        assert rc == 0 and math.isclose(float(lse[0, 0, 0]), 32 * 8 + math.log(16), rel_tol=2**-16)
        # (half a step of each weight, of their sum and of the result)
        assert ((out[0, :, 0].double() - v.mean(0)).abs() <= 2.0**-7 * v.abs().max()).all()
