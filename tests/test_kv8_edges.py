"""The 8-bit cache's kernels on the CPU simulation where inputs are extreme: garbage in
drafted rows that a tree does not see, with both kernels and every kind of share."""
import math

import pytest
import torch

import kv8_cases as K
import kv_edges as E
from test_kv8_sim import attn_inputs
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
    for kw in ({}, dict(max_len=1000)):
        rc, out, lse = K.sim_attention(sim, q, kn, vn, p, tabs, lens, par, None, **kw)
        assert rc == 0
        check_unseen(out, lse, args)


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
