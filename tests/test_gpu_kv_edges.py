"""GPU: the beam, tree-attention and cache calls where their inputs are extreme
(the CPU simulation's cases of test_kv_edges.py at larger sizes)."""
import pytest
import torch

import gpu_harness as H
import kv_cases as C
import kv_edges as E
from test_gpu_kv import cpu, dev

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
