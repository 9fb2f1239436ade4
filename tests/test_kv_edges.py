"""The beam, tree-attention and cache kernels on the CPU simulation where their
inputs are extreme: finite masks, garbage in rows that a tree does not see,
failed lengths, entries outside the pool."""
import math

import pytest
import torch

import kv_cases as C
import kv_edges as E
from test_kv_sim import BF16, F16, F32, beam_inputs, gen, sim  # noqa: F401  (sim: a fixture)


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
