"""GPU: the example that runs beam selection, tree attention and the cache's
calls together: speculated tokens are the greedy ones, in fewer passes; a beam
search's first beam scores at least what greedy decoding does."""
import importlib.util
import os

import pytest
import torch

import gpu_harness as H

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_speculation_and_beams_together(sampler):
    H.log("paged decode example")
    spec = importlib.util.spec_from_file_location("paged_decode", os.path.join(ROOT, "examples", "paged_decode.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    want, got, passes, scores, best = ex.main()
    torch.cuda.synchronize()
    assert got == want
    assert passes == 10  # (40 tokens, four a pass: three guessed right and the one sampled after them)
    model = ex.Model(sampler)
    one, hist = ex.beams(model, [5, 17, 400, 3, 250, 9], 1, 40)
    assert hist[0].tolist() == want
    # the search keeps the best prefixes, and 16 beams hold the greedy one here
    many, _ = ex.beams(model, [5, 17, 400, 3, 250, 9], 16, 40)
    assert torch.isfinite(many).all() and (many[:-1] >= many[1:]).all()
    assert torch.isfinite(scores).all() and (scores[:-1] >= scores[1:]).all()
