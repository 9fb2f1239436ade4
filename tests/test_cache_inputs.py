"""The cache calls check every tensor before anything is launched (CPU only:
no GPU is needed to reach these errors)."""
import pytest
import torch

import kv_cases as C
from tinygpt_amd.cache import CacheOps

BF16, I32 = torch.bfloat16, torch.int32


class Ops(CacheOps):
    """The methods without a handle: a call that passes the checks would be refused by the library."""

    _h, device = None, 0

    def _check(self, rc, what):
        raise AssertionError(f"{what} was called")


def attn_args(B=2, T=3, Hq=4, H=2, D=64, page=16):
    k, v = C.pools(torch.Generator().manual_seed(0), 1, 5, H, page, D, BF16)
    return dict(q=torch.zeros(B, T, Hq, D, dtype=BF16), k_new=torch.zeros(B, T, H, D, dtype=BF16),
                v_new=torch.zeros(B, T, H, D, dtype=BF16), k=k[0], v=v[0], tables=torch.zeros(B, 2, dtype=I32),
                lens=torch.zeros(B, dtype=I32), parents=torch.zeros(B, T, dtype=I32), out=torch.zeros(B, T, Hq, D, dtype=BF16))


@pytest.mark.parametrize("change,error,match", [
    ({}, ValueError, "device"),
    (dict(q=None), ValueError, "q must be a tensor"),
    (dict(q=3), TypeError, "q must be a tensor"),
    (dict(k=torch.zeros(5, 2, 16, 64)), TypeError, "bfloat16 or float16"),
    (dict(v=torch.zeros(5, 2, 2, 64, 4, dtype=BF16)), ValueError, "v must be"),
    (dict(v=torch.zeros(5, 2, 16, 64, dtype=BF16)), ValueError, "k must be"),
    (dict(k=torch.zeros(5, 16, 2, 64, dtype=BF16).transpose(1, 2)), ValueError, "contiguous"),
])
def test_attention(change, error, match):
    a = attn_args() | change
    with pytest.raises(error, match=match):
        Ops().tree_attention(stream=0, **a)


def test_numbers_and_counts():
    s = Ops()
    x, sc = torch.zeros(4, 50), torch.zeros(4)
    o = {n: torch.zeros(4, dtype=I32) for n in ("parents", "tokens", "hist", "hist_len")} | {"scores": torch.zeros(4)}
    with pytest.raises(ValueError, match="device"):
        s.beam_select(x, sc, 2, 2, out=dict(o), stream=0)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        s.beam_select(x.half(), sc, 2, 2, out=dict(o), stream=0)
    with pytest.raises(ValueError, match="unit stride"):
        s.beam_select(x.t(), sc, 2, 2, out=dict(o), stream=0)
    with pytest.raises(ValueError, match="32 bits"):
        s.beam_select(x, sc, 2, 1 << 40, out=dict(o), stream=0)
    with pytest.raises(TypeError):
        s.beam_select(x, sc, 2.5, 2, out=dict(o), stream=0)


def test_cache_calls():
    s = Ops()
    k, v = C.pools(torch.Generator().manual_seed(0), 2, 5, 1, 8, 16, BF16)
    rows = torch.zeros(2, 3, 4, 1, 16, dtype=BF16)
    tabs, lens = torch.zeros(3, 2, dtype=I32), torch.zeros(3, dtype=I32)
    out = torch.zeros(3, dtype=I32)
    with pytest.raises(ValueError, match="device"):
        s.kv_append(rows, rows, k, v, tabs, lens, lens_out=out, stream=0)
    with pytest.raises(ValueError, match="differ in layers"):
        s.kv_append(rows, rows, k, v[:1], tabs, lens, lens_out=out, stream=0)
    with pytest.raises(ValueError, match="k must be"):
        s.kv_fork(k[0], v[0], tabs, lens, lens, tables_out=tabs.clone(), lens_out=out, stream=0)
    o = dict(n_acc=out, tokens=torch.zeros(3, 4, dtype=I32), path=torch.zeros(3, 4, dtype=I32), lens=out.clone())
    par = torch.zeros(3, 4, dtype=I32)
    with pytest.raises(ValueError, match="device"):
        s.tree_commit(rows, rows, k, v, tabs, lens, par, par, par, out=o, stream=0)
