"""The 8-bit cache's and the rotation's calls check every tensor before anything
is launched (CPU only: no GPU is needed to reach these errors)."""
import pytest
import torch

import kv8_cases as K
from test_cache_inputs import Ops

BF16, I32 = torch.bfloat16, torch.int32


def attn_args(B=2, T=3, Hq=4, H=2, D=64, page=16):
    k, v, s = K.as_tensors([x[0] for x in K.pools(torch.Generator().manual_seed(0), 1, 5, H, page, D, BF16)])
    return dict(q=torch.zeros(B, T, Hq, D, dtype=BF16), k_new=torch.zeros(B, T, H, D, dtype=BF16),
                v_new=torch.zeros(B, T, H, D, dtype=BF16), k=k, v=v, tables=torch.zeros(B, 2, dtype=I32), scales=s,
                lens=torch.zeros(B, dtype=I32), parents=torch.zeros(B, T, dtype=I32), out=torch.zeros(B, T, Hq, D, dtype=BF16))


@pytest.mark.parametrize("change,error,match", [
    ({}, ValueError, "device"),
    (dict(scales=None), TypeError, "needs its scales"),
    (dict(scales=3), TypeError, "scales must be a tensor"),
    (dict(scales=torch.zeros(5, 2, 1, 2)), TypeError, "float8_e8m0fnu"),
    (dict(k=torch.zeros(5, 2, 16, 64, dtype=BF16)), TypeError, "float8_e4m3fn"),
    (dict(v=torch.zeros(5, 2, 2, 64, 8, dtype=torch.float8_e4m3fn)), ValueError, "v must be"),
    (dict(v=torch.zeros(5, 2, 16, 64, dtype=torch.float8_e4m3fn)), ValueError, "page / 16"),
    (dict(k=torch.zeros(5, 16, 2, 64, dtype=torch.float8_e4m3fn).transpose(1, 2)), ValueError, "contiguous"),
])
def test_attention(change, error, match):
    with pytest.raises(error, match=match):
        Ops().tree_attention(stream=0, **(attn_args() | change))


def test_writes_and_forks():
    s = Ops()
    k, v, sc = K.as_tensors(K.pools(torch.Generator().manual_seed(0), 2, 5, 1, 16, 16, BF16))
    rows = torch.zeros(2, 3, 4, 1, 16, dtype=BF16)
    tabs, lens = torch.zeros(3, 2, dtype=I32), torch.zeros(3, dtype=I32)
    out = torch.zeros(3, dtype=I32)
    with pytest.raises(ValueError, match="device"):
        s.kv_append(rows, rows, k, v, tabs, lens, lens_out=out, stream=0, scales=sc)
    with pytest.raises(TypeError, match="float8"):
        s.kv_fork(k, v, tabs, lens, lens, tables_out=tabs.clone(), lens_out=out, stream=0, scales=sc.float())
    with pytest.raises(ValueError, match="differ in layers"):
        s.kv_append(rows, rows, k, v[:1], tabs, lens, lens_out=out, stream=0, scales=sc)
    with pytest.raises(ValueError, match="k must be"):
        s.kv_fork(k[0], v[0], tabs, lens, lens, tables_out=tabs.clone(), lens_out=out, stream=0, scales=sc[0])
    o = dict(n_acc=out, tokens=torch.zeros(3, 4, dtype=I32), path=torch.zeros(3, 4, dtype=I32), lens=out.clone())
    par = torch.zeros(3, 4, dtype=I32)
    with pytest.raises(ValueError, match="device"):
        s.tree_commit(rows, rows, k, v, tabs, lens, par, par, par, out=o, stream=0, scales=sc)


def test_rotation():
    s = Ops()
    q, k = torch.zeros(2, 3, 4, 32, dtype=BF16), torch.zeros(2, 3, 1, 32, dtype=BF16)
    lens, f = torch.zeros(2, dtype=I32), torch.ones(16)
    with pytest.raises(ValueError, match="device"):
        s.rotate(q, k, lens, f, stream=0)
    with pytest.raises(ValueError, match="rotary"):
        s.rotate(q, k, lens, None, stream=0)
    with pytest.raises(ValueError, match="rotary"):
        s.rotate(q, k, lens, f[None], stream=0)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        s.rotate(q.float(), k, lens, f, stream=0)
    with pytest.raises(ValueError, match="q must be"):
        s.rotate(q[0], k, lens, f, stream=0)
    with pytest.raises(TypeError, match="k_new must be a tensor"):
        s.rotate(q, 5, lens, f, stream=0, k_out=k)
