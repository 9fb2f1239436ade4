"""Extreme inputs of the beam, tree-attention and cache tests, and what is
expected of them (shared by the CPU simulation's tests and the GPU's)."""
from __future__ import annotations

import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ beams

# (type, value of a masked id: a large finite number, as grammars and padded vocabularies write it)
MASKS = [(dt, v) for dt in (F32, BF16)
         for v in (-1e4, -1e9, -1e10, -1e12, -1e30, -1e38, -2.4e38, torch.finfo(dt).min)]


def mask_name(case):
    return f"{str(case[0])[6:]}{case[1]:.3g}"


def masked_logits(dt, value, V):
    """Requests of three beams: a few ids allowed in each row; all but the last ids masked in one, all ids in another;
    a padded vocabulary; a whole request at the mask's value, one with a single larger id in it."""
    g = gen(abs(int(value)) % 1000 + V)
    x = torch.randn(4 * 3, V, generator=g) * 3
    mask = torch.ones(12, V, dtype=torch.bool)
    for r in range(3):
        mask[r, torch.randperm(V, generator=g)[:40]] = False
    mask[3, -5:] = False       # one live thread in a chunk, and one chunk alone of a row
    mask[5, :7] = False        # (row 4: masked whole, beside rows that are not)
    mask[6:9, : V - V // 4] = False
    x = torch.where(mask, torch.tensor(value), x).to(dt)
    x[11, V // 2] = x[11, 0].double() * (1 - 2.0**-6)
    scores = -3 * torch.rand(12, generator=g).cumsum(0)
    return x, scores


def large_logits(dt, V):
    """Two beams each: rows around one large value, a few steps of the type apart, and rows with one huge id."""
    g = gen(V)
    rows = []
    for at in (1e6, 2.0**22 - 3, 2.0**22 + 3, 1e7, 1e9, 1e10, 1e20, 3e38):
        for sign in (-1, 1):
            step = at * torch.finfo(dt).eps
            rows.append(sign * at + torch.randint(-4, 4, (V,), generator=g).double() * max(step, 1.0))
            one = torch.randn(V, generator=g).double()
            one[int(torch.randint(0, V, (1,), generator=g))] = sign * at
            rows.append(one)
    x = torch.stack(rows).to(dt)
    assert torch.isfinite(x).all()
    return x, -3 * torch.rand(len(rows), generator=g)


def check_beam(got, want, x):
    # a total's one 32-bit rounding, the logsumexp's sum of 32-bit exponentials (relative 2^-21 at most), and the
    # 64-bit roundings of a logsumexp as large as the row's logits and of the difference from it, on both sides
    w = want["scores"]
    top = x.double().amax(1)[want["parents"].long().clamp(min=0)].abs()
    assert torch.equal(got["parents"], want["parents"]) and torch.equal(got["tokens"], want["tokens"])
    fin = torch.isfinite(w)
    assert torch.equal(fin, torch.isfinite(got["scores"]))
    err = (got["scores"].double() - w).abs()
    assert (err <= w.abs() * 2**-24 + 2**-21 + 4 * top * 2**-53)[fin].all(), float(err[fin].max())
