"""Beam search and tree speculation over a paged key/value cache, with a toy
attention-only model of random weights: what a server around the sampler runs
in a decode step.

    python examples/paged_decode.py

`Model.nodes` runs tokens (a prompt, one new token, a drafted tree) through the
layers with `tree_attention`; `greedy` and `beams` decode token by token
(`beam_select`, `kv_fork`, `kv_append`); `speculate` verifies a drafted tree at
a time (`tree_commit`) and gives the tokens that `greedy` gives.
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import tinygpt_amd as tg  # noqa: E402

DEV = "cuda:0"
I32 = torch.int32


class Model:
    def __init__(self, sampler, layers=2, q_heads=8, kv_heads=2, D=64, vocab=1000, page=16, pages=256, seed=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = lambda *shape: torch.randn(*shape, generator=g, device=DEV)
        self.s, self.L, self.Hq, self.H, self.D, self.V = sampler, layers, q_heads, kv_heads, D, vocab
        width = q_heads * D
        self.embed = r(vocab, width)
        # (a head that prefers one successor of each token, so that 16-bit rounding seldom decides between two)
        self.head = self.embed[torch.randperm(vocab, generator=g, device=DEV)].t().contiguous() * width**-0.5
        self.qkv = [r(width, (q_heads + 2 * kv_heads) * D) * width**-0.5 for _ in range(layers)]
        self.out = [r(width, width) * width**-0.5 for _ in range(layers)]
        self.k = torch.zeros(layers, pages, kv_heads, page, D, dtype=torch.bfloat16, device=DEV)
        self.v = torch.zeros(layers, pages, kv_heads, page // 8, D, 8, dtype=torch.bfloat16, device=DEV)
        self.page, self.pages = page, pages

    def nodes(self, tokens, tables, lens, parents=None):
        """Logits [B, T, V] after each node (a chain without parents) and the nodes' keys and values, every layer's."""
        B, T = tokens.shape
        x = self.embed[tokens.long()]
        k_new = torch.empty(self.L, B, T, self.H, self.D, dtype=self.k.dtype, device=DEV)
        v_new = torch.empty_like(k_new)
        for l in range(self.L):
            y = torch.nn.functional.rms_norm(x, x.shape[-1:]) @ self.qkv[l] * 2
            q, k, v = y.to(self.k.dtype).split([self.Hq * self.D, self.H * self.D, self.H * self.D], -1)
            k_new[l], v_new[l] = k.unflatten(-1, (self.H, self.D)), v.unflatten(-1, (self.H, self.D))
            o = self.s.tree_attention(q.unflatten(-1, (self.Hq, self.D)), k_new[l], v_new[l], self.k[l], self.v[l], tables, lens,
                                      parents=parents)
            x = x + 2 * o.flatten(2).float() @ self.out[l]
        return x @ self.head / 2, k_new, v_new

    def prefill(self, prompt, rows, slots):
        """`rows` sequences of their own pages that hold the prompt's tokens but the last."""
        tables = torch.arange(rows * slots, dtype=I32, device=DEV).view(rows, slots)
        lens = torch.zeros(rows, dtype=I32, device=DEV)
        chain = torch.tensor(prompt[:-1], dtype=I32, device=DEV).expand(rows, -1).contiguous()
        _, k_new, v_new = self.nodes(chain, tables, lens)
        return tables, self.s.kv_append(k_new, v_new, self.k, self.v, tables, lens)


def beams(model, prompt, W, steps):
    """The W best continuations of `steps` tokens, best first: (scores [W], tokens [W, steps])."""
    s, B = model.s, W
    slots = (len(prompt) + steps) // model.page + 2
    tables, lens = model.prefill(prompt, B, slots)
    scores = torch.full((B,), -torch.inf, device=DEV)
    scores[0] = 0.0  # (the beams start alike: one of them is alive)
    token = torch.full((B,), prompt[-1], dtype=I32, device=DEV)
    hist, hist_len = torch.full((B, steps), -1, dtype=I32, device=DEV), torch.zeros(B, dtype=I32, device=DEV)
    for _ in range(steps):
        logits, k_new, v_new = model.nodes(token[:, None], tables, lens)
        lens = s.kv_append(k_new, v_new, model.k, model.v, tables, lens)
        o = s.beam_select(logits[:, 0], scores, W, W, hist=hist, hist_len=hist_len)
        tables, lens = s.kv_fork(model.k, model.v, tables, lens, o["parents"], room=1)
        scores, token, hist, hist_len = o["scores"], o["tokens"], o["hist"], o["hist_len"]
    return scores, hist


def greedy(model, prompt, steps):
    return beams(model, prompt, 1, steps)[1][0].tolist()


def speculate(model, prompt, steps, draft, T=8):
    """Greedy decoding by verified trees: draft(tokens so far, T) gives a tree's tokens and parents (node 0: the
    last token).  Returns the tokens and the number of forward passes."""
    s = model.s
    tables, lens = model.prefill(prompt, 1, (len(prompt) + steps + T) // model.page + 2)
    params = tg.params_to_device(tg.make_params(T, temperature=0.0), DEV)
    u = torch.zeros(T, device=DEV)
    done, passes = list(prompt), 0
    while len(done) < len(prompt) + steps:
        tokens, parents = (torch.tensor([x], dtype=I32, device=DEV) for x in draft(done, T))
        logits, k_new, v_new = model.nodes(tokens, tables, lens, parents)
        sampled = s.sample(logits[0], params, u)[None]
        o = s.tree_commit(k_new, v_new, model.k, model.v, tables, lens, parents, tokens, sampled)
        lens = o["lens"]
        done += [t for t in o["tokens"][0].tolist() if t >= 0]
        passes += 1
    return done[len(prompt):len(prompt) + steps], passes


def main():
    sampler = tg.Sampler(device=0, max_batch=64, max_vocab=32000, max_hist=64)
    model = Model(sampler)
    prompt, steps, T = [5, 17, 400, 3, 250, 9], 40, 8
    want = greedy(model, prompt, steps)

    def draft(done, T):
        """A path that guesses three tokens right, and wrong siblings."""
        at = len(done) - len(prompt)
        right = (want + [0] * T)[at:at + 3]
        tokens = [done[-1], *right, 1, 2, 3, 4]
        return tokens[:T], [-1, 0, 1, 2, 0, 1, 2, 3][:T]

    got, passes = speculate(model, prompt, steps, draft, T)
    scores, best = beams(model, prompt, 4, steps)
    sampler.close()
    print(f"greedy      {want[:12]} ...")
    print(f"speculated  {got[:12]} ... in {passes} passes, equal: {got == want}")
    print(f"beams       {[round(x, 3) for x in scores.tolist()]}, best {best[0].tolist()[:12]} ...")
    return want, got, passes, scores, best


if __name__ == "__main__":
    main()
