"""Beam selection, tree attention, position rotation and the paged key/value cache on a sampler's
handle (torch tensors in, torch out; mixed into `Sampler`).

A cache is a pair of pools, keys [layers, pages, kv_heads, page, D] and values
[layers, pages, kv_heads, page / 8, D, 8] (bfloat16 or float16; one layer's
calls take them without the first dimension).  In 8 bits it is three: keys of
the same shape and values [layers, pages, kv_heads, page / 16, D, 16] in
float8_e4m3fn, and scales [layers, pages, kv_heads, page / 16, 2] in
float8_e8m0fnu, one of the keys and one of the values of each block of 16 tokens
of a head (page a multiple of 16, D of 16, at most 256); every call takes it
with `scales`, and bfloat16 or float16 rows.  A written block has the smallest
power of two as its scale with which its largest magnitude stays within 448, and
none below the one that it has while it holds earlier tokens of the sequence.
Token t of a sequence is slot t % page of page tables[sequence, t // page].  Every call checks its tensors
(type, layout, size, device) before anything is launched, runs on torch's
current stream or the one given, and neither allocates device memory (where
outputs are given) nor synchronises.
"""
from __future__ import annotations

import importlib.util
import os

from . import _lib

_torch_module = None
_calls_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch

        _torch_module = torch
    return _torch_module


def _calls():
    """The native checks and calls (csrc/tgs_cache_py.cpp), on the library that `_lib` loads."""
    global _calls_module
    if _calls_module is None:
        _torch()
        path = os.path.join(_lib.HERE, "_cache_calls.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
        spec = importlib.util.spec_from_file_location("tinygpt_amd._cache_calls", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _lib.load()
        module.bind(_lib.LIB_PATH)
        _calls_module = module
    return _calls_module


class CacheOps:
    """Methods of `Sampler` (self._L, self._h, self.device, self._check)."""

    def _call(self, name, stream, *args):
        """One native call on this handle; raises what its checks or its status say."""
        if stream is None:
            torch = _torch()
            raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
            stream = raw(self.device) if raw is not None else torch.cuda.current_stream(self.device).cuda_stream
        h = self._h
        rc = getattr(_calls_module or _calls(), name)(h.value if h is not None else 0, self.device, stream, *args)
        if rc:
            self._check(rc, "tgs_" + name)

    def _new(self, dtype, *shape):
        return _torch().empty(shape, dtype=dtype, device=f"cuda:{self.device}")

    def beam_select(self, logits, scores, W, n_out, hist=None, hist_len=None, out=None, vocab=None, stream=None):
        """The n_out best continuations of each request's W beams: logits
        [G * W, >= V] (float32 or bfloat16), scores float32 [G * W] (-inf: the
        beam has ended), optional histories int32 [G * W, H] with hist_len
        [G * W].  Returns `out`, a dict of scores, parents (rows of logits)
        and tokens [G * n_out], and with histories hist [G * n_out, H] and
        hist_len, best first, equal ones by the lower beam, then the lower id;
        past the last candidate -inf, -1, -1."""
        torch = _torch()
        i32 = torch.int32
        o = {} if out is None else out
        if len(o) < 5:  # (a caller that keeps its outputs gives them all)
            n = logits.shape[0] // max(W, 1) * max(n_out, 0)
            shapes = {"scores": (torch.float32, n), "parents": (i32, n), "tokens": (i32, n)}
            if hist is not None:
                shapes |= {"hist": (i32, n, *hist.shape[1:]), "hist_len": (i32, n)}
            for name, shape in shapes.items():
                if o.get(name) is None:
                    o[name] = self._new(*shape)
        self._call("beam_select", stream, logits, scores, W, n_out, -1 if vocab is None else vocab, hist, hist_len,
                   o["scores"], o["parents"], o["tokens"], o.get("hist"), o.get("hist_len"))
        return o

    def tree_attention(self, q, k_new, v_new, k, v, tables, lens, parents=None, max_len=None, scale=None, out=None,
                       lse=None, stream=None, scales=None):
        """Attention of T drafted nodes per sequence over the sequence's
        cached tokens, each node's ancestors and itself: q [B, T, q_heads, D],
        k_new and v_new [B, T, kv_heads, D] (any strides, D contiguous), k and
        v one layer's pools, tables int32 [B, slots], lens int32 [B], parents
        int32 [B, T] (an earlier node, -1: a root; None: a chain).  max_len:
        a bound of lens known on the host (sizes the launch), scale:
        1 / sqrt(D) when None.  Returns out [B, T, q_heads, D] (NaN for a sequence
        of the length -1 or with a page outside the pool); lse float32
        [B, T, q_heads], when given, gets the natural logsumexp of the scaled
        scores.  scales: of the layer, when the cache holds 8 bits (q and the new
        rows are of the type that the cache was written from)."""
        if out is None:
            out = self._new(q.dtype, *q.shape)
        self._call("tree_attention", stream, q, k_new, v_new, k, v, tables, lens, parents, -1 if max_len is None else max_len,
                   scale, out, lse, scales)
        return out

    def kv_append(self, k_new, v_new, k, v, tables, lens, counts=None, lens_out=None, stream=None, scales=None, rotary=None,
                  pairs=False):
        """Writes the first counts[b] (all, when None) of the T new rows of
        each sequence and layer, k_new and v_new [layers, B, T, kv_heads, D],
        behind its lens[b] tokens.  Returns lens_out int32 [B]: the new
        lengths, -1 where the rows did not fit (nothing is written there).
        scales: of an 8-bit cache.  rotary, float32 [R / 2]: pair j of a key's first
        R dimensions (a multiple of 16, at most 256) turns by position * rotary[j]
        on the way: dimensions j and j + R / 2, or with `pairs` the neighbours 2 j
        and 2 j + 1."""
        if lens_out is None:
            lens_out = self._new(_torch().int32, *tables.shape[:1])
        self._call("kv_append", stream, k_new, v_new, k, v, tables, lens, counts, lens_out, scales, rotary, pairs)
        return lens_out

    def rotate(self, q, k_new, lens, rotary, pairs=False, parents=None, q_out=None, k_out=None, stream=None):
        """Turns the queries and keys of T new nodes per sequence by their
        positions (lens[b], 0 where it is below, and the node's depth in its
        tree) as `kv_append` turns keys: q [B, T, q_heads, D] and k_new
        [B, T, kv_heads, D] (None: queries alone) of any strides, D contiguous,
        lens int32 [B], parents int32 [B, T] as in `tree_attention` (T at most
        64), or None: a chain of any length.  Returns (q_out, k_out); q_out=q
        and k_out=k_new turn them in place."""
        torch = _torch()
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if k_out is None and k_new is not None:
            k_out = torch.empty_like(k_new, memory_format=torch.contiguous_format)
        self._call("rotate", stream, q, k_new, lens, rotary, pairs, parents, q_out, k_out)
        return q_out, k_out

    def tree_commit(self, k_new, v_new, k, v, tables, lens, parents, draft, sampled, out=None, stream=None, scales=None):
        """Accepts each sequence's drafted tree as far as it agrees with the
        ids sampled after its nodes, and writes the path's rows to the cache:
        parents, draft, sampled int32 [B, T] (node 0 is the root), k_new and
        v_new [layers, B, T, kv_heads, D].  Returns `out`, a dict of n_acc
        [B], tokens [B, T] (accepted, then the one sampled at the last),
        path [B, T] and lens [B] (-1: the rows did not fit).  scales: of an
        8-bit cache."""
        o = {} if out is None else out
        for name in ("n_acc", "tokens", "path", "lens"):
            if o.get(name) is None:
                o[name] = self._new(_torch().int32, *(parents.shape if name in ("tokens", "path") else parents.shape[:1]))
        self._call("tree_commit", stream, k_new, v_new, k, v, tables, lens, parents, draft, sampled, o["n_acc"], o["tokens"],
                   o["path"], o["lens"], scales)
        return o

    def kv_fork(self, k, v, tables, lens, parents, room=1, tables_out=None, lens_out=None, stream=None, scales=None):
        """Reorders a cache's rows after a beam step: row r goes on from row
        parents[r].  Full pages are shared; the page that the next `room`
        tokens go to has one writer, the other rows get free pages of the pool
        (those that no row names any more) and copies.  Returns (tables_out
        [B, slots], lens_out [B]): -1 past the slots in use; length 0 for a
        parent outside the rows, -1 for a row that found no page, that names
        none where it has tokens, or whose parent's length was -1.  scales: of
        an 8-bit cache."""
        if tables_out is None:
            tables_out = self._new(_torch().int32, *tables.shape)
        if lens_out is None:
            lens_out = self._new(_torch().int32, *tables.shape[:1])
        self._call("kv_fork", stream, k, v, tables, lens, parents, room, tables_out, lens_out, scales)
        return tables_out, lens_out
