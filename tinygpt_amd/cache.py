"""Beam selection, tree attention and the paged key/value cache on a sampler's
handle (torch tensors in, torch out; mixed into `Sampler`).

A cache is a pair of pools, keys [layers, pages, kv_heads, page, D] and values
[layers, pages, kv_heads, page / 8, D, 8] (bfloat16 or float16; one layer's
calls take them without the first dimension).  Token t of a sequence is slot
t % page of page tables[sequence, t // page].  Every call checks its tensors
(type, layout, size, device) before anything is launched, runs on torch's
current stream or the one given, and neither allocates device memory (where
outputs are given) nor synchronises.
"""
from __future__ import annotations

import struct

from ._lib import TGS_BF16, TGS_F16

_CACHE = struct.Struct("PPqqqqiiiiii")   # tgs_kv_cache
_ROWS = struct.Struct("PPqqqqqqqq")      # tgs_kv_rows
_SEQS = struct.Struct("PPii")            # tgs_kv_seqs
_ATTN = struct.Struct("PqqqPPPiiif")     # tgs_attn

_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch

        _torch_module = torch
    return _torch_module


def _bad(fn, msg):
    raise ValueError(f"{fn}: {msg}")


def _ints(fn, torch, dev, name, t, *shape):
    """t is a contiguous int32 tensor of that shape on device index dev."""
    if t is None or t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        _bad(fn, f"{name} must be a contiguous int32 tensor of shape {tuple(shape)}")
    if t.get_device() != dev:
        _bad(fn, f"{name} must be on the handle's device (cuda:{dev})")


def _pools(fn, torch, dev, k, v, layered):
    """The cache's argument block, and (dtype, layers, pages, kv_heads, page, D)."""
    dims = 5 if layered else 4
    if k.dim() != dims or v.dim() != dims + 1:
        lead = "layers, " if layered else ""
        _bad(fn, f"k must be [{lead}pages, kv_heads, page, D], v [{lead}pages, kv_heads, page / 8, D, 8]")
    ks, vs, kt, vt = k.shape, v.shape, k.stride(), v.stride()
    if layered:
        L, kl, vl = ks[0], kt[0], vt[0]
        if vs[0] != L:
            _bad(fn, "k and v differ in layers")
        ks, vs, kt, vt = ks[1:], vs[1:], kt[1:], vt[1:]
    else:
        L, kl, vl = 1, 0, 0
    N, H, page, D = ks
    if vs != (N, H, page // 8, D, 8) or page % 8:
        _bad(fn, f"v must be [..., {N}, {H}, {page // 8}, {D}, 8] for k [..., {N}, {H}, {page}, {D}]")
    if kt[1:] != (page * D, D, 1) or vt[1:] != (page * D, 8 * D, 8, 1):
        _bad(fn, "a page of the cache must be contiguous")
    dt = k.dtype
    code = TGS_BF16 if dt is torch.bfloat16 else TGS_F16 if dt is torch.float16 else -1
    if code < 0 or v.dtype is not dt:
        raise TypeError(f"{fn}: the cache must be bfloat16 or float16")
    if k.get_device() != dev or v.get_device() != dev:
        _bad(fn, f"the cache must be on the handle's device (cuda:{dev})")
    if L == 1:
        kl = vl = 0
    block = _CACHE.pack(k.data_ptr(), v.data_ptr(), kl, kt[0], vl, vt[0], L, N, page, H, D, code)
    return block, (dt, L, N, H, page, D)


def _new_rows(fn, dev, k_new, v_new, shape, dt, layered):
    for name, t in (("k_new", k_new), ("v_new", v_new)):
        if t.dtype is not dt or t.shape != shape or t.stride(-1) != 1 or t.get_device() != dev:
            _bad(fn, f"{name} must be a {dt} tensor of shape {tuple(shape)} on cuda:{dev}, its last dimension contiguous")
    a, b = k_new.stride(), v_new.stride()
    if not layered:
        a, b = (0, *a), (0, *b)
    return _ROWS.pack(k_new.data_ptr(), v_new.data_ptr(), a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3])


def _sequences(fn, torch, dev, tables, lens):
    if tables is None or tables.dim() != 2:
        _bad(fn, "tables must be int32 [sequences, slots]")
    B, P = tables.shape
    _ints(fn, torch, dev, "tables", tables, B, P)
    _ints(fn, torch, dev, "lens", lens, B)
    return _SEQS.pack(tables.data_ptr(), lens.data_ptr(), B, P), B, P


def _out(fn, torch, dev, t, dtype, shape, name):
    if t is None:
        return torch.empty(shape, dtype=dtype, device=f"cuda:{dev}")
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous() or t.get_device() != dev:
        _bad(fn, f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{dev}")
    return t


def _apart(fn, outs, ins):
    """No output starts where an input does."""
    at = {t.data_ptr() for t in ins if t.numel()}
    for name, t in outs:
        if t.numel() and t.data_ptr() in at:
            _bad(fn, f"{name} must not be an input")


class CacheOps:
    """Methods of `Sampler` (self._L, self._h, self.device, self._check)."""

    def _raw_stream(self, torch, stream):
        if stream is not None:
            return stream
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        return raw(self.device) if raw is not None else torch.cuda.current_stream(self.device).cuda_stream

    def beam_select(self, logits, scores, W, n_out, hist=None, hist_len=None, out=None, vocab=None, stream=None):
        """The n_out best continuations of each request's W beams: logits
        [G * W, >= V] (float32 or bfloat16), scores float32 [G * W] (-inf: the
        beam has ended), optional histories int32 [G * W, H] with hist_len
        [G * W].  Returns `out`, a dict of scores, parents (rows of logits)
        and tokens [G * n_out], and with histories hist [G * n_out, H] and
        hist_len, best first, equal ones by the lower beam, then the lower id;
        past the last candidate -inf, -1, -1."""
        torch, fn, dev = _torch(), "beam_select", self.device
        if logits.dim() != 2 or logits.stride(1) != 1:
            _bad(fn, "logits must be [G * W, V] with unit stride along V")
        code = 0 if logits.dtype is torch.float32 else TGS_BF16 if logits.dtype is torch.bfloat16 else -1
        if code < 0:
            raise TypeError("beam_select: logits must be float32 or bfloat16")
        rows, width = logits.shape
        V = width if vocab is None else vocab
        if not 1 <= V <= width:
            _bad(fn, f"vocab {V} outside [1, {width}]")
        if W < 1 or rows % W:
            _bad(fn, f"{rows} rows are not requests of {W} beams")
        if logits.get_device() != dev:
            _bad(fn, f"logits must be on the handle's device (cuda:{dev})")
        if scores.dtype is not torch.float32 or scores.shape != (rows,) or not scores.is_contiguous() or scores.get_device() != dev:
            _bad(fn, f"scores must be a contiguous float32 tensor of {rows} elements on cuda:{dev}")
        G = rows // W
        n = G * n_out
        i32 = torch.int32
        o = {} if out is None else out
        o["scores"] = _out(fn, torch, dev, o.get("scores"), torch.float32, (n,), "out scores")
        o["parents"] = _out(fn, torch, dev, o.get("parents"), i32, (n,), "out parents")
        o["tokens"] = _out(fn, torch, dev, o.get("tokens"), i32, (n,), "out tokens")
        if (hist is None) != (hist_len is None):
            _bad(fn, "hist and hist_len go together")
        if hist is not None:
            if hist.dim() != 2 or hist.shape[1] < 1:
                _bad(fn, "hist must be int32 [G * W, H]")
            H = hist.shape[1]
            _ints(fn, torch, dev, "hist", hist, rows, H)
            _ints(fn, torch, dev, "hist_len", hist_len, rows)
            o["hist"] = oh = _out(fn, torch, dev, o.get("hist"), i32, (n, H), "out hist")
            o["hist_len"] = ol = _out(fn, torch, dev, o.get("hist_len"), i32, (n,), "out hist_len")
            _apart(fn, (("out hist", oh), ("out hist_len", ol)), (hist, hist_len))
            hp, lp, ohp, olp = hist.data_ptr(), hist_len.data_ptr(), oh.data_ptr(), ol.data_ptr()
        else:
            H, hp, lp, ohp, olp = 0, None, None, None, None
        _apart(fn, (("out scores", o["scores"]),), (scores,))
        rc = self._L.tgs_beam_select(
            self._h, logits.data_ptr(), code, G, W, V, logits.stride(0), scores.data_ptr(), n_out, hp, lp, H,
            o["scores"].data_ptr(), o["parents"].data_ptr(), o["tokens"].data_ptr(), ohp, olp,
            self._raw_stream(torch, stream))
        if rc:
            self._check(rc, "tgs_beam_select")
        return o

    def tree_attention(self, q, k_new, v_new, k, v, tables, lens, parents=None, max_len=None, scale=None, out=None,
                       lse=None, stream=None):
        """Attention of T drafted nodes per sequence over the sequence's
        cached tokens, each node's ancestors and itself: q [B, T, q_heads, D],
        k_new and v_new [B, T, kv_heads, D] (any strides, D contiguous), k and
        v one layer's pools, tables int32 [B, slots], lens int32 [B], parents
        int32 [B, T] (an earlier node, -1: a root; None: a chain).  max_len:
        a bound of lens known on the host, scale: 1 / sqrt(D) when None.
        Returns out [B, T, q_heads, D]; lse float32 [B, T, q_heads], when
        given, gets the natural logsumexp of the scaled scores."""
        torch, fn, dev = _torch(), "tree_attention", self.device
        cache, (dt, _, _, H, page, D) = _pools(fn, torch, dev, k, v, False)
        seqs, B, P = _sequences(fn, torch, dev, tables, lens)
        if q.dim() != 4 or q.shape[0] != B or q.shape[3] != D or q.dtype is not dt or q.stride(3) != 1 or q.get_device() != dev:
            _bad(fn, f"q must be a {dt} tensor of shape ({B}, T, q_heads, {D}) on cuda:{dev}, its last dimension contiguous")
        shape = q.shape
        _, T, Hq, _ = shape
        if Hq % H:
            _bad(fn, f"{Hq} query heads are no multiple of {H} key heads")
        rows = _new_rows(fn, dev, k_new, v_new, (B, T, H, D), dt, False)
        if parents is not None:
            _ints(fn, torch, dev, "parents", parents, B, T)
        out = _out(fn, torch, dev, out, dt, shape, "out")
        if lse is not None:
            lse = _out(fn, torch, dev, lse, torch.float32, (B, T, Hq), "lse")
        _apart(fn, (("out", out),), (q, k_new, v_new))
        qb, qt, qh, _ = q.stride()
        attn = _ATTN.pack(q.data_ptr(), qb, qt, qh, 0 if parents is None else parents.data_ptr(), out.data_ptr(),
                          0 if lse is None else lse.data_ptr(), T, Hq, P * page if max_len is None else max_len,
                          D ** -0.5 if scale is None else scale)
        rc = self._L.tgs_tree_attention(self._h, cache, rows, seqs, attn, self._raw_stream(torch, stream))
        if rc:
            self._check(rc, "tgs_tree_attention")
        return out

    def kv_append(self, k_new, v_new, k, v, tables, lens, counts=None, lens_out=None, stream=None):
        """Writes the first counts[b] (all, when None) of the T new rows of
        each sequence and layer, k_new and v_new [layers, B, T, kv_heads, D],
        behind its lens[b] tokens.  Returns lens_out int32 [B]: the new
        lengths, -1 where the rows did not fit (nothing is written there)."""
        torch, fn, dev = _torch(), "kv_append", self.device
        cache, (dt, L, _, H, _, D) = _pools(fn, torch, dev, k, v, True)
        seqs, B, _ = _sequences(fn, torch, dev, tables, lens)
        if k_new.dim() != 5:
            _bad(fn, "k_new and v_new must be [layers, B, T, kv_heads, D]")
        T = k_new.shape[2]
        rows = _new_rows(fn, dev, k_new, v_new, (L, B, T, H, D), dt, True)
        if counts is not None:
            _ints(fn, torch, dev, "counts", counts, B)
        lens_out = _out(fn, torch, dev, lens_out, torch.int32, (B,), "lens_out")
        _apart(fn, (("lens_out", lens_out),), (lens, tables) if counts is None else (lens, tables, counts))
        rc = self._L.tgs_kv_append(self._h, cache, rows, seqs, T, None if counts is None else counts.data_ptr(),
                                   lens_out.data_ptr(), self._raw_stream(torch, stream))
        if rc:
            self._check(rc, "tgs_kv_append")
        return lens_out

    def tree_commit(self, k_new, v_new, k, v, tables, lens, parents, draft, sampled, out=None, stream=None):
        """Accepts each sequence's drafted tree as far as it agrees with the
        ids sampled after its nodes, and writes the path's rows to the cache:
        parents, draft, sampled int32 [B, T] (node 0 is the root), k_new and
        v_new [layers, B, T, kv_heads, D].  Returns `out`, a dict of n_acc
        [B], tokens [B, T] (accepted, then the one sampled at the last),
        path [B, T] and lens [B] (-1: the rows did not fit)."""
        torch, fn, dev = _torch(), "tree_commit", self.device
        cache, (dt, L, _, H, _, D) = _pools(fn, torch, dev, k, v, True)
        seqs, B, _ = _sequences(fn, torch, dev, tables, lens)
        if k_new.dim() != 5:
            _bad(fn, "k_new and v_new must be [layers, B, T, kv_heads, D]")
        T = k_new.shape[2]
        rows = _new_rows(fn, dev, k_new, v_new, (L, B, T, H, D), dt, True)
        _ints(fn, torch, dev, "parents", parents, B, T)
        _ints(fn, torch, dev, "draft", draft, B, T)
        _ints(fn, torch, dev, "sampled", sampled, B, T)
        o = {} if out is None else out
        i32 = torch.int32
        o["n_acc"] = _out(fn, torch, dev, o.get("n_acc"), i32, (B,), "out n_acc")
        o["tokens"] = _out(fn, torch, dev, o.get("tokens"), i32, (B, T), "out tokens")
        o["path"] = _out(fn, torch, dev, o.get("path"), i32, (B, T), "out path")
        o["lens"] = _out(fn, torch, dev, o.get("lens"), i32, (B,), "out lens")
        _apart(fn, ((f"out {x}", o[x]) for x in ("n_acc", "tokens", "path", "lens")), (lens, tables, parents, draft, sampled))
        rc = self._L.tgs_tree_commit(self._h, cache, rows, seqs, T, parents.data_ptr(), draft.data_ptr(), sampled.data_ptr(),
                                     o["n_acc"].data_ptr(), o["tokens"].data_ptr(), o["path"].data_ptr(),
                                     o["lens"].data_ptr(), self._raw_stream(torch, stream))
        if rc:
            self._check(rc, "tgs_tree_commit")
        return o

    def kv_fork(self, k, v, tables, lens, parents, room=1, tables_out=None, lens_out=None, stream=None):
        """Reorders a cache's rows after a beam step: row r goes on from row
        parents[r].  Full pages are shared; the page that the next `room`
        tokens go to has one writer, the other rows get free pages of the pool
        (those that no row names any more) and copies.  Returns (tables_out
        [B, slots], lens_out [B]): -1 past the slots in use; length 0 for a
        parent outside the rows, -1 for a row that found no page."""
        torch, fn, dev = _torch(), "kv_fork", self.device
        cache, _ = _pools(fn, torch, dev, k, v, True)
        seqs, B, P = _sequences(fn, torch, dev, tables, lens)
        _ints(fn, torch, dev, "parents", parents, B)
        tables_out = _out(fn, torch, dev, tables_out, torch.int32, (B, P), "tables_out")
        lens_out = _out(fn, torch, dev, lens_out, torch.int32, (B,), "lens_out")
        _apart(fn, (("tables_out", tables_out), ("lens_out", lens_out)), (tables, lens, parents))
        rc = self._L.tgs_kv_fork(self._h, cache, seqs, parents.data_ptr(), room, tables_out.data_ptr(), lens_out.data_ptr(),
                                 self._raw_stream(torch, stream))
        if rc:
            self._check(rc, "tgs_kv_fork")
        return tables_out, lens_out
