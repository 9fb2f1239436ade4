"""Runs one beam, attention or cache call on the CPU simulation of the kernels
(built by the Makefile beside this file, under AddressSanitizer).  TEST
INFRASTRUCTURE ONLY."""
from __future__ import annotations

import fcntl
import os
import subprocess
import tempfile

import numpy as np
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
BIN = os.path.join(HERE, "build", "kv_case")


def build():
    os.makedirs(os.path.join(HERE, "build"), exist_ok=True)
    with open(os.path.join(HERE, "build", ".lock"), "w") as lk:
        fcntl.flock(lk, fcntl.LOCK_EX)
        subprocess.run(["make", "-s", f"-j{min(8, os.cpu_count() or 1)}", "-C", HERE], check=True)


def _raw(t):
    """The tensor's storage from its first element on, as bytes (strided tensors keep their gaps)."""
    t = t.detach()
    n = 1 + sum((s - 1) * st for s, st in zip(t.shape, t.stride())) if t.numel() else 0
    flat = torch.as_strided(t, (n,), (1,))
    return flat.contiguous().view(torch.uint8).numpy().tobytes() if n else b""


def call(op, arrays, num_cu=4, ws_words=1 << 20, timeout=600, **meta):
    """arrays: name -> tensor or None; those named o_* are outputs.  Returns
    (status, {name: tensor}) with the outputs and the pools k and v as they are afterwards."""
    with tempfile.TemporaryDirectory() as d:
        for name, t in arrays.items():
            if t is not None:
                with open(os.path.join(d, name + ".bin"), "wb") as f:
                    f.write(_raw(t))
        with open(os.path.join(d, "meta.txt"), "w") as f:
            for k, v in dict(meta, num_cu=num_cu, ws_words=ws_words).items():
                f.write(f"{k} {float(v)!r}\n")
        env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:max_malloc_fill_size=2147483647:malloc_fill_byte=190",
                   UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
        r = subprocess.run([BIN, op, d], capture_output=True, text=True, env=env, timeout=timeout)
        if r.returncode != 0:
            raise AssertionError(f"simulation failed ({r.returncode}):\n{r.stderr[-4000:]}")
        rc = int(r.stdout.split()[1])
        out = {}
        for name, t in arrays.items():
            p = os.path.join(d, name + ".out")
            if os.path.exists(p):
                flat = torch.from_numpy(np.fromfile(p, dtype=np.uint8)).view(t.dtype)
                out[name] = torch.as_strided(flat, t.shape, t.stride())
        return rc, out
