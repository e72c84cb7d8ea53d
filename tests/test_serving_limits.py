"""Calls of the operators for batches at the edges of what the header allows: as many rows as
fit, tables that lie, and calls of several threads at once."""

from __future__ import annotations

import ctypes
import subprocess

import numpy as np
import pytest

import gemma_hip
from gemma_hip import CACHE_I8
from test_serving import CSRC, F32, cuda, quantise, stream, values


def test_grids_of_the_cache_are_launchable(tmp_path):
    """kv_cache.h's grid, compiled for the host: every workgroup once, at most 2^32 - 1 threads a
    dimension, to the 2^24 workgroups that 2^25 rows by heads of 256 dims take."""
    src, so = tmp_path / "grid.cpp", tmp_path / "grid.so"
    src.write_text('#include "kv_cache.h"\n'
                   'extern "C" void grid(long n, int b, unsigned *o)'
                   ' { gh::KvGrid g = gh::kv_grid_of(n, b); o[0] = g.x; o[1] = g.y; o[2] = g.z; }\n'
                   'extern "C" long block(unsigned x, unsigned z) { return gh::kv_block(x, z); }\n')
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-I", CSRC, str(src), "-o",
                    str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.block.restype = ctypes.c_long
    for n in (1, 5, (1 << 22) - 1, 1 << 22, (1 << 22) + 1, 3 * (1 << 22) + 7, 1 << 24):
        o = (ctypes.c_uint * 3)()
        lib.grid(ctypes.c_long(n), 9, o)
        x, y, z = o
        assert y == 9 and x * 256 < 1 << 32 and 1 <= z <= 65535
        starts = [lib.block(0, k) for k in range(z)]
        assert starts[0] == 0 and all(b - a == x for a, b in zip(starts, starts[1:]))
        assert n <= starts[-1] + x < n + (1 << 22)


@pytest.mark.gpu
@pytest.mark.parametrize("flat", [False, True])
def test_as_many_rows_as_there_may_be(gh, flat):
    """2^25 rows of a key/value head of 256 dims written and read, of which the last 64 have a
    position; flat: beside sequences without rows."""
    import torch

    rows, hd, ln = 1 << 25, 256, 64
    rng = np.random.default_rng(1)
    k = torch.empty((rows, hd), device="cuda")
    v = torch.empty((rows, hd), device="cuda")
    x = rng.standard_normal((ln, hd)).astype(F32)
    k[-ln:] = cuda(x)
    batch = 3 if flat else 1
    lens = np.zeros(batch, np.int32)
    lens[0] = ln
    row0 = np.full(batch + 1, rows, np.int32)
    row0[0] = 0
    b = gemma_hip.batch(cuda(np.zeros((batch, 1), np.int32)), cuda(lens), cuda(row0), batch, 1, rows,
                        rows, ln)
    codes = torch.zeros((2, ln, hd), dtype=torch.int8, device="cuda")
    scales = torch.zeros((2, ln), device="cuda")
    c = gemma_hip.cache(codes[0], codes[1], scales[0], scales[1], CACHE_I8, 1, ln, 1, hd)
    gh.cache_write(c, b, k, 0, k, 0, stream())
    k[:4] = 5.0
    v[:4] = 5.0
    gh.cache_read(c, b, k, 0, v, 0, stream())
    torch.cuda.synchronize()
    want = values(*quantise(x, CACHE_I8), CACHE_I8)
    for t in (k, v):
        assert np.array_equal(t[-ln:].cpu().numpy(), want)
        assert not t[:4].any() and not t[rows // 2:rows // 2 + 4].any() and not t[-ln - 4:-ln].any()
    del k, v
    torch.cuda.empty_cache()
