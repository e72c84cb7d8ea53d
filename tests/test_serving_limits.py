"""Calls of the operators for batches at the edges of what the header allows: as many rows as
fit, tables that lie, and calls of several threads at once."""

from __future__ import annotations

import ctypes
import subprocess
import threading

import numpy as np
import pytest

import gemma_hip
from gemma_hip import CACHE_E4M3, CACHE_I8
from test_serving import CSRC, F32, Paged, cuda, quantise, stream, values


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


def attention_call(gh, seed, lens, heads=4, kv=1, hd=256):
    """A call of single tokens, and how many bytes its workspace takes."""
    import torch

    rng = np.random.default_rng(seed)
    p = Paged([(1, n) for n in lens], kv, hd, 64, CACHE_E4M3, rng)
    p.fill(rng)
    c, b = p.device(), p.batch()
    q = torch.randn((p.rows, heads * hd), device="cuda")
    out = torch.zeros_like(q)

    def call(work, s):
        gh.cache_attention(out, q, 0, c, b, heads, 0, 0.0625, 0.0, False, 0, work, s)

    call.out, call.keep = out, p
    return call, gh.cache_attention_work(c, b, heads, 0, 0)


@pytest.mark.gpu
def test_calls_with_workspaces_do_not_wait_for_those_without(gh):
    """A thread whose stream's workspace grows waits for that stream; one that brings a
    workspace of its own goes on meanwhile, and so does one that samples short rows."""
    import torch

    small, need0 = attention_call(gh, 1, [3000])
    large, need1 = attention_call(gh, 2, [4000] * 40)
    mine, need2 = attention_call(gh, 3, [3000])
    assert 0 < need0 < need1
    work = torch.empty(need2, dtype=torch.uint8, device="cuda")
    busy, free = torch.cuda.Stream(), torch.cuda.Stream()
    logits, u = torch.randn((1, 1000), device="cuda"), torch.rand(1, device="cuda")
    tokens = torch.empty(1, dtype=torch.int32, device="cuda")
    m = torch.randn((8192, 8192), device="cuda")
    to = torch.empty_like(m)
    torch.mm(m, m, out=to)
    small(None, busy.cuda_stream)
    mine(work, free.cuda_stream)
    torch.cuda.synchronize()
    want = mine.out.clone()
    mine.out.zero_()
    torch.cuda.synchronize()
    begun, errors = threading.Event(), []

    def grow():
        try:
            begun.set()
            large(None, busy.cuda_stream)
        except Exception as e:  # (shown by the main thread)
            errors.append(e)

    with torch.cuda.stream(busy):
        for _ in range(200):
            torch.mm(m, m, out=to)
        done = torch.cuda.Event()
        done.record()
    t = threading.Thread(target=grow)
    t.start()
    begun.wait()
    t.join(0.2)  # time to take the lock and to wait
    waiting = t.is_alive()
    mine(work, free.cuda_stream)
    gh.sample(tokens, None, logits, 0, 1, 1000, None, u, None, free.cuda_stream)
    early = not done.query()
    free.synchronize()
    t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert waiting, "the other thread's call was not waiting: this shows nothing"
    assert early, "a call with a workspace of its own waited for another thread's"
    assert torch.equal(mine.out, want)


def clamped(lens, row0, rows, max_rows, max_len):
    """(first row, rows, length) of every sequence, cut to the call's bounds."""
    out = []
    for i, ln in enumerate(lens):
        r0 = min(max(row0[i], 0), rows)
        out.append((r0, min(min(max(row0[i + 1], r0), rows) - r0, max_rows),
                    min(max(ln, 0), max_len)))
    return out


LIES = {  # lengths, first rows: of five rows, three a sequence at most, in 64 positions
    "few": ([2 ** 31 - 1, -5, 64], [0, 900, 2, 5]),
    "falling": ([70, 64, -2 ** 31], [4, 3, 1, -9]),
    "many": ([9, 64, 0, 2 ** 31 - 1, 33, -1, 64], [-7, 2, 2, 1, 2 ** 31 - 1, 3, 0, 5]),
}


@pytest.mark.gpu
@pytest.mark.parametrize("case", sorted(LIES))
@pytest.mark.parametrize("shared", [0, 16])
def test_tables_that_lie_lead_nowhere_else(gh, case, shared):
    """Whatever lengths, first rows and page ids say, cache_write touches no place but those
    that they name within the call's bounds, cache_read and attention no row but the call's
    sequences', and nothing beside any of the buffers."""
    import torch

    lens, row0 = LIES[case]
    rows, max_rows, max_len, hd, kv, page, npages, heads = 5, 3, 64, 128, 2, 16, 9, 4
    rng = np.random.default_rng(7)
    batch = len(lens)
    table = rng.permutation(np.arange(batch * 4) % (npages + 3)).reshape(batch, 4).astype(np.int32)
    table[0, 0], table[-1, -1], table[1, 3] = npages, -1, -2 ** 31
    pad = 4096  # before and behind every buffer

    def fenced(n, dtype, value):
        whole = torch.full((n + 2 * pad,), value, dtype=dtype, device="cuda")
        return whole, whole[pad:pad + n]

    ncode, nscale = npages * kv * page * hd, npages * kv * page
    codes = [fenced(ncode, torch.int8, 3) for _ in "kv"]
    scales = [fenced(nscale, torch.float32, 0.5) for _ in "kv"]
    reads = [fenced(rows * kv * hd, torch.float32, 7.0) for _ in "kv"]
    outs = fenced(rows * heads * hd, torch.float32, 7.0)
    every = codes + scales + reads + [outs]
    c = gemma_hip.cache(codes[0][1], codes[1][1], scales[0][1], scales[1][1], CACHE_I8, npages,
                        page, kv, hd)
    b = gemma_hip.batch(cuda(table), cuda(np.array(lens, np.int32)), cuda(np.array(row0, np.int32)),
                        batch, 4, rows, max_rows, max_len)
    x = torch.randn((rows, kv * hd), device="cuda")
    q = torch.randn((rows, heads * hd), device="cuda")
    gh.cache_write(c, b, x, 0, x, 0, stream())
    gh.cache_read(c, b, reads[0][1], 0, reads[1][1], 0, stream())
    gh.cache_attention(outs[1], q, 0, c, b, heads, 0, 0.1, 0.0, False, shared, None, stream())
    torch.cuda.synchronize()

    for whole, inner in every:
        edge = torch.cat([whole[:pad], whole[pad + inner.numel():]])
        assert (edge == edge[0]).all() and float(edge[0]) in (3.0, 0.5, 7.0)
    named, ours = np.zeros((npages, page), bool), np.zeros(rows, bool)
    for i, (r0, n, ln) in enumerate(clamped(lens, row0, rows, max_rows, max_len)):
        ours[r0:r0 + n] = True
        for pos in range(max(0, ln - n), ln):
            if 0 <= table[i, pos // page] < npages:
                named[table[i, pos // page], pos % page] = True
    for (_, code), (_, scale) in zip(codes, scales):
        same = (code.view(npages, kv, page, hd) == 3).all(3).all(1).cpu().numpy()
        assert same[~named].all() and (case != "few" or not same[named].any())
        same = (scale.view(npages, kv, page) == 0.5).all(1).cpu().numpy()
        assert same[~named].all()
    for _, inner in reads + [outs]:
        same = (inner.view(rows, -1) == 7.0).all(1).cpu().numpy()
        assert same[~ours].all()
