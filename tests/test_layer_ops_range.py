"""The operators between the products of a served batch where fp32 ends, at sums of many
terms, and calls that need none of the library's memory.  Definitions and bars are those of
test_layer_ops.py, or stand beside the test."""

from __future__ import annotations

import math
import threading

import numpy as np
import pytest

import gemma_hip
from gemma_hip import ADAPTER_BF16, ADAPTER_F16, ADAPTER_F32, NORM_LAYER, NORM_RMS
from test_layer_ops import (F32, F64, HALF, TYPES, adapters_expected, close_logs, codes_of_rows,
                            describe, normed, once)
from test_serving import cuda, stream

TOP = np.finfo(F32).max


# ---- norms ------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("x_scale", [1.0, 0.5, -2.0])
@pytest.mark.parametrize("rows,dim,kind", [(5, 8, NORM_RMS), (5, 2560, NORM_LAYER),
                                           (1030, 256, NORM_RMS), (1030, 1152, NORM_LAYER)])
def test_a_sum_without_a_block_is_clamped(gh, rows, dim, kind, x_scale):
    """x' = clamp(x_scale x) where there is no y, whatever x_scale: infinities become the largest
    values and their rows have finite norms and codes; NaN stays."""
    import torch

    rng = np.random.default_rng(dim)
    x = rng.standard_normal((rows, dim)).astype(F32)
    x[0, 2], x[1, 3], x[2, 1], x[3, :4] = np.inf, -np.inf, np.nan, (TOP, -TOP, np.inf, -np.inf)
    w = (rng.standard_normal(dim) * 0.2).astype(F32)
    with np.errstate(over="ignore"):
        want = np.clip((F64(x_scale) * x.astype(F64)), -F64(TOP), F64(TOP)).astype(F32)
    want[2, 1] = np.nan
    out, h = torch.empty((2, rows, dim), device="cuda").unbind(0)
    hq, hs = torch.empty((rows, dim), dtype=torch.int8, device="cuda"), \
        torch.empty(rows, device="cuda")
    gh.norm_residual(gemma_hip.residual(cuda(x), x_scale=x_scale, x_out=out, h=h, hq=hq, hs=hs,
                                        before=gemma_hip.norm(kind, cuda(w), None, 1.0)), rows, dim,
                     stream())
    assert np.array_equal(out.cpu().numpy(), want, equal_nan=True)
    got, q, s = h.cpu().numpy(), hq.cpu().numpy(), hs.cpu().numpy()
    fine = np.arange(rows) != 2
    assert once(got[fine], normed(want[fine], kind, w, None, 1.0))
    code, scale = codes_of_rows(got[fine])
    assert np.array_equal(q[fine], code) and np.array_equal(s[fine], scale)
    assert np.isnan(got[2]).all() and np.isnan(s[2]) and not q[2].any()


# ---- log probabilities --------------------------------------------------------------


def far_apart(vocab, t, rng, kind):
    """Rows of finite logits whose differences pass FLT_MAX, or are no more than some temperatures
    that fp32 holds as subnormals."""
    if kind == "ends":
        return rng.choice(np.array([-TOP, -3e38, 3e38, TOP], F32), vocab)
    if kind == "two":
        l = np.full(vocab, -3e38, F32)
        l[rng.integers(0, vocab, 1 + vocab // 3)] = 3e38
        return l
    if kind == "spread":
        return (rng.uniform(-1, 1, vocab) * F64(TOP)).astype(F32)
    if kind == "holes":
        l = (rng.uniform(-1, 1, vocab) * F64(TOP)).astype(F32)
        l[rng.random(vocab) < 0.3] = -np.inf
        l[rng.random(vocab) < 0.1] = np.nan
        return l
    if kind == "small":  # some temperatures apart
        return (rng.standard_normal(vocab) * 3 * F64(t)).astype(F32)
    l = (rng.standard_normal(vocab) * 3 * F64(t)).astype(F32)  # "mixed": far below as well
    l[rng.random(vocab) < 0.5] = -1e30
    return l


FAR = [(k, t) for k in ("ends", "two", "spread", "holes")
       for t in (np.inf, float(TOP), 3e38, 1e38, 1e37, 1.5, 1.0, 1e-40)] + \
      [(k, t) for k in ("small", "mixed") for t in (1e-45, 1e-42, 1e-40, 4e-39, 1e-38, 1e30)]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,ntop,times", [(2, 2, 1), (70, 9, 1), (2100, 64, 1), (5000, 5, 1),
                                              (40000, 12, 1), (3000, 4, 14), (9000, 7, 14)])
def test_logits_at_any_distance(gh, vocab, ntop, times):
    """Every kind of row at temperatures of its size, in one launch and in two; many rows are the
    same ones repeated."""
    import torch

    rng = np.random.default_rng(vocab)
    l = np.stack([far_apart(vocab, F32(t), rng, k) for k, t in FAR])
    t = np.array([t for _, t in FAR], F32)
    n = len(FAR)
    rows, targets = n * times, 3
    ids = rng.integers(0, vocab, (n, targets)).astype(np.int32)
    ids[:, 0], ids[:, 1] = np.nan_to_num(l, nan=-np.inf, posinf=np.inf).argmax(1), \
        np.nan_to_num(l, nan=np.inf).argmin(1)
    out = dict(logp=torch.empty((rows, targets), device="cuda"),
               rank=torch.empty((rows, targets), dtype=torch.int32, device="cuda"),
               entropy=torch.empty(rows, device="cuda"),
               top=torch.empty((rows, ntop), dtype=torch.int32, device="cuda"),
               top_logp=torch.empty((rows, ntop), device="cuda"))
    gh.logprobs(gemma_hip.scores(**out), cuda(l).repeat(times, 1), 0, rows, vocab,
                cuda(t).repeat(times), cuda(ids).repeat(times, 1), targets, ntop, None, stream())
    for v in out.values():
        again = v.view(times, -1)
        assert torch.equal(again, again[:1].expand_as(again))
    got = {k: v[:n].cpu().numpy() for k, v in out.items()}
    bad = []
    for r in range(n):
        logp, rank, h, top, tl = describe(l[r], F64(t[r]), ids[r], ntop)
        assert np.array_equal(got["rank"][r], rank) and np.array_equal(got["top"][r], top), FAR[r]
        if not (close_logs(got["logp"][r], logp) and close_logs(got["top_logp"][r], tl) and
                close_logs(got["entropy"][r], h)):
            bad.append((FAR[r], got["logp"][r], logp, got["entropy"][r], h))
    assert not bad, bad


# ---- adapters ---------------------------------------------------------------------


def one_adapter(gh, kind, a, b, x, scale=1.0, most=None):
    """A sequence's rows of zeros through one adapter, on the GPU: (result, definition in fp64, sums
    of the terms' magnitudes)."""
    import torch

    dt = {ADAPTER_F32: torch.float32, ADAPTER_BF16: torch.bfloat16, ADAPTER_F16: torch.float16}[kind]
    a, b, x = torch.from_numpy(a)[None].to(dt), torch.from_numpy(b)[None].to(dt), torch.from_numpy(x)
    (rows, k), (n, rank) = x.shape, b.shape[1:]
    base, scale = torch.zeros((rows, n)), torch.tensor([scale], dtype=torch.float32)
    ad = gemma_hip.adapters(cuda(np.array([0, rows], np.int32)), cuda(np.zeros(1, np.int32)),
                            scale.cuda(), 1, rows, most or rows, 1, rank, kind)
    jobs = gemma_hip.adapter_jobs([(a.cuda(), b.cuda(), n)])
    out = torch.full((rows, n), 7.0, device="cuda")
    gh.adapters_add(out, 0, base.cuda(), 0, ad, jobs, x.cuda(), 0, k, None, stream())
    with np.errstate(all="ignore"):
        want, size = adapters_expected(([rows], k, [n], rank, 1), [a], [b], x, base, scale, [0])
    return out.cpu().numpy().astype(F64), want, size


def agree(got, want, size, k, rank):
    """Within the bar where the definition is finite, the same infinity or NaN elsewhere."""
    room = (math.sqrt(3 * k) + math.sqrt(3 * rank) + 8) * HALF
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    with np.errstate(invalid="ignore"):
        assert (np.abs(got - want)[fine] <= room * size[fine]).all()


# by the row in one launch and in two (n), by tiles, by tiles whose waves share the matrices
ENDS = [(2, 70), (2, 9000), (3, 70), (40, 70), (100, 70), (100, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,n", ENDS)
@pytest.mark.parametrize("rank", [8, 40, 128])
@pytest.mark.parametrize("where", ["x", "u", "a", "b"])
def test_adapters_at_the_largest_values(gh, kind, rows, n, rank, where):
    """Values from the largest that rounds to a finite bf16 up to FLT_MAX, among the inputs, the
    first product's results and the matrices, beside ones that leave the answers finite."""
    k, rng = 136, np.random.default_rng(rows + n)
    ends = np.array([TOP, -TOP, 3.3961775e38, 3.3961777e38, -3.4e38, 1e38], F32)
    a, b = rng.standard_normal((rank, k)), rng.standard_normal((n, rank))
    x = rng.standard_normal((rows, k))
    if where == "x":
        a, b = a * 2.0 ** -10, b * 2.0 ** -10
    elif where == "u":  # the first inputs, as they are
        a, b = np.eye(rank, k), b * 2.0 ** -10
    else:
        x *= 2.0 ** -20
        a = a if where == "a" else np.eye(rank, k)
        b = b * 2.0 ** -10 if where == "a" else b
    a, b, x = a.astype(F32), b.astype(F32), x.astype(F32)
    if where in "xu":
        x[0, 1], x[-1, 2:8] = TOP, ends
        x[rows // 2, :6] = ends
    else:  # f16 ends at 65504, bf16 at 3.39e38
        m = a if where == "a" else b
        top = {"f32": 1.0, "bf16": 0.99, "f16": 65504 / F64(TOP)}[kind]
        m[1, 2:8], m[-1, 0] = (ends * top).astype(F32), F32(TOP * top)
    got, want, size = one_adapter(gh, TYPES[kind], a, b, x)
    assert np.isfinite(want).all() and size.max() < F64(TOP)
    agree(got, want, size, k, rank)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,n", ENDS)
@pytest.mark.parametrize("rank", [8, 40, 128])
def test_adapters_of_infinities(gh, kind, rows, n, rank):
    """An infinity or NaN in the inputs or the matrices comes out where it belongs, and nowhere
    else, a row of one beside a row of the other too."""
    k, rng = 136, np.random.default_rng(rows + n)
    a, b = (rng.random(s).astype(F32) + F32(0.5) for s in ((rank, k), (n, rank)))
    x = rng.random((rows, k)).astype(F32) + F32(0.5)
    for where in range(5):
        p, q, y = a.copy(), b.copy(), x.copy()
        if where == 0:
            y[0, 3], y[-1, k - 1] = np.inf, -np.inf
        elif where == 1:
            y[rows // 2, 7], q[5] = np.nan, -q[5]
        elif where == 2:
            p[rank - 1, 9], q[:, rank - 1] = np.inf, np.where(np.arange(n) % 3 == 0, 0.0, 1.0)
        else:
            q[5, 2], q[n - 1, rank - 1], q[6, 1] = np.inf, -np.inf, np.nan
        if where == 4:
            y[0, 3], y[-1, 1] = np.nan, np.inf
        got, want, size = one_adapter(gh, TYPES[kind], p, q, y)
        assert not np.isfinite(want).all()
        agree(got, want, size, k, rank)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 10240), (3, 10240), (1, 1 << 20), (3, 1 << 20)])
def test_adapters_of_many_inputs(gh, kind, rows, k):
    """Sums of equal terms, whose roundings all point one way.  Sums are fp32 over 4096 inputs at
    most and fp64 beyond.  By the row: 64 products to a lane's sum, 6 sums of lanes; by the tile 8
    steps of 2 times up to 6 products, 8 sums of waves; then the scale, u B of rank 8 in up to 9
    additions (6 products) and the base: 96 + 8 + 1 + 9 + 1 roundings of 2^-24 at most, and products
    off by 2^-22 twice: 7.4e-6 of the sum of magnitudes, below the 1e-5 that is promised."""
    rank, n, rng = 8, 24, np.random.default_rng(k)
    a = np.repeat((rng.random((rank, 1)) + 0.5).astype(F32), k, 1)
    b = np.repeat((rng.random((n, 1)) + 0.5).astype(F32), rank, 1)
    x = np.repeat((rng.random((rows, 1)) + 0.5).astype(F32), k, 1)
    got, want, size = one_adapter(gh, TYPES[kind], a, b, x)
    assert (np.abs(got - want) <= 1e-5 * size).all(), (np.abs(got - want) / size).max()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", [2, 3, 100])
@pytest.mark.parametrize("where", ["x", "u", "a"])
def test_adapters_of_the_smallest_values(gh, kind, rows, where):
    """bf16 pieces reach down to 2^-133, so in tiles a value counts to half that; its partner's
    magnitudes and the other matrix make of it what they do."""
    import torch

    k, n, rank, rng = 136, 70, 16, np.random.default_rng(rows)
    a, b = (rng.standard_normal(s).astype(F32) for s in ((rank, k), (n, rank)))
    x = rng.standard_normal((rows, k)).astype(F32)
    scale = 1.0
    if where == "x":
        x, scale = x * F32(1e-36), 1e30
    elif where == "u":
        scale = 1e-36
    elif kind == "f16":
        a = a * F32(1e-7)
    else:
        a, scale = a * F32(1e-36), 1e30
    got, want, size = one_adapter(gh, TYPES[kind], a, b, x, scale)
    dt = {"f32": F32, "f16": np.float16}.get(kind)
    p, q = (torch.from_numpy(m).to(torch.bfloat16).double().numpy() if dt is None else
            m.astype(dt).astype(F64) for m in (a, b))
    s, step = F64(F32(scale)), 2.0 ** -134
    # halves of the last piece's step: of the inputs, of A (its pieces), of u
    floor = s * step * (np.abs(p).sum(1) + np.abs(x.astype(F64)).sum(1)[:, None]) @ np.abs(q).T
    floor += step * np.abs(q).sum(1)
    room = (math.sqrt(3 * k) + math.sqrt(3 * rank) + 8) * HALF
    assert (np.abs(got - want) <= room * size + 1.01 * floor).all()


# ---- workspaces ---------------------------------------------------------------------


@pytest.mark.gpu
def test_calls_of_one_launch_wait_for_no_other_s_workspace(gh):
    """Short rows' log probabilities and single tokens' small adapters write no workspace: without
    one of their own they go on while another thread waits for the library's to grow."""
    import torch

    from test_serving_limits import attention_call

    small, need0 = attention_call(gh, 1, [3000])
    large, need1 = attention_call(gh, 2, [4000] * 40)
    assert 0 < need0 < need1
    busy, free = torch.cuda.Stream(), torch.cuda.Stream()
    logits, h = torch.randn((2, 3000), device="cuda"), torch.zeros(2, device="cuda")
    x, out = torch.randn((2, 64), device="cuda"), torch.zeros((2, 24), device="cuda")
    a, b = torch.randn((1, 8, 64), device="cuda"), torch.randn((1, 24, 8), device="cuda")
    row0, ids = cuda(np.array([0, 1, 2], np.int32)), cuda(np.zeros(2, np.int32))
    ad = gemma_hip.adapters(row0, ids, None, 2, 2, 1, 1, 8, ADAPTER_F32)
    jobs = gemma_hip.adapter_jobs([(a, b, 24)])
    zeros = torch.zeros_like(out)

    def calls():
        gh.logprobs(gemma_hip.scores(entropy=h), logits, 0, 2, 3000, None, None, 0, 0, None,
                    free.cuda_stream)
        gh.adapters_add(out, 0, zeros, 0, ad, jobs, x, 0, 64, None, free.cuda_stream)

    m = torch.randn((8192, 8192), device="cuda")
    to = torch.empty_like(m)
    torch.mm(m, m, out=to)
    small(None, busy.cuda_stream)
    torch.cuda.synchronize()
    calls()
    torch.cuda.synchronize()
    want = h.clone(), out.clone()
    h.zero_()
    out.zero_()
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
    calls()
    early = not done.query()
    free.synchronize()
    t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert waiting, "the other thread's call was not waiting: this shows nothing"
    assert early, "a call that needs no workspace waited for another thread's"
    assert torch.equal(h, want[0]) and torch.equal(out, want[1])


@pytest.mark.gpu
def test_log_probabilities_of_two_launches_on_two_streams(gh):
    """The library's own workspaces are a stream's: rows that take two launches, and so one, on two
    streams at once."""
    import torch

    streams = [torch.cuda.Stream() for _ in range(2)]
    logits = [torch.randn((3, 40000 + i), device="cuda") for i in range(2)]

    def one(i, s):
        o = dict(entropy=torch.empty(3, device="cuda"),
                 top=torch.empty((3, 12), dtype=torch.int32, device="cuda"))
        gh.logprobs(gemma_hip.scores(**o), logits[i], 0, 3, 40000 + i, None, None, 0, 12, None, s)
        return [o["entropy"], o["top"]]

    want = [one(i, stream()) for i in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(40):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, one(i, s.cuda_stream)))
    torch.cuda.synchronize()
    for i, g in got:
        assert all(torch.equal(x, y) for x, y in zip(g, want[i]))
