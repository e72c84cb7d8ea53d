"""The operators between the products of a served batch, one by one and together: rotary
positions (gemma_hip_rope, gemma_hip_rotary_freqs), rows appended to the paged cache
(gemma_hip_cache_append), norms around the residual sum (gemma_hip_norm_residual), adapters
(gemma_hip_adapters_add) and log probabilities (gemma_hip_logprobs), against plain numpy in 64
bits.

Bars.  rope, append's queries and the norms are fp64 rounded to fp32 once: half a step, 2^-24 of
the value, and 1e-13 of the row's largest for the fp64 roundings of both sides.  Codes follow
from such values by the cache's and gemma_hip_quantize's definitions: equal.  Adapters: fp32 sums
of k and then rank products, each product off by at most 2^-23 and each partial sum rounded:
errors grow by the root of the number of terms at most (they are as often up as down), so
(sqrt(3 k) + sqrt(3 rank) + 8) 2^-24 of the sum of magnitudes.  Log probabilities: an
exponent x octaves off by 3 roundings of 2^-24 x moves a weight 2^x by ln 2 times that; x 2^x
averages at most the entropy, 19 octaves, so 2.4e-6 of the sum if all errors pointed one way, and
32 + 6 additions 1e-6 at most: 4e-6 of the larger of 1 and the value."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

import gemma_hip
from gemma_hip import (ADAPTER_BF16, ADAPTER_F16, ADAPTER_F32, CACHE_E4M3, CACHE_I8, NORM_LAYER,
                       NORM_NONE, NORM_RMS, ROPE_BANDS, ROPE_HALF, ROPE_LINEAR, ROPE_NONE, ROPE_NTK,
                       ROPE_PAIRS, ROPE_YARN)
from test_serving import KINDS, Paged, attend, cuda, quantise, stream, values

F32, F64 = np.float32, np.float64
EPS = 1e-6
HALF = 2.0 ** -24


# ---- the definitions, in numpy ------------------------------------------------


def frequencies(rot, theta, scaling, factor=1.0, original=0.0, low=1.0, high=32.0):
    """(frequencies, amplitude), pair by pair."""
    out = []
    if scaling == ROPE_NTK:
        theta = theta * factor ** (rot / (rot - 2))
    for j in range(rot // 2):
        f = theta ** (-2 * j / rot)
        if scaling == ROPE_LINEAR:
            f = f / factor
        elif scaling == ROPE_BANDS:
            turns = original * f / (2 * math.pi)
            if turns <= low:
                f = f / factor
            elif turns < high:
                s = (turns - low) / (high - low)
                f = (1 - s) * f / factor + s * f
        elif scaling == ROPE_YARN:
            a, b = (rot * math.log(original / (n * 2 * math.pi)) / (2 * math.log(theta))
                    for n in (high, low))
            a, b = max(0, math.floor(a)), min(rot - 1, math.ceil(b))
            s = min(1.0, max(0.0, (j - a) / max(b - a, 0.001)))
            f = f / factor * s + f * (1 - s)
        out.append(f)
    return np.array(out), 0.1 * math.log(factor) + 1 if scaling == ROPE_YARN else 1.0


def rms(x, w, eps=EPS):
    x = x.astype(F64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + F64(F32(eps))) * (w.astype(F64) + 1)


def turn(x, pos, freq, amp, layout, angle32=False):
    """Heads x [rows][heads][hdim], fp64."""
    x = np.array(x, F64)
    n = len(freq)
    if angle32:
        angle = (freq.astype(F32)[None, :] * pos.astype(F32)[:, None]).astype(F64)
        c, s = (f(angle).astype(F32).astype(F64) for f in (np.cos, np.sin))
    else:
        angle = freq[None, :] * pos.astype(F64)[:, None]
        c, s = np.cos(angle), np.sin(angle)
    c, s = (F64(F32(amp)) * t[:, None, :] for t in (c, s))
    one, two = (slice(0, n), slice(n, 2 * n)) if layout == ROPE_HALF else \
        (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    a, b = x[..., one].copy(), x[..., two].copy()
    x[..., one], x[..., two] = a * c - b * s, a * s + b * c
    return x


def normed(x, kind, w, b, offset, eps=EPS):
    x = x.astype(F64)
    if kind == NORM_NONE:
        return x
    if kind == NORM_LAYER:
        x = x - x.mean(-1, keepdims=True)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + F64(F32(eps)))
    return x * (1.0 if w is None else w.astype(F64) + offset) + (0.0 if b is None else b)


def once(got, want):
    """got, fp32, is `want` rounded once, but for fp64 roundings."""
    got = got.astype(F64)
    room = HALF * np.abs(want) + 1e-13 * np.abs(want).max(-1, keepdims=True)
    return bool((np.abs(got - want) <= room).all())


def describe(l, t, ids, n):
    """One row of logits: log p and ranks of ids, the entropy, the first n tokens and theirs."""
    l = np.where(np.isnan(l), -np.inf, l.astype(F64))
    order = np.argsort(-l, kind="stable")
    place = np.empty(len(l), int)
    place[order] = np.arange(len(l))
    p = np.full(len(l), -np.inf)
    top = l.max()
    if top > -np.inf:
        if not t > 0:
            p[order[0]] = 0.0
        elif top == np.inf:
            p[l == top] = -math.log((l == top).sum())
        else:
            z = (l - top) / t if not np.isinf(t) else np.where(l > -np.inf, 0.0, -np.inf)
            p = z - math.log(np.exp(z).sum())
    q = p[p > -np.inf]
    best = [i for i in order[:n] if l[i] > -np.inf]
    fill = n - len(best)
    there = [0 <= i < len(l) for i in ids]
    return (np.array([p[i] if ok else -np.inf for i, ok in zip(ids, there)]),
            np.array([place[i] + 1 if ok else 0 for i, ok in zip(ids, there)]),
            -(np.exp(q) * q).sum() if len(q) else 0.0,
            np.array(best + [-1] * fill), np.array([p[i] for i in best] + [-np.inf] * fill))


def close_logs(got, want):
    with np.errstate(over="ignore"):  # answers are fp32: -inf below its range
        got, want = np.asarray(got, F64), np.asarray(want, F64).astype(F32).astype(F64)
    fine = np.isfinite(want)
    return np.array_equal(got[~fine], want[~fine]) and \
        bool((np.abs(got[fine] - want[fine]) <= 4e-6 * np.maximum(1, np.abs(want[fine]))).all())


# ---- without a GPU ---------------------------------------------------------------


@pytest.mark.parametrize("scaling,more", [
    (ROPE_NONE, {}), (ROPE_LINEAR, dict(factor=8.0)), (ROPE_NTK, dict(factor=4.0)),
    (ROPE_BANDS, dict(factor=8.0, original=8192.0, low=1.0, high=4.0)),
    (ROPE_YARN, dict(factor=16.0, original=4096.0, low=1.0, high=32.0)),
    (ROPE_YARN, dict(factor=1.0, original=64.0, low=30.0, high=31.0))])
@pytest.mark.parametrize("rot,theta", [(4, 10000.0), (36, 1e6), (128, 5e5), (256, 10000.0)])
def test_frequencies(scaling, more, rot, theta):
    f, amp = gemma_hip.rotary_freqs(rot, theta, scaling, **more)
    want, wamp = frequencies(rot, theta, scaling, **more)
    np.testing.assert_allclose(f, want, rtol=1e-13)
    assert amp == F32(wamp)


def test_frequencies_are_the_reference_s():
    from oracle.decode_oracle import rope_table

    for theta in (10000.0, 1e6):
        f, _ = gemma_hip.rotary_freqs(256, theta)
        pos = np.array([0, 1, 77, 131071])
        c, s = rope_table(theta, 256, pos)
        x = np.stack([np.ones((4, 1, 128)), np.zeros((4, 1, 128))], 2).reshape(4, 1, 256)
        y = turn(x, pos, f, 1.0, ROPE_HALF, angle32=True)
        assert np.array_equal(y[:, 0, :128].astype(F32), c)
        assert np.array_equal(y[:, 0, 128:].astype(F32), s)


def test_bad_frequencies_are_refused():
    def freqs(rot=8, theta=1e4, scaling=ROPE_NONE, **kw):
        return gemma_hip.rotary_freqs(rot, theta, scaling, **kw)

    for kw, word in ((dict(rot=6), "turning"), (dict(rot=0), "turning"), (dict(theta=1.0), "theta"),
                     (dict(theta=math.nan), "theta"), (dict(theta=math.inf), "theta"),
                     (dict(scaling=5), "scaling"), (dict(scaling=ROPE_LINEAR, factor=0.5), "factor"),
                     (dict(scaling=ROPE_NTK, factor=math.nan), "factor"),
                     (dict(scaling=ROPE_BANDS, factor=2.0, original=0.0), "bounds"),
                     (dict(scaling=ROPE_YARN, factor=2.0, original=64.0, low=2.0, high=2.0),
                      "bounds")):
        with pytest.raises(gemma_hip.GemmaHipError, match=word):
            freqs(**kw)


def test_definitions_catch_planted_mistakes():
    rng = np.random.default_rng(0)
    x, pos = rng.standard_normal((3, 2, 16)), np.array([1, 50, 1000])
    f, _ = frequencies(8, 1e4, ROPE_NONE)
    want = turn(x, pos, f, 1.0, ROPE_HALF)
    assert once(want.astype(F32), want)
    for other in (turn(x, pos, f, 1.0, ROPE_PAIRS), turn(x, pos + 1, f, 1.0, ROPE_HALF),
                  turn(x, pos, f, 1.001, ROPE_HALF), turn(x, pos, f * (1 + 1e-6), 1.0, ROPE_HALF)):
        assert not once(other.astype(F32), want)
    l = np.array([1.0, 3.0, 3.0, -np.inf, np.nan, 2.0])
    logp, rank, h, top, tl = describe(l, 1.0, [2, 1, 3, 9], 6)
    assert list(rank) == [2, 1, 5, 0] and list(top) == [1, 2, 5, 0, -1, -1]
    assert logp[0] == logp[1] == tl[0] and logp[2] == logp[3] == -np.inf and h > 0


def fake(off=0):
    """An address that no refused call reads."""
    return (1 << 20) + off


def refused(call, word):
    lib = gemma_hip.load()
    assert call(lib) == 1
    msg = lib.gemma_hip_last_error().decode()
    assert word in msg, msg


def test_bad_rotations_are_refused():
    def rope(lib, dst=fake(), ds=512, src=fake(), ss=512, rows=3, heads=2, hdim=256, pos=fake(),
             norm=None, rot=None):
        r = gemma_hip.Rotary(fake(), 256, ROPE_HALF, 0, 1.0) if rot is None else rot
        return lib.gemma_hip_rope(dst, ds, src, ss, rows, heads, hdim, pos, norm, EPS, r, None)

    R = gemma_hip.Rotary
    for kw, word in ((dict(dst=None), "null"), (dict(src=fake(4)), "aligned"), (dict(ds=508), "stride"),
                     (dict(ss=514), "multiple"), (dict(rows=-1), "shape"), (dict(heads=0), "shape"),
                     (dict(hdim=258), "shape"), (dict(hdim=260), "shape"), (dict(pos=None), "positions"),
                     (dict(rows=1 << 25, heads=2), "shape"), (dict(norm=fake(8)), "aligned"),
                     (dict(rot=R(fake(), 6, 0, 0, 1.0)), "turning"),
                     (dict(rot=R(fake(), 260, 0, 0, 1.0)), "turning"),
                     (dict(rot=R(fake(), -4, 0, 0, 1.0)), "turning"),
                     (dict(rot=R(fake(), 8, 2, 0, 1.0)), "layout"),
                     (dict(rot=R(None, 8, 0, 0, 1.0)), "frequencies"),
                     (dict(rot=R(fake(4), 8, 0, 0, 1.0)), "frequencies")):
        refused(lambda lib: rope(lib, **kw), word)
    refused(rope, "not initialised")


def test_bad_appends_are_refused():
    def append(lib, cache=(), batch=(), null=False, **kw):
        c = gemma_hip.cache(fake(), fake(), fake(), fake(), CACHE_I8, 4, 16, 1, 128)
        b = gemma_hip.batch(fake(), fake(), fake(), 2, 2, 5, 4, 30)
        for name, value in cache:
            setattr(c, name, value)
        for name, value in batch:
            setattr(b, name, value)
        a = dict(q=fake(), qs=256, k=fake(), ks=128, v=fake(), vs=128, o=fake(), os=256, n=2,
                 nq=None, nk=None, rot=gemma_hip.Rotary(fake(), 128, 0, 0, 1.0))
        a.update(kw)
        h = gemma_hip.heads(a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["o"], a["os"],
                            a["n"], a["nq"], a["nk"], EPS, a["rot"])
        return lib.gemma_hip_cache_append(c, b, None if null else h, None)

    for kw, word in ((dict(null=True), "null"), (dict(k=None), "null"), (dict(v=fake(8)), "aligned"),
                     (dict(ks=124), "stride"), (dict(q=None), "null"), (dict(o=None), "null"),
                     (dict(os=258), "multiple"), (dict(n=0), "heads"), (dict(n=1025), "heads"),
                     (dict(nk=fake(4)), "aligned"), (dict(cache=[("type", 3)]), "type"),
                     (dict(cache=[("hdim", 64)]), "cache"), (dict(batch=[("rows", 3)]), "batch"),
                     (dict(batch=[("rows", 1 << 25)]), "too many"),
                     (dict(batch=[("len", None)]), "null"),
                     (dict(rot=gemma_hip.Rotary(fake(), 132, 0, 0, 1.0)), "turning")):
        refused(lambda lib: append(lib, **kw), word)
    refused(append, "not initialised")


def test_bad_norms_are_refused():
    def call(lib, rows=3, dim=64, null=False, **kw):
        a = dict(x=fake(), y=fake(), before=gemma_hip.norm(NORM_RMS, fake()), h=fake())
        a.update(kw)
        return lib.gemma_hip_norm_residual(None if null else gemma_hip.residual(**a), rows, dim, None)

    for kw, word in ((dict(null=True), "null"), (dict(rows=-1), "shape"), (dict(dim=66), "shape"),
                     (dict(dim=0), "shape"), (dict(dim=24580), "shape"), (dict(x=None), "null"),
                     (dict(rows=(1 << 21) + 1), "shape"), (dict(y=fake(4)), "aligned"), (dict(x_stride=60), "stride"),
                     (dict(gate=fake(8)), "aligned"), (dict(h=fake(4)), "aligned"),
                     (dict(x_out=fake(), x_out_stride=66), "multiple"),
                     (dict(hq=fake()), "together"), (dict(hs=fake()), "together"),
                     (dict(hq=fake(2), hs=fake()), "aligned"),
                     (dict(hq=fake(), hs=fake(), hq_stride=62), "stride"),
                     (dict(before=gemma_hip.norm(3)), "norm"),
                     (dict(after=gemma_hip.norm(NORM_LAYER, fake(), fake(4))), "aligned")):
        refused(lambda lib: call(lib, **kw), word)
    refused(call, "not initialised")


def test_bad_adapters_are_refused():
    lib = gemma_hip.load()

    def call(lib, ad=(), jobs=((fake(), fake(), 40),), dst=fake(), ds=0, base=fake(), bs=0,
             src=fake(), ss=0, k=64, null=False):
        a = gemma_hip.adapters(fake(), fake(), fake(), 2, 5, 4, 3, 16, ADAPTER_BF16)
        for name, value in ad:
            setattr(a, name, value)
        return lib.gemma_hip_adapters_add(dst, ds, base, bs, None if null else a,
                                          gemma_hip.adapter_jobs(jobs), len(jobs), src, ss, k, None,
                                          0, None)

    j = (fake(), fake(), 40)
    for kw, word in ((dict(null=True), "null"), (dict(jobs=(j, j, j, j)), "shape"),
                     (dict(jobs=((None, fake(), 40),)), "null"), (dict(jobs=((fake(), fake(), 0),)), "shape"),
                     (dict(jobs=((fake(8), fake(), 40),)), "aligned"), (dict(k=60), "shape"),
                     (dict(k=0), "shape"), (dict(ad=[("rank", 12)]), "rank"),
                     (dict(ad=[("rank", 136)]), "rank"), (dict(ad=[("rank", 0)]), "rank"),
                     (dict(ad=[("type", 3)]), "type"), (dict(ad=[("rows", 3)]), "batch"),
                     (dict(ad=[("rows", 1 << 23)]), "batch"), (dict(ad=[("count", -1)]), "batch"),
                     (dict(ad=[("ids", None)]), "null"), (dict(dst=None), "null"),
                     (dict(ds=39), "stride"), (dict(bs=39), "stride"), (dict(src=fake(4)), "aligned"),
                     (dict(ss=66), "multiple")):
        refused(lambda lib: call(lib, **kw), word)
    refused(call, "not initialised")
    a = gemma_hip.adapters(fake(), fake(), fake(), 2, 5, 4, 3, 12, ADAPTER_BF16)
    assert lib.gemma_hip_adapters_work(a, 1, 64) == ctypes.c_size_t(-1).value


def test_bad_logits_are_refused():
    lib = gemma_hip.load()

    def call(lib, l=fake(), stride=0, rows=2, vocab=100, ids=fake(), nt=1, n=5, null=False):
        return lib.gemma_hip_logprobs(None if null else gemma_hip.scores(), l, stride, rows, vocab,
                                      None, ids, nt, n, None, 0, None)

    for kw, word in ((dict(null=True), "null"), (dict(l=None), "null"), (dict(ids=None), "null"),
                     (dict(stride=99), "stride"), (dict(rows=-1), "shape"), (dict(rows=65536), "shape"),
                     (dict(vocab=0), "shape"), (dict(vocab=(1 << 19) + 1), "shape"),
                     (dict(nt=65), "tokens"), (dict(nt=-1), "tokens"), (dict(n=65), "tokens"),
                     (dict(n=-1), "tokens")):
        refused(lambda lib: call(lib, **kw), word)
    refused(call, "not initialised")
    assert lib.gemma_hip_logprobs_work(1, 100, 65, 0) == ctypes.c_size_t(-1).value


# ---- rotary positions ---------------------------------------------------------


ROPES = [  # rows, heads, hdim, rot, layout, norm, angle32, stride
    (1, 1, 4, 4, ROPE_HALF, False, False, 0), (3, 2, 64, 64, ROPE_PAIRS, True, False, 0),
    (5, 3, 72, 36, ROPE_HALF, True, False, 220), (7, 5, 128, 128, ROPE_HALF, False, True, 0),
    (33, 4, 256, 256, ROPE_HALF, True, False, 1032), (2, 7, 96, 0, ROPE_HALF, True, False, 0),
    (9, 1, 256, 64, ROPE_PAIRS, True, True, 0), (40, 3, 68, 68, ROPE_PAIRS, False, False, 0),
    (6000, 3, 128, 64, ROPE_HALF, True, False, 384), (4099, 5, 256, 256, ROPE_PAIRS, True, False, 0),
    (1500, 17, 32, 32, ROPE_HALF, True, False, 0),
    (9000, 4, 64, 64, ROPE_HALF, True, True, 0), (5003, 7, 64, 16, ROPE_PAIRS, False, False, 452),
    (3001, 6, 256, 0, ROPE_HALF, True, False, 0), (8203, 3, 128, 96, ROPE_PAIRS, True, False, 0),
    (2601, 5, 256, 128, ROPE_HALF, True, True, 1284), (9001, 4, 64, 32, ROPE_HALF, False, False, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ROPES, ids=str)
def test_rope(gh, case):
    import torch

    rows, heads, hdim, rot, layout, norm, angle32, stride = case
    rng = np.random.default_rng(1)
    width = heads * hdim
    x = rng.standard_normal((rows, stride or width)).astype(F32)
    pos = rng.integers(-5, 131072, rows).astype(np.int32)
    pos[:2] = (0, 1 << 30)[:rows]
    w = (rng.standard_normal(hdim) * 0.2).astype(F32) if norm else None
    f, _ = gemma_hip.rotary_freqs(max(4, rot), 10000.0)
    r = gemma_hip.rotary(cuda(f), rot, layout, 1.25, angle32)
    y = x[:, :width].reshape(rows, heads, hdim)
    y = turn(rms(y, w) if norm else y, pos, f[:rot // 2], 1.25, layout, angle32)
    src, dst, dw = cuda(x), torch.full((rows, stride or width), 9.0, device="cuda"), \
        cuda(w) if norm else None
    for a, b in ((dst, src), (src, src)):  # into another buffer, and in place
        gh.rope(a, stride, b, stride, rows, heads, hdim, cuda(pos), dw, EPS, r, stream())
        got = a.cpu().numpy()
        assert once(got[:, :width].reshape(rows, heads, hdim), y)
        if stride:
            assert np.array_equal(got[:, width:], x[:, width:] if a is src else
                                  np.full_like(got[:, width:], 9.0))


@pytest.mark.gpu
def test_rope_keeps_what_is_not_finite_in_its_place(gh):
    x = np.ones((3, 2, 64), F32)
    x[0, 0, 5], x[1, 1, 40], x[2, 0, 63] = np.nan, np.inf, np.inf
    f, _ = gemma_hip.rotary_freqs(32, 10000.0)
    r = gemma_hip.rotary(cuda(f), 32, ROPE_HALF)
    dx, pos = cuda(x), cuda(np.array([3, 4, 5], np.int32))
    gh.rope(dx, 0, dx, 0, 3, 2, 64, pos, None, 0.0, r, stream())
    got = dx.cpu().numpy()
    bad = ~np.isfinite(got)
    assert sorted(map(tuple, np.argwhere(bad))) == [(0, 0, 5), (0, 0, 21), (1, 1, 40), (2, 0, 63)]
    dx, w = cuda(x), cuda(np.zeros(64, F32))
    gh.rope(dx, 0, dx, 0, 3, 2, 64, pos, w, EPS, r, stream())
    got = dx.cpu().numpy()
    assert np.isnan(got[0, 0]).all() and np.isfinite(got[0, 1]).all()
    assert np.isnan(got[1, 1, 40]) and (got[1, 1, 48:] == 0).all()  # the others over infinity


# ---- rows into the cache -------------------------------------------------------


APPENDS = {  # sequences (new rows, positions), q heads, kv heads, head dim, page, rot, layout, norm
    "one": ([(1, 1)], 1, 1, 128, 16, 128, ROPE_HALF, True),
    "steps": ([(1, 17), (1, 16), (1, 200), (1, 33)], 4, 1, 256, 16, 256, ROPE_HALF, True),
    "ragged": ([(3, 40), (0, 9), (17, 17), (1, 63), (0, 0), (30, 100)], 3, 1, 128, 32, 64,
               ROPE_PAIRS, True),
    "short": ([(5, 2), (4, 4), (3, 0)], 2, 2, 256, 16, 128, ROPE_HALF, True),
    "keys": ([(2, 70), (1, 30)], 0, 2, 128, 64, 128, ROPE_HALF, True),
    "plain": ([(9, 50)], 8, 4, 256, 64, 0, ROPE_HALF, False),
    "many": ([(1 + b % 3, 3 + b % 20) for b in range(200)], 2, 1, 128, 16, 128, ROPE_PAIRS, False),
    "prompt": ([(1500, 1600), (1, 5)], 8, 4, 256, 64, 256, ROPE_HALF, True),
    "prompt128": ([(2100, 2100)], 7, 1, 128, 256, 128, ROPE_PAIRS, True),
    "chunks": ([(1 + b % 19, 2 + b % 23) for b in range(220)], 7, 1, 128, 16, 64, ROPE_HALF, True),
    "chunks256": ([(40 + b, 45 + 3 * b % 70) for b in range(12)], 4, 2, 256, 32, 64, ROPE_PAIRS,
                  True),
    "keys256": ([(700, 800), (0, 5), (900, 900)], 0, 4, 256, 64, 256, ROPE_HALF, False),
}


def append_inputs(case, kind, seed, extra=3):
    seqs, nq, kv, hd, page, rot, layout, norm = case
    rng = np.random.default_rng(seed)
    p = Paged(seqs, kv, hd, page, kind, rng)
    rows = p.rows + extra  # some behind the last sequence
    x = rng.standard_normal((rows, (nq + 2 * kv) * hd)).astype(F32)
    wq, wk = ((rng.standard_normal(hd) * 0.2).astype(F32) if norm else None for _ in "qk")
    f, _ = gemma_hip.rotary_freqs(max(4, rot), 10000.0)
    return p, rows, x, wq, wk, f


def append_expected(case, p, x, wq, wk, f):
    """q's rows, and the cache's codes and scales after the call (in p)."""
    seqs, nq, kv, hd, page, rot, layout, norm = case
    pos = np.concatenate([np.arange(ln - n, ln) for n, ln in seqs]).astype(int)
    seq = np.repeat(np.arange(len(seqs)), [n for n, _ in seqs])
    y = x[:p.rows].reshape(p.rows, nq + 2 * kv, hd)

    def head(y, w):
        return turn(rms(y, w) if w is not None else y, pos, f[:rot // 2], 1.0, layout)

    k = head(y[:, nq:nq + kv], wk).astype(F32)
    v = y[:, nq + kv:]
    for r in range(p.rows):
        if pos[r] >= 0:
            for h in range(kv):
                p.put(seq[r], pos[r], k[r, h], h, "k")
                p.put(seq[r], pos[r], v[r, h], h, "v")
    return head(y[:, :nq], wq).reshape(p.rows, nq * hd)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("name", APPENDS)
def test_append(gh, name, kind):
    import torch

    case, kind = APPENDS[name], KINDS[kind]
    seqs, nq, kv, hd, page, rot, layout, norm = case
    p, rows, x, wq, wk, f = append_inputs(case, kind, 2)
    if name == "ragged":
        p.table[3, 1] = -1  # a page that isn't there
    if name in ("chunks", "keys256"):
        p.table[2, 0] = 1 << 30
    c, b = p.device(), None
    b = p.batch(rows=rows)
    dx, wqd, wkd = cuda(x), None if wq is None else cuda(wq), None if wk is None else cuda(wk)
    n = x.shape[1]
    q = torch.full((rows, max(1, nq * hd)), 5.0, device="cuda")
    heads = gemma_hip.heads(dx if nq else None, n, dx[:, nq * hd:], n, dx[:, (nq + kv) * hd:], n,
                            q if nq else None, 0, nq, wqd, wkd, EPS,
                            gemma_hip.rotary(cuda(f), rot, layout))
    gh.cache_append(c, b, heads, stream())
    want = append_expected(case, p, x, wq, wk, f)
    got = q.cpu().numpy()
    if nq:
        assert once(got[:p.rows].reshape(p.rows, nq, hd), want.reshape(p.rows, nq, hd))
    assert (got[p.rows:] == 5.0).all()
    for x_ in "kv":
        assert np.array_equal(p.d[x_][0].cpu().numpy(), p.codes[x_])
        assert np.array_equal(p.d[x_][1].cpu().numpy(), p.scales[x_], equal_nan=True)
    assert np.array_equal(dx.cpu().numpy(), x)


@pytest.mark.gpu
def test_append_is_rope_and_write(gh):
    """To the bit, with q in place in the products' buffer."""
    import torch

    case = APPENDS["ragged"]
    seqs, nq, kv, hd, page, rot, layout, norm = case
    p, rows, x, wq, wk, f = append_inputs(case, CACHE_I8, 3, extra=0)
    c, b = p.device(), p.batch()
    pos = cuda(np.concatenate([np.arange(ln - n, ln) for n, ln in seqs]).astype(np.int32))
    r = gemma_hip.rotary(cuda(f), rot, layout)
    dx, n, wq, wk = cuda(x), x.shape[1], cuda(wq), cuda(wk)
    gh.rope(dx, n, dx, n, rows, nq, hd, pos, wq, EPS, r, stream())
    gh.rope(dx[:, nq * hd:], n, dx[:, nq * hd:], n, rows, kv, hd, pos, wk, EPS, r, stream())
    gh.cache_write(c, b, dx[:, nq * hd:], n, dx[:, (nq + kv) * hd:], n, stream())
    want = [dx[:, :nq * hd].clone()] + [t.clone() for x_ in "kv" for t in p.d[x_]]
    c, dx = p.device(), cuda(x)
    gh.cache_append(c, b, gemma_hip.heads(dx, n, dx[:, nq * hd:], n, dx[:, (nq + kv) * hd:], n, dx,
                                          n, nq, wq, wk, EPS, r), stream())
    for g, w in zip([dx[:, :nq * hd]] + [t for x_ in "kv" for t in p.d[x_]], want):
        assert torch.equal(g.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8))
    assert np.array_equal(dx[:, nq * hd:].cpu().numpy(), x[:, nq * hd:])


@pytest.mark.gpu
def test_append_of_rows_that_are_not_finite(gh):
    """Codes of 0 and a NaN scale for their heads, the others as they are."""
    case = APPENDS["steps"]
    seqs, nq, kv, hd, page, rot, layout, norm = case
    p, rows, x, wq, wk, f = append_inputs(case, CACHE_E4M3, 4, extra=0)
    at = nq * hd
    x[0, at + 7], x[1, at + kv * hd + 3], x[2, at:at + hd] = np.nan, np.inf, 0.0
    c, b, dx, n = p.device(), p.batch(), cuda(x), x.shape[1]
    heads = gemma_hip.heads(None, 0, dx[:, at:], n, dx[:, at + kv * hd:], n, None, 0, 0, None,
                            cuda(wk), EPS, gemma_hip.rotary(cuda(f), rot, layout))
    gh.cache_append(c, b, heads, stream())
    append_expected(case, p, x, wq, wk, f)
    for x_ in "kv":
        assert np.array_equal(p.d[x_][0].cpu().numpy(), p.codes[x_])
        assert np.array_equal(p.d[x_][1].cpu().numpy(), p.scales[x_], equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,layout", [(128, ROPE_HALF), (256, ROPE_PAIRS)])
def test_many_rows_of_any_size_of_values(gh, kind, hd, layout):
    """Heads of zeros, subnormals, values at both ends of fp32, NaN and infinities among many rows:
    codes and scales to the bit those of rope and cache_write, other heads untouched by them."""
    import torch

    nq, kv, page, n = 3, 2, 64, 3000
    rng = np.random.default_rng(17)
    x = rng.standard_normal((n, nq + 2 * kv, hd)).astype(F32)
    sizes = np.array([1.0, 0.0, 1e-42, 1e-39, 1e-36, 1e-31, 1e-29, 1e30, 3e37], F32)
    x *= rng.choice(sizes, (n, nq + 2 * kv, 1))
    bad = rng.random((n, nq + 2 * kv)) < 0.1
    x[bad, 5] = rng.choice(np.array([np.nan, np.inf, -np.inf], F32), bad.sum())
    f, _ = gemma_hip.rotary_freqs(hd, 10000.0)
    r = gemma_hip.rotary(cuda(f), hd, layout)
    w = (nq + 2 * kv) * hd
    p = Paged([(n, n)], kv, hd, page, KINDS[kind], rng)
    pos = cuda(np.arange(n, dtype=np.int32))
    out = []
    for one in (False, True):
        c, b, dx = p.device(), p.batch(), cuda(x.reshape(n, w))
        if one:
            gh.cache_append(c, b, gemma_hip.heads(dx, w, dx[:, nq * hd:], w, dx[:, (nq + kv) * hd:],
                                                  w, dx, w, nq, None, None, EPS, r), stream())
            out.append([dx[:, :nq * hd].contiguous()])
        else:  # 64 rows at a time: by the kernel of few rows
            for i in range(0, n, 64):
                m = min(64, n - i)
                gh.rope(dx[i:], w, dx[i:], w, m, nq + kv, hd, pos[i:], None, EPS, r, stream())
            gh.cache_write(c, b, dx[:, nq * hd:], w, dx[:, (nq + kv) * hd:], w, stream())
            out.append([dx[:, :nq * hd].contiguous()])
        out[-1] += [t.clone() for k in "kv" for t in p.d[k]]
    for a, b in zip(*out):
        same = a.contiguous().view(torch.uint8) == b.contiguous().view(torch.uint8)
        if a.dtype == torch.float32:  # NaN is NaN
            same = same.view(*a.shape, 4).all(-1) | (a.isnan() & b.isnan())
        assert same.all()


@pytest.mark.gpu
def test_append_behind_four_gigabytes(gh):
    """Codes of pages whose addresses pass 32 bits, by one row and by many."""
    import torch

    kv, hd, page, npages = 4, 256, 64, 70000  # 4.6e9 codes of keys
    codes = torch.zeros((2, npages, kv, page, hd), dtype=torch.int8, device="cuda")
    scales = torch.zeros((2, npages, kv, page), device="cuda")
    c = gemma_hip.cache(codes[0], codes[1], scales[0], scales[1], CACHE_I8, npages, page, kv, hd)
    for n in (1, 1024):
        pages = -(-n // page)
        table = torch.arange(npages - pages, npages, device="cuda", dtype=torch.int32)[None]
        row0 = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        b = gemma_hip.batch(table, row0[1:], row0, 1, pages, n, n, n)
        x = torch.randn((n, 2 * kv * hd), device="cuda")
        gh.cache_append(c, b, gemma_hip.heads(None, 0, x, 2 * kv * hd, x[:, kv * hd:], 2 * kv * hd,
                                              None, 0, 0), stream())
        for i in range(2):
            got = codes[i, npages - pages:].float() * scales[i, npages - pages:, :, :, None]
            got = got.permute(0, 2, 1, 3).reshape(-1, kv * hd)[:n]
            off = (got - x[:, i * kv * hd:(i + 1) * kv * hd]).abs().view(n, kv, hd).amax(-1)
            # half a step, which is 1/127 of the head's largest, and six roundings of 2^-24 of up to
            # 127 steps (127 / amax, its product, the half added; 1 / 127, its product, the value's):
            # 6 * 127 * 2^-24 = 4.54e-5 steps, 9.1e-5 of half a step
            top = x[:, i * kv * hd:(i + 1) * kv * hd].abs().view(n, kv, hd).amax(-1)
            assert (off <= top / 254 * (1 + 9.1e-5)).all()
        assert not codes[:, :1000].any()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 62, 63, 64, 65, 200, 4000, 10000])
def test_rows_find_their_sequences(gh, batch):
    """Single rows, none and several, in batches around the search's steps."""
    import torch

    rng = np.random.default_rng(batch)
    n = rng.choice([0, 1, 1, 1, 2], batch)
    n[-1] = max(1, n[-1])
    ln = n + rng.integers(0, 3, batch)
    row0 = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    rows = int(row0[-1])
    kv, hd, page = 1, 128, 16
    codes = torch.zeros((2, batch, kv, page, hd), dtype=torch.int8, device="cuda")
    scales = torch.full((2, batch, kv, page), -1.0, device="cuda")
    c = gemma_hip.cache(codes[0], codes[1], scales[0], scales[1], CACHE_I8, batch, page, kv, hd)
    table = cuda(np.arange(batch, dtype=np.int32)[:, None])
    b = gemma_hip.batch(table, cuda(ln.astype(np.int32)), cuda(row0), batch, 1, rows, max(n), 5)
    x = torch.arange(1, rows + 1, device="cuda", dtype=torch.float32)[:, None].repeat(1, hd)
    gh.cache_append(c, b, gemma_hip.heads(None, 0, x, 0, x, 0, None, 0, 0), stream())
    got = scales.cpu().numpy()[:, :, 0]
    want = np.full((batch, page), -1.0, F32)
    for i in range(batch):
        for j in range(n[i]):
            want[i, ln[i] - n[i] + j] = F32(row0[i] + j + 1) * F32(1 / 127)
    assert np.array_equal(got[0], want) and np.array_equal(got[1], want)


# ---- norms and the residual sum ---------------------------------------------------


NORMS = [  # rows, dim, after, before, gate, stride
    (1, 4, NORM_RMS, NORM_RMS, None, 0), (3, 208, NORM_RMS, NORM_RMS, "rows", 216),
    (2, 1152, NORM_RMS, NORM_RMS, None, 0), (5, 1152, NORM_NONE, NORM_LAYER, "one", 1160),
    (700, 640, NORM_LAYER, NORM_RMS, "rows", 0), (4, 2564, NORM_RMS, NORM_LAYER, None, 0),
    (3, 6144, NORM_LAYER, NORM_LAYER, "one", 0), (2, 6148, NORM_RMS, NORM_RMS, "rows", 6152),
    (2, 24576, NORM_RMS, NORM_RMS, None, 0), (9, 512, NORM_NONE, NORM_NONE, None, 0),
    (3000, 256, NORM_RMS, NORM_RMS, None, 0), (1101, 704, NORM_LAYER, NORM_RMS, "rows", 712),
    (1030, 768, NORM_RMS, NORM_LAYER, "one", 0), (1027, 772, NORM_LAYER, NORM_LAYER, "rows", 0),
    (1300, 1152, NORM_RMS, NORM_RMS, "one", 1160), (1026, 1536, NORM_NONE, NORM_LAYER, None, 0),
    (1025, 2560, NORM_RMS, NORM_RMS, "rows", 0), (2, 5000, NORM_RMS, NORM_RMS, "one", 0),
    (2, 17000, NORM_LAYER, NORM_RMS, "rows", 0), (4100, 208, NORM_RMS, NORM_RMS, None, 216)]


def codes_of_rows(h):
    """gemma_hip_quantize of rows h: codes, and scales that are 1 for zeros."""
    code, scale = quantise(h, CACHE_I8)
    return code.view(np.int8), np.where(np.abs(h).max(-1) == 0, F32(1), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("case", NORMS, ids=str)
def test_norm_residual(gh, case):
    import torch

    rows, dim, after, before, gate, stride = case
    rng = np.random.default_rng(5)
    n = stride or dim
    x, y = (rng.standard_normal((rows, n)).astype(F32) * s for s in (3, 1))
    g = {"rows": rng.standard_normal((rows, n)).astype(F32),
         "one": rng.standard_normal((1, n)).astype(F32), None: None}[gate]
    w0, w1, b0, b1 = ((rng.standard_normal(dim) * 0.2).astype(F32) for _ in range(4))
    if rows > 2:
        x[1] = y[1] = 0.0
    args = dict(x_scale=0.5, y_scale=1.5, x_stride=stride, y_stride=stride, gate_stride=stride,
                gate_one=gate == "one", after=gemma_hip.norm(after, cuda(w0), cuda(b0), 1.0),
                before=gemma_hip.norm(before, cuda(w1), None, 0.0))
    z = normed(y[:, :dim], after, w0, b0, 1.0)
    want = 0.5 * x[:, :dim].astype(F64) + 1.5 * (1 if g is None else g[:, :dim].astype(F64)) * z
    dx, dy, dg = cuda(x), cuda(y), None if g is None else cuda(g)
    out, h = torch.full((2, rows, n), 7.0, device="cuda").unbind(0)
    hq = torch.full((rows, n), 7, dtype=torch.int8, device="cuda")
    hs = torch.zeros(rows, device="cuda")
    gh.norm_residual(gemma_hip.residual(dx, dy, dg, x_out=out, h=h, hq=hq, hs=hs,
                                        x_out_stride=stride, h_stride=stride, hq_stride=stride,
                                        **args), rows, dim, stream())
    got, hh, codes = out.cpu().numpy(), h.cpu().numpy(), hq.cpu().numpy()
    assert once(got[:, :dim], want)
    hw = normed(got[:, :dim], before, w1, None, 0.0)
    assert once(hh[:, :dim], hw)
    code, scale = codes_of_rows(hh[:, :dim])
    assert np.array_equal(codes[:, :dim], code) and np.array_equal(hs.cpu().numpy(), scale)
    if stride:
        assert (got[:, dim:] == 7).all() and (hh[:, dim:] == 7).all() and (codes[:, dim:] == 7).all()
    # in place, the norm alone: the same bits
    gh.norm_residual(gemma_hip.residual(dx, dy, dg, x_out=dx, x_out_stride=stride, **args), rows,
                     dim, stream())
    assert torch.equal(dx[:, :dim], out[:, :dim])
    h2 = torch.empty_like(h)
    only = dict(before=args["before"], x_stride=stride, h_stride=stride)
    gh.norm_residual(gemma_hip.residual(dx, h=h2, **only), rows, dim, stream())
    assert torch.equal(h2[:, :dim], h[:, :dim])


@pytest.mark.gpu
def test_norms_are_the_quantiser_s_and_the_decoder_s(gh):
    """Codes equal to gemma_hip_quantize's of the same rows."""
    import torch

    rows, dim = 40, 1152
    x = torch.randn((rows, dim), device="cuda") * 5
    w = torch.randn(dim, device="cuda") * 0.1
    h = torch.empty_like(x)
    hq, q = (torch.empty((rows, dim), dtype=torch.int8, device="cuda") for _ in "ab")
    hs, s = torch.empty((2, rows), device="cuda").unbind(0)
    gh.norm_residual(gemma_hip.residual(x, before=gemma_hip.norm(NORM_RMS, w, None, 1.0), h=h, hq=hq,
                                        hs=hs), rows, dim, stream())
    gh.quantize(q, s, h, dim, rows, dim, stream())
    assert torch.equal(q, hq) and torch.equal(s, hs)


@pytest.mark.gpu
def test_norm_residual_at_the_ends_of_fp32(gh):
    import torch

    big = 3.0e38
    x = np.full((5, 8), 1.0, F32)
    x[0], x[1, 2], x[2, 3], x[3], x[4] = big, np.nan, np.inf, 1e-30, 0.0
    y = x.copy()
    dx, h = cuda(x), torch.empty((5, 8), device="cuda")
    out, hs = torch.empty_like(h), torch.empty(5, device="cuda")
    hq = torch.empty((5, 8), dtype=torch.int8, device="cuda")
    gh.norm_residual(gemma_hip.residual(dx, cuda(y), x_out=out, h=h, hq=hq, hs=hs,
                                        before=gemma_hip.norm(NORM_RMS, eps=0.0)), 5, 8, stream())
    got, gh_, q, s = out.cpu().numpy(), h.cpu().numpy(), hq.cpu().numpy(), hs.cpu().numpy()
    top = np.finfo(F32).max
    assert (got[0] == top).all() and np.isnan(got[1, 2]) and got[2, 3] == top
    assert np.allclose(gh_[0], 1) and np.allclose(gh_[3], 1)
    assert np.isnan(gh_[1]).all() and np.isnan(s[1]) and not q[1].any()
    assert np.isfinite(gh_[2]).all() and q[2, 3] == 127
    assert np.isnan(gh_[4]).all() and np.isnan(s[4]) and not q[4].any()  # 0 / 0


# ---- adapters -------------------------------------------------------------------


TYPES = {"f32": ADAPTER_F32, "bf16": ADAPTER_BF16, "f16": ADAPTER_F16}
ADAPTERS = {  # rows of the sequences, k, outputs, rank, adapters
    "one": ([1], 8, [1], 8, 1), "steps": ([1] * 7, 208, [40, 17, 3], 16, 3),
    "spread": ([1] * 70, 1152, [256, 128], 8, 5), "odd": ([5, 0, 33, 1, 2], 136, [67], 24, 2),
    "wide": ([17, 64], 640, [300, 44, 8], 64, 2), "most": ([130], 72, [515], 128, 1),
    "prompts": ([300, 77, 0, 260], 2560, [512, 256, 256], 16, 3),
    "long": ([40], 10240, [65], 32, 2), "few": ([3, 4, 2], 1152, [1024, 256, 256], 16, 4),
    "three": ([900, 700], 264, [64, 100, 64], 16, 2), "two": ([300, 270], 200, [96, 40], 64, 2),
    "tiles": ([1 + i * 7 % 40 for i in range(90)], 72, [70, 3], 40, 4),
    "rank128": ([20, 3], 136, [130, 64], 128, 2), "tokens128": ([1] * 5, 200, [70, 130], 128, 3),
    "tokens32": ([1] * 6, 2560, [1024, 512, 512], 32, 3), "tokens16": ([1, 2], 6912, [1152], 16, 2),
    "more128": ([2, 1], 1152, [700, 30], 128, 2), "small128": ([1, 2], 72, [40], 128, 1),
    "pairs": ([1, 2, 0, 1], 1000, [65], 24, 2), "tall": ([129, 65, 64], 512, [129], 72, 2),
}


def adapter_inputs(case, kind, seed, device="cuda"):
    import torch

    rows, k, ns, rank, count = case
    g = torch.Generator().manual_seed(seed)
    dt = {ADAPTER_F32: torch.float32, ADAPTER_BF16: torch.bfloat16, ADAPTER_F16: torch.float16}[kind]
    a = [torch.randn((count, rank, k), generator=g).to(dt) for _ in ns]
    b = [torch.randn((count, n, rank), generator=g).to(dt) for n in ns]
    total = sum(rows)
    x, base = torch.randn((total, k), generator=g), torch.randn((total, sum(ns)), generator=g)
    scale = torch.rand(count, generator=g) + 0.5
    ids = np.random.default_rng(seed).integers(0, count, len(rows)).astype(np.int32)
    if len(ids) > 2:
        ids[1], ids[2] = -1, ids[0]
    return a, b, x, base, scale, ids


def adapters_expected(case, a, b, x, base, scale, ids):
    """The sums in fp64 and those of their terms' magnitudes."""
    rows, k, ns, rank, count = case
    want = base.double().numpy().copy()
    size = np.abs(want)
    ends = np.concatenate([[0], np.cumsum(rows)])
    for i, id in enumerate(ids):
        if not 0 <= id < count:
            continue
        r, at = slice(ends[i], ends[i + 1]), 0
        xs, s = x[r].double().numpy(), float(scale[id])
        for n, aj, bj in zip(ns, a, b):
            aj, bj = aj[id].double().numpy(), bj[id].double().numpy()
            want[r, at:at + n] += s * (xs @ aj.T) @ bj.T
            size[r, at:at + n] += s * (np.abs(xs) @ np.abs(aj).T) @ np.abs(bj).T
            at += n
    return want, size


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("name", ADAPTERS)
def test_adapters(gh, name, kind):
    import torch

    case = ADAPTERS[name]
    rows, k, ns, rank, count = case
    a, b, x, base, scale, ids = adapter_inputs(case, TYPES[kind], 7)
    total, n = sum(rows), sum(ns)
    row0 = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    ad = gemma_hip.adapters(cuda(row0), cuda(ids), scale.cuda(), len(rows), total + 2, max(rows),
                            count, rank, TYPES[kind])
    jobs = gemma_hip.adapter_jobs([(p.cuda(), q.cuda(), m) for p, q, m in zip(a, b, ns)])
    src = torch.zeros((total + 2, k + 4))
    src[:total, :k] = x
    src, out = src.cuda(), torch.full((total + 2, n + 3), 4.0, device="cuda")
    gh.adapters_add(out, n + 3, base.cuda(), 0, ad, jobs, src, k + 4, k, None, stream())
    got = out.cpu().double().numpy()
    want, size = adapters_expected(case, a, b, x, base, scale, ids)
    room = (math.sqrt(3 * k) + math.sqrt(3 * rank) + 8) * HALF
    assert (np.abs(got[:total, :n] - want) <= room * size).all()
    off = np.linalg.norm(got[:total, :n] - want) / np.linalg.norm(want)
    assert off < 1e-6, off
    assert (got[total:] == 4.0).all() and (got[:, n:] == 4.0).all()
    none = np.repeat(ids < 0, rows)
    assert np.array_equal(got[:total, :n][none], base.double().numpy()[none])
    # in place: the same bits, and rows of no adapter and no sequence as they were
    mine = torch.full((total + 2, n + 3), 4.0, device="cuda")
    mine[:total, :n] = base.cuda()
    work = torch.empty(gh.adapters_work(ad, len(ns), k), dtype=torch.uint8, device="cuda")
    gh.adapters_add(mine, n + 3, mine, n + 3, ad, jobs, src, k + 4, k, work, stream())
    assert torch.equal(mine, out)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_adapters_leave_rows_in_no_sequence(gh, kind):
    """Rows before the first sequence, behind max_rows of one and behind the last, and a table that
    falls: the others as if they weren't there; nothing that an adapter of another row holds, NaN and
    infinities among it, comes into a row."""
    import torch

    k, n, rank, count = 72, 70, 16, 3
    case = ([100], k, [n], rank, count)
    a, b, x, base, scale, _ = adapter_inputs(case, TYPES[kind], 12)
    a[0][2], b[0][2] = math.nan, math.inf
    for row0, max_rows in (([3, 20, 50, 52, 90], 18), ([3, 4, 5, 7, 9], 2)):
        ids = np.array([1, 2, 0, 1], np.int32)
        ad = gemma_hip.adapters(cuda(np.array(row0, np.int32)), cuda(ids), scale.cuda(), 4, 100,
                                max_rows, count, rank, TYPES[kind])
        out = torch.full((100, n), 4.0, device="cuda")
        jobs = gemma_hip.adapter_jobs([(a[0].cuda(), b[0].cuda(), n)])
        gh.adapters_add(out, 0, base.cuda(), 0, ad, jobs, x.cuda(), 0, k, None, stream())
        got = out.cpu().double().numpy()
        room = (math.sqrt(3 * k) + math.sqrt(3 * rank) + 8) * HALF
        left = np.ones(100, bool)
        for i, id in enumerate(ids):
            r = slice(row0[i], min(row0[i + 1], row0[i] + max_rows))
            left[r] = False
            if id == 2:
                assert not np.isfinite(got[r]).any()
                continue
            one = ([r.stop - r.start], k, [n], rank, count)
            want, size = adapters_expected(one, a, b, x[r], base[r], scale, [id])
            assert (np.abs(got[r] - want) <= room * size).all()
        assert (got[left] == 4.0).all()
    # a table that falls: no row outside of 0 .. 99 is touched (guards on both sides)
    out = torch.full((300, n), 4.0, device="cuda")
    ad = gemma_hip.adapters(cuda(np.array([50, 90, 10, -7, 1 << 30], np.int32)), cuda(ids),
                            scale.cuda(), 4, 100, 18, count, rank, TYPES[kind])
    gh.adapters_add(out[100:], 0, base.cuda(), 0, ad, jobs, x.cuda(), 0, k, None, stream())
    assert (out[:100] == 4.0).all() and (out[200:] == 4.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1 << 21, 1 << 22])
def test_adapters_of_the_last_of_many_rows(gh, rows):
    """As many rows as there may be, two of them in sequences."""
    import torch

    case = ([1, 1], 8, [8], 8, 2)
    a, b, x, base, scale, _ = adapter_inputs(case, ADAPTER_BF16, 15)
    ids = np.array([1, 0], np.int32)
    row0 = np.array([rows - 2, rows - 1, rows], np.int32)
    src, out = torch.zeros((2, rows, 8), device="cuda").unbind(0)
    src[rows - 2:], old = x.cuda(), torch.zeros((rows, 8), device="cuda")
    old[rows - 2:] = base.cuda()
    ad = gemma_hip.adapters(cuda(row0), cuda(ids), scale.cuda(), 2, rows, 1, 2, 8, ADAPTER_BF16)
    jobs = gemma_hip.adapter_jobs([(a[0].cuda(), b[0].cuda(), 8)])
    work = torch.empty(gh.adapters_work(ad, 1, 8), dtype=torch.uint8, device="cuda")
    gh.adapters_add(out, 0, old, 0, ad, jobs, src, 0, 8, work, stream())
    want, size = adapters_expected(case, a, b, x, base, scale, ids)
    room = (math.sqrt(24) + math.sqrt(24) + 8) * HALF
    assert (np.abs(out[rows - 2:].cpu().double().numpy() - want) <= room * size).all()
    assert not out[:rows - 2].any()


@pytest.mark.gpu
def test_adapters_without_scales_and_with_ids_that_lie(gh):
    import torch

    case = ([2, 2, 2, 2], 64, [24], 8, 2)
    rows, k, ns, rank, count = case
    a, b, x, base, scale, _ = adapter_inputs(case, ADAPTER_BF16, 8)
    ids = np.array([1, 2, -(1 << 31), (1 << 31) - 1], np.int32)
    row0 = np.array([0, 2, 4, 6, 8], np.int32)
    out = torch.empty((8, 24), device="cuda")
    jobs = gemma_hip.adapter_jobs([(a[0].cuda(), b[0].cuda(), 24)])
    ad = gemma_hip.adapters(cuda(row0), cuda(ids), None, 4, 8, 2, count, rank, ADAPTER_BF16)
    gh.adapters_add(out, 0, base.cuda(), 0, ad, jobs, x.cuda(), 0, k, None, stream())
    want, _ = adapters_expected(case, a, b, x, base, torch.ones(2), ids)
    assert np.abs(out.cpu().numpy() - want).max() < 1e-4
    assert torch.equal(out[2:].cpu(), base[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_adapters_of_any_size_of_values(gh, kind):
    """Rows of 1e-30 beside ones of 1e20, matrices with entries at the ends of f16."""
    import torch

    case = ([40, 1], 64, [24], 8, 1)
    rows, k, ns, rank, count = case
    a, b, x, base, scale, ids = adapter_inputs(case, TYPES[kind], 9)
    ids[:] = 0
    x[::3] *= 1e-30
    x[1::3] *= 1e20
    base[:] = 0.0
    a[0][0, 0, ::2] *= 2.0 ** 12
    a[0][0, 1, :] *= 2.0 ** -20
    row0 = np.array([0, 40, 41], np.int32)
    out = torch.empty((41, 24), device="cuda")
    jobs = gemma_hip.adapter_jobs([(a[0].cuda(), b[0].cuda(), 24)])
    ad = gemma_hip.adapters(cuda(row0), cuda(ids), scale.cuda(), 2, 41, 40, count, rank, TYPES[kind])
    gh.adapters_add(out, 0, base.cuda(), 0, ad, jobs, x.cuda(), 0, k, None, stream())
    want, size = adapters_expected(case, a, b, x, base, scale, ids)
    room = (math.sqrt(3 * k) + math.sqrt(3 * rank) + 8) * HALF
    assert (np.abs(out.cpu().numpy() - want) <= room * size).all()


# ---- log probabilities ------------------------------------------------------------


def row_of(name, vocab, rng):
    l = (rng.standard_normal(vocab) * 3).astype(F32)
    if name == "ties":
        l = np.round(l)
    elif name == "equal":
        l[:] = -1.5
    elif name == "peaked":
        l[rng.integers(vocab)] = 60.0
    elif name == "holes":
        l[rng.random(vocab) < 0.5] = -np.inf
        l[rng.random(vocab) < 0.1] = np.nan
    elif name == "lowest":
        l[rng.random(vocab) < 0.5] = np.finfo(F32).min
    elif name == "infinite":
        l[rng.integers(0, vocab, 3)] = np.inf
    elif name == "nothing":
        l[:] = -np.inf
        l[0] = np.nan
    elif name == "sorted":
        l = np.sort(l)
    elif name == "falling":
        l = -np.sort(l)
    elif name == "zeros":
        l = np.where(rng.random(vocab) < 0.5, F32(0.0), F32(-0.0)).astype(F32)
    elif name == "huge":
        l = (l * 1e36).astype(F32)
    return l


ROWS = ("normal", "ties", "equal", "peaked", "holes", "lowest", "infinite", "nothing", "sorted",
        "falling", "zeros", "huge")


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,stride,targets,ntop", [
    (1, 0, 1, 1), (2, 3, 2, 64), (63, 0, 1, 5), (64, 65, 3, 64), (65, 0, 1, 20), (1000, 1003, 8, 0),
    (2047, 0, 0, 7), (2048, 2048, 1, 64), (2049, 0, 2, 1), (16000, 16001, 64, 33),
    (70001, 0, 1, 64), (32768, 32769, 3, 64), (32769, 0, 3, 9), (66000, 0, 1, 0)])
@pytest.mark.parametrize("seed", [0, 1])
def test_logprobs(gh, vocab, stride, targets, ntop, seed):
    import torch

    rng = np.random.default_rng(seed)
    l = np.full((len(ROWS) * 2, stride or vocab), 1e30, F32)
    for i in range(len(l)):
        l[i, :vocab] = row_of(ROWS[i % len(ROWS)], vocab, rng)
    rows = len(l)
    t = np.where(np.arange(rows) < len(ROWS), F32(1.0), F32(0.6)).astype(F32)
    if seed:
        t[:8] = (0.0, -1.0, np.nan, np.inf, 1e-30, 0.0, 0.0, 0.0)
    ids = rng.integers(0, vocab, (rows, targets)).astype(np.int32)
    if targets > 1:
        ids[:, 0], ids[::2, 1] = np.nan_to_num(l[:, :vocab], nan=-np.inf).argmax(1), vocab
        ids[1::4, 1] = -1
    out = dict(logp=torch.full((rows, targets), 7.0, device="cuda"),
               rank=torch.full((rows, targets), 7, dtype=torch.int32, device="cuda"),
               entropy=torch.full((rows,), 7.0, device="cuda"),
               top=torch.full((rows, ntop), 7, dtype=torch.int32, device="cuda"),
               top_logp=torch.full((rows, ntop), 7.0, device="cuda"))
    gh.logprobs(gemma_hip.scores(**out), cuda(l), stride, rows, vocab, cuda(t), cuda(ids), targets,
                ntop, None, stream())
    got = {k: v.cpu().numpy() for k, v in out.items()}
    for r in range(rows):
        logp, rank, h, top, tl = describe(l[r, :vocab], F64(t[r]), ids[r], ntop)
        where = (ROWS[r % len(ROWS)], t[r])
        assert np.array_equal(got["rank"][r], rank), where
        assert np.array_equal(got["top"][r], top), where
        assert close_logs(got["logp"][r], logp), (where, got["logp"][r], logp)
        assert close_logs(got["top_logp"][r], tl), where
        assert close_logs(got["entropy"][r], h), (where, got["entropy"][r], h)


@pytest.mark.gpu
def test_infinite_logits_at_any_temperature(gh):
    """They share everything, also where the temperature is infinite and differences count nothing."""
    import torch

    rng = np.random.default_rng(3)
    l = np.stack([row_of("infinite", 5000, rng) for _ in range(3)])
    t, ids = np.array([np.inf, 1e-40, 3.0], F32), rng.integers(0, 5000, (3, 2)).astype(np.int32)
    ids[:, 0] = l.argmax(1)
    out = dict(logp=torch.empty((3, 2), device="cuda"), entropy=torch.empty(3, device="cuda"),
               top_logp=torch.empty((3, 8), device="cuda"))
    gh.logprobs(gemma_hip.scores(**out), cuda(l), 0, 3, 5000, cuda(t), cuda(ids), 2, 8, None,
                stream())
    for r in range(3):
        logp, _, h, _, tl = describe(l[r], F64(t[r]), ids[r], 8)
        assert close_logs(out["logp"][r].cpu(), logp) and close_logs(out["top_logp"][r].cpu(), tl)
        assert close_logs(out["entropy"][r].item(), h)


@pytest.mark.gpu
def test_logprobs_of_a_whole_vocabulary(gh):
    """262144 columns and the most there may be; answers left out; defaults."""
    import torch

    for vocab, rows in ((262144, 3), (1 << 19, 2)):
        rng = np.random.default_rng(vocab)
        l = np.stack([row_of(n, vocab, rng) for n in ("normal", "ties", "falling")[:rows]])
        ids = rng.integers(0, vocab, (rows, 1)).astype(np.int32)
        work = torch.empty(gh.logprobs_work(rows, vocab, 1, 64), dtype=torch.uint8, device="cuda")
        top = torch.empty((rows, 64), dtype=torch.int32, device="cuda")
        h = torch.empty(rows, device="cuda")
        dl, di = cuda(l), cuda(ids)
        gh.logprobs(gemma_hip.scores(top=top, entropy=h), dl, 0, rows, vocab, None, di, 1, 64, work,
                    stream())
        logp, rank = torch.empty((rows, 1), device="cuda"), torch.empty((rows, 1), dtype=torch.int32,
                                                                        device="cuda")
        gh.logprobs(gemma_hip.scores(logp=logp, rank=rank), dl, 0, rows, vocab, None, di, 1, 0, work,
                    stream())
        for r in range(rows):
            p, k, e, first, _ = describe(l[r], 1.0, ids[r], 64)
            assert np.array_equal(top[r].cpu().numpy(), first) and rank[r].item() == k[0]
            assert close_logs(logp[r].cpu().numpy(), p) and close_logs(h[r].item(), e)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,ntop,targets", [(70, 64, 1), (3023, 12, 2), (20000, 64, 0),
                                                (6145, 3, 0), (8000, 20, 1), (32768, 64, 2),
                                                (70000, 5, 1), (270000, 64, 1)])
def test_logprobs_of_many_rows(gh, vocab, ntop, targets):
    """More rows than compute units: rows that are repeated have the same answers, to the bit, and
    the first ones the definition's."""
    import torch

    rng = np.random.default_rng(vocab)
    kinds = [n for n in ROWS if n in ("normal", "ties", "equal", "holes", "falling", "nothing")]
    l = np.stack([row_of(n, vocab, rng) for n in kinds])
    ids = rng.integers(0, vocab, (len(l), targets)).astype(np.int32)
    t = np.array([1.0, 0.7, 0.0, 1.5, 1.0, 1.0], F32)
    times = 90  # 540 rows
    rows = len(l) * times
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
    got = {k: v[:len(l)].cpu().numpy() for k, v in out.items()}
    for r in range(len(l)):
        logp, rank, h, top, tl = describe(l[r], F64(t[r]), ids[r], ntop)
        assert np.array_equal(got["rank"][r], rank) and np.array_equal(got["top"][r], top), kinds[r]
        assert close_logs(got["logp"][r], logp) and close_logs(got["top_logp"][r], tl), kinds[r]
        assert close_logs(got["entropy"][r], h), kinds[r]


# ---- together ---------------------------------------------------------------------


def layer_state(seed, kind):
    """A served layer's weights and a ragged batch, in numpy."""
    rng = np.random.default_rng(seed)
    dim, heads, kv, hd = 256, 4, 2, 128
    seqs = [(1, 60), (1, 33), (7, 40), (1, 1), (20, 20)]
    p = Paged(seqs, kv, hd, 16, kind, rng)
    p.fill(rng, upto=[n for n, _ in seqs])
    n = (heads + 2 * kv) * hd
    st = dict(dim=dim, heads=heads, kv=kv, hd=hd, seqs=seqs, p=p, n=n)
    for name, shape, size in (("x", (p.rows, dim), 2), ("y", (p.rows, dim), 1),
                              ("w0", (dim,), 0.1), ("w1", (dim,), 0.1), ("nq", (hd,), 0.1),
                              ("nk", (hd,), 0.1), ("wqkv", (n, dim), dim ** -0.5),
                              ("a", (2, 8, dim), dim ** -0.5), ("b", (2, n, 8), 0.3)):
        st[name] = (rng.standard_normal(shape) * size).astype(F32)
    st["ids"] = np.array([0, -1, 1, 1, 0], np.int32)
    return st


class Layer:
    """The calls of a layer's first half on device buffers."""

    def __init__(self, gh, st):
        import torch

        self.gh, self.st, p = gh, st, st["p"]
        rows, dim, n, hd = p.rows, st["dim"], st["n"], st["hd"]
        q, kv = st["heads"] * hd, st["kv"] * hd
        self.c, self.b = p.device(), p.batch()
        d = self.d = {k: cuda(st[k]) for k in ("x", "y", "w0", "w1", "nq", "nk", "wqkv", "a", "b",
                                               "ids")}
        self.x, self.h = torch.empty((2, rows, dim), device="cuda").unbind(0)
        self.qkv = torch.empty((rows, n), device="cuda")
        self.q, self.out = torch.empty((2, rows, q), device="cuda").unbind(0)
        f, _ = gemma_hip.rotary_freqs(hd, 1e6, ROPE_LINEAR, 8.0)
        self.f, self.freq = f, cuda(f)
        self.spec = gemma_hip.residual(
            d["x"], d["y"], after=gemma_hip.norm(NORM_RMS, d["w0"], None, 1.0),
            before=gemma_hip.norm(NORM_RMS, d["w1"], None, 1.0), x_out=self.x, h=self.h)
        self.ad = gemma_hip.adapters(p.drow0, d["ids"], None, len(st["seqs"]), rows, max(p.n), 2, 8,
                                     ADAPTER_F32)
        self.jobs = gemma_hip.adapter_jobs([(d["a"], d["b"], n)])
        self.heads = gemma_hip.heads(self.qkv, n, self.qkv[:, q:], n, self.qkv[:, q + kv:], n,
                                     self.q, 0, st["heads"], d["nq"], d["nk"], EPS,
                                     gemma_hip.rotary(self.freq, hd))
        self.work = [torch.empty(max(1, k), dtype=torch.uint8, device="cuda") for k in
                     (gh.adapters_work(self.ad, 1, dim),
                      gh.cache_attention_work(self.c, self.b, st["heads"], 0, 0))]

    def run(self, s):
        gh, st, rows = self.gh, self.st, self.st["p"].rows
        gh.norm_residual(self.spec, rows, st["dim"], s)
        gh.matmul_f32(self.qkv, 0, self.d["wqkv"], 0, self.h, 0, rows, st["n"], st["dim"], s)
        gh.adapters_add(self.qkv, 0, self.qkv, 0, self.ad, self.jobs, self.h, 0, st["dim"],
                        self.work[0], s)
        gh.cache_append(self.c, self.b, self.heads, s)
        gh.cache_attention(self.out, self.q, 0, self.c, self.b, st["heads"], 0, st["hd"] ** -0.5,
                           0.0, False, 0, self.work[1], s)

    def expected(self):
        st = self.st
        p, hd, heads, kv = st["p"], st["hd"], st["heads"], st["kv"]
        x = st["x"].astype(F64) + rms(st["y"], st["w0"])
        h = rms(x, st["w1"])
        y = h @ st["wqkv"].astype(F64).T
        seq = np.repeat(np.arange(len(st["seqs"])), p.n)
        for r in range(p.rows):
            if st["ids"][seq[r]] >= 0:
                a, b = (st[k][st["ids"][seq[r]]].astype(F64) for k in "ab")
                y[r] += b @ (a @ h[r])
        pos = np.concatenate([np.arange(ln - n, ln) for n, ln in st["seqs"]])
        y = y.reshape(p.rows, heads + 2 * kv, hd)
        q = turn(rms(y[:, :heads], st["nq"]), pos, self.f, 1.0, ROPE_HALF)
        k = turn(rms(y[:, heads:heads + kv], st["nk"]), pos, self.f, 1.0, ROPE_HALF)
        for r in range(p.rows):
            for i in range(kv):
                p.put(seq[r], pos[r], k[r, i].astype(F32), i, "k")
                p.put(seq[r], pos[r], y[r, heads + kv + i].astype(F32), i, "v")
        out = np.zeros((p.rows, heads, hd))
        for b, ln in enumerate(p.len):
            for i in range(kv):
                ks, vs = p.seq_values(b, "k", i), p.seq_values(b, "v", i)
                for r in np.nonzero(seq == b)[0]:
                    for j in range(heads // kv):
                        out[r, i * (heads // kv) + j], _ = attend(
                            q[r, i * (heads // kv) + j], ks, vs, pos[r], ln, 0, hd ** -0.5, 0.0,
                            False)
        return x, out.reshape(p.rows, -1)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_a_layer_s_first_half(gh, kind):
    """Norm, product, adapters, append and attention against 64 bits.  The products' fp32 error
    (1e-6) moves a code by one step where a value lies that close to a border: a few in 10^5 of
    the codes, each 1/127 (e4m3: 1/16) of a value that counts for a share of the output."""
    st = layer_state(11, KINDS[kind])
    ly = Layer(gh, st)
    ly.run(stream())
    x, out = ly.expected()
    assert once(ly.x.cpu().numpy(), x)
    got = ly.out.cpu().numpy()
    off = np.linalg.norm(got - out) / np.linalg.norm(out)
    assert off < 1e-3, off
    same = [np.mean(st["p"].d[n][0].cpu().numpy() == st["p"].codes[n]) for n in "kv"]
    assert min(same) > 0.999, same


@pytest.mark.gpu
def test_captured_calls_follow_the_tables(gh):
    """Two graphs of the same calls with workspaces of their own, replayed in turn with eager work
    between, each replay against an eager run on the same inputs."""
    import torch

    layers = [Layer(gh, layer_state(20 + i, CACHE_I8)) for i in range(2)]
    eager = [Layer(gh, layer_state(20 + i, CACHE_I8)) for i in range(2)]
    logits = torch.randn((4, 5000), device="cuda")
    ids = torch.zeros((4, 1), dtype=torch.int32, device="cuda")
    outs = []

    def scored(work, s):
        o = dict(logp=torch.empty((4, 1), device="cuda"), entropy=torch.empty(4, device="cuda"),
                 top=torch.empty((4, 9), dtype=torch.int32, device="cuda"))
        spec = gemma_hip.scores(**o)
        return o, lambda: gh.logprobs(spec, logits, 0, 4, 5000, None, ids, 1, 9, work, s)

    graphs = []
    for ly in layers:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        work = torch.empty(gh.logprobs_work(4, 5000, 1, 9), dtype=torch.uint8, device="cuda")
        with torch.cuda.stream(s):
            o, call = scored(work, s.cuda_stream)
            ly.run(s.cuda_stream)
            call()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                ly.run(s.cuda_stream)
                call()
        graphs.append(g)
        outs.append((o, work))
    torch.cuda.synchronize()
    for step in range(4):
        for i, (g, ly, ref) in enumerate(zip(graphs, layers, eager)):
            x = torch.randn(ly.d["x"].shape, device="cuda")
            new = torch.tensor([step % 2, 1, -1, step % 3 - 1, 0], dtype=torch.int32, device="cuda")
            short = torch.tensor(ly.st["p"].len, dtype=torch.int32, device="cuda") - step % 2
            logits.copy_(torch.randn((4, 5000), device="cuda"))
            ids.fill_(step * 100 + i)
            for one in (ly, ref):
                one.d["x"].copy_(x)
                one.d["ids"].copy_(new)
                one.st["p"].dlen.copy_(short)
            g.replay()
            ref.run(stream())
            o, call = scored(outs[i][1].clone(), stream())
            call()
            torch.cuda.synchronize()
            assert torch.equal(ly.out, ref.out) and torch.equal(ly.q, ref.q)
            for n in "kv":
                assert torch.equal(ly.st["p"].d[n][0], ref.st["p"].d[n][0])
            for k in o:
                assert torch.equal(o[k], outs[i][0][k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(3, 40000), (600, 3000)])
def test_captured_log_probabilities_of_two_launches(gh, rows, vocab):
    """Replays on new logits, with eager work between, against eager calls."""
    import torch

    logits = torch.randn((rows, vocab), device="cuda")
    ids = torch.zeros((rows, 2), dtype=torch.int32, device="cuda")
    work = [torch.empty(gh.logprobs_work(rows, vocab, 2, 9), dtype=torch.uint8, device="cuda")
            for _ in "ab"]
    out = [dict(logp=torch.empty((rows, 2), device="cuda"), entropy=torch.empty(rows, device="cuda"),
                rank=torch.empty((rows, 2), dtype=torch.int32, device="cuda"),
                top=torch.empty((rows, 9), dtype=torch.int32, device="cuda")) for _ in "ab"]

    def call(i, s):
        gh.logprobs(gemma_hip.scores(**out[i]), logits, 0, rows, vocab, None, ids, 2, 9, work[i], s)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        call(0, s.cuda_stream)
    for step in range(4):
        logits.copy_(torch.randn((rows, vocab), device="cuda"))
        ids.fill_(step * 7)
        g.replay()
        call(1, stream())
        torch.cuda.synchronize()
        assert all(torch.equal(out[0][k], out[1][k]) for k in out[0])


@pytest.mark.gpu
def test_captured_calls_need_their_workspaces(gh):
    import torch

    case = ADAPTERS["steps"]
    rows, k, ns, rank, count = case
    a, b, x, base, scale, ids = adapter_inputs(case, ADAPTER_BF16, 7)
    ad = gemma_hip.adapters(cuda(np.arange(8, dtype=np.int32)), cuda(ids), scale.cuda(), 7, 7, 1,
                            count, rank, ADAPTER_BF16)
    jobs = gemma_hip.adapter_jobs([(p.cuda(), q.cuda(), m) for p, q, m in zip(a, b, ns)])
    out, base, x = torch.empty((7, sum(ns)), device="cuda"), base.cuda(), x.cuda()
    l = torch.randn((1, 100), device="cuda")
    h = torch.zeros(1, device="cuda")
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        if gh.adapters_work(ad, 3, k):
            with pytest.raises(gemma_hip.GemmaHipError, match="captured"):
                gh.adapters_add(out, 0, base, 0, ad, jobs, x, 0, k, None, s.cuda_stream)
        with pytest.raises(gemma_hip.GemmaHipError, match="captured"):
            gh.logprobs(gemma_hip.scores(entropy=h), l, 0, 1, 100, None, None, 0, 0, None,
                        s.cuda_stream)
        h.zero_()
    small = torch.empty(256, dtype=torch.uint8, device="cuda")
    with pytest.raises(gemma_hip.GemmaHipError, match="aligned"):
        gh.logprobs(gemma_hip.scores(entropy=h), l, 0, 1, 100, None, None, 0, 5, small[8:], stream())


@pytest.mark.gpu
def test_calls_on_two_streams(gh):
    """The library's own workspaces are a stream's: many calls on two of them at once."""
    import torch

    streams = [torch.cuda.Stream() for _ in range(2)]
    data = []
    for i in range(2):
        l = torch.randn((3, 30000 + i), device="cuda")
        case = ADAPTERS["few"]
        a, b, x, base, scale, ids = adapter_inputs(case, ADAPTER_F16, 30 + i)
        rows, k, ns, rank, count = case
        row0 = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        ad = gemma_hip.adapters(cuda(row0), cuda(ids), scale.cuda(), 3, 9, 4, count, rank, ADAPTER_F16)
        jobs = gemma_hip.adapter_jobs([(p.cuda(), q.cuda(), m) for p, q, m in zip(a, b, ns)])
        data.append((l, ad, jobs, x.cuda(), base.cuda(), k))

    def one(i, s):
        l, ad, jobs, x, base, k = data[i]
        o = dict(entropy=torch.empty(3, device="cuda"),
                 top=torch.empty((3, 12), dtype=torch.int32, device="cuda"))
        out = torch.empty_like(base)
        torch.cuda.synchronize() if s is None else None
        to = stream() if s is None else s.cuda_stream
        gh.logprobs(gemma_hip.scores(**o), l, 0, 3, l.shape[1], None, None, 0, 12, None, to)
        gh.adapters_add(out, 0, base, 0, ad, jobs, x, 0, k, None, to)
        return [o["entropy"], o["top"], out]

    want = [one(i, None) for i in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, one(i, s)))
    torch.cuda.synchronize()
    for i, g in got:
        assert all(torch.equal(x, y) for x, y in zip(g, want[i]))


@pytest.mark.gpu
def test_empty_calls(gh):
    import torch

    c = gemma_hip.cache(None, None, None, None, CACHE_I8, 1, 16, 1, 128)
    b = gemma_hip.batch(None, None, None, 0, 0, 0, 0, 0)
    gh.cache_append(c, b, gemma_hip.heads(None, 0, None, 0, None, 0, None, 0, 0), stream())
    gh.rope(None, 0, None, 0, 0, 1, 64, None, None, EPS, None, stream())
    gh.norm_residual(gemma_hip.residual(None), 0, 64, stream())
    ad = gemma_hip.adapters(None, None, None, 0, 0, 0, 0, 8, ADAPTER_F32)
    gh.adapters_add(None, 0, None, 0, ad, gemma_hip.adapter_jobs([(None, None, 8)]), None, 0, 8, None,
                    stream())
    gh.logprobs(gemma_hip.scores(), None, 0, 0, 100, None, None, 0, 0, None, stream())
    torch.cuda.synchronize()
