"""Attention over the 8-bit paged cache (gemma_hip_cache_attention) at values and scores of
any size that the cache and fp32 hold, against plain numpy in 64 bits.

The bar is relative to what a row weighs: the sum of weight times the largest |value| of a
position, over the sum of weights, so that large values which hardly count excuse no error of
small ones which do.  Scores s are fp32 sums of q's and the codes' products: off by about
2^-22 of |s| and that is the weights' relative error; the weights and the value sums add
about 2^-21.  2e-5 for scores up to 10 is some ten times both, and grows with |s| above.  An
output below 2^-126 is rounded to a whole number of fp32's least steps, 2^-149: half of one
added (a row whose weights lie on a position of zeros may answer 2^-140)."""

from __future__ import annotations

import numpy as np
import pytest

from test_serving import F32, F64, KINDS, Paged, cuda, stream

TOL = 2e-5


def attend(q, k, v, lo, hi, asc, cap):
    """One row and head over keys lo .. hi, in 64 bits: (output, the size of what it weighs, its
    largest |score|)."""
    k, v = k[lo:hi + 1].astype(F64), v[lo:hi + 1].astype(F64)
    s = k @ q.astype(F64) * asc
    if cap:
        s = np.tanh(s / cap) * cap
    p = np.exp(s - s.max())
    size = p @ np.abs(v).max(1) / p.sum()
    return p @ v / p.sum(), size, np.abs(s).max()


def check(gh, p, q, heads, asc, slide=0, cap=0.0, shared=0, step=1, exact=False):
    """exact: the scores are so in fp32, whatever their size."""
    import torch

    c = p.device()
    out = torch.full((p.rows, heads * p.hd), 3.0, device="cuda")
    gh.cache_attention(out, cuda(q), 0, c, p.batch(), heads, slide, asc, cap, False, shared, None,
                       stream())
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(p.rows, heads, p.hd)
    for b, (n, ln) in enumerate(p.seqs):
        for h in range(heads):
            k, v = (p.seq_values(b, x, h // (heads // p.kv)) for x in "kv")
            for i in range(0, n, step):
                pos = ln - n + i
                want, size, s = attend(q[p.row0[b] + i, h * p.hd:(h + 1) * p.hd], k, v,
                                       max(0, pos + 1 - slide) if slide else 0, pos, asc, cap)
                bar = TOL * size * (1.0 if exact else max(1.0, s / 10)) + 2.0 ** -150
                err = np.abs(got[p.row0[b] + i, h] - want).max()
                assert err <= bar, (b, i, h, err, bar)


# sequences (new rows, positions), heads, kv, head dim, window, shared, every so many rows checked:
# single tokens in one chunk and in many, prompt rows of 64 and 128 vectors a workgroup, behind a
# prefix that one launch takes with them and in a launch of its own
SHAPES = {
    "step": ([(1, 70), (2, 33), (1, 1)], 4, 1, 256, 0, 0, 1),
    "step_128": ([(1, 70), (3, 200)], 4, 2, 128, 7, 0, 1),
    "step_long": ([(1, 9000), (1, 40)], 4, 1, 256, 0, 0, 1),
    "prompt": ([(40, 90), (30, 30)], 4, 2, 256, 0, 0, 1),
    "prompt_128": ([(70, 500)], 4, 1, 128, 20, 0, 1),
    "prompt_large": ([(1300, 2600), (901, 1400)], 4, 1, 256, 0, 0, 97),
    "prompt_large_128": ([(1300, 2600), (901, 1400)], 8, 2, 128, 0, 0, 97),
    "prefix": ([(1, 150), (1, 97), (2, 200)], 4, 1, 256, 0, 96, 1),
    "prefix_mixed": ([(1, 150), (30, 140), (1, 97)], 4, 1, 128, 0, 96, 1),
}


def cache_of(name, kind, seed):
    seqs, heads, kv, hd, slide, shared, step = SHAPES[name]
    rng = np.random.default_rng(seed)
    p = Paged(seqs, kv, hd, 16, KINDS[kind], rng, shared=shared)
    p.fill(rng)
    q = rng.standard_normal((p.rows, heads * hd)).astype(F32)
    return p, q, rng


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("name,octaves", [
    (name, octaves) for name in sorted(SHAPES) for octaves in
    ([-85, 100] if "large" in name else [-50, -62, -70, -85, -110, 100])])
def test_values_of_one_size(gh, name, octaves, kind):
    """Values of about 2^octaves at every position."""
    _, heads, _, hd, slide, shared, step = SHAPES[name]
    p, q, _ = cache_of(name, kind, 3)
    p.scales["v"] *= F32(2.0) ** octaves
    check(gh, p, q, heads, hd ** -0.5, slide, 0.0, shared, step)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("name", ["step", "step_128", "step_long", "prompt", "prompt_128", "prefix",
                                  "prefix_mixed"])
def test_values_of_all_sizes(gh, name, kind):
    """Values from 2^-110 to 2^100 with weights that even them out, so that each row's largest
    contributions come from values of very different sizes, and zeros among them."""
    seqs, heads, kv, hd, slide, shared, step = SHAPES[name]
    p, q, rng = cache_of(name, kind, 4)
    u = rng.choice([-1.0, 1.0], hd)
    q[:] = np.tile(u, heads) * rng.choice([0.5, 1.0, 2.0], (p.rows, 1))
    asc = 1.0 / hd
    for page in range(p.codes["k"].shape[0]):  # keys c u: scores c times a row's 0.5, 1 or 2
        e = rng.integers(-110, 101, p.scales["v"][page].shape)
        c = (-e * np.log(2.0) + rng.standard_normal(e.shape)).astype(F32)
        live = np.isfinite(p.scales["k"][page])
        unit = np.where(u > 0, 64, -64).astype(np.int8).view(np.uint8) if kind == "i8" else \
            np.where(u > 0, 0x38, 0xb8).astype(np.uint8)  # +-64, and 1 in e4m3
        p.codes["k"][page][live] = unit
        p.scales["k"][page] = np.where(live, c / F32(64 if kind == "i8" else 1), np.nan)
        p.scales["v"][page] *= (F32(2.0) ** e).astype(F32) * (rng.random(e.shape) > 0.1)
    check(gh, p, q, heads, asc, slide, 0.0, shared, step)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_small_values_beside_zeros_and_unseen_large_ones(gh, rows, cap):
    """Rows of zeros are common (nothing has been written there yet) and answer zeros; values
    that no row sees, at any size, change nothing."""
    rng = np.random.default_rng(5)
    p = Paged([(rows, 100), (rows, 64)], 1, 128, 16, KINDS["i8"], rng)
    p.fill(rng)
    p.scales["v"] *= F32(2.0) ** -90
    for b in (0, 1):
        for pos in range(p.len[b]):
            page, at = p.table[b, pos // 16], pos % 16
            if pos < p.len[b] - rows - 8:
                p.scales["v"][page, 0, at] = F32(2.0) ** 100  # before every window
            elif pos % 3:
                p.scales["v"][page, 0, at], p.codes["v"][page, 0, at] = 0.0, 0
    q = rng.standard_normal((p.rows, 4 * 128)).astype(F32)
    check(gh, p, q, 4, 0.1, 9, cap)
    p.scales["v"][:], p.codes["v"][:] = 0.0, 0
    check(gh, p, q, 4, 0.1, 9, cap)


def scored_cache(name, kind, octaves, sign):
    """Keys that differ in their first dim alone: scores of exactly sign 2^octaves by asc 1 (q is
    a power of two in that dim, the rest meets codes of 0)."""
    p, q, rng = cache_of(name, kind, 6)
    a = octaves // 2
    q[:, ::p.hd] = F32(2.0) ** a
    code = 64 if kind == "i8" else 0x38
    live = np.isfinite(p.scales["k"])
    p.codes["k"][live] = 0
    p.codes["k"][..., 0][live] = code
    unit = F32(sign * 2.0 ** (octaves - a) / (64 if kind == "i8" else 1))
    p.scales["k"] = np.where(live, unit, np.nan).astype(F32)
    return p, q


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("octaves", [10, 23, 27, 30, 60, 100])
@pytest.mark.parametrize("name", ["step", "step_128", "step_long", "prompt", "prompt_128", "prefix",
                                  "prefix_mixed"])
def test_equal_scores_of_any_size(gh, name, octaves, sign, kind):
    """Every key scores the same, however much that is: the values' mean."""
    _, heads, _, hd, slide, shared, step = SHAPES[name]
    p, q = scored_cache(name, kind, octaves, sign)
    check(gh, p, q, heads, 1.0, slide, 0.0, shared, step, exact=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("octaves", [22, 24, 25, 26, 27, 28, 29, 31, 40])
@pytest.mark.parametrize("name", ["step", "prompt", "prefix"])
def test_scores_that_rise_by_their_last_place(gh, name, octaves, kind):
    """From tile to tile by 2^-23 of themselves, which is octaves where they are large."""
    _, heads, _, hd, slide, shared, step = SHAPES[name]
    p, q = scored_cache(name, kind, octaves, 1.0)
    for b, ln in enumerate(p.len):
        for pos in range(ln):
            page = p.table[b, pos // 16]
            unit = np.abs(p.scales["k"][page, :, pos % 16])
            up = F32(1.0 + (pos // 32) * 2.0 ** -23)
            p.scales["k"][page, :, pos % 16] = 2.0 ** np.floor(np.log2(unit)) * up
    check(gh, p, q, heads, 1.0, slide, 0.0, shared, step)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("octaves", [25, 27, 30, 60])
@pytest.mark.parametrize("name", ["step", "step_128", "step_long", "prompt", "prompt_128", "prefix",
                                  "prefix_mixed"])
def test_scores_that_come_from_far(gh, name, octaves, kind):
    """A sequence's first keys score -2^octaves and count for nothing beside the rest's 0: what
    their sums may have become is gone without a trace, but for a NaN among them."""
    import torch

    seqs, heads, _, hd, slide, shared, step = SHAPES[name]
    p, q = scored_cache(name, kind, octaves, -1.0)
    for b, ln in enumerate(p.len):
        for pos in range(ln // 2 if not shared else shared // 2, ln):
            p.scales["k"][p.table[b, pos // 16], :, pos % 16] = 0.0
    check(gh, p, q, heads, 1.0, slide, 0.0, shared, step, exact=True)
    if slide:
        return
    p.scales["k"][p.table[0, 0], :, 1] = np.nan  # seen by every row of the first sequence
    c = p.device()
    out = torch.zeros((p.rows, heads * hd), device="cuda")
    gh.cache_attention(out, cuda(q), 0, c, p.batch(), heads, 0, 1.0, 0.0, False, shared, None,
                       stream())
    torch.cuda.synchronize()
    sees = out[:p.n[0]].cpu().numpy()[[p.len[0] - p.n[0] + i >= 1 for i in range(p.n[0])]]
    assert np.isnan(sees).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("octaves", [0, -70])
@pytest.mark.parametrize("ahead", [80, 1000])
@pytest.mark.parametrize("name", ["step", "step_long", "prompt", "prompt_large", "prefix",
                                  "prefix_mixed"])
def test_positions_of_zeros_with_the_most_weight(gh, name, ahead, octaves, kind):
    """A position of zeros scores so many octaves above the others that these are 2^-80 of the
    sum, or nothing; then one further on scores above both."""
    _, heads, _, hd, slide, shared, step = SHAPES[name]
    p, q = scored_cache(name, kind, 0, 1.0)
    p.scales["v"] *= F32(2.0) ** octaves
    p.scales["k"] = np.where(np.isfinite(p.scales["k"]), 0, np.nan).astype(F32)
    unit = np.log(2.0) * ahead / (64 if kind == "i8" else 1)
    for b, ln in enumerate(p.len):
        if ln > 20:
            at = p.table[b, 1], slice(None), 3  # (position 19)
            p.scales["k"][at], p.scales["v"][at], p.codes["v"][at] = unit, 0.0, 0
    check(gh, p, q, heads, 1.0, slide, 0.0, shared, step)
    for b, ln in enumerate(p.len):
        if ln > 60:
            p.scales["k"][p.table[b, (ln - 5) // 16], :, (ln - 5) % 16] = 2.0 * unit
    check(gh, p, q, heads, 1.0, slide, 0.0, shared, step)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("low,high", [(-55, 75), (-100, 100), (-44, 110), (-59, 119)])
@pytest.mark.parametrize("name", sorted(SHAPES))
def test_small_values_first(gh, name, low, high, kind):
    """Scores near zero: the first keys' values are of 2^low, those from some key on of 2^high,
    beside whose M the sum of the first ones' weights, as large as those of the others, is still
    to be counted."""
    _, heads, _, hd, slide, shared, step = SHAPES[name]
    p, q, _ = cache_of(name, kind, 8)
    for b, ln in enumerate(p.len):
        for pos in range(ln):
            up = pos >= (shared or ln) * 2 // 3
            p.scales["v"][p.table[b, pos // 16], :, pos % 16] = F32(2.0) ** (high if up else low) / 127
    check(gh, p, q, heads, hd ** -0.5, 0, 0.0, shared, step)
