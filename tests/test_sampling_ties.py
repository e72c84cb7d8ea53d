"""gemma_hip_sample where logits are equal, as those rounded to few bits often are: running sums
then meet top-p's and the draw's targets exactly, and what the definition says of equality (the
fewest that sum to *at least* p, the first whose sum *exceeds* u times theirs) decides.  Against
whole numbers and fractions."""

from __future__ import annotations

from fractions import Fraction
from math import ceil, floor

import numpy as np
import pytest

import gemma_hip
from test_serving import F32, cuda, stream


def drawn(n, k, p, u):
    """Which of n equal tokens is drawn (from 0), and how many are kept."""
    kept = n if k <= 0 else min(n, k)
    if p < 1:
        kept = max(1, ceil(Fraction(float(p)) * kept))
    return min(floor(Fraction(float(u)) * kept), kept - 1), kept


def test_the_definition():
    assert drawn(2, 0, 0.5, 0.9) == (0, 1) and drawn(2, 0, F32(0.6), 0.5) == (1, 2)
    assert drawn(4, 0, 0.75, 0.0) == (0, 3) and drawn(10, 5, 1.0, 0.4) == (2, 5)
    assert drawn(10, 0, F32(0.1), 0.0) == (0, 2)  # 0.1 in fp32 is above 1/10


def settings_of(rng, rows, n):
    """Settings whose targets fall on borders between equal tokens, and beside them."""
    p = rng.choice([1.0, 0.5, 0.25, 0.75, 0.875, 0.0625, 0.1, 0.9, 0.3], rows).astype(F32)
    u = rng.choice([0.0, 0.5, 0.25, 0.75, 0.125, 0.625, 1 - 2.0 ** -24, 0.1, 0.7], rows).astype(F32)
    k = rng.choice([0, n, max(1, n // 2), max(1, n // 4), n + 5], rows).astype(np.int32)
    return p, u, k


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,n", [(2, 2), (4, 4), (16, 12), (1000, 1), (1000, 8), (1000, 500),
                                     (16384, 10000), (16384, 16384), (20000, 64), (262144, 2),
                                     (262144, 48), (262144, 2000), (262144, 100000),
                                     (262144, 262144), (524288, 524288)])
@pytest.mark.parametrize("others", ["none", "far"])
def test_equal_largest_logits(gh, vocab, n, others):
    """n tokens share the largest logit; the others are -inf, or so far below that top-k or
    their own weight (below 2^-300) leaves them out."""
    import torch

    rng = np.random.default_rng(vocab + n)
    rows = 24
    p, u, k = settings_of(rng, rows, n)
    if others == "far":
        k = np.minimum(np.where(k <= 0, n, k), n).astype(np.int32)
    temp = rng.choice([0.5, 1.0, 0.7, 1.3], rows).astype(F32)
    top = rng.standard_normal(rows).astype(F32) * F32(8)
    l = np.full((rows, vocab), -np.inf, F32)
    if others == "far":
        l[:] = top[:, None] - F32(300) - rng.random((rows, vocab)).astype(F32)
    at = np.stack([np.sort(rng.permutation(vocab)[:n]) for _ in range(rows)])
    np.put_along_axis(l, at, top[:, None].repeat(n, 1), 1)
    tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
    probs = torch.empty(rows, device="cuda")
    gh.sample(tokens, probs, cuda(l), 0, rows, vocab,
              gemma_hip.sampling(cuda(temp), cuda(k), cuda(p)), cuda(u), None, stream())
    torch.cuda.synchronize()
    tokens, probs = tokens.cpu().numpy(), probs.cpu().numpy()
    for i in range(rows):
        j, kept = drawn(n, int(k[i]), p[i], u[i])
        assert tokens[i] == at[i, j], (i, p[i], u[i], k[i], int(np.searchsorted(at[i], tokens[i])), j)
        # one rounding to fp32, and the weights' own
        assert abs(probs[i] - 1 / kept) <= (2.0 ** -24 + 2.0 ** -38) / kept
