"""The operators between the products of a served batch where fp32 ends.  Definitions and bars
are those of test_layer_ops.py, or stand beside the test."""

from __future__ import annotations

import numpy as np
import pytest

import gemma_hip
from gemma_hip import NORM_LAYER, NORM_RMS
from test_layer_ops import F32, F64, codes_of_rows, normed, once
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
