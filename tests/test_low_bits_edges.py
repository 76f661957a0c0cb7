"""8-bit rows and 4-bit weights where they meet their edges: what stands behind a matrix's last row, values next to the middle
between two codes, groups that stand for NaN behind a gate, the workspace's room, refusals.

What is planted is exact: sums of small whole numbers, powers of two.  So codes and scales are compared bit for bit.
"""
from __future__ import annotations

import ctypes
import gc
import math
import weakref

import pytest
import torch

from tests import kernel_refs as R
from tests.conftest import F32_MODEL_TOL, TINY, random_tokens
from tests.helpers import run_requests
from tests.test_low_bits import E2M1, E4M3, code_values, far, mx_engine, operands, ops, plain_mx_logits, powers, rnd, scale_rows, stands_for

GPU = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


# ---------------------------------------------------------------------------
# behind a matrix's last row
# ---------------------------------------------------------------------------

def set_scales_behind(m, byte):
    """The scale bytes of the rows that fill the last block of 128 behind the matrix's own."""
    r, kb = m.scales.shape[:2]
    at = torch.arange(m.rows, r * 128, device="cuda")
    m.scales.view(r, kb, 32, 4, 4)[at // 128, :, at % 32, at % 128 // 32] = byte


@GPU
@pytest.mark.parametrize("kernel,split", [(0, 0), (1, 0), (1, 4), (1, 8), (2, 0), (3, 0), (4, 2), (4, 4)])
@pytest.mark.parametrize("t,n,k", [(40, 144, 1024), (300, 144, 1030), (64, 400, 2048), (130, 16, 1024), (270, 560, 1100)])
def test_scales_behind_the_weights_rows_mean_nothing(t, n, k, kernel, split):
    o = ops()
    t = min(t, 64) if kernel == 1 else t
    x, w = operands(t, n, k, seed=n)
    whole = rnd(n + 100, k, seed=7)
    whole[n:, ::5] = torch.tensor([NAN, INF], device="cuda").repeat(50)[:, None]
    cut, clean = o.mx_weight(whole)[:n], o.mx_weight(whole[:n].contiguous())
    try:
        o.mx_set_kernel(kernel)
        o.mx_set_few(split)
        for epi in (1, 3, 4):
            three = dict(limit=1.5, alpha=1.702, up_add=1.0) if epi == 4 else {}
            got = []
            for weight, byte in ((clean, 127), (cut, None), (w, 127), (w, 255)):
                if byte is not None:
                    set_scales_behind(weight, byte)
                rows = o.MxRows.empty(t, n // 2)
                rows.codes.fill_(5)
                rows.scales.fill_(9)
                o.linear_mx(x, weight, rows, epi, **three)
                got.append((rows.codes, scale_rows(rows), o.linear_mx(x, weight, torch.full((t, n // 2), NAN, device="cuda"), epi, **three)))
            for a, b, what in ((got[0], got[1], "a weight's first rows"), (got[2], got[3], "scales of NaN behind them")):
                assert torch.equal(a[2], b[2]), f"{what}: values"
                assert torch.equal(a[1], b[1]), f"{what}: scales"
                assert torch.equal(a[0], b[0]), f"{what}: codes"
                assert not a[0][:, n // 2:].any() and (a[1][:, -(-(n // 2) // 32):] == 127).all(), "the padding is zeros of scale 1"
    finally:
        o.mx_set_kernel()
        o.mx_set_few()


@GPU
@pytest.mark.parametrize("t", [5, 40, 300])
def test_a_product_behind_a_cut_weight_is_finite(t):
    """Down behind gate and up, as a feed-forward has them: padding of scale NaN would take every sum along."""
    o = ops()
    x, _ = operands(t, 16, 256)
    gate_up, down = rnd(300, 256, seed=1), o.mx_weight(rnd(40, 72, seed=2))
    gate_up[150] = NAN
    act = o.MxRows.empty(t, 72)
    o.linear_mx(x, o.mx_weight(gate_up)[:144], act, o.EPI_GATED_GELU)
    out = o.linear_mx(act, down, torch.empty(t, 40, device="cuda"))
    assert torch.isfinite(out).all()
