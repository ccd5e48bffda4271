"""Rows that the norm reads twice: the residual's sum may be written over the input
or the residual, which the second pass reads. Tolerances: those of
test_gpu_rms_norm.py."""
from __future__ import annotations

import pytest
import torch

import practice_cuda_amd as pca
from test_gpu_rms_norm import check, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 3, 700])
@pytest.mark.parametrize("n", [16385, 16392, 20480, 40001, 65536, 65544])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_rows_and_in_place(dev, n, rows, dtype):
    x, w, r = tensors(dev, (rows, n), dtype, True, seed=n)
    codes, total = check(x, w, r)
    check(x, w)
    for into in ("residual", "x"):
        given = {"x": x.clone(), "residual": r.clone()}
        q, out = pca.rms_norm_quant(given["x"], w, residual=given["residual"], residual_out=given[into])
        assert out is given[into] and torch.equal(out, total)
        assert torch.equal(q.tensor.view(torch.uint8), codes.tensor.view(torch.uint8))
        assert torch.equal(q.dequant_scale, codes.dequant_scale)
