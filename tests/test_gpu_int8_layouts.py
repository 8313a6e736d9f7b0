"""Quantisation over what splits it: rows of one matrix shared by the CTAs of a cluster, rows longer than a CTA keeps,
each with and without RunningNorm's statistics, from every source type, bit for bit."""

import numpy as np
import pytest
import torch

from alphafly_b200.int8 import int8_linear, int8_matmul, quantize
from alphafly_b200.model import RunningNorm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _rand(*shape, seed=0):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


def _quantized(x):
    """The definition in numpy's float32 (IEEE division, rint to even): (q, scale)."""
    a = x.detach().cpu().float().numpy()
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(a).all(1)
        scale = (np.abs(a).max(1) / np.float32(127)).astype(np.float32)
        q = np.rint(a / scale[:, None])
    q = np.where((scale > 0)[:, None] & ~bad[:, None], np.clip(np.nan_to_num(q), -127, 127), 0)
    return q.astype(np.int8), np.where(bad, np.float32(np.nan), scale)


def _norm(k):
    norm = RunningNorm(k).to(DEV).eval()
    norm.mean.copy_(_rand(k, seed=1))
    norm.var.copy_(_rand(k, seed=2).abs() * 0.1)
    return norm


# columns: 321 values take a cluster of two CTAs, 641 four, 1,281 to 2,560 eight, more are read in spans
@pytest.mark.parametrize("layout", ["columns", "rows"])
@pytest.mark.parametrize("with_norm", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 321), (33, 640), (70, 641), (31, 1281), (256, 2333), (1120, 2333), (65, 2561), (9, 5000), (3, 20001)])
def test_quantize_across_clusters_and_spans(rows, k, dtype, with_norm, layout):
    x = (_rand(rows, k, seed=rows + k) * 2).to(dtype)
    x[rows // 2, k - 1] = 11.0                   # the largest magnitude in the last CTA's share
    if rows > 2:
        x[0, 3] = float("nan")                   # and a row without a scale by the first one's
        x[2] = 0.0
    norm = _norm(k) if with_norm else None
    rq, rs = _quantized(norm(x.float()) if with_norm else x)
    src = x.T.contiguous().T if layout == "columns" else x
    for _ in range(3):
        q, scale = quantize(src, norm)
        assert np.array_equal(scale.cpu().numpy(), rs, equal_nan=True)
        assert np.array_equal(q.cpu().numpy(), rq)


def test_a_backward_through_the_product_fails():
    """Rather than leave what lies before the product without a gradient."""
    x, (w, ws), bias = _rand(3, 40), quantize(_rand(6, 40, seed=1)), _rand(6, seed=2)
    q, scale = quantize(x)
    ref = int8_linear(x, w, ws, bias)
    leaf = x.clone().requires_grad_(True)
    other = torch.ones(3, 6, device=DEV, requires_grad=True)
    for y in (int8_linear(leaf * 1.0, w, ws, bias), int8_linear(x, w, ws, bias.clone().requires_grad_(True)),
              int8_matmul(q, scale, w, ws.clone().requires_grad_(True), bias)):
        assert torch.equal(y, ref)
        with pytest.raises(RuntimeError, match="has no gradient"):
            (y * other).sum().backward()
    for y in (int8_linear(leaf.detach(), w, ws, bias), int8_linear(x, w, ws, bias)):
        assert not y.requires_grad
        (y * other).sum().backward()
    with torch.no_grad():
        assert not int8_linear(leaf, w, ws, bias).requires_grad
    empty = int8_linear(torch.empty(3, 0, device=DEV, requires_grad=True), w[:, :0], ws, bias)
    assert empty.requires_grad and torch.equal(empty, bias.expand(3, 6))
