"""The 8-bit products (alphafly_b200.int8) against their definition: the quantiser bit for bit, the product in 64
bits; rows of zeros, infinities, NaN and subnormal numbers; every layout and type; odd sizes; the refusals."""

import ctypes

import numpy as np
import pytest
import torch

from alphafly_b200 import _lib
from alphafly_b200.gemm import status_word
from alphafly_b200.int8 import empty_rows, int8_linear, int8_matmul, quantize
from alphafly_b200.model import RunningNorm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# half the distance between neighbouring values of each type, relative
HALF_ULP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def _rand(*shape, seed=0):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


def _quantized(x):
    """The definition in numpy's float32 (IEEE division, rint to even): (q, scale)."""
    a = x.detach().cpu().float().numpy()
    with np.errstate(all="ignore"):
        top = np.abs(a).max(1) if a.shape[1] else np.zeros(len(a), np.float32)
        bad = ~np.isfinite(a).all(1)
        scale = (top / np.float32(127)).astype(np.float32)
        q = np.rint(a / scale[:, None])
    q = np.where((scale > 0)[:, None] & ~bad[:, None], np.clip(np.nan_to_num(q), -127, 127), 0)
    return q.astype(np.int8), np.where(bad, np.float32(np.nan), scale)


def _layout(x, layout):
    if layout == "columns":
        return x.T.contiguous().T
    if layout == "strided":                      # every other row of a wider matrix, off any 16-byte boundary
        wide = torch.full((2 * x.shape[0], x.shape[1] + 3), 77.0, dtype=x.dtype, device=x.device)
        wide[::2, 1:x.shape[1] + 1] = x
        return wide[::2, 1:x.shape[1] + 1]
    if layout == "scattered":                    # neither dimension has unit stride
        wide = torch.zeros(x.shape[0], 2 * x.shape[1], dtype=x.dtype, device=x.device)
        wide[:, ::2] = x
        return wide[:, ::2]
    return x.contiguous()


@pytest.mark.parametrize("layout", ["rows", "columns", "strided", "scattered"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 17), (33, 2333), (5, 4097), (130, 838), (1, 2333), (70, 64), (2, 20001)])
def test_quantize_is_its_definition_bit_for_bit(rows, k, dtype, layout):
    x = _layout((_rand(rows, k, seed=rows + k) * 2).clamp(-8, 8).to(dtype), layout)
    q, scale = quantize(x)
    rq, rs = _quantized(x)
    assert q.dtype == torch.int8 and q.shape == (rows, k) and q.stride(0) % 16 == 0
    assert np.array_equal(scale.cpu().numpy(), rs)
    assert np.array_equal(q.cpu().numpy(), rq)


@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("k", [5, 333])
def test_quantize_rows_of_special_values(k, layout):
    x = _rand(12, k, seed=3)
    x[0] = 0.0
    x[1, 2] = float("inf")
    x[2, k - 1] = float("-inf")
    x[3, 0] = float("nan")
    x[4] *= 1e-40                                # subnormal values, subnormal scale
    x[5] = 1e-45                                 # the scale underflows to 0
    x[6] *= 3e38 / x[6].abs().max()
    x[7] = -0.0
    x[8] = 2.0                                   # every quotient is 127
    x[9] = torch.arange(k, device=DEV) % 255 * 0.5 - 63.5   # quotients on .0 and .5
    x[9, 0] = 127.0
    x = _layout(x, layout)
    q, scale = quantize(x)
    rq, rs = _quantized(x)
    assert np.array_equal(scale.cpu().numpy(), rs, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), rq)
    assert np.isnan(rs[1:4]).all() and not rq[:4].any()
    w, ws = quantize(_rand(9, k, seed=4))
    y = int8_linear(x, w, ws, torch.ones(9, device=DEV))
    # row 6's products pass float32's range where the exact ones do
    exact = torch.from_numpy(rq * np.nan_to_num(rs.astype(np.float64))[:, None]).to(DEV) @ (w.double() * ws.double()[:, None]).T
    fits = (exact + 1).abs() < torch.finfo(torch.float32).max
    assert torch.isnan(y[1:4]).all() and torch.equal(torch.isfinite(y)[[0, *range(4, 12)]], fits[[0, *range(4, 12)]])
    assert torch.equal(y[[0, 5, 7]], torch.ones(3, 9, device=DEV))


@pytest.mark.parametrize("layout", ["rows", "columns"])
def test_quantize_normalises_like_running_norm(layout):
    norm = RunningNorm(301).to(DEV).eval()
    norm.mean.copy_(_rand(301, seed=1))
    norm.var.copy_(_rand(301, seed=2).abs() * 0.01)
    x = _layout(_rand(45, 301, seed=5), layout)
    rq, rs = _quantized(norm(x))
    q, scale = quantize(x, norm)
    # sqrt and both divisions round alike, so the normalised values are the module's own
    assert np.array_equal(scale.cpu().numpy(), rs)
    assert np.array_equal(q.cpu().numpy(), rq)
    with pytest.raises(ValueError, match="norm.mean"):
        quantize(x[:, :300], norm)


def _check_product(y, q, scale, w, w_scale, bias, dtype):
    """|y - ref| within: the sum's rounding to float32, two products and the final addition (4 float32 roundings of the
    terms), one rounding to the result's type, and that type's smallest step."""
    whole = q.cpu().double() @ w.cpu().double().T                    # exact: below 2^53
    part = whole * scale.cpu().double()[:, None] * w_scale.cpu().double()
    b = bias.cpu().double() if bias is not None else torch.zeros(w.shape[0], dtype=torch.float64)
    ref = part + b
    assert y.dtype == dtype and y.shape == ref.shape
    step = {torch.float16: 2.0**-25}.get(dtype, 0.0)
    limit = 4 * 2.0**-24 * (part.abs() + b.abs()) * 1.01 + HALF_ULP[dtype] * ref.abs() * 1.01 + step + 1e-38
    err = (y.cpu().double() - ref).abs()
    assert bool((err <= limit).all()), float((err / limit).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 5, 8, 9, 16, 33, 129, 300, 513])
@pytest.mark.parametrize("n,k", [(1, 1), (5, 3), (128, 16), (129, 127), (257, 129), (300, 2333), (515, 838)])
def test_product_over_sizes(rows, n, k, dtype):
    q, scale = quantize(_rand(rows, k, seed=rows))
    w, w_scale = quantize(_rand(n, k, seed=n + 7))
    bias = _rand(n, seed=1) if (rows + n) % 2 else None
    _check_product(int8_matmul(q, scale, w, w_scale, bias, dtype), q, scale, w, w_scale, bias, dtype)
    x = _rand(rows, k, seed=rows)
    assert torch.equal(int8_linear(x, w, w_scale, bias, out_dtype=dtype), int8_matmul(q, scale, w, w_scale, bias, dtype))
    assert int(status_word(DEV)) == 0


@pytest.mark.parametrize("rows,n,k", [(1120, 4171, 2333), (2048, 4171, 2333), (700, 17937, 838), (4500, 1000, 300)])
def test_product_at_the_networks_sizes(rows, n, k):
    q, scale = quantize(_rand(rows, k, seed=rows))
    w, w_scale = quantize(_rand(n, k, seed=n))
    bias = _rand(n, seed=2)
    _check_product(int8_matmul(q, scale, w, w_scale, bias), q, scale, w, w_scale, bias, torch.float32)
    assert int(status_word(DEV)) == 0


@pytest.mark.parametrize("rows", [1, 9, 200])
def test_longest_sum_is_exact(rows):
    """-128 times -128, 131071 times: one product below the overflow of int32."""
    q = empty_rows(rows, 131071, DEV).fill_(-128)
    w = empty_rows(3, 131071, DEV).fill_(-128)
    w[1] = 127
    one = torch.ones(rows, device=DEV)
    y = int8_matmul(q, one, w, torch.ones(3, device=DEV))
    ref = torch.tensor([131071 * 16384, -131071 * 16256, 131071 * 16384], dtype=torch.float64).float()
    assert torch.equal(y.cpu(), ref.expand(rows, 3))
    with pytest.raises(_lib.AfbError, match="131071"):
        int8_matmul(empty_rows(1, 131072, DEV), one[:1], empty_rows(1, 131072, DEV), one[:1])


@pytest.mark.parametrize("rows", [1, 6, 140])
def test_bytes_past_the_rows_do_not_count(rows):
    """Rows are padded to 16 bytes; the padding may hold anything."""
    k = 37
    q, scale = quantize(_rand(rows, k, seed=1))
    w, w_scale = quantize(_rand(50, k, seed=2))
    ref = int8_matmul(q, scale, w, w_scale)
    for t in (q, w):
        torch.as_strided(t, (t.shape[0], t.stride(0)), (t.stride(0), 1))[:, k:] = 113
    assert torch.equal(int8_matmul(q, scale, w, w_scale), ref)
    assert torch.equal(int8_linear(_rand(rows, k, seed=1), w, w_scale), ref)
    assert torch.equal(int8_matmul(q.contiguous()[:, :], scale, w.contiguous(), w_scale), ref)      # unaligned rows are copied


@pytest.mark.parametrize("rows", [1, 30, 260])
@pytest.mark.parametrize("type_,dtype", [(_lib.T_F32, torch.float32), (_lib.T_F16, torch.float16)])
def test_writes_stay_inside_the_result(rows, type_, dtype):
    """A result with a row stride beyond n and rows around it keeps what stood there."""
    n, k = 131, 50
    q, scale = quantize(_rand(rows, k, seed=1))
    w, w_scale = quantize(_rand(n, k, seed=2))
    wide = torch.full((rows + 2, n + 9), 55.0, dtype=dtype, device=DEV)
    y = wide[1:-1, 4:4 + n]
    p = ctypes.c_void_p
    _lib.call("afb_int8_matmul", rows, n, k, q.data_ptr(), q.stride(0), scale.data_ptr(), w.data_ptr(), w.stride(0),
              w_scale.data_ptr(), None, p(y.data_ptr()), type_, wide.stride(0), None, p(torch.cuda.current_stream().cuda_stream))
    ref = int8_matmul(q, scale, w, w_scale, out_dtype=dtype)
    assert torch.equal(y, ref)
    wide[1:-1, 4:4 + n] = 55.0
    assert bool((wide == 55.0).all())


def test_empty_sizes():
    w, w_scale = quantize(_rand(6, 40, seed=1))
    assert int8_linear(_rand(0, 40), w, w_scale).shape == (0, 6)
    assert int8_linear(_rand(3, 40), w[:0], w_scale[:0]).shape == (3, 0)
    bias = _rand(6, seed=2)
    y = int8_linear(_rand(3, 0), torch.empty(6, 0, dtype=torch.int8, device=DEV), w_scale, bias)
    assert torch.equal(y, bias.expand(3, 6))
    q, s = quantize(_rand(4, 0))
    assert q.shape == (4, 0) and torch.equal(s, torch.zeros(4, device=DEV))


def test_on_another_stream_and_in_a_graph():
    x = _rand(70, 333, seed=1)
    w, w_scale = quantize(_rand(90, 333, seed=2))
    ref = int8_linear(x, w, w_scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = int8_linear(x, w, w_scale)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        z = int8_linear(x, w, w_scale)
    x.mul_(2.0)                                  # the scales double, the 8-bit values stay
    g.replay()
    torch.testing.assert_close(z, 2 * ref, rtol=0, atol=0)


def test_refusals():
    x, (w, ws) = _rand(3, 40), quantize(_rand(6, 40))
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        int8_linear(x.double(), w, ws)
    with pytest.raises(TypeError, match="out_dtype"):
        int8_linear(x, w, ws, out_dtype=torch.int8)
    with pytest.raises(ValueError, match="inner dimensions"):
        int8_linear(x[:, :39], w, ws)
    with pytest.raises(ValueError, match="w must be int8"):
        int8_linear(x, w.float(), ws)
    with pytest.raises(ValueError, match="w_scale"):
        int8_linear(x, w, ws[:5])
    with pytest.raises(ValueError, match="bias"):
        int8_linear(x, w, ws, ws.double())
    with pytest.raises(RuntimeError, match="CUDA"):
        int8_linear(x.cpu(), w, ws)
    with pytest.raises(ValueError, match="rows, k"):
        quantize(x[0])
