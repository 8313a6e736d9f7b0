"""Argument errors of the 8-bit products and of distillation come back from the library without a GPU."""

import ctypes

import pytest

from alphafly_b200 import _lib

P = ctypes.c_void_p(256)


def _raises(match, name, *args):
    with pytest.raises(_lib.AfbError, match=match):
        _lib.call(name, *args)


def test_quantize_arguments():
    good = [4, 40, _lib.T_F32, P, 40, 0, None, None, 0.0, 0.0, P, 48, P, None]

    def bad(match, at, value):
        args = list(good)
        args[at] = value
        _raises(match, "afb_quantize_rows", *args)
    bad("negative size", 0, -1)
    bad("131071", 1, 131072)
    bad("element type", 2, 5)
    bad("NULL pointer", 3, None)
    bad("leading dimension", 4, 39)
    bad("together", 6, P)
    bad("16-byte", 11, 47)
    bad("16-byte", 10, ctypes.c_void_p(264))
    bad("aligned to its elements", 3, ctypes.c_void_p(257))
    _lib.call("afb_quantize_rows", 0, *good[1:])                  # nothing to do


def test_int8_product_arguments():
    good = [4, 9, 40, P, 48, P, P, 48, P, None, P, _lib.T_F16, 9, None, None]

    def bad(match, at, value):
        args = list(good)
        args[at] = value
        _raises(match, "afb_int8_matmul", *args)
    bad("k must be positive", 2, 0)
    bad("NULL pointer", 3, None)
    bad("NULL pointer", 8, None)
    bad("16-byte", 4, 41)
    bad("16-byte", 7, 41)
    bad("leading dimension", 12, 8)
    bad("element type", 11, -1)
    _lib.call("afb_int8_matmul", 0, *good[1:])
    assert _lib.load().afb_int8_linear_workspace(0, 7) == 0 and _lib.load().afb_int8_linear_workspace(300, 7) >= 300 * (16 + 4)
    _raises("workspace too small", "afb_int8_linear", 400, 9, 40, 0, P, 40, 0, None, None, 0.0, 0.0, P, 48, P, None, P, 0, 9, P, 10, None, None)


def test_top_logits_arguments():
    good = [3, 50, _lib.T_F32, P, 50, 4, 1.0, None, None, 0, P, P, P, None]

    def bad(match, at, value):
        args = list(good)
        args[at] = value
        _raises(match, "afb_top_logits", *args)
    bad("negative size", 0, -1)
    bad("1048576", 1, (1 << 20) + 1)
    bad("leading dimension", 4, 49)
    bad("between 1 and 256", 5, 257)
    bad("temperature", 6, 0.0)
    bad("temperature", 6, float("nan"))
    bad("valid flags", 7, P)
    bad("4096", 9, 4097)
    bad("NULL pointer", 10, None)
    _lib.call("afb_top_logits", 0, *good[1:])


def test_distill_loss_arguments():
    good = [3, 50, _lib.T_F32, P, 50, 4, P, P, None, 1.0, None, None, 0, None, 1.0, None, 0, 0, P, P, P, 50, None]

    def bad(match, at, value):
        args = list(good)
        args[at] = value
        _raises(match, "afb_distill_loss", *args)
    bad("needs row_loss", 18, None)
    bad("NULL pointer", 6, None)
    bad("leading dimension", 21, 49)
    bad("temperature", 9, -2.0)
    bad("aligned to its elements", 20, ctypes.c_void_p(258))
    bad("negative size", 16, -1)
