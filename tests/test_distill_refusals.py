"""Arguments of the distillation entry points that the library has to refuse on the host: a kernel would read past
them, or return what they do not mean.  No GPU is needed."""

import ctypes

import pytest

from alphafly_b200 import _lib

P = ctypes.c_void_p(256)
# afb_distill_loss: rows, moves, type, logits, ld, k, values, moves, log_rest, T, legal, valid, listed, weight, scale, upstream,
# its step, skip_ones, row_loss, loss, grad, ld of it, stream
LOSS = [3, 50, _lib.T_F32, P, 50, 4, P, P, None, 1.0, None, None, 0, None, 1.0, None, 0, 0, P, P, P, 50, None]


def _refused(match, name, good, **changes):
    args = list(good)
    for at, value in changes.items():
        args[int(at[1:])] = value
    with pytest.raises(_lib.AfbError, match=match):
        _lib.call(name, *args)


def test_rows_to_skip_are_named_by_an_upstream_gradient():
    """Without one the kernel would read it from address 0."""
    _refused("skip_ones needs", "afb_distill_loss", LOSS, _17=1)
    _refused("skip_ones needs", "afb_distill_loss", LOSS, _17=1, _10=P, _11=P, _12=8)


@pytest.mark.parametrize("temperature", [3.5e-39, 3e-39, 1e-45, float("inf")])
def test_temperatures_whose_inverse_is_not_finite(temperature):
    """log2(e) / T has to be: with an infinite one every term is NaN."""
    top = [3, 50, _lib.T_F32, P, 50, 4, 1.0, None, None, 0, P, P, P, None]
    _refused("temperature", "afb_top_logits", top, _6=temperature)
    _refused("temperature", "afb_distill_loss", LOSS, _9=temperature)


def test_temperatures_whose_square_is_not_finite():
    """The loss is a divergence times T^2: an infinite one makes 0 a NaN."""
    _refused("square of the temperature", "afb_distill_loss", LOSS, _9=1.9e19)
