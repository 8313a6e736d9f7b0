"""Selection and loss at their arguments' edges."""

import math

import pytest
import torch

from alphafly_b200.distill import distillation_loss, top_logits

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = math.inf


def _rand(*shape, seed=0):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


@pytest.mark.parametrize("dtype", DTYPES)
def test_lists_of_no_width_hold_no_move(dtype):
    x = _rand(4, 300, seed=1).to(dtype)
    empty = torch.zeros(4, 0, dtype=torch.int64, device=DEV), torch.zeros(4, 0, dtype=torch.bool, device=DEV)
    top = top_logits(x, 5, 2.0, legal=empty)
    assert (top.values == -INF).all() and (top.moves == -1).all() and (top.log_rest == -INF).all()
    named = top_logits(x, 5, 2.0)
    for rest in (False, True):
        leaf = x.clone().requires_grad_(True)
        losses = distillation_loss(leaf, named, legal=empty, rest=rest, reduction="none")
        grad, = torch.autograd.grad(losses.sum(), leaf)
        assert not losses.any() and not grad.any()
