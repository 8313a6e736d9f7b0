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


def test_one_row_of_any_stride():
    """A transposed column is a row whose stride, 1, lies below its length."""
    column = _rand(300, 1, seed=2)
    x, plain = column.T, column.reshape(1, 300).clone()
    assert x.stride() == (1, 1)
    top, ref = top_logits(x, 6), top_logits(plain, 6)
    for a, b in zip(top[:3], ref[:3]):
        assert torch.equal(a, b)
    leaf, leaf2 = column.clone().requires_grad_(True), plain.clone().requires_grad_(True)
    for scale in (1.0, 3.0):                     # the forward's gradient, and the backward's
        loss, loss2 = distillation_loss(leaf.T, top, rest=True), distillation_loss(leaf2, top, rest=True)
        assert torch.equal(loss, loss2)
        g, g2 = torch.autograd.grad(loss * scale, leaf)[0], torch.autograd.grad(loss2 * scale, leaf2)[0]
        assert torch.equal(g.T, g2)


@pytest.mark.parametrize("rows,v,k,dtype", [(2048, 4168, 32, torch.float32), (2048, 4168, 128, torch.float32), (64, 4168, 100, torch.float32),
                                            (1000, 32000, 64, torch.bfloat16), (1000, 12000, 200, torch.float16)])
def test_selection_repeats_bit_for_bit(rows, v, k, dtype):
    """Candidates are collected in any order; what is summed of them is not."""
    x = (_rand(rows, v, seed=k) * 2).to(dtype)
    first = top_logits(x, k, 2.0)
    for _ in range(30):
        again = top_logits(x, k, 2.0)
        for a, b in zip(first[:3], again[:3]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lists_over_the_most_moves(dtype):
    """1,048,576 moves with the longest lists and the most named moves: the loss over the lists is that of the listed
    logits side by side."""
    v, listed, k = 1 << 20, 4096, 256
    x = torch.zeros(2, v, dtype=dtype, device=DEV)
    moves = torch.stack([torch.randperm(v, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i))[:listed].sort().values for i in range(2)])
    moves[:, -1] = v - 1
    x.scatter_(1, moves, (_rand(2, listed, seed=3) * 2).to(dtype))
    legal = moves, torch.rand(2, listed, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)) < 0.9
    side = x.gather(1, moves).masked_fill(~legal[1], -INF)
    top, near = top_logits(x, k, 1.5, legal=legal), top_logits(side, k, 1.5)
    assert torch.equal(top.values, near.values) and torch.equal(top.moves, moves.gather(1, near.moves))
    leaf, leaf2 = x.clone().requires_grad_(True), side.clone().requires_grad_(True)
    losses = distillation_loss(leaf, top, legal=legal, rest=True, reduction="none")
    losses2 = distillation_loss(leaf2, near._replace(log_rest=top.log_rest), rest=True, reduction="none")
    # two orders of the same float32 sums
    torch.testing.assert_close(losses, losses2, rtol=1e-5, atol=1e-5)
    g, g2 = torch.autograd.grad(losses.sum(), leaf)[0], torch.autograd.grad(losses2.sum(), leaf2)[0]
    torch.testing.assert_close(g.gather(1, moves).float(), g2.float(), rtol=2.0**-7 if dtype == torch.bfloat16 else 2.0**-10, atol=1e-6)
    assert int((g != 0).sum()) <= int(legal[1].sum())


def test_calls_from_several_threads():
    """Threads that need different amounts of a kernel's shared memory get what one thread would."""
    from concurrent.futures import ThreadPoolExecutor
    cases = []
    for n, v in enumerate((30000, 70000, 300000, 700000, 1 << 20)):
        x, moves = _rand(2, v, seed=n), torch.arange(0, v, v // 50, device=DEV).repeat(2, 1)
        legal = moves, torch.ones_like(moves, dtype=torch.bool)
        cases += [(x, top_logits(x, 9), None), (x, top_logits(x, 9, legal=legal), legal)]
    torch.cuda.synchronize()

    def run(i):
        x, top, legal = cases[i % len(cases)]
        return distillation_loss(x, top, legal=legal, rest=True, reduction="none")
    order = [i * 7 % len(cases) for i in range(60)]
    with ThreadPoolExecutor(6) as pool:
        got = list(pool.map(run, order))
    torch.cuda.synchronize()
    ref = [run(i) for i in range(len(cases))]
    for i, losses in zip(order, got):
        assert torch.equal(losses, ref[i])


def test_targets_made_in_inference_mode():
    """The natural way to run a teacher; such tensors track no versions."""
    x, t = _rand(5, 400, seed=1), _rand(5, 400, seed=2)
    legal = torch.arange(60, device=DEV).repeat(5, 1), torch.rand(5, 60, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)) < 0.7
    weight = torch.rand(5, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4))
    with torch.inference_mode():
        made = top_logits(t, 6, 2.0, legal=legal)
        lists = tuple(a.clone() for a in legal)
        inside = distillation_loss(x, made, legal=lists, rest=True, weight=weight.clone(), reduction="none")
        own = weight.clone()
    plain = top_logits(t, 6, 2.0, legal=legal)
    ref = distillation_loss(x, plain, legal=legal, rest=True, weight=weight, reduction="none")
    assert made.values.is_inference() and torch.equal(inside, ref)
    grads = []
    for top, where, w in ((made, lists, own), (plain, legal, weight)):
        leaf = x.clone().requires_grad_(True)
        losses = distillation_loss(leaf, top, legal=where, rest=True, weight=w, reduction="none")
        assert torch.equal(losses, ref)
        grads.append(torch.autograd.grad(losses, leaf, torch.full_like(ref, 3.0))[0])
    assert torch.equal(*grads)


def test_targets_changed_before_the_backward_are_refused():
    leaf, top = _rand(3, 50, seed=1).requires_grad_(True), top_logits(_rand(3, 50, seed=2), 4)
    loss = distillation_loss(leaf, top)
    top.values.add_(1.0)
    with pytest.raises(RuntimeError, match="modified in place"):
        loss.backward()
