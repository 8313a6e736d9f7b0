"""Distillation (alphafly_b200.distill) against its definition in 64 bits: the selection with ties, masks and rows
that hold nothing; the loss and its gradient over all moves and legal lists, against the formula and against
differences of the 64-bit loss; scaled and repeated backwards; the refusals."""

import math

import numpy as np
import pytest
import torch

from alphafly_b200.distill import TopLogits, distillation_loss, top_logits

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_ULP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
INF = math.inf


def _rand(*shape, seed=0):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


def _lists(b, v, most, seed):
    """Distinct moves in random order; row 0 has none, row 1 one, the last all `most`."""
    rng = np.random.default_rng(seed)
    moves, valid = np.zeros((b, most), np.int64), np.zeros((b, most), bool)
    for i in range(b):
        n = {0: 0, 1: 1, b - 1: most}.get(i, int(rng.integers(1, most + 1)))
        at = np.sort(rng.permutation(most)[:n])              # gaps between the valid entries
        moves[i, at] = rng.permutation(v)[:n]
        valid[i, at] = True
    return torch.from_numpy(moves).to(DEV), torch.from_numpy(valid).to(DEV)


def _support(shape, legal):
    on = np.ones(shape, bool)
    if legal is not None:
        on[:] = False
        moves, valid = (t.cpu().numpy() for t in legal)
        for i in range(shape[0]):
            m = moves[i, valid[i]]
            on[i, m[(m >= 0) & (m < shape[1])]] = True
    return on


def _top_reference(logits, k, temperature, legal):
    x = logits.detach().cpu().float().numpy()
    b, v = x.shape
    on = _support(x.shape, legal) & ~np.isnan(x) & (x > -INF)
    values, moves, rest = np.full((b, k), -INF, np.float32), np.full((b, k), -1), np.full(b, -INF)
    for i in range(b):
        m = np.flatnonzero(on[i])
        m = m[np.lexsort((m, -x[i, m].astype(np.float64)))]
        n = min(k, len(m))
        values[i, :n], moves[i, :n] = x[i, m[:n]], m[:n]
        left = x[i, m[n:]].astype(np.float64) / np.float64(np.float32(temperature))
        if len(left):
            rest[i] = left.max() + np.log(np.exp(left - left.max()).sum())
    return values, moves, rest


def _check_top(logits, k, temperature=1.0, legal=None):
    top = top_logits(logits, k, temperature, legal)
    values, moves, rest = _top_reference(logits, k, temperature, legal)
    assert np.array_equal(top.values.cpu().numpy(), values)
    assert np.array_equal(top.moves.cpu().numpy(), moves)
    got = top.log_rest.cpu().double().numpy()
    fine = np.isfinite(rest)
    assert np.array_equal(got[~fine], rest[~fine])
    # the largest exponent's product, the terms' exponents and their sum: a few roundings of values up to |rest| + 20
    assert (np.abs(got - rest)[fine] <= 2.0**-21 * (np.abs(rest[fine]) + 20)).all()
    return top


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [1, 2, 31, 257, 1000, 4168, 9001, 40000])
@pytest.mark.parametrize("k", [1, 7, 32, 200, 256])
def test_top_logits_over_sizes(v, k, dtype):
    _check_top((_rand(5, v, seed=v + k) * 2).to(dtype), k, 1.7)


@pytest.mark.parametrize("v", [600, 5003])
@pytest.mark.parametrize("k", [16, 48, 80, 128, 190])
def test_top_logits_of_many_rows(v, k):
    """More than 1,024 rows are ranked by one warp each up to 160 candidates; half of the rows have equal values."""
    x = _rand(1100, v, seed=v + k) * 2
    x[::2] = (x[::2] * 4).round() / 4
    _check_top(x, k, 0.8)


@pytest.mark.parametrize("k", [100, 170, 256])
def test_top_logits_of_large_k(k):
    _check_top(_rand(40, 4168, seed=k), k)


@pytest.mark.parametrize("listed", [1, 30, 218, 1500, 4096])
@pytest.mark.parametrize("dtype", DTYPES)
def test_top_logits_of_legal_moves(listed, dtype):
    v = 4168
    x = (_rand(6, v, seed=listed) * 3).to(dtype)
    legal = _lists(6, v, listed, seed=listed)
    x[2, legal[0][2, 0]] = float("nan")
    top = _check_top(x, 8, 0.5, legal)
    assert (top.moves[0] == -1).all() and (top.values[0] == -INF).all() and float(top.log_rest[0]) == -INF


@pytest.mark.parametrize("v", [40, 4168, 30000])
def test_top_logits_ties_and_special_rows(v):
    x = _rand(12, v, seed=v)
    x[0] = 0.25                                   # all equal
    x[1] = -INF                                   # nothing
    x[2] = float("nan")                           # nothing
    x[3] = torch.finfo(torch.float32).min         # the type's lowest value is a value
    x[4, : v - 3] = -INF                          # three moves
    x[5] = x[5].round()                           # many ties
    x[6, ::2] = float("nan")
    x[7] = torch.where(torch.arange(v, device=DEV) % 2 == 0, 0.0, -0.0)   # one value
    x[8, v // 2] = INF
    x[9] *= 1e30
    x[10, 5] = 1e30                               # the rest far below the best
    x[11] = torch.linspace(1, -1, v, device=DEV)  # sorted: the best in one place
    for k in (1, 4, 33, 256):
        top = _check_top(x, k)
    assert torch.equal(top.moves[0, :min(v, 256)], torch.arange(min(v, 256), device=DEV))


def test_top_logits_rest_far_below_the_best():
    """The rest keeps its own size however far below the selected moves it lies."""
    x = _rand(3, 500, seed=1)
    x[:, 100:104] += 4000.0
    x[1] += 1e6
    _check_top(x, 4)
    _check_top(x, 3)
    _check_top(x, 2, 0.01)


def test_top_logits_strides_and_lists_that_repeat():
    base = _rand(7, 900, seed=2)
    _check_top(base[:, 3:703], 9)
    _check_top(base[::2], 9)
    _check_top(base.T, 5)
    moves = torch.tensor([[5, 5, -3, 700, 9, 5, 2000, 1]], device=DEV)
    valid = torch.tensor([[1, 1, 1, 1, 0, 1, 1, 1]], device=DEV).bool()
    top = top_logits(base[:1, :700], 4, legal=(moves, valid))
    ref = top_logits(base[:1, :700], 4, legal=(torch.tensor([[5, 1]], device=DEV), torch.ones(1, 2, dtype=torch.bool, device=DEV)))
    for a, b in zip(top[:3], ref[:3]):
        assert torch.equal(a, b)
    assert top_logits(base[:0], 3).moves.shape == (0, 3)


# -- the loss ------------------------------------------------------------------------------------------------

def _loss64(s, top, legal, rest, weight=None):
    """Per-position losses in float64 from the definition; differentiable in s (float64, CPU)."""
    t = float(np.float32(top.temperature))
    b, v = s.shape
    on = torch.from_numpy(_support((b, v), legal))
    out = []
    for i in range(b):
        named, z = [], []
        for m, value in zip(top.moves[i].tolist(), top.values[i].double().tolist()):
            if 0 <= m < v and bool(on[i, m]) and value > -INF and m not in named:
                named.append(m)
                z.append(value / t)
        si = torch.where(on[i], s[i] / t, -INF)
        if not named or bool((si == -INF).all()):
            out.append(s[i].sum() * 0.0 if bool(torch.isfinite(s[i]).all()) else torch.zeros((), dtype=torch.float64))
            continue
        r = float(top.log_rest[i]) if rest else -INF
        z = torch.tensor(z + ([r] if r > -INF else []), dtype=torch.float64)
        log_p = torch.log_softmax(z, 0)
        lse = torch.logsumexp(si, 0)
        log_q = si[named] - lse
        if r > -INF:
            other = torch.ones(v, dtype=torch.bool)
            other[named] = False
            log_q = torch.cat([log_q, (torch.logsumexp(si[other], 0) - lse)[None]])
        out.append((log_p.exp() * (log_p - log_q)).sum() * t * t)
    out = torch.stack(out)
    return out if weight is None else out * weight.cpu().double()


def _check_loss(s, top, legal=None, rest=False, weight=None):
    """The kernel's losses and gradient against the 64-bit ones.  Each log share comes from exponents of size up to
    A = 64 in float32, (A + 4) 2^-22 < 2e-5 of a share p or q; a loss term adds the rounding of its logarithms."""
    leaf = s.detach().clone().requires_grad_(True)
    b = s.shape[0]
    losses = distillation_loss(leaf, top, legal, rest, weight, reduction="none")
    mean = distillation_loss(leaf, top, legal, rest, weight)
    grad, = torch.autograd.grad(mean, leaf)
    s64 = s.detach().cpu().double().requires_grad_(True)
    ref = _loss64(s64, top, legal, rest, weight)
    ref_grad, = torch.autograd.grad(ref.sum() / b, s64)
    t = top.temperature
    w = torch.ones(b, dtype=torch.float64) if weight is None else weight.cpu().double()
    spread = (s.detach().float().cpu().double().abs().amax(1) / t + 20) * t * t * w
    assert losses.dtype == torch.float32 and mean.shape == ()
    assert bool(((losses.detach().cpu().double() - ref.detach()).abs() <= 2.0**-20 * spread).all())
    assert abs(float(mean.detach()) - float(ref.detach().mean())) <= 2.0**-20 * float(spread.mean())
    on = torch.from_numpy(_support(s.shape, legal))
    q = torch.softmax(torch.where(on, s64.detach() / t, -INF), 1).nan_to_num(0.0)
    p = torch.zeros_like(q)
    for i in range(b):
        for m, value in zip(top.moves[i].tolist(), top.values[i].double().tolist()):
            if 0 <= m < s.shape[1]:
                p[i, m] = max(float(p[i, m]), math.exp(value / t - float(top.values[i].double().max()) / t)) if value > -INF else p[i, m]
    share = (q + p + q / q.sum(1, keepdim=True).clamp(min=1e-300)) * t * w[:, None] / b
    # what the teacher leaves to the rest, spread like the student's own rest
    if rest:
        share = share + torch.where(p > 0, 0.0, q) / torch.where(p > 0, 0.0, q).sum(1, keepdim=True).clamp(min=1e-300) * t * w[:, None] / b
    step = {torch.float16: 2.0**-25}.get(s.dtype, 0.0)
    err = (grad.cpu().double() - ref_grad).abs()
    assert grad.dtype == s.dtype and grad.shape == s.shape
    assert bool((err <= 2e-5 * share + HALF_ULP[s.dtype] * ref_grad.abs() * 1.01 + step + 1e-37).all())
    assert bool((grad.cpu()[~on] == 0).all())
    return grad, ref_grad


def _teacher(b, v, k, t, seed, legal=None):
    return top_logits(_rand(b, v, seed=seed) * 2, k, t, legal)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v,k,t", [(1, 1, 1.0), (2, 1, 2.0), (50, 50, 1.0), (333, 7, 0.5), (4168, 32, 2.0), (4168, 256, 1.0), (20003, 64, 3.3)])
def test_loss_over_all_moves(v, k, t, dtype, rest):
    s = (_rand(4, v, seed=v) * 1.5).to(dtype)
    _check_loss(s, _teacher(4, v, k, t, seed=k), None, rest, torch.tensor([1.0, 0.0, 2.5, 0.3], device=DEV) if k == 7 else None)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("listed,k", [(1, 1), (40, 8), (218, 32), (2000, 16)])
def test_loss_over_legal_moves(listed, k, dtype, rest):
    legal = _lists(6, 4168, listed, seed=listed)
    s = (_rand(6, 4168, seed=3) * 2).to(dtype)
    grad, _ = _check_loss(s, _teacher(6, 4168, k, 1.0, seed=4, legal=legal), legal, rest)
    assert not grad[0].any()                                      # no legal move: nothing to learn
    if dtype == torch.float32:                                    # a teacher that names other moves: those are left out
        _check_loss(s, _teacher(6, 4168, k, 1.0, seed=5), legal, rest)


@pytest.mark.parametrize("rest", [False, True])
def test_loss_of_special_rows(rest):
    v, k = 600, 5
    s = _rand(9, v, seed=1)
    top = _teacher(9, v, k, 1.0, seed=2)
    moves, values = top.moves.clone(), top.values.clone()
    moves[0] = -1                                                 # names nothing
    values[1] = -INF
    moves[2, 1:] = -1                                             # one move
    moves[3, 3] = moves[3, 0]                                     # twice
    moves[4, 2] = v + 3                                           # out of range
    values[5, :4] -= 500.0                                        # shares that underflow
    s[6] -= 1e4                                                   # the student's size does not matter
    s[7] = torch.finfo(torch.float32).min / 4                     # uniform at the type's lowest values
    s[8, 10:] -= 300.0                                            # a rest that underflows beside the best
    top = TopLogits(values, moves, top.log_rest, 1.0)
    leaf = s.clone().requires_grad_(True)
    losses = distillation_loss(leaf, top, rest=rest, reduction="none")
    grad, = torch.autograd.grad(losses.sum(), leaf)
    assert torch.isfinite(losses).all() and torch.isfinite(grad).all()
    assert not losses[:2].any() and not grad[:2].any()
    keep = [0, 1, 2, 3, 4, 5, 6, 8]
    _check_loss(s[keep], TopLogits(values[keep], moves[keep], top.log_rest[keep], 1.0), None, rest)
    _check_loss(s[[7]].clamp(min=-1e3), TopLogits(values[[7]], moves[[7]], top.log_rest[[7]], 1.0), None, rest)
    # -inf for all, and NaN, stay in their rows
    s[2] = -INF
    s[3, 7] = float("nan")
    s[4, int(moves[4, 0])] = -INF
    leaf = s.clone().requires_grad_(True)
    losses = distillation_loss(leaf, top, rest=rest, reduction="none")
    grad, = torch.autograd.grad(losses.sum(), leaf)
    assert float(losses[2]) == 0 and not grad[2].any()
    assert math.isnan(float(losses[3])) and torch.isnan(grad[3]).all()
    assert float(losses[4]) == INF and torch.isfinite(grad[4]).all()
    assert torch.isfinite(losses[[0, 1, 5, 6, 7, 8]]).all()


@pytest.mark.parametrize("rest", [False, True])
def test_gradient_against_differences(rest):
    """Central differences of the 64-bit loss along random directions: error h^2/6 times a third derivative of order
    1 / T, h = 1e-4, and the kernel's own 2e-5."""
    b, v, k, t = 3, 300, 12, 1.5
    s, top = _rand(b, v, seed=6), _teacher(3, 300, k, t, seed=7)
    leaf = s.clone().requires_grad_(True)
    grad, = torch.autograd.grad(distillation_loss(leaf, top, rest=rest), leaf)
    base, h = s.cpu().double(), 1e-4
    for seed in range(5):
        d = torch.randn(b, v, dtype=torch.float64, generator=torch.Generator().manual_seed(seed))
        up, down = (_loss64(base + e * h * d, top, None, rest).mean() for e in (1, -1))
        slope = float((up - down) / (2 * h))
        got = float((grad.cpu().double() * d).sum())
        assert abs(got - slope) <= 2e-5 * float((grad.cpu().double().abs() * d.abs()).sum()) + 1e-7


@pytest.mark.parametrize("dtype", DTYPES)
def test_backward_scales_and_repeats(dtype):
    """An upstream gradient other than 1 is applied before the one rounding; a second backward gives the same."""
    b, v = 5, 700
    s, top = (_rand(b, v, seed=1)).to(dtype), _teacher(b, v, 6, 1.0, seed=2)
    up = torch.tensor([1.0, 0.0, 2.0, -3.0, 65536.0], device=DEV)
    leaf = s.clone().requires_grad_(True)
    losses = distillation_loss(leaf, top, rest=True, reduction="none")
    first, = torch.autograd.grad(losses, leaf, up, retain_graph=True)
    again, = torch.autograd.grad(losses, leaf, up)
    assert torch.equal(first, again)
    s64 = s.cpu().double().requires_grad_(True)
    ref, = torch.autograd.grad((_loss64(s64, top, None, True) * up.cpu().double()).sum(), s64)
    err = (first.cpu().double() - ref).abs()
    fine = ref.abs() < 60000 if dtype == torch.float16 else torch.ones_like(ref, dtype=torch.bool)
    assert bool((err <= 4e-5 * up.cpu().double().abs()[:, None] * 1.0 + HALF_ULP[dtype] * ref.abs() * 1.01 + 2.0**-25)[fine].all())
    leaf = s.clone().requires_grad_(True)
    g, = torch.autograd.grad(distillation_loss(leaf, top, rest=True) * 4096.0, leaf)
    leaf2 = s.clone().requires_grad_(True)
    g2, = torch.autograd.grad(distillation_loss(leaf2, top, rest=True, reduction="sum"), leaf2, torch.tensor(4096.0 / b, device=DEV))
    torch.testing.assert_close(g, g2, rtol=4 * HALF_ULP[dtype], atol=2.0**-24)


def test_reductions_and_repeatability():
    s, top = _rand(700, 4168, seed=1), _teacher(700, 4168, 16, 2.0, seed=2)
    w = torch.rand(700, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    losses = distillation_loss(s, top, weight=w, reduction="none")
    for reduction, ref in (("sum", losses.double().sum()), ("mean", losses.double().mean())):
        got = distillation_loss(s, top, weight=w, reduction=reduction)
        assert abs(float(got) - float(ref)) <= 2.0**-23 * float(ref)
        assert torch.equal(got, distillation_loss(s, top, weight=w, reduction=reduction))
    leaves = [s.clone().requires_grad_(True) for _ in range(2)]
    a, b = (torch.autograd.grad(distillation_loss(x, top, rest=True), x)[0] for x in leaves)
    assert torch.equal(a, b)
    with torch.no_grad():
        assert not distillation_loss(leaves[0], top).requires_grad


def test_loss_of_strided_logits_and_no_rows():
    wide, top = _rand(6, 1400, seed=1), _teacher(3, 700, 6, 1.0, seed=2)
    for view in (wide[::2, 1:701], wide[:3, :1400:2]):
        leaf = wide.clone().requires_grad_(True)
        sub = leaf[::2, 1:701] if view.stride(1) == 1 else leaf[:3, :1400:2]
        g, = torch.autograd.grad(distillation_loss(sub, top), leaf)
        flat = view.contiguous().requires_grad_(True)
        ref, = torch.autograd.grad(distillation_loss(flat, top), flat)
        got = g[::2, 1:701] if view.stride(1) == 1 else g[:3, :1400:2]
        assert torch.equal(got, ref)
    empty = _rand(0, 700).requires_grad_(True)
    loss = distillation_loss(empty, TopLogits(top.values[:0], top.moves[:0], top.log_rest[:0]), reduction="sum")
    assert float(loss) == 0 and torch.autograd.grad(loss, empty)[0].shape == (0, 700)


def test_refusals():
    x = _rand(3, 50)
    top = top_logits(x, 4)
    for bad in (0, 257):
        with pytest.raises(ValueError, match="between 1 and 256"):
            top_logits(x, bad)
    with pytest.raises(ValueError, match="temperature"):
        top_logits(x, 4, 0.0)
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        top_logits(x.double(), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        top_logits(x.cpu(), 4)
    with pytest.raises(ValueError, match="legal moves"):
        top_logits(x, 4, legal=(torch.zeros(2, 5, dtype=torch.int64, device=DEV), torch.zeros(2, 5, dtype=torch.bool, device=DEV)))
    with pytest.raises(ValueError, match="legal valid"):
        top_logits(x, 4, legal=(torch.zeros(3, 5, dtype=torch.int64, device=DEV), torch.zeros(3, 4, dtype=torch.bool, device=DEV)))
    with pytest.raises(ValueError, match="top.values"):
        distillation_loss(x[:2], top)
    with pytest.raises(ValueError, match="reduction"):
        distillation_loss(x, top, reduction="max")
    with pytest.raises(ValueError, match="weight"):
        distillation_loss(x, top, weight=torch.ones(2, device=DEV))
    from alphafly_b200 import _lib
    with pytest.raises(_lib.AfbError, match="4096 listed"):
        top_logits(x, 4, legal=(torch.zeros(3, 4097, dtype=torch.int64, device=DEV), torch.zeros(3, 4097, dtype=torch.bool, device=DEV)))
