"""Every kernel that the selection and the loss choose between, by its rule's sizes, against the definitions in 64 bits:
rows too long for shared memory, more rows than the device holds at once, rows that leave the common path among others,
lists around the length from which a bound is sought."""

import math

import pytest
import torch

from alphafly_b200.distill import TopLogits, distillation_loss, top_logits

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF_ULP = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}
INF = math.inf


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(*shape, seed=0):
    return torch.randn(*shape, device=DEV, generator=_gen(seed))


def _on(shape, legal):
    """(rows, moves) bool: the moves that take part."""
    if legal is None:
        return torch.ones(shape, dtype=torch.bool, device=DEV)
    moves, valid = legal
    ok = valid & (moves >= 0) & (moves < shape[1])
    on = torch.zeros(shape, dtype=torch.int32, device=DEV)
    return on.scatter_add_(1, moves.clamp(0, shape[1] - 1), ok.int()) > 0


def _check_top(logits, k, temperature=1.0, legal=None):
    top = top_logits(logits, k, temperature, legal)
    v = logits.shape[1]
    x = logits.double()
    x = torch.where(_on(x.shape, legal) & ~x.isnan(), x, -INF)
    best, moves = torch.sort(x, dim=1, descending=True, stable=True)         # ties to the lower move
    n = min(k, v)
    values = torch.full_like(top.values, -INF)
    values[:, :n] = best[:, :n].float()
    at = torch.full_like(top.moves, -1)
    at[:, :n] = torch.where(best[:, :n] > -INF, moves[:, :n], -1)
    assert torch.equal(top.values, values) and torch.equal(top.moves, at)
    rest = torch.logsumexp(best[:, n:] / temperature, 1) if v > n else torch.full((len(x),), -INF, dtype=torch.float64, device=DEV)
    got, fine = top.log_rest.double(), torch.isfinite(rest)
    assert torch.equal(got[~fine], rest[~fine])
    # the largest exponent's product, the terms' exponents and their sum: a few roundings of values up to |rest| + 20
    assert bool(((got - rest).abs() <= 2.0**-21 * (rest.abs() + 20))[fine].all())
    return top


@pytest.mark.parametrize("rows,v,dtype", [(300, 12000, F32), (300, 20000, F32), (260, 32000, BF16), (260, 60000, F16), (255, 32000, F32)])
@pytest.mark.parametrize("k", [1, 30, 50, 64, 90, 130, 256])
def test_selection_from_long_rows(rows, v, dtype, k):
    """256 and 512 threads a row, one warp or all of them ranking."""
    x = (_rand(rows, v, seed=k) * 2).to(dtype)
    x[::3] = (x[::3].float() * 4).round().to(dtype) / 4                      # many equal values
    x[1, 5:] = -INF
    x[2] = -INF
    _check_top(x, k, 1.3)


@pytest.mark.parametrize("listed", [31, 32, 33, 63, 64, 65, 71, 72, 73, 96, 127, 128, 129, 250])
@pytest.mark.parametrize("k", [1, 8, 60])
def test_selection_from_lists_around_the_bound(listed, k):
    rows, v = 300, 700
    x = (_rand(rows, v, seed=listed) * 3).half()
    x[::2] = x[::2].round()
    moves = torch.rand(rows, v, device=DEV, generator=_gen(k)).argsort(1)[:, :listed].contiguous()
    valid = torch.rand(rows, listed, device=DEV, generator=_gen(3)) < 0.8
    valid[0], valid[1] = False, True
    moves[2] = moves[2, 0]                                                    # one move over and over
    moves[3, 0], moves[3, listed // 2] = v, -5
    _check_top(x, k, 0.7, (moves, valid))


def _loss64(s, top, on, rest):
    """Losses of the rows in 64 bits, and the three parts whose sum of magnitudes bounds the gradient's rounding (without
    the temperature): the student's shares, the teacher's, and the teacher's rest spread like the student's."""
    t = top.temperature
    v = s.shape[1]
    at = top.moves.clamp(0, v - 1)
    kept = (top.moves >= 0) & (top.moves < v) & (top.values > -INF) & on.gather(1, at)
    first = torch.full((len(s), v), top.moves.shape[1], dtype=torch.int64, device=DEV)        # a move counts where it is named first
    place = torch.arange(top.moves.shape[1], device=DEV).expand_as(at)
    first.scatter_reduce_(1, at, torch.where(kept, place, top.moves.shape[1]), "amin")
    kept &= first.gather(1, at) == place
    z = torch.full((len(s), v + 1), -INF, dtype=torch.float64, device=DEV)
    r, c = kept.nonzero(as_tuple=True)
    z[r, at[r, c]] = top.values[r, c].double() / t
    named = z[:, :v] > -INF
    if rest:
        z[:, v] = top.log_rest.double()
    x = (s / t).masked_fill(~on, -INF)
    alive = kept.any(1) & (x > -INF).any(1)
    log_q = torch.log_softmax(torch.where(alive[:, None], x, 0.0), 1)
    log_rest = torch.zeros(len(s), dtype=torch.float64, device=DEV)
    if rest:                                         # of the moves that are not named; a row may have none (then p holds none)
        others = (log_q > -INF) & ~named
        some = others.any(1)
        log_rest = torch.where(some, torch.logsumexp(torch.where(some[:, None], log_q.masked_fill(~others, -INF), 0.0), 1), 0.0)
    z = torch.where(alive[:, None], z, 0.0)
    p, log_p = torch.softmax(z, 1), torch.log_softmax(z, 1)
    terms = torch.where(p > 0, p * (log_p - torch.cat([log_q, log_rest[:, None]], 1)), 0.0)
    q = log_q.detach().exp()
    spread = p[:, v:] * torch.where(named | (q == 0), 0.0, (log_q.detach() - log_rest.detach()[:, None]).exp()) if rest else 0.0
    shares = torch.where(alive[:, None], q + p[:, :v] + spread, 0.0)
    return torch.where(alive, terms.sum(1), 0.0) * t * t, shares


def _check_loss(s, top, legal=None, rest=False, weight=None, upstream=None):
    """The kernel's losses and gradient against the 64-bit ones.  Each log share comes from exponents of size up to A = 64
    in float32, (A + 4) 2^-22 < 2e-5 of a share; a loss term adds the rounding of its logarithms."""
    b, t = s.shape[0], top.temperature
    on = _on(s.shape, legal)
    leaf = s.detach().clone(memory_format=torch.preserve_format).requires_grad_(True) if s.is_contiguous() else s.detach().requires_grad_(True)
    losses = distillation_loss(leaf, top, legal, rest, weight, reduction="none")
    s64 = s.detach().double().requires_grad_(True)
    ref, shares = _loss64(s64, top, on, rest)
    w = torch.ones(b, dtype=torch.float64, device=DEV) if weight is None else weight.double()
    u = torch.ones(b, device=DEV) if upstream is None else upstream
    size = s.detach().double().masked_fill(~on, 0.0).abs().amax(1)
    assert bool(((losses.detach().double() - (ref * w).detach()).abs() <= 2.0**-20 * (size / t + 20) * t * t * w).all())
    grad, = torch.autograd.grad(losses, leaf, u)
    ref_grad, = torch.autograd.grad((ref * w * u.double()).sum(), s64)
    step = {F16: 2.0**-25}.get(s.dtype, 0.0)
    limit = 2e-5 * shares * t * (w * u.double().abs())[:, None] + HALF_ULP[s.dtype] * ref_grad.abs() * 1.01 + step + 1e-37
    assert grad.dtype == s.dtype and bool(((grad.double() - ref_grad).abs() <= limit).all())
    assert not grad[~on].any()
    mean = distillation_loss(leaf, top, legal, rest, weight)
    assert abs(float(mean) - float((ref * w).mean())) <= 2.0**-20 * float(((size / t + 20) * t * t * w).mean())
    g, = torch.autograd.grad(mean, leaf)
    ref_mean, = torch.autograd.grad((_loss64(s64, top, on, rest)[0] * w).mean(), s64)
    limit = 2e-5 * shares * t / b * w[:, None] + HALF_ULP[s.dtype] * ref_mean.abs() * 1.01 + step + 1e-37
    assert bool(((g.double() - ref_mean).abs() <= limit).all())


def _teacher(b, v, k, t, seed, legal=None):
    return top_logits(_rand(b, v, seed=seed) * 2, k, t, legal)


# 28,000 float32 or 56,000 16-bit moves are read twice from memory; 10,241 and 20,481 take 256 threads
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("v,dtype", [(10000, F32), (27000, F32), (29001, F32), (32000, F32), (12000, F16), (32000, BF16), (55000, BF16), (60001, F16), (64000, BF16)])
def test_loss_over_long_rows(v, dtype, rest):
    s = (_rand(6, v, seed=v) * 1.5).to(dtype)
    _check_loss(s, _teacher(6, v, 64, 2.0, seed=1), None, rest, upstream=torch.tensor([1.0, 2.0, 1.0, 0.0, -3.0, 0.5], device=DEV))
    _check_loss(s[:1], _teacher(1, v, 1, 1.0, seed=2), None, rest)


@pytest.mark.parametrize("v,dtype", [(4168, F32), (3001, F32), (32000, F32), (3001, F16), (32001, BF16), (60001, F16)])
@pytest.mark.parametrize("offset", [1, 3])
def test_loss_over_rows_off_any_boundary(v, dtype, offset):
    wide = (_rand(5, v + 9, seed=v) * 1.5).to(dtype)
    _check_loss(wide[:, offset:offset + v], _teacher(5, v, 20, 1.5, seed=3), None, True)


@pytest.mark.parametrize("v,dtype", [(600, F32), (4168, F16), (32000, F32), (60001, BF16)])
@pytest.mark.parametrize("rest", [False, True])
def test_loss_of_rows_that_leave_the_common_path(v, dtype, rest):
    """Between rows that do not, with named moves that repeat, are out of range or not there."""
    b, k = 12, 9
    s, top = (_rand(b, v, seed=v) * 1.5).to(dtype), _teacher(b, v, k, 1.0, seed=4)
    moves, values = top.moves.clone(), top.values.clone()
    lowest = torch.finfo(dtype).min
    moves[0] = -1                                    # names nothing
    moves[2, 3:6] = moves[2, 1]                      # a move four times
    moves[3, 0] = v + 2                              # the first out of range
    moves[4, 0] = moves[4, 1]                        # the first twice
    values[5, 1:] = -INF
    s[6] = -INF                                      # nothing to choose from
    s[7, v // 2:] = -INF                             # a mask of half of the moves ...
    moves[7] = torch.arange(k, device=DEV)           # ... the named ones outside it
    s[8, v // 2:] = lowest                           # the type's lowest value as a mask
    moves[8] = torch.arange(k, device=DEV)
    values[9] -= 60.0                                # the rest far above the named moves
    s[10] -= 50.0
    top = TopLogits(values, moves, top.log_rest, 1.0)
    on = _on(s.shape, None)
    ref, shares = _loss64(s.double(), top, on, rest)
    leaf = s.clone().requires_grad_(True)
    up = torch.where(torch.arange(b, device=DEV) % 2 == 0, 1.0, 3.0)
    losses = distillation_loss(leaf, top, rest=rest, reduction="none")
    grad, = torch.autograd.grad(losses, leaf, up)
    assert torch.isfinite(losses).all() and torch.isfinite(grad).all()
    assert not losses[[0, 6]].any() and not grad[[0, 6]].any()
    size = torch.where(s > lowest / 2, s.double(), 0.0).abs().amax(1)
    assert bool(((losses.double() - ref).abs() <= 2.0**-20 * (size + 80)).all())
    s64 = torch.where(s == -INF, -1e30, s.double()).requires_grad_(True)     # differentiable where the student's share is 0
    ref_grad, = torch.autograd.grad((_loss64(s64, top, on, rest)[0] * up.double()).sum(), s64)
    ref_grad[6] = 0.0
    step = {F16: 2.0**-25}.get(dtype, 0.0)
    limit = 2e-5 * shares * up.double()[:, None] + HALF_ULP[dtype] * ref_grad.abs() * 1.01 + step + 1e-37
    assert bool(((grad.double() - ref_grad).abs() <= limit).all())


@pytest.mark.parametrize("rows,v,k,dtype,rest", [(20000, 300, 7, F32, True), (9000, 1001, 12, F16, True), (3000, 4168, 32, F32, True),
                                                 (6000, 4168, 8, BF16, False), (1500, 8000, 16, F32, True), (1200, 12000, 16, BF16, True)])
def test_loss_of_more_rows_than_the_device_holds(rows, v, k, dtype, rest):
    """A CTA takes several rows: the next one's copy, its named moves, the marks of the last; every 7th row names a move
    twice, every 11th leaves the common path, upstream gradients of 1 and others mixed."""
    s, top = (_rand(rows, v, seed=rows) * 1.5).to(dtype), _teacher(rows, v, k, 2.0, seed=5)
    top.moves[::7, 1] = top.moves[::7, 0]
    top.moves[::13] = top.moves[::13].flip(1)
    s[::11] -= 300.0 if dtype == F32 else 40.0
    top.moves[5::11, 0] = -1
    weight = torch.rand(rows, device=DEV, generator=_gen(6))
    up = torch.where(torch.rand(rows, device=DEV, generator=_gen(7)) < 0.5, 1.0, 2.5)
    leaf = s.clone().requires_grad_(True)
    on = _on(s.shape, None)
    losses = distillation_loss(leaf, top, rest=rest, weight=weight, reduction="none")
    grad, = torch.autograd.grad(losses, leaf, up)
    s64 = s.double().requires_grad_(True)
    ref, shares = _loss64(s64, top, on, rest)
    ref_grad, = torch.autograd.grad((ref * weight * up.double()).sum(), s64)
    t, size = top.temperature, s.double().abs().amax(1)
    assert bool(((losses.double() - ref * weight).abs() <= 2.0**-20 * (size / t + 20) * t * t * weight).all())
    # a logit's exponent is as exact as the logit over T: its size comes before the shift by the row's largest
    a = 2e-5 + 2.0**-22 * size / t
    limit = (a * (weight * up).double())[:, None] * shares * t + HALF_ULP[dtype] * ref_grad.abs() * 1.01 + {F16: 2.0**-25}.get(dtype, 0.0) + 1e-37
    assert bool(((grad.double() - ref_grad).abs() <= limit).all())


@pytest.mark.parametrize("rows,v,listed,k,dtype", [(4000, 4168, 64, 8, F32), (5000, 900, 40, 200, F16), (700, 20000, 500, 32, BF16), (40, 5000, 4096, 256, F32)])
@pytest.mark.parametrize("rest", [False, True])
def test_loss_over_lists_of_many_rows(rows, v, listed, k, dtype, rest):
    """Lists with repeated, invalid and out-of-range moves; named moves that repeat or are not listed."""
    s = (_rand(rows, v, seed=listed) * 1.5).to(dtype)
    moves = torch.randint(0, v, (rows, listed), device=DEV, generator=_gen(1))
    valid = torch.rand(rows, listed, device=DEV, generator=_gen(2)) < 0.8
    moves[::5, 1] = v
    moves[::6, 0] = -1
    valid[3::17] = False
    top = top_logits(_rand(rows, v, seed=9) * 2, k, 1.5, (moves, valid))
    top.moves[::7, k // 2] = top.moves[::7, 0]
    top.moves[1::9, 0] = torch.randint(0, v, (len(top.moves[1::9]),), device=DEV, generator=_gen(3))
    up = torch.where(torch.rand(rows, device=DEV, generator=_gen(4)) < 0.5, 1.0, 0.25)
    _check_loss(s, top, (moves, valid), rest, torch.rand(rows, device=DEV, generator=_gen(5)), up)


@pytest.mark.parametrize("t", [0.5, 1.0, 2.0])
@pytest.mark.parametrize("v,listed", [(600, 0), (600, 60), (32000, 0)])
@pytest.mark.parametrize("rest", [False, True])
def test_teachers_masked_by_the_lowest_value(t, v, listed, rest):
    """A teacher whose illegal moves hold the type's lowest value, in one row all of them: over a temperature below 1 they leave
    float32's range."""
    teacher, s = _rand(5, v, seed=1) * 2, _rand(5, v, seed=2) * 1.5
    lowest = torch.finfo(F32).min
    teacher[0] = lowest
    teacher[1, 30:] = lowest
    teacher[2, 3:] = lowest
    legal = None
    if listed:
        legal = torch.arange(listed, device=DEV).repeat(5, 1), torch.ones(5, listed, dtype=torch.bool, device=DEV)
    top = top_logits(teacher, 8, t, legal)
    assert (top.moves >= 0).all() and not top.log_rest.isnan().any()
    _check_loss(s, top, legal, rest)
