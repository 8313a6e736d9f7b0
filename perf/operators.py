"""Cases of the 8-bit product and of the distillation operators, for timing and comparison.

``own`` False: the operators' plain form in elementary torch operations, 32 bits; True: the package's entry points
(``alphafly_b200.int8``, ``alphafly_b200.distill``).  ``exact`` has the definitions in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
N_MOVES = 4168          # policy indices of the network
N_OUT = 2333            # output neurons
N_IN = 17937            # sensory neurons
N_BASE = 838            # board features
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}


def _int8(name, rows, k, n, x, out, layout, bias=True):
    return {"name": name, "op": "int8", "rows": rows, "k": k, "n": n, "x": x, "out": out, "layout": layout, "bias": bias}


def _top(name, rows, v, k, x, temperature, listed_moves=0):
    return {"name": name, "op": "top", "rows": rows, "v": v, "k": k, "x": x, "temperature": temperature, "legal": listed_moves}


def _distill(name, rows, v, k, x, temperature, rest, train, listed_moves=0, weighted=False):
    return {"name": name, "op": "distill", "rows": rows, "v": v, "k": k, "x": x, "temperature": temperature, "rest": rest,
            "train": train, "legal": listed_moves, "weighted": weighted}


def listed():
    return [
        # one leaf of a search through the readout: latency
        _int8("int8 leaf readout", 1, N_OUT, N_MOVES + 3, "float32", "float32", "rows"),
        # a self-play round through the readout, the state as the recurrence leaves it (neurons, positions)
        _int8("int8 round readout", 1120, N_OUT, N_MOVES + 3, "float32", "float32", "columns"),
        # the input map of a training batch
        _int8("int8 batch input map", 2048, N_BASE, N_IN, "float16", "float16", "rows"),
        # a teacher over a pool of positions
        _int8("int8 pool readout", 35840, N_OUT, N_MOVES + 3, "float32", "float16", "rows"),
        # the best moves of one position
        _top("top single", 1, N_MOVES, 16, "float32", 1.0),
        # a self-play round, over each position's legal moves
        _top("top round legal", 1120, N_MOVES, 8, "float16", 1.0, 64),
        # the targets of a pool of positions
        _top("top pool", 35840, N_MOVES, 32, "float32", 2.0),
        # a larger vocabulary in a type with many equal values
        _top("top wide", 2048, 32000, 64, "bfloat16", 1.0),
        # a validation chunk: losses of the positions
        _distill("distill validation", 256, N_MOVES, 16, "float32", 1.0, False, False),
        # the training batch, the teacher's remaining moves as one class
        _distill("distill batch", 2048, N_MOVES, 32, "float32", 2.0, True, True),
        # the training batch over legal moves only, positions weighted
        _distill("distill batch legal", 2048, N_MOVES, 8, "float32", 1.0, False, True, 64, True),
        # a larger vocabulary
        _distill("distill wide", 4096, 32000, 64, "bfloat16", 2.0, True, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["int8", "top", "distill"])
    x = rng.choice(["float32", "float16", "bfloat16"])
    if op == "int8":
        k, n = _log(rng, 32, 4500), _log(rng, 16, 18000)
        rows = _log(rng, 1, max(1, min(35840, 300_000_000_000 // (k * n))))
        return {"op": op, "rows": rows, "k": k, "n": n, "x": x, "out": rng.choice(["float32", "float16", "bfloat16"]),
                "layout": rng.choice(["rows", "rows", "columns"]), "bias": rng.random() < 0.7}
    v = N_MOVES if rng.random() < 0.4 else _log(rng, 100, 40000)
    rows = _log(rng, 1, min(35840, 130_000_000 // v))
    k = min(_log(rng, 1, 128), v // 2)
    case = {"op": op, "rows": rows, "v": v, "k": k, "x": x, "temperature": rng.choice([1.0, 2.0, 0.5, round(rng.uniform(0.7, 4.0), 2)]),
            "legal": rng.choice([0, 0, min(v, _log(rng, 20, 218))])}
    if op == "distill":
        case.update(rest=rng.random() < 0.5, train=rng.random() < 0.75, weighted=rng.random() < 0.3)
    return case


# -- inputs -------------------------------------------------------------------------------------------------

def _padded_rows(rows, k):
    """(rows, k) int8 whose rows start on 16-byte boundaries, as the package's ``quantize`` lays them out."""
    return torch.zeros(rows, -(-k // 16) * 16, dtype=torch.int8, device=DEV)[:, :k]


def _legal_lists(rows, v, most, gen):
    """Move lists as a training batch holds them: distinct moves, 0 in the padding; about 1 row in 40 has none."""
    moves = torch.empty(rows, most, dtype=torch.int64, device=DEV)
    for lo in range(0, rows, 4096):
        part = moves[lo:lo + 4096]
        part.copy_(torch.rand(part.shape[0], v, device=DEV, generator=gen).argsort(1)[:, :most])
    count = (torch.rand(rows, 1, device=DEV, generator=gen) * most).long() + 1
    count[torch.rand(rows, 1, device=DEV, generator=gen) < 0.025] = 0
    valid = torch.arange(most, device=DEV) < count
    return moves.masked_fill_(~valid, 0), valid


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rows = case["rows"]
    if case["op"] == "int8":
        k, n = case["k"], case["n"]
        shape = (rows, k) if case["layout"] == "rows" else (k, rows)
        # normalised neuron activity, clipped like RunningNorm's output; positions differ in magnitude
        x = torch.randn(shape, device=DEV, generator=gen).mul_(1.5).clamp_(-8, 8)
        if case["layout"] == "columns":
            x = x.T
        x = x * (0.25 + torch.rand(rows, 1, device=DEV, generator=gen))
        x = x.to(DTYPES[case["x"]])
        w = torch.randn(n, k, device=DEV, generator=gen) * (0.5 + torch.rand(n, 1, device=DEV, generator=gen)) * k ** -0.5
        w_scale = w.abs().amax(1) / torch.full((n,), 127.0, device=DEV)
        wq = _padded_rows(n, k)
        wq.copy_((w / w_scale[:, None]).round())
        bias = torch.randn(n, device=DEV, generator=gen) * 0.3 if case["bias"] else None
        return {"case": case, "x": x, "wq": wq, "w_scale": w_scale, "bias": bias}
    v, dtype = case["v"], DTYPES[case["x"]]
    legal = _legal_lists(rows, v, case["legal"], gen) if case["legal"] else None
    teacher = torch.randn(rows, v, device=DEV, generator=gen).mul_(2.0).to(dtype)
    if case["op"] == "top":
        return {"case": case, "logits": teacher, "legal": legal}
    # a student that agrees with its teacher in part
    student = (teacher.float() * 0.6 + torch.randn(rows, v, device=DEV, generator=gen)).to(dtype)
    values, moves, log_rest = _plain_top(teacher, case["k"], case["temperature"], legal)
    del teacher
    weight = torch.rand(rows, device=DEV, generator=gen) * 2 if case["weighted"] else None
    return {"case": case, "logits": student.requires_grad_(case["train"]), "top": (values, moves, log_rest), "legal": legal, "weight": weight}


# -- plain forms --------------------------------------------------------------------------------------------

def _plain_int8(state):
    case = state["case"]
    x = state["x"].float()
    s = x.abs().amax(1) / torch.full((x.shape[0],), 127.0, device=x.device)
    q = (x / s[:, None]).round()
    y = (q @ state["wq"].float().T) * s[:, None] * state["w_scale"]
    if state["bias"] is not None:
        y = y + state["bias"]
    return y.to(DTYPES[case["out"]])


def _support(shape, legal):
    """(rows, v) bool: the moves that take part."""
    if legal is None:
        return torch.ones(shape, dtype=torch.bool, device=DEV)
    moves, valid = legal
    return torch.zeros(shape, dtype=torch.int32, device=DEV).scatter_add_(1, moves, valid.int()) > 0


def _log_sum_exp(x):
    """Over dim 1; -inf for a row of -inf."""
    m = x.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    return (m + (x - m).exp().sum(1, keepdim=True).log()).squeeze(1)


def _plain_top(logits, k, temperature, legal):
    x = logits.float()
    if legal is not None:
        x = torch.where(_support(x.shape, legal), x, -math.inf)
    values, moves = torch.sort(x, dim=1, descending=True, stable=True)
    rest = values[:, k:] / temperature
    values, moves = values[:, :k].contiguous(), moves[:, :k]
    moves = torch.where(values == -math.inf, -1, moves)
    log_rest = _log_sum_exp(rest) if rest.shape[1] else torch.full_like(values[:, 0], -math.inf)
    return values, moves, log_rest


def _softplus(d):
    """log(1 + exp(d))"""
    return d.clamp(min=0) + (-d.abs()).exp().log1p()


def _plain_distill(state):
    case, weight = state["case"], state["weight"]
    t, named, log_rest = state["top"]
    temp = case["temperature"]
    logits = state["logits"].detach()
    support = _support(logits.shape, state["legal"])
    s = torch.where(support, logits.float() / temp, -math.inf)
    at = named.clamp(min=0)
    kept = (named >= 0) & support.gather(1, at)
    some = kept.any(1)
    # the teacher over its named moves, the student over all
    z = torch.where(kept, t / temp, -math.inf)
    lse_z = torch.where(some, _log_sum_exp(z), 0.0)
    log_p = z - lse_z[:, None]
    s_at = torch.where(kept, s.gather(1, at), -math.inf)
    lse = torch.where(some, _log_sum_exp(s), 0.0)
    log_q = s_at - lse[:, None]
    loss_rest = 0.0
    if case["rest"]:
        # the moves it does not name as one class: log of its share = -softplus(log odds of the named moves)
        is_named = torch.zeros(s.shape, dtype=torch.int32, device=DEV).scatter_add_(1, at, kept.int()) > 0
        lse_rest = _log_sum_exp(torch.where(is_named, -math.inf, s))
        odds_p, odds_q = lse_z - log_rest, torch.where(some, _log_sum_exp(s_at), 0.0) - lse_rest
        log_p = log_p - _softplus(-odds_p)[:, None]
        p_rest = (-_softplus(odds_p)).exp()
        loss_rest = torch.where(p_rest > 0, p_rest * (_softplus(odds_q) - _softplus(odds_p)), 0.0)
    p = log_p.exp()
    loss = torch.where(p > 0, p * (log_p - log_q), 0.0).sum(1) + loss_rest
    loss = torch.where(some, loss, 0.0) * (temp * temp)
    if weight is not None:
        loss = loss * weight
    if not case["train"]:
        return loss
    ds = (s - lse[:, None]).exp() - torch.zeros_like(s).scatter_add_(1, at, p)
    if case["rest"]:
        safe = torch.where(lse_rest == -math.inf, 0.0, lse_rest)
        ds = ds - torch.where(is_named, 0.0, p_rest[:, None] * (s - safe[:, None]).exp())
    ds = torch.where(some[:, None], ds, 0.0) * (temp / s.shape[0])
    if weight is not None:
        ds = ds * weight[:, None]
    return loss.mean(), ds.to(logits.dtype)


def run(state):
    case = state["case"]
    if case["op"] == "int8":
        if not own:
            return _plain_int8(state)
        from alphafly_b200.int8 import int8_linear
        return int8_linear(state["x"], state["wq"], state["w_scale"], state["bias"], out_dtype=DTYPES[case["out"]])
    if case["op"] == "top":
        if not own:
            return _plain_top(state["logits"], case["k"], case["temperature"], state["legal"])
        from alphafly_b200.distill import top_logits
        top = top_logits(state["logits"], case["k"], temperature=case["temperature"], legal=state["legal"])
        return top.values, top.moves, top.log_rest
    if not own:
        return _plain_distill(state)
    from alphafly_b200.distill import TopLogits, distillation_loss
    top = TopLogits(*state["top"], case["temperature"])
    if not case["train"]:
        return distillation_loss(state["logits"], top, legal=state["legal"], rest=case["rest"], weight=state["weight"], reduction="none")
    loss = distillation_loss(state["logits"], top, legal=state["legal"], rest=case["rest"], weight=state["weight"])
    return loss.detach(), torch.autograd.grad(loss, state["logits"])[0]


def work(case):
    rows = case["rows"]
    if case["op"] == "int8":
        k, n = case["k"], case["n"]
        return {"bytes": rows * k * SIZE[case["x"]] + n * k + (8 if case["bias"] else 4) * n + rows * n * SIZE[case["out"]],
                "flops": 2 * rows * k * n}
    v, k, size, most = case["v"], case["k"], SIZE[case["x"]], case["legal"]
    read = rows * (most * (9 + size) if most else v * size)      # the lists and their logits, or all logits
    taken = rows * (most or v)
    targets = rows * (12 * k + 4)
    if case["op"] == "top":
        return {"bytes": read + targets, "flops": 4 * taken}
    out = rows * v * size + 4 if case["train"] else 4 * rows
    return {"bytes": read + targets + out + (4 * rows if case["weighted"] else 0), "flops": (8 if case["train"] else 4) * taken}


# -- the definitions in 64 bits -----------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "int8":
        return _exact_int8(state)
    return _exact_top(state) if case["op"] == "top" else _exact_distill(state)


def _exact_int8(state):
    """The quantiser's own roundings (scale and quotient to 32 bits, then to the nearest even whole number) are part
    of the definition; everything after them is exact."""
    x = state["x"].double()
    scale = (x.abs().max(dim=1).values / 127.0).float().double()
    whole = torch.round((x / scale[:, None]).float().double())
    y = torch.einsum("ik,jk->ij", whole, state["wq"].double())
    y *= scale[:, None]
    y *= state["w_scale"].double()[None]
    return y if state["bias"] is None else y + state["bias"].double()


def _sortable(x):
    """32-bit floats -> whole numbers in the same order (no NaN)."""
    bits = x.float().view(torch.int32).long()
    return torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))


def _takes_part(state):
    """(rows, v) bool from the lists, row by row of the list's columns."""
    rows, v = state["logits"].shape
    if state["legal"] is None:
        return None
    moves, valid = state["legal"]
    on = torch.zeros(rows, v, dtype=torch.bool, device=DEV)
    r, c = valid.nonzero(as_tuple=True)
    on[r, moves[r, c]] = True
    return on


def _exact_top(state):
    case, x = state["case"], state["logits"].detach()
    rows, v = x.shape
    k, on = case["k"], _takes_part(state)
    order = _sortable(x) * v + (v - 1 - torch.arange(v, device=DEV))      # one key a move: ties to the lowest
    never = torch.iinfo(torch.int64).min
    if on is not None:
        order = torch.where(on, order, never)
    best, moves = torch.topk(order, k, dim=1, sorted=True)
    values = x.double().gather(1, moves)
    gone = best == never
    values = values.masked_fill(gone, -math.inf)
    left = torch.ones(rows, v, dtype=torch.bool, device=DEV) if on is None else on
    left = left.scatter(1, moves, False)
    z = (x.double() / case["temperature"]).masked_fill(~left, -math.inf)
    return values, moves.masked_fill(gone, -1), torch.logsumexp(z, 1)


def _exact_distill(state):
    case = state["case"]
    temp = case["temperature"]
    s = state["logits"].detach().double() / temp
    on = _takes_part(state)
    if on is not None:
        s = s.masked_fill(~on, -math.inf)
    t, named, log_rest = (a.double() if a.is_floating_point() else a for a in state["top"])
    rows, v = s.shape
    # the teacher's distribution as a dense target, and what it leaves to the other moves
    z = torch.full((rows, v + 1), -math.inf, dtype=torch.float64, device=DEV)
    r, c = (named >= 0).nonzero(as_tuple=True)
    z[r, named[r, c]] = t[r, c] / temp
    if on is not None:
        z[:, :v] = z[:, :v].masked_fill(~on, -math.inf)
    if case["rest"]:
        z[:, v] = log_rest
    alive = (z[:, :v] > -math.inf).any(1) & (s > -math.inf).any(1)
    chosen = z[:, :v] > -math.inf
    p = torch.softmax(z, 1)
    log_q = torch.log_softmax(s, 1)
    log_q_rest = torch.logsumexp(log_q.masked_fill(chosen, -math.inf), 1) if case["rest"] else torch.zeros(rows, dtype=torch.float64, device=DEV)
    both = torch.cat([log_q, log_q_rest[:, None]], 1)
    terms = torch.xlogy(p, p) - torch.where(p > 0, p * both, 0.0)
    loss = torch.where(alive, terms.sum(1), 0.0) * temp ** 2
    w = torch.ones(rows, dtype=torch.float64, device=DEV) if state["weight"] is None else state["weight"].double()
    if not case["train"]:
        return loss * w
    grad = log_q.exp() - p[:, :v]
    if case["rest"]:
        inside = torch.where(chosen, 0.0, (log_q - log_q_rest[:, None]).exp())
        grad = grad - p[:, v:] * inside
    if on is not None:
        grad = grad.masked_fill(~on, 0.0)
    grad = torch.where(alive[:, None], grad, 0.0) * (w[:, None] * temp / rows)
    return (loss * w).mean(), grad
