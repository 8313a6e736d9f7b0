"""A network learning from another one: the 8-bit readout of the teacher, its best moves as targets, and train_step
with them, on the small synthetic graph."""

import numpy as np
import pytest
import torch

from oracle import oracle as orc
from alphafly_b200 import synth
from alphafly_b200.distill import distillation_loss, teacher_targets
from alphafly_b200.encoding import N_MOVES
from alphafly_b200.model import Evaluator, FlyChessNet, ModelConfig, ShardedEvaluator
from alphafly_b200.train import Sample, TrainConfig, loss_terms, make_batch, make_optimizer, policy_cross_entropy, train_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _net(steps, seed):
    inst = synth.small()
    net = FlyChessNet(inst.conn, ModelConfig(steps=steps))
    synth.apply(net.brain, inst)
    w, b = synth.encoder_weights(len(inst.in_idx))
    gen = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        net.encoder.weight.copy_(torch.from_numpy(w))
        net.encoder.bias.copy_(torch.from_numpy(b))
        params = dict(net.named_parameters())
        for k, v in synth.head_weights(len(inst.out_idx)).items():
            params[k].copy_(torch.from_numpy(v))
        for name in ("policy_from.weight", "policy_to.weight"):
            params[name].normal_(0, 0.05, generator=gen)
    net = net.to(DEV)
    with torch.no_grad():                                 # the normaliser's statistics from a batch of boards
        r = net.brain_output(torch.from_numpy(synth.boards(256, seed=seed)).to(DEV)).T.float()
        net.norm.mean.copy_(r.mean(0))
        net.norm.var.copy_(r.var(0) + 1e-6)
        net.norm.initialised.fill_(True)
    return net.eval()


@pytest.fixture(scope="module")
def teacher():
    return _net(6, 3)


def _batch(b, seed, none=()):
    rng = np.random.default_rng(seed)
    x = synth.boards(b, seed).astype(np.float16)
    samples = []
    for i in range(b):
        idx = rng.choice(N_MOVES, 0 if i in none else int(rng.integers(1, 60)), replace=False)
        samples.append(Sample(x[i], idx, rng.dirichlet(np.ones(len(idx))) if len(idx) else np.zeros(0), float(rng.uniform(-1, 1)),
                              int(rng.integers(3))))
    return make_batch(samples, DEV)


def _int8_bound(r, w):
    """By how much an 8-bit product may be off: half a step of each factor, all of one sign."""
    s, t = r.abs().amax(1, keepdim=True) / 127, w.abs().amax(1, keepdim=True) / 127
    return s / 2 * w.abs().sum(1) + r.abs().sum(1, keepdim=True) * (t / 2).T + r.shape[1] * s * t.T / 4


@pytest.mark.parametrize("batch", [1, 5, 64, 300])
def test_int8_heads_are_within_their_steps(teacher, batch):
    x = torch.from_numpy(synth.boards(batch, seed=batch)).to(DEV)
    with torch.no_grad():
        out = teacher.brain_output(x)
        logits, wdl = teacher.int8_heads(out)
        r = teacher.norm(out.T.float()).double()
        w, b = (t.double() for t in teacher._folded())
        ref = r @ w.T + b
    assert logits.shape == (batch, N_MOVES) and wdl.shape == (batch, 3) and logits.dtype == torch.float32
    err = (torch.cat([logits, wdl], 1).double() - ref).abs()
    assert bool((err <= _int8_bound(r, w) * 1.001 + 1e-5).all())
    # the errors are independent, so their size is that of a random sum: sqrt(3 n) below the bound, tenfold allowed
    assert float(err.pow(2).mean().sqrt()) <= 10 * float(_int8_bound(r, w).pow(2).mean().sqrt()) / (3 * r.shape[1]) ** 0.5


def test_forward_and_evaluator_take_the_readout_that_is_set(teacher):
    x = synth.boards(70, seed=5).astype(np.float16)
    xd = torch.from_numpy(x).to(DEV)
    with torch.no_grad():
        plain, _ = teacher(xd)
        teacher.infer_heads = "int8"
        try:
            logits, wdl = teacher(xd)
            direct = teacher.int8_heads(teacher.brain_output(xd))
            assert torch.equal(logits, direct[0]) and torch.equal(wdl, direct[1]) and not torch.equal(logits, plain)
            rows, cols = np.repeat(np.arange(70), 4), np.random.default_rng(1).integers(0, N_MOVES, 280)
            ev = Evaluator(teacher, DEV)
            legal, values = ev(x, rows, cols)
            # the graph runs 256 positions, as does this (the recurrence rounds by its schedule, which goes by the batch)
            padded = torch.zeros(256, xd.shape[1], dtype=xd.dtype, device=DEV)
            padded[:70] = xd
            logits, wdl = (t[:70] for t in teacher(padded))
            np.testing.assert_allclose(legal, logits.cpu().numpy()[rows, cols], rtol=0, atol=0)
            np.testing.assert_allclose(values, teacher.expected_value(wdl).cpu().numpy(), rtol=1e-6, atol=1e-6)
            teacher.policy.bias.add_(1.0)                    # a training phase between rounds reaches the captured graph
            moved, _ = ev(x, rows, cols)
            np.testing.assert_allclose(moved, legal + 1.0, rtol=1e-6, atol=1e-5)
            teacher.policy.bias.sub_(1.0)
            sharded = ShardedEvaluator(teacher, [DEV])
            np.testing.assert_allclose(sharded(x, rows, cols)[0], ev(x, rows, cols)[0], rtol=0, atol=0)
            assert teacher.device_status() == 0
            teacher.infer_heads = "int4"
            with pytest.raises(ValueError, match="infer_heads"):
                teacher(xd)
        finally:
            teacher.infer_heads = "float32"
        assert torch.equal(teacher(xd)[0], plain)


@pytest.mark.parametrize("heads", ["float32", "int8"])
def test_teacher_targets_are_the_best_legal_moves(teacher, heads):
    batch = _batch(40, 7, none=(3,))
    teacher.infer_heads = heads
    try:
        top = teacher_targets(teacher, batch.x, 8, 1.5, legal=(batch.moves, batch.valid))
        with torch.no_grad():
            logits, _ = teacher(batch.x)
    finally:
        teacher.infer_heads = "float32"
    legal = logits.gather(1, batch.moves).masked_fill(~batch.valid, -float("inf"))
    best = legal.sort(1, descending=True)
    n = min(8, best.values.shape[1])
    assert torch.equal(top.values[:, :n], best.values[:, :n])
    assert torch.equal(logits.gather(1, top.moves.clamp(min=0))[top.moves >= 0], top.values[top.moves >= 0])
    rest = torch.logsumexp(best.values[:, 8:].double() / 1.5, 1)
    torch.testing.assert_close(top.log_rest.double(), rest, rtol=1e-6, atol=1e-5)
    assert top.temperature == 1.5 and (top.moves[3] == -1).all() and not teacher.training


@pytest.mark.parametrize("rest,share", [(False, 1.0), (True, 1.0), (True, 0.3)])
def test_train_step_with_a_teacher(teacher, rest, share):
    """The parameters' gradients against autograd through the plain float32 form of the loss on the same logits; the loss
    falls over a few steps."""
    student = _net(4, 11).train()
    batch = _batch(48, 9, none=(0, 17))
    top = teacher_targets(teacher, batch.x, 6, 2.0, legal=(batch.moves, batch.valid))
    net = _net(4, 11).train()
    logits, _ = net(batch.x)
    s = logits.gather(1, batch.moves).masked_fill(~batch.valid, -1e30) / 2.0
    named = (batch.moves[:, :, None] == top.moves[:, None]).to(logits.dtype) * batch.valid[:, :, None]     # (B, K, k)
    lse = torch.logsumexp(s, 1, keepdim=True)
    log_q = torch.einsum("bk,bkn->bn", s - lse, named)
    other = s.masked_fill(named.sum(2) > 0, -1e30)
    z = top.values / 2.0
    if rest:
        z = torch.cat([z, top.log_rest[:, None]], 1)
        log_q = torch.cat([log_q, torch.logsumexp(other, 1, keepdim=True) - lse], 1)
    alive = batch.valid.any(1)
    z = torch.where(alive[:, None], z, 0.0)
    log_p = torch.log_softmax(z, 1)
    p = log_p.exp()
    plain = torch.where((p > 0) & alive[:, None], p * (log_p - log_q), 0.0).sum(1).mean() * 4.0
    expected = share * plain + (1 - share) * policy_cross_entropy(logits, batch)
    expected.backward()
    opt = make_optimizer(student, TrainConfig())
    policy, value, _ = loss_terms(student, batch, 0.5, top, share, rest)
    assert abs(float(policy) - float(expected)) <= 1e-5 * abs(float(expected))
    policy.backward()
    for (name, a), (_, b) in zip(student.named_parameters(), net.named_parameters()):
        if b.grad is None or float(b.grad.abs().max()) == 0:
            assert a.grad is None or float(a.grad.abs().max()) < 1e-7, name
        else:
            assert orc.rel_l2(a.grad.cpu().numpy(), b.grad.cpu().numpy()) < 1e-4, name
    # the normaliser's statistics moved in the forward above; the steps go on from there
    losses = [train_step(student, opt, batch, DEV, q_ratio=0.5, teacher=top, teacher_share=share, teacher_rest=rest)["policy_loss"]
              for _ in range(12)]
    assert losses[-1] < losses[0] and all(np.isfinite(losses))
    assert student.device_status() == 0
    with torch.no_grad():
        per = distillation_loss(student(batch.x)[0], top, legal=(batch.moves, batch.valid), rest=rest, reduction="none")
    assert float(per[0]) == 0 and float(per[17]) == 0
