"""A network that is evaluated in inference mode, trained, and evaluated again in any mode."""

import numpy as np
import pytest
import torch

from alphafly_b200 import gemm, synth
from alphafly_b200.distill import teacher_targets
from alphafly_b200.encoding import N_FEATURES
from alphafly_b200.model import Evaluator, FlyChessNet, ModelConfig

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _net(dtype, heads):
    gen = torch.Generator().manual_seed(2)
    net = FlyChessNet(synth.tiny(60, 600), ModelConfig(steps=3))
    with torch.no_grad():
        for p in (*net.encoder.parameters(), *net.policy.parameters(), *net.value.parameters()):
            p.normal_(0, 0.1, generator=gen)
    net = net.to(DEV).eval()
    net.infer_dtype, net.infer_heads = dtype, heads
    return net


@pytest.mark.parametrize("heads", ["float32", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_what_a_network_keeps_outlives_inference_mode(dtype, heads):
    net, fresh = _net(dtype, heads), _net(dtype, heads)
    x = (torch.rand(40, N_FEATURES, generator=torch.Generator().manual_seed(1)) < 0.05).half()
    xd, rows, cols = x.to(DEV), np.arange(40), np.arange(40) * 7
    gemm._status.clear()
    ev, fresh_ev = Evaluator(net, DEV), Evaluator(fresh, DEV)
    with torch.inference_mode():
        before = net(xd)[0].clone()
        legal = ev(x.numpy(), rows, cols)[0]
        assert torch.equal(teacher_targets(net, xd, 5).values, before.sort(1, descending=True).values[:, :5])
    with torch.no_grad():
        assert torch.equal(net(xd)[0], before)
        for n in (net, fresh):                   # a step of training
            for p in n.parameters():
                p.add_(0.01)
        after = net(xd)[0]
        assert not torch.equal(after, before) and torch.equal(after, fresh(xd)[0])
        moved = ev(x.numpy(), rows, cols)[0]
        assert np.array_equal(moved, fresh_ev(x.numpy(), rows, cols)[0]) and not np.array_equal(moved, legal)
    with torch.inference_mode():
        assert torch.equal(net(xd)[0], after)
    net._map_status(xd.device).fill_(4)
    assert net.device_status() == 4 and net.device_status() == 0
