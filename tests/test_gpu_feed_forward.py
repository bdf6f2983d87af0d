"""The linear layer, its gradients, the buckets, the clip and the orthogonalised step together,
as ``examples/feed_forward_muon.py`` runs them: against the same network in plain torch, recorded
against eager, and over enough steps for the loss to fall."""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from hybrid_training_amd import StepGraph

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "feed_forward_muon.py")


def _training(device, seed=0, **options):
    spec = importlib.util.spec_from_file_location("feed_forward_muon", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    torch.manual_seed(seed)
    return module.Training(**{**dict(width=96, hidden=260, blocks=2, tokens=150, device=device), **options})


def _fill(training, seed):
    gen = torch.Generator(device=training.x.device).manual_seed(seed)
    training.x.copy_(torch.randn(training.x.shape, device=training.x.device, generator=gen))
    training.target.copy_(torch.sin(training.x.float()))


def test_prediction_and_gradients_match_plain_torch(device):
    training = _training(device)
    _fill(training, 1)
    training.optimizer.step = lambda: None  # look at the packed, unclipped gradients
    training.max_norm = 0.0
    seen = {}
    training.optimizer.clip_grad_norm = lambda _: seen.update(
        {n: p.grad.clone() for n, p in training.network.named_parameters()})
    prediction = training.step()
    x = training.x.double()
    weights = {n: p.detach().double().requires_grad_(True) for n, p in training.network.named_parameters()}
    for b in range(2):
        hidden = torch.nn.functional.gelu(x @ weights[f"{b}.up.weight"].t() + weights[f"{b}.up.bias"], approximate="tanh")
        x = hidden @ weights[f"{b}.down.weight"].t() + weights[f"{b}.down.bias"] + x
    x = x @ weights["2.weight"].t() + weights["2.bias"]
    (x - training.target.double()).square().mean().backward()
    # float32 sums of a few hundred terms through five products: relative 1e-5
    assert float((prediction.double() - x).norm() / x.norm()) < 1e-5
    for name, w in weights.items():
        assert float((seen[name].double() - w.grad).norm() / w.grad.norm()) < 1e-5, name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_recorded_steps_equal_eager_ones(device, dtype):
    eager, recorded = _training(device, dtype=dtype), _training(device, dtype=dtype)
    for t in (eager, recorded):
        _fill(t, 1)
        t.step()
    graph = StepGraph(recorded.step)
    for k in range(2, 6):
        _fill(eager, k)
        _fill(recorded, k)
        want = eager.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(graph.output, want), k
        for p, q in zip(recorded.network.parameters(), eager.network.parameters()):
            assert torch.equal(p, q), k


def test_the_loss_falls(device):
    training = _training(device, tokens=512)
    losses = []
    for k in range(40):
        _fill(training, k)
        losses.append(training.loss(training.step()))
    assert sum(losses[-5:]) < 0.5 * sum(losses[:5])
