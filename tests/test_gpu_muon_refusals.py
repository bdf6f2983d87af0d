"""A refused orthogonalised step leaves parameters, step counters and state as they were."""

from __future__ import annotations

import copy

import pytest
import torch

from hybrid_training_amd import (
    NativeKernelError,
    OptimizerConfig,
    StepGraph,
    UnsupportedFeatureError,
    muon,
)
from hybrid_training_amd.errors import ConfigurationError

from .test_gpu_muon import build, set_grads

pytestmark = pytest.mark.gpu


def _optimizer(device, stepped):
    vector = torch.nn.Parameter(torch.ones(11, device=device))
    params, opt = build(device, [(32, 23), (130, 70)], others=[vector], others_config=OptimizerConfig(learning_rate=1e-3))
    vector.grad = torch.ones_like(vector)
    if stepped:
        opt.step()
        set_grads(params, torch.float32, 9)
    return params, vector, opt


def _contents(params, vector, opt):
    torch.cuda.synchronize()
    tensors = [t.detach().clone() for t in [*params, vector, *(p.grad for p in [*params, vector])]]
    return tensors, opt.state_dict()["state"], copy.deepcopy([{k: v for k, v in g.items() if k != "params"}
                                                              for g in opt.inner.param_groups])


def _same(a, b):
    assert all(torch.equal(x, y) for x, y in zip(a[0], b[0]))
    assert a[1].keys() == b[1].keys()
    for index, entry in a[1].items():
        assert entry.keys() == b[1][index].keys()
        assert all(torch.equal(value, b[1][index][key]) for key, value in entry.items())
    assert a[2] == b[2]


@pytest.mark.parametrize("stepped", [False, True], ids=["first", "later"])
@pytest.mark.parametrize("option,value,error", [
    ("scale", "unit", UnsupportedFeatureError),
    ("product_dtype", "bfloat16", UnsupportedFeatureError),
    ("product_dtype", "int3", ConfigurationError),
    ("steps", 0, ConfigurationError),
    ("coefficients", (1.0, 2.0), ConfigurationError),
    ("momentum", "high", ValueError),
])
def test_options_that_no_kernel_takes(device, stepped, option, value, error):
    params, vector, opt = _optimizer(device, stepped)
    good = opt.inner.param_groups[-1][option]
    opt.inner.param_groups[-1][option] = value
    before = _contents(params, vector, opt)
    with pytest.raises(error):
        opt.step()
    _same(before, _contents(params, vector, opt))
    opt.inner.param_groups[-1][option] = good
    opt.step()
    assert not torch.equal(params[0], before[0][0]) and not torch.equal(vector, before[0][2])


@pytest.mark.parametrize("stepped", [False, True], ids=["first", "later"])
@pytest.mark.parametrize("cause", ["limits", "storage", "momentum"])
def test_sizes_and_memory_that_run_out(device, stepped, cause, monkeypatch):
    params, vector, opt = _optimizer(device, stepped)
    before = _contents(params, vector, opt)

    def refuse(*_, **__):
        raise NativeKernelError("past the limits of one call") if cause == "limits" else torch.OutOfMemoryError("full")

    if cause == "limits":
        monkeypatch.setattr(muon, "_call_groups", refuse)
    elif cause == "storage":
        monkeypatch.setattr(muon, "_call_groups", lambda *_: [([0, 1], 1 << 60)])  # no device holds it
    else:
        if stepped:
            del opt.inner.state[params[1]]["momentum_buffer"]
            before = _contents(params, vector, opt)
        monkeypatch.setattr(muon.MuonOptimizer, "_zero_state", refuse)
    with pytest.raises(NativeKernelError if cause == "limits" else torch.OutOfMemoryError):
        opt.step()
    _same(before, _contents(params, vector, opt))
    monkeypatch.undo()
    opt.step()
    assert not torch.equal(params[0], before[0][0]) and not torch.equal(vector, before[0][2])


def test_a_recording_that_would_create_the_momentum(device):
    """The others hold their state already; only the matrices' is missing."""
    params, vector, opt = _optimizer(device, True)
    for p in params:
        opt.inner.state.pop(p)
    before = _contents(params, vector, opt)
    with pytest.raises(UnsupportedFeatureError, match="momentum buffer"):
        StepGraph(opt.step)
    _same(before, _contents(params, vector, opt))
