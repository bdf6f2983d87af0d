"""What the matrix operators refuse, or split, on the host before any launch.  Runs on any host."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from hybrid_training_amd import UnsupportedFeatureError, fused_linear, linear


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A tangent is not dropped: no kernel carries it, whichever argument holds it."""
    monkeypatch.setattr(linear, "_check", lambda *_: None)
    monkeypatch.setattr(linear, "_forward", lambda x, w, b, r, *_, **__: (x.detach() @ w.detach().t(), None))
    x, w, b, r = torch.randn(2, 4), torch.randn(3, 4), torch.randn(3), torch.randn(2, 3)
    with forward_ad.dual_level():
        for at in range(4):
            given = [x, w, b, r]
            given[at] = forward_ad.make_dual(given[at], torch.ones_like(given[at]))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(UnsupportedFeatureError, match="forward-mode"):
                    fused_linear(given[0], given[1], given[2], residual=given[3])
            given[at - 1] = given[at - 1].clone().requires_grad_(True)
            with pytest.raises(UnsupportedFeatureError, match="forward-mode"):
                fused_linear(given[0], given[1], given[2], residual=given[3])
        # a level without a tangent is an ordinary call
        assert torch.equal(fused_linear(x, w, b, residual=r), x @ w.t())
    assert torch.equal(fused_linear(x, w, b, residual=r), x @ w.t())
