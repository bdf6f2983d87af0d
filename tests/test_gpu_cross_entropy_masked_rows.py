"""Rows whose mask leaves no word: the softmax of nothing but -inf is not a number, at every size."""

from __future__ import annotations

import math

import pytest
import torch

from hybrid_training_amd import linear_cross_entropy

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
# one workgroup, the kernel for few tokens (of a loss alone), tiles
SHAPES = [(16, 32, 97), (5, 64, 20011), (100, 64, 300), (300, 64, 3000)]


def _inputs(tokens, inner, vocab, dtype):
    gen = torch.Generator(device=DEV).manual_seed(1)
    w = (torch.randn(vocab, inner, device=DEV, generator=gen) * inner**-0.5).to(dtype)
    x = torch.randn(tokens, inner, device=DEV, generator=gen).to(dtype)
    return x, w, torch.randint(vocab, (tokens,), device=DEV, generator=gen)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_no_word_is_left(dtype, shape, smoothing):
    x, w, target = _inputs(*shape, dtype)
    b = torch.full((shape[2],), -math.inf, device=DEV, dtype=dtype)
    target[1] = -100
    valid = target != -100
    losses = linear_cross_entropy(x, w, target, b, reduction="none", label_smoothing=smoothing)
    assert torch.isnan(losses[valid]).all() and losses[1] == 0
    for reduction in ("mean", "sum"):
        assert torch.isnan(linear_cross_entropy(x, w, target, b, reduction=reduction, label_smoothing=smoothing))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    loss = linear_cross_entropy(x, w, target, b, label_smoothing=smoothing)
    assert torch.isnan(loss)
    dx, dw, db = torch.autograd.grad(loss, leaves)
    assert torch.isnan(dx[valid]).all() and (dx[1] == 0).all()
    assert torch.isnan(dw).all() and torch.isnan(db).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_one_row_alone(dtype, shape):
    """A row at -inf everywhere is not a number; a target at -inf beside other words has an infinite loss."""
    x, w, target = _inputs(*shape, dtype)
    w[:, 0] = 1.0
    want = linear_cross_entropy(x, w, target, reduction="none")
    x[3, 0] = -math.inf
    got = linear_cross_entropy(x, w, target, reduction="none")
    assert torch.isnan(got[3])
    others = torch.arange(shape[0], device=DEV) != 3
    assert torch.equal(got[others], want[others])
    x[3, 0] = 0.0
    b = torch.zeros(shape[2], device=DEV, dtype=dtype)
    b[target[2]] = -math.inf
    got = linear_cross_entropy(x, w, target, b, reduction="none")
    assert got[2] == math.inf and torch.isfinite(got[target != target[2]]).all()
