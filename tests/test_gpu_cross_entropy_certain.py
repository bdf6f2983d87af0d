"""Gradients of nearly certain targets, every word of them, relative to what they are.

Where a target stands far above the other words, its row's dz is 1 - p for the target and as much, shared
out, for the others.  With e the error of a logit, (inner + 2) 2^-24 of its products' magnitudes, and
s = 4 e + 12 2^-24 max|z| + 2^-20 for the units, differences and exponentials in float32, a word's
probability is off by

* s of itself,
* 2^-11 of itself where its exponential is held in fp16 (2-byte tensors), or half of fp16's smallest
  step, 2^-25, times the probability of the largest word of its tile, the target aside;

and its dz by u more, half a step of the tensors' dtype.  float16's dz of equal tokens stand 2^13 times as
large: half of their smallest step is 2^-38.  The target's dz, a float32 sum, is off by s and u of
itself.  Products add as many 2^-24 of their magnitudes as they have terms.
"""

from __future__ import annotations

import math

import pytest
import torch

from hybrid_training_amd import linear_cross_entropy

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
LIFTS, INNER = 16, 80  # targets, each with a column of its own that lifts it


def _inputs(tokens, vocab, dtype, above):
    """Hidden states whose targets stand ``above`` over the largest other word; the words' rows share a component."""
    gen = torch.Generator(device=DEV).manual_seed(tokens + vocab)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    w = torch.zeros(vocab, INNER, device=DEV)
    w[:, LIFTS:] = 0.5 * normal(1, INNER - LIFTS) + 0.125 * normal(vocab, INNER - LIFTS)
    words = torch.randperm(vocab, device=DEV, generator=gen)[:LIFTS]
    w[words, torch.arange(LIFTS, device=DEV)] = 1.0
    w = w.to(dtype)
    which = torch.randint(LIFTS, (tokens,), device=DEV, generator=gen)
    target = words[which]
    x = torch.zeros(tokens, INNER, device=DEV)
    x[:, LIFTS:] = 0.25 * normal(tokens, INNER - LIFTS)
    x = x.to(dtype)
    b = (0.25 * normal(vocab)).to(dtype)
    z = x.double() @ w.double().t() + b.double()
    at = target[:, None]
    own = z.gather(1, at).squeeze(1)
    z.scatter_(1, at, -math.inf)
    x[torch.arange(tokens, device=DEV), which] = (above + z.amax(1) - own).to(dtype)
    return x, w, b, target


def _exact(x, w, b, target, scale):
    """(dx, dw, db) of the summed loss times ``scale`` in float64, and bounds on their errors."""
    x64, w64, b64, at = x.double(), w.double(), b.double(), target[:, None]
    z = x64 @ w64.t() + b64
    e = ((x.shape[1] + 2) * 2.0**-24 * (x64.abs() @ w64.abs().t() + b64.abs())).amax(1, keepdim=True)
    s = 4 * e + 12 * 2.0**-24 * z.abs().amax(1, keepdim=True) + 2.0**-20
    others = z.clone().scatter_(1, at, -math.inf)
    p = torch.exp(others - torch.logsumexp(z, 1, keepdim=True))
    missing = p.sum(1, keepdim=True)
    dz = p.scatter(1, at, -missing)
    u = torch.finfo(x.dtype).eps / 2
    off = p * (s + u)
    if x.dtype != torch.float32:
        off = off + torch.maximum(p * 2.0**-11, 2.0**-25 * p.amax(1, keepdim=True))
    off = off.scatter(1, at, missing * (s + u))
    if x.dtype == torch.float16:
        off = off + 2.0**-38
    along, across = z.shape[1] * 2.0**-24, z.shape[0] * 2.0**-24
    want = dz @ w64, dz.t() @ x64, dz.sum(0)
    near = (off @ w64.abs() + along * (dz.abs() @ w64.abs()), off.t() @ x64.abs() + across * (dz.abs().t() @ x64.abs()),
            off.sum(0) + across * dz.abs().sum(0))
    return [t * scale for t in want], [t * scale for t in near]


@pytest.mark.parametrize("dtype, above", [(d, a) for d in (torch.float32, torch.bfloat16, torch.float16)
                                          for a in (11.5, 12.0, 16.0, 18.0, 20.0, 25.0)])
@pytest.mark.parametrize("vocab", [40, 300, 3000])
@pytest.mark.parametrize("tokens", [100, 300])
def test_every_word_keeps_its_gradient(dtype, above, vocab, tokens):
    x, w, b, target = _inputs(tokens, vocab, dtype, above)
    scale = 2.0**20 if dtype == torch.float16 else 1.0  # a loss scale; 1e-8 alone is a float16 subnormal
    want, near = _exact(x, w, b, target, scale)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    loss = linear_cross_entropy(x, w, target, b, reduction="sum")
    found = torch.autograd.grad(loss, leaves, torch.tensor(scale, device=DEV))
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for name, g, t, off in zip(("dx", "dw", "db"), found, want, near):
        # what float16 cannot hold is infinite: 2^20 times a dw of 0.1 is past its 65504
        wild = torch.isinf(g)
        assert (t[wild].abs() + off[wild] > torch.finfo(dtype).max).all() and (g[wild].sign() == t[wild].sign()).all()
        g, t, off = g.double()[~wild], t[~wild], off[~wild]
        past = (g - t).abs() - (off * (1 + u) + u * t.abs() + tiny)
        assert (past <= 0).all(), f"{name}: {float((g - t).norm() / t.norm()):.3g} of itself off"
    # a row of dz adds up to nothing, and so do the bias's gradients
    if torch.isfinite(found[2]).all():
        assert abs(float(found[2].double().sum())) <= float((near[2] * (1 + u) + u * want[2].abs() + tiny).sum())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [200, 3000])
def test_a_target_that_is_alone(dtype, vocab):
    """Every other word at -inf: a probability of 1, no loss and no gradient anywhere."""
    x, w, b, target = _inputs(100, vocab, dtype, 3.0)
    target.fill_(vocab // 2)
    b.fill_(-math.inf)
    b[vocab // 2] = 0.5
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    loss = linear_cross_entropy(x, w, target, b, reduction="sum")
    assert loss == 0
    assert all((g == 0).all() for g in torch.autograd.grad(loss, leaves))
    with torch.no_grad():
        for rows in (5, 100):
            assert (linear_cross_entropy(x[:rows], w, target[:rows], b, reduction="none") == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_vocabulary_of_one_word(dtype):
    x = torch.randn(100, 4000, device=DEV).to(dtype)
    w = torch.randn(1, 4000, device=DEV).to(dtype)
    target = torch.zeros(100, dtype=torch.int64, device=DEV)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    loss = linear_cross_entropy(x, w, target, reduction="sum")
    assert loss == 0 and all((g == 0).all() for g in torch.autograd.grad(loss, leaves))
