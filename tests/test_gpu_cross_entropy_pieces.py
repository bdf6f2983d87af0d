"""Steps of more rows than one piece holds whose weight's gradient is formed in the largest tiles, from
hidden states with the tokens along a row, and carried from piece to piece."""

from __future__ import annotations

import pytest
import torch

from hybrid_training_amd import linear_cross_entropy

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("inner", [520, 333])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_sums_over_pieces(dtype, inner, reduction):
    """17000 rows of 66000 words are 2.2e9 bytes of exponentials: two pieces.  Bounds as for one piece (a
    logit's error e, (inner + 2) 2^-24 of its products' magnitudes; 4 e, u, 2^-11 and 2^-20 of a probability, with 2^-25 of
    the largest other one; float16's dz 2^-25 beside 2^13 or more), and one float32 addition a piece."""
    tokens, vocab = 17000, 66000
    gen = torch.Generator(device=DEV).manual_seed(inner)
    w = (torch.randn(vocab, inner, device=DEV, generator=gen) * inner**-0.5).to(dtype)
    target = torch.randint(vocab, (tokens,), device=DEV, generator=gen)
    x = (torch.randn(tokens, inner, device=DEV, generator=gen) + 8 * w[target].float()).to(dtype)
    target[torch.rand(tokens, device=DEV, generator=gen) < 0.02] = -100
    c = torch.exp2(4 * torch.rand(tokens, device=DEV, generator=gen)) if reduction == "none" else torch.ones(tokens, device=DEV)
    x.requires_grad_(True), w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, target, reduction=reduction)
    # 16 at most: a float16 dW of a word that many tokens share stays in range
    found = torch.autograd.grad(loss, [x, w], c if reduction == "none" else None)
    x, w = x.detach(), w.detach()
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    floor = 2.0**-38 * float(c.max()) * 2 if dtype == torch.float16 else 0.0
    w64 = w.double()
    dw = torch.zeros(vocab, inner, dtype=torch.float64, device=DEV)
    dw_off = torch.zeros_like(dw)
    total = near_total = 0.0
    for at in range(0, tokens, 1000):
        part = slice(at, at + 1000)
        valid = (target[part] != -100)[:, None].double()
        words = target[part].clamp_min(0)[:, None]
        x64, grads = x[part].double(), c[part, None].double() * valid
        z = x64 @ w64.t()
        e = ((inner + 2) * 2.0**-24 * (x64.abs() @ w64.abs().t())).amax(1, keepdim=True)
        log_sum = torch.logsumexp(z, 1, keepdim=True)
        each = (log_sum - z.gather(1, words)) * valid
        near = (2 * e + 2.0**-21 * (1 + log_sum.abs() + z.gather(1, words).abs())) * valid
        total, near_total = total + float(each.sum()), near_total + float(near.sum())
        if reduction == "none":
            assert ((loss.detach()[part].double()[:, None] - each).abs() <= near).all()
        p = torch.exp(z - log_sum)
        one = torch.zeros_like(p).scatter_(1, words, 1.0)
        size = torch.where(one > 0, 1 - p, p)
        dz = grads * torch.where(one > 0, -size, size)
        off = grads * (size * (u + 2.0**-11 + 2.0**-20) + 4 * e * p + 2.0**-25 * (p * (1 - one)).amax(1, keepdim=True)) + floor * valid
        want = dz @ w64
        bound = off @ w64.abs() + vocab * 2.0**-24 * (dz.abs() @ w64.abs())
        past = (found[0][part].double() - want).abs() - (bound * (1 + u) + u * want.abs() + tiny)
        assert (past <= 0).all()
        assert (found[0][part][valid[:, 0] == 0] == 0).all()
        dw += dz.t() @ x64
        dw_off += off.t() @ x64.abs() + tokens * 2.0**-24 * (dz.abs().t() @ x64.abs())
    if reduction == "sum":
        assert abs(float(loss.detach()) - total) <= near_total + 2.0**-22 * total
    past = (found[1].double() - dw).abs() - (dw_off * (1 + u) + u * dw.abs() + tiny)
    assert (past <= 0).all()
