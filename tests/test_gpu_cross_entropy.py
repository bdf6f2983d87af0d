"""The loss over a vocabulary and its gradients against the definition in float64.

Bounds.  A logit is a float32 sum of ``inner`` products: off by at most e = (inner + 2) 2^-24 times the
sum of its products' magnitudes.  A loss is off by 2 e and a few float32 roundings of its parts.
A probability is off by 2 e relative, by 2^-11 where its exponential is held in fp16 (and 2^-24
absolute, fp16's smallest steps), and the gradient of a logit is rounded to the tensors' dtype, half a step u;
its products are float32 sums of as many terms as they have, counted as n 2^-24 of the magnitudes.
Results are rounded once more, bfloat16 ones twice where the loss is scaled.
"""

from __future__ import annotations

import math

import pytest
import torch

from hybrid_training_amd import LinearCrossEntropy, StepGraph, cross_entropy, linear_cross_entropy
from hybrid_training_amd.errors import ShardingError, UnsupportedFeatureError

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(tokens, inner, vocab, dtype, *, bias=False, ignored=0.0, seed=0, strength=8.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    w = (normal(vocab, inner) * max(inner, 1) ** -0.5).to(dtype)
    target = torch.randint(vocab, (tokens,), device=DEV, generator=gen)
    x = (normal(tokens, inner) + strength * torch.rand(tokens, 1, device=DEV, generator=gen) * w[target].float()).to(dtype)
    b = (normal(vocab) * 0.5).to(dtype) if bias else None
    target[torch.rand(tokens, device=DEV, generator=gen) < ignored] = -100
    return x, w, b, target


def _exact(x, w, b, target, *, smoothing=0.0, grads=None, ignore=-100):
    """Losses of every token and, for token gradients c, (dx, dw, db) with bounds on their errors
    before the last rounding."""
    valid = target != ignore
    rows = torch.nonzero(valid).squeeze(1)
    x64, w64 = x[rows].double(), w.double()
    z = x64 @ w64.t() + (0 if b is None else b.double())
    e = (x.shape[1] + 2) * 2.0**-24 * (x64.abs() @ w64.abs().t() + (0 if b is None else b.double().abs()))
    e = e.amax(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    at = target[rows][:, None].long()
    part = lse - (1 - smoothing) * z.gather(1, at) - (smoothing * z.mean(1, keepdim=True) if smoothing else 0)
    loss = torch.zeros(target.shape, dtype=torch.float64, device=DEV).index_put_((rows,), part.squeeze(1))
    near = torch.zeros_like(loss).index_put_(
        (rows,), (2 * e + 2.0**-21 * (1 + lse.abs() + z.gather(1, at).abs())).squeeze(1))
    if grads is None:
        return loss, near
    c = grads.double()[rows][:, None]
    p = torch.exp(z - lse)
    one = torch.zeros_like(p).scatter_(1, at, 1.0)
    dz = c * (p - (1 - smoothing) * one - smoothing / w.shape[0])
    u = torch.finfo(x.dtype).eps / 2
    held = 0.0 if x.dtype == torch.float32 else 1.0
    # the products sum dz, but smoothing subtracts from p: errors are relative to the parts
    size = c.abs() * (p * (1 - one) + (1 - p) * one + smoothing / w.shape[0])
    off = size * (u + held * 2.0**-11 + 2.0**-20) + 4 * e * c.abs() * p + held * 2.0**-23 * c.abs()
    terms = dz.shape[1] * 2.0**-24
    dx = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    dx_off = torch.zeros_like(dx)
    dx[rows] = dz @ w64
    dx_off[rows] = off @ w64.abs() + terms * (dz.abs() @ w64.abs())
    terms = dz.shape[0] * 2.0**-24
    dw, dw_off = dz.t() @ x64, off.t() @ x64.abs() + terms * (dz.abs().t() @ x64.abs())
    db, db_off = dz.sum(0), off.sum(0) + terms * dz.abs().sum(0)
    return loss, near, (dx, dw, db), (dx_off, dw_off, db_off)


def _close(got, want, off, twice=False):
    u = torch.finfo(got.dtype).eps / 2 * (2 if twice else 1)
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    near = off * (1 + u) + u * want.abs() + tiny
    assert torch.isfinite(got).all()
    past = (got.double() - want).abs() - near
    assert (past <= 0).all(), f"{past.max():.3g} past the bound"


SHAPES = [(20, 0, 30), (300, 64, 20011), (1, 1, 1), (1, 64, 97), (3, 5, 2), (16, 32, 97), (17, 23, 63), (16, 768, 5003), (64, 96, 256), (130, 64, 257),
          (300, 501, 1000), (257, 128, 4096), (1500, 40, 333), (2049, 16, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("options", [dict(), dict(bias=True, ignored=0.3, smoothing=0.1)], ids=["plain", "all"])
def test_losses_and_gradients(dtype, shape, options):
    smoothing = options.get("smoothing", 0.0)
    x, w, b, target = _inputs(*shape, dtype, bias="bias" in options, ignored=options.get("ignored", 0.0))
    if "ignored" in options:
        target[-1] = 0  # one token at least
    count = int((target != -100).sum())
    loss, near, grads, offs = _exact(x, w, b, target, smoothing=smoothing,
                                     grads=torch.full(target.shape, 1.0 / count, device=DEV))
    got = linear_cross_entropy(x, w, target, b, reduction="none", label_smoothing=smoothing)
    assert got.dtype == torch.float32 and got.shape == target.shape
    assert ((got.double() - loss).abs() <= near).all() and (got[target == -100] == 0).all()
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    for reduction, divide in (("mean", count), ("sum", 1)):
        with torch.no_grad():
            evaluated = linear_cross_entropy(x, w, target, b, reduction=reduction, label_smoothing=smoothing)
        got = linear_cross_entropy(x, w, target, b, reduction=reduction, label_smoothing=smoothing)
        for value in (got, evaluated):
            assert abs(float(value.detach()) - float(loss.sum()) / divide) <= float(near.sum()) / divide + 2.0**-22 * float(loss.sum())
        found = torch.autograd.grad(got, leaves)
        scale = count / divide
        for g, want, off in zip(found, grads, offs):
            assert g.dtype == dtype
            _close(g, want * scale, off * scale)
        assert (found[0][target == -100] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_separate_losses_take_each_tokens_gradient(dtype):
    x, w, b, target = _inputs(200, 48, 777, dtype, bias=True, ignored=0.2)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    c = torch.randn(200, device=DEV) * torch.exp2(torch.randn(200, device=DEV) * 4)
    c[5] = 0.0
    _, _, grads, offs = _exact(x.detach(), w.detach(), b.detach(), target, grads=c)
    loss = linear_cross_entropy(x, w, target, b, reduction="none")
    found = torch.autograd.grad(loss, leaves, c)
    # fp16's dz stands at a common power of two: its smallest steps are those of the largest gradient
    extra = 2.0**-24 * float(c.abs().max()) if dtype == torch.float16 else 0.0
    sums = (w.detach().double().abs().sum(0)[None], x.detach().double().abs().sum(0)[None], torch.tensor(200.0, device=DEV))
    for g, want, off, s in zip(found, grads, offs, sums):
        _close(g, want, off + extra * s)
    assert (found[0][5] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1.0, 1024.0, 0.3])
@pytest.mark.parametrize("tokens, held", [(20, None), (20, 0), (100, None), (100, 0), (900, None)])
def test_the_losss_own_gradient(dtype, scale, tokens, held, monkeypatch):
    x, w, b, target = _inputs(tokens, 40, 300, dtype, bias=True)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    _, _, grads, offs = _exact(x.detach(), w.detach(), b.detach(), target,
                               grads=torch.full((tokens,), scale / tokens, device=DEV))
    if held is not None:  # as for a large weight
        monkeypatch.setattr(cross_entropy, "_HOLD_ELEMENTS", held)
    loss = linear_cross_entropy(x, w, target, b)
    first = torch.autograd.grad(loss, leaves, torch.tensor(scale, device=DEV), retain_graph=True)
    kept = [g.clone() for g in first]
    again = torch.autograd.grad(loss, leaves, torch.tensor(scale, device=DEV))
    for g, k, a, want, off in zip(first, kept, again, grads, offs):
        _close(g, want, off, twice=True)
        assert torch.equal(g, k) and torch.equal(g, a)


def test_a_loss_scale_keeps_what_float16_flushes():
    """Gradients near 1e-8 are zero in float16; scaled by 2^16 before they are rounded, they are not."""
    x, w, b, target = _inputs(4096, 64, 512, torch.float16)
    x = (x * 2.0**-10).requires_grad_(True)
    w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, target)
    scaled, = torch.autograd.grad(loss, [w], torch.tensor(65536.0, device=DEV))
    _, _, grads, offs = _exact(x.detach(), w.detach(), None, target, grads=torch.full((4096,), 16.0, device=DEV))
    _close(scaled, grads[1], offs[1])
    assert (scaled == 0).float().mean() < 0.01


@pytest.mark.parametrize("tokens", [7, 500])
@pytest.mark.parametrize("garbage", [math.nan, math.inf, -math.inf])
def test_ignored_tokens_reach_nothing(tokens, garbage):
    x, w, b, target = _inputs(tokens, 33, 400, torch.bfloat16, bias=True)
    hidden = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    hidden[::3] = True
    target[hidden] = -7
    outputs = []
    for fill in (0.0, garbage):
        x2 = x.clone()
        x2[hidden] = fill
        leaves = [t.detach().clone().requires_grad_(True) for t in (x2, w, b)]
        loss = linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], ignore_index=-7)
        outputs.append([loss.detach(), *torch.autograd.grad(loss, leaves),
                        linear_cross_entropy(x2, w, target, b, ignore_index=-7, reduction="none")])
    for a, c in zip(*outputs):
        assert torch.isfinite(a).all() and torch.equal(a, c)
    assert (outputs[1][1][hidden] == 0).all()


@pytest.mark.parametrize("tokens", [4, 40])
@pytest.mark.parametrize("dtype", DTYPES)
def test_no_token_carries_a_loss(tokens, dtype):
    x, w, b, target = _inputs(tokens, 24, 50, dtype, bias=True)
    target.fill_(-100)
    assert (linear_cross_entropy(x, w, target, b, reduction="none") == 0).all()
    assert linear_cross_entropy(x, w, target, b, reduction="sum") == 0
    assert torch.isnan(linear_cross_entropy(x, w, target, b))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    for reduction in ("mean", "sum"):
        for g in torch.autograd.grad(linear_cross_entropy(x, w, target, b, reduction=reduction), leaves):
            assert (g == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_tokens(dtype):
    x, w, b, target = _inputs(0, 24, 50, dtype, bias=True)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    assert linear_cross_entropy(x, w, target, b, reduction="none").shape == (0,)
    loss = linear_cross_entropy(x, w, target, b, reduction="sum")
    assert loss == 0 and all((g == 0).all() for g in torch.autograd.grad(loss, leaves))
    assert torch.isnan(linear_cross_entropy(x, w, target, b))
    none = linear_cross_entropy(x, w, target, b, reduction="none")
    assert all((g == 0).all() for g in torch.autograd.grad(none, leaves, torch.zeros(0, device=DEV)))


@pytest.mark.parametrize("tokens", [3, 50])
@pytest.mark.parametrize("bad", [50, -1, 1 << 40])
def test_targets_out_of_range_are_not_a_number(tokens, bad):
    x, w, b, target = _inputs(tokens, 24, 50, torch.bfloat16)
    target[1] = bad
    losses = linear_cross_entropy(x, w, target, reduction="none")
    assert torch.isnan(losses[1]) and torch.isfinite(losses[0]) and torch.isfinite(losses[2:]).all()
    x.requires_grad_(True)
    loss = linear_cross_entropy(x, w, target)
    dx, = torch.autograd.grad(loss, [x])
    assert torch.isnan(loss) and torch.isnan(dx[1]).all() and torch.isfinite(dx[0]).all()


@pytest.mark.parametrize("tokens", [5, 70])
@pytest.mark.parametrize("dtype", DTYPES)
def test_words_masked_out_by_the_bias(tokens, dtype):
    """Words at -inf, whole tiles of them, take no probability and get no gradient; logits far below
    zero elsewhere keep their differences."""
    vocab = 900
    x, w, b, target = _inputs(tokens, 32, vocab, dtype, bias=True)
    b = (b.float() - 500.0).to(dtype)
    b[300:] = -math.inf
    target %= 300
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    want, near, grads, offs = _exact(x.detach(), w.detach()[:300], b.detach()[:300], target,
                                     grads=torch.full((tokens,), 1.0 / tokens, device=DEV))
    losses = linear_cross_entropy(x.detach(), w.detach(), target, b.detach(), reduction="none")
    assert ((losses.double() - want).abs() <= near).all()
    dx, dw, db = torch.autograd.grad(linear_cross_entropy(x, w, target, b), leaves)
    _close(dx, grads[0], offs[0])
    _close(dw[:300], grads[1], offs[1])
    _close(db[:300], grads[2], offs[2])
    assert (dw[300:] == 0).all() and (db[300:] == 0).all()


def test_a_nearly_certain_target_keeps_its_gradient():
    """1 - p of 1e-5 is far under fp16's and bfloat16's steps next to 1."""
    tokens, vocab = 20, 300
    w = torch.zeros(vocab, 64, device=DEV, dtype=torch.bfloat16)
    w[0, 0] = 1.0
    x = torch.zeros(tokens, 64, device=DEV, dtype=torch.bfloat16)
    x[:, 0] = math.log(vocab - 1) + 11.5
    target = torch.zeros(tokens, dtype=torch.int64, device=DEV)
    x.requires_grad_(True)
    loss = linear_cross_entropy(x, w, target, reduction="sum")
    dx, = torch.autograd.grad(loss, [x])
    z = x.detach()[:, 0].double()
    missing = 1.0 - torch.exp(z) / (torch.exp(z) + vocab - 1)
    assert ((dx[:, 0].double() + missing).abs() <= missing * (2.0**-8 + 2.0**-9)).all()
    assert abs(float(loss.detach()) + float(torch.log1p(-missing).sum())) <= tokens * 2.0**-19


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens, vocab", [(3, 40), (4, 3000), (40, 3000), (300, 700)])
@pytest.mark.parametrize("above", [11.5, 18.0, 25.0])
def test_the_loss_of_a_nearly_certain_target_is_the_others_sum(dtype, tokens, vocab, above):
    """log(1 + s) for an s down to 1e-11, which fp32 would lose beside the target's 1.  One logit z is not zero
    and has one product; its unit, the difference of two tiles' largest and the exponentials are
    off by at most 6 z + 16 float32 roundings."""
    w = torch.zeros(vocab, 64, device=DEV, dtype=dtype)
    w[1, 0] = 1.0
    x = torch.zeros(tokens, 64, device=DEV, dtype=dtype)
    x[:, 0] = math.log(vocab - 1) + above
    target = torch.ones(tokens, dtype=torch.int64, device=DEV)
    z = x[:, 0].double()
    others = (vocab - 1) * torch.exp(-z)
    off = (6 * z + 16) * 2.0**-24
    loss = linear_cross_entropy(x, w, target, reduction="none")
    assert ((loss.double() / torch.log1p(others) - 1).abs() <= off).all()
    if dtype != torch.float16:  # whose dz of 1e-11 would be a subnormal
        u = torch.finfo(dtype).eps / 2
        dx, = torch.autograd.grad(linear_cross_entropy(x.requires_grad_(True), w, target, reduction="sum"), [x])
        assert ((dx[:, 0].double() * (1 + others) / -others - 1).abs() <= off + 2 * u + 2.0**-22).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [9, 150, 390])
def test_layouts(dtype, tokens):
    """Strides, offsets and shapes other than dense ones give the dense ones' bits."""
    x, w, b, target = _inputs(tokens, 64, 333, dtype, bias=True)
    dense = [t.clone().requires_grad_(True) for t in (x, w, b)]
    loss = linear_cross_entropy(dense[0], dense[1], target, dense[2])
    want = [loss.detach(), *torch.autograd.grad(loss, dense)]
    wide = torch.zeros(tokens, 200, device=DEV, dtype=dtype)
    wide[:, 8:72] = x
    stretched = torch.zeros(2 * 333, 64, device=DEV, dtype=dtype)
    stretched[::2] = w
    every = torch.zeros(2 * 333, device=DEV, dtype=dtype)
    every[::2] = b
    many = torch.zeros(tokens, 3, dtype=torch.int32, device=DEV)
    many[:, 1] = target
    views = [wide[:, 8:72].requires_grad_(True), stretched[::2].requires_grad_(True), every[::2].requires_grad_(True)]
    loss = linear_cross_entropy(views[0], views[1], many[:, 1], views[2])
    for a, c in zip(want, [loss.detach(), *torch.autograd.grad(loss, views)]):
        assert torch.equal(a, c)
    # rows off 16 bytes take another way through the same sums: the bounds of any other call
    odd = torch.zeros(333 * 64 + 1, device=DEV, dtype=dtype)
    odd[1:] = w.reshape(-1)
    shifted = [x.clone().requires_grad_(True), odd[1:].view(333, 64).requires_grad_(True), b.clone().requires_grad_(True)]
    _, _, grads, offs = _exact(x, w, b, target, grads=torch.full((tokens,), 1.0 / tokens, device=DEV))
    for g, t, off in zip(torch.autograd.grad(linear_cross_entropy(shifted[0], shifted[1], target, shifted[2]), shifted),
                         grads, offs):
        _close(g, t, off)
    # leading dimensions
    if tokens % 3 == 0:
        cube = x.view(3, -1, 64).clone().requires_grad_(True)
        loss = linear_cross_entropy(cube, w, target.view(3, -1), b)
        dx, = torch.autograd.grad(loss, [cube])
        assert dx.shape == cube.shape and torch.equal(dx.view(-1, 64), want[1])
        assert linear_cross_entropy(x.view(3, -1, 64), w, target.view(3, -1), b, reduction="none").shape == (3, tokens // 3)


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 2), (1, 2)])
def test_some_gradients_alone(which):
    x, w, b, target = _inputs(90, 72, 500, torch.bfloat16, bias=True)
    every = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(linear_cross_entropy(every[0], every[1], target, every[2]), every)
    some = [t.clone().requires_grad_(i in which) for i, t in enumerate((x, w, b))]
    found = torch.autograd.grad(linear_cross_entropy(some[0], some[1], target, some[2]), [some[i] for i in which])
    for i, g in zip(which, found):
        assert torch.equal(g, want[i])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_more_rows_than_one_piece_holds(dtype):
    """18000 x 65537 exponentials pass 2 GiB: the sums over rows are carried from piece to piece."""
    tokens, inner, vocab = 18000, 24, 65537
    x, w, b, target = _inputs(tokens, inner, vocab, dtype, bias=True, ignored=0.05)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    loss = linear_cross_entropy(x, w, target, b, reduction="sum")
    found = torch.autograd.grad(loss, leaves)
    want = [torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in leaves]
    offs = [torch.zeros_like(t) for t in want]
    total = near = 0.0
    for i in range(0, tokens, 1000):
        part = slice(i, i + 1000)
        loss64, close, grads, off = _exact(x.detach()[part], w.detach(), b.detach(), target[part],
                                           grads=torch.ones(1000, device=DEV))
        total, near = total + float(loss64.sum()), near + float(close.sum())
        want[0][part], offs[0][part] = grads[0], off[0]
        for k in (1, 2):
            want[k] += grads[k]
            offs[k] += off[k] + 2.0**-20 * grads[k].abs()
    assert abs(float(loss) - total) <= near + 2.0**-22 * total
    for g, t, off in zip(found, want, offs):
        _close(g, t, off)


def test_rows_far_apart():
    """Rows 2^20 elements apart, past 4 GiB, are read where they lie and give the dense ones' bits."""
    x, w, _, target = _inputs(2500, 64, 3000, torch.bfloat16)
    dense = [t.clone().requires_grad_(True) for t in (x, w)]
    loss = linear_cross_entropy(*dense, target)
    want = [loss.detach(), *torch.autograd.grad(loss, dense)]
    far = []
    for t in (x, w):
        room = torch.empty(t.shape[0], 1 << 20, dtype=t.dtype, device=DEV)
        room[:, :64] = t
        far.append(room[:, :64].requires_grad_(True))
    loss = linear_cross_entropy(*far, target)
    for a, c in zip(want, [loss.detach(), *torch.autograd.grad(loss, far)]):
        assert torch.equal(a, c)


def test_hidden_states_past_32_bits():
    """1.1e6 x 2048 hidden states.  All but the last 1000 tokens' are zero, so the weight's gradient is a
    sum of 1000 terms, whose bound holds, from the end of the tensor."""
    tokens, inner, vocab, last = 1_100_000, 2048, 64, 1000
    some, w, _, words = _inputs(last, inner, vocab, torch.bfloat16)
    x = torch.zeros(tokens, inner, dtype=torch.bfloat16, device=DEV)
    x[-last:] = some
    target = torch.arange(tokens, device=DEV) % vocab
    target[-last:] = words
    dx, dw = torch.autograd.grad(
        linear_cross_entropy(x.requires_grad_(True), w.requires_grad_(True), target, reduction="sum"), [x, w])
    x, w = x.detach(), w.detach()
    ones = torch.ones(tokens, device=DEV)
    _, _, grads, offs = _exact(x[-last:], w, None, target[-last:], grads=ones[-last:])
    _close(dw, grads[1], offs[1])
    for at in range(0, tokens, 50_000):
        part = slice(at, at + 50_000)
        _, _, grads, offs = _exact(x[part], w, None, target[part], grads=ones[part])
        _close(dx[part], grads[0], offs[0])


def test_a_weight_past_32_bits():
    """33 tokens over the largest vocabulary, a weight of 2.2e9 elements."""
    tokens, inner, vocab = 33, 2112, (1 << 20) - 64
    gen = torch.Generator(device=DEV).manual_seed(3)
    w = torch.empty(vocab, inner, dtype=torch.bfloat16, device=DEV).normal_(0, inner**-0.5, generator=gen)
    target = torch.randint(vocab, (tokens,), device=DEV, generator=gen)
    target[0], target[1] = vocab - 1, 0
    x = (torch.randn(tokens, inner, device=DEV, generator=gen) + 12 * w[target].float()).bfloat16()
    loss = linear_cross_entropy(x.requires_grad_(True), w.requires_grad_(True), target, reduction="sum")
    dx, dw = torch.autograd.grad(loss, [x, w])
    x, w = x.detach(), w.detach()
    chunks = [slice(i, min(i + 65536, vocab)) for i in range(0, vocab, 65536)]
    x64 = x.double()
    z = torch.cat([x64 @ w[c].double().t() for c in chunks], 1)
    e = torch.stack([(x64.abs() @ w[c].double().abs().t()).amax(1, keepdim=True) for c in chunks]).amax(0)
    e = e * (inner + 2) * 2.0**-24
    lse = torch.logsumexp(z, 1, keepdim=True)
    p, one = torch.exp(z - lse), torch.zeros_like(z).scatter_(1, target[:, None], 1.0)
    exact = (lse.squeeze(1) - z.gather(1, target[:, None]).squeeze(1)).sum()
    assert abs(float(loss.detach()) - float(exact)) <= float((2 * e + 2.0**-21 * (1 + 2 * z.abs().amax(1, keepdim=True) + lse)).sum())
    dz = p - one
    off = dz.abs() * (2.0**-8 + 2.0**-11 + 2.0**-20) + 4 * e * p + 2.0**-23
    want, near = torch.zeros_like(x64), torch.zeros_like(x64)
    for c in chunks:
        w64 = w[c].double()
        want += dz[:, c] @ w64
        near += off[:, c] @ w64.abs() + vocab * 2.0**-24 * (dz[:, c].abs() @ w64.abs())
        _close(dw[c], dz[:, c].t() @ x64, off[:, c].t() @ x64.abs() + tokens * 2.0**-24 * (dz[:, c].abs().t() @ x64.abs()))
    _close(dx, want, near)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("inner, vocab", [(700, 28501), (28501, 700)])
def test_a_last_round_of_few_tiles(dtype, inner, vocab):
    """336 tiles of 256 of the weight's gradient: a round, and 81 whose sums are split."""
    x, w, b, target = _inputs(8192, inner, vocab, dtype, bias=True, ignored=0.01)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    found = torch.autograd.grad(linear_cross_entropy(x, w, target, b, reduction="sum"), leaves)
    ones = torch.ones(8192, device=DEV)
    _, _, grads, offs = _exact(x.detach(), w.detach(), b.detach(), target, grads=ones)
    for g, want, off in zip(found, grads, offs):
        _close(g, want, off)


def test_gradients_against_differences():
    x, w, b, target = _inputs(6, 8, 40, torch.float32, bias=True)
    x64, w64, b64 = x.double(), w.double(), b.double()
    target[2] = -100
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    found = torch.autograd.grad(linear_cross_entropy(x, w, target, b, label_smoothing=0.2), leaves)

    def value(x64, w64, b64):
        return _exact(x64, w64, b64, target, smoothing=0.2)[0].sum() / 5

    step = 1e-5
    for which, g in enumerate(found):
        for flat in (0, g.numel() // 2, g.numel() - 1):
            moved = []
            for sign in (1, -1):
                at = [t.clone() for t in (x64, w64, b64)]
                at[which].view(-1)[flat] += sign * step
                moved.append(float(value(*at)))
            # central differences: step^2 of a third derivative (a few at most), 1e-16 / step of rounding
            assert abs(float(g.reshape(-1)[flat]) - (moved[0] - moved[1]) / (2 * step)) <= 2e-6


def test_equal_inputs_give_equal_bits():
    x, w, b, target = _inputs(700, 96, 3001, torch.bfloat16, bias=True, ignored=0.1)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    runs = []
    for _ in range(3):
        loss = linear_cross_entropy(x, w, target, b)
        runs.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
    assert all(torch.equal(a, c) for other in runs[1:] for a, c in zip(runs[0], other))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(16, 32, 97), (16, 768, 5003), (130, 64, 257), (300, 501, 1000), (1801, 200, 4099), (700, 1, 9000)],
                         ids=lambda s: "x".join(map(str, s)))
def test_nothing_comes_from_unwritten_memory(dtype, shape, monkeypatch):
    """Results and working storage that hold NaN before the call give the same bits."""
    x, w, b, target = _inputs(*shape, dtype, bias=True, ignored=0.4)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def call():
        loss = linear_cross_entropy(x, w, target, b, label_smoothing=0.1)
        with torch.no_grad():
            each = linear_cross_entropy(x, w, target, b, reduction="none")
        return [loss.detach(), each, *torch.autograd.grad(loss, leaves)]

    want = call()
    empty = torch.empty

    def poisoned(*args, **options):
        t = empty(*args, **options)
        return t.fill_(255 if t.dtype == torch.uint8 else math.nan)

    monkeypatch.setattr(cross_entropy.torch, "empty", poisoned)
    found = call()
    monkeypatch.undo()
    for a, c in zip(want, found):
        assert torch.isfinite(a).all() and torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("ignored", [0.0, 0.5, 0.9, 0.995])
def test_few_rows_of_many_tokens(dtype, ignored):
    """Sums of dx are split by how many tokens carry a loss, which only the device knows."""
    x, w, _, target = _inputs(1500, 264, 9001, dtype, ignored=ignored)
    target[3] = 5
    c = torch.full(target.shape, 1.0, device=DEV)
    _, _, grads, offs = _exact(x, w, None, target, grads=c)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    found = torch.autograd.grad(linear_cross_entropy(x, w, target, reduction="sum"), leaves)
    for g, want, off in zip(found, grads, offs):
        _close(g, want, off)


def test_two_streams_at_once():
    cases = [_inputs(300, 128, 2000, torch.bfloat16, seed=s) for s in (1, 2)]
    want, found = [], [None, None]
    for x, w, _, target in cases:
        w.requires_grad_(True)
        loss = linear_cross_entropy(x, w, target)
        want.append([loss.detach(), *torch.autograd.grad(loss, [w])])
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for i, (s, (x, w, _, target)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                loss = linear_cross_entropy(x, w, target)
                found[i] = [loss.detach(), *torch.autograd.grad(loss, [w])]
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for one, other in zip(want, found) for a, c in zip(one, other))


def test_recorded_and_replayed():
    """Replays read new hidden states, targets (another number of them ignored) and weights."""
    x, w, b, target = _inputs(200, 64, 1000, torch.bfloat16, bias=True)
    head = LinearCrossEntropy(64, 1000, bias=True, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        head.weight.copy_(w)
        head.bias.copy_(b)
    hidden = x.clone().requires_grad_(True)
    words = target.clone()

    def fixed():
        loss = head(hidden, words)
        return (loss.detach(), *torch.autograd.grad(loss, [hidden, head.weight, head.bias]))

    fixed()
    torch.cuda.synchronize()
    graph = StepGraph(fixed)
    for seed in range(1, 5):
        x, w, b, target = _inputs(200, 64, 1000, torch.bfloat16, bias=True, ignored=0.2 * seed, seed=seed)
        with torch.no_grad():
            hidden.copy_(x)
            words.copy_(target)
            head.weight.copy_(w)
            head.bias.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        taped = [t.clone() for t in graph.output]
        for a, c in zip(taped, fixed()):
            assert torch.equal(a, c)


def test_recording_beside_a_living_eager_loss():
    """Its nodes belong to the default stream, which cannot join the recording: refused, until it is gone."""
    x, w, _, target = _inputs(100, 32, 300, torch.bfloat16)
    w.requires_grad_(True)
    w.grad = torch.zeros_like(w)

    def step():
        loss = linear_cross_entropy(x, w, target)
        loss.backward()
        return loss.detach()

    want = step()
    alive = linear_cross_entropy(x, w, target)
    with pytest.raises(UnsupportedFeatureError, match="still alive"):
        StepGraph(step)
    alive.backward()
    kept = alive.detach()
    del alive
    graph = StepGraph(step)
    w.grad.zero_()
    once = torch.autograd.grad(linear_cross_entropy(x, w, target), [w])[0]
    for count in (1, 2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(graph.output, want) and torch.equal(kept, want)
        assert torch.equal(w.grad, once * count)


def test_refusals():
    x, w, b, target = _inputs(10, 16, 40, torch.bfloat16, bias=True)
    for call, error, match in (
        (lambda: linear_cross_entropy(x, w, target[:9]), ShardingError, "one target per token"),
        (lambda: linear_cross_entropy(x, w[:, :8], target), ShardingError, "inner size"),
        (lambda: linear_cross_entropy(x, w[:0], target), ShardingError, "empty"),
        (lambda: linear_cross_entropy(x, w, target, b[:3]), ShardingError, "per word"),
        (lambda: linear_cross_entropy(x, w.float(), target), UnsupportedFeatureError, "dtype"),
        (lambda: linear_cross_entropy(x.double(), w.double(), target), UnsupportedFeatureError, "dtype"),
        (lambda: linear_cross_entropy(x, w, target.float()), UnsupportedFeatureError, "whole numbers"),
        (lambda: linear_cross_entropy(x, w, target.cpu()), UnsupportedFeatureError, "HIP device"),
        (lambda: linear_cross_entropy(x, w, target, reduction="max"), UnsupportedFeatureError, "reduction"),
        (lambda: linear_cross_entropy(x, w, target, label_smoothing=1.5), UnsupportedFeatureError, "smoothing"),
        (lambda: LinearCrossEntropy(4, 4, reduction="max"), UnsupportedFeatureError, "reduction"),
    ):
        with pytest.raises(error, match=match):
            call()
    huge = torch.zeros(1, device=DEV, dtype=torch.bfloat16).expand(1 << 20, 16)
    with pytest.raises(UnsupportedFeatureError, match="limits"):
        linear_cross_entropy(x, huge, target)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(UnsupportedFeatureError, match="forward-mode"):
            linear_cross_entropy(dual, w, target)
