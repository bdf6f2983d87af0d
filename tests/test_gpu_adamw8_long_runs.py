"""AdamW with moments in 8 bits over many steps, where rounding errors of one step add up.

Codes of first moments have 4 significant bits, those of roots of second moments 5, and both are evenly
spaced under 2^-14 of their block's largest.  A step that moves a value by less than half a code has to
move it all the same: to one of the two codes around it, the upper one as often as the value lies near it.
"""

from __future__ import annotations

import math

import pytest
import torch

from hybrid_training_amd import GroupHandle, OptimizerConfig, ShardedOptimizer, StepGraph, moments8

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
LR = 1e-3


def _optimizer(params, betas, **options) -> ShardedOptimizer:
    config = OptimizerConfig(learning_rate=LR, betas=betas, eps=1e-12, state_format="8bit", **options)
    return ShardedOptimizer(params, config, norm_group=GroupHandle.trivial("world"), device=DEV)


def _parameter(numel, dtype=torch.float32):
    p = torch.nn.Parameter(torch.zeros(numel, dtype=dtype, device=DEV))
    p.grad = torch.zeros_like(p)
    return p


def _codes(optimizer, p):
    return [optimizer.inner.state[p][k].clone() for k in moments8.STATE_KEYS]


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.95, 0.95), (0.9, 0.99), (0.9, 0.999), (0.95, 0.999)])
@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16])
def test_roots_follow_their_gradients(betas, grad_dtype):
    """Half of every block's gradients become 4 times smaller.  4000 steps later the roots are the ones
    of float64 moments of the same gradients.

    A step changes a root by (1 - b2) / 2 |g^2 / v - 1| of itself, 0.484 (1 - b2) on average, and a code is at
    most 1/16: rounding without bias adds at most k = 0.484 (1 - b2) / 16 of it to the square of a root, and 4 k to
    the relative variance of v.  Both fade as b2^t.  Where gradients stay as they are, sums over all steps give v 0.03
    of itself and a root a variance of 0.0151, 0.123 of it.  In the other half v(s) = 1 + 15 e^-s, s in units of 1 / (1 - b2)
    steps, and the sums of k v(s) e^(s - T) and of 4 k v(s)^2 e^(2 s - 2 T) up to T = 4, over v(T) = 1.27 and its
    square, give v 0.049 and a root 0.158; further on (b2 below 0.999) they come to those of the first half.
    The root of a mean lies up to half a variance below the mean of roots, so the mean is within 0.03.
    Nearest rounding (b2 up to 0.96) is off by at most half a code, 1/32, and by what one more step takes back.
    """
    blocks = 64
    gen = torch.Generator(device=DEV).manual_seed(7)
    p = _parameter(256 * blocks)
    if grad_dtype != p.dtype:
        p.grad = None
        p.grad_dtype = None
        p.grad = torch.zeros(256 * blocks, dtype=grad_dtype, device=DEV)
    optimizer = _optimizer([p], betas)
    size = torch.ones(blocks, 256, device=DEV)
    v = torch.zeros(256 * blocks, dtype=torch.float64, device=DEV)
    for step in range(5000):
        if step == 1000:
            size[:, ::2] = 0.25
        p.grad.copy_((torch.randn(blocks, 256, device=DEV, generator=gen) * size).view(-1))
        v.mul_(betas[1]).add_(p.grad.double().square(), alpha=1 - betas[1])
        optimizer.step()
    ratio = (optimizer.moments()[0][1].double() / v).sqrt().view(blocks, 256)
    for part, off in ((ratio[:, ::2], 0.158), (ratio[:, 1::2], 0.123)):
        assert abs(float(part.mean()) - 1) <= 0.03
        assert float((part - 1).square().mean()) <= off**2 + 0.03**2


@pytest.mark.parametrize("betas", [(0.8, 0.9), (0.9, 0.95), (0.95, 0.95), (0.9, 0.999), (0.95, 0.999)])
def test_an_element_without_gradients_comes_to_rest(betas):
    """Every fourth element's gradient is zero from step 50 on, in blocks whose others go on.  Its first moment
    leaves the normal codes by b1^t within 300 steps and is then a code or two that each step drops with a
    probability of 1 - b1 at least: 0.95^400 of 16384 elements is none.  Nothing moves such an element."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    numel = 1 << 16
    p = _parameter(numel)
    optimizer = _optimizer([p], betas)
    still = torch.arange(numel, device=DEV) % 4 == 0
    still[: numel // 2 : 8] = False
    small = torch.where(torch.arange(numel, device=DEV) % 8 == 4, 1e-3, 1.0)
    for step in range(1000):
        g = torch.randn(numel, device=DEV, generator=gen) * small
        if step >= 50:
            g[still] = 0.0
        p.grad.copy_(g)
        optimizer.step()
        if step == 800:
            before = p.detach().clone()
    assert (optimizer.moments()[0][0][still] == 0).all()
    assert torch.equal(p.detach()[still], before[still])
    assert (p.detach()[~still] != before[~still]).float().mean() > 0.99


@pytest.mark.parametrize("betas", [(0.99, 0.999), (0.9, 0.95)])
@pytest.mark.parametrize("step", [16, 17, 1000])
def test_one_step_rounds_to_a_neighbour_without_bias(betas, step):
    """Every value is held as one of the two codes around it; the errors, in codes, average to none: they are
    within 1 and independent, so their mean over n elements is within 5 / sqrt(n).  Up to step 16, and from
    there on for normal codes where b1 is at most 15/16 or b2 at most 0.96, the nearer one is taken."""
    numel = 1 << 20
    gen = torch.Generator(device=DEV).manual_seed(step)
    p = _parameter(numel)
    optimizer = _optimizer([p], betas, weight_decay=0.0)

    def spread():
        return torch.exp2(-24 * torch.rand(numel, device=DEV, generator=gen))

    m = spread() * (torch.randint(2, (numel,), device=DEV, generator=gen) * 2 - 1)
    v = spread().square()
    m[::256], v[::256] = 1.0, 1.0  # every block's largest
    payload = optimizer.state_dict()
    payload["state"] = {0: {"step": torch.tensor(step - 1.0), "exp_avg": m, "exp_avg_sq": v}}
    optimizer.load_state_dict(payload)
    (m0, v0), = optimizer.moments()
    g = torch.randn(numel, device=DEV, generator=gen) * m.abs()
    g[::256] = 1.0
    p.grad.copy_(g)
    optimizer.step()
    (m1, v1), = optimizer.moments()
    m64 = m0.double() + (1 - betas[0]) * (g.double() - m0.double())
    r64 = (v0.double() * betas[1] + (1 - betas[1]) * g.double().square()).sqrt()
    scales = optimizer.inner.state[p]["moment_scales"].double().repeat_interleave(256, 0)  # every block's largest
    slow = (1 - betas[0] < 1 / 16, 1 - betas[1] < 0.04)
    for which, (exact, held, bits, free) in enumerate(((m64.abs(), m1.double().abs(), 4, slow[0]),
                                                       (r64, v1.double().sqrt(), 5, slow[1]))):
        exact, held = exact / scales[:, which], held / scales[:, which]
        code = torch.exp2(torch.floor(torch.log2(exact.clamp_min(2.0**-14))) - (bits - 1))
        at, to = exact / code, held / code
        off = to - at
        normal = exact >= 2.0**-14
        # float32 arithmetic before the rounding: 2^-20 of the value; a code is at most 2^4 units up
        slop = 2.0**-20 * 32
        assert (off.abs() <= 1 + slop).all()
        if bits == 5:
            kept = exact >= 2.0**-18  # a smaller positive root is raised to the smallest code
            off, normal, at = off[kept], normal[kept], at[kept]
        for part, nearest in ((normal, step <= 16 or not free), (~normal, step <= 16)):
            errors = off[part]
            assert errors.numel() > 10_000
            if nearest:
                assert (errors.abs() <= 0.5 + slop).all()
            else:
                assert abs(float(errors.mean())) <= 5 / math.sqrt(errors.numel())
                # what lies between two codes goes to the upper one as often as it lies near it
                share = at[part] - torch.floor(at[part])
                farther = float((errors.abs() > 0.5).double().mean() - torch.minimum(share, 1 - share).mean())
                assert abs(farther) <= 5 / math.sqrt(errors.numel())
                for low in (0.1, 0.3, 0.5, 0.7):
                    some = (share > low) & (share < low + 0.2)
                    assert abs(float(errors[some].sum())) <= 5 * math.sqrt(int(some.sum()))


def test_a_value_on_a_code_stays():
    """Moments that a step does not change are held exactly, rounded without bias or not."""
    p = _parameter(2048)
    optimizer = _optimizer([p], (0.99, 0.999))
    every = torch.arange(2048, device=DEV) % 112 + 8  # the normal codes of a first moment up to 240
    m = every.to(torch.uint8).view(torch.float8_e4m3fn).float().clamp_max(256.0)
    payload = optimizer.state_dict()
    payload["state"] = {0: {"step": torch.tensor(500.0), "exp_avg": m, "exp_avg_sq": m.square()}}
    optimizer.load_state_dict(payload)
    (m0, v0), = optimizer.moments()
    p.grad.copy_(m0)  # m + 0.01 (g - m) = m
    optimizer.step()
    assert torch.equal(optimizer.moments()[0][0], m0)


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.9, 0.999)])
def test_recorded_steps_round_as_eager_ones(betas):
    """A step recorded as the third is replayed past the sixteenth; equal inputs give equal bits."""
    eager, taped = _parameter(5003), _parameter(5003)
    a, b = _optimizer([eager], betas), _optimizer([taped], betas)
    gen = torch.Generator(device=DEV).manual_seed(11)

    def new_grads():
        g = torch.randn(5003, device=DEV, generator=gen) * torch.exp2(-8 * torch.rand(5003, device=DEV, generator=gen))
        for p in (eager, taped):
            p.grad.copy_(g)

    for _ in range(2):
        new_grads()
        a.step()
        b.step()
    graph = StepGraph(b.step)
    for _ in range(40):
        new_grads()
        a.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, taped)
        assert all(torch.equal(x, y) for x, y in zip(_codes(a, eager), _codes(b, taped)))


def test_a_list_rounds_as_each_tensor_alone():
    sizes = [1 + 53 * i for i in range(100)]
    together, alone = [_parameter(n) for n in sizes], [_parameter(n) for n in sizes]
    one, each = _optimizer(together, (0.95, 0.999)), [_optimizer([p], (0.95, 0.999)) for p in alone]
    gen = torch.Generator(device=DEV).manual_seed(5)
    for _ in range(20):
        for p, q in zip(together, alone):
            g = torch.randn(p.shape, device=DEV, generator=gen)
            p.grad.copy_(g)
            q.grad.copy_(g)
        one.step()
        for o in each:
            o.step()
    for p, q, o in zip(together, alone, each):
        assert torch.equal(p, q)
        assert all(torch.equal(x, y) for x, y in zip(_codes(one, p), _codes(o, q)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_is_not_finite_stays_alone(dtype):
    """Past the sixteenth step as before it: NaN and infinite gradients are held as NaN where they are."""
    p = _parameter(700, dtype)
    optimizer = _optimizer([p], (0.95, 0.999))
    gen = torch.Generator(device=DEV).manual_seed(2)
    for step in range(30):
        p.grad.copy_(torch.randn(700, device=DEV, generator=gen) * torch.exp2(-10 * torch.rand(700, device=DEV, generator=gen)))
        if step == 25:
            p.grad[5], p.grad[300] = math.inf, math.nan
        optimizer.step()
    (m, v), = optimizer.moments()
    wild = torch.zeros(700, dtype=torch.bool, device=DEV)
    wild[5] = wild[300] = True
    for t in (m, v):
        assert torch.equal(~torch.isfinite(t), wild)
    assert torch.equal(torch.isnan(p.detach()), wild)
