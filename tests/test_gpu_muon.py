"""Orthogonalised matrices and the optimizer step along them, against float64.

Bounds, relative in the Frobenius norm.  float32 products: four norm-wise roundings of 2^-24 a
step, grown by at most a^5 = 3.4445^5 = 485 over the run, 1.2e-4.  float16 products read x, A
and B with independent rounding errors of rms 0.58 2^-11 = 2.8e-4: about six of them a step
enter (b A + c A A) x, which is at most 2.8 |x|, so 1.9e-3 a step and 4.3e-3 over five; 5e-3 is
allowed.  The result's own rounding comes on top.  The momentum is elementwise: four fp32
roundings of |v| + |g|.
"""

from __future__ import annotations

import math

import pytest
import torch

from hybrid_training_amd import (
    GroupHandle,
    MuonConfig,
    MuonOptimizer,
    NativeKernelError,
    OptimizerConfig,
    ShardedOptimizer,
    ShardingError,
    StepGraph,
    UnsupportedFeatureError,
    _native,
    orthogonalize,
)
from hybrid_training_amd.errors import ConfigurationError

pytestmark = pytest.mark.gpu

A, B, C = COEFFICIENTS = (3.4445, -4.7750, 2.0315)
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
PRODUCT = {torch.float16: 5e-3, torch.float32: 1.2e-4}
SHAPES = [(1, 1), (1, 32), (32, 1), (32, 23), (23, 32), (7, 5), (3, 100), (64, 64), (64, 128), (129, 64), (65, 130),
          (300, 77), (77, 300), (9, 1030), (512, 512), (130, 1030), (1030, 131), (1000, 1001), (2100, 40)]


def exact(u, steps=5, coefficients=COEFFICIENTS, eps=1e-12):
    a, b, c = coefficients
    x = u.double()
    x = x / max(float(x.norm()), eps)
    if x.shape[0] > x.shape[1]:
        return exact(u.t(), steps, coefficients, eps).t()
    for _ in range(steps):
        gram = x @ x.t()
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x


def gradient(device, rows, cols, dtype=torch.float32, seed=0, kind="noise"):
    gen = torch.Generator(device=device).manual_seed(seed * 100003 + rows * 1009 + cols)
    m = torch.randn(rows, cols, device=device, generator=gen)
    if kind == "low_rank":
        left = torch.randn(rows, 4, device=device, generator=gen)
        m = 0.05 * m + left @ torch.randn(4, cols, device=device, generator=gen)
    return (m * 1e-3).to(dtype)


def off(got, want):
    return float((got.double() - want).norm() / want.norm().clamp_min(1e-300))


@pytest.mark.parametrize("product", [torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("kind", ["noise", "low_rank"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalize(device, shape, kind, product):
    print(shape, kind, product, flush=True)
    g = gradient(device, *shape, kind=kind)
    want = exact(g)
    (got,) = orthogonalize([g], product_dtype=product)
    assert got.shape == g.shape and got.dtype == g.dtype
    assert off(got, want) < PRODUCT[product]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_a_list_of_mixed_sizes(device, dtype):
    """Wide and tall together, more matrices than one call takes, an empty one among them."""
    shapes = [(40, 60), (60, 40), (256, 256), (0, 5), (1, 9), (9, 1), (300, 20), (33, 33), (200, 264)] * 3
    matrices = [gradient(device, *s, dtype, seed=i) for i, s in enumerate(shapes)]
    product = torch.float32 if dtype == torch.float32 else torch.float16
    results = orthogonalize(matrices)
    assert [r.dtype for r in results] == [dtype] * len(shapes)
    for m, r in zip(matrices, results):
        assert r.shape == m.shape
        if m.numel():
            assert off(r, exact(m)) < PRODUCT[product] + UNIT[dtype]
    # each alone: the same bits, whatever shares its launches
    for i in (0, 1, 2, 5, 8):
        assert torch.equal(orthogonalize([matrices[i]])[0], results[i])


@pytest.mark.parametrize("shape", [(9001, 16), (16, 9001), (50257, 64), (70, 6000), (2600, 129), (129, 2600), (4100, 250),
                                   (255, 7001)], ids=str)
def test_long_thin_matrices(device, shape):
    """Gram sums in parts, of odd lengths, beside matrices whose sums are whole; the bits stay a
    matrix's own."""
    shapes = [shape, (300, 300), shape, (40, 20)]
    for dtype, product in ((torch.bfloat16, torch.float16), (torch.float32, torch.float32)):
        matrices = [gradient(device, *s, dtype, seed=i) for i, s in enumerate(shapes)]
        results = orthogonalize(matrices)
        for m, r in zip(matrices, results):
            assert off(r, exact(m)) < PRODUCT[product] + UNIT[dtype]
            assert torch.equal(orthogonalize([m])[0], r)


def test_large_matrices_take_the_large_tiles(device):
    for shape in ((4200, 4104), (4104, 4200)):
        g = gradient(device, *shape, torch.bfloat16)
        assert off(orthogonalize([g])[0], exact(g)) < PRODUCT[torch.float16] + UNIT[torch.bfloat16]
    g = gradient(device, 2100, 2060)
    assert off(orthogonalize([g])[0], exact(g)) < PRODUCT[torch.float32]


def test_options(device):
    g = gradient(device, 48, 90)
    for steps, coefficients in ((1, COEFFICIENTS), (3, (1.5, -0.5, 0.0)), (9, (1.875, -1.25, 0.375))):
        got = orthogonalize([g], steps=steps, coefficients=coefficients)[0]
        assert off(got, exact(g, steps, coefficients)) < PRODUCT[torch.float32]
    assert orthogonalize([g], dtype=torch.bfloat16)[0].dtype == torch.bfloat16
    assert orthogonalize([]) == []
    # below eps the norm no longer scales
    small = g * 1e-3
    assert off(orthogonalize([small], eps=1.0, steps=1)[0], exact(small, 1, eps=1.0)) < PRODUCT[torch.float32]
    # any layout
    assert torch.equal(orthogonalize([g.t().contiguous().t()])[0], orthogonalize([g])[0])
    assert torch.equal(orthogonalize([torch.cat([g, g], 1)[:, 10:60]])[0],
                       orthogonalize([torch.cat([g, g], 1)[:, 10:60].contiguous()])[0])


@pytest.mark.parametrize("product", [torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("shape", [(24, 40), (300, 200)], ids=str)
def test_magnitudes_zeros_and_nonfinite_values(device, shape, product):
    g = gradient(device, *shape)
    want = exact(g)
    for scale in (2.0**-90, 2.0**60):  # float32 holds it; its square it does not
        assert off(orthogonalize([g * scale], eps=0.0, product_dtype=product)[0], want) < PRODUCT[product]
    assert not orthogonalize([torch.zeros_like(g)], product_dtype=product)[0].any()
    for value in (float("nan"), float("inf")):
        bad = g.clone()
        bad[3, 5] = value
        clean, dirty = orthogonalize([g, bad], product_dtype=product)
        assert not bool(dirty.isfinite().all())
        assert torch.equal(clean, orthogonalize([g], product_dtype=product)[0])  # its neighbour is untouched
    lonely = torch.zeros_like(g)
    lonely[2, 7] = 3.0  # one singular value: x is a single element of size near 1
    got = orthogonalize([lonely], product_dtype=product)[0]
    assert off(got, exact(lonely)) < PRODUCT[product] and int((got != 0).sum()) == 1


def test_side_stream_and_repeated_bits(device):
    matrices = [gradient(device, 300, 500), gradient(device, 500, 129)]
    want = orthogonalize(matrices, product_dtype="float16")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            got = orthogonalize(matrices, product_dtype="float16")
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- the optimizer ---------------------------------------------------------------------
def build(device, shapes, master=torch.float32, grad=torch.float32, config=None, others=(), seed=0, **options):
    gen = torch.Generator(device=device).manual_seed(seed)
    params = [torch.nn.Parameter((torch.randn(*s, device=device, generator=gen) * 0.02).to(master)) for s in shapes]
    config = config or MuonConfig(learning_rate=3e-4, weight_decay=0.1)
    opt = MuonOptimizer(params, config, norm_group=GroupHandle.trivial("world"), device=device, others=others, **options)
    set_grads(params, grad, seed)
    return params, opt


def set_grads(params, grad, seed, scale=1.0):
    for i, p in enumerate(params):
        if p.dtype != grad:
            p.grad_dtype = None
        p.grad = (gradient(p.device, *p.shape, seed=seed * 31 + i + 1) * scale).to(grad)


def expect(p, g, v, config, mul=1.0):
    """Parameter, momentum and how far each may be, in float64, from one step."""
    g, v = g.double() * mul, v.double()
    v = config.momentum * v + (1 - config.momentum) * g
    u = (1 - config.momentum) * g + config.momentum * v if config.nesterov else v
    rows, cols = p.shape
    scale = 0.2 * math.sqrt(max(rows, cols)) if config.scale == "rms" else math.sqrt(max(1.0, rows / cols))
    move = config.learning_rate * scale * exact(u, config.steps, config.coefficients, config.eps)
    new = (1 - config.learning_rate * config.weight_decay) * p.double() - move
    product = PRODUCT[torch.float32 if config.product_dtype == "float32" else torch.float16]
    far = product * float(move.norm()) + (UNIT[p.dtype] + 2.0**-22) * float(new.norm())
    return new, v, far


def holds(p, v, want, grads):
    new, velocity, far = want
    assert float((p.detach().double() - new).norm()) <= far
    assert bool(((v.double() - velocity).abs() <= 2.0**-21 * (velocity.abs() + grads.double().abs()) + 1e-37).all())


PAIRS = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float16)]


@pytest.mark.parametrize("pair", PAIRS, ids=str)
@pytest.mark.parametrize("config", [
    MuonConfig(learning_rate=3e-4, weight_decay=0.1),
    MuonConfig(learning_rate=0.02, momentum=0.9, nesterov=False, scale="spectral", product_dtype="float32"),
    MuonConfig(learning_rate=1e-3, momentum=0.0, steps=3, weight_decay=0.0),
], ids=["rms", "spectral", "no_momentum"])
def test_steps(device, pair, config):
    params, opt = build(device, [(32, 23), (200, 300), (300, 136), (1, 32), (64, 64)], *pair, config=config)
    buffers = [torch.zeros(p.shape, dtype=torch.float32, device=device) for p in params]
    for step in range(3):
        set_grads(params, pair[1], step)
        wants = [expect(p.detach(), p.grad, v, config) for p, v in zip(params, buffers)]
        grads = [p.grad.clone() for p in params]
        versions = [p._version for p in params]
        opt.step()
        for p, g, want, before in zip(params, grads, wants, versions):
            v = opt.inner.state[p]["momentum_buffer"]
            assert v.dtype == torch.float32 and p._version > before and torch.equal(p.grad, g)
            holds(p, v, want, g)
        buffers = [opt.inner.state[p]["momentum_buffer"].clone() for p in params]


@pytest.mark.parametrize("options", [{}, {"clip_in_step": True}, {"defer_clip": True}], ids=["in_place", "in_step", "defer"])
@pytest.mark.parametrize("pair", [PAIRS[0], PAIRS[2]], ids=str)
def test_clip_placements(device, options, pair):
    config = MuonConfig(learning_rate=3e-4, weight_decay=0.1)
    params, opt = build(device, [(48, 60), (300, 200)], *pair, config=config, **options)
    set_grads(params, pair[1], 3, scale=1e3)
    grads = [p.grad.clone() for p in params]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    mul = 1.0 / (norm + 1e-6)
    assert mul < 1
    assert abs(float(opt.clip_grad_norm(1.0)) - norm) < 1e-9 * norm
    clipped = [p.grad.clone() for p in params]
    opt.step()
    for p, g, c in zip(params, grads, clipped):
        # in place the clipped gradient has been rounded to its dtype; the step's own clip has not
        want = expect(p.detach(), c if not options else g, torch.zeros_like(p, dtype=torch.float32), config,
                      1.0 if not options else mul)
        v = opt.inner.state[p]["momentum_buffer"]
        assert bool(((v.double() - want[1]).abs() <= 2.0**-20 * want[1].abs() + 1e-37).all())
        if "defer_clip" in options:
            assert torch.equal(p.grad, g)
        else:
            assert torch.equal(p.grad, (g.float() * torch.tensor(mul, dtype=torch.float32, device=device)).to(g.dtype))


def test_others_are_stepped_as_by_the_sharded_optimizer(device):
    config = OptimizerConfig(learning_rate=1e-3, weight_decay=0.01)
    vectors = [torch.nn.Parameter(torch.randn(n, device=device)) for n in (7, 300)]
    twins = [torch.nn.Parameter(p.detach().clone()) for p in vectors]
    params, opt = build(device, [(40, 50)], others=vectors, others_config=config)
    plain = ShardedOptimizer(twins, config, norm_group=GroupHandle.trivial("world"), device=device)
    for step in range(2):
        set_grads(params, torch.float32, step)
        for p, q in zip(vectors, twins):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
        opt.step()
        plain.step()
    assert all(torch.equal(p, q) for p, q in zip(vectors, twins))
    assert opt.parameters[:2] == tuple(vectors) and opt.state_bytes() > 0
    norm = float(opt.clip_grad_norm(0.0))
    total = sum(float(p.grad.double().square().sum()) for p in [*vectors, *params])
    assert abs(norm - math.sqrt(total)) < 1e-9 * norm


def test_missing_gradients_are_skipped(device):
    params, opt = build(device, [(20, 30), (30, 20)])
    params[0].grad = None
    before = params[0].detach().clone()
    opt.step()
    assert torch.equal(params[0], before) and "momentum_buffer" not in opt.inner.state.get(params[0], {})


@pytest.mark.parametrize("master", [torch.float32, torch.bfloat16], ids=str)
def test_state_dict_round_trip(device, master):
    vector = torch.nn.Parameter(torch.randn(9, device=device))
    params, opt = build(device, [(24, 40), (40, 24)], master, master, others=[vector])
    vector.grad = torch.randn_like(vector)
    opt.step()
    payload = opt.state_dict()
    assert payload["state"][1]["momentum_buffer"].dtype == torch.float32
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = torch.nn.Parameter(vector.detach().clone())
    twin = MuonOptimizer(copies, MuonConfig(learning_rate=1.0), norm_group=GroupHandle.trivial("world"), device=device,
                         others=[other])
    twin.load_state_dict(payload)
    for p, q in zip(params, copies):
        assert torch.equal(opt.inner.state[p]["momentum_buffer"], twin.inner.state[q]["momentum_buffer"])
        q.grad = p.grad = gradient(device, *p.shape, master, seed=5)
    other.grad = vector.grad
    opt.step()
    twin.step()
    assert all(torch.equal(p, q) for p, q in zip([*params, vector], [*copies, other]))


def test_recorded_steps_replay_as_eager_ones(device):
    shapes = [(32, 23), (130, 70), (70, 260)]
    vector, vector_twin = (torch.nn.Parameter(torch.ones(11, device=device)) for _ in range(2))
    params, opt = build(device, shapes, others=[vector])
    twins, eager = build(device, shapes, others=[vector_twin])
    vector.grad, vector_twin.grad = torch.ones_like(vector), torch.ones_like(vector)
    for o in (opt, eager):
        o.clip_grad_norm(1.0)
        o.step()
    graph = StepGraph(lambda: (opt.clip_grad_norm(1.0), opt.step()))
    for k in range(4):
        for p, q in zip(params, twins):
            p.grad.copy_(gradient(device, *p.shape, seed=50 + k))
            q.grad.copy_(p.grad)
        if k == 2:  # a schedule moves the learning rate and the momentum
            for o in (opt, eager):
                o.set_learning_rate(1e-4)
                o.inner.param_groups[-1]["momentum"] = 0.9
        graph.replay()
        torch.cuda.synchronize()
        eager.clip_grad_norm(1.0)
        eager.step()
        for p, q in zip([*params, vector], [*twins, vector_twin]):
            assert torch.equal(p, q), k
        for p, q in zip(params, twins):
            assert torch.equal(opt.inner.state[p]["momentum_buffer"], eager.inner.state[q]["momentum_buffer"])
    opt.inner.param_groups[-1]["steps"] = 4
    with pytest.raises(UnsupportedFeatureError, match="record the step again"):
        graph.replay()


def test_first_step_cannot_be_recorded(device):
    params, opt = build(device, [(20, 30)])
    with pytest.raises(UnsupportedFeatureError, match="momentum buffer"):
        StepGraph(opt.step)


def test_refusals(device):
    good = torch.nn.Parameter(torch.randn(4, 6, device=device))
    group = GroupHandle.trivial("world")
    make = lambda matrices, **k: MuonOptimizer(matrices, MuonConfig(), norm_group=group, device=device, **k)  # noqa: E731
    with pytest.raises(ShardingError, match="no trainable matrices"):
        make([])
    with pytest.raises(ShardingError, match="whole matrices"):
        make([torch.nn.Parameter(torch.randn(24, device=device))])
    with pytest.raises(ShardingError, match="twice"):
        make([good], others=[good])
    with pytest.raises(UnsupportedFeatureError, match="float32, bfloat16 or float16"):
        make([torch.nn.Parameter(torch.randn(4, 6, device=device, dtype=torch.float64))])
    with pytest.raises(UnsupportedFeatureError, match="device memory"):
        make([torch.nn.Parameter(torch.randn(4, 6))])
    with pytest.raises(UnsupportedFeatureError, match="AdamW"):
        make([good], others_config=OptimizerConfig(name="sgd"))
    for bad in ({"learning_rate": 0.0}, {"momentum": 1.0}, {"steps": 0}, {"steps": 65}, {"scale": "none"}, {"eps": -1.0},
                {"coefficients": (1.0, 2.0)}, {"coefficients": (1.0, 2.0, float("nan"))}, {"product_dtype": "bfloat16"}):
        with pytest.raises(ConfigurationError):
            MuonConfig(**bad)
    m = good.detach()
    with pytest.raises(ShardingError, match="matrix"):
        orthogonalize([m[0]])
    with pytest.raises(UnsupportedFeatureError, match="one dtype"):
        orthogonalize([m, m.half()])
    with pytest.raises(UnsupportedFeatureError, match="one dtype"):
        orthogonalize([m.double()])
    with pytest.raises(UnsupportedFeatureError, match="results"):
        orthogonalize([m], dtype=torch.float64)
    with pytest.raises(UnsupportedFeatureError, match="products read"):
        orthogonalize([m], product_dtype=torch.bfloat16)
    with pytest.raises(UnsupportedFeatureError, match="HIP device"):
        orthogonalize([m.cpu()])
    with pytest.raises(ConfigurationError):
        orthogonalize([m], steps=0)
    opt = make([good])
    good.grad = torch.randn_like(good)
    opt.inner.state[good]["momentum_buffer"] = torch.zeros(4, 6, dtype=torch.bfloat16, device=device)
    with pytest.raises(ShardingError, match="float32 tensor"):
        opt.step()
    lib = _native.library()
    one = _native.int64_array([4])
    assert lib.hbt_orthogonal_workspace(one, _native.int64_array([-1]), 1, _native.DTYPE_F16) == -1
    large = torch.randn(80, 200, device=device)  # small matrices need no workspace
    status = lib.hbt_orthogonalize(_native.pointer_array([large.data_ptr()]), _native.pointer_array([large.data_ptr()]),
                                   _native.int64_array([80]), _native.int64_array([200]), 1, 0, 0, 0, 5, A, B, C, 0.0,
                                   None, 0, None)
    with pytest.raises(NativeKernelError, match="workspace"):
        _native.check(status, "test")
