"""AdamW with moments in 8 bits, against the definition in float64.

A first moment has 4 significant bits: the nearest code is at most half a step away, 2^-4 of the
value, or 2^-18 of its block's largest below the smallest normal code (steps of 2^-17).  A root of
a second moment has 5: 2^-5 of the value, 2^-19 of the largest, or 2^-18 where a positive root
is raised to the smallest code.  The float32 arithmetic before that adds a few 2^-24 (and 2^-23 of
what cancels), counted as 2^-20 of the operands.  Parameters are compared with the float64 update
of the same state within their own rounding and 8 float32 roundings of what is added up.
"""

from __future__ import annotations

import math

import pytest
import torch

from hybrid_training_amd import (
    FlatParamHandle,
    FSDPConfig,
    GradScaler,
    GradScalerConfig,
    GroupHandle,
    MixedPrecisionConfig,
    MuonConfig,
    MuonOptimizer,
    OptimizerConfig,
    ShardedOptimizer,
    StepGraph,
    collect_flat_shard_payload,
    load_flat_shard_checkpoint,
    write_checkpoint,
)
from hybrid_training_amd import moments8
from hybrid_training_amd.errors import ShardingError, UnsupportedFeatureError

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
BLOCK = 256
LR, B1, B2, EPS, WD = 1e-3, 0.9, 0.99, 1e-8, 0.1
SLOP = 2.0**-20
PAIRS = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float16)]


def _config(**options) -> OptimizerConfig:
    return OptimizerConfig(learning_rate=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_format="8bit", **options)


def _optimizer(params, config=None, **options) -> ShardedOptimizer:
    return ShardedOptimizer(params, config or _config(), norm_group=GroupHandle.trivial("world"), device=DEV, **options)


def _params(sizes, dtype=torch.float32, grad_dtype=None, seed=0, offset=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    params = []
    for n in sizes:
        def normal():
            return torch.randn(n + offset, device=DEV, generator=gen)

        p = torch.nn.Parameter((normal() * 0.1).to(dtype)[offset:])
        grad = (normal() * torch.exp2(normal() * 2) * 1e-2).to(grad_dtype or dtype)[offset:]
        if grad.dtype != p.dtype:
            p.grad_dtype = None
        p.grad = grad
        params.append(p)
    return params


def _new_grads(params, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for p in params:
        p.grad.copy_(torch.randn(p.shape, device=DEV, generator=gen) * 1e-2)


def _codes(optimizer, p):
    return [optimizer.inner.state[p][k].clone() for k in moments8.STATE_KEYS]


def _top(values: torch.Tensor) -> torch.Tensor:
    """Every element's block maximum of |values|, non-finite ones aside."""
    flat = values.abs().reshape(-1)
    flat = torch.where(torch.isfinite(flat), flat, 0)
    missing = -flat.numel() % BLOCK
    rows = torch.cat([flat, flat.new_zeros(missing)]).view(-1, BLOCK)
    return rows.amax(1, keepdim=True).expand(-1, BLOCK).reshape(-1)[: values.numel()].view(values.shape)


def _check_held(m, v, m64, r64, slop_m, slop_r):
    """Decoded moments against exact ones, before rounding off by at most the slops."""
    near = torch.maximum(m64.abs() * 2.0**-4, _top(m64) * 2.0**-18) + 2 * slop_m
    assert ((m.double() - m64).abs() <= near).all()
    near = torch.maximum(r64 * 2.0**-5, _top(r64) * 2.0**-18) + 2 * slop_r
    assert ((v.double().sqrt() - r64).abs() <= near).all()
    assert ((v > 0) == (r64 > 0)).all()


@pytest.mark.parametrize("sizes", [[0, 1, 255], [256, 257], [5000, 3, 100_001]])
def test_encode_and_decode(sizes):
    gen = torch.Generator(device=DEV).manual_seed(5)
    params = [torch.empty(n, device=DEV) for n in sizes]
    pairs = [(torch.randn(n, device=DEV, generator=gen) * torch.exp2(torch.randn(n, device=DEV, generator=gen) * 5),
              torch.rand(n, device=DEV, generator=gen) * torch.exp2(torch.randn(n, device=DEV, generator=gen) * 9))
             for n in sizes]
    states = [moments8.zero_state(p) for p in params]
    moments8.encode(pairs, states, DEV)
    held = moments8.decode(params, states, DEV)
    for (m, v), (dm, dv) in zip(pairs, held):
        _check_held(dm, dv, m.double(), v.double().sqrt(), m.abs().double() * 2.0**-23, v.double().sqrt() * 2.0**-23)
        if m.numel():  # a block's largest values are held exactly (the second by its rounded root)
            assert torch.equal(dm.abs().max(), m.abs().max())
            assert torch.equal(dv.max(), v.max().sqrt().square())
    # what was decoded encodes to the same bits
    again = [moments8.zero_state(p) for p in params]
    moments8.encode(held, again, DEV)
    for a, b in zip(states, again):
        assert all(torch.equal(a[k], b[k]) for k in moments8.STATE_KEYS)
    for (m, v), (bm, bv) in zip(held, moments8.decode(params, states, DEV, torch.bfloat16)):
        assert torch.equal(bm, m.bfloat16()) and torch.equal(bv, v.bfloat16())


def test_every_code_stands_for_its_value():
    """256 codes in one block: e4m3 over 256 as torch reads them, and the root's exponent and mantissa."""
    p = torch.empty(256, device=DEV)
    state = moments8.zero_state(p)
    every = torch.arange(256, device=DEV).to(torch.uint8)
    state["moment_codes"].view(64, 2, 4).copy_(every.view(64, 1, 4).expand(64, 2, 4))
    state["moment_scales"].copy_(torch.tensor([[3.0, 0.75]]))
    (m, v), = moments8.decode([p], [state], DEV)
    first = every.view(torch.float8_e4m3fn).float() * (3.0 / 256)
    assert torch.equal(torch.isnan(m), torch.isnan(first)) and torch.equal(m.nan_to_num(0), first.nan_to_num(0))
    e, f = torch.arange(256) // 16, torch.arange(256) % 16
    root = torch.where(e > 0, torch.ldexp((16.0 + f), e - 19), torch.ldexp(f.float(), torch.tensor(-18))) * 0.75
    root[255] = math.nan
    assert torch.equal(v.cpu()[:255], root[:255].square()) and torch.isnan(v[255])


@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: "-".join(str(t).split(".")[1] for t in p))
@pytest.mark.parametrize("offset", [0, 1])
def test_step_against_float64(pair, offset):
    dtype, grad_dtype = pair
    sizes = [1, 4, 255, 256, 257, 2047, 4099, 70_001]
    params = _params(sizes, dtype, grad_dtype, offset=offset)
    optimizer = _optimizer(params)
    for step in range(1, 4):
        _new_grads(params, step)
        before = [(p.detach().double(), p.grad.double()) for p in params]
        state = optimizer.moments() if step > 1 else [(torch.zeros_like(g), torch.zeros_like(g)) for _, g in before]
        optimizer.step()
        for p, (old, g), (m0, v0), (m, v) in zip(params, before, state, optimizer.moments()):
            m64 = B1 * m0.double() + (1 - B1) * g
            r64 = (B2 * v0.double() + (1 - B2) * g.square()).sqrt()
            size = m0.double().abs() + g.abs()
            _check_held(m, v, m64, r64, size * SLOP, r64 * SLOP)
            update = LR / (1 - B1**step) * m64 / (r64 / math.sqrt(1 - B2**step) + EPS)
            # m's rounding errors are relative to what it is summed from, the update's to m's
            spread = LR / (1 - B1**step) * size / (r64 / math.sqrt(1 - B2**step) + EPS)
            new = old - LR * WD * old - update
            eps = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
            tiny = torch.finfo(torch.float16).smallest_normal * eps if dtype == torch.float16 else 0.0
            near = eps * new.abs() + tiny + 8 * 2.0**-24 * (1 + eps) * (old.abs() + spread)
            assert ((p.detach().double() - new).abs() <= near).all()


def test_a_list_longer_than_a_launch_steps_as_each_alone():
    sizes = [1 + 37 * i for i in range(130)]
    together, alone = _params(sizes), _params(sizes)
    one = _optimizer(together)
    each = [_optimizer([p]) for p in alone]
    for seed in (1, 2):
        for params in (together, alone):
            _new_grads(params, seed)
        one.step()
        for o in each:
            o.step()
    for p, q, o in zip(together, alone, each):
        assert torch.equal(p, q)
        assert all(torch.equal(a, b) for a, b in zip(_codes(one, p), _codes(o, q)))


def test_elements_past_32_bits():
    """A parameter of 2^31 + 300 elements: its last blocks step and decode as they do alone."""
    numel, last = (1 << 31) + 300, (1 << 16) + 300
    whole = torch.nn.Parameter(torch.zeros(numel, dtype=torch.bfloat16, device=DEV))
    whole.grad = torch.zeros_like(whole)
    alone, = _params([last], torch.bfloat16)
    with torch.no_grad():
        whole[-last:] = alone
    optimizers = [_optimizer([whole]), _optimizer([alone])]
    for step in (1, 2):
        _new_grads([alone], step)
        whole.grad[-last:] = alone.grad
        for optimizer in optimizers:
            optimizer.step()
    assert torch.equal(whole.detach()[-last:], alone.detach())
    assert not whole.detach()[: numel - last].any()
    (far, near), (other, beside) = (o.moments(torch.bfloat16)[0] for o in optimizers)
    assert torch.equal(far[-last:], other) and torch.equal(near[-last:], beside)
    assert not far[: numel - last].any() and not near[: numel - last].any()


def test_zeros_tiny_and_non_finite_gradients():
    params = _params([1024])
    p = params[0]
    optimizer = _optimizer(params)
    g = torch.zeros(1024, device=DEV)
    g[256:512] = 1e-33          # first moments under 2^-100: held as zeros
    g[512], g[513] = math.inf, math.nan
    g[514:768] = 0.5
    g[768], g[769] = 1.0, 1e-7  # a root under the smallest code beside a large one
    p.grad.copy_(g)
    old = p.detach().clone()
    optimizer.step()
    (m, v), = optimizer.moments()
    decayed = old * torch.tensor(1 - LR * WD, device=DEV)
    assert torch.equal(m[:512], torch.zeros(512, device=DEV)) and torch.equal(v[:256], torch.zeros(256, device=DEV))
    assert torch.equal(p[:256].detach(), decayed[:256])
    assert torch.isnan(m[512:514]).all() and torch.isnan(v[512:514]).all()
    assert torch.isfinite(m[514:]).all() and torch.isfinite(v[514:]).all() and torch.isfinite(p[514:].detach()).all()
    assert (m[514:768] == m[514]).all() and m[514] > 0
    assert v[769] > 0 and v[769] <= (2.0**-18 * 1.0001) ** 2 * v[768]
    # a block of nothing finite has zero scales and keeps NaN everywhere
    state = moments8.zero_state(torch.empty(256))
    state = {k: v.to(DEV) for k, v in state.items()}
    wild = torch.tensor([math.inf, -math.inf, math.nan, math.inf] * 64, device=DEV)
    moments8.encode([(wild, wild.abs())], [state], DEV)
    (wm, wv), = moments8.decode([wild], [state], DEV)
    assert (state["moment_scales"] == 0).all() and torch.isnan(wm).all() and torch.isnan(wv).all()
    # the next step starts from them: the element that was not finite stays so, alone
    p.grad.copy_(torch.full((1024,), 0.1, device=DEV))
    optimizer.step()
    assert torch.isnan(p[512:514]).all() and torch.isfinite(p[514:]).all() and torch.isfinite(p[:512]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clip_placements_agree(dtype):
    runs = []
    for options in ({}, {"clip_in_step": True}, {"defer_clip": True}):
        params = _params([700, 33_000], dtype)
        optimizer = _optimizer(params, **options)
        for seed in (3, 4):
            _new_grads(params, seed)
            unclipped = [p.grad.clone() for p in params]
            optimizer.clip_grad_norm(0.25)
            optimizer.step()
        grads = [p.grad for p in params]
        assert all(torch.equal(a, b) for a, b in zip(grads, unclipped)) == ("defer_clip" in options)
        runs.append([p.detach() for p in params] + [c for p in params for c in _codes(optimizer, p)])
        if "defer_clip" not in options:
            runs[-1] += grads
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@pytest.mark.parametrize("deferred", [False, True])
def test_a_loss_scale_is_taken_off(deferred):
    plain, scaled = _params([9000], torch.float16), _params([9000], torch.float16)
    a, b = _optimizer(plain), _optimizer(scaled)
    scaler = GradScaler(GradScalerConfig(enabled=True, init_scale=64.0), GroupHandle.trivial(), DEV,
                        defer_unscale=deferred)
    scaled[0].grad.mul_(64.0)
    a.step()
    assert scaler.step(b, scaled)
    assert torch.equal(plain[0], scaled[0]) and torch.equal(plain[0].grad, scaled[0].grad)
    assert all(torch.equal(x, y) for x, y in zip(_codes(a, plain[0]), _codes(b, scaled[0])))


def test_state_dict_returns_the_same_bits_and_crosses_formats():
    params = _params([300, 4097])
    optimizer = _optimizer(params)
    for seed in (1, 2):
        _new_grads(params, seed)
        optimizer.step()
    payload = optimizer.state_dict()
    assert payload["state"][0]["exp_avg"].dtype == torch.float32 and not payload["state"][0]["exp_avg"].is_cuda
    restored = _optimizer(params)
    restored.load_state_dict(payload)
    for p in params:
        assert all(torch.equal(x, y) for x, y in zip(_codes(optimizer, p), _codes(restored, p)))
        assert restored.inner.state[p]["step"] == 2
    # to moments in the master's dtype and back
    wide = ShardedOptimizer(params, OptimizerConfig(learning_rate=LR, betas=(B1, B2), weight_decay=WD),
                            norm_group=GroupHandle.trivial("world"), device=DEV)
    wide.load_state_dict(payload)
    assert torch.equal(wide.inner.state[params[1]]["exp_avg"], optimizer.moments()[1][0])
    back = _optimizer(params)
    back.load_state_dict(wide.state_dict())
    for p in params:
        assert all(torch.equal(x, y) for x, y in zip(_codes(optimizer, p), _codes(back, p)))
    assert optimizer.state_bytes() < sum(p.numel() for p in params) * 2 + 4096


def test_recorded_steps_equal_eager_ones():
    eager, taped = _params([500, 12_345]), _params([500, 12_345])
    a, b = _optimizer(eager), _optimizer(taped)
    for params, optimizer in ((eager, a), (taped, b)):
        _new_grads(params, 1)
        optimizer.clip_and_step(1.0)
    graph = StepGraph(lambda: b.clip_and_step(1.0))
    for seed in range(2, 6):
        for optimizer in (a, b):
            optimizer.set_learning_rate(LR / seed)
        for params in (eager, taped):
            _new_grads(params, seed)
        a.clip_and_step(1.0)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(eager, taped):
            assert torch.equal(p, q) and a.inner.state[p]["step"] == b.inner.state[q]["step"]
            assert all(torch.equal(x, y) for x, y in zip(_codes(a, p), _codes(b, q)))
    b.load_state_dict(b.state_dict())
    with pytest.raises(UnsupportedFeatureError, match="record the step again"):
        graph.replay()


def test_steps_on_another_stream():
    here, there = _params([50_000]), _params([50_000])
    a, b = _optimizer(here), _optimizer(there)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for seed in (1, 2):
        _new_grads(here, seed)
        a.step()
        with torch.cuda.stream(side):
            _new_grads(there, seed)
            b.step()
            moments = b.moments()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(here[0], there[0])
    assert all(torch.equal(x, y) for x, y in zip(a.moments()[0], moments[0]))


def test_beside_orthogonalised_matrices():
    """MuonOptimizer's other parameters hold their moments in 8 bits as ShardedOptimizer's do."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    matrix = torch.nn.Parameter(torch.randn(48, 32, device=DEV, generator=gen))
    vectors, alone = _params([48, 300]), _params([48, 300])
    muon = MuonOptimizer([matrix], MuonConfig(), norm_group=GroupHandle.trivial("world"), device=DEV, others=vectors,
                         others_config=_config())
    single = _optimizer(alone)
    for seed in (1, 2):
        matrix.grad = torch.randn(48, 32, device=DEV, generator=gen)
        for params in (vectors, alone):
            _new_grads(params, seed)
        muon.step()
        single.step()
    assert all(torch.equal(p, q) for p, q in zip(vectors, alone))
    moments = muon.moments()
    assert moments[2] is None and torch.equal(moments[1][0], single.moments()[1][0])
    payload, momentum = muon.state_dict(), muon.inner.state[matrix]["momentum_buffer"].clone()
    muon.load_state_dict(payload)
    assert torch.equal(muon.inner.state[matrix]["momentum_buffer"], momentum)
    assert all(torch.equal(x, y) for x, y in zip(_codes(muon, vectors[1]), _codes(single, alone[1])))


@pytest.mark.parametrize("group", [2, 3])
def test_a_checkpoint_restores_the_moments_at_another_width(tmp_path, group):
    named = [("a", torch.nn.Parameter(torch.randn(301, 50, device=DEV))), ("b", torch.nn.Parameter(torch.randn(77, device=DEV)))]
    total = 301 * 50 + 77

    def world(size):
        handles = [FlatParamHandle(named, None, GroupHandle.local_view("shard", size, r), FSDPConfig(),
                                   MixedPrecisionConfig(), DEV, keep_originals=True) for r in range(size)]
        return handles, [_optimizer([h.flat_param]) for h in handles]

    handles, optimizers = world(2)
    for h, o in zip(handles, optimizers):
        h.flat_param.grad = torch.randn(h.shard_numel, device=DEV) * 1e-2
        o.step()
    shards = [(r, *collect_flat_shard_payload(h, rank=r, optimizer=o)) for r, (h, o) in enumerate(zip(handles, optimizers))]
    path = write_checkpoint(tmp_path, 1, shards, topology={"fsdp": 2})
    readers, restored = world(group)
    for h, o in zip(readers, restored):
        load_flat_shard_checkpoint(path, h, optimizer=o)
    for k in (0, 1):
        saved = torch.cat([o.moments()[0][k].reshape(-1) for o in optimizers])[:total]
        found = torch.cat([o.moments()[0][k].reshape(-1) for o in restored])[:total]
        if group == 2:
            assert torch.equal(saved, found)
        else:  # other blocks, rounded once more: half a step of 4 or of 5 bits, or of the smallest code
            if k == 1:
                saved, found = saved.sqrt(), found.sqrt()
            step = 2.0**-4 if k == 0 else 2.0**-5
            assert ((saved - found).abs() <= saved.abs() * (step + 2.0**-22) + 2.0**-18 * saved.abs().max()).all()
    assert all(o.inner.state[h.flat_param]["step"] == 1 for h, o in zip(readers, restored))


def test_state_that_does_not_fit_is_refused():
    params = _params([300])
    p = params[0]
    optimizer = _optimizer(params)
    optimizer.step()
    before = [p.detach().clone(), *_codes(optimizer, p)]
    kept = optimizer.inner.state[p]["moment_codes"]
    for wrong in (kept[:1], kept.float(), kept.cpu()):
        optimizer.inner.state[p]["moment_codes"] = wrong
        with pytest.raises(ShardingError, match="moment_codes"):
            optimizer.step()
    optimizer.inner.state[p]["moment_codes"] = kept
    assert optimizer.inner.state[p]["step"] == 1
    assert all(torch.equal(x, y) for x, y in zip(before, [p.detach(), *_codes(optimizer, p)]))
    payload = optimizer.state_dict()
    payload["state"][0]["exp_avg"] = torch.zeros(7)
    with pytest.raises(ShardingError, match="one value per element"):
        optimizer.load_state_dict(payload)
    with pytest.raises(UnsupportedFeatureError, match="float32 or bfloat16"):
        optimizer.moments(torch.float16)
    with pytest.raises(UnsupportedFeatureError, match="8-bit moments"):
        _optimizer([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64, device=DEV))])
    with pytest.raises(UnsupportedFeatureError, match="8-bit moments"):
        _optimizer([torch.nn.Parameter(torch.zeros(4))])
