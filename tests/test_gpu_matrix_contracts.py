"""What the matrix operators promise at their entry points beyond plain results: the gradients of a
pre-activation past its dtype's range, the bits the iterate is held in, matrices that hold a
non-finite value, working storage that is missing or short, outputs over inputs, and layers whose
parameters are views into a flat FSDP unit."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from hybrid_training_amd import (
    FlatParamHandle,
    FSDPConfig,
    FusedLinear,
    GroupHandle,
    MixedPrecisionConfig,
    OptimizerConfig,
    ShardedOptimizer,
    _native,
    fused_linear,
    orthogonalize,
)

from .test_gpu_linear import DTYPES, close, make, reference
from .test_gpu_muon import PRODUCT, exact, gradient, off

pytestmark = pytest.mark.gpu


# ---- values ----------------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [40, 100])  # one workgroup's backward pass, and the slope pass
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
def test_slopes_of_preactivations_past_float16(device, name, tokens):
    """z = +-320000 is infinite as float16 keeps it; the slopes there are still 1 and 0."""
    x = torch.full((tokens, 8), 200.0, dtype=torch.float16, device=device).requires_grad_(True)
    w = torch.tensor([[200.0], [-200.0]], dtype=torch.float16, device=device).expand(2, 8).contiguous().requires_grad_(True)
    b = torch.zeros(2, dtype=torch.float16, device=device).requires_grad_(True)
    y = fused_linear(x, w, b, activation=name)
    y.backward(torch.ones_like(y))
    assert torch.equal(y, torch.tensor([float("inf"), 0.0], dtype=y.dtype, device=device).expand(tokens, 2))
    assert b.grad.tolist() == [tokens, 0]
    assert torch.equal(x.grad, torch.full_like(x, 200.0))
    assert torch.equal(w.grad, torch.tensor([[200.0 * tokens], [0.0]], dtype=w.dtype, device=device).expand(2, 8))


@pytest.mark.parametrize("tokens", [40, 100])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
def test_a_nan_preactivation_has_nan_gradients(device, name, dtype, tokens):
    x, w, b, _, dy = make(device, tokens, 24, 32, dtype, residual=False)
    x[3, 5] = float("nan")
    leaf = x.clone().requires_grad_(True)
    fused_linear(leaf, w, b, activation=name).backward(dy)
    rows = torch.arange(tokens, device=device) != 3
    assert bool(leaf.grad[3].isnan().all()) and bool(leaf.grad[rows].isfinite().all())


@pytest.mark.parametrize("steps", [1, 2, 3])
@pytest.mark.parametrize("shape", [(200, 300), (1400, 1001), (136, 20000), (4100, 4100)], ids=str)
def test_the_iterate_beside_float16_products_keeps_22_bits(device, shape, steps):
    """With b = c = 0 a step is x = a x: what is left is how the iterate is held.

    The fp16 value of x leaves at most 2^-11 |x|, whose own fp16 rounding is 2^-11 of that: 2^-22 a
    pair, three more fp32 roundings a step, once more for u / |u| (its norm, factor and product).
    Below fp16's normal range, 2^-14, the pair is 2^-36 off at most, in units of 1 / scale, where the
    iterate's scale is a power of two of at least half the square root of the longer side."""
    g = gradient(device, *shape)
    (got,) = orthogonalize([g], steps=steps, coefficients=(1.0, 0.0, 0.0), dtype=torch.float32, product_dtype="float16")
    want = g.double() / g.double().norm()
    unit = 2.0**-36 / (0.5 * max(shape) ** 0.5)
    bound = steps * (2.0**-22 * want.abs() + 3 * 2.0**-24 * want.abs() + unit) + 3 * 2.0**-24 * want.abs()
    excess = ((got.double() - want).abs() - bound).max()
    assert float(excess) <= 0, f"{float(excess):.3e} past its bound, of elements near {float(want.abs().mean()):.3e}"


@pytest.mark.parametrize("product", [torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("shape", [(24, 40), (90, 70), (300, 200), (200, 300), (9001, 16)], ids=str)
def test_a_nonfinite_value_reaches_its_whole_matrix(device, shape, value, product):
    bad = gradient(device, *shape)
    bad[3, 5] = value
    clean = gradient(device, *shape, seed=1)
    found = orthogonalize([clean, bad, clean], product_dtype=product)
    assert not bool(found[1].isfinite().any())
    assert bool(found[0].isfinite().all()) and torch.equal(found[0], found[2])


# ---- working storage and overlaps ------------------------------------------------------------
def call(x, w, b, r, y, activation=3, space=None):
    lib, (tokens, inner), outer = _native.library(), x.shape, w.shape[0]
    ldr = 0 if r is None else r.stride(0)
    _native.check(lib.hbt_linear(
        x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), b.data_ptr(), None if r is None else r.data_ptr(), ldr,
        y.data_ptr(), y.stride(0), None, 0, tokens, inner, outer, _native.dtype_code(x.dtype), activation,
        None if space is None else space.data_ptr(), 0 if space is None else space.numel(),
        _native.stream_of(x.device)), "test")
    return y


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(64, 4096, 64), (65, 2085, 70)], ids=str)
def test_working_storage_that_is_short_or_missing(device, shape, dtype):
    """The sum is split less, or not at all; every result keeps the bound of a sum in any order."""
    x, w, b, r, dy = make(device, *shape, dtype)
    need = _native.library().hbt_linear_workspace(shape[0], shape[1], shape[2], _native.dtype_code(dtype))
    part = 4 * shape[0] * ((shape[2] + 3) // 4 * 4)
    assert need >= 3 * part
    want, _, bound = reference(x, w, b, r, dy, "gelu_tanh")
    for nbytes in (0, part, 2 * part, 3 * part - 1, need):
        guard = torch.full((nbytes + 256,), 7, dtype=torch.uint8, device=device)
        space = guard[:nbytes] if nbytes else None
        close(call(x, w, b, r, torch.empty_like(r), space=space), want, bound["y"], f"{nbytes} bytes")
        assert bool((guard[nbytes:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(3, 90, 50), (64, 4096, 64), (130, 129, 257), (300, 520, 264), (1000, 64, 50000)], ids=str)
def test_the_result_may_be_the_residual(device, shape, dtype):
    """Few rows, a split sum, tiles of each kind and a result in two launches."""
    print(shape, dtype, flush=True)
    x, w, b, r, _ = make(device, *shape, dtype)
    space = torch.empty(1 << 24, dtype=torch.uint8, device=device)
    want = call(x, w, b, r, torch.empty_like(r), space=space)
    assert torch.equal(call(x, w, b, r, r, space=space), want)


@pytest.mark.parametrize("product", [_native.DTYPE_F16, _native.DTYPE_F32])
@pytest.mark.parametrize("shape", [(24, 40), (40, 24), (300, 70), (200, 264), (264, 200), (9001, 16)], ids=str)
def test_an_output_may_be_its_input(device, shape, product):
    """A matrix in one workgroup, with float32 and with float16 products, and a Gram sum in parts."""
    lib, g = _native.library(), gradient(device, *shape)
    rows, cols = _native.int64_array([shape[0]]), _native.int64_array([shape[1]])
    space = torch.empty(max(lib.hbt_orthogonal_workspace(rows, cols, 1, product), 1), dtype=torch.uint8, device=device)

    def run(source, result):
        _native.check(lib.hbt_orthogonalize(
            _native.pointer_array([source.data_ptr()]), _native.pointer_array([result.data_ptr()]), rows, cols, 1, 0, 0,
            product, 5, 3.4445, -4.7750, 2.0315, 1e-12, space.data_ptr(), space.numel(), _native.stream_of(device)), "test")
        return result

    want = run(g, torch.empty_like(g))
    assert off(want, exact(g)) < PRODUCT[torch.float16 if product == _native.DTYPE_F16 else torch.float32]
    assert torch.equal(run(g, g), want)


# ---- layers inside a flat unit -----------------------------------------------------------------
class Pair(nn.Module):
    def __init__(self, device, dtype):
        super().__init__()
        # the odd bias leaves the second layer's weight off 16 bytes
        self.up = FusedLinear(40, 33, activation="gelu_tanh", device=device, dtype=dtype)
        self.down = FusedLinear(33, 24, device=device, dtype=dtype)

    def forward(self, x, residual):
        return self.down(self.up(x), residual=residual)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("tokens", [5, 50, 130])
def test_layers_of_a_flat_unit(device, tokens, dtype):
    """Parameters as views into a gathered buffer, its bytes freed between the forward and the
    backward pass, the buffer's gradient reduced and stepped."""
    torch.manual_seed(0)
    plain = Pair(device, dtype)
    unit = Pair(device, dtype)
    unit.load_state_dict(plain.state_dict())
    named = list(unit.named_parameters())
    places = {id(p): [(unit.get_submodule(n.rpartition(".")[0]), n.rpartition(".")[2])] for n, p in named}
    handle = FlatParamHandle(named, places, GroupHandle.trivial("shard"), FSDPConfig(), MixedPrecisionConfig(), device)
    x, r, dy = (torch.randn(tokens, n, device=device).to(dtype) for n in (40, 24, 24))
    full = handle.gather_full().requires_grad_(True)
    handle.bind_views(full)
    assert unit.down.weight.data_ptr() % 16 != 0
    got = unit(x, r)
    handle.reshard()
    handle.refill(full)
    got.backward(dy)
    want = plain(x, r)
    want.backward(dy)
    # The same sums in another order (whole rows, and rows off 16 bytes): a few roundings of each value.
    near = 2.0**-6 if dtype == torch.bfloat16 else 1e-5
    assert float((got.float() - want.float()).norm()) <= near * float(want.float().norm())
    sizes = [p.numel() for _, p in plain.named_parameters()]
    for (name, p), part in zip(plain.named_parameters(), full.grad.split([*sizes, full.numel() - sum(sizes)])):
        assert float((part.view(p.shape).float() - p.grad.float()).norm()) <= near * float(p.grad.float().norm()), name
    optimizer = ShardedOptimizer([handle.flat_param], OptimizerConfig(learning_rate=1e-2),
                                 norm_group=GroupHandle.trivial("world"), device=device)
    before = handle.flat_param.detach().clone()
    handle.flat_param.grad = handle.reduce_scatter_gradient(full.grad)
    optimizer.step()
    assert not torch.equal(handle.flat_param, before) and bool(handle.flat_param.isfinite().all())
