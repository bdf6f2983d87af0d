"""What the matrix operators promise at their entry points beyond plain results: the gradients of a
pre-activation past its dtype's range, the bits the iterate is held in."""

from __future__ import annotations

import pytest
import torch

from hybrid_training_amd import fused_linear, orthogonalize

from .test_gpu_linear import DTYPES, make
from .test_gpu_muon import gradient

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
