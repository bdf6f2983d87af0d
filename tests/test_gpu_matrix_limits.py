"""The matrix operators at the edges of their layouts: long sums that end inside a k-tile, aligned
windows of NaN buffers, rows far apart, offsets past 32 bits, and the loss scaler around the
orthogonalised step."""

from __future__ import annotations

import pytest
import torch

from hybrid_training_amd import (
    GradScaler,
    GradScalerConfig,
    GroupHandle,
    MuonConfig,
    MuonOptimizer,
    fused_linear,
    orthogonalize,
)

from .test_gpu_linear import DTYPES, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("inner", [8, 40, 72, 120, 200, 264, 1016])
def test_aligned_sums_that_end_inside_a_tile(device, inner, dtype):
    """Rows on 16 bytes and a sum that is no whole number of k-tiles, in all three products."""
    print(inner, dtype, flush=True)
    check(*make(device, inner + 16, inner, 136, dtype), "none")
    check(*make(device, 136, 144, inner, dtype), "gelu_tanh")


@pytest.mark.parametrize("shape", [(1000, 64, 50000), (8200, 64, 2100), (2048, 65536, 2048)], ids=str)
def test_last_rounds_and_split_sums_of_large_tiles(device, shape):
    """Results whose last columns or rows are formed in smaller tiles, and a long sum split over
    large ones, with everything the epilogue does."""
    print(shape, flush=True)
    check(*make(device, *shape, torch.bfloat16), "relu")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(136, 72, 200), (520, 264, 312)], ids=str)
def test_aligned_windows_of_nan(device, shape, dtype):
    """Windows whose rows start on 16 bytes are read where they lie; nothing beside them is."""
    x, w, b, r, dy = make(device, *shape, dtype)

    def window(t):
        wide = torch.full((t.shape[0] + 16, t.shape[1] + 16), float("nan"), dtype=dtype, device=device)
        inside = wide[8 : 8 + t.shape[0], 8 : 8 + t.shape[1]]
        inside.copy_(t)
        return inside

    check(window(x), window(w), b, window(r), window(dy), "silu")


def test_rows_further_apart_than_the_kernels_address(device):
    x, w, b, r, _ = make(device, 20, 64, 48, torch.bfloat16)
    spread = torch.zeros(20, (1 << 20) + 8, dtype=torch.bfloat16, device=device)
    spread[:, :64] = x
    assert torch.equal(fused_linear(spread[:, :64], w, b, residual=r), fused_linear(x, w, b, residual=r))


def test_linear_past_32_bit_offsets(device):
    """An input of more than 2**31 elements, and 2**32 bytes, read by rows and by columns."""
    tokens, inner, outer = 66000, 33024, 24
    gen = torch.Generator(device=device).manual_seed(0)
    x = torch.empty(tokens, inner, dtype=torch.bfloat16, device=device)
    for part in x.split(4096):
        part.normal_(generator=gen)
    w = (torch.randn(outer, inner, device=device, generator=gen) / inner**0.5).to(torch.bfloat16).requires_grad_(True)
    dy = torch.randn(tokens, outer, device=device, generator=gen).to(torch.bfloat16)
    y = fused_linear(x, w)
    (dw,) = torch.autograd.grad(y, w, dy)
    for rows in (slice(0, 64), slice(tokens - 64, tokens)):
        want = x[rows].float() @ w.detach().float().t()
        assert float((y[rows].float() - want).abs().max()) < 2.0**-8 * float(want.abs().max()) + 1e-3
    want = torch.zeros(outer, 128, dtype=torch.float64, device=device)
    for first in range(0, tokens, 4096):
        want += dy[first : first + 4096].double().t() @ x[first : first + 4096, -128:].double()
    # bf16 rounding of the result, and a float32 sum of 66000 terms
    assert float((dw[:, -128:].double() - want).abs().max()) < 2.0**-8 * float(want.abs().max()) + 1e-2


@pytest.mark.parametrize("tall", [False, True])
def test_orthogonalize_past_32_bit_offsets(device, tall):
    side, length = 136, 1 << 20  # 2**27 elements a matrix, sixteen of them and one that is looked at
    gen = torch.Generator(device=device).manual_seed(1)
    shape = (length, side) if tall else (side, length)
    filler = torch.randn(*shape, device=device, generator=gen).to(torch.bfloat16)
    looked_at = torch.randn(*shape, device=device, generator=gen).to(torch.bfloat16)
    got = orthogonalize([filler] * 16 + [looked_at], steps=2)[-1]
    x = looked_at.float()
    x = x if not tall else x.t()
    x = x / x.norm()
    for _ in range(2):
        gram = x @ x.t()
        x = 3.4445 * x + (-4.7750 * gram + 2.0315 * gram @ gram) @ x
    x = x.t() if tall else x
    assert float((got.float() - x).norm() / x.norm()) < 5e-3 + 2.0**-8
    assert float((got[-5:].float() - x[-5:]).norm() / x[-5:].norm()) < 2e-2


def test_a_single_matrix_past_32_bit_offsets(device):
    """2100 x 2**20: its own elements pass 2**31."""
    side, length = 2100, 1 << 20
    gen = torch.Generator(device=device).manual_seed(2)
    u = torch.empty(side, length, dtype=torch.bfloat16, device=device)
    for part in u.split(128):
        part.normal_(generator=gen)
    (got,) = orthogonalize([u], steps=1)
    x = u.float()
    x /= x.norm()
    gram = x @ x.t()
    poly = -4.7750 * gram + 2.0315 * gram @ gram
    for rows in (slice(0, 8), slice(side - 8, side)):
        want = 3.4445 * x[rows] + poly[rows] @ x
        assert float((got[rows].float() - want).norm() / want.norm()) < 5e-3 + 2.0**-8


def test_loss_scaler_around_the_step(device):
    """Scaled gradients step as unscaled ones do; an overflow skips the step."""
    world = GroupHandle.trivial("world")
    shape, scale = (96, 200), 1024.0
    first = torch.randn(*shape, device=device) * 0.02
    gradient = torch.randn(*shape, device=device) * 1e-3
    results = []
    for scaled in (False, True):
        p = torch.nn.Parameter(first.clone())
        opt = MuonOptimizer([p], MuonConfig(learning_rate=1e-3), norm_group=world, device=device)
        p.grad = gradient * scale if scaled else gradient.clone()
        if scaled:
            scaler = GradScaler(GradScalerConfig(enabled=True, init_scale=scale), world, device)
            scaler.unscale_([p])
            opt.clip_grad_norm(0.05)
            scaler.step(opt, [p], already_unscaled=True)
            scaler.update()
            results.append(p.detach().clone())
            before = p.detach().clone()
            p.grad = torch.full_like(p, float("inf"))
            scaler.unscale_([p])
            scaler.step(opt, [p], already_unscaled=True)
            assert torch.equal(p, before)
        else:
            opt.clip_grad_norm(0.05)
            opt.step()
            results.append(p.detach().clone())
    assert torch.equal(*results)  # a power of two scales exactly
