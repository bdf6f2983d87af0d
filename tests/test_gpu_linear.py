"""The fused linear layer against its definition in float64, forward and backward.

Bounds, per element, derived from the arithmetic: a product of K terms summed in fp32 in any
order is off by at most K 2^-24 sum |x| |w|; a store rounds once (unit u of the dtype); the
backward pass reads z rounded once, which moves act'(z) by at most max |act''| u |z| (below
0.8 for GELU, 0.5 for SiLU, 0 for ReLU); 2-byte activations use exponentials and reciprocals
good to a few 2^-23, held here to 2^-18.
"""

from __future__ import annotations

import math

import pytest
import torch

from hybrid_training_amd import FusedLinear, ShardingError, UnsupportedFeatureError, fused_linear

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
#: The smallest step of each dtype near zero (fp16's subnormals).
FLOOR = {torch.bfloat16: 1e-37, torch.float16: 2.0**-24, torch.float32: 1e-37}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SHAPES = [
    (1, 1, 1), (1, 23, 32), (16, 23, 32), (17, 64, 64), (5, 7, 3), (130, 129, 257), (257, 8, 1), (33, 1000, 65),
    (128, 128, 128), (300, 520, 264), (1, 4097, 1000), (2, 4096, 33), (64, 4096, 64), (65, 2085, 70),
    (2100, 72, 2050), (4100, 200, 4100),
]


def activation64(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def make(device, tokens, inner, outer, dtype, bias=True, residual=True):
    gen = torch.Generator(device=device).manual_seed(tokens * 7 + inner * 3 + outer)
    draw = lambda *shape, scale=1.0: (torch.randn(*shape, device=device, generator=gen) * scale).to(dtype)  # noqa: E731
    return (draw(tokens, inner), draw(outer, inner, scale=max(inner, 1) ** -0.5), draw(outer) if bias else None,
            draw(tokens, outer) if residual else None, draw(tokens, outer))


def reference(x, w, b, r, dy, name):
    """Results and gradients in float64, and the per-element bounds of each."""
    u, floor = UNIT[x.dtype], FLOOR[x.dtype]
    leaves = [None if t is None else t.detach().double().requires_grad_(True) for t in (x, w, b, r)]
    X, W, B, R = leaves
    z = X @ W.t()
    z = z if B is None else z + B
    y = activation64(z, name)
    y = y if R is None else y + R
    (slope,) = torch.autograd.grad(activation64(z, name).sum(), z, retain_graph=True)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.double())
    found = dict(zip([k for k, t in zip("xwbr", leaves) if t is not None], grads))
    with torch.no_grad():
        eps, coarse = 2.0**-24, 0.0 if x.dtype == torch.float32 else 2.0**-18
        tokens, inner = x.shape
        outer = w.shape[0]
        product = (inner + 4) * eps * (X.abs() @ W.abs().t() + (0 if B is None else B.abs()))
        bound = {"y": 1.2 * product + u * y.abs() + (coarse + 8 * eps) * (z.abs() + y.abs()) + floor}
        dY = dy.double()
        dz = dY * slope
        curve = {"none": 0.0, "relu": 0.0, "silu": 0.5}.get(name, 0.8)
        first = dY.abs() * (curve * (product + u * z.abs() * (name != "none")) + coarse + 8 * eps) + floor
        if name == "relu":  # z near 0 may change sign with the product's rounding
            first = first + dY.abs() * (z.abs() <= 1.2 * product)
        rounded = first + u * dz.abs() * (name != "none")
        bound["x"] = rounded @ W.abs() + (outer + 4) * eps * (dz.abs() @ W.abs()) + u * found["x"].abs() + floor
        bound["w"] = (rounded.t() @ X.abs() + (tokens + 4) * eps * (dz.abs().t() @ X.abs()) + u * found["w"].abs()
                      + floor)
        bound["b"] = first.sum(0) + (tokens + 4) * eps * dz.abs().sum(0) + floor
        if B is not None:
            bound["b"] = bound["b"] + u * found["b"].abs()
    return y.detach(), found, bound


def close(got, want, bound, what):
    assert got.shape == want.shape
    excess = (got.double() - want).abs() - bound
    assert bool((excess <= 0).all()), f"{what}: {float(excess.max()):.3e} past its bound"


def run(x, w, b, r, dy, name):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, r)]
    y = fused_linear(leaves[0], leaves[1], leaves[2], activation=name, residual=leaves[3])
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    return y.detach(), dict(zip([k for k, t in zip("xwbr", leaves) if t is not None], grads))


def check(x, w, b, r, dy, name):
    want, grads, bound = reference(x, w, b, r, dy, name)
    y, got = run(x, w, b, r, dy, name)
    assert y.dtype == x.dtype
    close(y, want, bound["y"], "y")
    for key in [k for k in "xwb" if k in grads]:
        close(got[key], grads[key], bound[key], "d" + key)
    if "r" in got:
        assert torch.equal(got["r"], dy)
    with torch.no_grad():  # without a graph: the same kernel, z not stored
        assert torch.equal(fused_linear(x, w, b, activation=name, residual=r), y)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(device, shape, dtype):
    print(shape, dtype, flush=True)
    check(*make(device, *shape, dtype), "gelu")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_epilogues(device, name, bias, residual, dtype):
    check(*make(device, 70, 90, 50, dtype, bias, residual), name)
    check(*make(device, 3, 90, 50, dtype, bias, residual), name)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(0, 8, 8), (8, 0, 8), (8, 8, 0), (40, 0, 33), (0, 0, 0)], ids=str)
def test_empty_sides(device, shape, dtype):
    tokens, inner, outer = shape
    x, w, b, r, dy = make(device, *shape, dtype)
    y, grads = run(x, w, b, r, dy, "none")
    assert torch.equal(y, (b.float() + r.float()).to(dtype) if tokens and outer else y.new_zeros(tokens, outer))
    assert torch.equal(grads["x"], (dy.float() @ w.float()).to(dtype) if inner and outer else torch.zeros_like(x))
    assert grads["w"].shape == w.shape and (tokens or not grads["w"].any())
    assert grads["b"].shape == b.shape and (tokens or not grads["b"].any())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(3, 37, 45), (66, 37, 45), (140, 200, 136)], ids=str)
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_operands_inside_wider_rows_of_nan(device, shape, dtype, offset):
    """Every operand is a window of a buffer of NaN: nothing outside it may be read into a
    result, at any alignment of its first element and of its rows."""
    tokens, inner, outer = shape
    x, w, b, r, dy = make(device, *shape, dtype)

    def window(t, extra):
        wide = torch.full((t.shape[0] + 2, t.shape[1] + offset + extra), float("nan"), dtype=dtype, device=device)
        inside = wide[1 : 1 + t.shape[0], offset : offset + t.shape[1]]
        inside.copy_(t)
        return inside

    check(window(x, 3), window(w, 8), b, window(r, 1), window(dy, 5), "silu")


def test_other_layouts(device):
    x, w, b, r, dy = make(device, 24, 40, 56, torch.bfloat16)
    want = fused_linear(x, w, b, residual=r)
    assert torch.equal(fused_linear(x, w.t().contiguous().t(), b, residual=r), want)  # W stored transposed
    assert torch.equal(fused_linear(x.t().contiguous().t(), w, b, residual=r), want)
    assert torch.equal(fused_linear(x.view(2, 3, 4, 40), w, b, residual=r.view(2, 3, 4, 56)).view(24, 56), want)
    assert torch.equal(fused_linear(x[0], w, b, residual=r[0]), fused_linear(x[:1], w, b, residual=r[:1])[0])
    shared = x[:1].expand(24, 40)  # rows that share their memory
    assert torch.equal(fused_linear(shared, w, b, residual=r), fused_linear(shared.contiguous(), w, b, residual=r))
    spread = torch.zeros(112, dtype=b.dtype, device=device)
    spread[::2] = b
    assert torch.equal(fused_linear(x, w, spread[::2], residual=r), want)
    # a broadcast gradient (the loss is a sum)
    leaf = w.clone().requires_grad_(True)
    fused_linear(x, leaf, b).sum().backward()
    (dw,) = torch.autograd.grad(fused_linear(x, leaf, b), leaf, torch.ones_like(dy))
    assert torch.equal(leaf.grad, dw)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_nonfinite_values_stay_in_their_rows(device, dtype):
    x, w, b, r, dy = make(device, 150, 70, 80, dtype)
    clean = fused_linear(x, w, b, activation="gelu_tanh", residual=r)
    x[7, 3], x[80, 69] = float("nan"), float("inf")
    got = fused_linear(x, w, b, activation="gelu_tanh", residual=r)
    rows = torch.ones(150, dtype=torch.bool, device=device)
    rows[7] = rows[80] = False
    assert torch.equal(got[rows], clean[rows])
    assert bool(got[7].isnan().all()) and not bool(got[80].isfinite().all())
    assert bool(fused_linear(x[7:8], w, b, activation="relu").isnan().all())


@pytest.mark.parametrize("tokens", [40, 100])  # one workgroup's backward pass, and the slope pass
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
def test_slopes_far_from_zero(device, name, dtype, tokens):
    # z is the bias, whose square and cube pass float32: the slopes are 0 and 1, the sums whole numbers.
    b = torch.tensor([1e25, -1e25, 100.0, -120.0], device=device, dtype=dtype).requires_grad_(True)
    x = torch.zeros(tokens, 8, device=device, dtype=dtype)
    w = torch.zeros(4, 8, device=device, dtype=dtype)
    y = fused_linear(x, w, b, activation=name)
    y.backward(torch.ones_like(y))
    with torch.no_grad():
        assert torch.equal(y, b.clamp_min(0).expand(tokens, 4))
    assert b.grad.tolist() == [tokens, 0, tokens, 0]


def test_gradients_match_differences(device):
    x, w, b, r, dy = make(device, 6, 9, 7, torch.float32)
    for name in ("gelu", "gelu_tanh", "silu"):
        _, grads = run(x, w, b, r, dy, name)
        for key, t in zip("xwb", (x, w, b)):
            step, parts = 1e-4, [v.double() for v in (x, w, b)]
            base = parts["xwb".index(key)]
            flat = base.reshape(-1)
            numeric = torch.zeros_like(flat)
            for i in range(flat.numel()):
                values = []
                for sign in (1, -1):
                    moved = flat.clone()
                    moved[i] += sign * step
                    args = list(parts)
                    args["xwb".index(key)] = moved.view_as(base)
                    values.append(float((activation64(args[0] @ args[1].t() + args[2], name) * dy.double()).sum()))
                numeric[i] = (values[0] - values[1]) / (2 * step)
            # differences: step^2 times a third derivative (below 1e-7 here); fp32 gradients 1e-5
            assert float((grads[key].double().reshape(-1) - numeric).abs().max()) < 1e-5 * (1 + float(numeric.abs().max()))


def test_only_the_wanted_gradients(device):
    x, w, b, r, dy = make(device, 40, 30, 20, torch.float32)
    full = run(x, w, b, r, dy, "gelu")[1]
    for wanted in ("x", "w", "b", "r", "wb"):
        leaves = {k: t.detach().requires_grad_(k in wanted) for k, t in zip("xwbr", (x, w, b, r))}
        y = fused_linear(leaves["x"], leaves["w"], leaves["b"], activation="gelu", residual=leaves["r"])
        for key, g in zip(wanted, torch.autograd.grad(y, [leaves[k] for k in wanted], dy)):
            assert torch.equal(g, full[key])


def test_side_stream_and_repeated_bits(device):
    x, w, b, r, dy = make(device, 2000, 300, 130, torch.float16)
    want = run(x, w, b, r, dy, "silu")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            got = run(x, w, b, r, dy, "silu")
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and all(torch.equal(got[1][k], want[1][k]) for k in want[1])


def test_recorded_graph_replays(device):
    x, w, b, r, dy = make(device, 64, 4096, 64, torch.bfloat16)  # a split sum with its workspace
    eager = lambda: fused_linear(x, w, b, activation="gelu", residual=r)  # noqa: E731
    eager()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = eager()
    for k in range(3):
        x.copy_(torch.randn_like(x.float()).to(x.dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager()), k


def test_module(device):
    layer = FusedLinear(23, 32, activation="relu", device=device)
    plain = torch.nn.Linear(23, 32, device=device)
    plain.load_state_dict(layer.state_dict())
    x = torch.randn(16, 23, device=device)
    torch.testing.assert_close(layer(x), torch.relu(plain(x)), rtol=1e-5, atol=1e-6)
    assert "activation='relu'" in repr(layer)


def test_refusals(device):
    x, w, b, r, _ = make(device, 4, 8, 6, torch.float32)
    with pytest.raises(UnsupportedFeatureError, match="unknown activation"):
        fused_linear(x, w, activation="swish")
    with pytest.raises(ShardingError, match="inner size"):
        fused_linear(x, w.t())
    with pytest.raises(ShardingError, match="one value per output"):
        fused_linear(x, w, b[:5])
    with pytest.raises(ShardingError, match="result's shape"):
        fused_linear(x, w, b, residual=r[:3])
    with pytest.raises(UnsupportedFeatureError, match="one dtype"):
        fused_linear(x, w.half())
    with pytest.raises(UnsupportedFeatureError, match="one dtype"):
        fused_linear(x.double(), w.double())
    with pytest.raises(UnsupportedFeatureError, match="HIP device"):
        fused_linear(x.cpu(), w)
    with pytest.raises(UnsupportedFeatureError, match="unknown activation"):
        FusedLinear(4, 4, activation="tanh")
