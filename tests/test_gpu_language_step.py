"""The loss over a vocabulary and the 8-bit AdamW step in the training step that both are made for.

A small language model (an embedding shared with the output head, two fused layers) takes steps:
forward, the loss with its gradients, bucket pack, global clip, the 8-bit update, eagerly and
recorded into a graph.
"""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn as nn

from hybrid_training_amd import (
    BucketedGradients,
    DDPConfig,
    FlatParamHandle,
    FSDPConfig,
    FusedLinear,
    GradScaler,
    GradScalerConfig,
    GroupHandle,
    LinearCrossEntropy,
    MixedPrecisionConfig,
    OptimizerConfig,
    ShardedOptimizer,
    StepGraph,
    linear_cross_entropy,
)
from hybrid_training_amd import moments8

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
VOCAB, WIDTH, TOKENS, HIDDEN = 1003, 64, 300, 128
CONFIG = OptimizerConfig(learning_rate=1e-3, weight_decay=0.01, state_format="8bit")


class Model(nn.Module):
    def __init__(self, dtype: torch.dtype) -> None:
        super().__init__()
        torch.manual_seed(3)
        options = dict(device=DEV, dtype=dtype)
        self.embedding = nn.Embedding(VOCAB, WIDTH, **options)
        self.up = FusedLinear(WIDTH, HIDDEN, activation="gelu_tanh", **options)
        self.down = FusedLinear(HIDDEN, WIDTH, **options)
        self.head = LinearCrossEntropy(WIDTH, VOCAB, bias=True, **options)

    def hidden(self, tokens: torch.Tensor) -> torch.Tensor:
        x = self.embedding(tokens)
        return self.down(self.up(x), residual=x)

    def forward(self, tokens: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
        return self.head(self.hidden(tokens), target)


def _batch(seed: int) -> tuple[torch.Tensor, torch.Tensor]:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    tokens = torch.randint(VOCAB, (TOKENS,), device=DEV, generator=gen)
    target = torch.roll(tokens, -1)
    target[torch.rand(TOKENS, device=DEV, generator=gen) < 0.1 * seed] = -100
    return tokens, target


class Training:
    """A model, its buckets and optimizer; the hidden states' step alone can be recorded (torch's
    embedding gradient sums in no fixed order, so it is left out of what is compared bit for bit)."""

    def __init__(self, dtype: torch.dtype) -> None:
        self.model = Model(dtype)
        self.x = torch.zeros(TOKENS, WIDTH, device=DEV, dtype=dtype)
        self.target = torch.zeros(TOKENS, dtype=torch.int64, device=DEV)
        named = [(n, p) for n, p in self.model.named_parameters() if not n.startswith("embedding")]
        self.params = [p for _, p in named]
        world = GroupHandle.trivial("world")
        self.buckets = BucketedGradients(named, world, DDPConfig())
        self.optimizer = ShardedOptimizer(self.params, CONFIG, norm_group=world, device=DEV, defer_clip=True)

    def step(self) -> torch.Tensor:
        m = self.model
        loss = m.head(m.down(m.up(self.x), residual=self.x), self.target)
        loss.backward()
        self.buckets.synchronize()
        self.optimizer.clip_and_step(0.5)
        for p in self.params:
            p.grad.zero_()
        return loss.detach()

    def fill(self, seed: int) -> None:
        tokens, target = _batch(seed)
        with torch.no_grad():
            self.x.copy_(self.model.embedding(tokens))
            self.target.copy_(target)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_recorded_steps_equal_eager_ones(dtype):
    eager, taped = Training(dtype), Training(dtype)
    for t in (eager, taped):
        t.fill(1)
        t.step()
    graph = StepGraph(taped.step)
    for seed in range(2, 6):
        for t in (eager, taped):
            t.fill(seed)
        loss = eager.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(loss) and torch.equal(loss, graph.output)
        for p, q in zip(eager.params, taped.params):
            assert torch.equal(p, q)
            a, b = eager.optimizer.inner.state[p], taped.optimizer.inner.state[q]
            assert a["step"] == b["step"] and all(torch.equal(a[k], b[k]) for k in moments8.STATE_KEYS)


def test_gradients_of_a_whole_model_with_shared_weights():
    """The embedding's weight is the head's too: its gradient is the sum of both uses.  Against
    float64 autograd; fp32 sums of at most 1003 terms through four layers stay within 2^-14 of the
    largest gradient of each tensor (1003 2^-24 a product, four of them and their slopes)."""
    model = Model(torch.float32)
    model.head.weight = model.embedding.weight
    tokens, target = _batch(2)
    loss = model(tokens, target)
    loss.backward()
    wide = {n: p.detach().double().requires_grad_(True) for n, p in model.named_parameters()}
    e = wide["embedding.weight"]
    x = e[tokens]
    z = x @ wide["up.weight"].t() + wide["up.bias"]
    h = z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z**3))
    out = h @ wide["down.weight"].t() + wide["down.bias"] + x
    rows = target != -100
    want = torch.nn.functional.cross_entropy(out[rows] @ e.t() + wide["head.bias"], target[rows])
    grads = torch.autograd.grad(want, list(wide.values()))
    assert abs(float(loss.detach()) - float(want.detach())) <= 2.0**-18 * float(want.detach())
    for (name, p), g in zip(model.named_parameters(), grads):
        assert (p.grad.double() - g).abs().max() <= 2.0**-14 * g.abs().max(), name


def test_a_loss_scaled_float16_step():
    """fp16 throughout: the scaled loss's gradients are the unscaled ones times a power of two, a
    step that overflows is skipped, and the next one is taken."""
    training = Training(torch.float16)
    scaler = GradScaler(GradScalerConfig(enabled=True, init_scale=2.0**12), GroupHandle.trivial(), DEV)
    training.fill(1)
    m = training.model

    def backward(x: torch.Tensor) -> None:
        for p in training.params:
            p.grad = None
        scaler.scale(m.head(m.down(m.up(x), residual=x), training.target)).backward()

    backward(training.x)
    scaled = [p.grad.clone() for p in training.params]
    for p in training.params:
        p.grad = None
    m.head(m.down(m.up(training.x), residual=training.x), training.target).backward()
    for p, g in zip(training.params, scaled):
        # both round to fp16 once per product; the unscaled one also to fp16's smallest steps
        near = (p.grad.double().abs() * 2.0**-9 + 2.0**-23) + 2.0**-9 * p.grad.double().abs().max()
        assert ((g.double() / 2.0**12 - p.grad.double()).abs() <= near).all()
    backward(training.x)
    before = [p.detach().clone() for p in training.params]
    assert scaler.step(training.optimizer, training.params)
    assert any(not torch.equal(a, p) for a, p in zip(before, training.params))
    held = [p.detach().clone() for p in training.params]
    scaler.update()
    backward(torch.full_like(training.x, math.inf))
    assert not scaler.step(training.optimizer, training.params)
    assert all(torch.equal(a, p) for a, p in zip(held, training.params))
    assert all(training.optimizer.inner.state[p]["step"] == 1 for p in training.params)
    scaler.update()
    backward(training.x)
    assert scaler.step(training.optimizer, training.params)


def test_on_a_flat_shard():
    """The head's weight and bias as views into an FSDP unit's gathered flat parameter, off 16
    bytes, its shard stepped in 8 bits: the gradients are the plain ones', the shard moves as a
    parameter of its own would."""
    torch.manual_seed(0)
    named = [("bias", nn.Parameter(torch.randn(333, device=DEV))),
             ("weight", nn.Parameter(torch.randn(333, 48, device=DEV) * 0.1))]
    world = GroupHandle.local_view("shard", 1, 0)
    handle = FlatParamHandle(named, None, world, FSDPConfig(), MixedPrecisionConfig(), DEV, keep_originals=True)
    x, target = torch.randn(90, 48, device=DEV), torch.randint(333, (90,), device=DEV)
    full = handle.full_tensors()
    bias, weight = full["bias"], full["weight"]
    leaves = [bias.detach().requires_grad_(True), weight.detach().requires_grad_(True)]
    grads = torch.autograd.grad(linear_cross_entropy(x, leaves[1], target, leaves[0]), leaves)
    plain = [named[0][1].detach().clone().requires_grad_(True), named[1][1].detach().clone().requires_grad_(True)]
    want = torch.autograd.grad(linear_cross_entropy(x, plain[1], target, plain[0]), plain)
    for g, w in zip(grads, want):
        assert (g - w).abs().max() <= 2.0**-18 * w.abs().max()
    flat = torch.zeros(handle.padded_numel, device=DEV)
    flat[: 333 * 49] = torch.cat([want[0], want[1].reshape(-1)])
    handle.flat_param.grad = flat[: handle.shard_numel].clone()
    alone = nn.Parameter(handle.flat_param.detach().clone())
    alone.grad = handle.flat_param.grad.clone()
    one = ShardedOptimizer([handle.flat_param], CONFIG, norm_group=GroupHandle.trivial("world"), device=DEV)
    two = ShardedOptimizer([alone], CONFIG, norm_group=GroupHandle.trivial("world"), device=DEV)
    assert torch.equal(one.clip_and_step(0.1), two.clip_and_step(0.1))
    assert torch.equal(handle.flat_param.detach(), alone.detach())
