"""Train a residual feed-forward network with the fused linear layer and orthogonalised updates.

Each block is ``x + down(gelu(up(x)))``, its activation, biases and residual in the two products'
epilogues (``FusedLinear``).  The gradients are packed into DDP buckets, clipped by their global
norm, and the weight matrices move along their orthogonalised momenta while biases take AdamW
steps (``MuonOptimizer``).  The whole step (forward, backward, pack, clip, update) is recorded
into a HIP graph after one eager step and replayed.

    python examples/feed_forward_muon.py --width 256 --hidden 1024 --blocks 4 --steps 100
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "build-your-own-hybrid-distributed-training_amd"))

from hybrid_training_amd import (  # noqa: E402
    BucketedGradients,
    DDPConfig,
    FusedLinear,
    GroupHandle,
    MuonConfig,
    MuonOptimizer,
    OptimizerConfig,
    StepGraph,
)


class Block(nn.Module):
    """``x + down(gelu(up(x)))``: two products, nothing between them."""

    def __init__(self, width: int, hidden: int, **options) -> None:
        super().__init__()
        self.up = FusedLinear(width, hidden, activation="gelu_tanh", **options)
        self.down = FusedLinear(hidden, width, **options)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.down(self.up(x), residual=x)


class Training:
    """A network, its buckets and optimizer, and one step over fixed input buffers."""

    def __init__(self, *, width: int, hidden: int, blocks: int, tokens: int, device: torch.device,
                 dtype: torch.dtype = torch.float32, learning_rate: float = 3e-3, max_norm: float = 1.0) -> None:
        options = dict(device=device, dtype=dtype)
        self.network = nn.Sequential(*[Block(width, hidden, **options) for _ in range(blocks)],
                                     FusedLinear(width, width, **options))
        self.max_norm = max_norm
        self.x = torch.zeros(tokens, width, **options)
        self.target = torch.zeros(tokens, width, **options)
        named = list(self.network.named_parameters())
        matrices = [p for _, p in named if p.dim() == 2]
        others = [p for _, p in named if p.dim() != 2]
        world = GroupHandle.trivial("world")
        self.buckets = BucketedGradients(named, world, DDPConfig())
        self.optimizer = MuonOptimizer(matrices, MuonConfig(learning_rate=learning_rate, weight_decay=0.01),
                                       norm_group=world, device=device, others=others,
                                       others_config=OptimizerConfig(learning_rate=learning_rate))

    def step(self) -> torch.Tensor:
        """Forward, backward, bucket pack, clip and update; the prediction.

        The mean squared error's gradient is formed element by element, so that no library
        reduction is recorded; :meth:`loss` reduces the returned prediction eagerly."""
        y = self.network(self.x)
        error = y.detach() - self.target
        y.backward(error * (2.0 / error.numel()))
        self.buckets.synchronize()
        self.optimizer.clip_grad_norm(self.max_norm)
        self.optimizer.step()
        for p in self.network.parameters():  # the buckets' views stay bound
            p.grad.zero_()
        return y.detach()

    def loss(self, prediction: torch.Tensor) -> float:
        return float((prediction.float() - self.target.float()).square().mean())


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--width", type=int, default=256)
    parser.add_argument("--hidden", type=int, default=1024)
    parser.add_argument("--blocks", type=int, default=4)
    parser.add_argument("--tokens", type=int, default=2048)
    parser.add_argument("--steps", type=int, default=100)
    parser.add_argument("--dtype", choices=["float32", "bfloat16", "float16"], default="float32")
    args = parser.parse_args()
    device = torch.device("cuda", 0)
    torch.manual_seed(0)
    training = Training(width=args.width, hidden=args.hidden, blocks=args.blocks, tokens=args.tokens, device=device,
                        dtype=getattr(torch, args.dtype))
    teacher = torch.randn(args.width, args.width, device=device) / args.width**0.5

    def fill() -> None:
        x = torch.randn(args.tokens, args.width, device=device)
        training.x.copy_(x)
        training.target.copy_(torch.tanh(x @ teacher))

    fill()
    first = training.loss(training.step())  # eager: creates the optimizer state and binds the buckets
    graph = StepGraph(training.step)
    for step in range(1, args.steps):
        fill()
        graph.replay()
        if step % max(1, args.steps // 10) == 0:
            print(f"step {step}: loss {training.loss(graph.output):.5f}", flush=True)
    print(f"loss {first:.5f} -> {training.loss(graph.output):.5f}", flush=True)


if __name__ == "__main__":
    main()
