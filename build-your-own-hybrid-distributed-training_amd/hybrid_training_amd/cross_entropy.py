"""Softmax cross entropy over a large vocabulary, from hidden states and the output head's weight.

:func:`linear_cross_entropy` is ``cross_entropy(x W^T + bias, target)`` without the logits in
memory (``hbt_linear_cross_entropy``): a tile of logits becomes its rows' statistics in the
workgroup that forms it.  With gradients wanted, the exponentials of a piece of the rows (at
most 2 GiB in 16 bits; float32 tensors keep 32) stand in working storage until the two products that follow
have read them, so nothing of that size outlives the call.

A summed or averaged loss computes its gradients in the forward pass, where the exponentials are,
and the backward pass multiplies them by the loss's own gradient: 6 operations for each token,
word and hidden value instead of 8.  Separate losses (``reduction="none"``), whose gradients are
known only then, and few float16 tokens of a large weight form the logits again in the backward pass.

Sums and statistics are float32 or wider, and so is the loss.  The gradient of the logits is rounded once to the
tensors' dtype, for the matrix cores; before that the probabilities of 2-byte tensors are held in fp16, to 2^-11 of
themselves or 2^-25 of the largest one beside them, the target's aside.  float16's gradients of separate losses share
one power of two, so tokens whose loss counts far less than the largest one's keep fewer digits.  Gradients of bfloat16 tensors are held rounded between
the passes, so a loss scaled by anything but a power of two rounds them twice; those of float16
tensors are held in float32, and a loss scale keeps what float16 alone would flush to zero.  No
atomics run, so equal inputs give equal bits.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _native
from .errors import ShardingError, UnsupportedFeatureError, format_error
from .linear import _holds_tangent, _rows

__all__ = ["LinearCrossEntropy", "REDUCTIONS", "linear_cross_entropy"]

#: Reduction names and their HBT_LOSS_* codes.
REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_INTEGERS = (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8)
#: Sizes that the kernels address (hbt_linear_cross_entropy's limits).
_MAX_SIDE, _MAX_TOKENS = (1 << 20) - 64, 1 << 24
_WHO = "cross_entropy.linear_cross_entropy"
#: Gradients of float16 tensors are computed in the forward pass and held in float32 from so many tokens
#: on, or for weights of fewer elements.  For few tokens of a large weight, writing and reading its
#: gradient costs more than forming the logits again.  Held and not, in us, for 32, 512, 768 and 1024 tokens:
#: 50257 x 768 (39M elements) 207 and 234, 353 and 376, 419 and 449, 480 and 532; 32768 x 2048 (67M) 294 and 260, 436
#: and 408, 541 and 552, 610 and 641; 128256 x 2048 921 and 716, 1439 and 1356, 1801 and 1861, 2153 and 2295;
#: 128256 x 4096 (525M) 1683 and 1219, 2635 and 2451, 3362 and 3405, 4017 and 4248.
_HOLD_TOKENS, _HOLD_ELEMENTS = 768, 3 << 24


def _check(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: torch.Tensor | None, reduction: str,
           label_smoothing: float) -> None:
    if reduction not in REDUCTIONS:
        raise UnsupportedFeatureError(format_error(_WHO, "unknown reduction", expected=sorted(REDUCTIONS),
                                                   observed=reduction))
    if not 0.0 <= label_smoothing <= 1.0:
        raise UnsupportedFeatureError(format_error(_WHO, "label_smoothing must lie in [0, 1]", expected="0 <= s <= 1",
                                                   observed=label_smoothing))
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ShardingError(
            format_error(_WHO, "x must end in the weight's inner size",
                         expected="x [..., inner] and weight [vocabulary, inner]",
                         observed=f"x {tuple(x.shape)}, weight {tuple(weight.shape)}"))
    vocab, inner = weight.shape
    if vocab < 1:
        raise ShardingError(format_error(_WHO, "the vocabulary is empty", observed=tuple(weight.shape)))
    if bias is not None and tuple(bias.shape) != (vocab,):
        raise ShardingError(format_error(_WHO, "the bias must hold one value per word", expected=(vocab,),
                                         observed=tuple(bias.shape)))
    if target.shape != x.shape[:-1]:
        raise ShardingError(format_error(_WHO, "there must be one target per token", expected=tuple(x.shape[:-1]),
                                         observed=tuple(target.shape)))
    given = [t for t in (x, weight, bias) if t is not None]
    for t in (*given, target):
        if not t.is_cuda:
            _native.require_device_tensor(t, _WHO)
        if t.device != x.device:
            raise ShardingError(format_error(_WHO, "x, weight, bias and target must be on one device",
                                             expected=str(x.device), observed=str(t.device)))
    if x.dtype not in _DTYPES or any(t.dtype != x.dtype for t in given):
        raise UnsupportedFeatureError(
            format_error(_WHO, "x, weight and bias share one dtype of bfloat16, float16 or float32",
                         observed=[str(t.dtype) for t in given]))
    if target.dtype not in _INTEGERS:
        raise UnsupportedFeatureError(format_error(_WHO, "targets are whole numbers", expected="int64",
                                                   observed=str(target.dtype)))
    if vocab > _MAX_SIDE or inner > _MAX_SIDE or target.numel() > _MAX_TOKENS:
        raise UnsupportedFeatureError(
            format_error(_WHO, "sizes past the kernels' limits",
                         expected=f"a vocabulary and an inner size of at most {_MAX_SIDE}, {_MAX_TOKENS} tokens",
                         observed=f"{target.numel()} tokens of {inner} over {vocab} words"))


def _compute(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, target: torch.Tensor, options: tuple,
             wants: tuple[bool, bool, bool], dloss: torch.Tensor | None = None):
    """(loss, [dx, dw, dbias], None where not wanted); with the loss's own gradient ``dloss`` (None, [...]).
    Without it, gradients of float16 tensors are float32."""
    ignore_index, reduction, smoothing = options
    vocab, inner = weight.shape
    device, dtype = x.device, x.dtype
    separate = reduction == "none"
    held = torch.float32 if dtype == torch.float16 and dloss is None else dtype
    loss = torch.empty(target.shape if separate else (), dtype=torch.float32, device=device) if dloss is None else None
    if dloss is not None:
        dloss = dloss.to(torch.float32).contiguous()
    grads = [torch.empty(t.shape, dtype=held, device=device) if want else None
             for t, want in zip((x, weight, bias), wants)]
    words = target.reshape(-1)
    if words.dtype != torch.int64 or not words.is_contiguous():
        words = words.to(torch.int64).contiguous()
    tokens = words.numel()
    if loss is None and not any(g is not None and g.numel() for g in grads):
        return loss, grads  # of an inner size of 0
    if tokens == 0:
        if loss is not None and not separate:
            loss.fill_(math.nan if reduction == "mean" else 0.0)
        for g in grads:
            if g is not None:
                g.zero_()
        return loss, grads
    rows, ldx = _rows(x, inner)
    w, ldw = _rows(weight, inner)
    b = None if bias is None else bias.contiguous()
    code, held_code = _native.dtype_code(dtype), _native.dtype_code(held)
    with _native.device_guard(device):
        lib = _native.library()
        mask = sum(bit for bit, g in zip((1, 2, 4), grads) if g is not None)
        size = x.element_size()
        aligned = (w.data_ptr() | ldw * size | inner * size) & 15 == 0
        nbytes = lib.hbt_linear_cross_entropy_workspace(tokens, inner, vocab, code, mask, held_code, smoothing, aligned)
        if nbytes < 0:
            _native.check(int(nbytes), "cross_entropy.hbt_linear_cross_entropy_workspace")
        space = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        at = [None if g is None else g.data_ptr() for g in grads]
        across = max(inner, 1)
        _native.check(lib.hbt_linear_cross_entropy(
            rows.data_ptr(), ldx, w.data_ptr(), ldw, None if b is None else b.data_ptr(), words.data_ptr(),
            dloss.data_ptr() if dloss is not None and separate else None,
            dloss.data_ptr() if dloss is not None and not separate else None,
            None if loss is None else loss.data_ptr(), at[0], across, at[1], across, at[2], tokens, inner, vocab, code,
            held_code, ignore_index, smoothing, REDUCTIONS[reduction], None if space is None else space.data_ptr(), nbytes,
            _native.stream_of(device)),
            "cross_entropy.hbt_linear_cross_entropy")
    return loss, grads


class _Scaling:
    """The call that multiplies ``grads`` by the loss's own gradient, a device scalar, into ``dtype``:
    in place where they are in it already, which reads and writes nothing for a factor of 1.

    Laid out in the forward pass: the backward one runs on autograd's own thread, where host
    code is slower."""

    def __init__(self, grads: list[torch.Tensor | None], dtype: torch.dtype) -> None:
        present = [g for g in grads if g is not None]
        self.device, held = present[0].device, present[0].dtype
        self.results = grads
        if held != dtype:
            self.results = [None if g is None else torch.empty(g.shape, dtype=dtype, device=g.device) for g in grads]
        self._held = grads
        self._tables = (
            _native.pointer_array([g.data_ptr() for g in present]),
            _native.pointer_array([r.data_ptr() for r in self.results if r is not None]),
            _native.int64_array([g.numel() for g in present]), len(present), _native.dtype_code(held),
            _native.dtype_code(dtype))

    def run(self, factor: torch.Tensor) -> list[torch.Tensor | None]:
        if factor.dtype != torch.float32:
            factor = factor.to(torch.float32)
        with _native.device_guard(self.device):
            _native.check(_native.library().hbt_scale_round(*self._tables, factor.data_ptr(),
                                                            _native.stream_of(self.device)),
                          "cross_entropy.hbt_scale_round")
        return self.results


def _refuse_eager_nodes(ctx, device: torch.device) -> None:
    """Refuse to record a step whose tensors still hang on an eager step's autograd nodes.

    Autograd runs a leaf's node on the stream that first used it, for as long as any loss keeps the node
    alive.  Where that was the default stream, which cannot join a recording, the recorded backward pass
    would end the process.  Each node notes its stream."""
    stream = _native.stream_of(device)
    for node, _ in ctx.next_functions:
        if node is not None and node.metadata.setdefault("linear_cross_entropy_stream", stream) != stream:
            if not node.metadata["linear_cross_entropy_stream"] and _native.capturing():
                raise UnsupportedFeatureError(
                    format_error(_WHO, "a loss of an eager step is still alive, and its parameters' autograd nodes with it",
                                 resolution="delete it, or keep loss.detach(), before recording a step"))


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, target, options):
        _refuse_eager_nodes(ctx, x.device)
        ctx.options, ctx.scaling = options, None
        ctx.holds = options[1] != "none" and (x.dtype != torch.float16 or target.numel() >= _HOLD_TOKENS
                                              or weight.numel() < _HOLD_ELEMENTS)
        if not ctx.holds:
            loss, _ = _compute(x, weight, bias, target, options, (False, False, False))
        else:
            wants = (x.requires_grad, weight.requires_grad, bias is not None and bias.requires_grad)
            loss, grads = _compute(x, weight, bias, target, options, wants)
            ctx.scaling = _Scaling(grads, x.dtype)
        ctx.save_for_backward(x, weight, bias, target)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        scaling, ctx.scaling = ctx.scaling, None  # its gradients become the leaves' own
        if scaling is not None:
            dx, dw, db = scaling.run(dloss)
            return dx, dw, db, None, None
        x, weight, bias, target = ctx.saved_tensors
        wants = ctx.needs_input_grad[:3]
        if ctx.holds:  # a second backward pass, with the first one's bits
            _, grads = _compute(x, weight, bias, target, ctx.options, wants)
            grads = _Scaling(grads, x.dtype).run(dloss)
        else:
            _, grads = _compute(x, weight, bias, target, ctx.options, wants, dloss)
        return *grads, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: torch.Tensor | None = None,
                         *, ignore_index: int = -100, reduction: str = "mean",
                         label_smoothing: float = 0.0) -> torch.Tensor:
    """The cross entropy of ``x weight^T + bias`` against ``target``, in float32, differentiable once
    (backwards; a forward-mode tangent is refused).

    ``x`` is ``[..., inner]``, ``weight`` ``[vocabulary, inner]`` and ``bias`` ``[vocabulary]``, of one
    dtype: bfloat16, float16 or float32; ``target`` holds whole numbers and has ``x``'s leading
    shape.  ``ignore_index``, ``reduction`` (``"mean"`` over the tokens that are not ignored,
    ``"sum"``, ``"none"``) and ``label_smoothing`` are ``torch.nn.functional.cross_entropy``'s.  An
    ignored token has no part in anything, whatever its row of ``x`` holds, and costs nothing but
    its look at the target; a mean over none is NaN, with zero gradients.  A target out of range makes its
    loss and the gradients NaN, and so does a row whose logits are all -inf.  Any strides are accepted, as by :func:`fused_linear`.

    With gradients wanted, a summed or averaged loss computes them here (see the module), so call
    it under ``torch.no_grad()`` to evaluate.  Before a step is recorded (:class:`StepGraph`), let go of the
    losses of eager steps over the same tensors, or keep ``loss.detach()``: recording beside them is refused.
    """
    _check(x, weight, target, bias, reduction, label_smoothing)
    if _holds_tangent(x, weight, bias):
        raise UnsupportedFeatureError(
            format_error(_WHO, "forward-mode derivatives have no kernel",
                         resolution="differentiate backwards, or use torch.nn.functional.cross_entropy inside a dual level"))
    options = (int(ignore_index), reduction, float(label_smoothing))
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _LinearCrossEntropy.apply(x, weight, bias, target, options)
    return _compute(x, weight, bias, target, options, (False, False, False))[0]


class LinearCrossEntropy(nn.Module):
    """An output head and its loss: ``torch.nn.Linear``'s parameters over a vocabulary, and
    :func:`linear_cross_entropy` of what they would give.  To share an embedding's weight,
    assign it: ``head.weight = embedding.weight``."""

    def __init__(self, in_features: int, vocabulary: int, bias: bool = False, *, ignore_index: int = -100,
                 reduction: str = "mean", label_smoothing: float = 0.0, device: torch.device | str | None = None,
                 dtype: torch.dtype | None = None) -> None:
        super().__init__()
        if reduction not in REDUCTIONS:
            raise UnsupportedFeatureError(format_error("cross_entropy.LinearCrossEntropy", "unknown reduction",
                                                       expected=sorted(REDUCTIONS), observed=reduction))
        self.in_features, self.vocabulary = in_features, vocabulary
        self.ignore_index, self.reduction, self.label_smoothing = ignore_index, reduction, label_smoothing
        self.weight = nn.Parameter(torch.empty(vocabulary, in_features, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.empty(vocabulary, device=device, dtype=dtype)) if bias else None
        self.reset_parameters()

    def reset_parameters(self) -> None:
        """Uniform in +-1/sqrt(in_features), weight and bias."""
        bound = 1 / math.sqrt(self.in_features) if self.in_features > 0 else 0.0
        with torch.no_grad():
            self.weight.uniform_(-bound, bound)
            if self.bias is not None:
                self.bias.uniform_(-bound, bound)

    def forward(self, x: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
        return linear_cross_entropy(x, self.weight, target, self.bias, ignore_index=self.ignore_index,
                                    reduction=self.reduction, label_smoothing=self.label_smoothing)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, vocabulary={self.vocabulary}, bias={self.bias is not None}, "
                f"ignore_index={self.ignore_index}, reduction={self.reduction!r}, "
                f"label_smoothing={self.label_smoothing}")
