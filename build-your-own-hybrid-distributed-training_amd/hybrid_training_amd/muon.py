"""Orthogonalised updates of matrix parameters on HIP: :func:`orthogonalize` and
:class:`MuonOptimizer`.

A matrix's update direction ``u`` (its momentum) is replaced by the nearest matrix with
orthonormal rows or columns, up to a few per cent in its singular values, through ``steps``
Newton-Schulz products from ``x = u / |u|``::

    A = x x^T (over the shorter side);  x = a x + (b A + c A A) x

and the parameter moves by ``-lr * scale * x`` after its weight decay.  One call updates up to
32 matrices of any sizes (``hbt_muon_step``): the momentum and the norm in one pass over the
gradients, the products on the matrix cores with every matrix of a phase in one launch, the
parameter written by the last product's epilogue.

Every sum and the momentum are float32, the norm float64.  ``product_dtype`` says what the
products read: ``float16``, whose 11 bits leave the result about 2e-3 off its exact value
(relative, in the Frobenius norm), or ``float32``.  Matrices whose shorter side is at most 128 take
``float32`` products either way.  The iterate takes 32 bits: float32, or beside ``float16``
products their fp16 value and an fp16 remainder (22 bits of mantissa).
"""

from __future__ import annotations

import ctypes
import math
from collections.abc import Callable, Iterable, Sequence

import torch
import torch.nn as nn
from torch.autograd.graph import increment_version

from . import _native
from .config import MuonConfig, OptimizerConfig, check_newton_schulz, resolve_dtype
from .errors import ShardingError, UnsupportedFeatureError, format_error
from .groups import GroupHandle
from .host_staging import is_host
from .optim import (
    NormResult,
    ShardedOptimizer,
    _check_recorded_grad,
    _mul_ptr,
    _pending_unscale,
    _RecordedOperands,
    _replay_error,
    _replay_groups,
    _unrecordable,
    _write_back_flag,
    scale_gradients,
)

__all__ = ["MuonOptimizer", "orthogonalize"]

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
#: Working storage one call may ask for before a list of matrices is split (a single matrix may
#: need more): 32 matrices of a few thousand squared fit.
_WORKSPACE_CAP = 4 << 30
#: Sides the kernels address, and the elements of one call (hbt_orthogonalize's limits).
_MAX_SIDE, _MAX_ELEMENTS = 1 << 20, 1 << 34


def _call_groups(shapes: Sequence[tuple[int, int]], product: int) -> list[tuple[list[int], int]]:
    """(indices, workspace bytes) of the calls a list of matrices is split into, in order: at
    most ``MAX_MATRICES`` matrices, ``_MAX_ELEMENTS`` elements and ``_WORKSPACE_CAP`` bytes each."""
    lib = _native.library()

    def need(indices: list[int]) -> int:
        nbytes = lib.hbt_orthogonal_workspace(_native.int64_array([shapes[i][0] for i in indices]),
                                              _native.int64_array([shapes[i][1] for i in indices]), len(indices),
                                              product)
        if nbytes < 0:
            _native.check(int(nbytes), "muon.hbt_orthogonal_workspace")
        return nbytes

    groups: list[tuple[list[int], int]] = []
    for first in range(0, len(shapes), _native.MAX_MATRICES):
        indices = list(range(first, min(first + _native.MAX_MATRICES, len(shapes))))
        elements = [shapes[i][0] * shapes[i][1] for i in indices]
        if sum(elements) <= _MAX_ELEMENTS and (nbytes := need(indices)) <= _WORKSPACE_CAP:
            groups.append((indices, nbytes))
            continue
        part: list[int] = []
        taken = held = 0
        for i, count in zip(indices, elements):
            size = need([i])  # whole 256-byte units: a call's need is their sum
            if part and (taken + size > _WORKSPACE_CAP or held + count > _MAX_ELEMENTS):
                groups.append((part, taken))
                part, taken, held = [], 0, 0
            part.append(i)
            taken += size
            held += count
        groups.append((part, taken))
    return groups


def _product_code(product_dtype: torch.dtype | str | None, result: torch.dtype) -> int:
    if product_dtype is None:
        product_dtype = torch.float32 if result == torch.float32 else torch.float16
    product = resolve_dtype(product_dtype)
    if product not in (torch.float16, torch.float32):
        raise UnsupportedFeatureError(
            format_error("muon.orthogonalize", "the products read float16 or float32", observed=str(product)))
    return _native.dtype_code(product)


def orthogonalize(
    matrices: Sequence[torch.Tensor],
    *,
    steps: int = 5,
    coefficients: tuple[float, float, float] = (3.4445, -4.7750, 2.0315),
    eps: float = 1e-12,
    dtype: torch.dtype | None = None,
    product_dtype: torch.dtype | str | None = None,
) -> list[torch.Tensor]:
    """The Newton-Schulz form of every matrix, ``steps`` products from ``x = u / max(|u|, eps)``.

    ``matrices`` are 2-D device tensors of any sizes, float32, bfloat16 or float16, of one
    dtype; the results have their shapes, in ``dtype`` (default: theirs).  ``product_dtype``
    (default: float32 for float32 results, else float16) is what the matrix cores read; sums
    are float32 either way.  A zero matrix gives zeros; one holding a
    non-finite value comes out non-finite.  Layouts other than dense rows go through a copy.  Not
    differentiable.
    """
    who = "muon.orthogonalize"
    matrices = list(matrices)
    check_newton_schulz("orthogonalize", steps, coefficients, eps)
    if not matrices:
        return []
    kind, device = matrices[0].dtype, matrices[0].device
    for m in matrices:
        if not m.is_cuda:
            _native.require_device_tensor(m, who)
        if m.dim() != 2:
            raise ShardingError(format_error(who, "every tensor must be a matrix", expected="2 dimensions",
                                             observed=tuple(m.shape)))
        if m.dtype != kind or kind not in _DTYPES:
            raise UnsupportedFeatureError(
                format_error(who, "the matrices share one dtype of float32, bfloat16 or float16",
                             observed=sorted({str(v.dtype) for v in matrices})))
        if m.device != device:
            raise ShardingError(format_error(who, "the matrices must be on one device", expected=str(device),
                                             observed=str(m.device)))
    result = kind if dtype is None else resolve_dtype(dtype)
    if result not in _DTYPES:
        raise UnsupportedFeatureError(format_error(who, "results are float32, bfloat16 or float16",
                                                   observed=str(result)))
    product = _product_code(product_dtype, result)
    sources = [m.detach().contiguous() for m in matrices]
    outputs = [torch.empty(m.shape, dtype=result, device=device) for m in sources]
    lib = _native.library()
    with _native.device_guard(device):
        stream = _native.stream_of(device)
        for indices, nbytes in _call_groups([tuple(m.shape) for m in sources], product):
            space = torch.empty(nbytes, dtype=torch.uint8, device=device)
            _native.check(lib.hbt_orthogonalize(
                _native.pointer_array([sources[i].data_ptr() for i in indices]),
                _native.pointer_array([outputs[i].data_ptr() for i in indices]),
                _native.int64_array([sources[i].shape[0] for i in indices]),
                _native.int64_array([sources[i].shape[1] for i in indices]), len(indices), _native.dtype_code(kind),
                _native.dtype_code(result), product, int(steps), *map(float, coefficients), float(eps),
                space.data_ptr(), nbytes, stream), "muon.hbt_orthogonalize")
    return outputs


class _Groups(torch.optim.AdamW):
    """The torch object that owns groups and state; its ``step`` is never called.  AdamW's
    restore hook expects a step count in every state, which a matrix's does not have."""

    def __setstate__(self, state) -> None:
        torch.optim.Optimizer.__setstate__(self, state)


class MuonOptimizer(ShardedOptimizer):
    """Orthogonalised momentum steps for matrices, AdamW for ``others``, with one global-norm clip.

    ``matrices`` are whole 2-D device parameters (float32, bfloat16 or float16): a layer's
    weight under DDP, where every rank holds it.  A flat FSDP shard holds parts of matrices and
    is refused.  Embeddings, biases and norms go into ``others``, which ``others_config`` (an
    AdamW :class:`OptimizerConfig`) steps.  The clip, its placements, the loss scaler, learning
    rates, recording into a ``StepGraph`` and the state dict work as in
    :class:`ShardedOptimizer`; ``inner.param_groups[-1]`` holds the matrices' options
    (``lr``, ``momentum``, ``nesterov``, ``weight_decay``, ``steps``, ``coefficients``,
    ``norm_eps``, ``scale``, ``product_dtype``) and ``inner.state[p]["momentum_buffer"]`` the float32
    momentum.

    A clip or loss-scale factor that the step applies (``clip_in_step``, ``defer_clip``) multiplies
    the gradient in float32 without rounding to the gradient's dtype in between.
    """

    def __init__(
        self,
        matrices: Iterable[nn.Parameter],
        config: MuonConfig,
        *,
        norm_group: GroupHandle,
        device: torch.device,
        others: Iterable[nn.Parameter] = (),
        others_config: OptimizerConfig | None = None,
        recorder=None,
        defer_clip: bool = False,
        clip_in_step: bool = False,
    ) -> None:
        who = "muon.MuonOptimizer"
        chosen = [p for p in matrices if p.requires_grad]
        rest = [p for p in others if p.requires_grad]
        if not chosen:
            raise ShardingError(format_error(who, "no trainable matrices were supplied", observed=0,
                                             resolution="use ShardedOptimizer for parameters that are not matrices"))
        seen: set[int] = set()
        for p in [*chosen, *rest]:
            if id(p) in seen:
                raise ShardingError(format_error(who, "a parameter was supplied twice", observed=tuple(p.shape)))
            seen.add(id(p))
            if is_host(p):
                raise UnsupportedFeatureError(
                    format_error(who, "parameters and their state stay in device memory here", observed=str(p.device),
                                 resolution="step host-resident shards with ShardedOptimizer"))
        for p in chosen:
            if p.dim() != 2:
                raise ShardingError(
                    format_error(who, "an orthogonalised step needs whole matrices", expected="2 dimensions",
                                 observed=tuple(p.shape),
                                 resolution="pass flat shards, vectors and convolutions as others"))
            if p.dtype not in _DTYPES:
                raise UnsupportedFeatureError(
                    format_error(who, "matrices must be float32, bfloat16 or float16", observed=str(p.dtype)))
            if max(p.shape) > _MAX_SIDE:
                raise UnsupportedFeatureError(
                    format_error(who, "a matrix's sides are limited", expected=f"at most {_MAX_SIDE}",
                                 observed=tuple(p.shape)))
        if others_config is None:
            others_config = OptimizerConfig(learning_rate=config.learning_rate, weight_decay=config.weight_decay)
        if others_config.name != "adamw" or others_config.cpu_offload_state:
            raise UnsupportedFeatureError(
                format_error(who, "the other parameters are stepped by AdamW with its state on the device",
                             observed=others_config))
        super().__init__([*rest, *chosen], others_config, norm_group=norm_group, device=device, recorder=recorder,
                         defer_clip=defer_clip, clip_in_step=clip_in_step)
        self._muon_config = config
        self._due: list[_Batch] = []
        self._space: torch.Tensor | None = None
        self._recording: _native.GraphRecording | None = None
        self._matrices = {id(p) for p in chosen}
        options = dict(lr=config.learning_rate, weight_decay=config.weight_decay, momentum=config.momentum,
                       nesterov=config.nesterov, steps=config.steps, coefficients=config.coefficients,
                       norm_eps=config.eps, scale=config.scale, product_dtype=config.product_dtype)
        # The object that owns groups and state: AdamW's group of the others, if any, then the matrices'.
        defaults = {k: v for k, v in self._optimizer.param_groups[0].items() if k != "params"}
        groups = [{**defaults, "params": rest}] if rest else []
        self._optimizer = _Groups([*groups, {**defaults, "params": chosen, **options}], lr=config.learning_rate)

    # -- update ----------------------------------------------------------------------
    def _is_matrix(self, p: nn.Parameter) -> bool:
        return id(p) in self._matrices

    def _stepped_parameters(self):
        """The others' share of the step, for the AdamW kernels.

        By then the matrices' share, :attr:`_due`, is planned and its memory is allocated, so that
        whatever it is refused for leaves every parameter, counter and state as it was."""
        self._due = []
        others, batches = [], {}
        recording = self._recording = self._recording_check()
        for item in super()._stepped_parameters():
            if not self._is_matrix(item[1]):
                others.append(item)
                continue
            group, p, grad, state = item
            if torch.float64 in (p.dtype, grad.dtype):
                raise UnsupportedFeatureError(format_error("muon.MuonOptimizer.step", "float64 matrices have no kernel",
                                                           observed=f"parameter {p.dtype}, gradient {grad.dtype}"))
            buffer = state.get("momentum_buffer") if state else None
            if buffer is None:
                if recording is not None:
                    raise _unrecordable("the first step creates the momentum buffer")
            elif (buffer.dtype != torch.float32 or buffer.shape != p.shape or buffer.device != p.device
                  or not buffer.is_contiguous()):
                raise ShardingError(
                    format_error("muon.MuonOptimizer.step", "a momentum buffer must be a dense float32 tensor beside "
                                 "its parameter", expected=f"{tuple(p.shape)} on {p.device}",
                                 observed=f"{buffer.dtype} {tuple(buffer.shape)} on {buffer.device}"))
            check_newton_schulz("MuonOptimizer.step", group["steps"], group["coefficients"], group["norm_eps"])
            unscale = _pending_unscale(grad)
            key = (id(group), p.dtype, grad.dtype, unscale)
            batch = batches.get(key)
            if batch is None:
                batch = batches[key] = _Batch(group, p.dtype, grad.dtype, unscale)
            batch.params.append(p)
            batch.grads.append(grad)
            batch.buffers.append(buffer)
            batch.fresh |= buffer is None
        due = list(batches.values())
        for batch in due:
            batch.plan()
        if due:
            # One call's kernels follow another's on the stream, so all share the largest's storage.
            self._space = torch.empty(max(n for batch in due for _, n in batch.calls), dtype=torch.uint8,
                                      device=self._device)
            for batch in due:
                if batch.fresh:
                    batch.buffers = [self._zero_state(p, "momentum_buffer") if v is None else v
                                     for p, v in zip(batch.params, batch.buffers)]
        self._due = due
        return others

    def _run_adamw_step(self, grad_mul: NormResult | None, write_back: bool) -> None:
        try:
            super()._run_adamw_step(grad_mul, write_back)
            with _native.device_guard(self._device):
                for batch in self._due:
                    self._step_batch(batch, grad_mul)
                    if _write_back_flag(write_back, grad_mul, batch.unscale):
                        # In-place semantics: .grad ends as the reference's multiplies leave it.
                        scale_gradients(batch.grads, batch.gdtype, batch.unscale, _mul_ptr(grad_mul, batch.gdtype),
                                        self._device, "muon.hbt_scale_inplace")
        finally:
            self._due, self._space, self._recording = [], None, None

    def _step_batch(self, batch: "_Batch", grad_mul: NormResult | None) -> None:
        """Matrices of one group and dtype pair, in calls of up to 32."""
        lib = _native.library()
        stream = _native.stream_of(self._device)
        space, recording = self._space, self._recording
        decay, lr, momentum, rest = batch.scalars
        if batch.fresh:
            for p, buffer in zip(batch.params, batch.buffers):
                self._optimizer.state[p]["momentum_buffer"] = buffer
        slot = None
        if recording is not None:
            slot = recording.new_slot()
            recording.steps.append(_RecordedMuon(self, recording.record_address(slot), batch))
        for indices, nbytes in batch.calls:
            params, grads, buffers, scales = batch.of(indices)
            _native.check(lib.hbt_muon_step(
                _native.pointer_array([p.data_ptr() for p in params]),
                _native.pointer_array([g.data_ptr() for g in grads]),
                _native.pointer_array([v.data_ptr() for v in buffers]),
                _native.int64_array([p.shape[0] for p in params]), _native.int64_array([p.shape[1] for p in params]),
                (ctypes.c_float * len(params))(*scales), len(params), _native.dtype_code(batch.pdtype), _native.dtype_code(batch.gdtype), batch.product,
                batch.unscale, _mul_ptr(grad_mul, batch.gdtype), momentum, rest, *batch.options, decay, lr,
                None if slot is None else slot.data_ptr(), space.data_ptr(), nbytes, stream), "muon.hbt_muon_step")
            increment_version(params + buffers)

    # -- state -----------------------------------------------------------------------
    def _zero_state(self, p: torch.Tensor, key: str) -> torch.Tensor:
        if key == "momentum_buffer":
            return torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return super()._zero_state(p, key)

    def _place_state(self, value: torch.Tensor, reference: torch.Tensor, key: str) -> torch.Tensor:
        if key == "momentum_buffer":  # float32 whatever the parameter's dtype
            return torch.empty(reference.shape, dtype=torch.float32, device=reference.device).copy_(
                value.detach().reshape(reference.shape))
        return super()._place_state(value, reference, key)

    def load_state_dict(self, payload) -> None:
        super().load_state_dict(payload)
        # torch's optimizer casts loaded state to its parameter's dtype; the momentum is float32.
        for index, entry in payload["state"].items():
            if "momentum_buffer" in entry:
                p = self._parameters[int(index)]
                self._optimizer.state[p]["momentum_buffer"] = self._place_state(entry["momentum_buffer"], p,
                                                                                "momentum_buffer")

    def __repr__(self) -> str:
        return (f"MuonOptimizer(matrices={len(self._matrices)}, "
                f"others={len(self._parameters) - len(self._matrices)}, norm_group={self._norm_group.name!r})")


def _step_scalars(group: dict) -> tuple[float, float, float, float]:
    """decay, learning rate, momentum and 1 - momentum of a step, as Python doubles."""
    lr, momentum = float(group["lr"]), float(group["momentum"])
    return 1.0 - lr * float(group["weight_decay"]), lr, momentum, 1.0 - momentum


def _update_scale(rule: str, shape: Sequence[int]) -> float:
    """What multiplies the learning rate for a matrix of ``shape`` (see :class:`MuonConfig`)."""
    rows, cols = (max(int(s), 1) for s in shape)
    if rule == "rms":
        return 0.2 * math.sqrt(max(rows, cols))
    if rule == "spectral":
        return math.sqrt(max(1.0, rows / cols))
    raise UnsupportedFeatureError(format_error("muon.MuonOptimizer.step", "unknown update scale",
                                               expected=["rms", "spectral"], observed=rule))


class _Batch:
    """The matrices of one group and dtype pair that a step moves, and the calls that do."""

    def __init__(self, group: dict, pdtype: torch.dtype, gdtype: torch.dtype, unscale: float) -> None:
        self.group, self.pdtype, self.gdtype, self.unscale = group, pdtype, gdtype, unscale
        self.params: list[nn.Parameter] = []
        self.grads: list[torch.Tensor] = []
        self.buffers: list[torch.Tensor | None] = []
        self.fresh = False  # some buffers are not in the optimizer's state yet

    def plan(self) -> None:
        """Everything the calls are formed from that can be refused."""
        group = self.group
        self.scalars = _step_scalars(group)
        self.options = (int(bool(group["nesterov"])), int(group["steps"]), *map(float, group["coefficients"]),
                        float(group["norm_eps"]))
        self.product = _product_code(group["product_dtype"], self.pdtype)
        self.scales = [_update_scale(group["scale"], p.shape) for p in self.params]
        self.calls = _call_groups([p.shape for p in self.params], self.product)

    def of(self, indices: list[int]) -> tuple[list, list, list, list]:
        """Parameters, gradients, momenta and scales of one call."""
        lists = (self.params, self.grads, self.buffers, self.scales)
        return lists if len(self.calls) == 1 else tuple([values[i] for i in indices] for values in lists)


class _RecordedMuon:
    """The matrices' share of a step recorded into a graph, whose kernels read decay, learning
    rate and momentum from a slot that each replay rewrites."""

    def __init__(self, optimizer: MuonOptimizer, record: int, batch: _Batch) -> None:
        self._optimizer = optimizer
        self._record = record
        self._params = batch.params
        self._grad_ptrs = [g.data_ptr() for g in batch.grads]
        self._operands = _RecordedOperands(optimizer, self._params, ("momentum_buffer",))
        self._fixed = _fixed_options(batch.group)

    @property
    def parameters(self) -> list[nn.Parameter]:
        return self._params

    def prepare(self) -> Callable[[], None]:
        opt = self._optimizer
        groups = _replay_groups(opt, self._params)
        for p, ptr in zip(self._params, self._grad_ptrs):
            _check_recorded_grad(p, ptr)
        self._operands.check([opt._optimizer.state[p] for p in self._params])
        found = {(_step_scalars(groups[id(p)]), _fixed_options(groups[id(p)])) for p in self._params}
        if len(found) != 1:
            raise _replay_error("the matrices recorded in one call no longer share their options")
        scalars, fixed = found.pop()
        if fixed != self._fixed:
            raise _replay_error("steps, coefficients, eps, nesterov, scale or product_dtype changed, which are part "
                                "of the recorded launches")
        ctypes.memmove(self._record, (ctypes.c_float * 4)(*scalars), 16)
        return self._operands.bump_versions


def _fixed_options(group: dict) -> tuple:
    return (bool(group["nesterov"]), int(group["steps"]), tuple(map(float, group["coefficients"])),
            float(group["norm_eps"]), group["scale"], str(group["product_dtype"]))
