"""The linear layer with its bias, activation and residual in the product's epilogue.

:func:`fused_linear` computes ``act(x W^T + bias) + residual`` in one kernel (``hbt_linear``),
and its backward pass ``dz = dy act'(z)``, ``dx = dz W``, ``dW = dz^T x`` and the bias gradient in
one call (``hbt_linear_backward``).  :class:`FusedLinear` is the module
around it, with ``torch.nn.Linear``'s parameters and initialisation.

Sums are held in float32; every stored value is rounded once to the tensors' dtype.  With an
activation the backward pass keeps ``z = x W^T + bias`` in that dtype and forms ``act'`` from
it; a ReLU without a residual keeps its result, which has the same sign, in its place.  No atomics run, so equal inputs give equal bits.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native
from .errors import ShardingError, UnsupportedFeatureError, format_error

__all__ = ["ACTIVATIONS", "FusedLinear", "fused_linear"]

#: Activation names and their HBT_ACT_* codes.  ``gelu`` is the exact (erf) form, ``gelu_tanh``
#: the tanh approximation GPT-2 trains with.
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
#: Elements between rows that the kernels address (hbt_linear's limit).
_MAX_LD = 1 << 20
_DX, _DW, _DBIAS = 1, 2, 4


def _rows(t: torch.Tensor, cols: int) -> tuple[torch.Tensor, int]:
    """``t`` as rows of ``cols`` consecutive elements and the distance between them: a view
    where its strides allow one, else a dense copy."""
    if t.dim() != 2:
        t = t.reshape(-1, cols) if cols else t.reshape(math.prod(t.shape[:-1]), 0)
    rows = t.shape[0]
    if cols <= 1 or t.stride(1) == 1:
        if rows <= 1:
            return t, max(cols, 1)
        ld = t.stride(0)
        if max(cols, 1) <= ld <= _MAX_LD:
            return t, ld
    t = t.contiguous()
    return t, max(cols, 1)


def _workspace(nbytes: int, device: torch.device) -> tuple[torch.Tensor | None, int]:
    """(tensor to keep, address) of working storage, or nothing where none is needed."""
    if nbytes <= 0:
        return None, 0
    space = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return space, space.data_ptr()


def _check(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, residual: torch.Tensor | None,
           activation: str) -> None:
    dtype, device = x.dtype, x.device
    if (activation in ACTIVATIONS and dtype in _DTYPES and x.is_cuda and weight.dim() == 2 and x.dim() > 0
            and x.shape[-1] == weight.shape[1] and weight.dtype == dtype and weight.device == device
            and (bias is None or (bias.shape == weight.shape[:1] and bias.dtype == dtype and bias.device == device))
            and (residual is None or (residual.shape == x.shape[:-1] + weight.shape[:1] and residual.dtype == dtype
                                      and residual.device == device))):
        return
    _refuse(x, weight, bias, residual, activation)


def _refuse(x, weight, bias, residual, activation) -> None:
    """Name what :func:`_check` found wrong."""
    who = "linear.fused_linear"
    if activation not in ACTIVATIONS:
        raise UnsupportedFeatureError(format_error(who, "unknown activation", expected=sorted(ACTIVATIONS),
                                                   observed=activation))
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ShardingError(
            format_error(who, "x must end in the weight's inner size",
                         expected="x [..., inner] and weight [outer, inner]",
                         observed=f"x {tuple(x.shape)}, weight {tuple(weight.shape)}"))
    outer = weight.shape[0]
    if bias is not None and tuple(bias.shape) != (outer,):
        raise ShardingError(format_error(who, "the bias must hold one value per output", expected=(outer,),
                                         observed=tuple(bias.shape)))
    if residual is not None and residual.shape != (*x.shape[:-1], outer):
        raise ShardingError(format_error(who, "the residual must have the result's shape",
                                         expected=(*x.shape[:-1], outer), observed=tuple(residual.shape)))
    given = [t for t in (x, weight, bias, residual) if t is not None]
    for t in given:
        _native.require_device_tensor(t, who)
    if x.dtype not in _DTYPES or any(t.dtype != x.dtype for t in given):
        raise UnsupportedFeatureError(
            format_error(who, "x, weight, bias and residual share one dtype of bfloat16, float16 or float32",
                         observed=[str(t.dtype) for t in given]))
    raise ShardingError(format_error(who, "x, weight, bias and residual must be on one device",
                                     expected=str(x.device), observed=[str(t.device) for t in given]))


def _forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, residual: torch.Tensor | None,
             activation: str, keep: bool) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The result and, with ``keep``, z."""
    outer, inner = weight.shape
    shape = (*x.shape[:-1], outer)
    rows, ldx = _rows(x, inner)
    tokens = rows.shape[0]
    w, ldw = _rows(weight, inner)
    y = x.new_empty(shape)
    z = x.new_empty((tokens, outer)) if keep else None
    if tokens == 0 or outer == 0:
        return y, z
    b = None if bias is None else bias.contiguous()
    r, ldr = (None, 0) if residual is None else _rows(residual, outer)
    code = _native.dtype_code(x.dtype)
    device = x.device
    with _native.device_guard(device):
        lib = _native.library()
        nbytes = lib.hbt_linear_workspace(tokens, inner, outer, code) if tokens > 16 else 0
        space, address = _workspace(nbytes, device)
        status = lib.hbt_linear(
            rows.data_ptr(), ldx, w.data_ptr(), ldw, None if b is None else b.data_ptr(),
            None if r is None else r.data_ptr(), ldr, y.data_ptr(), outer, None if z is None else z.data_ptr(), outer,
            tokens, inner, outer, code, ACTIVATIONS[activation], address, nbytes, _native.stream_of(device))
    if status:
        _native.check(status, "linear.hbt_linear")
    return y, z


def _holds_tangent(*given: torch.Tensor | None) -> bool:
    """Whether a tensor is dual: part of a forward-mode derivative."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # no level is open
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in given)


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        from_result = activation == "relu" and residual is None
        y, z = _forward(x, weight, bias, residual, activation, keep=activation != "none" and not from_result)
        ctx.activation = activation
        ctx.save_for_backward(x, weight, y if from_result else z)
        return y

    # The backward pass runs on autograd's own thread, where host code is slower: it does as
    # little as it can before its one call.
    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        if not (want_x or want_w or want_b):
            return None, None, None, dy if want_r else None, None
        x, weight, z = ctx.saved_tensors
        outer, inner = weight.shape
        device, dtype, across = x.device, x.dtype, max(inner, 1)
        g, ldg = _rows(dy, outer)
        tokens = g.shape[0]
        wants, ldx, ldw = 0, 0, 0
        xs = ws = dx = dw = db = x_at = w_at = dx_at = dw_at = db_at = None
        if want_x:
            wants = _DX
            ws, ldw = _rows(weight, inner)
            dx = x.new_empty(x.shape)
            w_at, dx_at = ws.data_ptr(), dx.data_ptr()
        if want_w:
            wants |= _DW
            xs, ldx = _rows(x, inner)
            dw = weight.new_empty(weight.shape)
            x_at, dw_at = xs.data_ptr(), dw.data_ptr()
        if want_b:
            wants |= _DBIAS
            db = weight.new_empty(outer)
            db_at = db.data_ptr()
        code, activation = _native.dtype_code(dtype), ACTIVATIONS[ctx.activation]
        lib = _native.library()
        with _native.device_guard(device):
            nbytes = lib.hbt_linear_backward_workspace(tokens, inner, outer, code, activation, wants)
            space, address = _workspace(nbytes, device)
            status = lib.hbt_linear_backward(
                g.data_ptr(), ldg, x_at, ldx, w_at, ldw, None if z is None else z.data_ptr(), max(outer, 1), dx_at, across,
                dw_at, across, db_at, tokens, inner, outer, code, activation, address, nbytes, _native.stream_of(device))
        if status:
            _native.check(status, "linear.hbt_linear_backward")
        return dx, dw, db, dy if want_r else None, None


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                 activation: str = "none", residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x weight^T + bias) + residual`` in one kernel, differentiable once (backwards; a
    forward-mode tangent is refused).

    ``x`` is ``[..., inner]``, ``weight`` ``[outer, inner]``, ``bias`` ``[outer]`` and
    ``residual`` ``[..., outer]``, all of one dtype: bfloat16, float16 or float32.  Any strides
    are accepted; rows of consecutive elements up to 2**20 apart are read where they lie, other
    layouts through a dense copy.  ``activation`` is one of :data:`ACTIVATIONS`.
    """
    _check(x, weight, bias, residual, activation)
    if _holds_tangent(x, weight, bias, residual):
        raise UnsupportedFeatureError(
            format_error("linear.fused_linear", "forward-mode derivatives have no kernel",
                         resolution="differentiate backwards, or use torch.nn.functional.linear inside a dual level"))
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _FusedLinear.apply(x, weight, bias, residual, activation)
    return _forward(x, weight, bias, residual, activation, keep=False)[0]


class FusedLinear(nn.Module):
    """``torch.nn.Linear`` with an activation, and a residual given to :meth:`forward`, in its
    product's epilogue.  Parameters, their names and their initialisation are
    ``torch.nn.Linear``'s."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, *, activation: str = "none",
                 device: torch.device | str | None = None, dtype: torch.dtype | None = None) -> None:
        super().__init__()
        if activation not in ACTIVATIONS:
            raise UnsupportedFeatureError(format_error("linear.FusedLinear", "unknown activation",
                                                       expected=sorted(ACTIVATIONS), observed=activation))
        self.in_features, self.out_features, self.activation = in_features, out_features, activation
        self.weight = nn.Parameter(torch.empty(out_features, in_features, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.empty(out_features, device=device, dtype=dtype)) if bias else None
        self.reset_parameters()

    def reset_parameters(self) -> None:
        """Uniform in +-1/sqrt(in_features), weight and bias."""
        bound = 1 / math.sqrt(self.in_features) if self.in_features > 0 else 0.0
        with torch.no_grad():
            self.weight.uniform_(-bound, bound)
            if self.bias is not None:
                self.bias.uniform_(-bound, bound)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        return fused_linear(x, self.weight, self.bias, activation=self.activation, residual=residual)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, activation={self.activation!r}")
