"""AdamW's moments held in 8 bits: the state tensors of one parameter and the calls that read
and write them (``hbt_adamw8_step_numbered``, ``hbt_moments8_encode``, ``hbt_moments8_decode``).

``ShardedOptimizer`` holds its state this way with ``OptimizerConfig(state_format="8bit")``.  Every
256 consecutive elements share two float32 scales, the largest first moment and the largest root of a second
moment among them; beside these an element takes one byte for its first moment (e4m3, 4
significant bits) and one for the root of its second (5 significant bits): 2.03 bytes of state an
element instead of 8.

A code is rounded to nearest where a step moves it by more than rounding can lose; elsewhere, as for
the roots at the default beta2 of 0.999, without bias, by random numbers that follow from the step and the
element's place: a root is then off by up to an eighth of itself, as often up as down, and equal runs
stay equal bit by bit.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from . import _native
from .errors import ShardingError, UnsupportedFeatureError, format_error

__all__ = ["BLOCK", "STATE_KEYS", "check_state", "decode", "encode", "zero_state"]

#: Consecutive elements that share their scales.
BLOCK = 256
#: A parameter's state: codes, [blocks][groups of four][first moments and roots][four], and scales,
#: [blocks][first moments and roots].
STATE_KEYS = ("moment_codes", "moment_scales")
_CODES, _SCALES = STATE_KEYS


def _blocks(numel: int) -> int:
    return (numel + BLOCK - 1) // BLOCK


def zero_state(p: torch.Tensor) -> dict[str, torch.Tensor]:
    """Zero moments beside ``p``."""
    blocks = _blocks(p.numel())
    return {_CODES: torch.zeros(blocks, 2 * BLOCK, dtype=torch.uint8, device=p.device),
            _SCALES: torch.zeros(blocks, 2, dtype=torch.float32, device=p.device)}


def check_state(p: torch.Tensor, state: dict, operation: str) -> None:
    """Refuse codes or scales that are not the ones :func:`zero_state` lays out."""
    blocks = (p.numel() + 255) >> 8
    codes, scales = state.get(_CODES), state.get(_SCALES)
    if (codes is not None and scales is not None and codes.dtype is torch.uint8 and scales.dtype is torch.float32
            and codes.numel() == blocks << 9 and scales.numel() == blocks << 1 and codes.is_contiguous()
            and scales.is_contiguous() and codes.is_cuda and scales.is_cuda
            and codes.get_device() == scales.get_device() == p.get_device()
            and not (codes.data_ptr() | scales.data_ptr()) & 7):
        return
    for key, value, count, dtype in ((_CODES, codes, blocks << 9, torch.uint8), (_SCALES, scales, blocks << 1, torch.float32)):
        if (value is None or value.dtype != dtype or value.numel() != count or value.device != p.device
                or not value.is_contiguous() or value.data_ptr() % 8):
            raise ShardingError(
                format_error(operation, f"the state {key!r} must lie dense beside its parameter",
                             expected=f"{count} of {dtype} on {p.device}",
                             observed=None if value is None else f"{value.numel()} of {value.dtype} on {value.device}",
                             resolution="set moments through load_state_dict, which encodes them"))


def tables(states: Sequence[dict]) -> tuple:
    """The pointer tables of a call over ``states``."""
    return (_native.pointer_array([s[_CODES].data_ptr() for s in states]),
            _native.pointer_array([s[_SCALES].data_ptr() for s in states]))


def _chunks(items: Sequence) -> list:
    return [items[i : i + _native.MAX_ADAMW8_TENSORS] for i in range(0, len(items), _native.MAX_ADAMW8_TENSORS)]


def encode(pairs: Sequence[tuple[torch.Tensor, torch.Tensor]], states: Sequence[dict], device: torch.device) -> None:
    """Hold (first, second) moments, dense float32 device tensors, in ``states``."""
    lib = _native.library()
    with _native.device_guard(device):
        stream = _native.stream_of(device)
        for chunk in _chunks(list(zip(pairs, states))):
            held = [s for _, s in chunk]
            _native.check(lib.hbt_moments8_encode(
                _native.pointer_array([m.data_ptr() for (m, _), _ in chunk]),
                _native.pointer_array([v.data_ptr() for (_, v), _ in chunk]), *tables(held),
                _native.int64_array([m.numel() for (m, _), _ in chunk]), len(chunk), stream),
                "optim.hbt_moments8_encode")


#: Smaller results share one allocation: a tensor costs more to allocate than to decode.
_SHARED_MAX = 1 << 18


def _results(params: Sequence[torch.Tensor], dtype: torch.dtype, device: torch.device) -> list:
    """Uninitialised (first, second) tensors shaped like ``params``."""
    small = [i for i, p in enumerate(params) if p.numel() <= _SHARED_MAX]
    out: list = [None] * len(params)
    if len(small) > 1:
        sizes = []
        for i in small:
            n = params[i].numel()
            sizes += (n, -n % 64, n, -n % 64)  # each starts on a 128-byte line
        parts = torch.empty(sum(sizes), dtype=dtype, device=device).split(sizes)
        for k, i in enumerate(small):
            m, v, shape = parts[4 * k], parts[4 * k + 2], params[i].shape
            out[i] = (m, v) if len(shape) == 1 else (m.view(shape), v.view(shape))
    for i, p in enumerate(params):
        if out[i] is None:
            out[i] = (torch.empty(p.shape, dtype=dtype, device=device), torch.empty(p.shape, dtype=dtype, device=device))
    return out


def decode(params: Sequence[torch.Tensor], states: Sequence[dict], device: torch.device,
           dtype: torch.dtype = torch.float32) -> list[tuple[torch.Tensor, torch.Tensor]]:
    """The (first, second) moments that ``states`` stand for, shaped like ``params``."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise UnsupportedFeatureError(format_error("optim.moments", "moments are decoded to float32 or bfloat16",
                                                   observed=str(dtype)))
    lib = _native.library()
    out = _results(params, dtype, device)
    with _native.device_guard(device):
        stream = _native.stream_of(device)
        for chunk in _chunks(list(zip(out, states))):
            held = [s for _, s in chunk]
            _native.check(lib.hbt_moments8_decode(
                *tables(held), _native.pointer_array([m.data_ptr() for (m, _), _ in chunk]),
                _native.pointer_array([v.data_ptr() for (_, v), _ in chunk]),
                _native.int64_array([m.numel() for (m, _), _ in chunk]), len(chunk), _native.dtype_code(dtype), stream),
                "optim.hbt_moments8_decode")
    return out
