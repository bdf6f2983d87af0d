"""AdamW's moments held in 8 bits: the state tensors of one parameter and the calls that read
and write them (``hbt_adamw8_step``, ``hbt_moments8_encode``, ``hbt_moments8_decode``).

``ShardedOptimizer`` holds its state this way with ``OptimizerConfig(state_format="8bit")``.  Every
256 consecutive elements share two float32 scales, the largest first moment and the largest root of a second
moment among them; beside these an element takes one byte for its first moment (e4m3, 4
significant bits) and one for the root of its second (5 significant bits): 2.03 bytes of state an
element instead of 8.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from . import _native
from .errors import ShardingError, UnsupportedFeatureError, format_error

__all__ = ["BLOCK", "STATE_KEYS", "check_state", "decode", "encode", "zero_state"]

#: Consecutive elements that share their scales.
BLOCK = 256
#: A parameter's state: codes and scales of the first moment and of the second one's root.
STATE_KEYS = ("exp_avg_codes", "exp_avg_sq_codes", "exp_avg_scales", "exp_avg_sq_scales")


def _blocks(numel: int) -> int:
    return (numel + BLOCK - 1) // BLOCK


def zero_state(p: torch.Tensor) -> dict[str, torch.Tensor]:
    """Zero moments beside ``p``."""
    blocks = _blocks(p.numel())
    codes = torch.zeros(2, blocks * BLOCK, dtype=torch.uint8, device=p.device)
    scales = torch.zeros(2, blocks, dtype=torch.float32, device=p.device)
    return dict(zip(STATE_KEYS, (codes[0], codes[1], scales[0], scales[1])))


def check_state(p: torch.Tensor, state: dict, operation: str) -> None:
    """Refuse codes or scales that are not the ones :func:`zero_state` lays out."""
    blocks = _blocks(p.numel())
    for key, count, dtype in zip(STATE_KEYS, (blocks * BLOCK, blocks * BLOCK, blocks, blocks),
                                 (torch.uint8, torch.uint8, torch.float32, torch.float32)):
        value = state.get(key)
        if (value is None or value.dtype != dtype or value.numel() != count or value.device != p.device
                or not value.is_contiguous() or (count and value.data_ptr() % 4)):
            raise ShardingError(
                format_error(operation, f"the state {key!r} must lie dense beside its parameter",
                             expected=f"{count} of {dtype} on {p.device}",
                             observed=None if value is None else f"{value.numel()} of {value.dtype} on {value.device}",
                             resolution="set moments through load_state_dict, which encodes them"))


def tables(states: Sequence[dict]) -> tuple:
    """The four pointer tables of a call over ``states``."""
    return tuple(_native.pointer_array([s[key].data_ptr() for s in states]) for key in STATE_KEYS)


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


def decode(params: Sequence[torch.Tensor], states: Sequence[dict], device: torch.device,
           dtype: torch.dtype = torch.float32) -> list[tuple[torch.Tensor, torch.Tensor]]:
    """The (first, second) moments that ``states`` stand for, shaped like ``params``."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise UnsupportedFeatureError(format_error("optim.moments", "moments are decoded to float32 or bfloat16",
                                                   observed=str(dtype)))
    lib = _native.library()
    out = [(torch.empty(p.shape, dtype=dtype, device=p.device), torch.empty(p.shape, dtype=dtype, device=p.device))
           for p in params]
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
