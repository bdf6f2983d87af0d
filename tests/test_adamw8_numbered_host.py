"""What the numbered 8-bit step refuses before any launch, and the scalars it is given, without a device."""

from __future__ import annotations

import ctypes
import math

from hybrid_training_amd import _native
from hybrid_training_amd.optim import _adamw8_scalars, _adamw_scalars


def test_bad_calls_are_refused():
    lib = _native.library()
    scalars = (1.0, None, 1.0, 0.1, 0.9, 0.1, 1.0, 1e-8, -1e-3, 17, None, 0, None)
    none = (None,) * 5
    step = lib.hbt_adamw8_step_numbered
    assert step(*none, 0, 0, 0, *scalars) == 0 and lib.hbt_last_error() == b""
    for call in ((*none, 81, 0, 0, *scalars), (*none, 1, 0, 0, *scalars), (*none, 0, 0, 2, *scalars),
                 (*none, 0, 0, 0, *scalars[:-2], 1, None), (*none, 0, 0, 0, *scalars[:-3], ctypes.c_void_p(4098), 0, None)):
        assert step(*call) == -1
        assert lib.hbt_last_error().startswith(b"hbt_adamw8_step_numbered: ")
    step(*none, 0, 0, 0, *scalars)  # leaves no message behind


def test_the_step_is_a_whole_number_of_32_bits():
    group = {"lr": 1e-3, "betas": (0.9, 0.999), "weight_decay": 0.0, "eps": 1e-8}
    for step, number in ((1.0, 1), (17.0, 17), (2.0**24, 1 << 24), (1e12, (1 << 32) - 1), (math.inf, (1 << 32) - 1)):
        scalars = _adamw8_scalars(group, step)
        assert scalars[-1] == number and isinstance(scalars[-1], int)
        assert scalars[:4] == _adamw_scalars(group, step)[:4]
