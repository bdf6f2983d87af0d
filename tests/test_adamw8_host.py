"""What 8-bit moments refuse before anything touches a device, and the codes' arithmetic on the host."""

from __future__ import annotations

import ctypes

import pytest
import torch

from hybrid_training_amd import OptimizerConfig, _native, moments8
from hybrid_training_amd.errors import ConfigurationError


def test_configuration():
    assert OptimizerConfig().state_format == "master"
    assert OptimizerConfig(state_format="8bit").state_format == "8bit"
    with pytest.raises(ConfigurationError, match="state format"):
        OptimizerConfig(state_format="4bit")
    with pytest.raises(ConfigurationError, match="AdamW"):
        OptimizerConfig(name="sgd", state_format="8bit")
    with pytest.raises(ConfigurationError, match="device memory"):
        OptimizerConfig(cpu_offload_state=True, state_format="8bit")


@pytest.mark.parametrize("numel", [0, 1, 256, 257])
def test_state_is_laid_out_in_whole_blocks(numel):
    state = moments8.zero_state(torch.empty(numel))
    blocks = -(-numel // 256)
    assert tuple(state) == moments8.STATE_KEYS
    assert [state[k].numel() for k in moments8.STATE_KEYS] == [blocks * 512, blocks * 2]
    assert all(state[k].data_ptr() % 8 == 0 for k in moments8.STATE_KEYS if numel)


def test_the_library_refuses_bad_tables_before_any_launch():
    lib = _native.library()
    scalars = (1.0, None, 1.0, 0.1, 0.9, 0.1, 1.0, 1e-8, -1e-3, None, 0, None)
    none = (None,) * 5
    assert lib.hbt_adamw8_step(*none, 81, 0, 0, *scalars) == -1
    assert b"hbt_adamw8_step: count" in lib.hbt_last_error()
    assert lib.hbt_adamw8_step(*none, 1, 0, 0, *scalars) == -1
    assert lib.hbt_adamw8_step(*none, 0, 0, 2, *scalars) == -1
    assert b"dtypes (0, 2)" in lib.hbt_last_error()
    assert lib.hbt_adamw8_step(*none, 0, 3, 3, *scalars) == -1
    assert lib.hbt_adamw8_step(*none, 0, 0, 0, *scalars[:-2], 1, None) == -1
    assert lib.hbt_adamw8_step(*none, 0, 0, 0, *scalars[:-3], ctypes.c_void_p(4098), 0, None) == -1
    assert lib.hbt_adamw8_step(*none, 0, 0, 0, *scalars) == 0
    one, odd, n = _native.pointer_array([4096]), _native.pointer_array([4100]), _native.int64_array([1])
    assert lib.hbt_adamw8_step(one, one, odd, one, n, 1, 0, 0, *scalars) == -1
    assert b"off 8 bytes" in lib.hbt_last_error()
    assert lib.hbt_adamw8_step(one, one, one, one, _native.int64_array([-1]), 1, 0, 0, *scalars) == -1
    zero = _native.pointer_array([0])
    assert lib.hbt_adamw8_step(zero, one, one, one, n, 1, 0, 0, *scalars) == -1
    assert lib.hbt_moments8_encode(*none, 81, None) == -1
    assert lib.hbt_moments8_decode(*none, 0, 2, None) == -1
    assert b"out_dtype 2" in lib.hbt_last_error()
    assert lib.hbt_moments8_decode(*none, 0, 1, None) == 0
