"""The matrix operators' host side: refusals before any launch, working storage, splits of lists.
Runs on any host."""

from __future__ import annotations

import ctypes

import pytest
import torch

from hybrid_training_amd import MuonConfig, MuonOptimizer, GroupHandle, UnsupportedFeatureError, _native, fused_linear, muon
from hybrid_training_amd.errors import ConfigurationError, NativeKernelError

FAKE = ctypes.c_void_p(4096)


def linear(lib, x=FAKE, ldx=8, w=FAKE, ldw=8, y=FAKE, ldy=8, z=None, ldz=8, r=None, ldr=8, m=4, k=8, n=8, dtype=0, act=0):
    return lib.hbt_linear(x, ldx, w, ldw, None, r, ldr, y, ldy, z, ldz, m, k, n, dtype, act, None, 0, None)


def backward(lib, dx=FAKE, dw=FAKE, db=None, m=100, k=8, n=8, dtype=0, act=0, z=None, lddy=8):
    return lib.hbt_linear_backward(FAKE, lddy, FAKE, 8, FAKE, 8, z, 8, dx, 8, dw, 8, db, m, k, n, dtype, act, None, 0, None)


def orthogonalize(lib, rows, cols, count=1, product=2, steps=5, dtype=0, eps=0.0, address=4096):
    table = _native.pointer_array([address] * max(len(rows), 1))
    return lib.hbt_orthogonalize(table, table, _native.int64_array(rows), _native.int64_array(cols), count, dtype, dtype,
                                 product, steps, 1.0, 1.0, 1.0, eps, None, 0, None)


def test_linear_refuses_bad_arguments():
    lib = _native.library()
    assert linear(lib, m=-1) == -1 and b"negative" in lib.hbt_last_error()
    assert linear(lib, dtype=3) == -1 and b"dtype 3" in lib.hbt_last_error()
    assert linear(lib, act=5) == -1 and b"activation" in lib.hbt_last_error()
    assert linear(lib, x=None) == -1 and b"x is null" in lib.hbt_last_error()
    assert linear(lib, y=None) == -1 and linear(lib, w=None) == -1
    assert linear(lib, ldx=7) == -1 and b"overlap" in lib.hbt_last_error()
    assert linear(lib, z=FAKE, ldz=7) == -1 and linear(lib, r=FAKE, ldr=7) == -1
    assert linear(lib, ldw=(1 << 20) + 1) == -2 and b"at most" in lib.hbt_last_error()
    assert linear(lib, m=1 << 28) == -2
    assert linear(lib, m=0) == 0 and linear(lib, n=0) == 0  # nothing to do, nothing launched
    assert lib.hbt_last_error() == b""


def test_linear_backward_refuses_bad_arguments():
    lib = _native.library()
    assert backward(lib, dtype=3) == -1 and backward(lib, act=-1) == -1 and backward(lib, k=-1) == -1
    assert backward(lib, act=1) == -1 and b"z is null" in lib.hbt_last_error()
    assert backward(lib, act=1, z=FAKE) == -1 and b"workspace" in lib.hbt_last_error()
    assert backward(lib, lddy=3) == -1
    assert backward(lib, dx=None, dw=None, m=8) == 0  # nothing asked for
    assert lib.hbt_linear_backward_workspace(100, 8, 8, 0, 0, 8) == -1
    assert lib.hbt_linear_backward_workspace(100, 8, 8, 7, 0, 1) == -1
    assert lib.hbt_linear_workspace(-1, 8, 8, 0) == -1
    assert lib.hbt_linear_workspace(16, 1 << 14, 64, 1) == 0  # few rows take no working storage
    assert lib.hbt_linear_workspace(64, 1 << 14, 64, 1) > 0  # one tile's long sum is split
    # dz with an activation: padded rows of 16 bytes
    assert lib.hbt_linear_backward_workspace(1000, 8, 77, 1, 2, 1) >= 1000 * 80 * 2


def test_orthogonalize_refuses_bad_arguments():
    lib = _native.library()
    assert orthogonalize(lib, [4], [4], count=33) == -1 and b"count" in lib.hbt_last_error()
    assert orthogonalize(lib, [4], [4], product=1) == -1 and b"product" in lib.hbt_last_error()
    assert orthogonalize(lib, [4], [4], steps=0) == -1 and orthogonalize(lib, [4], [4], steps=65) == -1
    assert orthogonalize(lib, [-4], [4]) == -1
    assert orthogonalize(lib, [(1 << 20) + 1], [4]) == -2
    assert orthogonalize(lib, [1 << 19], [1 << 19]) == -2
    assert orthogonalize(lib, [200], [200], dtype=3) == -1
    assert orthogonalize(lib, [200], [200], eps=-1.0) == -1
    assert orthogonalize(lib, [200], [200], address=0) == -1 and b"null" in lib.hbt_last_error()
    assert orthogonalize(lib, [200], [200]) == -1 and b"workspace" in lib.hbt_last_error()
    assert orthogonalize(lib, [0, 3], [5, 0], count=2) == 0  # empty matrices are skipped
    none = lib.hbt_muon_step(None, None, None, None, None, None, 1, 0, 0, 2, 1.0, None, 0.9, 0.1, 1, 5, 1.0, 1.0, 1.0, 0.0,
                             1.0, 0.1, None, None, 0, None)
    assert none == -1
    with pytest.raises(NativeKernelError):
        _native.check(none, "test")


def test_working_storage_adds_up_and_lists_are_split(monkeypatch):
    lib = _native.library()
    shapes = [(200, 300), (300, 200), (64, 64), (1, 4000), (513, 129)]

    def need(indices):
        return lib.hbt_orthogonal_workspace(_native.int64_array([shapes[i][0] for i in indices]),
                                            _native.int64_array([shapes[i][1] for i in indices]), len(indices), 2)

    assert need(range(5)) == sum(need([i]) for i in range(5))
    assert need([2]) == 0  # a small matrix stays in one workgroup
    assert muon._call_groups(shapes, 2) == [([0, 1, 2, 3, 4], need(range(5)))]
    many = [(200, 300)] * 70
    groups = muon._call_groups(many, 2)
    assert [len(i) for i, _ in groups] == [32, 32, 6] and sum((i for i, _ in groups), []) == list(range(70))
    monkeypatch.setattr(muon, "_WORKSPACE_CAP", need([0]) * 3)
    groups = muon._call_groups(many[:8], 2)
    assert [i for i, _ in groups] == [[0, 1, 2], [3, 4, 5], [6, 7]]
    assert all(nbytes == need([0]) * len(i) for i, nbytes in groups)
    monkeypatch.setattr(muon, "_WORKSPACE_CAP", 1)  # a single matrix may need more than the cap
    assert [i for i, _ in muon._call_groups(many[:2], 2)] == [[0], [1]]


def test_host_tensors_and_bad_options_are_refused():
    x = torch.zeros(2, 4)
    with pytest.raises(UnsupportedFeatureError, match="HIP device"):
        fused_linear(x, torch.zeros(3, 4))
    with pytest.raises(UnsupportedFeatureError, match="HIP device"):
        muon.orthogonalize([x])
    with pytest.raises(UnsupportedFeatureError, match="device memory"):
        MuonOptimizer([torch.nn.Parameter(x)], MuonConfig(), norm_group=GroupHandle.trivial("world"),
                      device=torch.device("cpu"))
    for options in ({"steps": 1.5}, {"coefficients": (1.0,)}, {"eps": float("inf")}, {"scale": "unit"}, {"momentum": -0.1}):
        with pytest.raises(ConfigurationError):
            MuonConfig(**options)
    assert MuonConfig(coefficients=[1, 2, 3]).coefficients == (1.0, 2.0, 3.0)
    assert muon._update_scale("rms", (100, 400)) == 0.2 * 20 and muon._update_scale("spectral", (400, 100)) == 2.0
