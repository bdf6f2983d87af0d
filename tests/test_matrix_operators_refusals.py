"""What the matrix operators refuse, or split, on the host before any launch.  Runs on any host."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

import hybrid_training_amd
from hybrid_training_amd import UnsupportedFeatureError, _native, fused_linear, linear, muon
from hybrid_training_amd.errors import NativeKernelError


@pytest.fixture(autouse=True)
def _no_error_is_left():
    """The last refused call's message stays with the thread until a call succeeds."""
    yield
    assert _native.library().hbt_linear_workspace(8, 8, 8, 0) == 0


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A tangent is not dropped: no kernel carries it, whichever argument holds it."""
    monkeypatch.setattr(linear, "_check", lambda *_: None)
    monkeypatch.setattr(linear, "_forward", lambda x, w, b, r, *_, **__: (x.detach() @ w.detach().t(), None))
    x, w, b, r = torch.randn(2, 4), torch.randn(3, 4), torch.randn(3), torch.randn(2, 3)
    with forward_ad.dual_level():
        for at in range(4):
            given = [x, w, b, r]
            given[at] = forward_ad.make_dual(given[at], torch.ones_like(given[at]))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(UnsupportedFeatureError, match="forward-mode"):
                    fused_linear(given[0], given[1], given[2], residual=given[3])
            given[at - 1] = given[at - 1].clone().requires_grad_(True)
            with pytest.raises(UnsupportedFeatureError, match="forward-mode"):
                fused_linear(given[0], given[1], given[2], residual=given[3])
        # a level without a tangent is an ordinary call
        assert torch.equal(fused_linear(x, w, b, residual=r), x @ w.t())
    assert torch.equal(fused_linear(x, w, b, residual=r), x @ w.t())


HUGE = [1 << 26, (1 << 26) + 1, 1 << 31, 1 << 48, 1 << 50, (1 << 63) - 1]


def test_working_storage_of_sizes_past_the_limits():
    """-1 wherever the call itself refuses, whatever the arithmetic on such sizes gives.  In a process
    of its own: a division by zero ended it."""
    code = f"""
from hybrid_training_amd import _native
lib = _native.library()
for tokens in {HUGE}:
    for wants in (1, 2, 4, 7):
        print(lib.hbt_linear_backward_workspace(tokens, 8, 100, 0, 1, wants))
    print(lib.hbt_linear_workspace(tokens, 8, 100, 1))
    print(lib.hbt_linear_backward_workspace(8, tokens, tokens, 1, 1, 7), lib.hbt_linear_workspace(8, tokens, tokens, 1))
"""
    path = os.path.dirname(os.path.dirname(hybrid_training_amd.__file__))
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                          env={**os.environ, "PYTHONPATH": path})
    assert done.returncode == 0, done.returncode
    values = [int(v) for v in done.stdout.split()]
    each = len(values) // len(HUGE)
    assert each == 7 and all(v >= 0 for v in values[:5])  # 2^26 rows are within the limits
    assert values[5:each] == [-1, -1]  # a product of 2^26 by 2^26 is not
    assert values[each:] == [-1] * (len(values) - each)


def test_working_storage_names_what_it_refuses():
    lib = _native.library()
    assert lib.hbt_linear_workspace(8, 8, -1, 0) == -1 and b"negative" in lib.hbt_last_error()
    assert lib.hbt_linear_backward_workspace(8, 8, 8, 0, 9, 1) == -1 and b"activation" in lib.hbt_last_error()
    assert lib.hbt_linear_backward_workspace(8, 8, 8, 0, 0, 8) == -1 and b"wanted" in lib.hbt_last_error()
    assert lib.hbt_linear_workspace(1 << 27, 8, 8, 0) == -1 and b"launch limits" in lib.hbt_last_error()
    assert lib.hbt_linear_workspace(8, 8, 8, 0) == 0 and lib.hbt_last_error() == b""


def test_lists_past_a_calls_elements_are_split(monkeypatch):
    """A call takes 2^34 elements; a list of matrices that each fit takes as many calls as it needs."""
    side = 1 << 16  # 2^32 elements a matrix
    groups = muon._call_groups([(side, side)] * 9, _native.DTYPE_F16)
    assert sum((indices for indices, _ in groups), []) == list(range(9))
    monkeypatch.setattr(muon, "_WORKSPACE_CAP", 1 << 62)  # the elements alone
    groups = muon._call_groups([(side, side)] * 9, _native.DTYPE_F16)
    assert [indices for indices, _ in groups] == [[0, 1, 2, 3], [4, 5, 6, 7], [8]]
    lib = _native.library()
    for indices, nbytes in groups:
        sides = _native.int64_array([side] * len(indices))
        assert lib.hbt_orthogonal_workspace(sides, sides, len(indices), _native.DTYPE_F16) == nbytes > 0
    # small matrices, which take no working storage, among them
    assert [i for i, _ in muon._call_groups([(side, side)] * 4 + [(8, 8)], _native.DTYPE_F16)] == [[0, 1, 2, 3], [4]]
    assert muon._call_groups([], _native.DTYPE_F16) == []
    with pytest.raises(NativeKernelError, match="past the limits"):
        muon._call_groups([(8, 8), (1 << 18, 1 << 18)], _native.DTYPE_F16)
