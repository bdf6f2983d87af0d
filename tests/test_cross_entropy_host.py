"""What the loss over a vocabulary refuses, and its working storage, without a device."""

from __future__ import annotations

import ctypes

import pytest
import torch

from hybrid_training_amd import LinearCrossEntropy, _native, linear_cross_entropy
from hybrid_training_amd.errors import UnsupportedFeatureError

GIB = 1 << 30


def test_host_tensors_are_refused():
    head = LinearCrossEntropy(8, 20)
    assert [tuple(p.shape) for p in head.parameters()] == [(20, 8)]
    assert "vocabulary=20" in repr(head)
    with pytest.raises(UnsupportedFeatureError, match="HIP device"):
        head(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(UnsupportedFeatureError, match="reduction"):
        linear_cross_entropy(torch.zeros(3, 8), torch.zeros(20, 8), torch.zeros(3, dtype=torch.int64), reduction="avg")


def test_working_storage():
    size = _native.library().hbt_linear_cross_entropy_workspace
    assert size(0, 64, 100, 1, 0, 1, 0.0, 1) == 0
    assert size(16, 32, 97, 0, 7, 0, 0.0, 1) == 0  # a small call's stands in LDS
    # one token over a large vocabulary: statistics alone
    assert 0 < size(1, 4096, 128256, 1, 0, 1, 0.0, 1) < 1 << 20
    # evaluation never holds logits, training at most 2 GiB of exponentials beside rows, fp32 sums and at most
    # 1024 tiles' parts of dx's sums
    assert size(8192, 4096, 128256, 1, 0, 1, 0.0, 1) < 8192 * 4096 * 2 + (1 << 28) + (8 << 20)
    one = size(8192, 4096, 128256, 1, 3, 1, 0.0, 1)
    parts = 1024 * 256 * 256 * 4
    assert one < 2 * GIB + 8192 * 4096 * 2 + parts + (1 << 27)
    more = size(16384, 4096, 128256, 1, 3, 1, 0.0, 1)
    assert more < 2 * GIB + 16384 * 4096 * 2 + 4 * 128256 * 4096 + parts + (1 << 27)
    assert size(32768, 4096, 128256, 1, 3, 1, 0.0, 1) - more < 16384 * 4096 * 2 + (4 << 20)
    # a 2-byte weight off 16 bytes is copied for many tokens, an fp32 one is not
    assert size(8192, 64, 50257, 1, 0, 1, 0.0, 0) - size(8192, 64, 50257, 1, 0, 1, 0.0, 1) > 50257 * 64 * 2 - (1 << 20)
    assert size(8192, 64, 50257, 0, 0, 0, 0.0, 0) == size(8192, 64, 50257, 0, 0, 0, 0.0, 1)
    # fp32 results carry the sums themselves
    assert size(16384, 4096, 128256, 1, 3, 0, 0.0, 1) < more - 4 * 128256 * 4096 + (1 << 20)
    assert size(10, 64, 10000, 1, 0, 1, 0.1, 1) > size(10, 64, 10000, 1, 0, 1, 0.0, 1)
    for bad in ((-1, 64, 100, 1, 0, 1), (1, -1, 100, 1, 0, 1), (1, 64, 0, 1, 0, 1), (1, 64, 100, 3, 0, 1),
                (1, 64, 100, 1, 8, 1), (1, 64, 100, 1, 1, 2), (1, 64, (1 << 20), 1, 0, 1), (1, 1 << 20, 100, 1, 0, 1),
                ((1 << 24) + 1, 64, 100, 1, 0, 1)):
        assert size(*bad, 0.0, 1) == -1 and _native.library().hbt_last_error()
    assert size(0, 64, 100, 1, 0, 1, 0.0, 1) == 0  # leaves no message behind


def test_the_library_refuses_bad_calls_before_any_launch():
    lib = _native.library()
    p = ctypes.c_void_p(4096)

    def call(x=p, ldx=64, w=p, ldw=64, target=p, token_grads=None, loss=p, dx=None, lddx=0, dw=None, lddw=0, tokens=4,
             inner=64, vocab=10000, dtype=1, grad_dtype=1, smoothing=0.0, reduction=0, space=p, nbytes=1 << 30):
        return lib.hbt_linear_cross_entropy(x, ldx, w, ldw, None, target, token_grads, None, loss, dx, lddx, dw, lddw, None,
                                            tokens, inner, vocab, dtype, grad_dtype, -100, smoothing, reduction, space,
                                            nbytes, None)

    for wrong in (dict(tokens=0), dict(tokens=-1), dict(vocab=0), dict(dtype=3), dict(x=None), dict(w=None),
                  dict(ldx=63), dict(ldw=(1 << 20) + 1), dict(target=None), dict(loss=None), dict(smoothing=-0.1),
                  dict(smoothing=float("nan")), dict(reduction=3), dict(reduction=1, token_grads=p),
                  dict(dx=p, lddx=63), dict(dw=p, lddw=63), dict(dx=p, lddx=64, grad_dtype=2), dict(space=None),
                  dict(nbytes=16), dict(space=ctypes.c_void_p(4100))):
        assert call(**wrong) in (-1, -2), wrong
        assert b"hbt_linear_cross_entropy" in lib.hbt_last_error()
    one, four = _native.pointer_array([4096]), _native.int64_array([4])
    assert lib.hbt_scale_round(None, None, None, 1, 0, 1, p, None) == -1
    assert lib.hbt_scale_round(one, one, four, 5, 0, 0, p, None) == -1
    assert lib.hbt_scale_round(one, one, four, 1, 0, 1, p, None) == -1  # in place with two dtypes
    assert lib.hbt_scale_round(one, one, four, 1, 1, 0, p, None) == -1
    assert lib.hbt_scale_round(one, one, four, 1, 0, 0, None, None) == -1
    assert lib.hbt_scale_round(_native.pointer_array([4096, 8192]), _native.pointer_array([4096, 12288]),
                               _native.int64_array([4, 4]), 2, 0, 0, p, None) == -1
    assert lib.hbt_scale_round(one, one, _native.int64_array([-4]), 1, 0, 0, p, None) == -1
    assert lib.hbt_scale_round(None, None, None, 0, 0, 1, None, None) == 0  # nothing to do, and no message left behind
