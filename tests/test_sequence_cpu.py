"""Sequence operators: what can be said without a GPU."""
from __future__ import annotations

import math

import pytest
import torch

from kernel_matmul_b200 import ops


def test_tensors_on_the_cpu_are_refused():
    x = torch.randn(4, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.decay_attention(x, x, x, torch.zeros(2))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.decay_attention_step(x, x, x, torch.zeros(2), torch.zeros(4, 2, 8, 8))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.rotary(x, x, torch.arange(4), torch.ones(4))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.global_norm([x])
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.clip_global_norm_([x], 1.0)
    with pytest.raises(RuntimeError):
        ops.rotary("x", None, torch.arange(4), torch.ones(4))


def test_bad_values_are_refused():
    with pytest.raises(ValueError):
        ops.global_norm([])
    with pytest.raises(ValueError):
        ops.clip_global_norm_([torch.zeros(1)], -1.0)
    with pytest.raises(ValueError):
        ops.clip_global_norm_([torch.zeros(1)], math.nan)
    x = torch.randn(4, 2, 8)
    with pytest.raises(ValueError):
        ops.decay_attention(x, x, x, torch.zeros(2), path="nodes")
    for kw in (dict(scaling="other"), dict(scaling="parts", factor=2.0), dict(base=0.0), dict(factor=0.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(8, device="cpu", **kw)
    with pytest.raises(ValueError):
        ops.rotary_frequencies(7, device="cpu")


def test_rotary_frequencies():
    f, s = ops.rotary_frequencies(8, base=100.0, device="cpu")
    assert s == 1.0 and torch.allclose(f, torch.tensor([100.0 ** (-i / 4) for i in range(4)], dtype=torch.float64), rtol=1e-15)
    half, _ = ops.rotary_frequencies(8, base=100.0, scaling="linear", factor=2.0, device="cpu")
    assert torch.equal(half, f / 2)
    b, _ = ops.rotary_frequencies(8, base=100.0, scaling="base", factor=4.0, device="cpu")
    assert b[0] == f[0] and abs(b[-1] * 4 / f[-1] - 1) < 1e-14
    p, s = ops.rotary_frequencies(64, scaling="parts", factor=8.0, original_tokens=4096, device="cpu")
    full, _ = ops.rotary_frequencies(64, device="cpu")
    turns = 4096 * full / (2 * math.pi)
    assert torch.equal(p[turns >= 32], full[turns >= 32]) and torch.allclose(p[turns <= 1], full[turns <= 1] / 8, rtol=1e-15)
    assert s == 0.1 * math.log(8.0) + 1.0
    assert ops.rotary_frequencies(0, device="cpu")[0].shape == (0,)


@pytest.mark.parametrize("field, value", [("reverse", 3), ("reverse", -1), ("states", 3), ("path", 3), ("dk", 0), ("dv", 129), ("group", 0),
                                          ("tokens", -1), ("tokens", 2**31), ("dtype", 9), ("out_dtype", 2)])
def test_bad_problems_are_refused(field, value):
    import ctypes

    from kernel_matmul_b200._lib import KmDecayProblem, lib

    good = dict(dtype=0, out_dtype=0, reverse=0, path=0, sequences=1, tokens=8, groups=2, group=1, dk=16, dv=16, packed=0, states=0, scale=1.0)
    p = KmDecayProblem(**{**good, field: value})
    calls = [lambda q: lib.km_decay_attention(q, *[None] * 4, None, None, None, None, None, 0, None),
             lambda q: lib.km_decay_gradient(q, *[None] * 4, None, None, None, None, None, None, 0, None)]
    for call in calls:
        assert call(KmDecayProblem(**good)) != 0 and b"null argument" in lib.km_last_error()
        assert call(p) != 0 and b"null" not in lib.km_last_error()
        assert call(ctypes.POINTER(KmDecayProblem)()) != 0 and b"null problem" in lib.km_last_error()
    assert lib.km_decay_attention_workspace_bytes(p) == 0
