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
