"""Packed sequences: what stands in the rows of other sequences, or in rows of no sequence, reaches no result of a sequence."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from kernel_matmul_b200 import ops  # noqa: E402

DEV = "cuda"
FORMS = [(torch.float32, "fma"), (torch.bfloat16, "fma"), (torch.bfloat16, "tc"), (torch.float16, "fma"), (torch.float16, "tc")]
# (lengths, tokens behind the last sequence)
PACKS = [([140, 60, 200], 30), ([1, 127, 5, 128, 3, 129, 64], 7), ([100], 200), ([31, 0, 33, 17], 1)]


def run(x, starts, path, cotangents):
    inputs = [x[n].requires_grad_() for n in ("q", "k", "v", "log_decay", "initial")]
    o, s = ops.decay_attention(*inputs[:4], initial_state=inputs[4], sequence_starts=starts, return_state=True, path=path)
    grads = torch.autograd.grad([o, s], inputs, cotangents)
    # (a tensor's gradient comes back without a graph, and the next call takes fresh leaves)
    return dict(zip(("o", "state", "dq", "dk", "dv", "dlog_decay", "dinitial"), (o.detach(), s.detach(), *grads)))


def make(lengths, tail, dtype, heads, groups, dk, dv):
    n = sum(lengths) + tail
    x = {"q": (n, heads, dk), "k": (n, groups, dk), "v": (n, groups, dv), "go": (n, heads, dv)}
    x = {name: torch.randn(shape, device=DEV).to(dtype) for name, shape in x.items()}
    x["log_decay"] = -(2.0 ** -torch.arange(1.0, heads + 1, device=DEV))
    x["initial"] = torch.randn(len(lengths), heads, dk, dv, device=DEV)
    x["gs"] = torch.randn(len(lengths), heads, dk, dv, device=DEV)
    return x, torch.tensor([0, *lengths], device=DEV).cumsum(0).to(torch.int32)


def compare(x, rows, values, starts, path, sequences):
    """The results with ``values`` in ``rows`` of all operands and of the result's gradient, against those without: the same bits in
    all other rows and in all other sequences' states."""
    clean = {n: t.clone() for n, t in x.items()}
    want = run(clean, starts, path, [clean["go"], clean["gs"]])
    spoilt = {n: t.clone() for n, t in x.items()}
    for name in ("q", "k", "v", "go"):
        spoilt[name][rows] = values(spoilt[name][rows])
    got = run(spoilt, starts, path, [spoilt["go"], spoilt["gs"]])
    keep = torch.ones(x["q"].shape[0], dtype=torch.bool, device=DEV)
    keep[rows] = False
    others = torch.ones(len(x["initial"]), dtype=torch.bool, device=DEV)
    for i in sequences:
        others[i] = False
        keep[starts[i] : starts[i + 1]] = False
    for name in ("o", "dq", "dk", "dv"):
        assert want[name][keep].isfinite().all()
        assert torch.equal(got[name][keep], want[name][keep]), name
    for name in ("state", "dinitial"):
        assert torch.equal(got[name][others], want[name][others]), name
    return got, want


def not_finite(x):
    y = torch.full_like(x, math.nan)
    y[:, :, ::3] = math.inf
    y[:, :, 1::3] = -math.inf
    return y


@pytest.mark.parametrize("dims", [(2, 2, 64, 64), (4, 2, 128, 40), (3, 1, 40, 128)], ids=str)
@pytest.mark.parametrize("dtype, path", FORMS, ids=str)
@pytest.mark.parametrize("lengths, tail", PACKS, ids=str)
def test_rows_of_no_sequence_reach_no_result(lengths, tail, dtype, path, dims):
    """Padding behind the last sequence may hold anything: no result depends on it, the gradient of the decays included, and it has none."""
    x, starts = make(lengths, tail, dtype, *dims)
    rows = slice(sum(lengths), None)
    got, want = compare(x, rows, not_finite, starts, path, [])
    assert torch.equal(got["dlog_decay"], want["dlog_decay"]) and got["dlog_decay"].isfinite().all()
    for name in ("o", "dq", "dk", "dv"):
        assert not got[name][rows].any(), name


@pytest.mark.parametrize("dtype, path", FORMS, ids=str)
@pytest.mark.parametrize("lengths, tail", PACKS[:2], ids=str)
def test_another_sequence_reaches_no_result(lengths, tail, dtype, path):
    x, starts = make(lengths, tail, dtype, 2, 1, 64, 72)
    for bad in range(len(lengths)):
        first = int(starts[bad])
        for at in {first, first + lengths[bad] // 2, first + lengths[bad] - 1}:
            compare(x, slice(at, at + 1), not_finite, starts, path, [bad])


@pytest.mark.parametrize("dtype, path", FORMS, ids=str)
def test_the_size_of_a_neighbour_reaches_no_result(dtype, path):
    """fp16 operands are scaled by the largest of a row: that row's own."""
    x, starts = make([90, 100], 20, dtype, 2, 2, 64, 64)
    for name in ("q", "k", "v", "go"):
        x[name][:90] *= 2.0**-9
    compare(x, slice(90, None), lambda y: y.sign() * 2.0**12, starts, path, [1])
