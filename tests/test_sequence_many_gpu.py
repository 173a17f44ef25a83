"""Packed sequences in numbers: many of them, rows before the first and behind the last, starts that make no sense."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from kernel_matmul_b200 import ops  # noqa: E402

DEV = "cuda"
FORMS = [(torch.float32, "fma"), (torch.bfloat16, "tc"), (torch.float16, "tc")]


def grads(q, k, v, g, s0, starts, path, go, gs):
    inputs = [t.detach().requires_grad_() for t in (q, k, v, g, s0)]
    o, s = ops.decay_attention(*inputs[:4], initial_state=inputs[4], sequence_starts=starts, return_state=True, path=path)
    return [o.detach(), s.detach(), *torch.autograd.grad([o, s], inputs, [go, gs])]


@pytest.mark.parametrize("dtype, path", FORMS, ids=str)
@pytest.mark.parametrize("count, length", [(33, 7), (1025, 1), (40_000, 3), (40, 1100), (1100, 260)])
def test_packed_sequences_are_those_of_a_batch(count, length, dtype, path):
    """The same bits as a batch of the same sequences, but where a sequence is cut in one form and not in the other."""
    heads, d = 2, 16
    draw = lambda *s: torch.randn(s, device=DEV)  # noqa: E731
    q, k, v, go = (draw(count, length, heads, d).to(dtype) for _ in range(4))
    s0, gs, g = draw(count, heads, d, d), draw(count, heads, d, d), torch.tensor([-0.3, -0.01], device=DEV)
    starts = torch.arange(count + 1, device=DEV, dtype=torch.int32) * length
    want = grads(q, k, v, g, s0, None, path, go, gs)
    got = grads(*(t.flatten(0, 1) for t in (q, k, v)), g, s0, starts, path, go.flatten(0, 1), gs)
    for name, a, b in zip(("o", "state", "dq", "dk", "dv", "dlog_decay", "dinitial"), got, want):
        b = b.reshape(a.shape)
        if name == "dlog_decay":  # (sums over all sequences, in another order)
            assert torch.allclose(a, b, rtol=1e-4, atol=1e-3 * count**0.5)
        elif length <= 256:
            assert torch.equal(a, b), name
        else:  # the state between segments is rounded to 32 bits once more, results as they are anyway: two of their steps at most
            assert ((a.float() - b.float()).norm() <= 2 * torch.finfo(a.dtype).eps * b.float().norm() + 1e-5).all(), name


@pytest.mark.parametrize("dtype, path", FORMS, ids=str)
@pytest.mark.parametrize("before, behind", [(0, 0), (5000, 0), (0, 5000), (700, 2500), (1, 1)])
def test_rows_around_the_sequences_are_zero(before, behind, dtype, path):
    lengths, heads, d = [300, 0, 2600, 1, 0], 2, 64
    n = before + sum(lengths) + behind
    q, k, v = (torch.randn(n, heads, d, device=DEV).to(dtype).requires_grad_() for _ in range(3))
    g = torch.tensor([-0.3, -0.01], device=DEV)
    starts = torch.tensor([before, *lengths], device=DEV).cumsum(0).to(torch.int32)
    torch.full((n, heads, d), float("nan"), device=DEV, dtype=dtype)  # (freed at once: what the results' memory may hold)
    o = ops.decay_attention(q, k, v, g, sequence_starts=starts, path=path)
    got = [o.detach(), *torch.autograd.grad(o, [q, k, v], torch.ones_like(o))]
    inside = slice(before, before + sum(lengths))
    o = ops.decay_attention(q[inside], k[inside], v[inside], g, sequence_starts=starts - before, path=path)
    want = [o.detach(), *torch.autograd.grad(o, [q, k, v], torch.ones_like(o))]
    for name, a, b in zip(("o", "dq", "dk", "dv"), got, want):
        assert not a[:before].any() and not a[n - behind :].any(), name
        b = b if name == "o" else b[inside]
        # (sequences may be cut at other places)
        assert (a[inside].float() - b.float()).norm() <= 2 * torch.finfo(dtype).eps * b.float().norm() + 1e-5, name


@pytest.mark.parametrize("dtype, path", FORMS, ids=str)
def test_many_starts_that_make_no_sense_stay_inside(dtype, path):
    """Results are undefined, but nothing is read or written out of range."""
    t, count = 3000, 20_001
    q, k, v = (torch.randn(t, 1, 16, device=DEV).to(dtype).requires_grad_() for _ in range(3))
    g = torch.tensor([-0.1], device=DEV).requires_grad_()
    guard = [torch.full((1 << 20,), 7.0, device=DEV) for _ in range(4)]
    swing = torch.zeros(count, dtype=torch.int32, device=DEV)
    swing[1::2] = t
    for starts in (swing, t - swing, torch.randint(-t, 2 * t, (count,), device=DEV, dtype=torch.int32), torch.full((count,), t, device=DEV, dtype=torch.int32)):
        o, s = ops.decay_attention(q, k, v, g, sequence_starts=starts, return_state=True, path=path)
        torch.autograd.grad(o.sum() + s.sum(), [q, k, v, g])
    ops.check()
    assert all((x == 7.0).all() for x in guard)
