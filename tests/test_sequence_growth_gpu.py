"""Linear attention with log decays above zero (states that grow): a learnable decay may step there."""
from __future__ import annotations

import pytest
import torch

from sequence_reference import attention, attention_with_scales, half_step

pytestmark = pytest.mark.gpu

from kernel_matmul_b200 import ops  # noqa: E402

DEV = "cuda"
FORMS = [(torch.float32, "fma"), (torch.bfloat16, "fma"), (torch.bfloat16, "tc"), (torch.float16, "fma"), (torch.float16, "tc")]
# tokens, log decays of the two heads, size of v and of the result's gradient (so that results stay in fp16's range:
# they grow by up to e^(g tokens))
CASES = [(300, (0.02, 0.011), 2.0**-6), (140, (0.1, -0.5), 2.0**-10), (128, (0.1, 0.02), 2.0**-10), (129, (0.05, 0.0), 2.0**-7), (1000, (0.008, 0.004), 2.0**-9)]


@pytest.mark.parametrize("dims", [(2, 64, 64), (1, 128, 72)], ids=str)
@pytest.mark.parametrize("dtype, path", FORMS, ids=str)
@pytest.mark.parametrize("tokens, g, size", CASES, ids=str)
def test_growing_states(tokens, g, size, dtype, path, dims):
    """Results and gradients against 64 bits, as 2-norms over a sequence.

    With N(0, 1) operands the terms of a result have random signs, so that roundings of terms add up as the terms do: each rounding of
    operands to 16 bits (the state's copy, P, the result) is off by at most half a step of its term, and three of them by at
    most sqrt(3) half steps of the result in the 2-norm; sums in fp32, whose terms go through fewer than 64 roundings (16 steps of the
    sums of a chunk in three parts, two a chunk): 64 x 2^-24 = 3.8e-6 of all fp32 results and on top of the others.

    The gradient of a decay is one number to a head, sum_i go_i (d o_i / d g) of terms of random signs, and may come out as close to zero as
    it likes, where its error does not: that is to be held against what such a sum is in the mean, sqrt(sum_i (go_i d o_i / d g)^2)."""
    groups, dk, dv = dims
    x = dict(q=torch.randn(2, tokens, 2, dk, device=DEV).to(dtype), k=torch.randn(2, tokens, groups, dk, device=DEV).to(dtype),
             v=(torch.randn(2, tokens, groups, dv, device=DEV) * size).to(dtype), log_decay=torch.tensor(g, device=DEV),
             initial=torch.randn(2, 2, dk, dv, device=DEV) * size)
    go = (torch.randn(2, tokens, 2, dv, device=DEV) * size).to(dtype)
    gs = torch.randn(2, 2, dk, dv, device=DEV) * size
    want = attention_with_scales({n: t.double() for n, t in x.items()}, dk**-0.5, None, [go.double(), gs.double()])[0]
    inputs = [t.requires_grad_() for t in x.values()]
    o, s = ops.decay_attention(*inputs[:4], initial_state=inputs[4], return_state=True, path=path)
    grads = torch.autograd.grad([o, s], inputs, [go, gs])
    exact = {n: t.detach().double() for n, t in x.items()}
    rest = lambda g: attention(exact["q"], exact["k"], exact["v"], g, dk**-0.5, exact["initial"], None)  # noqa: E731
    slope, state_slope = torch.func.jvp(rest, (exact["log_decay"],), (torch.ones_like(exact["log_decay"]),))[1]
    terms = ((go.double() * slope) ** 2).sum((0, 1, 3)) + ((gs.double() * state_slope) ** 2).sum((0, 2, 3))
    for name, y in zip(("o", "state", "dq", "dk", "dv", "dlog_decay", "dinitial"), (o, s, *grads)):
        y, w, narrow = y.detach().double(), want[name], name not in ("state", "dlog_decay", "dinitial") and dtype != torch.float32
        if narrow and dtype == torch.float16:  # (values that fp16 does not hold are infinite)
            inside = w.abs() < torch.finfo(dtype).max
            assert (y[~inside].abs() >= torch.finfo(dtype).max).all() and inside.float().mean() > 0.99
            y, w = y[inside], w[inside]
        assert y.isfinite().all(), name
        bound = 64 * 2.0**-24 + (3**0.5 * half_step(dtype) if narrow else 0.0)
        size = terms.sqrt().norm() if name == "dlog_decay" else w.norm()
        # values below the type's normal range are off by half of its smallest step
        absolute = 0.5 * torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps * w.numel() ** 0.5
        assert (y - w).norm() <= bound * size + absolute, f"{name}: {((y - w).norm() / size).item():.2e}"


def test_packed_sequences_that_grow():
    """The FMA pipe's results, for sequences that end inside a chunk and chunks that are cut into segments."""
    lengths, heads, d = [60, 140, 1, 1300], 2, 64
    starts = torch.tensor([0, *lengths], device=DEV).cumsum(0).to(torch.int32)
    q, k, v = (torch.randn(sum(lengths), heads, d, device=DEV).half() for _ in range(3))
    g = torch.tensor([0.01, 0.002], device=DEV)
    v = v * 2.0**-14
    got = ops.decay_attention(q, k, v, g, sequence_starts=starts, path="tc", return_state=True)
    want = ops.decay_attention(q, k, v, g, sequence_starts=starts, path="fma", return_state=True)
    for a, b, bound in zip(got, want, (3 * half_step(torch.float16), 128 * 2.0**-24)):
        assert b.isfinite().all() and (a.double() - b.double()).norm() <= bound * b.double().norm()
