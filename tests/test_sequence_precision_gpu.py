"""How far results of the linear attention with decay are from 64 bits, as 2-norms: what the parts of the operands buy."""
from __future__ import annotations

import math

import pytest
import torch

from sequence_reference import attention, attention_with_scales, half_step

pytestmark = pytest.mark.gpu

from kernel_matmul_b200 import ops  # noqa: E402

DEV = "cuda"


def evaluate(dtype, path, tokens, heads, groups, dk, dv, decays, sizes=(1.0, 1.0, 1.0, 1.0), initial=True, batch=2):
    """Relative 2-norm errors of results and gradients; ``sizes`` of q, k, v and of the result's gradient."""
    draw = lambda *s: torch.randn(s, device=DEV)  # noqa: E731
    x = dict(q=(draw(batch, tokens, heads, dk) * sizes[0]).to(dtype), k=(draw(batch, tokens, groups, dk) * sizes[1]).to(dtype),
             v=(draw(batch, tokens, groups, dv) * sizes[2]).to(dtype), log_decay=decays,
             initial=draw(batch, heads, dk, dv) * (sizes[1] * sizes[2] if initial else 0.0))
    go = (draw(batch, tokens, heads, dv) * sizes[3]).to(dtype)
    gs = draw(batch, heads, dk, dv) * (sizes[0] * sizes[3])
    want = attention_with_scales({n: t.double() for n, t in x.items()}, dk**-0.5, None, [go.double(), gs.double()])[0]
    inputs = [t.requires_grad_() for t in x.values()]
    o, s = ops.decay_attention(*inputs[:4], initial_state=inputs[4] if initial else None, return_state=True, path=path)
    used = inputs if initial else inputs[:4]
    grads = torch.autograd.grad([o, s], used, [go, gs])
    names = ("o", "state", "dq", "dk", "dv", "dlog_decay", "dinitial")
    return {n: ((y.detach().double() - want[n]).norm() / want[n].norm()).item() for n, y in zip(names, (o, s, *grads))}


def slopes(heads):
    return -(2.0 ** (-8.0 * torch.arange(1, heads + 1, device=DEV) / heads))


FORMS = [(torch.bfloat16, "fma"), (torch.bfloat16, "tc"), (torch.float16, "fma"), (torch.float16, "tc")]


# An fp32 evaluation of states is within 1.5e-7 of 64 bits: 3 times that.  One part of the keys less makes it 2.4e-6 in bf16 (two parts, 2^-17)
# and 2e-4 in fp16 (one part).  The gradient of a decay is a sum over tokens of terms of either sign; over 8 heads an
# fp32 evaluation is within 4e-7, and with parts of the keys left out at 5e-6: 2e-6.
STATES, DECAYS = 5e-7, 2e-6


@pytest.mark.parametrize("dtype, path", FORMS, ids=str)
@pytest.mark.parametrize("tokens, groups, dk, dv", [(300, 4, 64, 64), (1100, 8, 128, 72), (2100, 8, 40, 128)])
def test_states_and_gradients_of_decays_are_those_of_32_bits(dtype, path, tokens, groups, dk, dv):
    e = evaluate(dtype, path, tokens, 8, groups, dk, dv, slopes(8))
    assert e["state"] <= STATES and e["dinitial"] <= STATES and e["dlog_decay"] <= DECAYS, e


@pytest.mark.parametrize("path", ["fma", "tc"])
@pytest.mark.parametrize("fast", [False, True])
@pytest.mark.parametrize("sizes", [(1.0, 1.0, 1.0, 1.0), (1.0, 1e-2, 1.0, 1.0), (1e-2, 1e-1, 1.0, 1e-2), (1.0, 1e-3, 1.0, 1e-3), (1e-3, 1e-3, 1e-3, 1e-3),
                                   (300.0, 100.0, 1.0, 1.0)], ids=str)
def test_small_fp16_operands_keep_their_bits(path, fast, sizes):
    """Decayed operands lie below fp16's normal range where the operands themselves are small (normalised keys, gradients)."""
    decays = torch.full((8,), -0.256, device=DEV) if fast else slopes(8)
    e = evaluate(torch.float16, path, 700, 8, 8, 64, 64, decays, sizes)
    assert e["state"] <= STATES and e["dinitial"] <= STATES and e["dlog_decay"] <= DECAYS, e


@pytest.mark.parametrize("dtype, path", FORMS, ids=str)
def test_results_of_one_chunk_are_rounded_once(dtype, path):
    """Without a state that comes in, a result of one chunk is P v: rounded once, P in two parts.

    A value m 2^e with m spread over [1, 2) evenly in its logarithm, rounded to nearest with a half step u, is off by an error spread
    evenly over +- u 2^e: relative 2-norm u sqrt(1/3) / sqrt(E m^2) = u sqrt(1/3) / sqrt(3 / (2 ln 2)) = 0.392 u.  A second rounding
    of the same size (P in one part) makes it 0.555 u.  In between, for what the spread of m differs: 0.46 u."""
    e = evaluate(dtype, path, 128, 8, 8, 64, 64, slopes(8), initial=False, batch=8)
    assert e["o"] <= 0.46 * half_step(dtype), e
    # the gradient of q is the same product; those of k and v have the state's gradient in them, whose copy is rounded once more: 0.555 u, and
    # the same margin on top
    assert e["dq"] <= 0.46 * half_step(dtype) and max(e["dk"], e["dv"]) <= 0.65 * half_step(dtype), e


@pytest.mark.parametrize("dtype, path", FORMS, ids=str)
def test_results_of_many_chunks_are_rounded_twice(dtype, path):
    """The state's copy and the result: 0.555 u (above), with the same margin."""
    e = evaluate(dtype, path, 1100, 8, 8, 64, 64, slopes(8))
    assert max(e["o"], e["dq"], e["dk"], e["dv"]) <= 0.65 * half_step(dtype), e
    assert not math.isnan(sum(e.values()))


@pytest.mark.parametrize("dtype, path", [*FORMS, (torch.float32, "fma")], ids=str)
def test_gradients_of_fast_decays(dtype, path):
    """A decay of e^g leaves its gradient terms of e^g and smaller: each head's is held against sqrt(sum_i (go_i d o_i / d g)^2), what a sum
    of its terms' random signs is in the mean (the last state and its gradient among them).  A term goes through fewer than 64 roundings to
    24 bits or more; and the exponent of a decay, g log2(e) d, is rounded three times (log2(e), both products), which makes the decay
    wrong by 3 |g| d 2^-24 of itself, where d = 1 for all terms that count."""
    decays = -torch.tensor([1.0, 4.0, 8.0, 12.0, 16.0, 24.0, 40.0, 60.0], device=DEV)
    draw = lambda d: torch.randn(2, 300, 8, d, device=DEV).to(dtype)  # noqa: E731
    q, k, v, go = draw(64), draw(64), draw(40), draw(40)
    gs = torch.randn(2, 8, 64, 40, device=DEV)
    zero = torch.zeros_like(gs, dtype=torch.float64)
    rest = lambda x: attention(q.double(), k.double(), v.double(), x, 64**-0.5, zero, None)  # noqa: E731
    slope, state_slope = torch.func.jvp(rest, (decays.double(),), (torch.ones(8, device=DEV, dtype=torch.float64),))[1]
    terms = (go.double() * slope).transpose(1, 2).flatten(2), (gs.double() * state_slope).flatten(2)  # (batch, heads, terms)
    for used in ((0,), (1,), (0, 1)):
        g = decays.clone().requires_grad_()
        results = ops.decay_attention(q, k, v, g, return_state=True, path=path)
        (got,) = torch.autograd.grad([results[i] for i in used], g, [(go, gs)[i] for i in used])
        x = torch.cat([terms[i] for i in used], -1)
        error = (got.double() - x.sum((0, 2))).abs() / x.square().sum((0, 2)).sqrt()
        assert (error <= (64 + 3 * decays.abs()) * 2.0**-24).all(), error
