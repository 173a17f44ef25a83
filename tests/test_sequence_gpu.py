"""The sequence operators against 64 bits (tests/sequence_reference.py has the reference and the tolerances)."""
from __future__ import annotations

import math

import pytest
import torch

from sequence_reference import attention_with_scales, half_step, rotate, tolerance

pytestmark = pytest.mark.gpu

from kernel_matmul_b200 import gp, ops  # noqa: E402

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda"


def randn(*shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device=DEV) * scale).to(dtype)


def decays(heads, kind="slopes"):
    if kind == "none":
        return torch.zeros(heads, device=DEV)
    g = -(2.0 ** (-8.0 * torch.arange(1, heads + 1, device=DEV) / heads))
    if kind == "mixed":  # from everything forgotten at once to nothing ever
        g[0] = -math.inf
        g[-1] = 0.0
    return g


def starts_of(lengths, first=0):
    return torch.tensor([first, *lengths]).cumsum(0).to(torch.int32).to(DEV)


def paths(dtype):
    return ["fma"] if dtype == torch.float32 else ["fma", "tc"]


CASES = [
    # batch, tokens, heads, groups, dk, dv, decay; lengths of packed sequences instead of a batch
    dict(batch=1, tokens=1, heads=1, groups=1, dk=1, dv=1),
    dict(batch=2, tokens=5, heads=3, groups=3, dk=8, dv=16),
    dict(batch=1, tokens=128, heads=2, groups=2, dk=128, dv=128),
    dict(batch=2, tokens=129, heads=4, groups=2, dk=64, dv=64),
    dict(batch=1, tokens=257, heads=2, groups=1, dk=33, dv=77, decay="mixed"),
    dict(batch=1, tokens=1100, heads=2, groups=2, dk=128, dv=64, decay="none"),
    dict(batch=3, tokens=700, heads=4, groups=1, dk=72, dv=128),
    dict(batch=1, tokens=4100, heads=1, groups=1, dk=128, dv=128),
    dict(lengths=[1, 0, 130, 31, 1, 256], tail=5, heads=2, groups=1, dk=64, dv=64),
    dict(lengths=[900, 3, 0, 1500], tail=0, heads=3, groups=3, dk=40, dv=128, decay="mixed"),
    dict(lengths=[0, 0], tail=9, heads=2, groups=2, dk=16, dv=16),
    dict(lengths=[17] * 70, tail=300, heads=2, groups=2, dk=32, dv=32),
    dict(lengths=[3, 5000, 0, 1, 2600], tail=1, heads=2, groups=1, dk=64, dv=128),
    dict(batch=2, tokens=3000, heads=2, groups=2, dk=128, dv=40),
]


def make(case, dtype):
    packed = "lengths" in case
    tokens = sum(case["lengths"]) + case["tail"] if packed else case["tokens"]
    batch = 1 if packed else case["batch"]
    count = len(case["lengths"]) if packed else batch
    heads, groups, dk, dv = case["heads"], case["groups"], case["dk"], case["dv"]
    x = dict(q=randn(batch, tokens, heads, dk, dtype=dtype), k=randn(batch, tokens, groups, dk, dtype=dtype),
             v=randn(batch, tokens, groups, dv, dtype=dtype), log_decay=decays(heads, case.get("decay", "slopes")),
             initial=randn(count, heads, dk, dv, scale=2.0))
    return x, packed, tokens, count


def call(x, case, packed, path, **kw):
    q, k, v = (x[n][0] if packed else x[n] for n in ("q", "k", "v"))
    starts = starts_of(case["lengths"]) if packed else None
    return ops.decay_attention(q, k, v, x["log_decay"], initial_state=x["initial"], sequence_starts=starts, return_state=True, path=path, **kw)


def compare(got, want, sizes, dtype, case, tokens):
    for name, y in got.items():
        value, magnitude = want[0][name], want[1][name]
        bound = tolerance(name, value, magnitude, dtype, tokens, case["dk"], case["dv"], case["heads"] // case["groups"])
        error = (y.double().reshape(value.shape) - value).abs()
        worst = (error / bound).max().item() if error.numel() else 0.0
        assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_attention(case, dtype):
    for path in paths(dtype):
        x, packed, tokens, _ = make(case, dtype)
        o, s = call(x, case, packed, path)
        assert o.dtype == dtype and s.dtype == torch.float32
        want = attention_with_scales({n: t.double() for n, t in x.items()}, case["dk"] ** -0.5, case.get("lengths"))
        compare({"o": o, "state": s}, want, None, dtype, case, tokens)
        if packed and case["tail"]:
            assert not o[-case["tail"] :].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_attention_gradients(case, dtype):
    for path in paths(dtype):
        x, packed, tokens, count = make(case, dtype)
        if case.get("decay") == "mixed":
            x["log_decay"][0] = -30.0  # the gradient of a decay of exactly zero is 0 * inf in any formula with it
        go = randn(*x["q"].shape[:3], case["dv"], dtype=dtype)
        gs = randn(count, case["heads"], case["dk"], case["dv"], scale=0.5)
        for t in x.values():
            t.requires_grad_()
        o, s = call(x, case, packed, path)
        grads = torch.autograd.grad([o, s], list(x.values()), [go[0] if packed else go, gs])
        for g, t in zip(grads, x.values()):
            assert g.dtype == t.dtype and g.shape == t.shape
        got = {"d" + n: g for n, g in zip(x, grads)}
        if packed and case["tail"]:
            go[:, -case["tail"] :] = 0
        want = attention_with_scales({n: t.detach().double() for n, t in x.items()}, case["dk"] ** -0.5, case.get("lengths"),
                                     [go.double(), gs.double()])
        compare(got, want, None, dtype, case, tokens)
        if packed and case["tail"]:
            assert not got["dq"][:, -case["tail"] :].any() and not got["dv"][:, -case["tail"] :].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [CASES[3], CASES[4], CASES[7], CASES[12], dict(batch=1, tokens=700, heads=2, groups=2, dk=65, dv=65)],
                         ids=lambda c: "-".join(str(v) for v in c.values()))
def test_attention_gradients_without_states(case, dtype):
    """No state comes in and none is asked for: the passes of the gradient return 16-bit results alone."""
    for path in paths(dtype):
        x, packed, tokens, _ = make(case, dtype)
        if case.get("decay") == "mixed":
            x["log_decay"][0] = -30.0
        x["initial"].zero_()
        go = randn(*x["q"].shape[:3], case["dv"], dtype=dtype)
        leaves = [x[n].requires_grad_() for n in ("q", "k", "v", "log_decay")]
        q, k, v = (t[0] if packed else t for t in leaves[:3])
        o = ops.decay_attention(q, k, v, leaves[3], sequence_starts=starts_of(case["lengths"]) if packed else None, path=path)
        grads = torch.autograd.grad(o, leaves, go[0] if packed else go)
        if packed and case["tail"]:
            go[:, -case["tail"] :] = 0
        want = attention_with_scales({n: t.detach().double() for n, t in x.items()}, case["dk"] ** -0.5, case.get("lengths"),
                                     [go.double(), torch.zeros_like(x["initial"]).double()])
        compare({"dq": grads[0], "dk": grads[1], "dv": grads[2], "dlog_decay": grads[3]}, want, None, dtype, case, tokens)


def test_attention_gradient_against_differences():
    """Central differences of the fp64 reference are no check of the op, so the op itself is differenced, in fp32: a loss that is
    linear in the op's results; step h = 2^-6, errors h^2 / 6 of third derivatives and 2^-24 sum|terms| / h."""
    q, k, v = randn(1, 40, 2, 8), randn(1, 40, 2, 8), randn(1, 40, 2, 4)
    g, s0 = torch.tensor([-0.5, -0.05], device=DEV), randn(1, 2, 8, 4)
    go, gs = randn(1, 40, 2, 4), randn(1, 2, 8, 4)
    inputs = [q, k, v, g, s0]

    def loss(*x):
        o, s = ops.decay_attention(*x[:4], initial_state=x[4], return_state=True)
        return (o.double() * go.double()).sum() + (s.double() * gs.double()).sum()

    for t in inputs:
        t.requires_grad_()
    grads = torch.autograd.grad(loss(*inputs), inputs)
    h = 2.0**-6
    with torch.no_grad():
        for i, (t, grad) in enumerate(zip(inputs, grads)):
            direction = torch.randn_like(t)
            up, down = list(inputs), list(inputs)
            up[i], down[i] = t + h * direction, t - h * direction
            difference = (loss(*up) - loss(*down)).item() / (2 * h)
            slope = (grad.double() * direction.double()).sum().item()
            # o is linear in q, k, v and s0; third derivative in g: distance^3 weights of a few hundred, h^2 / 6 = 4e-5
            third = 4e-5 * 40.0**2 if i == 3 else 0.0
            assert abs(difference - slope) <= 1e-3 * abs(slope) + third * (1 + abs(slope)) * 0.1 + 0.05


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_strides(dtype):
    """Operands in other orders of dims, with gaps, reversed roles of heads and tokens, unaligned starts and stride 0."""
    b, t, h, d = 2, 150, 3, 40
    base = randn(b, t, h, d, dtype=dtype)
    forms = [
        base.transpose(1, 2).contiguous().transpose(1, 2),
        base.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0),
        randn(b, t, h, 2 * d, dtype=dtype)[..., 1 : d + 1],
        randn(b, t + 3, h, d, dtype=dtype)[:, 3:],
        randn(b, t, 1, d, dtype=dtype).expand(b, t, h, d),
        randn(1, t, h, d, dtype=dtype).expand(b, t, h, d),
    ]
    g = decays(h)
    for path in paths(dtype):
        for f in forms:
            for which in range(3):
                x = [base, base.flip(1), base.flip(3)]
                x[which] = f
                got = ops.decay_attention(*x, g, path=path)
                want = ops.decay_attention(*(y.contiguous() for y in x), g, path=path)
                assert torch.equal(got, want)


def test_attention_strided_state_and_batches():
    q, k, v = (randn(2, 3, 50, 2, 16) for _ in range(3))
    g, s0 = decays(2), randn(2, 3, 2, 16, 16)
    o, s = ops.decay_attention(q, k, v, g, initial_state=s0.transpose(-1, -2), return_state=True)
    for i in range(2):
        o1, s1 = ops.decay_attention(q[i], k[i], v[i], g, initial_state=s0[i].transpose(-1, -2).contiguous(), return_state=True)
        assert torch.equal(o[i], o1) and torch.equal(s[i], s1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_in_parts_and_tokens(dtype):
    """A prompt in one go, in parts, and its last tokens one by one: the same recurrence."""
    b, t, h, d = 2, 300, 2, 64
    q, k, v = (randn(b, t, h, d, dtype=dtype) for _ in range(3))
    g = decays(h)
    x = dict(q=q, k=k, v=v, log_decay=g, initial=torch.zeros(b, h, d, d, device=DEV))
    want = attention_with_scales({n: y.double() for n, y in x.items()}, d**-0.5, None)
    case = dict(dk=d, dv=d, heads=h, groups=h)
    o1, s = ops.decay_attention(q[:, :131], k[:, :131], v[:, :131], g, return_state=True)
    o2, s = ops.decay_attention(q[:, 131:290], k[:, 131:290], v[:, 131:290], g, initial_state=s, return_state=True)
    outs = [o1, o2]
    for i in range(290, t):
        outs.append(ops.decay_attention_step(q[:, i], k[:, i], v[:, i], g, s)[:, None])
    compare({"o": torch.cat(outs, 1), "state": s}, want, None, dtype, case, t)


def test_values_that_are_not_finite_stay_in_their_sequence():
    lengths = [140, 60, 200]
    for dtype in DTYPES:
        for path in paths(dtype):
            q, k, v = (randn(400, 2, 32, dtype=dtype) for _ in range(3))
            g = decays(2)
            want = ops.decay_attention(q, k, v, g, sequence_starts=starts_of(lengths), path=path)
            for t in (q, k, v):
                t[150, 1] = math.nan
                t[160, 1] = math.inf
            got = ops.decay_attention(q, k, v, g, sequence_starts=starts_of(lengths), path=path)
            assert torch.equal(got[:140], want[:140]) and torch.equal(got[200:], want[200:]) and torch.equal(got[:, 0], want[:, 0])
            assert torch.isnan(got[150:200, 1]).any()


@pytest.mark.parametrize("dk, dv", [(5, 6), (63, 70), (67, 63), (126, 127)])
def test_an_infinite_value_reaches_its_column_of_later_tokens(dk, dv):
    """With positive q and k every sum is +inf from that token on and finite elsewhere: nothing behind dk meets it as 0 * inf."""
    n, at, col = 150, 40, dv - 1
    q, k = (torch.rand(n, 2, dk, device=DEV) + 0.1 for _ in range(2))
    v = randn(n, 2, dv)
    v[at, :, col] = math.inf
    o, s = ops.decay_attention(q, k, v, torch.full((2,), -0.125, device=DEV), sequence_starts=starts_of([n]), return_state=True)
    assert torch.isposinf(o[at:, :, col]).all() and o[:at].isfinite().all() and o[:, :, :col].isfinite().all()
    assert torch.isposinf(s[..., col]).all() and s[..., :col].isfinite().all()


def test_sequence_starts_out_of_range_are_clamped():
    q, k, v = (randn(100, 1, 8) for _ in range(3))
    g = decays(1)
    wild = torch.tensor([-5, 40, 2**31 - 1], dtype=torch.int32, device=DEV)
    tame = torch.tensor([0, 40, 100], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.decay_attention(q, k, v, g, sequence_starts=wild), ops.decay_attention(q, k, v, g, sequence_starts=tame))
    first = torch.tensor([30, 60], dtype=torch.int32, device=DEV)
    o = ops.decay_attention(q, k, v, g, sequence_starts=first)
    assert not o[:30].any() and not o[60:].any()
    assert torch.equal(o[30:60], ops.decay_attention(q[30:60], k[30:60], v[30:60], g))
    none = torch.tensor([0], dtype=torch.int32, device=DEV)
    assert not ops.decay_attention(q, k, v, g, sequence_starts=none).any()


def test_attention_without_tokens():
    q, k, v = (randn(2, 0, 3, 8) for _ in range(3))
    s0 = randn(2, 3, 8, 8)
    o, s = ops.decay_attention(q, k, v, decays(3), initial_state=s0, return_state=True)
    assert o.shape == (2, 0, 3, 8) and torch.equal(s, s0)
    o, s = ops.decay_attention(q.bfloat16(), k.bfloat16(), v.bfloat16(), decays(3), return_state=True)
    assert not s.any()
    o, s = ops.decay_attention(q[:, :, :0], k[:, :, :0], v[:, :, :0], decays(0), return_state=True)
    assert o.shape == (2, 0, 0, 8) and s.shape == (2, 0, 8, 8)


def test_only_the_state_is_used():
    q, k, v = (randn(1, 70, 2, 16).requires_grad_() for _ in range(3))
    _, s = ops.decay_attention(q, k, v, decays(2), return_state=True)
    gq, gk, gv = torch.autograd.grad(s.sum(), [q, k, v], allow_unused=True)
    assert gq is None or not gq.any()
    assert gk.any() and gv.any()


def test_a_second_derivative_is_refused():
    q, k, v = (randn(1, 7, 1, 8).requires_grad_() for _ in range(3))
    o = ops.decay_attention(q, k, v, decays(1))
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(o.sum(), q, create_graph=True)


def test_other_stream_and_graph():
    q, k, v = (randn(2, 300, 2, 64, dtype=torch.bfloat16) for _ in range(3))
    g = decays(2)
    states = randn(2, 2, 64, 64)
    want, ws = ops.decay_attention(q, k, v, g, return_state=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.decay_attention(q, k, v, g)
    side.synchronize()
    assert torch.equal(got, want)
    kept = states.clone()
    one = ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, kept)
    positions, (frequencies, _) = torch.arange(300, device=DEV), ops.rotary_frequencies(64)
    turned = ops.rotary(q, k, positions, frequencies)
    grads = [randn(1000), randn(33, dtype=torch.bfloat16)]
    before = [t.clone() for t in grads]
    norm = ops.global_norm(grads)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o, s = ops.decay_attention(q, k, v, g, return_state=True)
        step = ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, states)
        q2, k2 = ops.rotary(q, k, positions, frequencies)
        n = ops.clip_global_norm_(grads, 1.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want) and torch.equal(s, ws) and torch.equal(step, one) and torch.equal(states, kept)
    assert torch.equal(q2, turned[0]) and torch.equal(k2, turned[1]) and torch.equal(n, norm)
    # new inputs in the same buffers
    q.copy_(randn(*q.shape, dtype=q.dtype))
    for t, b in zip(grads, before):
        t.copy_(b * 2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, ops.decay_attention(q, k, v, g)) and torch.allclose(n, 2 * norm)
    assert abs(ops.global_norm(grads).item() - 1.0) < 2.0**-8


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,heads,groups,dk,dv", [(1, 1, 1, 1, 1), (3, 4, 2, 64, 64), (70, 6, 6, 128, 128), (5, 2, 1, 33, 47), (40, 32, 8, 128, 100)])
def test_step(dtype, rows, heads, groups, dk, dv):
    pool = rows + 3
    q, k, v = randn(rows, heads, dk, dtype=dtype), randn(rows, groups, dk, dtype=dtype), randn(rows, groups, dv, dtype=dtype)
    g, states = decays(heads), randn(pool, heads, dk, dv)
    slots = torch.randperm(pool, device=DEV)[:rows].to(torch.int32)
    want = states.double()
    r = heads // groups
    new = torch.exp(g.double())[:, None, None] * want[slots.long()] + k.double().repeat_interleave(r, 1)[..., None] * v.double().repeat_interleave(r, 1)[..., None, :]
    size = torch.exp(g.double())[:, None, None] * want[slots.long()].abs() + k.double().abs().repeat_interleave(r, 1)[..., None] * v.double().abs().repeat_interleave(r, 1)[..., None, :]
    want[slots.long()] = new
    o = ops.decay_attention_step(q, k, v, g, states, slots=slots)
    expected = torch.einsum("bhi,bhij->bhj", q.double(), new) * dk**-0.5
    magnitude = torch.einsum("bhi,bhij->bhj", q.double().abs(), size) * dk**-0.5
    bound = magnitude * (dk + 8) * 2.0**-24 + expected.abs() * half_step(dtype) + torch.finfo(dtype).smallest_normal
    assert ((o.double() - expected).abs() <= bound).all()
    full = torch.zeros_like(want)
    full[slots.long()] = size
    assert ((states.double() - want).abs() <= full * 6 * 2.0**-24).all()


def test_step_padding_and_repeated_slots():
    """Rows without a state, and several tokens of one sequence in a batch: as if the rows came one after the other."""
    rows, heads, d = 9, 3, 64
    q, k, v = (randn(rows, heads, d, dtype=torch.bfloat16) for _ in range(3))
    g = decays(heads)
    for kind in (torch.int32, torch.int64):
        slots = torch.tensor([2, -1, 0, 2, 5, 2, 0, 1 << 30, 1], device=DEV).to(kind)
        states = randn(5, heads, d, d)
        serial = states.clone()
        want = torch.zeros(rows, heads, d, device=DEV, dtype=torch.bfloat16)
        for r, slot in enumerate(slots.tolist()):
            if 0 <= slot < 5:
                want[r] = ops.decay_attention_step(q[r : r + 1], k[r : r + 1], v[r : r + 1], g, serial[slot : slot + 1])[0]
        got = ops.decay_attention_step(q, k, v, g, states, slots=slots)
        assert torch.equal(got, want) and torch.equal(states, serial)


def test_step_strided_states():
    q, k, v = (randn(4, 2, 24) for _ in range(3))
    pool = randn(6, 2, 24, 30)
    view, copy = pool[1:5, :, :, 3:27], pool[1:5, :, :, 3:27].clone()
    outside = pool.clone()
    a = ops.decay_attention_step(q, k, v, decays(2), view)
    b = ops.decay_attention_step(q, k, v, decays(2), copy)
    assert torch.equal(view, copy)
    # sums of 24 products in another order: each off by (24 + 8) half steps of the sum of their magnitudes at most
    magnitude = torch.einsum("bhi,bhij->bhj", q.double().abs(), copy.double().abs()) * 24**-0.5
    assert ((a.double() - b.double()).abs() <= 2 * 32 * 2.0**-24 * magnitude).all()
    outside[1:5, :, :, 3:27] = copy
    assert torch.equal(pool, outside)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.decay_attention_step(q, k, v, decays(2), copy.transpose(-1, -2))


# ------------------------------------------------------------------------------------------ rotary


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,groups,dim,turned", [(1, 1, 1, 2, 2), (33, 4, 2, 64, 64), (700, 3, 1, 80, 40), (65, 2, 2, 7, 6), (129, 8, 8, 128, 96), (9, 2, 1, 16, 0), (1500, 2, 1, 4096, 4096)])
def test_rotary(dtype, interleaved, tokens, heads, groups, dim, turned):
    q, k = randn(2, tokens, heads, dim, dtype=dtype), randn(2, tokens, groups, dim, dtype=dtype)
    frequencies, scale = ops.rotary_frequencies(turned, scaling="parts", factor=4.0, original_tokens=2048)
    positions = torch.randint(0, 1 << 20, (2, 1), device=DEV) + torch.arange(tokens, device=DEV)
    q.requires_grad_(), k.requires_grad_()
    out = ops.rotary(q, k, positions, frequencies, interleaved=interleaved, scale=scale)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    grads = torch.autograd.grad(out, [q, k], [gq, gk])
    for y, x, inverse in [(out[0], q, False), (out[1], k, False), (grads[0], gq, True), (grads[1], gk, True)]:
        want = rotate(x.detach(), positions, frequencies, interleaved, scale, inverse)
        size = rotate_magnitude(x.detach().double().abs(), turned, interleaved, scale)
        # two products and their sum, cosine and sine good to 2 steps, the angle to 2^-24 half turns: pi 2^-24
        bound = size * 10 * 2.0**-24 + want.abs() * half_step(dtype) + torch.finfo(dtype).smallest_normal
        assert ((y.detach().double() - want).abs() <= bound).all()
        if turned < dim:
            assert torch.equal(y[..., turned:], x[..., turned:])


def rotate_magnitude(x, turned, interleaved, scale):
    y = x.clone()
    a, b = (slice(0, turned, 2), slice(1, turned, 2)) if interleaved else (slice(0, turned // 2), slice(turned // 2, turned))
    y[..., a] = y[..., b] = (x[..., a] + x[..., b]) * scale
    return y


def test_rotary_forms():
    frequencies, _ = ops.rotary_frequencies(32)
    q = randn(2, 3, 40, 4, 32, dtype=torch.bfloat16)
    positions = torch.arange(40, device=DEV)
    want, none = ops.rotary(q, None, positions, frequencies)
    assert none is None
    for p in (positions.int(), positions.float(), positions.expand(2, 3, 40), positions[None], positions[None, None].expand(2, 1, 40)):
        assert torch.equal(ops.rotary(q, None, p, frequencies)[0], want)
    moved = q.transpose(-2, -3).contiguous().transpose(-2, -3)
    assert torch.equal(ops.rotary(moved, None, positions, frequencies)[0], want)
    odd = torch.empty(2, 3, 40, 4, 33, device=DEV, dtype=torch.bfloat16)[..., 1:]
    odd.copy_(q)
    assert torch.equal(ops.rotary(odd, None, positions, frequencies)[0], want)
    wide = ops.rotary(q.permute(4, 0, 1, 2, 3).contiguous().permute(1, 2, 3, 4, 0), q[..., :1, :], positions, frequencies)
    assert torch.equal(wide[0], want) and torch.equal(wide[1], want[..., :1, :])
    assert ops.rotary(q[:, :, :0], None, positions[:0], frequencies)[0].shape == (2, 3, 0, 4, 32)
    # far positions, and times that are not whole
    far = torch.tensor([2**40 + 1, -7], device=DEV)
    x = randn(2, 1, 32)
    assert ((ops.rotary(x, None, far, frequencies)[0].double() - rotate(x, far, frequencies, False, 1.0)).abs() < 1e-3).all()
    times = torch.tensor([0.25, 1e4 + 0.5], device=DEV)
    assert ((ops.rotary(x, None, times, frequencies)[0].double() - rotate(x, times, frequencies, False, 1.0)).abs() < 1e-5).all()


def test_rotary_second_derivative():
    frequencies, _ = ops.rotary_frequencies(8)
    positions = torch.arange(5, device=DEV)
    x = randn(5, 2, 8).requires_grad_()
    y, _ = ops.rotary(x, None, positions, frequencies)
    (g,) = torch.autograd.grad((y**3).sum(), x, create_graph=True)
    (h,) = torch.autograd.grad((g * g.detach()).sum(), x)
    xd = x.detach().double().requires_grad_()
    angle = positions.double()[:, None, None] * frequencies
    c, s = angle.cos(), angle.sin()
    yd = torch.cat([xd[..., :4] * c - xd[..., 4:] * s, xd[..., :4] * s + xd[..., 4:] * c], -1)
    (gd,) = torch.autograd.grad((yd**3).sum(), xd, create_graph=True)
    (hd,) = torch.autograd.grad((gd * gd.detach()).sum(), xd)
    assert torch.allclose(h.double(), hd, rtol=1e-4, atol=1e-4)


# ------------------------------------------------------------------------------------------ norm


def exact_norm(tensors):
    return math.sqrt(sum((t.double() ** 2).sum().item() for t in tensors))


@pytest.mark.parametrize("sizes", [[1], [3, 0, 5], [65537, 7, 1 << 20], [11] * 1500, [5_000_011, 1]])
def test_norm_and_clipping(sizes):
    tensors = [randn(n, dtype=DTYPES[i % 3]) for i, n in enumerate(sizes)]
    want = exact_norm(tensors)
    norm = ops.global_norm(tensors)
    assert norm.shape == () and norm.dtype == torch.float32
    # squares and sums of up to 128 of them in fp32 (a thread's share of a chunk), fp64 beyond: off by 131 half steps, its root by half
    assert abs(norm.item() - want) <= want * 66 * 2.0**-24
    before = [t.clone() for t in tensors]
    assert torch.equal(ops.clip_global_norm_(tensors, want * 2), norm)
    assert all(torch.equal(a, b) for a, b in zip(tensors, before))
    assert torch.equal(ops.clip_global_norm_(tensors, want / 3), norm)
    factor = want / 3 / (want + 1e-6)
    for a, b in zip(tensors, before):
        exact = b.double() * factor
        assert ((a.double() - exact).abs() <= exact.abs() * (half_step(a.dtype) + 70 * 2.0**-24) + torch.finfo(a.dtype).smallest_normal).all()


def test_norm_of_extreme_values():
    for big in (1e30, 1e-30, 3e38, 1e-38):
        x = torch.full((70_000,), big, device=DEV)
        x[::2] = 0.0
        assert abs(ops.global_norm([x]).item() / exact_norm([x]) - 1) < 1e-6 or math.isinf(torch.tensor(exact_norm([x])).float().item())
    assert ops.global_norm([torch.zeros(100_000, device=DEV)]).item() == 0.0
    assert math.isinf(ops.global_norm([torch.tensor([math.inf, 1.0], device=DEV)]).item())
    bad = [torch.tensor([math.nan, 1.0], device=DEV)]
    assert math.isnan(ops.clip_global_norm_(bad, 1.0).item()) and torch.isnan(bad[0]).all()
    zero = [torch.zeros(5, device=DEV)]
    ops.clip_global_norm_(zero, 0.0)
    assert not zero[0].any()
    kept = randn(10)
    copy = kept.clone()
    ops.clip_global_norm_([kept], math.inf)
    assert torch.equal(kept, copy)


def test_norm_of_views():
    base = randn(64, 64, dtype=torch.bfloat16)
    part, turned, odd = base[1:40, 2:30], base.t(), base.flatten()[1:1001]
    for t in (part, turned, odd):
        assert abs(ops.global_norm([t]).item() - exact_norm([t])) <= exact_norm([t]) * 66 * 2.0**-24
    copy = base.clone()
    norm = exact_norm([part])
    ops.clip_global_norm_([part], norm / 2)
    copy[1:40, 2:30] *= 0.5
    assert torch.allclose(base.float(), copy.float(), rtol=2.0**-7, atol=0.0)
    # the same tensor twice counts once
    x = randn(100)
    want = exact_norm([x])
    assert abs(ops.global_norm([x, x]).item() - want) < 1e-4 * want
    ops.clip_global_norm_([x, x], want / 2)
    assert abs(exact_norm([x]) - want / 2) < 1e-4 * want


def test_training_step_together():
    """Positions, layer, loss, gradients, clipping, in the order of a training step, in fp32 against autograd in 64 bits."""
    b, t, h, groups, d = 2, 200, 4, 2, 16
    q, k, v = randn(b, t, h, d), randn(b, t, groups, d), randn(b, t, groups, d)
    g = decays(h)
    leaves = [q, k, v, g]
    frequencies, _ = ops.rotary_frequencies(d)
    positions = torch.arange(t, device=DEV)
    for x in leaves:
        x.requires_grad_()
    qr, kr = ops.rotary(q, k, positions, frequencies)
    o = ops.decay_attention(qr, kr, v, g)
    grads = list(torch.autograd.grad((o**2).mean(), leaves))
    norm = ops.clip_global_norm_(grads, 0.01)

    x = [y.detach().double().requires_grad_() for y in leaves]
    angle = positions.double()[:, None, None] * frequencies
    c, s = angle.cos(), angle.sin()
    turn = lambda y: torch.cat([y[..., : d // 2] * c - y[..., d // 2 :] * s, y[..., : d // 2] * s + y[..., d // 2 :] * c], -1)  # noqa: E731
    from sequence_reference import attention

    od, _ = attention(turn(x[0]), turn(x[1]), x[2], x[3], d**-0.5, torch.zeros(b, h, d, d, device=DEV, dtype=torch.float64), None)
    want = torch.autograd.grad((od**2).mean(), x)
    wn = math.sqrt(sum((y**2).sum().item() for y in want))
    assert abs(norm.item() - wn) <= 1e-5 * wn and wn > 0.01
    for y, z in zip(grads, want):
        z = z * (0.01 / (wn + 1e-6))
        assert (y.double() - z).norm() <= 1e-5 * z.norm()


def test_mll_gradient_clipped():
    x = torch.sort(torch.rand(500, device=DEV) * 10)[0]
    y = torch.sin(x)
    params = torch.tensor([1.0, 1.0], device=DEV)
    probes = torch.randint(0, 2, (500, 5), device=DEV).float() * 2 - 1
    kw = dict(cutoff=4.0, probes=probes, cg_iterations=30)
    a = gp.mll_gradient("rbf", x, params, 0.1, y, **kw)
    both = torch.cat([a.grad_params.flatten(), a.grad_sigma2.flatten()]).double()
    c = gp.mll_gradient("rbf", x, params, 0.1, y, max_grad_norm=both.norm().item() / 10, **kw)
    clipped = torch.cat([c.grad_params.flatten(), c.grad_sigma2.flatten()]).double()
    assert torch.allclose(clipped, both / 10, rtol=1e-4)


def test_refusals():
    q, k, v = (randn(5, 2, 8) for _ in range(3))
    g = decays(2)
    f, _ = ops.rotary_frequencies(8)
    p = torch.arange(5, device=DEV)
    bad = [
        lambda: ops.decay_attention(q.double(), k, v, g),
        lambda: ops.decay_attention(q, k.bfloat16(), v, g),
        lambda: ops.decay_attention(q, k, v, g.double()),
        lambda: ops.decay_attention(q, k, v, g[:1]),
        lambda: ops.decay_attention(q, k[:4], v, g),
        lambda: ops.decay_attention(q, k, v[:, :1], g),
        lambda: ops.decay_attention(q[:, :1], k, v, g[:1]),
        lambda: ops.decay_attention(q, k, v, g, path="tc"),
        lambda: ops.decay_attention(randn(5, 2, 129), randn(5, 2, 129), v, g),
        lambda: ops.decay_attention(q, k, v, g, initial_state=randn(2, 8, 9)),
        lambda: ops.decay_attention(q, k, v, g, initial_state=randn(2, 8, 8).bfloat16()),
        lambda: ops.decay_attention(q, k, v, g, sequence_starts=torch.tensor([0, 5], device=DEV)),
        lambda: ops.decay_attention(q[None], k[None], v[None], g, sequence_starts=starts_of([5])),
        lambda: ops.decay_attention(q.cpu(), k, v, g),
        lambda: ops.decay_attention(q, k, v, g.cpu()),
        lambda: ops.decay_attention_step(q, k, v, g, randn(4, 2, 8, 8)),
        lambda: ops.decay_attention_step(q, k, v, g, randn(5, 2, 8, 8).bfloat16()),
        lambda: ops.decay_attention_step(q, k, v, g, randn(1, 2, 8, 8).expand(5, 2, 8, 8)),
        lambda: ops.decay_attention_step(q, k, v, g, randn(5, 2, 8, 8), slots=torch.zeros(4, dtype=torch.int32, device=DEV)),
        lambda: ops.decay_attention_step(q.requires_grad_(), k, v, g, randn(5, 2, 8, 8)),
        lambda: ops.rotary(q, None, p[:4], f),
        lambda: ops.rotary(q, None, p.double(), f),
        lambda: ops.rotary(q, k[:, :, :4], p, f),
        lambda: ops.rotary(q, None, p, torch.cat([f, f])),
        lambda: ops.rotary(q, None, p, f.clone().requires_grad_()),
        lambda: ops.global_norm([q.double()]),
        lambda: ops.global_norm([q, torch.zeros(3)]),
        lambda: ops.clip_global_norm_([randn(10)[:6], torch.zeros(1, device=DEV).expand(4)], 1.0),
        lambda: ops.clip_global_norm_([randn(3).requires_grad_()], 1.0),
    ]
    x = randn(10)
    bad.append(lambda: ops.clip_global_norm_([x[:6], x[4:]], 1.0))
    for i, f_ in enumerate(bad):
        with pytest.raises(RuntimeError):
            f_()
            pytest.fail(f"call {i} was accepted")
    for f_ in (lambda: ops.global_norm([]), lambda: ops.clip_global_norm_([x], -1.0), lambda: ops.clip_global_norm_([x], math.nan),
               lambda: ops.decay_attention(q, k, v, g, path="nodes")):
        with pytest.raises(ValueError):
            f_()


def test_sequence_starts_that_decrease_stay_inside():
    """Sequences that overlap are not supported: their results are undefined, but nothing is read or written out of range, and
    other tensors keep their values."""
    t = 5000
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v = (randn(t, 2, 64, dtype=dtype).requires_grad_() for _ in range(3))
        g = decays(2).requires_grad_()
        guard = [torch.full((1 << 20,), 7.0, device=DEV) for _ in range(4)]
        for starts in ([0, t, 0, t, 0, t], [t, 0], [0, t, -3, t + 50, 10, 5, t]):
            o, s = ops.decay_attention(q, k, v, g, sequence_starts=torch.tensor(starts, dtype=torch.int32, device=DEV), return_state=True)
            torch.autograd.grad(o.sum() + s.sum(), [q, k, v, g])
        ops.check()
        assert all((x == 7.0).all() for x in guard)


@pytest.fixture
def short_waits():
    """A function that makes every hand-off wait of the tensor-core kernels give up at its first test."""
    from kernel_matmul_b200._lib import lib

    try:
        yield lambda: lib.km_selftest_set_wait_polls(0)
    finally:
        assert lib.km_selftest_set_wait_polls(-1) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,dim", [(100, 64), (1000, 128), (3000, 40)])
def test_attention_that_gives_up_reports_and_poisons_its_results(dtype, tokens, dim, short_waits):
    from kernel_matmul_b200._lib import lib

    q, k, v = (randn(2, tokens, 2, dim, dtype=dtype).requires_grad_() for _ in range(3))
    g = decays(2).requires_grad_()
    inputs = [q, k, v, g]
    o, s = ops.decay_attention(q, k, v, g, return_state=True)
    cotangents = [torch.randn_like(o), torch.randn_like(s)]
    want = torch.autograd.grad([o, s], inputs, cotangents, retain_graph=True)
    torch.cuda.synchronize()
    assert short_waits() == 0
    bad, bad_state = (x.detach() for x in ops.decay_attention(q, k, v, g, return_state=True))
    torch.cuda.synchronize()  # the launches end by themselves
    assert torch.isnan(bad).all() and torch.isnan(bad_state).all()
    with pytest.raises(ops.KernelGaveUpError, match="decay_attention"):
        ops.check()
    grads = torch.autograd.grad([o, s], inputs, cotangents, retain_graph=True)
    torch.cuda.synchronize()
    assert all(torch.isnan(x).all() for x in grads)
    with pytest.raises(ops.KernelGaveUpError):
        ops.check()
    assert lib.km_selftest_set_wait_polls(-1) == 0
    again = torch.autograd.grad([o, s], inputs, cotangents)
    ops.check()
    assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_training_step_in_a_graph():
    """Forward pass, gradients and clipping captured and replayed with other values in the same buffers."""
    q, k, v = (randn(2, 200, 2, 64, dtype=torch.bfloat16).requires_grad_() for _ in range(3))
    g = decays(2).requires_grad_()
    frequencies, _ = ops.rotary_frequencies(64)
    positions = torch.arange(200, device=DEV)

    def step():
        a, b = ops.rotary(q, k, positions, frequencies)
        o = ops.decay_attention(a, b, v, g)
        grads = list(torch.autograd.grad(o.float().square().mean(), [q, k, v, g]))
        return [o.detach(), *grads, ops.clip_global_norm_(grads, 0.01)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        with torch.no_grad():
            for t in (q, k, v):
                t.copy_(randn(*t.shape, dtype=t.dtype))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_gives_the_same_bits_again(dtype):
    """Sums are added up in a fixed order, and no hand-off between warps is left to chance."""
    cases = [(2, 3000, 4, 2, 128, 128), (1, 9000, 2, 2, 64, 128), (3, 700, 4, 4, 128, 64), (1, 5000, 3, 3, 64, 64)]
    for b, t, h, groups, dk, dv in cases:
        q, k, v = randn(b, t, h, dk, dtype=dtype), randn(b, t, groups, dk, dtype=dtype), randn(b, t, groups, dv, dtype=dtype)
        g, s0 = decays(h), randn(b, h, dk, dv)
        inputs = [x.requires_grad_() for x in (q, k, v, g, s0)]
        go, gs = randn(b, t, h, dv, dtype=dtype), randn(b, h, dk, dv)
        want = None
        for _ in range(8):
            o, s = ops.decay_attention(q, k, v, g, initial_state=s0, return_state=True)
            got = [o.detach(), s.detach(), *torch.autograd.grad([o, s], inputs, [go, gs])]
            assert want is None or all(torch.equal(a, c) for a, c in zip(got, want))
            want = got
