"""The sequence operators, as cases to time and compare.

``rotary``     ``ops.rotary``: rotary positions of queries and keys, with ``grad`` also back through them
``attention``  ``ops.decay_attention``: linear attention with a decay for each head over whole
               sequences, with ``grad`` also the gradients of everything that can have one
``step``       ``ops.decay_attention_step``: one more token for each of many sequences whose states
               live in a pool
``clip``       ``ops.clip_global_norm_``: norm over many gradients, and clipping to it

Head sizes, token counts and types are generic.  Log decays are the slopes ``-2^(-8 (h + 1) / H)``, from
a memory of one token to one of some hundreds, or none at all.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # One new token of each of eight sequences on its way into the step below: launch and host time.
        dict(name="rotary_token", kind="rotary", batch=8, tokens=1, q_heads=16, k_heads=16, dim=64, rotary_dim=64, interleaved=False,
             scaling="none", dtype="bfloat16", grad=False),
        # A prompt of a long context whose frequencies are scaled by parts, grouped key heads.
        dict(name="rotary_prompt", kind="rotary", batch=2, tokens=8192, q_heads=32, k_heads=8, dim=128, rotary_dim=128,
             interleaved=False, scaling="parts", dtype="bfloat16", grad=False),
        # Training on ragged lengths, interleaved pairs, half of each head rotated, in fp16.
        dict(name="rotary_partial_train", kind="rotary", batch=3, tokens=2047, q_heads=12, k_heads=12, dim=80, rotary_dim=40,
             interleaved=True, scaling="linear", dtype="float16", grad=True),
        # Short requests packed into one batch, rows left over behind them, states kept for the tokens that follow.
        dict(name="attention_packed_short", kind="attention", batch=0, tokens=777, sequences=6, tail=13, heads=8, kv_heads=8, dk=64,
             dv=64, decay="slopes", dtype="float16", state=True, grad=False),
        # One long prompt: all the parallelism is in the heads and along the prompt.
        dict(name="attention_prompt", kind="attention", batch=1, tokens=16384, sequences=0, tail=0, heads=16, kv_heads=16, dk=128,
             dv=128, decay="slopes", dtype="bfloat16", state=True, grad=False),
        # Many long documents packed, four query heads to one key head, odd lengths.
        dict(name="attention_packed_long", kind="attention", batch=0, tokens=32749, sequences=17, tail=0, heads=32, kv_heads=8,
             dk=128, dv=128, decay="slopes", dtype="bfloat16", state=False, grad=False),
        # A training step's forward and backward pass, with the gradient of the decays.
        dict(name="attention_train", kind="attention", batch=4, tokens=4096, sequences=0, tail=0, heads=16, kv_heads=16, dk=128,
             dv=128, decay="slopes", dtype="bfloat16", state=False, grad=True),
        # The same in fp32 on odd sizes with a state carried between segments, the precision of the other operators here.
        dict(name="attention_train_f32", kind="attention", batch=2, tokens=1001, sequences=0, tail=0, heads=6, kv_heads=3, dk=40,
             dv=72, decay="slopes", dtype="float32", state=True, grad=True),
        # A single user's next token.
        dict(name="step_single", kind="step", rows=1, pool=1, heads=16, kv_heads=16, dk=64, dv=64, decay="slopes", dtype="bfloat16"),
        # The next token of a full serving batch, states in a larger pool.
        dict(name="step_batch", kind="step", rows=192, pool=256, heads=32, kv_heads=8, dk=128, dv=128, decay="slopes",
             dtype="bfloat16"),
        # Gradients of a few kernel parameters and a small network, below the bound: the norm alone.
        dict(name="clip_small", kind="clip", tensors=14, elements=50021, dtype="float32", clipped=False),
        # Gradients of a large network, matrices in bf16 and vectors in fp32, above the bound.
        dict(name="clip_large", kind="clip", tensors=290, elements=420_000_000, dtype="bfloat16", clipped=True),
    ]


def _spread(rng, low, high):
    """A whole number between ``low`` and ``high``, uniform in its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["rotary", "attention", "attention", "attention", "step", "clip"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    decay = rng.choice(["slopes", "slopes", "none"])
    size = rng.choice([16, 32, 40, 64, 64, 72, 96, 128, 128, rng.randint(8, 128)])
    if kind == "rotary":
        dim = max(2, size)
        heads = _spread(rng, 1, 8)
        group = rng.choice([1, 1, 2, 4])
        batch = rng.randint(1, 4)
        tokens = _spread(rng, 1, 100_000_000 // (batch * heads * (group + 1) * dim * 2))
        return dict(kind=kind, batch=batch, tokens=min(tokens, 16384), q_heads=heads * group, k_heads=heads, dim=dim,
                    rotary_dim=rng.choice([dim // 2 * 2, max(2, dim // 4 * 2)]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "parts"]), dtype=dtype, grad=rng.random() < 0.5)
    if kind == "attention":
        grad = rng.random() < 0.5
        kv_heads = _spread(rng, 1, 16)
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        batch = rng.choice([0, 1, 2, 4])
        budget = (33_000_000 if grad else 130_000_000) // (4 if dtype == "float32" else 1)
        tokens = _spread(rng, 1, min(32768 if batch < 2 else 8192, budget // (heads * 128 * max(batch, 1))))
        sequences = rng.randint(1, min(24, max(1, tokens // 8))) if batch == 0 else 0
        return dict(kind=kind, batch=batch, tokens=tokens, sequences=sequences, tail=rng.randint(0, tokens // 8) if batch == 0 else 0,
                    heads=heads, kv_heads=kv_heads, dk=size, dv=rng.choice([size, size, rng.randint(8, 128)]), decay=decay, dtype=dtype,
                    state=rng.random() < 0.5, grad=grad)
    if kind == "step":
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        rows = _spread(rng, 1, 192)
        return dict(kind=kind, rows=rows, pool=rows + rng.randint(0, 64), heads=kv_heads * rng.choice([1, 1, 2]), kv_heads=kv_heads,
                    dk=size, dv=rng.choice([size, rng.randint(8, 128)]), decay=decay, dtype=dtype)
    tensors = _spread(rng, 1, 400)
    return dict(kind=kind, tensors=tensors, elements=_spread(rng, max(tensors, 1000), 400_000_000), dtype=dtype,
                clipped=rng.random() < 0.5)


# ------------------------------------------------------------------------------------ inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _frequencies(case):
    """Angular frequencies of the pairs in 64 bits, and the factor on the rotated values."""
    half = case["rotary_dim"] // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    if case["scaling"] == "linear":
        return (freq / 4.0).cuda(), 1.0
    if case["scaling"] == "parts":
        # long waves are stretched eightfold, short ones kept, the rest in between
        turns = 4096.0 * freq / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return (freq / 8.0 * (1.0 - keep) + freq * keep).cuda(), 0.1 * math.log(8.0) + 1.0
    return freq.cuda(), 1.0


def _log_decay(case):
    heads = case["heads"]
    if case["decay"] == "none":
        return torch.zeros(heads, device="cuda")
    return -(2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float32, device="cuda") / heads))


def _sequence_lengths(case, seed):
    total, count = case["tokens"] - case["tail"], case["sequences"]
    rng = random.Random(seed)
    cuts = sorted(rng.randint(0, total) for _ in range(count - 1))
    if count >= 4:
        cuts[1] = cuts[0]  # an empty sequence among them
    return [b - a for a, b in zip([0, *cuts], [*cuts, total])]


def _tensor_sizes(case):
    """Sizes of a network's tensors: matrices that grow, and a short vector behind every third."""
    count, total = case["tensors"], case["elements"]
    weights = [0.001 if i % 3 == 2 else 1.0 + (i % 7) for i in range(count)]
    sizes = [max(1, int(total * w / sum(weights))) for w in weights]
    return [n | 1 if i % 3 == 2 else n for i, n in enumerate(sizes)]


def _wide(case):
    """The types of a network's tensors: the short vectors are fp32."""
    return [torch.float32 if i % 3 == 2 else DTYPES[case["dtype"]] for i in range(case["tensors"])]


def prepare(case, seed):
    gen = _generator(seed)
    kind = case["kind"]
    dtype = DTYPES[case["dtype"]]
    if kind == "rotary":
        shape = (case["batch"], case["tokens"])
        q = _normal(gen, (*shape, case["q_heads"], case["dim"]), dtype)
        k = _normal(gen, (*shape, case["k_heads"], case["dim"]), dtype)
        first = torch.randint(0, 100_000, (case["batch"], 1), generator=gen, device="cuda")
        frequencies, scale = _frequencies(case)
        state = dict(case=case, q=q, k=k, positions=first + torch.arange(case["tokens"], device="cuda"), frequencies=frequencies,
                     scale=scale)
        if case["grad"]:
            state.update(q=q.requires_grad_(), k=k.requires_grad_(), gq=_normal(gen, q.shape, dtype), gk=_normal(gen, k.shape, dtype))
        return state
    if kind == "attention":
        lead = (case["tokens"],) if case["batch"] == 0 else (case["batch"], case["tokens"])
        count = case["sequences"] if case["batch"] == 0 else case["batch"]
        state = dict(case=case, q=_normal(gen, (*lead, case["heads"], case["dk"]), dtype),
                     k=_normal(gen, (*lead, case["kv_heads"], case["dk"]), dtype),
                     v=_normal(gen, (*lead, case["kv_heads"], case["dv"]), dtype), log_decay=_log_decay(case), initial=None,
                     starts=None, lengths=None)
        if case["batch"] == 0:
            lengths = _sequence_lengths(case, seed)
            state.update(lengths=lengths, starts=torch.tensor([0, *lengths]).cumsum(0).to(torch.int32).cuda())
        if case["state"]:
            state["initial"] = _normal(gen, (count, case["heads"], case["dk"], case["dv"]), torch.float32, 3.0)
        if case["grad"]:
            for name in ("q", "k", "v", "log_decay", "initial"):
                if state[name] is not None:
                    state[name].requires_grad_()
            state["go"] = _normal(gen, (*lead, case["heads"], case["dv"]), dtype)
            state["gs"] = _normal(gen, (count, case["heads"], case["dk"], case["dv"]), torch.float32, 0.1) if case["state"] else None
        return state
    if kind == "step":
        rows, heads = case["rows"], case["heads"]
        return dict(case=case, q=_normal(gen, (rows, heads, case["dk"]), dtype), k=_normal(gen, (rows, case["kv_heads"], case["dk"]), dtype),
                    v=_normal(gen, (rows, case["kv_heads"], case["dv"]), dtype), log_decay=_log_decay(case),
                    pool=_normal(gen, (case["pool"], heads, case["dk"], case["dv"]), torch.float32, 3.0),
                    slots=torch.randperm(case["pool"], generator=gen, device="cuda")[:rows].to(torch.int32))
    # gradients are views of one bucket for each type, every one on a boundary of 128 elements
    sizes, wide = _tensor_sizes(case), _wide(case)
    room = [-(-n // 128) * 128 for n in sizes]
    buckets = {t: torch.zeros(sum(r for r, w in zip(room, wide) if w == t), dtype=t, device="cuda") for t in dict.fromkeys(wide)}
    tensors, used = [], dict.fromkeys(buckets, 0)
    for n, r, t in zip(sizes, room, wide):
        tensors.append(buckets[t][used[t] : used[t] + n].copy_(_normal(gen, (n,), t, 0.01)))
        used[t] += r
    norm = 0.01 * math.sqrt(sum(sizes))
    return dict(case=case, tensors=tensors, buckets=list(buckets.values()), max_norm=norm * (0.5 if case["clipped"] else 2.0))


# ------------------------------------------------------------------------------------ plain forms


def _rotate(x, cos, sin, case, scale):
    """Plain rotary positions of ``x (batch, tokens, heads, dim)`` in 32 bits."""
    r = case["rotary_dim"]
    y, rest = x.float()[..., :r], x.float()[..., r:]
    a, b = (y[..., 0::2], y[..., 1::2]) if case["interleaved"] else (y[..., : r // 2], y[..., r // 2 :])
    c, s = cos[:, :, None] * scale, sin[:, :, None] * scale
    u, w = a * c - b * s, a * s + b * c
    y = torch.stack([u, w], dim=-1).flatten(-2) if case["interleaved"] else torch.cat([u, w], dim=-1)
    return torch.cat([y, rest], dim=-1).to(x.dtype)


def _plain_rotary(state):
    case, scale = state["case"], state["scale"]
    angle = state["positions"].double()[..., None] * state["frequencies"]
    cos, sin = angle.cos().float(), angle.sin().float()
    out = {"q": _rotate(state["q"].detach(), cos, sin, case, scale), "k": _rotate(state["k"].detach(), cos, sin, case, scale)}
    if case["grad"]:  # the transposed rotation
        out["dq"], out["dk"] = _rotate(state["gq"], cos, -sin, case, scale), _rotate(state["gk"], cos, -sin, case, scale)
    return out


def _chunked(q, k, v, log_decay, scale, state, chunk=128):
    """Linear attention with decay over ``q, k (batch, heads, tokens, dk)``, ``v`` alike, from ``state``: chunks one after
    the other, the tokens inside one against each other through a masked matrix."""
    outs = []
    g = log_decay[:, None, None]
    for first in range(0, q.shape[2], chunk):
        qc, kc, vc = (x[:, :, first : first + chunk] for x in (q, k, v))
        n = qc.shape[2]
        t = torch.arange(n, device=q.device, dtype=torch.float32)
        distance = t[:, None] - t[None, :]
        weight = torch.where(distance >= 0, torch.exp(g * distance.clamp_min(0.0)), torch.zeros((), device=q.device))
        inside = ((qc @ kc.transpose(-1, -2)) * weight) @ vc
        before = torch.exp(g * (t[:, None] + 1.0)) * (qc @ state)
        outs.append((inside + before) * scale)
        state = torch.exp(g * n) * state + (kc * torch.exp(g * (n - 1.0 - t[:, None]))).transpose(-1, -2) @ vc
    return (torch.cat(outs, dim=2) if outs else q.new_zeros(*q.shape[:3], v.shape[-1])), state


def _plain_attention(state):
    case = state["case"]
    scale = case["dk"] ** -0.5
    names = [n for n in ("q", "k", "v", "log_decay", "initial") if state[n] is not None]
    with torch.set_grad_enabled(case["grad"]):
        x = {n: state[n].detach().float().requires_grad_(case["grad"]) for n in names}
        group = case["heads"] // case["kv_heads"]
        k, v = (x[n].repeat_interleave(group, dim=-2) for n in ("k", "v"))
        q = x["q"]
        count = case["sequences"] if case["batch"] == 0 else case["batch"]
        initial = x.get("initial")
        if initial is None:
            initial = torch.zeros(count, case["heads"], case["dk"], case["dv"], device="cuda")
        if case["batch"] == 0:
            outs, states, first = [], [], 0
            for i, n in enumerate(state["lengths"]):
                part = [y[first : first + n].transpose(0, 1)[None] for y in (q, k, v)]
                o, s = _chunked(*part, x["log_decay"], scale, initial[i : i + 1])
                outs.append(o[0].transpose(0, 1))
                states.append(s)
                first += n
            outs.append(torch.zeros(case["tokens"] - first, case["heads"], case["dv"], device="cuda"))
            o, s = torch.cat(outs), torch.cat(states)
        else:
            o, s = _chunked(*(y.transpose(1, 2) for y in (q, k, v)), x["log_decay"], scale, initial)
            o = o.transpose(1, 2)
        out = {"o": o.detach().to(state["q"].dtype)}
        if case["state"]:
            out["state"] = s.detach()
        if case["grad"]:
            results, cotangents = ([o, s], [state["go"].float(), state["gs"]]) if case["state"] else ([o], [state["go"].float()])
            for n, grad in zip(names, torch.autograd.grad(results, [x[n] for n in names], cotangents)):
                out["d" + n] = grad.to(state[n].dtype)
    return out


def _plain_step(state):
    case = state["case"]
    slots = state["slots"].long()
    group = case["heads"] // case["kv_heads"]
    q = state["q"].float()
    k, v = (state[n].float().repeat_interleave(group, dim=1) for n in ("k", "v"))
    s = torch.exp(state["log_decay"])[:, None, None] * state["pool"][slots] + k[..., :, None] * v[..., None, :]
    state["pool"][slots] = s
    o = (q[..., :, None] * s).sum(dim=-2) * case["dk"] ** -0.5
    return {"o": o.to(state["q"].dtype), "pool": state["pool"]}


def _plain_clip(state):
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for t in state["tensors"]:
        total += t.float().square().sum(dtype=torch.float64)
    norm = total.sqrt()
    factor = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    for t in state["tensors"]:
        t.copy_(t.float() * factor)
    return {"norm": norm.float(), "buckets": state["buckets"]}


def run(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "clip" and case["clipped"]:
        # a bound that tightens from pass to pass: gradients that are within it already would not be clipped again
        state["max_norm"] *= 0.995
    if not own:
        return {"rotary": _plain_rotary, "attention": _plain_attention, "step": _plain_step, "clip": _plain_clip}[kind](state)
    from kernel_matmul_b200 import ops

    if kind == "rotary":
        q, k = ops.rotary(state["q"], state["k"], state["positions"], state["frequencies"], interleaved=case["interleaved"],
                          scale=state["scale"])
        out = {"q": q.detach(), "k": k.detach()}
        if case["grad"]:
            out["dq"], out["dk"] = torch.autograd.grad([q, k], [state["q"], state["k"]], [state["gq"], state["gk"]])
        return out
    if kind == "attention":
        result = ops.decay_attention(state["q"], state["k"], state["v"], state["log_decay"], initial_state=state["initial"],
                                     sequence_starts=state["starts"], return_state=case["state"])
        results = list(result) if case["state"] else [result]
        out = dict(zip(("o", "state"), (r.detach() for r in results)))
        if case["grad"]:
            names = [n for n in ("q", "k", "v", "log_decay", "initial") if state[n] is not None]
            grads = torch.autograd.grad(results, [state[n] for n in names], [state["go"], state["gs"]][: len(results)])
            out.update({"d" + n: grad for n, grad in zip(names, grads)})
        return out
    if kind == "step":
        o = ops.decay_attention_step(state["q"], state["k"], state["v"], state["log_decay"], state["pool"], slots=state["slots"])
        return {"o": o, "pool": state["pool"]}
    return {"norm": ops.clip_global_norm_(state["tensors"], state["max_norm"]), "buckets": state["buckets"]}


# ------------------------------------------------------------------------------------ floors


def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "float32" else 2
    if kind == "rotary":
        rows = case["batch"] * case["tokens"]
        heads, passes = case["q_heads"] + case["k_heads"], 2 if case["grad"] else 1
        return {"bytes": passes * (2 * rows * heads * case["dim"] * size) + rows * 8 + case["rotary_dim"] * 4,
                "flops": passes * 3 * rows * heads * case["rotary_dim"]}
    if kind == "attention":
        rows = case["tokens"] * max(case["batch"], 1)
        q, k = rows * case["heads"] * case["dk"] * size, rows * case["kv_heads"] * case["dk"] * size
        v, o = rows * case["kv_heads"] * case["dv"] * size, rows * case["heads"] * case["dv"] * size
        state = (case["sequences"] or case["batch"]) * case["heads"] * case["dk"] * case["dv"] * 4 if case["state"] else 0
        product = 2 * rows * case["heads"] * case["dk"] * case["dv"]
        # forward: q, k, v, states in; o, states out.  Backward: q, k, v, do, states in; dq, dk, dv, state gradient out.
        return {"bytes": q + k + v + o + 2 * state + (2 * (q + k + v) + o + 3 * state if case["grad"] else 0),
                "flops": product * (2 + (5 if case["grad"] else 0))}
    if kind == "step":
        states = case["rows"] * case["heads"] * case["dk"] * case["dv"]
        vectors = case["rows"] * (case["heads"] + case["kv_heads"]) * (case["dk"] + case["dv"])
        return {"bytes": 2 * states * 4 + vectors * size, "flops": 5 * states}
    sizes = _tensor_sizes(case)
    total = sum(n * t.itemsize for n, t in zip(sizes, _wide(case)))
    elements = sum(sizes)
    return {"bytes": total * (3 if case["clipped"] else 1), "flops": elements * (3 if case["clipped"] else 2)}


# ------------------------------------------------------------------------------------ 64 bits


def _exact_rotary(state):
    case, r = state["case"], state["case"]["rotary_dim"]
    phase = torch.polar(torch.full((), float(state["scale"]), dtype=torch.float64, device="cuda").expand(*state["positions"].shape, r // 2),
                        state["positions"].double()[..., None] * state["frequencies"])[:, :, None]

    def turn(x, factor):
        x = x.detach().double()
        pairs = x[..., :r].unflatten(-1, (r // 2, 2) if case["interleaved"] else (2, r // 2))
        last = -1 if case["interleaved"] else -2
        z = torch.complex(pairs.select(last, 0), pairs.select(last, 1)) * factor
        return torch.cat([torch.stack([z.real, z.imag], dim=last).flatten(-2), x[..., r:]], dim=-1)

    out = {"q": turn(state["q"], phase), "k": turn(state["k"], phase)}
    if case["grad"]:
        out.update(dq=turn(state["gq"], phase.conj()), dk=turn(state["gk"], phase.conj()))
    return out


def _exact_head(q, k, v, g, initial, go, gs, scale, out):
    """One head of one sequence through the whole matrix ``W[t, s] = e^(g (t - s)) q_t . k_s`` in blocks of rows."""
    n = q.shape[0]
    t = torch.arange(n, device=q.device, dtype=torch.float64)
    decay = torch.exp(g * (t + 1.0))[:, None]
    out["o"][:] = decay * (q @ initial) * scale
    rest = torch.exp(g * (n - 1.0 - t))[:, None]
    carried = torch.exp(g * n)
    out["state"][:] = carried * initial + (k * rest).T @ v
    if go is not None:
        go = go * scale
        out["dq"][:] = decay * (go @ initial.T)
        out["dk"] += rest * (v @ gs.T)
        out["dv"] += rest * (k @ gs)
        out["dinitial"][:] = (decay * q).T @ go + carried * gs
        dg = (decay * (t + 1.0)[:, None] * (q @ initial) * go).sum() + n * carried * (initial * gs).sum()
        dg = dg + (((n - 1.0 - t)[:, None] * rest * k) @ gs * v).sum()
    for a in range(0, n, 2048):
        b = min(a + 2048, n)
        distance = t[a:b, None] - t[None, :b]
        mask = torch.where(distance >= 0, torch.exp(g * distance.clamp_min(0.0)), torch.zeros((), dtype=torch.float64, device=q.device))
        weights = mask * (q[a:b] @ k[:b].T)
        out["o"][a:b] += weights @ v[:b] * scale
        if go is not None:
            back = go[a:b] @ v[:b].T
            dg = dg + (distance * weights * back).sum()
            out["dv"][:b] += weights.T @ go[a:b]
            back *= mask
            out["dq"][a:b] += back @ k[:b]
            out["dk"][:b] += back.T @ q[a:b]
    if go is not None:
        out["dlog_decay"] += dg


def _exact_attention(state):
    case = state["case"]
    grad = case["grad"]
    packed = case["batch"] == 0
    x = {n: state[n].detach().double() for n in ("q", "k", "v", "log_decay")}
    if packed:
        x.update({n: x[n][None] for n in ("q", "k", "v")})
    count = case["sequences"] if packed else case["batch"]
    shape = (count, case["heads"], case["dk"], case["dv"])
    zeros = dict(dtype=torch.float64, device="cuda")
    initial = torch.zeros(shape, **zeros) if state["initial"] is None else state["initial"].detach().double()
    go = state["go"].double().reshape(*x["q"].shape[:3], case["dv"]) if grad else None
    gs = (torch.zeros(shape, **zeros) if state["gs"] is None else state["gs"].double()) if grad else None
    out = {"o": torch.zeros(*x["q"].shape[:3], case["dv"], **zeros), "state": torch.zeros(shape, **zeros)}
    if grad:
        out.update({"d" + n: torch.zeros_like(x[n]) for n in x}, dinitial=torch.zeros(shape, **zeros))
    lengths = state["lengths"] if packed else [case["tokens"]] * count
    first = 0
    for i, n in enumerate(lengths):
        row, rows = (0, slice(first, first + n)) if packed else (i, slice(0, n))
        for h in range(case["heads"]):
            kv = h // (case["heads"] // case["kv_heads"])
            heads = {"q": h, "o": h, "dq": h, "k": kv, "v": kv, "dk": kv, "dv": kv}
            views = {key: out[key][row, rows, head] for key, head in heads.items() if key in out}
            views.update({key: out[key][i, h] for key in ("state", "dinitial") if key in out})
            if grad:
                views["dlog_decay"] = out["dlog_decay"][h : h + 1]
            _exact_head(x["q"][row, rows, h], x["k"][row, rows, kv], x["v"][row, rows, kv], x["log_decay"][h], initial[i, h],
                        go[row, rows, h] if grad else None, gs[i, h] if grad else None, case["dk"] ** -0.5, views)
        first += n
    if packed:
        out.update({n: out[n][0] for n in ("o", "dq", "dk", "dv") if n in out})
    if not case["state"]:
        out = {n: y for n, y in out.items() if n not in ("state", "dinitial")}
    return out


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return _exact_rotary(state)
    if kind == "attention":
        out = _exact_attention(state)
        order = ["o", "state", "dq", "dk", "dv", "dlog_decay", "dinitial"]
        return {n: out[n] for n in order if n in out}
    if kind == "step":
        slots = state["slots"].long()
        q, k, v = (state[n].double() for n in ("q", "k", "v"))
        head = torch.arange(case["heads"], device="cuda") // (case["heads"] // case["kv_heads"])
        pool = state["pool"].double()
        for row, slot in enumerate(slots.tolist()):
            pool[slot] = pool[slot] * state["log_decay"].double().exp()[:, None, None] + torch.einsum("hi,hj->hij", k[row, head], v[row, head])
        return {"o": torch.einsum("bhi,bhij->bhj", q, pool[slots]) / math.sqrt(case["dk"]), "pool": pool}
    bound = state["max_norm"] * (0.995 if case["clipped"] else 1.0)
    norm = math.sqrt(sum(torch.linalg.vector_norm(t.double()).item() ** 2 for t in state["tensors"]))
    factor = min(1.0, bound / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda"), "buckets": [b.double() * factor for b in state["buckets"]]}
