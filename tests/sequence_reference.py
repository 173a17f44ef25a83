"""The sequence operators in 64 bits, from their definitions, and how far results in fewer bits may be off.

A result is a sum of products of inputs.  With every rounding of a term off by at most half a step, the error is at most
(number of roundings a term goes through) x (half a step) x (sum of the terms' magnitudes), and that sum is the same
expression of the inputs' magnitudes: the reference is evaluated a second time on those."""
from __future__ import annotations

import torch

HALF = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention(q, k, v, log_decay, scale, initial, lengths):
    """``q (batch, tokens, heads, dk)`` etc. in 64 bits; ``lengths``: None, or those of the packed sequences of one batch."""
    group = q.shape[2] // k.shape[2]
    k, v = k.repeat_interleave(group, dim=2), v.repeat_interleave(group, dim=2)
    if lengths is None:
        o, s = _sequences(q, k, v, log_decay, scale, initial)
        return o, s
    outs, states, first = [], [], 0
    for i, n in enumerate(lengths):
        rows = slice(first, first + n)
        o, s = _sequences(q[:, rows], k[:, rows], v[:, rows], log_decay, scale, initial[i : i + 1])
        outs.append(o), states.append(s)
        first += n
    outs.append(torch.zeros_like(q[:, first:, :, :1]).expand(-1, -1, -1, v.shape[3]))
    return torch.cat(outs, 1), torch.cat(states)


def _sequences(q, k, v, log_decay, scale, initial):
    n = q.shape[1]
    t = torch.arange(n, device=q.device, dtype=torch.float64)
    distance = t[:, None] - t[None, :]
    g = log_decay.clamp_min(-1e30)  # (-inf * 0)
    weight = torch.exp(g[:, None, None] * distance.clamp_min(0.0)) * (distance >= 0)
    pairs = torch.einsum("bthi,bshi->bhts", q, k) * weight
    o = torch.einsum("bhts,bshj->bthj", pairs, v)
    o = o + torch.exp(g * (t[:, None] + 1.0))[None, :, :, None] * torch.einsum("bthi,bhij->bthj", q, initial)
    rest = torch.exp(g * (n - 1.0 - t[:, None]))
    s = torch.exp(g * float(n))[None, :, None, None] * initial + torch.einsum("bthi,th,bthj->bhij", k, rest, v)
    return o * scale, s


def attention_with_scales(inputs, scale, lengths, cotangents=None):
    """Results (and with ``cotangents`` for the output and the state also the gradients of all inputs) and the sums of their terms'
    magnitudes.  ``inputs``: dict of q, k, v, log_decay, initial in 64 bits."""
    out = []
    for f in (lambda x: x, torch.abs):
        x = {n: (f(t) if n != "log_decay" else t).detach().requires_grad_(cotangents is not None) for n, t in inputs.items()}
        o, s = attention(x["q"], x["k"], x["v"], x["log_decay"], scale, x["initial"], lengths)
        r = {"o": o.detach(), "state": s.detach()}
        if cotangents is not None:
            grads = torch.autograd.grad([o, s], list(x.values()), [f(c) for c in cotangents])
            r.update({"d" + n: g for n, g in zip(x, grads)})
        out.append(r)
    return out


def tolerance(name, value, magnitude, dtype, tokens, dk, dv, group):
    """Bound on the error of result ``name`` for operands of type ``dtype``: sums of products in fp32 (a term is rounded in the
    dot products, in its decay -- whose exponent, up to 40 where the term counts, is rounded to fp32 -- in the sums over tokens and over a
    group's heads, and a few more times); 16-bit operands of the second product round a term once more (P, or the state), and
    the result is rounded to its type.  States of 16-bit operands are sums of decayed keys held in two parts: 2^-17 and, below
    fp16's range, 2^-25 absolute."""
    sums = (dk + dv + tokens + group + 96) * 2.0**-24
    if dtype == torch.float32 or name == "dlog_decay":
        return magnitude * sums + 1e-30
    if name in ("state", "dinitial"):
        return magnitude * (sums + 2.0**-17) + tokens * 2.0**-23
    return magnitude * (sums + half_step(dtype) * 1.01) + value.abs() * half_step(dtype) + torch.finfo(dtype).smallest_normal


def rotate(x, positions, frequencies, interleaved, scale, inverse=False):
    """``x (.., tokens, heads, dim)`` in 64 bits."""
    r = 2 * frequencies.shape[0]
    angle = positions.double()[..., None, None] * frequencies.double()
    c, s = angle.cos() * scale, angle.sin() * scale * (-1.0 if inverse else 1.0)
    x = x.double()
    y = x.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., first] * s + x[..., second] * c
    return y
