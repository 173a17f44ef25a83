"""Sequence operators under forms of calls of PyTorch's that would go past their kernels."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from kernel_matmul_b200 import ops  # noqa: E402

DEV = "cuda"


def calls():
    q, k, v = (torch.randn(5, 2, 8, device=DEV) for _ in range(3))
    g = torch.tensor([-0.5, -0.1], device=DEV)
    f, _ = ops.rotary_frequencies(8)
    p = torch.arange(5, device=DEV)
    s = torch.randn(5, 2, 8, 8, device=DEV)
    return {
        "rotary": (lambda x: ops.rotary(x, None, p, f)[0], q),
        "attention": (lambda x: ops.decay_attention(x, k, v, g), q),
        "step": (lambda x: ops.decay_attention_step(x, k, v, g, s), q),
        "norm": (lambda x: ops.global_norm([x, k]), q),
        "clip": (lambda x: ops.clip_global_norm_([x, k], 1.0), q),
    }


@pytest.mark.parametrize("name", ["rotary", "attention", "step", "norm", "clip"])
def test_recordings_without_the_kernels_are_refused(name):
    """torch.jit.trace and make_fx see the allocation of a result and not the kernel that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    f, x = calls()[name]
    with pytest.raises(RuntimeError, match="record"):
        torch.jit.trace(f, (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="record"):
        make_fx(f)(x)
    f(x)  # (and nothing of that stays)


@pytest.mark.parametrize("name", ["rotary", "attention", "step", "norm", "clip"])
def test_forward_mode_and_transforms_are_refused(name):
    f, x = calls()[name]
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError):
            f(dual)
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(torch.stack([x, x]))
    f(x)


def test_saved_tensors_may_be_moved_away():
    """Hooks on what the graph saves: the backward pass works on what they give back."""
    q, k, v = (torch.randn(150, 2, 64, device=DEV, dtype=torch.bfloat16).requires_grad_() for _ in range(3))
    g = torch.tensor([-0.5, -0.1], device=DEV).requires_grad_()
    f, _ = ops.rotary_frequencies(64)
    p = torch.arange(150, device=DEV)

    def step():
        a, b = ops.rotary(q, k, p, f)
        return torch.autograd.grad(ops.decay_attention(a, b, v, g).float().square().sum(), [q, k, v, g])

    want = step()
    with torch.autograd.graph.save_on_cpu():
        got = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_gradient_of_a_norm_is_refused_and_not_left_out():
    x, y = torch.randn(10, device=DEV).requires_grad_(), torch.randn(3, device=DEV)
    norm = ops.global_norm([x, y])
    assert abs(norm.item() - torch.cat([x, y]).norm().item()) < 1e-5
    with pytest.raises(RuntimeError, match="no gradient"):
        (x.sum() + norm).backward()
    with torch.no_grad():
        assert not ops.global_norm([x]).requires_grad
    assert not ops.global_norm([x.detach(), y]).requires_grad


def test_a_tensor_that_is_listed_twice_counts_once():
    """Whatever stands between, another view from the same element on among it."""
    base = torch.randn(20, 36, device=DEV)
    square = lambda t: t.double().square().sum().item()  # noqa: E731
    for views, once in (([base, base[:10], base], [base, base[:10]]), ([base, base.view(-1), base[:1], base, base[:1], base.view(-1)], [base, base, base[:1]]),
                        ([base[:, 3:], base[:2, 3:5], base[:, 3:], base[5:]], [base[:, 3:], base[:2, 3:5], base[5:]])):
        want = sum(square(t) for t in once) ** 0.5
        # squares and sums of up to 128 of them in fp32, fp64 beyond: off by 131 half steps, its root by half
        assert abs(ops.global_norm(views).item() - want) <= want * 66 * 2.0**-24


# ------------------------------------------------------------------------------------------ views of one buffer


def clipped_apart(views, base):
    """Clipping ``views`` of ``base`` gives what clipping copies of them gives, and leaves the rest of ``base``."""
    copies = [t.clone() for t in views]
    outside = base.clone()
    norm = ops.clip_global_norm_(copies, 0.5)
    got = ops.clip_global_norm_(views, 0.5)
    # (the copies lie elsewhere: sums in another order)
    assert abs(got.item() - norm.item()) <= 1e-5 * norm.item()
    for a, b in zip(views, copies):
        assert torch.allclose(a.float(), b.float(), rtol=2 * torch.finfo(a.dtype).eps, atol=0.0)
    mask = torch.zeros_like(base, dtype=torch.bool)
    flat = mask.flatten()
    for t in views:
        torch.as_strided(flat, t.size(), t.stride(), t.storage_offset() - base.storage_offset()).fill_(True)
    assert torch.equal(base.flatten()[~flat], outside.flatten()[~flat])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_slices_of_one_buffer_are_clipped(dtype):
    new = lambda *s: torch.randn(s, device=DEV).to(dtype)  # noqa: E731
    base = new(20, 36)
    clipped_apart(list(base.chunk(3, dim=1)), base)
    base = new(20, 36)
    clipped_apart([base[:, 24:], base[5:, :12], base[3:17, 12:20]], base)
    base = new(36, 20).t()
    clipped_apart([base[2:, :12], base[:2, 3:]], base.t())
    base = new(4, 6, 5, 8)
    clipped_apart([base[:, :3, :, 2:6], base[1:, 3:, 1:3], base[:, :3, :, 6:], base[2:, :3, :, :2]], base)
    base = new(100)
    clipped_apart([base[::2], base[1::2]], base)
    base = new(101)
    clipped_apart([base[::3], base[2::3], base[1:50:3]], base)


def test_slices_that_overlap_are_refused():
    base = torch.randn(20, 36, device=DEV)
    before = base.clone()
    line = base.flatten()
    for views in ([base[:, :13], base[:, 12:]], [base[:10], base[9:]], [base[:, :12], base[3:4]], [base[::2], base[2:3]], [base, base[:, 5:]],
                  [base, base.t()], [line[::2], line[::3]], [line[:1], line[0:700:5]]):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.clip_global_norm_(list(views), 0.5)
    assert torch.equal(base, before)
    assert abs(ops.global_norm([base, base[:, 5:]]).item() - math.sqrt(base.square().sum().item() + base[:, 5:].square().sum().item())) < 1e-3


# ------------------------------------------------------------------------------------------ bounds that are not finite


def test_an_infinite_bound_gives_what_the_formula_gives():
    x = torch.randn(10, device=DEV)
    kept = x.clone()
    ops.clip_global_norm_([x], math.inf)
    assert torch.equal(x, kept)
    x[3] = math.nan
    assert math.isnan(ops.clip_global_norm_([x], math.inf).item()) and x.isnan().all()  # inf / (nan + eps)
    y = torch.tensor([math.inf, 1.0], device=DEV)
    assert math.isinf(ops.clip_global_norm_([y], math.inf).item()) and y.isnan().all()  # inf / (inf + eps)
    y = torch.tensor([math.inf, 1.0], device=DEV)
    ops.clip_global_norm_([y], 1.0)  # 1 / inf = 0
    assert y[0].isnan() and y[1] == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_factors_below_the_range_of_fp32(dtype):
    x = (torch.randn(100_003, device=DEV) * 1e37).to(dtype)
    exact, norm = x.double(), x.double().norm().item()
    for bound in (1e3, 1.0, 1e-3):
        y = x.clone()
        ops.clip_global_norm_([y], bound, eps=0.0)
        want = exact * (bound / norm)
        assert bound / norm < 1e-36
        # the norm, the factor, two products and the result's rounding
        assert ((y.double() - want).abs() <= want.abs() * (70 * 2.0**-24 + torch.finfo(dtype).eps / 2) + 2.0**-149).all()
