"""Sequence operators: what their C entry points refuse before they launch anything."""
from __future__ import annotations

import ctypes

import pytest

from kernel_matmul_b200._lib import KmDecayProblem, KmView, lib

ANY = ctypes.c_void_p(4096)  # (never read: the call is refused)


def view(data=4096):
    return KmView(data=data, batch_stride=(0, 0, 0, 0), stride=(16, 1))


def refused(rc, text):
    assert rc != 0 and text in lib.km_last_error(), lib.km_last_error()


@pytest.mark.parametrize("missing", range(4))
def test_gradient_without_an_operand(missing):
    p = KmDecayProblem(dtype=0, out_dtype=0, reverse=0, path=0, sequences=1, tokens=8, groups=2, group=1, dk=16, dv=16, packed=0, states=0, scale=1.0)
    need = lib.km_decay_gradient_workspace_bytes(p)
    views = [view(None if i == missing else 4096) for i in range(4)]
    refused(lib.km_decay_gradient(p, *views, ANY, None, None, None, ANY, ANY, need, None), b"null pointer")


@pytest.mark.parametrize("missing", range(4))
def test_attention_without_an_operand(missing):
    p = KmDecayProblem(dtype=0, out_dtype=0, reverse=0, path=0, sequences=1, tokens=8, groups=2, group=1, dk=16, dv=16, packed=0, states=0, scale=1.0)
    views = [view(None if i == missing else 4096) for i in range(4)]
    refused(lib.km_decay_attention(p, *views, ANY, None, None, None, ANY, 0, None), b"null pointer")


def step(rows=1, pool=1, groups=1, group=1, states=4096, dv=16):
    v = view()
    return lib.km_decay_step(0, rows, pool, groups, group, 16, dv, v, v, v, v, ANY, view(states), 3, ANY, 1.0, None)


def test_step_without_states():
    refused(step(states=None), b"null pointer")


@pytest.mark.parametrize("rows, groups, group", [(2**30, 4, 1), (2**31 - 1, 2**16, 2**14), (2**31 - 1, 2**15, 2**15 + 1), (2**30, 2**15, 2**15), (2**31 - 1, 2**30, 1)])
def test_step_with_more_pairs_than_fit_a_launch(rows, groups, group):
    for dv in (16, 127):  # (127: four CTAs to a pair)
        refused(step(rows, 1, groups, group, dv=dv), b"2^31")


@pytest.mark.parametrize("rows, groups, group, dim", [(2**31, 2**31, 1, 4), (2**32, 2**32, 2, 1), (2**40, 1, 2**30, 1), (2**62, 1, 1, 4)])
def test_group_sums_with_more_values_than_there_are(rows, groups, group, dim):
    refused(lib.km_group_sums(0, rows, groups, group, dim, ANY, ANY, None), b"2^60")


def test_workspaces_off_their_boundary():
    p = KmDecayProblem(dtype=1, out_dtype=1, reverse=0, path=0, sequences=1, tokens=100_000, groups=2, group=1, dk=16, dv=16, packed=0, states=0, scale=1.0)
    off, v = ctypes.c_void_p(4100), view()
    need = lib.km_decay_attention_workspace_bytes(p)
    assert need > 0
    refused(lib.km_decay_attention(p, v, v, v, v, ANY, None, None, None, off, need, None), b"16-byte aligned")
    refused(lib.km_decay_gradient(p, v, v, v, v, ANY, None, None, None, ANY, off, lib.km_decay_gradient_workspace_bytes(p), None), b"16-byte aligned")
    one = (ctypes.c_void_p * 1)(4096), (ctypes.c_int64 * 1)(4), (ctypes.c_int32 * 1)(0)
    refused(lib.km_global_norm(1, *one, 0, 0.0, 0.0, ANY, off, lib.km_global_norm_workspace_bytes(1), None), b"16-byte aligned")


@pytest.mark.parametrize("states", [1, -1, 3])
def test_workspaces_that_hold_something_else(states):
    p = KmDecayProblem(dtype=0, out_dtype=0, reverse=0, path=0, sequences=1, tokens=8, groups=2, group=1, dk=16, dv=16, packed=0, states=states, scale=1.0)
    v = view()
    refused(lib.km_decay_attention(p, v, v, v, v, ANY, None, None, None, ANY, 0, None), b"states must be")
