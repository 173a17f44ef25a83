"""Results that leave value by value, many chunks one after the other: the tile they leave through is loaded again behind them."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from kernel_matmul_b200 import ops  # noqa: E402

DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dk, dv", [(128, 77), (64, 33), (128, 127), (64, 100)])
def test_results_that_are_stored_value_by_value_are_those_that_are_not(dtype, dk, dv):
    """Rows of dv values that lie on no boundary of 16 bytes have no tensor map; with zeros up to the next multiple of 8 columns
    they have one.  The columns do not depend on each other (in fp16 the scalings are those of rows of scores and of columns of v)."""
    wide = (dv + 7) // 8 * 8
    for batch, tokens, heads in [(3, 2500, 4), (160, 700, 1)]:
        q, k = (torch.randn(batch, tokens, heads, dk, device=DEV).to(dtype) for _ in range(2))
        v = torch.zeros(batch, tokens, heads, wide, device=DEV, dtype=dtype)
        v[..., :dv] = torch.randn(batch, tokens, heads, dv, device=DEV).to(dtype)
        g = torch.full((heads,), -0.01, device=DEV)
        want, state = ops.decay_attention(q, k, v, g, return_state=True, path="tc")
        for _ in range(4):
            got, other = ops.decay_attention(q, k, v[..., :dv], g, return_state=True, path="tc")
            assert torch.equal(got, want[..., :dv]) and torch.equal(other, state[..., :dv])
