"""The 4-bit operators where their first tests did not look: scales next to nothing."""

from __future__ import annotations

import pytest
import torch

from test_fp4_gpu import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1e-9, 1e-30, 1e-38])
def test_zero_queries_under_a_tiny_scale(mlb, cuda, dtype, scale):
    """Keys past a row's end stay masked however small the scale is: every key that is seen weighs the same."""
    for how in ("plain", "odd"):
        st = Step(mlb, cuda, 8, 2, 64, [(70, 1), (200, 1), (9, 20), (0, 1)], dtype, how=how)
        st.q[::2] = 0.0
        st.q_dev.copy_(st.q)
        for tables, pages in ((True, 0), (False, 0), (False, 2)):
            st.check(st.run(mlb, cuda, tables, pages, scale=scale), scale=scale)
