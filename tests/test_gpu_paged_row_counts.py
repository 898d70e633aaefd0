"""PAGED_ATTENTION around the row counts at which another kernel or tile takes over."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_paged import Setup, attention64, check_attention, rows, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 80, 128, 192])
@pytest.mark.parametrize("group,n", [(1, 7), (1, 8), (1, 9), (1, 16), (1, 17), (1, 31), (1, 32), (1, 33), (4, 8),
                                     (4, 9), (3, 16), (1, 49), (7, 7), (4, 13), (1, 63), (8, 8), (1, 65), (5, 13),
                                     (1, 81), (2, 64), (1, 129)])
def test_rows_of_a_head(gpu, torch, dtype, d, group, n):
    s = Setup(torch, [(n, n + 150), (1, 300), (n, n)], 2, d, 16, seed=n)
    hq = 2 * group
    q, q64 = rows(torch, np.random.default_rng(n), s.tokens, hq * d, dtype)
    o = torch.full((s.tokens, hq, d), float("nan"), dtype=q.dtype, device="cuda")
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, s.batch, q.view(s.tokens, hq, d), o)
    check_attention(o, *attention64(s, q64, hq, True, 0), dtype)
