"""What the paged kernels' numbers promise, where it is hardest to keep.

Bounds follow from the arithmetic, each beside its use.  Scores are off by 2^-21 of sum |q||k| scale
("size"), so a softmax weight by 2^-20 (1 + size) relatively with the exponential's part; 16-bit rows
round weights to 11 bits more.
"""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_paged import HALF_ULP, Setup, attention64, rows, torch  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------
# Pages of zeros
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("small", [1e-3, 1e-6, 1e-9, 1e-20, 1e-28])
@pytest.mark.parametrize("spans", [[(1, 400), (6, 200)], [(200, 400)], [(1, 9000)]], ids=["few", "many", "joined"])
@pytest.mark.parametrize("zeros", ["first", "middle", "most", "all"])
def test_zero_pages_beside_small_values(gpu, torch, dtype, small, spans, zeros):
    """A page of zeros counts in the softmax's sum alone: it takes nothing from the others' bits."""
    hq, hk, d, ps = 4, 2, 64, 16
    s = Setup(torch, spans, hk, d, ps, seed=3)
    s.vs *= np.float32(small * 60)                         # scales of 0.5 to 1.5 times `small`
    for b, (_, length) in enumerate(spans):
        need = -(-length // ps)
        gone = {"first": range(1), "middle": range(need // 2, need // 2 + 2), "all": range(need),
                "most": [i for i in range(need) if i % 5]}[zeros]
        for i in gone:
            s.vs[s.table[b, i]] = 0
    s.dvs.copy_(torch.from_numpy(s.vs))
    q, q64 = rows(torch, np.random.default_rng(1), s.tokens, hq * d, dtype)
    o = torch.full((s.tokens, hq, d), float("nan"), dtype=q.dtype, device="cuda")
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, s.batch, q.view(s.tokens, hq, d), o)
    want, size, most = attention64(s, q64, hq, True, 0)
    # the output's own rounding: relative, or half of the type's smallest number (f32's are flushed)
    least = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}[dtype]
    tol = most * (2.0 ** -20 * (1 + size) + (0 if dtype == "f32" else 2.0 ** -11))
    tol = tol + np.abs(want) * HALF_ULP[dtype] + least
    off = np.abs(o.double().cpu().numpy() - want)
    assert (off <= tol).all(), (off / tol).max()
