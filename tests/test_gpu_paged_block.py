"""The decoder block over the paged 8-bit cache (llm_paged.PagedBlock) against the block with
its f32 cache (llm_block.B200Block), sequence by sequence.

The two differ by the cache's rounding: half a step of a page's largest value, 0.3 % of it as an
rms error, about 1 % of a value's own size (a page's largest is some 3-4 times that).  Attention
averages values and perturbs scores by as much, and the output adds the result to its input, so
the rows agree within 2 % of their norm.
"""
from __future__ import annotations

import numpy as np
import pytest

import vnpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.mark.parametrize("page_size", [16, 64])
def test_sequences_of_any_lengths_step_together(b200_lib, torch, page_size):
    from llm_block import B200Block, BlockConfig
    from llm_paged import PagedBlock
    cfg = BlockConfig(d=256, heads=4, inter=704, cap=64)
    gen = torch.Generator().manual_seed(3)
    prompts = {"a": 20, "b": 1, "c": 33}
    rows = {s: torch.randn((n + 6, cfg.d), generator=gen) for s, n in prompts.items()}
    want = {}
    for s, n in prompts.items():
        with vnpu.Device(b200_lib) as dev:
            blk = B200Block(cfg, b200_lib, dev, torch)
            x = rows[s].cuda()
            torch.cuda.synchronize()
            out = []
            for i, j in [(0, n)] * (n > 1) + [(i, i + 1) for i in range(n if n > 1 else 0, n + 6)]:
                y = blk.forward(x[i:j], i)
                assert dev.sync() == vnpu.OK
                out.append(y.clone())
            torch.cuda.synchronize()
            want[s] = torch.cat(out).cpu()
            blk.close()
    with vnpu.Device(b200_lib) as dev:
        blk = PagedBlock(cfg, b200_lib, dev, torch, pages=24, page_size=page_size)
        got = {s: [] for s in prompts}
        x = torch.cat([rows[s][:n] for s, n in prompts.items()]).cuda()
        steps = [(x, dict(prompts))]
        for i in range(6):
            steps.append((torch.cat([rows[s][n + i:n + i + 1] for s, n in prompts.items()]).cuda(),
                          dict.fromkeys(prompts, 1)))
        for x, counts in steps:
            y = blk.step(x, counts)
            assert dev.sync() == vnpu.OK
            for s, part in zip(counts, y.cpu().split(list(counts.values()))):
                got[s].append(part)
        used = 24 - len(blk.free)
        assert used == sum(-(-(n + 6) // page_size) for n in prompts.values())
        for s in prompts:
            a, b = torch.cat(got[s]).double(), want[s].double()
            assert ((a - b).norm(dim=1) <= 2e-2 * b.norm(dim=1)).all()
        blk.release("a")
        assert len(blk.free) == 24 - used + -(-26 // page_size) and "a" not in blk.length
        with pytest.raises(RuntimeError):
            blk.step(torch.zeros((2001, cfg.d), device="cuda"), {"b": 1, "d": 2000})
        assert blk.length["b"] == 7 and "d" not in blk.length
        with pytest.raises(ValueError):
            blk.step(torch.zeros((3, cfg.d), device="cuda"), {"b": 2})
        blk.close()
    assert np.isfinite(a.numpy()).all()
