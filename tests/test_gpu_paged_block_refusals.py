"""What PagedBlock.step refuses, before it takes pages or enqueues anything."""
from __future__ import annotations

import pytest

import vnpu

pytestmark = pytest.mark.gpu


def test_step_refuses_rows_it_cannot_read(b200_lib):
    torch = pytest.importorskip("torch")
    from llm_block import BlockConfig
    from llm_paged import PagedBlock
    cfg = BlockConfig(d=256, heads=4, inter=704, cap=64)
    with vnpu.Device(b200_lib) as dev:
        blk = PagedBlock(cfg, b200_lib, dev, torch, pages=4, page_size=16)
        x = torch.zeros((6, cfg.d), device="cuda")
        for rows, counts in [(x.half(), {"a": 6}), (x.double(), {"a": 6}), (x.cpu(), {"a": 6}),
                             (x[::2], {"a": 3}), (x.t().contiguous().t(), {"a": 6}), (x[:, :128], {"a": 6}),
                             (x[:, None], {"a": 6}), (x, {"a": 7, "b": -1}), (x, {})]:
            with pytest.raises(ValueError):
                blk.step(rows, counts)
        assert len(blk.free) == 4 and not blk.length and not blk.pages
        assert blk.step(x[:0], {"a": 0}).shape == (0, cfg.d) and len(blk.free) == 4
        y = blk.step(x, {"a": 2, "b": 4})
        assert y.shape == x.shape and dev.sync() == vnpu.OK
        blk.close()
