"""The decoder blocks' calls beside a caller's own stream.

The library's stream does not wait for torch's streams by itself, nor they for it.  A block's call is
ordered with the stream that is current where it is made, as a torch operator is: what was enqueued
there before is seen, the result may be used there at once, and inputs may be overwritten or freed.
One side is held back in each test, so that an order that is missing shows every time.
"""
from __future__ import annotations

import pytest

import vnpu

pytestmark = pytest.mark.gpu

HOLD = 20_000_000      # clocks, about 10 ms


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def caller_stream(torch, name):
    return torch.cuda.Stream() if name == "own" else torch.cuda.default_stream()


class Late:
    """Holds back the caller's stream, the library's, or (None) has all done after each call."""

    def __init__(self, torch, held):
        self.torch, self.held = torch, held

    def here(self, name, stream):
        if self.held == name:
            with self.torch.cuda.stream(stream):
                self.torch.cuda._sleep(HOLD)

    def done(self):
        if self.held is None:
            self.torch.cuda.synchronize()


def run_block(b200_lib, torch, held, caller, fused):
    from llm_block import B200Block, BlockConfig
    cfg = BlockConfig(d=256, heads=4, inter=704, cap=48)
    gen = torch.Generator().manual_seed(1)
    late, outs = Late(torch, held), []
    with vnpu.Device(b200_lib) as dev:
        blk = B200Block(cfg, b200_lib, dev, torch, fused=fused)
        stream = caller_stream(torch, caller)
        sources = [torch.randn((n, cfg.d), generator=gen).cuda() for n in (20, 1, 1)]
        inputs = [torch.zeros_like(x) for x in sources]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for source, x, pos in zip(sources, inputs, (0, 20, 21)):
                late.here("caller", stream)
                x.copy_(source)
                late.done()
                late.here("library", blk.stream)
                y = blk.forward(x, pos)
                late.done()
                outs.append(y.clone())
                x.fill_(float("nan"))
        torch.cuda.synchronize()
        assert dev.sync() == vnpu.OK
        blk.close()
    return outs


@pytest.mark.parametrize("held", ["caller", "library"])
@pytest.mark.parametrize("caller", ["default", "own"])
@pytest.mark.parametrize("fused", [True, False])
def test_block_forward_is_ordered_with_the_callers_stream(b200_lib, torch, held, caller, fused):
    want = run_block(b200_lib, torch, None, caller, fused)
    for a, b in zip(run_block(b200_lib, torch, held, caller, fused), want):
        assert torch.equal(a, b)


def run_replay(b200_lib, torch, held, caller):
    from llm_block import B200Block, BlockConfig
    cfg = BlockConfig(d=256, heads=4, inter=704, cap=48)
    gen = torch.Generator().manual_seed(2)
    late, outs = Late(torch, held), []
    with vnpu.Device(b200_lib) as dev:
        blk = B200Block(cfg, b200_lib, dev, torch)
        prompt, tokens = (torch.randn(n, cfg.d, generator=gen).cuda() for n in (20, 4))
        xin = torch.zeros((1, cfg.d), device="cuda")
        torch.cuda.synchronize()
        blk.forward(prompt, 0)
        torch.cuda.synchronize()
        y = blk.capture_decode(xin)
        blk.pos.fill_(20)
        torch.cuda.synchronize()
        stream = caller_stream(torch, caller)
        with torch.cuda.stream(stream):
            for token in tokens:
                late.here("caller", stream)
                xin.copy_(token[None])
                late.done()
                late.here("library", blk.stream)
                blk.replay_decode()
                late.done()
                outs.append(y.clone())
                xin.fill_(float("nan"))
        torch.cuda.synchronize()
        assert dev.sync() == vnpu.OK
        blk.close()
    return outs


@pytest.mark.parametrize("held", ["caller", "library"])
@pytest.mark.parametrize("caller", ["default", "own"])
def test_block_replay_is_ordered_with_the_callers_stream(b200_lib, torch, held, caller):
    want = run_replay(b200_lib, torch, None, caller)
    for a, b in zip(run_replay(b200_lib, torch, held, caller), want):
        assert torch.equal(a, b)


def run_paged(b200_lib, torch, held, caller):
    from llm_block import BlockConfig
    from llm_paged import PagedBlock
    cfg = BlockConfig(d=256, heads=4, inter=704, cap=64)
    gen = torch.Generator().manual_seed(3)
    prompts = {"a": 20, "b": 1, "c": 33}
    late, outs = Late(torch, held), []
    with vnpu.Device(b200_lib) as dev:
        blk = PagedBlock(cfg, b200_lib, dev, torch, pages=24, page_size=16)
        stream, submit = caller_stream(torch, caller), dev.submit

        def submit_late(cmds, event=None):
            late.here("library", blk.stream)
            return submit(cmds, event)

        dev.submit = submit_late
        sources = [torch.randn((n, cfg.d), generator=gen).cuda() for n in [54] + [3] * 6]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for i, source in enumerate(sources):
                late.here("caller", stream)
                x = source * 1
                late.done()
                y = blk.step(x, dict(prompts) if i == 0 else dict.fromkeys(prompts, 1))
                late.done()
                outs.append(y * 1)
                y.fill_(float("nan"))
                del x, y
                for _ in range(3):            # of the sizes of x and y, in their places
                    torch.full((source.shape[0], cfg.d), float("nan"), device="cuda")
        torch.cuda.synchronize()
        assert dev.sync() == vnpu.OK
        blk.close()
    return outs


@pytest.mark.parametrize("held", ["caller", "library"])
@pytest.mark.parametrize("caller", ["default", "own"])
def test_paged_steps_of_temporaries(b200_lib, torch, held, caller):
    """Inputs and outputs that go as soon as they are used, no sync between steps."""
    want = run_paged(b200_lib, torch, None, caller)
    for a, b in zip(run_paged(b200_lib, torch, held, caller), want):
        assert torch.equal(a, b)
