"""The decoder block (llm_block.py) for many sequences over one paged 8-bit cache.

A step takes the new tokens of any number of sequences, prompts and single
tokens together, as packed rows: RMSNORM_QUANTIZE_I8 -> MATMUL_I8 (QKV) ->
PAGED_KV_APPEND, which reads the parts of the QKV rows in place, rotates queries
and keys and appends -> PAGED_ATTENTION -> QUANTIZE_I8 -> MATMUL_I8_RESIDUAL (O)
-> RMSNORM_QUANTIZE_I8 -> MATMUL_I8_SWIGLU -> QUANTIZE_I8 -> MATMUL_I8_RESIDUAL
(down).  Pages are taken from a pool as sequences grow and given back when they
end; the block table and the lengths live on the device.

    python npuxl-improved_b200/llm_paged.py      # prompts of 8 users, then 64 steps
"""
from __future__ import annotations

import numpy as np

import vnpu
from llm_block import BlockConfig, _cmd, make_weights, ordered_on


class PagedBlock:
    """The block's weights and a pool of `pages` pages of `page_size` tokens."""

    def __init__(self, cfg: BlockConfig, lib, dev, torch, pages: int, page_size: int = 64,
                 max_batch: int = 64):
        self.cfg, self.lib, self.dev, self.t = cfg, lib, dev, torch
        self.stream = torch.cuda.ExternalStream(lib.b200_stream_handle(dev.stream))
        self.page_size, self.max_batch = page_size, max_batch
        w, (n1, n2) = make_weights(cfg)
        self.n1, self.n2 = torch.from_numpy(n1).cuda(), torch.from_numpy(n2).cuda()
        self.w = {}
        for name, f in w.items():
            K, N = f.shape
            fd = torch.from_numpy(f).cuda()
            B8 = torch.empty((K, N), dtype=torch.int8, device="cuda")
            sb = torch.empty(N, device="cuda")
            torch.cuda.synchronize()
            dev.quantize_i8(fd, B8, sb, K, N, vnpu.QUANT_PER_COLUMN)
            self.w[name] = (dev.pack(B8.data_ptr(), sb.data_ptr(), K, N), K, N)
        shape = (pages, cfg.heads, page_size, cfg.head_dim)
        # what a page holds before its first token is never read: nothing to clear
        self.k, self.v = (torch.empty(shape, dtype=torch.int8, device="cuda") for _ in range(2))
        self.ks, self.vs = (torch.empty(shape[:2], device="cuda") for _ in range(2))
        self.cache = vnpu.paged_cache(self.k, self.v, self.ks, self.vs)
        self.free = list(range(pages - 1, -1, -1))
        self.pages, self.length = {}, {}          # of each sequence

    def close(self):
        for (w, _, _) in self.w.values():
            self.dev.unpack(w)

    def release(self, seq) -> None:
        """Gives a sequence's pages back (the steps that used them are on the stream before any
        that will)."""
        self.free += self.pages.pop(seq, [])
        self.length.pop(seq, None)

    def _grow(self, counts: dict) -> None:
        """Pages for all of the new tokens, or none and an error."""
        need = {s: -(-(self.length.get(s, 0) + n) // self.page_size) - len(self.pages.get(s, ()))
                for s, n in counts.items()}
        if sum(need.values()) > len(self.free):
            raise RuntimeError(f"the pool is out of pages: {sum(need.values())} wanted, "
                               f"{len(self.free)} free")
        for s, n in counts.items():
            self.length[s] = self.length.get(s, 0) + n
            self.pages.setdefault(s, []).extend(self.free.pop() for _ in range(need[s]))

    def step(self, x, counts: dict):
        """x: [tokens][d] f32 on the device, the rows of `counts`' sequences in its order;
        counts: sequence -> its number of new tokens.  Returns [tokens][d].  The step runs on the
        library's stream, ordered with the stream that is current where it is called."""
        t, cfg = self.t, self.cfg
        T, d, H, hd = x.shape[0], cfg.d, cfg.heads, cfg.head_dim
        if T != sum(counts.values()) or not counts or len(counts) > self.max_batch or min(counts.values()) < 0:
            raise ValueError("rows of x and counts differ, or the batch is too large")
        if x.dtype != t.float32 or tuple(x.shape) != (T, d) or not x.is_contiguous() or not x.is_cuda:
            raise ValueError(f"x: contiguous float32 of shape {(T, d)} on the device, got {x.dtype} "
                             f"{tuple(x.shape)} with strides {x.stride()} on {x.device}")
        if T == 0:
            return t.empty((0, d), device="cuda")
        self._grow(counts)
        width = max(len(self.pages[s]) for s in counts)
        table = np.full((len(counts), width), -1, np.int32)
        for row, s in zip(table, counts):
            row[:len(self.pages[s])] = self.pages[s]
        cu = np.concatenate([[0], np.cumsum(list(counts.values()))]).astype(np.int32)
        lens = np.array([self.length[s] for s in counts], np.int32)
        y = t.empty((T, d), device="cuda")        # the caller's stream's memory, as x is
        with ordered_on(t, self.stream):
            dev = lambda a: t.from_numpy(a).cuda(non_blocking=False)  # noqa: E731
            table, cu, lens = dev(table), dev(cu), dev(lens)
            new = lambda *shape, dtype=t.float32: t.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
            batch = vnpu.paged_batch(table, cu, lens, T, max(counts.values()))

            def norm(src, weight, name):
                K = self.w[name][1]
                a8, sa = new(T, K, dtype=t.int8), new(T)
                return a8, sa, vnpu.b200_command(vnpu.OP_B200_RMSNORM_QUANTIZE_I8, vnpu.RmsnormQuantizeArgs(
                    vnpu.ptr(src), vnpu.ptr(weight), None, vnpu.ptr(a8), vnpu.ptr(sa), T, K, cfg.eps, 0))

            def projection(src, residual, name, out):
                w, K, N = self.w[name]
                a8, sa = new(T, K, dtype=t.int8), new(T)
                return [
                    _cmd(vnpu.OP_QUANTIZE_I8, "quantize_i8", vnpu.QuantizeI8Args(
                        vnpu.ptr(src), vnpu.ptr(a8), vnpu.ptr(sa), T, K, 0, 0)),
                    vnpu.b200_command(vnpu.OP_B200_MATMUL_I8_RESIDUAL, vnpu.MatmulI8ResidualArgs(
                        vnpu.ptr(a8), w, vnpu.ptr(sa), None, vnpu.ptr(residual), vnpu.ptr(out), T, K, N,
                        0, 0, 0, 0, 0))]

            w, K, N = self.w["qkv"]
            a8, sa, pre = norm(x, self.n1, "qkv")
            qkv, att = new(T, N), new(T, H, hd)
            q, k, v = qkv.split(d, dim=1)
            cmds = [pre, _cmd(vnpu.OP_MATMUL_I8, "matmul_i8", vnpu.MatmulI8Args(
                        vnpu.ptr(a8), w, vnpu.ptr(sa), None, vnpu.ptr(qkv), T, K, N, 0, 0, 0, vnpu.UNIT_GPU)),
                    # the rotated queries take the projection's place
                    vnpu.paged_kv_append_cmd(self.cache, batch, q, k, v, q, q_heads=H, theta=cfg.theta),
                    vnpu.paged_attention_cmd(self.cache, batch, q.unflatten(1, (H, hd)), att,
                                             max_length=int(max(self.length[s] for s in counts)))]
            x1 = new(T, d)
            more = projection(att, x, "o", x1)
            w, K, N = self.w["gate_up"]
            b8, sb, pre = norm(x1, self.n2, "gate_up")
            ff = new(T, cfg.inter)
            last = projection(ff, x1, "down", y)
            cmds += more + [pre, vnpu.b200_command(vnpu.OP_B200_MATMUL_I8_SWIGLU, vnpu.MatmulI8SwigluArgs(
                vnpu.ptr(b8), w, vnpu.ptr(sb), None, vnpu.ptr(ff), T, K, N, 0, 0, 0, 1.0, 0))] + last
            self.lib.check(self.dev.submit(cmds), "submit")
            # all but x and y is the caching allocator's memory of this stream: it may go now
        return y


def main():
    import time

    import torch

    lib = vnpu.Lib(vnpu.LIB_PATH)
    with vnpu.Device(lib) as dev:
        block = PagedBlock(BlockConfig(), lib, dev, torch, pages=256)
        gen = torch.Generator(device="cuda").manual_seed(0)
        prompts = {i: 100 + 37 * i for i in range(8)}
        x = torch.randn((sum(prompts.values()), block.cfg.d), generator=gen, device="cuda")
        y = block.step(x, prompts)
        dev.sync()
        start = time.perf_counter()
        steps = 64
        for _ in range(steps):
            y = block.step(torch.randn((8, block.cfg.d), generator=gen, device="cuda"),
                           dict.fromkeys(prompts, 1))
        assert dev.sync() == vnpu.OK
        ms = (time.perf_counter() - start) / steps * 1e3
        print(f"8 users, {sum(prompts.values())} prompt tokens, {steps} steps: {ms:.3f} ms a step, "
              f"{len(block.free)} of 256 pages free, |y| {float(y.norm()):.3f}")
        block.close()


if __name__ == "__main__":
    main()
