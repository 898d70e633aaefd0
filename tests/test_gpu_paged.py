"""The paged 8-bit key/value cache: PAGED_KV_APPEND, PAGED_KV_READ and PAGED_ATTENTION
(include/vnpu_b200.h) against their definitions in 64 bits, in numpy.

Tolerances follow from the arithmetic and are stated where they are used:
* a rotation is off by the 32-bit rounding of the angle (2^-24 of at most pi), the sine's and
  cosine's (2 ulp) and three roundings of the products: 8 * 2^-24 of |pair|, plus the row type's
  half unit in the last place;
* a stored value is at most half a code from what was given (plus the rotation's error), a page's
  older values at most half a new code from what they were;
* a read is one 32-bit product, rounded once: equal to the bit;
* attention: scores are off by 2^-21 of sum |q||k| (22-bit queries, 32-bit sums), so weights by
  that much relatively; with 16-bit rows the weights are rounded to 11 bits.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import vnpu

pytestmark = pytest.mark.gpu

HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # relative, an ulp to be safe


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def dt(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Setup:
    """A cache with pages in a shuffled order and the sequences' arrays on the device."""

    def __init__(self, torch, spans, kv_heads, d, ps, seed=0, slack=2, stride_extra=1):
        rng = np.random.default_rng(seed)
        self.torch, self.spans, self.ps, self.d, self.hk = torch, spans, ps, d, kv_heads
        need = [-(-length // ps) for _, length in spans]
        self.pages = sum(need) + slack
        order = rng.permutation(self.pages)
        self.table = np.full((len(spans), max(need + [1]) + stride_extra), 2 ** 31 - 1, np.int32)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = order[at:at + k]
            at += k
        self.k = rng.integers(-127, 128, (self.pages, kv_heads, ps, d)).astype(np.int8)
        self.v = rng.integers(-127, 128, (self.pages, kv_heads, ps, d)).astype(np.int8)
        self.ks = rng.uniform(0.5, 1.5, (self.pages, kv_heads)).astype(np.float32) / 60
        self.vs = rng.uniform(0.5, 1.5, (self.pages, kv_heads)).astype(np.float32) / 60
        unused = np.ones(self.pages, bool)
        for b, k in enumerate(need):
            unused[self.table[b, :k]] = False
        self.ks[unused] = np.nan          # nothing of these may be looked at
        self.vs[unused] = np.inf
        self.cu = np.concatenate([[0], np.cumsum([n for n, _ in spans])]).astype(np.int32)
        self.lens = np.array([length for _, length in spans], np.int32)
        self.tokens = int(self.cu[-1])
        dev = lambda a: torch.from_numpy(a.copy()).cuda()  # noqa: E731
        self.dk, self.dv, self.dks, self.dvs = dev(self.k), dev(self.v), dev(self.ks), dev(self.vs)
        self.dtable, self.dcu, self.dlens = dev(self.table), dev(self.cu), dev(self.lens)
        self.cache = vnpu.paged_cache(self.dk, self.dv, self.dks, self.dvs)
        self.batch = vnpu.paged_batch(self.dtable, self.dcu, self.dlens, self.tokens,
                                      max([n for n, _ in spans] + [0]))
        torch.cuda.synchronize()

    def seq_codes(self, which, b):
        """Codes [length][heads][d] and scales [length][heads] of sequence b, in 64 bits."""
        length = self.spans[b][1]
        pages = self.table[b, : -(-length // self.ps)]
        codes, scale = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        c = codes[pages].astype(np.float64).transpose(0, 2, 1, 3).reshape(-1, self.hk, self.d)
        return c[:length], np.repeat(scale[pages].astype(np.float64), self.ps, 0)[:length]


def rows(torch, rng, n, width, dtype, extra=0):
    """A device tensor [n][width] (row stride width + extra) and its values in 64 bits."""
    x = torch.from_numpy(rng.standard_normal((max(n, 1), width + extra)).astype(np.float32))
    x = x.to(dt(torch, dtype)).cuda()[:n, :width]
    return x, x.double().cpu().numpy()


# ------------------------------------------------------------------------------------------------
# Attention
# ------------------------------------------------------------------------------------------------
def attention64(s, q, hq, causal, window, scale=None):
    """Outputs [tokens][hq][d], and for each row sum |q||k| scale at its largest and max |v|."""
    d, g = s.d, hq // s.hk
    out = np.zeros((s.tokens, hq, d))
    size = np.zeros((s.tokens, hq, 1))
    most = np.zeros((s.tokens, hq, 1))
    scale = scale or 1 / np.sqrt(d)
    for b, (n, length) in enumerate(s.spans):
        k, ks = s.seq_codes("k", b)
        v, vs = s.seq_codes("v", b)
        k, v = k * ks[:, :, None], v * vs[:, :, None]
        at = np.arange(length)
        pos = length - n + np.arange(n)
        seen = np.ones((n, length), bool)
        if causal:
            seen &= at[None] <= pos[:, None]
        if window:
            seen &= at[None] > pos[:, None] - window
        for h in range(hq):
            x = q[s.cu[b]:s.cu[b + 1]].reshape(n, hq, d)[:, h]
            w = (x @ k[:, h // g].T) * scale
            w = np.where(seen, w, -np.inf)
            top = w.max(1, keepdims=True, initial=-np.inf)
            p = np.exp(w - np.where(np.isinf(top), 0, top))
            total = p.sum(1, keepdims=True)
            o = (p @ v[:, h // g]) / np.where(total > 0, total, 1)
            sl = slice(s.cu[b], s.cu[b + 1])
            out[sl, h] = o
            if length:
                size[sl, h] = ((np.abs(x) @ np.abs(k[:, h // g]).T) * scale).max(1, keepdims=True)
                most[sl, h] = np.abs(v[:, h // g]).max()
    return out, size, most


def check_attention(got, want, size, most, dtype):
    got = got.double().cpu().numpy()
    # weights: 2 * 2^-21 of the score's terms and 2^-20 of sums and exponentials; 16-bit rows round
    # each weight to 11 bits; then the output's own rounding
    tol = most * (2.0 ** -20 * (1 + size) + (0 if dtype == "f32" else 2.0 ** -11))
    tol = tol + np.abs(want) * HALF_ULP[dtype] + 1e-30
    bad = np.abs(got - want) > tol
    assert np.isfinite(got).all()
    assert not bad.any(), (bad.sum(), np.abs(got - want).max(), np.argwhere(bad)[:4])


SPANS = {
    "one": [(1, 1)],
    "decode": [(1, 5), (1, 300), (1, 1), (1, 129), (1, 128)],
    "long": [(1, 5000)],
    "mixed": [(3, 3), (0, 40), (7, 200), (1, 64), (0, 0), (20, 333)],
    "prefill": [(150, 150), (33, 400)],
    "rows": [(130, 257), (64, 64), (1, 700)],
}


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hk,d,ps", [(4, 4, 128, 64), (8, 2, 64, 16), (6, 1, 96, 32),
                                        (3, 3, 256, 128), (5, 1, 16, 16), (16, 1, 144, 256)])
@pytest.mark.parametrize("spans", ["one", "decode", "long", "mixed", "prefill", "rows"])
def test_attention(gpu, torch, dtype, hq, hk, d, ps, spans):
    s = Setup(torch, SPANS[spans], hk, d, ps, seed=len(spans))
    rng = np.random.default_rng(1)
    q, q64 = rows(torch, rng, s.tokens, hq * d, dtype)
    o = torch.full((s.tokens, hq, d), float("nan"), dtype=q.dtype, device="cuda")
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, s.batch, q.view(s.tokens, hq, d), o)
    check_attention(o, *attention64(s, q64, hq, True, 0), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("causal,window", [(False, 0), (True, 1), (True, 100), (False, 37),
                                           (True, 128), (True, 100000)])
@pytest.mark.parametrize("spans", ["mixed", "prefill", "long", "rows"])
def test_attention_masks(gpu, torch, dtype, causal, window, spans):
    hq, hk, d, ps = 4, 2, 128, 16
    s = Setup(torch, SPANS[spans], hk, d, ps)
    q, q64 = rows(torch, np.random.default_rng(2), s.tokens, hq * d, dtype)
    o = torch.full((s.tokens, hq, d), float("nan"), dtype=q.dtype, device="cuda")
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, s.batch, q.view(s.tokens, hq, d), o, causal=causal, window=window)
    check_attention(o, *attention64(s, q64, hq, causal, window), dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_ragged_rows_of_many(gpu, torch, dtype, d):
    """More sequences than a CTA has threads, most of them short, some without rows."""
    rng = np.random.default_rng(5)
    spans = [(int(rng.integers(0, 3)), int(rng.integers(2, 90))) for _ in range(300)]
    spans[37] = (200, 900)
    s = Setup(torch, spans, 2, d, 32)
    q, q64 = rows(torch, rng, s.tokens, 4 * d, dtype)
    o = torch.full((s.tokens, 4, d), float("nan"), dtype=q.dtype, device="cuda")
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, s.batch, q.view(s.tokens, 4, d), o)
    check_attention(o, *attention64(s, q64, 4, True, 0), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spans", [[(40, 60000)], [(300, 20000), (5, 9000), (1, 30000)]])
def test_attention_long_runs_of_key_tiles(gpu, torch, dtype, spans):
    """Tens of thousands of keys under a few hundred rows: every CTA walks many tiles of one
    block, and blocks are joined from many CTAs."""
    s = Setup(torch, spans, 1, 128, 64)
    q, q64 = rows(torch, np.random.default_rng(6), s.tokens, 2 * 128, dtype)
    o = torch.full((s.tokens, 2, 128), float("nan"), dtype=q.dtype, device="cuda")
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, s.batch, q.view(s.tokens, 2, 128), o)
    check_attention(o, *attention64(s, q64, 2, True, 0), dtype)


@pytest.mark.parametrize("dtype,extra", [("f32", 3), ("f32", 4), ("bf16", 1), ("f16", 8), ("f16", 4)])
def test_attention_strided_rows_and_in_place(gpu, torch, dtype, extra):
    """Rows with gaps of odd and even sizes, unaligned bases, and the output over the queries."""
    hq, hk, d = 4, 2, 64
    s = Setup(torch, SPANS["mixed"], hk, d, 16)
    rng = np.random.default_rng(3)
    full = torch.from_numpy(rng.standard_normal((s.tokens, hq * d + extra)).astype(np.float32))
    full = full.to(dt(torch, dtype)).cuda()
    for base in (0, extra):
        x = full.clone()
        q = x[:, base:base + hq * d]
        q64 = q.double().cpu().numpy()
        want = attention64(s, q64, hq, True, 0)
        args = vnpu.PagedAttentionArgs(s.cache, s.batch, q.data_ptr(), q.data_ptr(), x.stride(0),
                                       x.stride(0), hq, vnpu._paged_dtype(q), 1, 0, 0, 0.0)
        torch.cuda.synchronize()
        gpu._run(vnpu.b200_command(vnpu.OP_B200_PAGED_ATTENTION, args), "paged_attention")
        check_attention(q.reshape(s.tokens, hq, d), *want, dtype)
        rest = torch.ones(hq * d + extra, dtype=torch.bool)
        rest[base:base + hq * d] = False
        assert torch.equal(x[:, rest], full[:, rest])       # the gaps keep what they held


@pytest.mark.parametrize("scale", [0.03, 2.0, -0.5])
def test_attention_scale_and_large_scores(gpu, torch, scale):
    """Scores of hundreds: the running maximum moves far, most weights vanish."""
    s = Setup(torch, [(1, 700), (40, 300)], 2, 128, 64)
    q, q64 = rows(torch, np.random.default_rng(4), s.tokens, 4 * 128, "f32")
    o = torch.empty((s.tokens, 4, 128), device="cuda")
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, s.batch, q.view(-1, 4, 128), o, scale=scale)
    want, size, most = attention64(s, q64, 4, True, 0, scale)
    check_attention(o, want, np.abs(size), most, "f32")


def test_attention_rows_of_any_size(gpu, torch):
    """Queries of 1e-30 and 1e30, of zeros, and of bf16's largest numbers; pages whose scale is 0."""
    s = Setup(torch, [(6, 200)], 1, 128, 16)
    for page in s.table[0, 2:4]:
        s.vs[page] = 0
        s.ks[page] = 0
    s.dks.copy_(torch.from_numpy(s.ks))
    s.dvs.copy_(torch.from_numpy(s.vs))
    q = torch.randn((6, 1, 128), generator=torch.Generator().manual_seed(0))
    q = (q * torch.tensor([1e-30, 1.0, 0.0, 1e3, 1e-3, 1e-38])[:, None, None]).to(torch.bfloat16).cuda()
    o = torch.empty_like(q)
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, s.batch, q, o)
    q64 = q.double().cpu().numpy().reshape(6, -1)
    check_attention(o, *attention64(s, q64, 1, True, 0), "bf16")


def test_attention_bad_values_stay_in_their_row(gpu, torch):
    """A NaN or an infinity in one query leaves the other rows' bits alone."""
    s = Setup(torch, [(9, 150), (1, 30)], 1, 64, 16)
    q = torch.randn((10, 2, 64), generator=torch.Generator().manual_seed(0)).cuda()
    clean, dirty = torch.empty_like(q), torch.empty_like(q)
    bad = q.clone()
    bad[3, 1, 7] = float("nan")
    bad[5, 0, 0] = float("inf")
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, s.batch, q, clean)
    gpu.paged_attention(s.cache, s.batch, bad, dirty)
    keep = torch.ones((10, 2), dtype=torch.bool)
    keep[3, 1] = keep[5, 0] = False
    assert torch.equal(clean[keep], dirty[keep])
    assert torch.isnan(dirty[3, 1]).all()


def test_attention_is_repeatable(gpu, torch):
    s = Setup(torch, [(1, 9000), (1, 70), (3, 2000)], 2, 128, 64)
    q, _ = rows(torch, np.random.default_rng(4), s.tokens, 8 * 128, "bf16")
    outs = [torch.empty((s.tokens, 8, 128), dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    for o in outs:
        gpu.paged_attention(s.cache, s.batch, q.view(-1, 8, 128), o)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_attention_rows_past_the_sequences_are_left_alone(gpu, torch):
    s = Setup(torch, [(2, 20)], 1, 64, 16)
    batch = vnpu.paged_batch(s.dtable, s.dcu, s.dlens, 5)       # 5 rows, the sequences have 2
    q = torch.randn((5, 1, 64), device="cuda")
    o = torch.full((5, 1, 64), 7.0, device="cuda")
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, batch, q, o)
    assert (o[2:] == 7.0).all() and not (o[:2] == 7.0).any()


# ------------------------------------------------------------------------------------------------
# Append and read
# ------------------------------------------------------------------------------------------------
def rotate64(x, pos, rotary, theta, scaling, interleaved):
    """x [rows][heads][d] in 64 bits."""
    x = x.copy()
    j = np.arange(rotary // 2)
    angle = (pos[:, None] * (scaling * theta ** (-2.0 * j / rotary)))[:, None, :]
    a, b = ((slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else
            (slice(0, rotary // 2), slice(rotary // 2, rotary)))
    p, q = x[..., a].copy(), x[..., b].copy()
    x[..., a] = p * np.cos(angle) - q * np.sin(angle)
    x[..., b] = p * np.sin(angle) + q * np.cos(angle)
    return x


def check_append(s, q_out, q64, k64, v64, hq, dtype, rotary, theta=10000.0, scaling=1.0,
                 interleaved=False):
    pos = np.concatenate([length - n + np.arange(n) for n, length in s.spans])
    if q_out is not None:
        got = q_out.double().cpu().numpy().reshape(s.tokens, hq, s.d)
        x = q64.reshape(s.tokens, hq, s.d)
        want = rotate64(x, pos, rotary, theta, scaling, interleaved) if rotary else x
        size = np.abs(x).max(-1, keepdims=True) * 2
        assert (np.abs(got - want) <= size * 2.0 ** -21 + np.abs(want) * HALF_ULP[dtype]).all()
    touched = np.zeros((s.pages, s.ps), bool)
    for which, x in (("k", k64), ("v", v64)):
        x = x.reshape(s.tokens, s.hk, s.d)
        if which == "k" and rotary:
            x = rotate64(x, pos, rotary, theta, scaling, interleaved)
        size = np.abs(x).max(-1) * 2 * 2.0 ** -21                      # the rotation's error
        codes0, scale0 = (s.k, s.ks) if which == "k" else (s.v, s.vs)
        codes = (s.dk if which == "k" else s.dv).cpu().numpy()
        scale = (s.dks if which == "k" else s.dvs).cpu().numpy()
        row = 0
        seen = set()
        for b, (n, length) in enumerate(s.spans):
            start = length - n
            if n == 0:
                continue
            for p in range(start // s.ps, (length - 1) // s.ps + 1):
                page = s.table[b, p]
                seen.add(int(page))
                lo, hi = max(start, p * s.ps), min(length, (p + 1) * s.ps)
                r = slice(row + lo - start, row + hi - start)
                sl = slice(lo - p * s.ps, hi - p * s.ps)
                touched[page, sl] = True
                most = np.abs(x[r]).max((0, 2)) / 127
                old = scale0[page].astype(np.float64) if lo > p * s.ps else np.zeros(s.hk)
                now = np.maximum(old, most)
                assert (np.abs(scale[page] - now) <= now * 2.0 ** -22 + size[r].max(0) / 127).all()
                now = scale[page].astype(np.float64)
                stored = codes[page, :, sl].astype(np.float64) * now[:, None, None]
                off = np.abs(stored - x[r].transpose(1, 0, 2))
                assert (off <= now[:, None, None] * (0.5 + 1e-4) + size[r].max()).all()
                kept = codes0[page, :, :lo - p * s.ps].astype(np.float64) * old[:, None, None]
                now_kept = codes[page, :, :lo - p * s.ps].astype(np.float64) * now[:, None, None]
                assert (np.abs(kept - now_kept) <= now[:, None, None] * (0.5 + 1e-4)).all()
                if (now == old).any():       # scales that did not grow keep their codes
                    h = now == old
                    assert (codes[page, h, :lo - p * s.ps] == codes0[page, h, :lo - p * s.ps]).all()
            row += n
        rest = np.ones(s.pages, bool)
        rest[list(seen)] = False
        assert np.array_equal(codes[rest], codes0[rest])
        assert np.array_equal(scale[rest].view(np.uint32), scale0[rest].view(np.uint32))
        for page in seen:                     # slots past the new tokens are not written
            last = np.flatnonzero(touched[page])[-1] + 1
            assert np.array_equal(codes[page, :, last:], codes0[page, :, last:])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hq,hk,d,ps,rotary,interleaved", [
    (4, 4, 128, 64, 128, False), (8, 2, 64, 16, 64, True), (6, 1, 96, 32, 32, False),
    (3, 3, 256, 128, 256, False), (1, 1, 16, 16, 16, True), (5, 1, 256, 256, 0, False),
    (2, 1, 80, 64, 48, True)])
@pytest.mark.parametrize("spans", ["one", "decode", "mixed", "prefill"])
def test_append(gpu, torch, dtype, hq, hk, d, ps, rotary, interleaved, spans):
    s = Setup(torch, SPANS[spans], hk, d, ps, seed=7)
    rng = np.random.default_rng(11)
    qkv, x64 = rows(torch, rng, s.tokens, (hq + 2 * hk) * d, dtype)
    qkv[: s.tokens // 2] *= 0.25               # some pages' scales grow, some stay
    x64 = qkv.double().cpu().numpy()
    q, k, v = qkv.split([hq * d, hk * d, hk * d], dim=1)
    q_out = torch.empty((s.tokens, hq, d), dtype=q.dtype, device="cuda")
    torch.cuda.synchronize()
    gpu.paged_kv_append(s.cache, s.batch, q, k, v, q_out, q_heads=hq, interleaved=interleaved,
                        rope=rotary > 0, rotary_dim=rotary)
    parts = np.split(x64, [hq * d, (hq + hk) * d], axis=1)
    check_append(s, q_out, *parts, hq, dtype, rotary, interleaved=interleaved)


@pytest.mark.parametrize("theta,scaling", [(500000.0, 1.0), (10000.0, 0.25), (100.0, 8.0)])
def test_append_far_positions(gpu, torch, theta, scaling):
    """Positions of two million: the angles are as exact as at the start."""
    s = Setup(torch, [(3, 3)], 1, 128, 64)
    length = 2_000_003
    table = torch.full((1, length // 64 + 1), -1, dtype=torch.int32, device="cuda")
    table[0, length // 64] = int(s.table[0, 0])
    table[0, (length - 3) // 64] = int(s.table[0, 0])
    lens = torch.tensor([length], dtype=torch.int32, device="cuda")
    batch = vnpu.paged_batch(table, s.dcu, lens, 3)
    q, q64 = rows(torch, np.random.default_rng(0), 3, 128, "f32")
    k, k64 = rows(torch, np.random.default_rng(1), 3, 128, "f32")
    out = torch.empty((3, 1, 128), device="cuda")
    torch.cuda.synchronize()
    gpu.paged_kv_append(s.cache, batch, q, k, k, out, q_heads=1, theta=theta, scaling=scaling)
    pos = length - 3 + np.arange(3)
    # 64-bit references lose 2^-53 of an angle of 2e6 rad: 2e-10, far below the tolerance
    want = rotate64(q64.reshape(3, 1, 128), pos, 128, float(np.float32(theta)), scaling, False)
    size = np.abs(q64).max() * 2
    assert np.abs(out.double().cpu().numpy() - want).max() <= size * 2.0 ** -21


def test_append_rounds_and_grows(gpu, torch):
    """Token by token into one page: each scale is the running maximum, each older code is rounded
    again only where the scale grew; a page begun anew forgets its last scale."""
    s = Setup(torch, [(1, 1)], 2, 16, 16)
    rng = np.random.default_rng(3)
    values = rng.standard_normal((20, 32)).astype(np.float32) * np.linspace(0.1, 3, 20)[:, None].astype(np.float32)
    page = int(s.table[0, 0])
    codes = np.zeros((2, 16, 16))
    scale = np.zeros(2, np.float32)
    for i in range(16):
        x = torch.from_numpy(values[i:i + 1]).cuda()
        s.dlens.fill_(i + 1)
        torch.cuda.synchronize()
        gpu.paged_kv_append(s.cache, s.batch, None, x, x, None, rope=False)
        v = values[i].reshape(2, 16)
        now = np.maximum(scale, np.abs(v).max(1) / np.float32(127)).astype(np.float32)
        codes[:, :i] = np.rint(codes[:, :i] * (scale / now)[:, None, None].astype(np.float32))
        inv = (np.float32(1) / now).astype(np.float32)
        codes[:, i] = np.rint((v * inv[:, None]).astype(np.float32))
        scale = now
        assert np.array_equal(s.dvs[page].cpu().numpy(), scale)
        assert np.array_equal(s.dv[page, :, :i + 1].cpu().numpy(), codes[:, :i + 1].astype(np.int8))
        assert np.array_equal(s.dk[page, :, :i + 1].cpu().numpy(), codes[:, :i + 1].astype(np.int8))
    x = torch.full((1, 32), 1e-3, device="cuda")
    s.dlens.fill_(1)
    torch.cuda.synchronize()
    gpu.paged_kv_append(s.cache, s.batch, None, x, x, None, rope=False)
    assert np.allclose(s.dvs[page].cpu().numpy(), 1e-3 / 127, rtol=1e-6)


def test_append_zeros_nan_and_infinity(gpu, torch):
    s = Setup(torch, [(4, 4)], 1, 16, 16)
    x = torch.zeros((4, 16), device="cuda")
    torch.cuda.synchronize()
    gpu.paged_kv_append(s.cache, s.batch, None, x, x, None, rope=False)
    page = int(s.table[0, 0])
    assert s.dvs[page, 0] == 0 and (s.dv[page, 0, :4] == 0).all()
    x[1, 0], x[1, 1], x[2, 2], x[3, 3], x[3, 4] = float("nan"), 2.0, float("inf"), float("-inf"), -1.0
    torch.cuda.synchronize()
    gpu.paged_kv_append(s.cache, s.batch, None, x, x, None, rope=False)
    assert abs(float(s.dvs[page, 0]) - 2 / 127) < 1e-8
    got = s.dv[page, 0, :4].cpu().numpy()
    want = np.zeros((4, 16), np.int8)
    want[1, 1], want[2, 2], want[3, 3], want[3, 4] = 127, 127, -127, -64
    assert np.array_equal(got, want)


def test_append_in_place_and_odd_strides(gpu, torch):
    """The rotated queries over the queries, rows of an odd stride, q only read where given."""
    hq, hk, d = 3, 2, 48
    s = Setup(torch, SPANS["mixed"], hk, d, 16)
    rng = np.random.default_rng(0)
    width = (hq + 2 * hk) * d
    x = torch.from_numpy(rng.standard_normal((s.tokens, width + 3)).astype(np.float32)).to(torch.bfloat16).cuda()
    x64 = x.double().cpu().numpy()[:, 1:1 + width]
    view = x[:, 1:1 + width]
    q, k, v = view.split([hq * d, hk * d, hk * d], dim=1)
    torch.cuda.synchronize()
    gpu.paged_kv_append(s.cache, s.batch, q, k, v, q, q_heads=hq)
    check_append(s, q, *np.split(x64, [hq * d, (hq + hk) * d], axis=1), hq, "bf16", d)
    assert np.array_equal(view[:, hq * d:].double().cpu().numpy(), x64[:, hq * d:])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift", [16, 8, 4, 1], ids=lambda e: f"from{e}")
@pytest.mark.parametrize("gap", [0, 16, 8, 1], ids=lambda e: f"gap{e}")
@pytest.mark.parametrize("spans", ["decode", "mixed"])
def test_places_of_rotated_queries(gpu, torch, dtype, shift, gap, spans):
    """Rotated queries to bases and rows of every alignment: the same values, nothing beside them."""
    hq, hk, d, ps = 4, 2, 64, 16
    s = Setup(torch, SPANS[spans], hk, d, ps)
    rng = np.random.default_rng(6)
    q = rows(torch, rng, s.tokens, hq * d, dtype)[0]
    k, v = (rows(torch, rng, s.tokens, hk * d, dtype)[0] for _ in range(2))
    width = hq * d + gap
    flat = torch.full((shift + s.tokens * width,), 5.0, dtype=dt(torch, dtype), device="cuda")
    out = flat[shift:].view(s.tokens, width)[:, :hq * d]
    want = torch.empty((s.tokens, hq * d), dtype=dt(torch, dtype), device="cuda")
    torch.cuda.synchronize()
    for o in (out, want):
        gpu.paged_kv_append(s.cache, s.batch, q, k, v, o, q_heads=hq)
    assert torch.equal(out, want)
    assert bool((flat[:shift] == 5).all()) and bool((flat[shift:].view(s.tokens, width)[:, hq * d:] == 5).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("spans", ["one", "decode", "mixed", "prefill"])
@pytest.mark.parametrize("hk,d,ps", [(2, 128, 64), (3, 48, 16), (1, 256, 256)])
@pytest.mark.parametrize("layout", ["rows", "heads", "gaps"])
def test_read(gpu, torch, dtype, spans, hk, d, ps, layout):
    s = Setup(torch, SPANS[spans], hk, d, ps)
    make = lambda *shape: torch.full(shape, 5.0, dtype=dt(torch, dtype), device="cuda")  # noqa: E731
    if layout == "rows":
        outs = [make(s.tokens, hk, d) for _ in range(2)]
    elif layout == "heads":
        outs = [make(hk, s.tokens, d).transpose(0, 1) for _ in range(2)]
    else:
        outs = [make(s.tokens, hk, d + 5)[:, :, :d] for _ in range(2)]
    torch.cuda.synchronize()
    gpu.paged_kv_read(s.cache, s.batch, *outs)
    for which, o in zip("kv", outs):
        codes, scale = (s.k, s.ks) if which == "k" else (s.v, s.vs)
        want = np.concatenate([
            (codes[s.table[b, p // ps], :, p % ps].astype(np.float32) *
             scale[s.table[b, p // ps]][:, None])[None]
            for b, (n, length) in enumerate(s.spans) for p in range(length - n, length)])
        assert torch.equal(o.cpu(), torch.from_numpy(want).to(o.dtype))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift", [16, 8, 4, 1], ids=lambda e: f"from{e}")
@pytest.mark.parametrize("gap", [0, 16, 8, 1], ids=lambda e: f"gap{e}")
@pytest.mark.parametrize("spans", [[(300, 300), (5, 40)], [(5, 40), (1, 300)]], ids=["many", "few"])
def test_places_of_outputs(gpu, torch, dtype, shift, gap, spans):
    """Read-back and attention to bases and rows of every alignment: the same values, nothing beside them."""
    hk, d, ps = 2, 64, 16
    s = Setup(torch, spans, hk, d, ps)
    q, _ = rows(torch, np.random.default_rng(5), s.tokens, hk * d, dtype)
    q = q.view(s.tokens, hk, d)
    width = hk * d + gap
    flat = [torch.full((shift + s.tokens * width,), 5.0, dtype=dt(torch, dtype), device="cuda") for _ in range(3)]
    outs = [x[shift:].view(s.tokens, width)[:, :hk * d] for x in flat]
    dense = [torch.empty((s.tokens, hk * d), dtype=dt(torch, dtype), device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    for k, v, o in (outs, dense):
        gpu.paged_kv_read(s.cache, s.batch, k.unflatten(1, (hk, d)), v.unflatten(1, (hk, d)))
        gpu.paged_attention(s.cache, s.batch, q, o.unflatten(1, (hk, d)))
    for x, o, want in zip(flat, outs, dense):
        assert torch.equal(o, want)
        assert bool((x[:shift] == 5).all()) and bool((x[shift:].view(s.tokens, width)[:, hk * d:] == 5).all())


def test_read_one_output_feeds_attention_f32(gpu, torch):
    """The cache taken out head-major for ATTENTION_F32 gives what PAGED_ATTENTION gives."""
    hk, d, n = 4, 128, 96
    s = Setup(torch, [(n, n)], hk, d, 32)
    k, v = (torch.empty((hk, n, d), device="cuda") for _ in range(2))
    q, q64 = rows(torch, np.random.default_rng(9), n, hk * d, "f32")
    paged, dense = torch.empty((n, hk, d), device="cuda"), torch.empty((hk, n, d), device="cuda")
    torch.cuda.synchronize()
    gpu.paged_kv_read(s.cache, s.batch, k.transpose(0, 1), v.transpose(0, 1))
    gpu.paged_kv_read(s.cache, s.batch, k.transpose(0, 1), None)
    gpu.paged_attention(s.cache, s.batch, q.view(n, hk, d), paged)
    qh = q.view(n, hk, d).transpose(0, 1).contiguous()
    torch.cuda.synchronize()
    gpu.attention(qh, k, v, None, dense, 1, hk, n, n, d, causal=1)
    want, size, most = attention64(s, q64, hk, True, 0)
    check_attention(paged, want, size, most, "f32")
    # ATTENTION_F32's exponential is the reference's degree-5 polynomial: 2e-6 relative
    assert (np.abs(dense.transpose(0, 1).double().cpu().numpy() - want) <=
            most * (2.0 ** -20 * (1 + size) + 2e-5)).all()


# ------------------------------------------------------------------------------------------------
# Streams, graphs, host operands, refusals
# ------------------------------------------------------------------------------------------------
def test_step_in_a_graph_follows_the_device_arrays(gpu, torch):
    """Append and attention captured once: the lengths advance on the device between replays."""
    hq, hk, d, ps = 4, 2, 64, 16
    s = Setup(torch, [(1, 14), (1, 35)], hk, d, ps, slack=0)   # pages for the later tokens
    s.dlens.copy_(torch.tensor([10, 31]))
    qkv = torch.empty((2, (hq + 2 * hk) * d), dtype=torch.bfloat16, device="cuda")
    q, k, v = qkv.split([hq * d, hk * d, hk * d], dim=1)
    q_rot = torch.empty((2, hq, d), dtype=torch.bfloat16, device="cuda")
    o = torch.empty_like(q_rot)
    torch.cuda.synchronize()
    graph = gpu.capture([
        vnpu.paged_kv_append_cmd(s.cache, s.batch, q, k, v, q_rot, q_heads=hq),
        vnpu.paged_attention_cmd(s.cache, s.batch, q_rot, o)])
    for step in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(step)))
        torch.cuda.synchronize()
        gpu.replay(graph)
        assert gpu.sync() == vnpu.OK
        s.k, s.v = s.dk.cpu().numpy(), s.dv.cpu().numpy()
        s.ks, s.vs = s.dks.cpu().numpy(), s.dvs.cpu().numpy()
        s.spans = [(1, 10 + step), (1, 31 + step)]
        q64 = q_rot.double().cpu().numpy().reshape(2, -1)
        check_attention(o, *attention64(s, q64, hq, True, 0), "bf16")
        s.dlens.add_(1)
    gpu.lib.b200_graph_destroy(graph)


@pytest.mark.parametrize("dtype,spans", [("bf16", [(1, 3000), (1, 200)]), ("f32", [(70, 900), (3, 500)])])
def test_graphs_keep_their_own_workspaces(gpu, torch, dtype, spans):
    """Two captured attentions whose parts are joined, replayed in turns: each gives what the plain
    call gives."""
    s = Setup(torch, spans, 2, 128, 64)
    qs = [rows(torch, np.random.default_rng(i), s.tokens, 4 * 128, dtype)[0].view(-1, 4, 128) for i in range(2)]
    want, got = [torch.empty_like(q) for q in qs], [torch.empty_like(q) for q in qs]
    torch.cuda.synchronize()
    for q, o in zip(qs, want):
        gpu.paged_attention(s.cache, s.batch, q, o)
    graphs = [gpu.capture([vnpu.paged_attention_cmd(s.cache, s.batch, q, o)]) for q, o in zip(qs, got)]
    for _ in range(3):
        for o in got:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for g in graphs + graphs:
            gpu.replay(g)
        assert gpu.sync() == vnpu.OK
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for g in graphs:
        gpu.lib.b200_graph_destroy(g)


def test_two_streams_read_one_cache(gpu, torch):
    """Attention on two streams at once, nothing between them: workspaces are not shared."""
    s = Setup(torch, [(1, 6000), (1, 900), (80, 1500)], 2, 128, 64)
    one = vnpu.paged_batch(s.dtable[:2], s.dcu[:3], s.dlens[:2], 2, 1)
    q, q64 = rows(torch, np.random.default_rng(4), s.tokens, 4 * 128, "bf16")
    q = q.view(-1, 4, 128)
    want, size, most = attention64(s, q64, 4, True, 0)
    other = C.c_void_p()
    gpu.lib.check(gpu.lib.stream_create(gpu.dev, 0, C.byref(other)), "stream_create")
    outs = [torch.empty((2 if i % 2 else s.tokens, 4, 128), dtype=torch.bfloat16, device="cuda") for i in range(8)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        cmd = (vnpu.Command * 1)(vnpu.paged_attention_cmd(s.cache, one if i % 2 else s.batch,
                                                          q[:2] if i % 2 else q, o))
        assert gpu.lib.stream_submit(other if i % 4 < 2 else gpu.stream, cmd, 1, None) == vnpu.OK
    assert gpu.sync() == vnpu.OK and gpu.lib.stream_sync(other) == vnpu.OK
    gpu.lib.stream_destroy(other)
    for i, o in enumerate(outs):
        n = len(o)
        check_attention(o, want[:n], size[:n], most[:n], "bf16")


def test_pools_of_more_than_four_gigabytes(gpu, torch):
    """Pages whose offsets pass 32 bits: append, read and attention at the end of a 4.6 GB pool."""
    hk, d, ps, n = 4, 256, 256, 300
    pages = 4_600_000_000 // (hk * d * ps)
    k, v = (torch.empty((pages, hk, ps, d), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((pages, hk), float("nan"), device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, pages // 2 + 7]], dtype=torch.int32, device="cuda")
    cu, lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, n], [n]))
    cache, batch = vnpu.paged_cache(k, v, ks, vs), vnpu.paged_batch(table, cu, lens, n)
    x = torch.randn((3, n, hk, d), generator=torch.Generator().manual_seed(1)).cuda()
    back = torch.empty((2, n, hk, d), device="cuda")
    q, o = torch.empty_like(x[0]), torch.empty_like(x[0])
    torch.cuda.synchronize()
    gpu.paged_kv_append(cache, batch, x[0].flatten(1), x[1].flatten(1), x[2].flatten(1), q.flatten(1),
                        q_heads=hk, rope=False)
    gpu.paged_kv_read(cache, batch, back[0], back[1])
    step = x[1:].abs().amax() / 127
    assert (back - x[1:]).abs().max() <= 0.5001 * step
    gpu.paged_attention(cache, batch, q, o)
    w = torch.einsum("qhd,khd->hqk", x[0].double(), back[0].double()) / 16
    w = w.masked_fill(torch.ones((n, n), device="cuda").triu(1).bool(), -float("inf")).softmax(-1)
    want = torch.einsum("hqk,khd->qhd", w, back[1].double())
    assert (o.double() - want).abs().max() <= back[1].abs().max() * 2.0 ** -20 * (1 + 16 * 4 * 4)


def test_host_rows_are_staged(gpu, torch):
    hq, hk, d = 2, 2, 64
    s = Setup(torch, SPANS["mixed"], hk, d, 16)
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal((s.tokens, hq * d)).astype(np.float32) for _ in range(3))
    q_out, o = np.empty_like(q), np.empty_like(q)
    batch = vnpu.PagedBatch(vnpu.ptr(s.table), vnpu.ptr(s.cu), vnpu.ptr(s.lens), len(s.spans),
                            s.table.shape[1], s.tokens, 0)
    gpu._run(vnpu.b200_command(vnpu.OP_B200_PAGED_KV_APPEND, vnpu.PagedKvAppendArgs(
        s.cache, batch, vnpu.ptr(q), vnpu.ptr(k), vnpu.ptr(v), vnpu.ptr(q_out), 0, 0, 0, 0, hq, 0,
        0, 0, 0.0, 0.0)), "append")
    check_append(s, torch.from_numpy(q_out), q.astype(np.float64), k.astype(np.float64),
                 v.astype(np.float64), hq, "f32", d)
    s.k, s.v = s.dk.cpu().numpy(), s.dv.cpu().numpy()
    s.ks, s.vs = s.dks.cpu().numpy(), s.dvs.cpu().numpy()
    gpu._run(vnpu.b200_command(vnpu.OP_B200_PAGED_ATTENTION, vnpu.PagedAttentionArgs(
        s.cache, batch, vnpu.ptr(q_out), vnpu.ptr(o), 0, 0, hq, 0, 1, 0, 0, 0.0)), "attention")
    want = attention64(s, q_out.astype(np.float64), hq, True, 0)
    check_attention(torch.from_numpy(o).view(s.tokens, hq, d), *want, "f32")


def test_no_rows_is_no_work(gpu, torch):
    s = Setup(torch, [(0, 20), (0, 0)], 1, 64, 16)
    before = s.dk.clone()
    one = torch.full((1, 1, 64), 3.0, device="cuda")
    torch.cuda.synchronize()
    for args, op in ((vnpu.PagedKvAppendArgs(s.cache, s.batch, None, one.data_ptr(), one.data_ptr(),
                                             None, 0, 0, 0, 0, 0, 0, 0, 0, 0.0, 0.0),
                      vnpu.OP_B200_PAGED_KV_APPEND),
                     (vnpu.PagedKvReadArgs(s.cache, s.batch, one.data_ptr(), None, 0, 0, 0, 0),
                      vnpu.OP_B200_PAGED_KV_READ),
                     (vnpu.PagedAttentionArgs(s.cache, s.batch, one.data_ptr(), one.data_ptr(), 0, 0,
                                              1, 0, 1, 0, 0, 0.0), vnpu.OP_B200_PAGED_ATTENTION)):
        gpu._run(vnpu.b200_command(op, args), "no work")
        s.batch.batch = 0
        gpu._run(vnpu.b200_command(op, args), "no work")
        s.batch.batch = 2
    assert torch.equal(before, s.dk) and (one == 3.0).all()


def _status(lib, cmd):
    """Status of one command on a device of its own: the event's, and the sync's after it."""
    with vnpu.Device(lib) as dev:
        ev = C.c_void_p()
        lib.check(lib.event_create(C.byref(ev)), "event")
        arr = (vnpu.Command * 1)(cmd)
        assert lib.stream_submit(dev.stream, arr, 1, ev) == vnpu.OK
        st, sync = lib.event_wait(ev, 5000), dev.sync()
        lib.event_destroy(ev)
        return st, sync


BAD_CACHE = [("K", None), ("V_scale", None), ("num_pages", 0), ("heads", 0), ("page_size", 48),
             ("page_size", 8), ("page_size", 512), ("head_dim", 24), ("head_dim", 272),
             ("head_dim", 0), ("K", "odd"), ("V", "host")]


@pytest.mark.parametrize("field,value", BAD_CACHE)
def test_refused_caches(b200_lib, gpu, torch, field, value):
    s = Setup(torch, [(1, 20)], 1, 64, 16)
    host = np.zeros(64, np.int8)
    if value == "odd":
        value = s.dk.data_ptr() + 8
    elif value == "host":
        value = host.ctypes.data
    x = torch.zeros((1, 1, 64), device="cuda")
    cache = vnpu.PagedCache.from_buffer_copy(s.cache)
    setattr(cache, field, value)
    torch.cuda.synchronize()
    before = s.dk.clone()
    for cmd in (vnpu.b200_command(vnpu.OP_B200_PAGED_KV_APPEND, vnpu.PagedKvAppendArgs(
                    cache, s.batch, None, x.data_ptr(), x.data_ptr(), None, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)),
                vnpu.b200_command(vnpu.OP_B200_PAGED_KV_READ, vnpu.PagedKvReadArgs(
                    cache, s.batch, x.data_ptr(), x.data_ptr(), 0, 0, 0, 0)),
                vnpu.b200_command(vnpu.OP_B200_PAGED_ATTENTION, vnpu.PagedAttentionArgs(
                    cache, s.batch, x.data_ptr(), x.data_ptr(), 0, 0, 1, 0, 1, 0, 0, 0))):
        event, sync = _status(b200_lib, cmd)
        assert event != vnpu.OK and sync == vnpu.ERR_DEVICE_ERROR
    assert torch.equal(before, s.dk)


def test_refused_arguments(b200_lib, gpu, torch):
    s = Setup(torch, [(1, 20)], 2, 64, 16)
    x = torch.zeros((1, 2, 64), device="cuda")
    p = x.data_ptr()
    torch.cuda.synchronize()
    append = lambda **kw: vnpu.b200_command(vnpu.OP_B200_PAGED_KV_APPEND, vnpu.PagedKvAppendArgs(  # noqa: E731
        **{**dict(cache=s.cache, batch=s.batch, Q=p, K=p, V=p, Q_out=p, q_heads=2), **kw}))
    attend = lambda **kw: vnpu.b200_command(vnpu.OP_B200_PAGED_ATTENTION, vnpu.PagedAttentionArgs(  # noqa: E731
        **{**dict(cache=s.cache, batch=s.batch, Q=p, O=p, q_heads=2, causal=1), **kw}))
    read = lambda **kw: vnpu.b200_command(vnpu.OP_B200_PAGED_KV_READ, vnpu.PagedKvReadArgs(  # noqa: E731
        **{**dict(cache=s.cache, batch=s.batch, K_out=p), **kw}))
    no_table = vnpu.PagedBatch.from_buffer_copy(s.batch)
    no_table.block_table = None
    no_stride = vnpu.PagedBatch.from_buffer_copy(s.batch)
    no_stride.table_stride = 0
    bad = [append(K=None), append(Q=None), append(Q_out=None), append(q_heads=0), append(flags=4),
           append(rotary_dim=80), append(rotary_dim=24), append(dtype=3), append(ldk=64),
           append(K=p + 2), append(ldq=256, ldqo=0), append(batch=no_table), append(batch=no_stride),
           attend(q_heads=3), attend(q_heads=0), attend(Q=None), attend(O=None), attend(causal=2),
           attend(dtype=5), attend(ldq=100), attend(scale=float("nan")), attend(Q=p + 1),
           attend(batch=no_table), read(K_out=None), read(dtype=4), read(ld_head=32), read(ld_row=32),
           read(K_out=p + 2)]
    for cmd in bad:
        event, sync = _status(b200_lib, cmd)
        assert event != vnpu.OK and sync == vnpu.ERR_DEVICE_ERROR


@pytest.mark.parametrize("what", ["page", "negative page", "length", "short length", "rows",
                                  "max_tokens", "falling"])
def test_device_arrays_are_checked(b200_lib, gpu, torch, what):
    """Arrays that point outside the cache, the table or the rows: the kernels leave the sequence
    out and the stream reports it; the other sequence and the rest of memory are untouched."""
    hq, hk, d = 2, 1, 64
    s = Setup(torch, [(2, 40), (2, 20)], hk, d, 16)
    table, cu, lens, tokens, most = s.dtable.clone(), s.dcu.clone(), s.dlens.clone(), 4, 2
    if what == "page":
        table[0] = s.pages
    elif what == "negative page":
        table[0] = -1
    elif what == "length":
        lens[0] = 16 * table.shape[1] + 1
    elif what == "short length":
        lens[0] = 1
    elif what == "rows":
        cu[2] = 5
    elif what == "max_tokens":
        most = 1
    else:
        cu[1] = 5
    batch = vnpu.paged_batch(table, cu, lens, tokens, most)
    x = torch.randn((4, (hq + 2 * hk) * d), device="cuda")
    q, k, v = x.split([hq * d, hk * d, hk * d], dim=1)
    out = torch.zeros((4, hq, d), device="cuda")
    back = torch.zeros((4, hk, d), device="cuda")
    torch.cuda.synchronize()
    for cmd in (vnpu.paged_kv_append_cmd(s.cache, batch, q, k, v, out, q_heads=hq),
                vnpu.paged_kv_read_cmd(s.cache, batch, back, None),
                vnpu.paged_attention_cmd(s.cache, batch, out, out.clone())):
        _, sync = _status(b200_lib, cmd)
        assert sync == vnpu.ERR_DEVICE_ERROR
    seen = set(s.table[0, :3]) | set(s.table[1, :2])
    rest = [p for p in range(s.pages) if p not in seen]
    assert np.array_equal(s.dk.cpu().numpy()[rest], s.k[rest])
    assert (gpu.sync()) == vnpu.OK


@pytest.mark.parametrize("bad", range(5))
def test_every_single_token_sequence_is_checked(b200_lib, gpu, torch, bad):
    """One token a sequence, one bad page among five: reported wherever it is, the others appended."""
    s = Setup(torch, [(1, 10 + i) for i in range(5)], 1, 64, 16)
    table = s.dtable.clone()
    table[bad] = s.pages + 5
    batch = vnpu.paged_batch(table, s.dcu, s.dlens, 5, 1)
    x = torch.full((5, 64), 50.0, device="cuda")
    q = torch.zeros((5, 1, 64), device="cuda")
    torch.cuda.synchronize()
    cmds = [vnpu.paged_kv_append_cmd(s.cache, batch, None, x, x, None, rope=False),
            vnpu.paged_kv_read_cmd(s.cache, batch, q.clone(), None),
            vnpu.paged_attention_cmd(s.cache, batch, q, q.clone())]
    for cmd in cmds:
        _, sync = _status(b200_lib, cmd)
        assert sync == vnpu.ERR_DEVICE_ERROR
    for b in range(5):
        new = s.dv[int(s.table[b, 0]), 0, 9 + b].cpu()
        if b != bad:
            assert (new == 127).all()
        else:
            assert np.array_equal(new, s.v[int(s.table[b, 0]), 0, 9 + b])


def test_python_helpers_refuse(torch):
    k = torch.zeros((2, 1, 16, 64), dtype=torch.int8)
    sc = torch.zeros((2, 1))
    with pytest.raises(ValueError):
        vnpu.paged_cache(k, k[:1], sc, sc)
    with pytest.raises(ValueError):
        vnpu.paged_cache(k.float(), k, sc, sc)
    cache = vnpu.paged_cache(k, k, sc, sc)
    i = torch.zeros((1, 1), dtype=torch.int32)
    with pytest.raises(TypeError):
        vnpu.paged_batch(i.long(), i[0].repeat(2), i[0], 1)
    with pytest.raises(ValueError):
        vnpu.paged_batch(i, i[0], i[0], 1)
    batch = vnpu.paged_batch(i, i[0].repeat(2), i[0], 1)
    x = torch.zeros((1, 2, 64))
    with pytest.raises(TypeError):
        vnpu.paged_attention_cmd(cache, batch, x, x.half())
    with pytest.raises(ValueError):
        vnpu.paged_attention_cmd(cache, batch, x[:, :, ::2], x)
