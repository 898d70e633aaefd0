"""What the paged kernels' numbers promise, where it is hardest to keep.

Bounds follow from the arithmetic, each beside its use.  Scores are off by 2^-21 of sum |q||k| scale
("size"), so a softmax weight by 2^-20 (1 + size) relatively with the exponential's part; 16-bit rows
round weights to 11 bits more.
"""
from __future__ import annotations

import numpy as np
import pytest

import vnpu
from test_gpu_paged import HALF_ULP, Setup, attention64, dt, rows, torch  # noqa: F401

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


# ------------------------------------------------------------------------------------------------
# Long runs of keys
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("length", [1024, 8192, 32768, 131072])
@pytest.mark.parametrize("rows_of", ["few", "many"])
def test_error_does_not_grow_with_the_keys(gpu, torch, dtype, length, rows_of):
    """Every CTA walks all keys of its rows (as many row tiles as CTAs, one shared prefix): the
    error against the output's own size, which falls with the keys, stays what it is at 1024.

    An output is a weighted mean of values of either sign; errors of the weights (2^-20 (1 + size),
    each its own) come out as that part of the output's rms, 16-bit weights as 2^-11 / sqrt(12) of
    it, and the output's rounding as at most its half unit in the last place.  What is common to all
    weights (a sum that is not rounded to nearest) is a part of the output itself: 2^-19."""
    hk, d, ps = 4, 128, 64
    g, batch, n = (1, 112, 1) if rows_of == "few" else (4, 37, 64)      # x 4 heads: 448 and 148 row tiles
    hq, pages = g * hk, length // ps
    gen = torch.Generator(device="cuda").manual_seed(length)
    k, v = (torch.randint(-127, 128, (pages, hk, ps, d), generator=gen, device="cuda", dtype=torch.int8)
            for _ in range(2))
    ks, vs = (torch.rand((pages, hk), generator=gen, device="cuda") * 0.01 + 0.01 for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(batch, 1)
    cu = torch.arange(0, (batch + 1) * n, n, dtype=torch.int32, device="cuda")
    lens = torch.full((batch,), length, dtype=torch.int32, device="cuda")
    q = torch.randn((batch * n, hq, d), generator=gen, device="cuda").to(dt(torch, dtype))
    o = torch.empty_like(q)
    torch.cuda.synchronize()
    gpu.paged_attention(vnpu.paged_cache(k, v, ks, vs), vnpu.paged_batch(table, cu, lens, batch * n, n), q, o,
                        causal=False)
    sample = torch.arange(0, batch * n, 37 if rows_of == "many" else 1, device="cuda")[:112]
    error = square = size = 0.0
    for h in range(hq):
        kk = (k[:, h // g].double() * ks[:, h // g, None, None].double()).reshape(length, d)
        vv = (v[:, h // g].double() * vs[:, h // g, None, None].double()).reshape(length, d)
        x = q[sample, h].double()
        w = torch.softmax((x @ kk.T) / d ** 0.5, -1)
        want = w @ vv
        size = max(size, float((x.abs() @ kk.abs().T).max()) / d ** 0.5)
        error += float((o[sample, h].double() - want).square().sum())
        square += float(want.square().sum())
    tol = 2.0 ** -20 * (1 + size) + 2.0 ** -19
    if dtype == "f16":
        tol += 2.0 ** -11 / 12 ** 0.5 + HALF_ULP[dtype]
    assert error ** 0.5 <= tol * square ** 0.5, (error / square) ** 0.5 / tol


# ------------------------------------------------------------------------------------------------
# One key
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [1e-25, 1e-9, 1e-4, 1.0, 1e3, 1e20])
@pytest.mark.parametrize("spans", [[(1, 200), (5, 70)], [(130, 300)]], ids=["few", "many"])
def test_one_key_gives_its_value(gpu, torch, dtype, size, spans):
    """A window of one: the output is the cached value, whatever its page's scale.  A weight is rounded
    to 22 bits (11 for 16-bit rows), the scale's reciprocal by 2^-23, the sum, its reciprocal and the
    output's product by 2^-24 each."""
    if dtype == "f16" and size not in (1e-4, 1.0):
        pytest.skip("past what f16 holds")
    hk, d, ps = 2, 64, 16
    s = Setup(torch, spans, hk, d, ps)
    s.vs *= np.float32(size)
    s.dvs.copy_(torch.from_numpy(s.vs))
    q, _ = rows(torch, np.random.default_rng(3), s.tokens, hk * d, dtype)
    o = torch.empty((s.tokens, hk, d), dtype=q.dtype, device="cuda")
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, s.batch, q.view(s.tokens, hk, d), o, window=1)
    want = []
    for b, (n, length) in enumerate(spans):
        v, vs = s.seq_codes("v", b)
        want.append((v * vs[:, :, None])[length - n:])
    want = np.concatenate(want)
    part = (2.0 ** -22 if dtype == "f32" else 2.0 ** -11) + 2.0 ** -23 + 4 * 2.0 ** -24
    off = np.abs(o.double().cpu().numpy() - want)
    tol = np.abs(want) * (part + HALF_ULP[dtype]) + (2.0 ** -25 if dtype == "f16" else 0)
    assert (off <= tol).all(), (off / (tol + 1e-300)).max()


# ------------------------------------------------------------------------------------------------
# Rows of one sign
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("spans", ["few", "many"])
@pytest.mark.parametrize("size", [50, 1000, 16000])
def test_scores_of_rows_of_one_sign(gpu, torch, dtype, spans, size):
    """Two keys with scores of thousands, a few units apart, values +1 and -1: the output is
    tanh((s0 - s1) / 2), which shows the scores' errors.  All query elements are positive.

    Each score may be off by 2^-21 of its size (16-bit queries are exact), the output by half their
    difference's error; weights of 16-bit rows by 2^-11, f32 queries have 22 bits: another 2^-22."""
    d, ps, n = 128, 16, 600
    rng = np.random.default_rng(size)
    s = Setup(torch, [(1, 2)] * n if spans == "few" else [(200, 200)] * 3, 1, d, ps)
    if spans == "few":
        q = rng.uniform(0.5, 1.5, (n, d))
        k0 = rng.integers(-127, 128, (n, d))
        k1 = k0.copy()
        for _ in range(6):             # moves of one code from one place to another: sums stay alike
            i, j = rng.integers(0, d, (2, n))
            r = np.arange(n)
            step = np.minimum(rng.integers(1, 40, n), np.minimum(127 - k1[r, i], 127 + k1[r, j]))
            k1[r, i] += step
            k1[r, j] -= step
        s.k[s.table[:, 0], 0, 0], s.k[s.table[:, 0], 0, 1] = k0, k1
        s.v[s.table[:, 0], 0, 0], s.v[s.table[:, 0], 0, 1] = 127, -127
    else:
        # keys in pairs within a page, only the first two of each sequence are near the top
        q = rng.uniform(0.5, 1.5, (600, d))
        for b in range(3):
            for page in s.table[b, :13]:
                s.k[page] = -127
                s.v[page] = 127
            page = s.table[b, 0]
            k0 = rng.integers(-60, 128, d)
            k1 = k0.copy()
            for _ in range(6):
                i, j = rng.integers(0, d, 2)
                step = min(int(rng.integers(1, 40)), 127 - k1[i], 127 + k1[j])
                k1[i] += step
                k1[j] -= step
            s.k[page, 0, 0], s.k[page, 0, 1] = k0, k1
            s.v[page, 0, 0], s.v[page, 0, 1] = 127, -127
    s.ks[:], s.vs[:] = 1 / 64, 1 / 127
    for x, y in ((s.dk, s.k), (s.dv, s.v), (s.dks, s.ks), (s.dvs, s.vs)):
        x.copy_(torch.from_numpy(y))
    q = torch.from_numpy(q.astype(np.float32)).to(dt(torch, dtype)).cuda()
    scale = size / (d * 1.0)                               # |q| is 1 and |k| 1 on the average
    scale = float(np.float32(scale))
    o = torch.empty((s.tokens, 1, d), dtype=q.dtype, device="cuda")
    torch.cuda.synchronize()
    gpu.paged_attention(s.cache, s.batch, q.view(-1, 1, d), o, causal=False, scale=scale)
    want, sizes, _ = attention64(s, q.double().cpu().numpy(), 1, False, 0, scale)
    assert (np.abs(want) < 0.9).mean() > (0.02 if size > 1000 else 0.1)     # rows that show something
    tol = sizes * 2.0 ** -21 * (1.5 if dtype == "f32" else 1) + 2.0 ** -20
    tol = tol + (0 if dtype == "f32" else 2.0 ** -11) + np.abs(want) * HALF_ULP[dtype]
    off = np.abs(o.double().cpu().numpy() - want)
    assert (off <= tol).all(), ((off / tol).max(), (off > tol).sum())


# ------------------------------------------------------------------------------------------------
# Append: angles and codes
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("single", [True, False], ids=["single", "runs"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_angles_of_keys(gpu, torch, single, interleaved):
    """One pair (1, 0) a head and page: the page's scale is the larger of |cos| and |sin| over 127,
    in 32 bits.  The angle is off by 2^-24 of at most pi/4 off a quarter turn, sine and cosine by 2
    units in the last place (2^-23 of values above 1/2), the scale's division by half a unit."""
    d, ps, hk, n = 16, 16, 8, 512
    rng = np.random.default_rng(7)
    starts = rng.integers(0, 200_000, n) // ps * ps         # each token opens a page
    table = np.full((n, 200_000 // ps + 1), -1, np.int32)
    table[np.arange(n), starts // ps] = np.arange(n)
    k = torch.zeros((n, hk, d), device="cuda")
    for h in range(hk):
        k[:, h, 2 * h if interleaved else h] = 1.0
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
    codes = [torch.zeros((n, hk, ps, d), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((n, hk), device="cuda") for _ in range(2)]
    cache = vnpu.paged_cache(*codes, *scales)
    batch = vnpu.paged_batch(dev(table), dev(np.arange(n + 1)), dev(starts + 1), n, 1 if single else 2)
    torch.cuda.synchronize()
    gpu.paged_kv_append(cache, batch, None, k.flatten(1), k.flatten(1), None, interleaved=interleaved)
    angle = starts[:, None] * 10000.0 ** (-2.0 * np.arange(hk) / d)
    want = np.maximum(np.abs(np.cos(angle)), np.abs(np.sin(angle))) / 127
    off = np.abs(scales[0].double().cpu().numpy() / want - 1)
    assert off.max() <= np.pi / 4 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -24 + 1e-10, off.max()


@pytest.mark.parametrize("single", [True, False], ids=["single", "runs"])
def test_codes_are_to_nearest(gpu, torch, single):
    """A code is x / scale to nearest: off by half a code and the 32-bit quotient's rounding, 2^-24
    of at most 127.  Whole and half multiples of a scale that is no power of two go to even."""
    d, ps, hk = 256, 16, 4
    n = 1024
    rng = np.random.default_rng(8)
    x = rng.standard_normal((n, hk, d)).astype(np.float32)
    x[:16, 0] = rng.integers(-254, 255, (16, d)) * np.float32(1.5)     # scale 3, halves of it
    x[:16, 0, 0] = 381.0
    spans = [(1, 1)] * n if single else [(n, n)]
    s = Setup(torch, spans, hk, d, ps)
    if single:
        x[::7, 0] = rng.integers(-254, 255, x[::7, 0].shape) * np.float32(1.5)
        x[::7, 0, 0] = 381.0
    dx = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    gpu.paged_kv_append(s.cache, s.batch, None, dx.flatten(1), dx.flatten(1), None, rope=False)
    for codes, scale in ((s.dk, s.dks), (s.dv, s.dvs)):
        codes, scale = codes.cpu().numpy().astype(np.float64), scale.cpu().numpy().astype(np.float64)
        if single:
            got, per = codes[s.table[:, 0], :, 0], scale[s.table[:, 0]]
        else:
            pages = s.table[0, :n // ps]
            got = codes[pages].transpose(0, 2, 1, 3).reshape(n, hk, d)
            per = np.repeat(scale[pages], ps, 0)
        y = x / per[:, :, None]
        off = np.abs(got - y)
        assert off.max() <= 0.5 + 127 * 2.0 ** -24, off.max() - 0.5
        halves = np.abs(y - np.trunc(y)) == 0.5
        assert halves.sum() > 100 and np.array_equal(got[halves], np.rint(y[halves]))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_codes_of_16_bit_values(gpu, torch, dtype):
    """16-bit values are often exactly between two codes of their largest over 127, though not of that
    scale's 32-bit rounding: the code is the 32-bit quotient's nearest, ties to even, to the bit."""
    d, ps, hk, n = 128, 64, 8, 1024
    s = Setup(torch, [(n, n)], hk, d, ps)
    x = torch.randn((n, hk * d), generator=torch.Generator().manual_seed(4)).to(
        torch.bfloat16 if dtype == "f32" else dt(torch, dtype)).to(dt(torch, dtype)).cuda()
    torch.cuda.synchronize()
    gpu.paged_kv_append(s.cache, s.batch, None, x, x, None, rope=False)
    x = x.float().cpu().numpy().reshape(n, hk, d)
    for codes, scale in ((s.dk, s.dks), (s.dv, s.dvs)):
        pages = s.table[0, :n // ps]
        got = codes.cpu().numpy()[pages].transpose(0, 2, 1, 3).reshape(n, hk, d)
        per = np.repeat(scale.cpu().numpy()[pages], ps, 0)[:, :, None]
        assert np.array_equal(per, np.repeat(np.abs(x).reshape(-1, ps, hk, d).max((1, 3)) / np.float32(127), ps, 0)[:, :, None])
        assert np.array_equal(got, np.rint(x / per).astype(np.int8))
