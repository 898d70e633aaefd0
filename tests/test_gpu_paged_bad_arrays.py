"""Device arrays that describe no rows, pages or tokens, with enough rows for the many-row kernel of
PAGED_ATTENTION (more than 48 a key/value head): found on the device, left out and reported."""
from __future__ import annotations

import numpy as np
import pytest

import vnpu
from test_gpu_paged import Setup, _status, attention64, check_attention, rows, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def guarded(torch, tokens, heads, d, dtype, fill=7.0):
    """An output with rows before and after it that nothing may write."""
    flat = torch.full((tokens + 64, heads, d), fill, dtype=dtype, device="cuda")
    return flat, flat[32:32 + tokens]


@pytest.mark.parametrize("dtype,d", [("f32", 128), ("bf16", 64), ("f16", 128)])
@pytest.mark.parametrize("batch", [9, 40, 1500])
def test_rows_that_fall_and_rise_again(b200_lib, gpu, torch, dtype, d, batch):
    """cu = 0, T, 0, T, ...: every second sequence looks right by itself, together they have far
    more blocks of rows than `tokens` has (room for T * group / 256 + batch)."""
    n, hq, hk = 300, 8, 2
    s = Setup(torch, [(n, n)], hk, d, 16)
    need = (batch + 1) // 2 * -(-n * 4 // 256)
    assert need > n * 4 // 256 + batch
    cu = torch.tensor([0, n] * (batch // 2 + 1), dtype=torch.int32)[:batch + 1].cuda()
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    table = s.dtable.repeat(batch, 1)
    q, _ = rows(torch, np.random.default_rng(0), n, hq * d, dtype)
    flat, o = guarded(torch, n, hq, d, q.dtype)
    torch.cuda.synchronize()
    _, sync = _status(b200_lib, vnpu.paged_attention_cmd(
        s.cache, vnpu.paged_batch(table, cu, lens, n), q.view(n, hq, d), o))
    assert sync == vnpu.ERR_DEVICE_ERROR
    assert bool((flat == 7).all())
    # and the same stream's good numbers right after
    gpu.paged_attention(s.cache, s.batch, q.view(n, hq, d), o)
    check_attention(o, *attention64(s, q.double().cpu().numpy(), hq, True, 0), dtype)
    assert bool((flat[:32] == 7).all()) and bool((flat[-32:] == 7).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("what", ["page", "negative page", "length", "short length", "negative length",
                                  "rows", "max_tokens", "falling", "negative rows"])
def test_bad_numbers_of_many_rows(b200_lib, gpu, torch, dtype, what):
    hq, hk, d = 4, 2, 64
    s = Setup(torch, [(70, 90), (60, 200)], hk, d, 16)
    table, cu, lens, tokens, most = s.dtable.clone(), s.dcu.clone(), s.dlens.clone(), 130, 70
    if what == "page":
        table[0] = s.pages
    elif what == "negative page":
        table[0] = -1
    elif what == "length":
        lens[0] = 16 * table.shape[1] + 1
    elif what == "short length":
        lens[0] = 69
    elif what == "negative length":
        lens[0] = -5
    elif what == "rows":
        cu[2] = 131
    elif what == "max_tokens":
        most = 65
    elif what == "falling":
        cu[1] = 130 + 1
    else:
        cu[0] = -1
    q, q64 = rows(torch, np.random.default_rng(1), tokens, hq * d, dtype)
    flat, o = guarded(torch, tokens, hq, d, q.dtype)
    torch.cuda.synchronize()
    _, sync = _status(b200_lib, vnpu.paged_attention_cmd(
        s.cache, vnpu.paged_batch(table, cu, lens, tokens, most), q.view(tokens, hq, d), o))
    assert sync == vnpu.ERR_DEVICE_ERROR
    assert bool((flat[:32] == 7).all()) and bool((flat[-32:] == 7).all())
    bad = {"rows": 1, "falling": 2}.get(what, 0)        # the sequence left out; 2: both
    want, size, top = attention64(s, q64, hq, True, 0)
    if bad != 1 and "page" not in what:
        assert bool((o[:70] == 7).all())
    if bad == 0:
        check_attention(o[70:], want[70:], size[70:], top[70:], dtype)
    elif bad == 1:
        check_attention(o[:70], want[:70], size[:70], top[:70], dtype)
        assert bool((o[70:] == 7).all())
    assert bool(torch.isfinite(o).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_steps_than_can_be_counted(b200_lib, torch, dtype):
    """Every page the same one, 2^31 keys, 256 and 512 blocks of rows: nearly 2^33 steps of 256
    rows by a tile of keys.  Left out and reported, nothing is written."""
    n = 1024 if dtype == "f32" else 2048                   # tiles of 64 and of 128 keys
    heads, d, ps, length = 64, 16, 256, 0x7fffff00
    codes = torch.zeros((1, 1, ps, d), dtype=torch.int8, device="cuda")
    scale = torch.ones((1, 1), device="cuda")
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.zeros((1, length // ps + 1), dtype=torch.int32, device="cuda")
    q = torch.zeros((n, heads, d), device="cuda").to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    flat, o = guarded(torch, n, heads, d, q.dtype)
    assert (n * heads // 256) * ((length - n) // (64 if dtype == "f32" else 128)) >= 2 ** 32
    torch.cuda.synchronize()
    _, sync = _status(b200_lib, vnpu.paged_attention_cmd(
        vnpu.paged_cache(codes, codes, scale, scale),
        vnpu.paged_batch(table, ints(0, n), ints(length), n), q, o))
    assert sync == vnpu.ERR_DEVICE_ERROR
    assert bool((flat == 7).all())
