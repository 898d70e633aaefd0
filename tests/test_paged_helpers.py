"""The packet builders of the paged cache refuse tensors that the kernels would read or write past:
fewer rows than the batch has tokens, rows that are one and the same, other element types."""
from __future__ import annotations

import pytest

import vnpu

torch = pytest.importorskip("torch")


@pytest.fixture
def cache():
    k, scale = torch.zeros((3, 2, 16, 32), dtype=torch.int8), torch.zeros((3, 2))
    return vnpu.paged_cache(k, k.clone(), scale, scale.clone())


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.fixture
def batch():
    return vnpu.paged_batch(torch.zeros((2, 3), dtype=torch.int32), ints(0, 3, 4), ints(3, 1), 4)


def rows(n=4, heads=2, d=32, dtype=torch.float32):
    return torch.zeros((n, heads * d), dtype=dtype)


def test_good_rows_pass(cache, batch):
    q, k, v = torch.zeros((6, 8 * 32)).split([128, 64, 64], dim=1)           # more rows than tokens
    vnpu.paged_kv_append_cmd(cache, batch, q, k, v, q, q_heads=4)
    vnpu.paged_kv_append_cmd(cache, batch, None, k, v, None)
    for out in (torch.zeros((4, 2, 32)), torch.zeros((2, 5, 32)).transpose(0, 1), torch.zeros((4, 2, 40))[:, :, :32]):
        vnpu.paged_kv_read_cmd(cache, batch, out, out)
    o = torch.zeros((4, 4, 32))
    vnpu.paged_attention_cmd(cache, batch, o, o)
    one = vnpu.paged_batch(torch.zeros((1, 3), dtype=torch.int32), ints(0, 1), ints(1), 1)
    vnpu.paged_attention_cmd(cache, one, o[:1], o[:1])
    vnpu.paged_kv_append_cmd(cache, one, None, k[:1].expand(1, -1), v[:1], None)


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("what", ["short", "broadcast", "overlapping", "wide"])
def test_append_rows(cache, batch, which, what):
    args = [rows(heads=4), rows(), rows(), rows(heads=4)]
    width = args[which].shape[1]
    args[which] = {"short": args[which][:3], "broadcast": args[which][:1].expand(4, -1),
                   "overlapping": torch.zeros(5 * width).as_strided((4, width), (width // 2, 1)),
                   "wide": torch.zeros((4, width + 1))}[what]
    with pytest.raises(ValueError):
        vnpu.paged_kv_append_cmd(cache, batch, *args, q_heads=4)


@pytest.mark.parametrize("which", range(2))
@pytest.mark.parametrize("what", ["short", "one row", "one head"])
def test_read_outputs(cache, batch, which, what):
    bad = {"short": torch.zeros((3, 2, 32)), "one row": torch.zeros((1, 2, 32)).expand(4, -1, -1),
           "one head": torch.zeros((4, 1, 32)).expand(-1, 2, -1)}[what]
    good = torch.zeros((4, 2, 32)) if what == "short" else None
    for pair in ((bad, good), (good, bad), (bad, bad.clone() if what == "short" else bad)):
        with pytest.raises(ValueError):
            vnpu.paged_kv_read_cmd(cache, batch, *(pair if which == 0 else pair[::-1]))


@pytest.mark.parametrize("which", range(2))
@pytest.mark.parametrize("what", ["short", "broadcast"])
def test_attention_rows(cache, batch, which, what):
    args = [torch.zeros((4, 4, 32)) for _ in range(2)]
    args[which] = args[which][:3] if what == "short" else args[which][:1].expand(4, -1, -1)
    with pytest.raises(ValueError):
        vnpu.paged_attention_cmd(cache, batch, *args)


def test_types_and_tables(cache):
    k, scale = torch.zeros((3, 2, 16, 32), dtype=torch.int8), torch.zeros((3, 2))
    with pytest.raises(ValueError):
        vnpu.paged_cache(k.to(torch.uint8), k, scale, scale)
    table = torch.zeros((2, 3), dtype=torch.int32)
    with pytest.raises(TypeError):
        vnpu.paged_batch(table.to(torch.uint32), ints(0, 3, 4), ints(3, 1), 4)
    with pytest.raises(ValueError):
        vnpu.paged_batch(table[:1].expand(2, -1), ints(0, 3, 4), ints(3, 1), 4)


def test_table_rows_are_whole(cache):
    """Some columns of a wider table: its rows are read by their stride, the last one too."""
    wide = torch.zeros((3, 8), dtype=torch.int32)
    cu, lens = ints(0, 1, 2, 3), ints(1, 1, 1)
    assert vnpu.paged_batch(wide[:, :5], cu, lens, 3).table_stride == 8
    assert vnpu.paged_batch(wide[:2, 4:], cu[:3], lens[:2], 2).table_stride == 8
    with pytest.raises(ValueError):
        vnpu.paged_batch(wide[:, 4:], cu, lens, 3)
    assert vnpu.paged_batch(wide[2:, 4:], cu[:2], lens[:1], 1).table_stride == 4
