"""PAGED_KV_READ into host memory: the same bytes as into device memory, whatever the layout."""
from __future__ import annotations

import numpy as np
import pytest

import vnpu
from test_gpu_paged import SPANS, Setup, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["apart", "rows", "heads", "tokens", "head rows", "one"])
@pytest.mark.parametrize("spans", ["one", "mixed", "prefill"])
def test_read_to_host_memory(gpu, torch, layout, spans):
    hk, d, ps = 3, 48, 16
    s = Setup(torch, SPANS[spans], hk, d, ps)
    t = s.tokens
    # places of K and V in one buffer, in elements: first elements, and the strides of both
    places = {"apart": (0, t * hk * d + 5, hk * d, d), "rows": (0, hk * d, 2 * hk * d + 3, d),
              "heads": (0, d, 2 * hk * d, 2 * d), "tokens": (hk * t * d, 0, d, t * d),
              "head rows": (0, t * d, d, 2 * t * d), "one": (7, None, hk * d, d)}
    k_at, v_at, ld_row, ld_head = places[layout]
    host = np.full(2 * hk * d * t + 3 * t + 64, 5.0, np.float32)
    device = torch.from_numpy(host.copy()).cuda()
    torch.cuda.synchronize()
    for base in (host.ctypes.data, device.data_ptr()):
        at = lambda x: None if x is None else base + 4 * x  # noqa: E731
        gpu._run(vnpu.b200_command(vnpu.OP_B200_PAGED_KV_READ, vnpu.PagedKvReadArgs(
            s.cache, s.batch, at(k_at), at(v_at), ld_row, ld_head, 0, 0)), "paged_kv_read")
    assert np.array_equal(host, device.cpu().numpy())
    assert (host != 5.0).sum() == (1 if v_at is None else 2) * t * hk * d
