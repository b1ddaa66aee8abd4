"""The 4-bit paged cache where arithmetic and launches change their way: numbers that are not finite, groups and tokens of very
different size, work cut through many requests, and what a cache's bytes are on either device."""
import pytest
import torch

from omni_infer_b200 import ops
from omni_infer_b200.ops import kv4
from test_kv4_ops import BOTH, Filled, _gen


def _places(f, b):
    t = torch.arange(f.lens[b])
    return f.table[b].long()[t // f.block], t % f.block


# ----------------------------------------------------------------------------- numbers that are not finite
@BOTH
@pytest.mark.parametrize("room", [0, 1 << 28])
@pytest.mark.parametrize("scale", [float("nan"), float("inf")])
@pytest.mark.parametrize("lens", [[70, 2, 0], [1000, 2, 0]])
def test_scales_that_are_not_finite(monkeypatch, dev, lens, scale, room):
    """No softmax of them is a number: rows that see a token are NaN, and so is the weight of all that a row sees; rows that see none
    are zero all the same."""
    monkeypatch.setattr(kv4, "KEPT_SCORES", room)
    rows, hkv, d = 3, 2, 64
    f = Filled(2, lens, hkv, d, 16, dev)
    q = torch.randn(len(lens) * rows, 4, d, generator=_gen(0)).bfloat16().to(dev)
    w = torch.ones(f.k_cache.shape[:3], device=dev)
    out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, scale, weights=w).cpu().view(len(lens), rows, 4, d)
    want = torch.ones(w.shape)
    for b, n in enumerate(lens):
        for r in range(rows):
            row = out[b, r]
            assert row.isnan().all() if n - rows + 1 + r > 0 else (row == 0).all(), f"request {b}, row {r}"
        blk, t = _places(f, b)
        want[blk, :, t] = float("nan")
    assert torch.equal(w.cpu().nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0))


@BOTH
@pytest.mark.parametrize("room", [0, 1 << 28])
def test_a_query_that_is_not_finite(monkeypatch, dev, room):
    """The first of three rows: NaN for itself and for the weights of what it sees.  The last two tokens are seen by the other rows
    alone, and their weights are numbers."""
    monkeypatch.setattr(kv4, "KEPT_SCORES", room)
    n, rows, d = 50, 3, 64
    f = Filled(4, [n], 1, d, 16, dev)
    q = torch.randn(rows, 2, d, generator=_gen(1)).bfloat16()
    q[0, 1, 7] = float("nan")
    w = torch.zeros(f.k_cache.shape[:3], device=dev)
    out = ops.kv4_decode(q.to(dev), f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 0.125, weights=w).cpu()
    assert out[0, 1].isnan().all() and out.isnan().sum() == d
    blk, t = _places(f, 0)
    assert torch.equal(w.cpu()[blk, 0, t].isnan(), torch.arange(n) < n - rows + 1)
