"""The 4-bit paged cache where arithmetic and launches change their way: numbers that are not finite, groups and tokens of very
different size, work cut through many requests, and what a cache's bytes are on either device."""
import pytest
import torch

from omni_infer_b200 import ops
from omni_infer_b200.ops import kv4
from test_kv4_ops import BOTH, Filled, _gen

cuda = [pytest.mark.gpu]


def _on_both(*sizes):
    """Sizes for both devices, and behind a None those for a GPU alone: writing long caches takes the CPU too long."""
    at = sizes.index(None) if None in sizes else len(sizes)
    return [("cpu", *s) for s in sizes[:at]] + [pytest.param("cuda", *s, marks=cuda) for s in sizes if s is not None]


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


@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("dev,n", _on_both((100,), None, (3000,)))
def test_a_nan_value_whose_weight_is_zero(dev, n, rows):
    """0 NaN is NaN: whether a row gives a NaN goes by what it sees, not by where a token lies or by how small its weight has become.
    The token's score is 25,600 below the others'."""
    d = 128
    for j in sorted({5, 40, n // 2, n - 3, n - 1}):
        f = Filled(n, [n], 1, d, 16, dev)
        f.k[0] *= 0.1
        f.k[0][j] = -200.0
        f.v[0][j, 0, 3] = float("nan")
        ops.kv4_write(f.k[0].to(dev), f.v[0].to(dev), f.slots[0].to(dev), f.k_cache, f.v_cache)
        q = torch.ones(rows, 8, d, dtype=torch.bfloat16, device=dev)
        out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 1.0).cpu()
        nan = torch.zeros(rows, 8, d, dtype=torch.bool)
        for r in range(rows):
            nan[r, :, :64] = j < n - rows + 1 + r
        assert torch.equal(out.isnan(), nan), f"token {j}"
