"""Attention over the 4-bit paged cache where arithmetic is hardest: numbers that are not finite, groups and tokens of very different
size, and scores that move far, within bounds that notice a tenth."""
import pytest
import torch

import kv4_oracle as O
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


# ----------------------------------------------------------------------------- sizes
def _bound(q, keys, values, h, m, scale):
    """One row's heads [rep, d] of key/value head h that see m stored tokens -> result, weights, relative error of the weights, and what the result may
    be off by.  Weights and sums as the oracle has them.  A product step p is rounded to fp16 after a power of two for each row and
    group that brings the largest such product so far to 2^7 at least: it is off by 2^-11 of itself, or below fp16's normal numbers by 2^-25, which
    (code - 8) <= 8 multiplies: 2^-29 of the row's largest step p for each of the m tokens at most."""
    k, k_step, k_low = (x[:m, h] for x in keys)
    v, v_step, v_low = (x[:m, h] for x in values)
    o, p, rel, mass, _ = O.attention(q, k, v, scale, k_step, k_low, v_step, v_low)
    mid = (v_low + 8 * v_step).repeat_interleave(64, -1)
    far = (v - mid).abs()
    top = (p[:, :, None] * v_step[None]).amax(1).repeat_interleave(64, -1)
    carried = 2.0 ** -11 * (p @ far) + (m + 16) * 2.0 ** -24 * (p @ (far + mid.abs())) + m * 2.0 ** -29 * top
    return o, p, rel, 2.0 ** -8 * o.abs() + (1 + 2.0 ** -8) * (rel * mass + carried) + 1e-38


def _check(f, q, rows, scale, out, weights=None, most_rel=0.05):
    """Against the formula; weights are those of a call with decay 0.  The bounds must be tight enough to notice a mistake: weights are
    known to a twentieth at least."""
    rep = q.shape[1] // f.hkv
    q, out = q.cpu(), out.cpu().double()
    for b, n in enumerate(f.lens):
        keys, values = O.stored(f.k[b]), O.stored(f.v[b])
        for h in range(f.hkv):
            sums, tol = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
            for r in range(rows):
                m, got = n - rows + 1 + r, out[b * rows + r, h * rep:(h + 1) * rep]
                if m <= 0:
                    assert (got == 0).all()
                    continue
                o, p, rel, bound = _bound(q[b * rows + r, h * rep:(h + 1) * rep], keys, values, h, m, scale)
                assert rel.max() < most_rel, f"the bound says nothing: {rel.max():.3g}"
                assert ((got - o).abs() <= bound).all(), f"request {b}, row {r}, head {h}: {((got - o).abs() / bound).max():.3g} bounds off"
                sums[:m] += p.sum(0)
                tol[:m] += (p * rel).sum(0)
            if weights is not None and n:
                blk, t = _places(f, b)
                w = weights.cpu().double()[blk, h, t]
                assert ((w - sums).abs() <= tol + 2.0 ** -21 * sums + rows * rep * 2.0 ** -126).all(), f"weights of request {b}, head {h}"


def _few_columns(g, n, hq, d, size=1.0, columns=4):
    """Queries of a few columns: their scores, and what a worst case makes of fp32 sums, stay small against keys of any step."""
    q = torch.zeros(n, hq, d)
    q[:, :, torch.randperm(d, generator=g)[:columns]] = size * torch.randn(n, hq, columns, generator=g)
    return q.bfloat16()


@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("dev,d,n", _on_both((128, 60), None, (128, 300), (64, 300), (256, 700), (128, 4000)))
def test_value_groups_of_very_different_size(dev, d, n, rows):
    """A group of a head is as exact beside one that is 2^60 times as large as it is alone."""
    for down in (12, 20, 24, 32, 60):
        f = Filled(down, [n], 2, d, 16, dev)
        f.v[0][:, 0, :64] *= 2.0 ** -down
        f.v[0][:, 1, -64:] *= 2.0 ** down
        ops.kv4_write(f.k[0].to(dev), f.v[0].to(dev), f.slots[0].to(dev), f.k_cache, f.v_cache)
        q = _few_columns(_gen(n), rows, 8, d, 3.0).to(dev)
        out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, d ** -0.5)
        _check(f, q, rows, d ** -0.5, out)


@pytest.mark.parametrize("up", [20, 30, 60])
@pytest.mark.parametrize("weight", [-18, -27, -60, 2])
@pytest.mark.parametrize("dev,n,rows", _on_both((110, 2), None, (300, 1), (300, 3), (4000, 1)))
def test_tokens_of_very_large_values_and_small_weight(dev, n, rows, weight, up):
    """Values 2^up times the others', of tokens with scores that half the heads put at 2^weight of the others' and the other half nowhere in
    particular: what a row gets of the others has to keep its bits."""
    d = 64
    g = _gen(n + up - weight)
    for where in (slice(0, 1), slice(90, 91), slice(n - 3, n), slice(96, 128), slice(40, n)):
        f = Filled(up, [n], 1, d, 16, dev)
        f.k[0] = (f.k[0] * 0.25).bfloat16()
        f.k[0][:, :, :32] = 0
        f.k[0][where] = 0
        f.k[0][where, :, :32] = 1.0
        f.v[0][where] = (f.v[0][where].float() * 2.0 ** up).bfloat16()
        ops.kv4_write(f.k[0].to(dev), f.v[0].to(dev), f.slots[0].to(dev), f.k_cache, f.v_cache)
        q = torch.zeros(rows, 8, d)
        q[:, :, 40:44] = torch.randn(rows, 8, 4, generator=g)
        q[:, ::2, 0] = weight * 0.6931471805599453
        q = q.bfloat16().to(dev)
        out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 1.0)
        _check(f, q, rows, 1.0, out)


@BOTH
@pytest.mark.parametrize("room", [0, 1 << 28])
@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("shape", ["up", "down", "peak", "waves"])
def test_scores_that_move_far_within_known_bounds(monkeypatch, dev, shape, rows, room):
    """The running maximum, with the sums that it rescales, follows scores over 600 and more.  The columns 64 and up of a key are alike, so that
    their step is 0 and scores of any size have a small error, and the results' bounds are small against them: a result or weight
    that is a tenth too large does not pass."""
    monkeypatch.setattr(kv4, "KEPT_SCORES", room)
    d, n = 128, 960
    f = Filled(9, [n], 1, d, 64, dev)
    t = torch.arange(n).float()
    lift = {"up": t / 3, "down": (n - t) / 3, "peak": 250.0 * (t == 321), "waves": 160 + 160 * torch.sin(t / 40) * t / n}[shape]
    f.k[0][:, 0, 64:] = torch.round(lift).clamp(0, 256)[:, None].bfloat16()
    ops.kv4_write(f.k[0].to(dev), f.v[0].to(dev), f.slots[0].to(dev), f.k_cache, f.v_cache)
    q = torch.zeros(rows, 8, d)
    q[:, :, 3:7] = torch.randn(rows, 8, 4, generator=_gen(1)) * 0.5
    q[:, :, 70] = torch.tensor([5.0, 1.0, 0.25, 0.0, -1.0, -5.0, 3.0, 2.0])
    q = q.bfloat16().to(dev)
    w = torch.full(f.k_cache.shape[:3], 0.25, device=dev)
    out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 0.5, weights=w, decay=0.0)
    _check(f, q, rows, 0.5, out, w)
    for wrong in (lambda: _check(f, q, rows, 0.5, out * 1.1), lambda: _check(f, q, rows, 0.5, out * 0), lambda: _check(f, q, rows, 0.5, out, w * 1.1)):
        with pytest.raises(AssertionError, match="bounds off|weights of"):
            wrong()


@BOTH
@pytest.mark.parametrize("q_size,scale", [(10.0, 0.09), (0.01, 0.09), (3e4, 1e-4), (2.0, -0.3), (1e-30, 1e29)])
def test_queries_of_any_size_within_known_bounds(dev, q_size, scale):
    for rows, d in ((1, 128), (5, 64), (2, 256)):
        f = Filled(5, [333, 64], 2, d, 16, dev)
        q = _few_columns(_gen(d), 2 * rows, 16, d, q_size, 3).to(dev)
        w = torch.zeros(f.k_cache.shape[:3], device=dev)
        out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, scale, weights=w, decay=0.0)
        _check(f, q, rows, scale, out, w)
