"""The 4-bit paged key/value cache: every op against its formula in 64 bits, on the CPU (references) and on the GPU (kernels)."""
import pytest
import torch

import kv4_oracle as O
from omni_infer_b200 import ops
from omni_infer_b200.ops import _native as nat
from omni_infer_b200.ops import kv4

GPU = pytest.param("cuda", marks=pytest.mark.gpu)
BOTH = pytest.mark.parametrize("dev", ["cpu", GPU])


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(g, *shape, levels=True):
    x = torch.randn(*shape, generator=g)
    if levels:
        x = x + 4 * torch.randn(shape[-1], generator=g) * (torch.rand(shape[-1], generator=g) < 0.1)
    return x.bfloat16()


class Filled:
    """Caches whose requests hold known rows, in shuffled blocks; everything else holds NaN scales."""

    def __init__(self, seed, lens, hkv, d, block, dev, spare=2, k_scale=1.0, v_scale=1.0):
        g = _gen(seed)
        self.lens, self.hkv, self.d, self.block, self.dev = lens, hkv, d, block, dev
        width = max(1, -(-max(lens + [1]) // block)) + 1
        blocks = len(lens) * width + spare
        self.table = torch.randperm(blocks, generator=g)[:len(lens) * width].view(len(lens), width).to(torch.int32)
        self.k_cache, self.v_cache = ops.kv4_cache(blocks, block, hkv, d, dev)
        self.k_cache.fill_(0xff)
        self.v_cache.fill_(0xff)
        self.k = [_rows(g, n, hkv, d) * k_scale for n in lens]
        self.v = [_rows(g, n, hkv, d, levels=False) * v_scale for n in lens]
        self.slots = [self.table[b].long()[torch.arange(n) // block] * block + torch.arange(n) % block for b, n in enumerate(lens)]
        if sum(lens):
            ops.kv4_write(torch.cat(self.k).to(dev), torch.cat(self.v).to(dev), torch.cat(self.slots).to(dev), self.k_cache, self.v_cache)
        self.table_dev = self.table.to(dev)
        self.lens_dev = torch.tensor(lens, dtype=torch.int32, device=dev)


# ----------------------------------------------------------------------------- rows
@BOTH
@pytest.mark.parametrize("T,hkv,d,block", [(1, 1, 64, 16), (7, 2, 128, 48), (65, 4, 128, 128), (33, 3, 256, 32), (130, 8, 64, 64)])
def test_rows_are_what_the_formula_says(dev, T, hkv, d, block):
    """Every value equals the formula's, rounded to bf16 once: the codes of a group and its bf16 step and lowest value are exact
    functions of bf16 inputs, and so is code * step + lowest up to that rounding."""
    g = _gen(T + d)
    blocks = T // block + 3
    k, v = _rows(g, T, hkv, d), _rows(g, T, hkv, d, levels=False) * 0.01
    slots = torch.randperm(blocks * block, generator=g)[:T]
    kc, vc = ops.kv4_cache(blocks, block, hkv, d, dev)
    weights = torch.full((blocks, hkv, block), 5.0, device=dev)
    positions = torch.full((blocks, hkv, block), -7, dtype=torch.int32, device=dev)
    pos = torch.arange(T) + 100
    ops.kv4_write(k.to(dev), v.to(dev), slots.to(dev), kc, vc, weights=weights, positions=positions, token_positions=pos.to(dev))
    rk, rv = ops.kv4_read(kc, vc, slots.to(dev))
    for got, x in ((rk, k), (rv, v)):
        assert torch.equal(got.cpu(), O.stored(x)[0].float().bfloat16())
    w, p = weights.cpu().transpose(1, 2).flatten(0, 1), positions.cpu().transpose(1, 2).flatten(0, 1)
    assert (w[slots] == 0).all() and (p[slots] == pos[:, None].int()).all()
    rest = torch.ones(blocks * block, dtype=torch.bool)
    rest[slots] = False
    assert (w[rest] == 5).all() and (p[rest] == -7).all()
    empty = ops.kv4_read(kc, vc, torch.arange(blocks * block)[rest].to(dev))
    assert all((e == 0).all() for e in empty), "other slots are left as they were"


@BOTH
def test_rows_of_any_pitch_and_slots_to_skip(dev):
    g = _gen(3)
    T, hkv, d, block = 21, 2, 128, 16
    for off in (0, 1):                                       # odd offsets: no aligned wide loads
        big = torch.randn(T, hkv + 3, d + 9, generator=g).bfloat16().to(dev)
        k, v = big[:, 1:1 + hkv, off:off + d], big[:, 2:2 + hkv, off + 5:off + 5 + d]
        slots = torch.arange(T) * 2
        slots[4] = slots[9] = -1
        kc, vc = ops.kv4_cache(4, block, hkv, d, dev)
        ops.kv4_write(k, v, slots.to(dev), kc, vc)
        rk, rv = ops.kv4_read(kc, vc, slots.to(dev))
        for got, x in ((rk, k), (rv, v)):
            want = O.stored(x)[0].float().bfloat16()
            want[4] = want[9] = 0
            assert torch.equal(got.cpu(), want)
        odd = ops.kv4_read(kc, vc, (torch.arange(T) * 2 + 1).to(dev))
        assert all((o == 0).all() for o in odd)


@BOTH
def test_groups_at_the_edges_of_the_format(dev):
    """Constant groups are exact, groups with a NaN or an infinity are NaN as a whole and leave the others alone, and ranges from
    the smallest to nearly the largest bf16 numbers follow the formula."""
    hkv, d, block = 1, 128, 16
    x = torch.randn(9, hkv, d, generator=_gen(8)).bfloat16()
    x[0] = 3.25
    x[1] = 0
    x[2, 0, 70] = float("nan")
    x[3, 0, 5] = float("inf")
    x[4, 0, 100] = float("-inf")
    x[5] = (x[5].double() * 1e30).bfloat16()
    x[6] = (x[6].double() * 1e-30).bfloat16()
    x[7] = x[7] + 1000
    x[8, 0, 0], x[8, 0, 1] = 3e38, -3e38                    # the range is beyond fp32
    slots = torch.arange(9)
    kc, vc = ops.kv4_cache(1, block, hkv, d, dev)
    ops.kv4_write(x.to(dev), x.flip(0).contiguous().to(dev), slots.to(dev), kc, vc)
    rk, rv = ops.kv4_read(kc, vc, slots.to(dev))
    want = O.stored(x)[0].float().bfloat16()
    for i, grp in ((2, 1), (3, 0), (4, 1), (8, 0)):
        assert want[i, 0, grp * 64:grp * 64 + 64].isnan().all() and not want[i, 0, (1 - grp) * 64:(1 - grp) * 64 + 64].isnan().any()
    assert torch.equal(rk.cpu().nan_to_num(nan=77.0), want.nan_to_num(nan=77.0))
    assert torch.equal(rv.cpu().nan_to_num(nan=77.0), want.flip(0).nan_to_num(nan=77.0))
    assert (rk[0] == 3.25).all() and (rk[1] == 0).all()


@BOTH
@pytest.mark.parametrize("d", [64, 128, 256])
def test_groups_of_all_exponents(dev, d):
    """Columns of every size within a group, ties between codes, the smallest steps, and ranges just below the largest fp32 number, where
    15 steps are beyond it and 15 steps and the lowest value are not."""
    g, T, hkv, block = _gen(d), 96, 2, 16
    x = torch.randn(T, hkv, d, generator=g)
    sign = torch.sign(x)
    x[0:16] = torch.randint(-8, 9, (16, hkv, d), generator=g).float() / 2                      # ties
    x[16:32] = torch.exp2(torch.randint(-133, 127, (16, hkv, d), generator=g).float()) * sign[16:32]
    x[32:48] *= torch.exp2(torch.randint(-133, 120, (16, hkv, 1), generator=g).float())
    x[48:64] = torch.randint(0, 16, (16, hkv, d), generator=g) * 2.0 ** -133 - 2.0 ** -130      # the smallest bf16 numbers
    x[64:80] = torch.randint(0, 31, (16, hkv, d), generator=g) * 2.0 ** torch.randint(-20, 20, (16, hkv, 1), generator=g)
    x[80:96, :, 0::64], x[80:96, :, 1::64] = 2.5e38, torch.linspace(-8.6e37, -9.1e37, 16)[:, None, None].expand(16, hkv, d // 64)
    x = x.bfloat16()
    slots = torch.randperm(T, generator=g)
    kc, vc = ops.kv4_cache(T // block, block, hkv, d, dev)
    ops.kv4_write(x.to(dev), x.flip(0).contiguous().to(dev), slots.to(dev), kc, vc)
    want = O.stored(x)[0].float().bfloat16()
    for got, w in zip(ops.kv4_read(kc, vc, slots.to(dev)), (want, want.flip(0))):
        assert torch.equal(got.cpu().isnan(), w.isnan())
        assert torch.equal(got.cpu()[~w.isnan()], w[~w.isnan()])


@BOTH
def test_no_rows(dev):
    kc, vc = ops.kv4_cache(1, 16, 2, 64, dev)
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=dev)
    ops.kv4_write(none, none, torch.empty(0, dtype=torch.int64, device=dev), kc, vc)
    k, v = ops.kv4_read(kc, vc, torch.empty(0, dtype=torch.int64, device=dev))
    assert k.shape == v.shape == (0, 2, 64)
    table, lens = torch.zeros(0, 1, dtype=torch.int32, device=dev), torch.zeros(0, dtype=torch.int32, device=dev)
    assert ops.kv4_decode(torch.empty(0, 4, 64, dtype=torch.bfloat16, device=dev), kc, vc, table, lens, 1.0).shape == (0, 4, 64)
    w, p = torch.zeros(1, 2, 16, device=dev), torch.zeros(1, 2, 16, dtype=torch.int32, device=dev)
    keep, kept = ops.kv4_keep(w, p, table, lens, lens, 4)
    assert keep.shape == (0, 2, 4) and kept.shape == (0,)
    ops.kv4_move(kc, vc, table, keep)


# ----------------------------------------------------------------------------- attention
def _check_decode(f, q, rows, scale, out, weights=None, old=None, decay=0.0):
    """Against the formula, within the bound that the oracle derives."""
    hq, rep = q.shape[1], q.shape[1] // f.hkv
    q, out = q.cpu(), out.cpu().double()
    place = weights.cpu().double() if weights is not None else None
    want_w = old.cpu().double().clone() if old is not None else None
    tol_w = torch.zeros_like(want_w) if want_w is not None else None
    for b, n in enumerate(f.lens):
        k, k_step, k_low = O.stored(f.k[b])
        v, v_step, v_low = O.stored(f.v[b])
        t = torch.arange(n)
        blk = f.table[b].long()[t // f.block]
        for h in range(f.hkv):
            sums, tol = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
            for r in range(rows):
                m, got = n - rows + 1 + r, out[b * rows + r, h * rep:(h + 1) * rep]
                if m <= 0:
                    assert (got == 0).all()
                    continue
                o, p, rel, mass, carried = O.attention(q[b * rows + r, h * rep:(h + 1) * rep], k[:m, h], v[:m, h], scale, k_step[:m, h], k_low[:m, h],
                                                       v_step[:m, h], v_low[:m, h])
                bound = 2.0 ** -8 * o.abs() + (1 + 2.0 ** -8) * (rel * mass + carried) + 1e-38
                assert ((got - o).abs() <= bound).all(), f"request {b}, row {r}, head {h}: {((got - o).abs() - bound).max():.3g} over the bound"
                sums[:m] += p.sum(0)
                tol[:m] += (p * rel).sum(0)
            if want_w is not None and n:
                before = want_w[blk, h, t % f.block]
                want_w[blk, h, t % f.block] = sums + (before * decay if decay else 0)
                # and each of the rows * rep terms may be flushed below the smallest normal number
                tol_w[blk, h, t % f.block] = tol + 2.0 ** -21 * (sums + abs(decay) * before.abs()) + rows * rep * 2.0 ** -126
    if want_w is not None:
        assert ((place - want_w).abs() <= tol_w).all(), f"weights off by {((place - want_w).abs() - tol_w).max():.3g} over the bound"


SHAPES = [
    # lens, rows, hq, hkv, d, block
    ([1], 1, 1, 1, 64, 16),
    ([0, 1, 2, 15, 16, 17, 0], 1, 4, 2, 128, 16),
    ([63, 64, 65, 127, 128, 129], 1, 8, 1, 128, 64),
    ([300, 5, 77], 1, 32, 4, 128, 128),
    ([191, 193, 1], 2, 14, 2, 64, 48),
    ([2, 3, 100, 0], 4, 6, 6, 256, 32),
    ([513], 5, 16, 1, 128, 256),
    ([40, 1000], 16, 16, 2, 128, 128),
    ([70, 31], 3, 5, 1, 256, 16),
    ([2100], 1, 12, 4, 64, 80),
    # many rows a key/value head
    ([65], 33, 1, 1, 128, 16),
    ([700, 0, 64, 8], 9, 8, 1, 128, 64),
    ([100, 3, 257], 20, 10, 1, 64, 32),
    ([1030], 17, 24, 3, 128, 128),
    ([5000], 16, 8, 1, 128, 128),
]


@BOTH
@pytest.mark.parametrize("mode", ["plain", "set", "add"])
@pytest.mark.parametrize("lens,rows,hq,hkv,d,block", SHAPES)
def test_attention(dev, lens, rows, hq, hkv, d, block, mode):
    f = Filled(sum(lens) + d, lens, hkv, d, block, dev)
    g = _gen(11)
    q = (1.3 * torch.randn(len(lens) * rows, hq + 2, d, generator=g)).bfloat16().to(dev)[:, 1:1 + hq]
    if mode == "plain":
        out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, d ** -0.5)
        assert out.shape == (len(lens) * rows, hq, d) and out.dtype == torch.bfloat16
        return _check_decode(f, q, rows, d ** -0.5, out)
    old = torch.rand(f.k_cache.shape[:3], generator=g)
    if mode == "set":
        old[f.table[0, 0]] = float("nan")                    # dropped unread below the lengths, left beyond them
        for b, n in enumerate(lens):
            for i in range(n, f.table.shape[1] * block):
                old[f.table[b, i // block], :, i % block] = 0.5
    w = old.clone().to(dev)
    decay = 0.0 if mode == "set" else 0.75
    out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, d ** -0.5, max_seq_len=max(lens), weights=w, decay=decay)
    if mode == "set":
        old = old.nan_to_num(nan=0.5)
    _check_decode(f, q, rows, d ** -0.5, out, w, old, decay)


@pytest.mark.gpu
@pytest.mark.parametrize("bound", [None, 1, 700, 10 ** 6])
@pytest.mark.parametrize("B,n,hkv,rep", [(1, 4000, 1, 8), (2, 9001, 2, 5), (40, 700, 4, 2)])
def test_attention_is_split_over_long_caches(bound, B, n, hkv, rep):
    """However the launch is shaped: a bound that is wrong, too small or missing changes nothing but speed."""
    lens = [n - 13 * i for i in range(B)]
    f = Filled(n, lens, hkv, 128, 64, "cuda")
    q = torch.randn(B, hkv * rep, 128, generator=_gen(2)).bfloat16().cuda()
    w = torch.zeros(f.k_cache.shape[:3], device="cuda")
    out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 128 ** -0.5, max_seq_len=bound, weights=w)
    _check_decode(f, q, 1, 128 ** -0.5, out, w, torch.zeros(f.k_cache.shape[:3]), 1.0)


@BOTH
@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("q_scale,k_scale,v_scale,scale", [(40.0, 1.0, 1.0, 0.09), (1.0, 1.0, 1e-20, 0.09), (1.0, 1.0, 1e6, 0.09), (0.0, 1.0, 1.0, 0.09),
                                                         (1.0, 100.0, 1.0, 1e-3), (1.0, 1.0, 1.0, -0.3), (1.0, 1.0, 1.0, 0.0)])
def test_attention_of_any_magnitude(dev, q_scale, k_scale, v_scale, scale, rows):
    f = Filled(5, [333, 64], 2, 128, 16, dev, k_scale=k_scale, v_scale=v_scale)
    q = (q_scale * torch.randn(2 * rows, 16, 128, generator=_gen(7))).bfloat16().to(dev)
    w = torch.zeros(f.k_cache.shape[:3], device=dev)
    out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, scale, weights=w, decay=0.0)
    _check_decode(f, q, rows, scale, out, w, torch.zeros(f.k_cache.shape[:3]))


@BOTH
@pytest.mark.parametrize("shift", [1, 3, 8])
def test_queries_of_any_pitch(dev, shift):
    """Rows and heads that do not start on 16 bytes, and the largest and smallest bf16 numbers."""
    f = Filled(17, [150, 3], 2, 128, 32, dev, k_scale=1e-3)
    q = torch.randn(4, 9, 128 + 16, generator=_gen(3)).bfloat16()[:, 1:7, shift:shift + 128]
    q[1] *= 1e-38
    q[2] *= 1e37
    q = q.to(dev) if dev == "cpu" else torch.randn(4, 9, 128 + 16, device=dev).bfloat16()[:, 1:7, shift:shift + 128].copy_(q)
    out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 1e-34)
    _check_decode(f, q, 2, 1e-34, out)


@BOTH
@pytest.mark.parametrize("outlier", [300.0, 3000.0, 65536.0])
def test_queries_with_one_large_column(dev, outlier):
    """A column that outweighs the others by far, with keys that are all alike there: the softmax goes by the other columns, which have
    to keep their bits.  The large product is 4 outlier scale in an fp32 sum of some 20 steps (16 columns a step and a few more):
    an error of 20 * 2^-24 of it at most, twice that in the weights; an error of half a step in an 8th bit of the other columns would
    be over 100 times that for the first two."""
    d, n, scale = 128, 200, 0.09
    f = Filled(31, [n], 2, d, 16, dev)
    f.k[0][:, :, 9] = 4.0
    ops.kv4_write(f.k[0].to(dev), f.v[0].to(dev), f.slots[0].to(dev), f.k_cache, f.v_cache)
    q = torch.randn(1, 12, d, generator=_gen(1))
    q[:, ::2, 9] = outlier
    q = q.bfloat16().to(dev)
    w = torch.zeros(f.k_cache.shape[:3], device=dev)
    ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, scale, weights=w, decay=0.0)
    k = O.stored(f.k[0])[0]
    blk, t = f.table[0].long()[torch.arange(n) // 16], torch.arange(n) % 16
    for h in range(2):
        p = torch.softmax(q[0, 6 * h:6 * h + 6].double().cpu() @ k[:, h].T * scale, -1).sum(0)
        assert ((w.cpu()[blk, h, t].double() - p).abs() <= p * (1e-5 + 2 * 20 * 2.0 ** -24 * 4 * outlier * scale)).all()


@BOTH
@pytest.mark.parametrize("rows", [1, 5])
def test_rising_scores(dev, rows):
    """Scores that rise, fall and stand still along the cache by far more than what an exponential holds: the running maximum has to
    follow them."""
    d, n = 128, 640
    for shape in ("up", "down", "peak"):
        f = Filled(9, [n], 1, d, 64, dev)
        t = torch.arange(n).float()
        lift = {"up": t, "down": n - t, "peak": 500.0 * (t == 321)}[shape]
        f.k[0][:, 0, 0] = (lift * 2).bfloat16()
        ops.kv4_write(f.k[0].to(dev), f.v[0].to(dev), f.slots[0].to(dev), f.k_cache, f.v_cache)
        q = torch.randn(rows, 8, d, generator=_gen(1))
        q[:, :, 0] = torch.tensor([4.0, 1.0, 0.25, 0.0, -1.0, -4.0, 30.0, 2.0])
        q = q.bfloat16().to(dev)
        w = torch.zeros(f.k_cache.shape[:3], device=dev)
        out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 0.5, weights=w, decay=0.0)
        _check_decode(f, q, rows, 0.5, out, w, torch.zeros(f.k_cache.shape[:3]))


@BOTH
@pytest.mark.parametrize("rows", [1, 20])
def test_nan_stays_where_it_is_seen(dev, rows):
    n = 100
    f = Filled(21, [n, n], 2, 128, 16, dev)
    f.v[0][50, 1, 3] = float("nan")                          # a value of request 0, head 1: the columns of its group
    f.k[1][20, 0, 0] = float("inf")                          # a key of request 1, head 0: all columns of the head's queries
    f.v[1][n - 1, 1, 100] = float("-inf")                    # a value that only the last row sees
    for b in (0, 1):
        ops.kv4_write(f.k[b].to(dev), f.v[b].to(dev), f.slots[b].to(dev), f.k_cache, f.v_cache)
    q = torch.randn(2 * rows, 4, 128, generator=_gen(1)).bfloat16().to(dev)
    out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 0.1).cpu().view(2, rows, 4, 128)
    nan = torch.zeros(2, rows, 4, 128, dtype=torch.bool)
    nan[0, :, 2:, :64] = True
    nan[1, :, :2] = True
    nan[1, -1, 2:, 64:] = True
    assert torch.equal(out.isnan(), nan)


# ----------------------------------------------------------------------------- eviction
def _state(seed, lens, hkv, block, dev, ties=False, nans=False):
    g = _gen(seed)
    width = max(1, -(-max(lens + [1]) // block))
    blocks = len(lens) * width + 1
    table = torch.randperm(blocks, generator=g)[:len(lens) * width].view(len(lens), width).to(torch.int32)
    w = torch.exp(3 * torch.randn(blocks, hkv, block, generator=g) - 4)
    if ties:
        w = torch.round(w * 4) / 4
        w = torch.where(torch.rand(w.shape, generator=g) < 0.2, -0.0 * w, w)
    if nans:
        w = torch.where(torch.rand(w.shape, generator=g) < 0.1, torch.full_like(w, float("nan")), w)
        w = torch.where(torch.rand(w.shape, generator=g) < 0.1, -w, w)
    pos = torch.full((blocks, hkv, block), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for h in range(hkv):
            p = torch.randperm(n + 5, generator=g)[:n].to(torch.int32)
            for i in range(n):
                pos[table[b, i // block], h, i % block] = p[i]
    return table, w, pos, [n + 5 for n in lens]


@BOTH
@pytest.mark.parametrize("ties,nans", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("lens,hkv,block,budget,first,last", [([1], 1, 16, 1, 0, 0), ([40, 0, 20, 21, 300], 2, 16, 20, 4, 7), ([1500, 1025], 1, 64, 1024, 0, 1024),
                                                              ([129, 128, 127], 3, 128, 128, 64, 64), ([700], 2, 48, 3, 1, 2), ([90, 33], 1, 16, 500, 10, 10)])
def test_keep(dev, lens, hkv, block, budget, first, last, ties, nans):
    table, w, pos, seen = _state(sum(lens) + budget, lens, hkv, block, dev, ties, nans)
    keep, kept = ops.kv4_keep(w.to(dev), pos.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                              torch.tensor(seen, dtype=torch.int32, device=dev), budget, keep_first=first, keep_last=last)
    assert keep.shape == (len(lens), hkv, budget) and kept.tolist() == [min(n, budget) for n in lens]
    for b, n in enumerate(lens):
        t = torch.arange(n)
        blk = table[b].long()[t // block]
        for h in range(hkv):
            want = O.keep(w[blk, h, t % block].tolist(), pos[blk, h, t % block].tolist(), n, seen[b], budget, first, last)
            assert keep[b, h].tolist() == want + [-1] * (budget - len(want)), f"request {b}, head {h}"


@pytest.mark.gpu
@pytest.mark.parametrize("bound", [None, 10, 50_000])
@pytest.mark.parametrize("lens,budget", [([50_000, 41_003, 4097, 300], 4096), ([330_000], 300_001)])
def test_keep_of_long_requests(lens, budget, bound):
    """Whatever the launch is shaped by, and with more places than shared memory holds."""
    g, hkv, block = _gen(budget), 2, 128
    width = -(-max(lens) // block)
    blocks = len(lens) * width
    table = torch.randperm(blocks, generator=g).view(len(lens), width).to(torch.int32)
    w = torch.round(torch.rand(blocks, hkv, block, generator=g) * 3000) / 7          # many equal ones
    pos = torch.randint(0, max(lens), (blocks, hkv, block), generator=g, dtype=torch.int32)
    seen = [n - n // 9 for n in lens]
    keep, kept = ops.kv4_keep(w.cuda(), pos.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(seen, dtype=torch.int32).cuda(),
                              budget, keep_first=3, keep_last=100, max_seq_len=bound)
    assert kept.tolist() == [min(n, budget) for n in lens]
    for b, n in enumerate(lens):
        wb, pb = (x[table[b].long()].transpose(0, 1).flatten(1)[:, :n] for x in (w, pos))
        for h in range(hkv):
            want = O.keep(wb[h].tolist(), pb[h].tolist(), n, seen[b], budget, 3, 100)
            assert keep[b, h].tolist() == want + [-1] * (budget - len(want))


@pytest.mark.gpu
@pytest.mark.parametrize("hkv,block,off,lens", [(1, 10, 0, [2001, 30]), (3, 16, 1, [5000, 999]), (3, 16, 2, [20_000, 4099]), (33, 64, 0, [17_001, 9000])])
def test_keep_of_any_block_and_address(hkv, block, off, lens):
    """Blocks of other sizes than a cache's, numbers that do not start on 16 bytes, and more heads than clusters find room for at once."""
    g, budget, width = _gen(hkv), 500, -(-max(lens) // block)
    blocks = len(lens) * width
    table = torch.randperm(blocks, generator=g).view(len(lens), width).to(torch.int32)
    w = torch.exp(3 * torch.randn(blocks, hkv, block, generator=g))
    pos = torch.randint(0, max(lens), w.shape, generator=g, dtype=torch.int32)
    wd, pd = (torch.empty(x.numel() + off, dtype=x.dtype, device="cuda")[off:].view(x.shape).copy_(x) for x in (w, pos))
    n = torch.tensor(lens, dtype=torch.int32)
    keep, _ = ops.kv4_keep(wd, pd, table.cuda(), n.cuda(), n.cuda(), budget, keep_first=5, keep_last=20)
    want, _ = ops.kv4_keep(w, pos, table, n, n, budget, keep_first=5, keep_last=20)
    assert torch.equal(keep.cpu(), want)


@BOTH
@pytest.mark.parametrize("d,block,hkv", [(64, 16, 3), (128, 48, 2), (256, 32, 1)])
def test_move(dev, d, block, hkv):
    """The named tokens, their weights and positions in their places, bit for bit; every other place as it was."""
    lens, budget = [200, 97, 30, 0], 41
    f = Filled(d, lens, hkv, d, block, dev)
    shape = tuple(f.k_cache.shape[:3])
    w = torch.rand(shape, generator=_gen(1))
    pos = torch.randint(0, 1000, shape, generator=_gen(2), dtype=torch.int32)
    keep = torch.full((len(lens), hkv, budget), -1, dtype=torch.int32)
    g = _gen(3)
    for b, n in enumerate(lens):
        for h in range(hkv):
            far = (budget + torch.randperm(max(0, n - budget), generator=g)).tolist()
            for j in range(min(n, budget)):
                keep[b, h, j] = far.pop() if far and torch.rand((), generator=g) < 0.5 else j
    everything = torch.arange(shape[0] * block, device=dev)
    before = [x.cpu() for x in ops.kv4_read(f.k_cache, f.v_cache, everything)]
    wd, pd = w.to(dev), pos.to(dev)
    ops.kv4_move(f.k_cache, f.v_cache, f.table_dev, keep.to(dev), weights=wd, positions=pd)
    want = [x.clone() for x in before] + [w.clone(), pos.clone()]
    for b, n in enumerate(lens):
        for h in range(hkv):
            for j in range(min(n, budget)):
                s = int(keep[b, h, j])
                fb, ft, tb, tt = int(f.table[b, s // block]), s % block, int(f.table[b, j // block]), j % block
                for i in (0, 1):
                    want[i][tb * block + tt, h] = before[i][fb * block + ft, h]
                want[2][tb, h, tt], want[3][tb, h, tt] = w[fb, h, ft], pos[fb, h, ft]
    got = [x.cpu() for x in ops.kv4_read(f.k_cache, f.v_cache, everything)] + [wd.cpu(), pd.cpu()]
    for a, b in zip(got, want):
        assert torch.equal(a.float().nan_to_num(nan=1e9), b.float().nan_to_num(nan=1e9))


# ----------------------------------------------------------------------------- without room for scores
@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["set", "add"])
@pytest.mark.parametrize("lens,rows,hq,hkv,d,block", SHAPES)
def test_weights_of_scores_that_are_not_kept(monkeypatch, lens, rows, hq, hkv, d, block, mode):
    monkeypatch.setattr(kv4, "KEPT_SCORES", 0)
    test_attention("cuda", lens, rows, hq, hkv, d, block, mode)


@pytest.mark.gpu
def test_long_and_extreme_scores_that_are_not_kept(monkeypatch):
    monkeypatch.setattr(kv4, "KEPT_SCORES", 0)
    for bound in (None, 1, 700):
        test_attention_is_split_over_long_caches(bound, 2, 9001, 2, 5)
    for rows in (1, 5):
        test_rising_scores("cuda", rows)
        test_attention_of_any_magnitude("cuda", 40.0, 1.0, 1.0, 0.09, rows)
        test_attention_of_any_magnitude("cuda", 1.0, 1.0, 1.0, -0.3, rows)


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 1 << 28])
@pytest.mark.parametrize("d,rows,hq,hkv", [(64, 16, 32, 2), (128, 256, 1, 1), (256, 32, 8, 1), (128, 51, 5, 1)])
def test_weights_of_the_most_rows(monkeypatch, d, rows, hq, hkv, room):
    monkeypatch.setattr(kv4, "KEPT_SCORES", room)
    lens = [290, 17, 0]
    f = Filled(d, lens, hkv, d, 32, "cuda")
    q = torch.randn(len(lens) * rows, hq, d, generator=_gen(5)).bfloat16().cuda()
    w = torch.ones(f.k_cache.shape[:3], device="cuda")
    out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, d ** -0.5, weights=w, decay=0.25)
    _check_decode(f, q, rows, d ** -0.5, out, w, torch.ones(f.k_cache.shape[:3]), 0.25)


@BOTH
@pytest.mark.parametrize("room", [0, 1 << 28])
def test_weights_of_a_nan(monkeypatch, dev, room):
    """A key that is not finite makes the weights of its head's whole request NaN, and no others."""
    monkeypatch.setattr(kv4, "KEPT_SCORES", room)
    lens = [100, 900]
    f = Filled(21, lens, 2, 128, 16, dev)
    f.k[1][20, 0, 0] = float("inf")
    ops.kv4_write(f.k[1].to(dev), f.v[1].to(dev), f.slots[1].to(dev), f.k_cache, f.v_cache)
    q = torch.randn(2, 6, 128, generator=_gen(1)).bfloat16().to(dev)
    w = torch.full(f.k_cache.shape[:3], 0.5, device=dev)
    ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 0.1, weights=w, decay=0.5)
    nan = torch.zeros(w.shape, dtype=torch.bool)
    for i in range(lens[1]):
        nan[f.table[1, i // 16], 0, i % 16] = True
    assert torch.equal(w.isnan().cpu(), nan)


@pytest.mark.gpu
def test_weights_of_a_wide_table():
    """A table far wider than the requests: nothing of it counts but what they have."""
    f = Filled(3, [130, 64, 1], 2, 128, 64, "cuda")
    wide = torch.full((3, 2000), -1, dtype=torch.int32, device="cuda")
    wide[:, :f.table_dev.shape[1]] = f.table_dev
    q = torch.randn(3, 6, 128, generator=_gen(2)).bfloat16().cuda()
    for bound in (None, 130):
        w = torch.ones(f.k_cache.shape[:3], device="cuda")
        out = ops.kv4_decode(q, f.k_cache, f.v_cache, wide, f.lens_dev, 0.1, max_seq_len=bound, weights=w, decay=0.5)
        _check_decode(f, q, 1, 0.1, out, w, torch.ones(f.k_cache.shape[:3]), 0.5)


# ----------------------------------------------------------------------------- together
@BOTH
def test_a_request_with_a_budget(dev):
    """Tokens written one at a time, read by attention that adds up its weights, and cut down to the budget whenever a block over it
    has filled up: every step equals the same steps on lists of plain rows."""
    g = _gen(4)
    B, hkv, rep, d, block, budget = 2, 2, 3, 64, 16, 32
    kc, vc = ops.kv4_cache(2 * 4, block, hkv, d, dev)
    table = torch.randperm(8, generator=g).view(2, 4).to(torch.int32).to(dev)
    w, pos = torch.zeros(8, hkv, block, device=dev), torch.zeros(8, hkv, block, dtype=torch.int32, device=dev)
    lens = [0, 0]
    mine = [[[] for _ in range(hkv)] for _ in range(B)]      # per head: [key row, value row, key steps, key lows, value steps, weight, position, value lows]
    for step in range(75):
        live = [b for b in range(B) if b == 0 or step >= 20]  # the second request comes later
        k, v = _rows(g, B, hkv, d), _rows(g, B, hkv, d, levels=False)
        q = torch.randn(B, hkv * rep, d, generator=g).bfloat16()
        slots = torch.full((B,), -1, dtype=torch.int64)
        seen = [step + 1, max(0, step - 19)]
        for b in live:
            slots[b] = int(table[b, lens[b] // block]) * block + lens[b] % block
            lens[b] += 1
            (ks, kst, kl), (vs, vst, vl) = O.stored(k[b]), O.stored(v[b])
            for h in range(hkv):
                mine[b][h].append([ks[h], vs[h], kst[h], kl[h], vst[h], 0.0, seen[b] - 1, vl[h]])
        n = torch.tensor(lens, dtype=torch.int32, device=dev)
        at = torch.tensor(seen, device=dev) - 1
        ops.kv4_write(k.to(dev), v.to(dev), slots.to(dev), kc, vc, weights=w, positions=pos, token_positions=at)
        out = ops.kv4_decode(q.to(dev), kc, vc, table, n, d ** -0.5, max_seq_len=64, weights=w).cpu().double()
        for b in live:
            for h in range(hkv):
                rows = mine[b][h]
                ks, vs, kst, kl, vst, vl = (torch.stack([r[i] for r in rows]) for i in (0, 1, 2, 3, 4, 7))
                o, p, rel, mass, carried = O.attention(q[b, h * rep:(h + 1) * rep], ks, vs, d ** -0.5, kst, kl, vst, vl)
                assert ((out[b, h * rep:(h + 1) * rep] - o).abs() <= 2.0 ** -8 * o.abs() + 1.01 * (rel * mass + carried)).all(), f"step {step}"
                blk, t = table[b].long().cpu()[torch.arange(lens[b]) // block], torch.arange(lens[b]) % block
                now = w.cpu()[blk, h, t]
                want = torch.tensor([r[5] for r in rows], dtype=torch.float64) + p.sum(0)
                assert torch.allclose(now.double(), want, rtol=1e-4, atol=1e-6)
                for r, x in zip(rows, now.tolist()):
                    r[5] = x                                  # eviction goes by what the op holds
        if max(lens) == budget + block:
            keep, kept = ops.kv4_keep(w, pos, table, n, torch.tensor(seen, dtype=torch.int32, device=dev), budget, keep_first=2, keep_last=5)
            ops.kv4_move(kc, vc, table, keep, weights=w, positions=pos)
            for b in range(B):
                for h in range(hkv):
                    rows = mine[b][h]
                    place = O.keep([r[5] for r in rows], [r[6] for r in rows], len(rows), seen[b], budget, 2, 5)
                    assert keep[b, h, :len(place)].tolist() == place
                    mine[b][h] = [list(rows[j]) for j in place]
            lens = kept.tolist()
    assert max(lens) < budget + block and seen[0] == 75


@pytest.mark.gpu
def test_graphs_and_streams():
    """Two captured graphs over the same caches, replayed on two streams in turn with new contents and lengths, give what eager calls
    give; a call on another stream than the tensors' own as well."""
    d, block, hkv, hq, B = 128, 64, 2, 10, 3
    f = Filled(33, [1500, 700, 64], hkv, d, block, "cuda")
    shape = f.k_cache.shape[:3]
    qs = [torch.randn(B, hq, d, generator=_gen(i)).bfloat16().cuda() for i in range(2)]
    ws = [torch.zeros(shape, device="cuda") for _ in range(2)]
    pos = torch.arange(shape[0] * hkv * block, device="cuda", dtype=torch.int32).view(shape)
    seen = torch.full((B,), 10 ** 6, dtype=torch.int32, device="cuda")
    lens = f.lens_dev.clone()

    def step(i):
        out = ops.kv4_decode(qs[i], f.k_cache, f.v_cache, f.table_dev, lens, 0.1, max_seq_len=64, weights=ws[i], decay=0.0)
        return (out, *ops.kv4_keep(ws[i], pos, f.table_dev, lens, seen, 50))

    step(0)
    side = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for n in ([1500, 700, 64], [3, 0, 50], [1499, 51, 1]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        for i in range(2):
            qs[i].copy_(torch.randn(B, hq, d, generator=_gen(n[0] + i)))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(side[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        got = [[x.clone() for x in o] for o in outs]
        with torch.cuda.stream(side[0]):
            want = [step(i) for i in range(2)]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_the_same_call_gives_the_same_bits():
    f = Filled(12, [5000, 4000], 2, 128, 64, "cuda")
    q = torch.randn(4, 32, 128, generator=_gen(0)).bfloat16().cuda()
    first = None
    for _ in range(3):
        w = torch.zeros(f.k_cache.shape[:3], device="cuda")
        out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 0.1, weights=w)
        first = first or (out, w)
        assert torch.equal(out, first[0]) and torch.equal(w, first[1])


@pytest.mark.gpu
def test_far_slots():
    """Byte offsets beyond 32 bits: the last blocks of a cache of over 4 GB."""
    hkv, d, block = 8, 128, 128
    blocks = 70_000                                          # 5.2 GB of keys
    kc, vc = (torch.empty(blocks, hkv, block, d * 9 // 16, dtype=torch.uint8, device="cuda") for _ in range(2))
    n, g = 300, _gen(6)
    table = torch.tensor([[blocks - 1, 3, blocks - 2, 0]], dtype=torch.int32)
    slots = table[0].long()[torch.arange(n) // block] * block + torch.arange(n) % block
    f = Filled.__new__(Filled)
    f.lens, f.hkv, f.d, f.block, f.table = [n], hkv, d, block, table
    f.k, f.v = [_rows(g, n, hkv, d)], [_rows(g, n, hkv, d)]
    w, pos = torch.zeros(blocks, hkv, block, device="cuda"), torch.zeros(blocks, hkv, block, dtype=torch.int32, device="cuda")
    ops.kv4_write(f.k[0].cuda(), f.v[0].cuda(), slots.cuda(), kc, vc, weights=w, positions=pos, token_positions=torch.arange(n).cuda())
    assert torch.equal(ops.kv4_read(kc, vc, slots.cuda())[0].cpu(), O.stored(f.k[0])[0].float().bfloat16())
    q = torch.randn(1, 16, d, generator=g).bfloat16().cuda()
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    out = ops.kv4_decode(q, kc, vc, table.cuda(), lens, 0.1, weights=w)
    _check_decode(f, q, 1, 0.1, out)
    keep, _ = ops.kv4_keep(w, pos, table.cuda(), lens, lens, 200)
    ops.kv4_move(kc, vc, table.cuda(), keep, weights=w, positions=pos)
    for h in range(hkv):
        rows = ops.kv4_read(kc, vc, slots[:200].cuda())[1][:, h].cpu()
        assert torch.equal(rows, O.stored(f.v[0][keep[0, h].cpu().long(), h])[0].float().bfloat16())


# ----------------------------------------------------------------------------- refusals
def _args(dev="cpu"):
    kc, vc = ops.kv4_cache(3, 16, 2, 64, dev)
    return dict(kc=kc, vc=vc, k=torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=dev), slots=torch.arange(4, device=dev),
                q=torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev), table=torch.zeros(2, 2, dtype=torch.int32, device=dev),
                lens=torch.zeros(2, dtype=torch.int32, device=dev), w=torch.zeros(3, 2, 16, device=dev), pos=torch.zeros(3, 2, 16, dtype=torch.int32, device=dev),
                keep=torch.full((2, 2, 8), -1, dtype=torch.int32, device=dev))


REFUSED = {
    "cache type": lambda a: ops.kv4_read(a["kc"].float(), a["vc"].float(), a["slots"]),
    "caches differ": lambda a: ops.kv4_read(a["kc"], a["vc"][:2], a["slots"]),
    "caches with gaps": lambda a: ops.kv4_read(a["kc"][:, :, ::2], a["vc"][:, :, ::2], a["slots"]),
    "row size": lambda a: ops.kv4_read(a["kc"].view(3, 2, 48, 12), a["vc"].view(3, 2, 48, 12), a["slots"]),
    "block size": lambda a: ops.kv4_read(a["kc"][:, :, :8].contiguous(), a["vc"][:, :, :8].contiguous(), a["slots"]),
    "head size to make": lambda a: ops.kv4_cache(1, 16, 2, 96),
    "block size to make": lambda a: ops.kv4_cache(1, 24, 2, 64),
    "slot type": lambda a: ops.kv4_read(a["kc"], a["vc"], a["slots"].int()),
    "slots missing": lambda a: ops.kv4_write(a["k"], a["k"], a["slots"][:3], a["kc"], a["vc"]),
    "row type": lambda a: ops.kv4_write(a["k"].float(), a["k"].float(), a["slots"], a["kc"], a["vc"]),
    "row heads": lambda a: ops.kv4_write(a["k"][:, :1], a["k"], a["slots"], a["kc"], a["vc"]),
    "row columns with gaps": lambda a: ops.kv4_write(torch.zeros(4, 2, 128).bfloat16()[:, :, ::2], a["k"], a["slots"], a["kc"], a["vc"]),
    "positions alone": lambda a: ops.kv4_write(a["k"], a["k"], a["slots"], a["kc"], a["vc"], positions=a["pos"]),
    "weights shape": lambda a: ops.kv4_write(a["k"], a["k"], a["slots"], a["kc"], a["vc"], weights=a["w"][:2]),
    "query type": lambda a: ops.kv4_decode(a["q"].float(), a["kc"], a["vc"], a["table"], a["lens"], 1.0),
    "query head size": lambda a: ops.kv4_decode(torch.zeros(2, 4, 128).bfloat16(), a["kc"], a["vc"], a["table"], a["lens"], 1.0),
    "query heads": lambda a: ops.kv4_decode(a["q"][:, :3], a["kc"], a["vc"], a["table"], a["lens"], 1.0),
    "uneven rows": lambda a: ops.kv4_decode(torch.zeros(3, 4, 64).bfloat16(), a["kc"], a["vc"], a["table"], a["lens"], 1.0),
    "table type": lambda a: ops.kv4_decode(a["q"], a["kc"], a["vc"], a["table"].long(), a["lens"], 1.0),
    "table rows": lambda a: ops.kv4_decode(a["q"], a["kc"], a["vc"], a["table"][:1], a["lens"], 1.0),
    "lengths type": lambda a: ops.kv4_decode(a["q"], a["kc"], a["vc"], a["table"], a["lens"].long(), 1.0),
    "decode weights type": lambda a: ops.kv4_decode(a["q"], a["kc"], a["vc"], a["table"], a["lens"], 1.0, weights=a["w"].double()),
    "table too wide": lambda a: ops.kv4_decode(a["q"], a["kc"], a["vc"], torch.empty(1 << 26, dtype=torch.int32).expand(len(a["lens"]), -1), a["lens"], 0.1),
    "budget too small": lambda a: ops.kv4_keep(a["w"], a["pos"], a["table"], a["lens"], a["lens"], 4, keep_first=3, keep_last=2),
    "no budget": lambda a: ops.kv4_keep(a["w"], a["pos"], a["table"], a["lens"], a["lens"], 0),
    "positions type": lambda a: ops.kv4_keep(a["w"], a["pos"].long(), a["table"], a["lens"], a["lens"], 4),
    "seen missing": lambda a: ops.kv4_keep(a["w"], a["pos"], a["table"], a["lens"], a["lens"][:1], 4),
    "keep type": lambda a: ops.kv4_move(a["kc"], a["vc"], a["table"], a["keep"].long()),
    "keep heads": lambda a: ops.kv4_move(a["kc"], a["vc"], a["table"], a["keep"][:, :1].contiguous()),
}


@pytest.mark.parametrize("what", list(REFUSED))
def test_refusals(what):
    with pytest.raises(AssertionError):
        REFUSED[what](_args())


@pytest.mark.gpu
def test_caches_off_16_bytes_are_refused():
    buf = torch.zeros(2 * 16 * 36 + 8, dtype=torch.uint8, device="cuda")[8:].view(1, 2, 16, 36)
    kc, vc = ops.kv4_cache(1, 16, 2, 64, "cuda")
    with pytest.raises(RuntimeError, match="omni_kv4_read"):
        ops.kv4_read(kc, buf, torch.zeros(1, dtype=torch.int64, device="cuda"))


@pytest.mark.gpu
def test_weights_of_too_many_rows_are_refused():
    a = _args("cuda")
    q = torch.zeros(2 * 129, 4, 64, dtype=torch.bfloat16, device="cuda")
    ops.kv4_decode(q, a["kc"], a["vc"], a["table"], a["lens"], 1.0)
    with pytest.raises(AssertionError, match="256"):
        ops.kv4_decode(q, a["kc"], a["vc"], a["table"], a["lens"], 1.0, weights=a["w"])


@pytest.mark.gpu
def test_blocks_and_slots_outside_the_cache_are_skipped_and_reported():
    def reported(f):
        f()
        torch.cuda.synchronize()
        with pytest.raises(nat.KernelProtocolError, match="out of bounds.*4-bit cache"):
            nat.check_status()
    a = _args("cuda")
    far = torch.tensor([0, 3 * 16, 10 ** 12, 5], device="cuda")
    reported(lambda: ops.kv4_write(a["k"] + 1, a["k"] + 1, far, a["kc"], a["vc"]))
    k, v = ops.kv4_read(a["kc"], a["vc"], torch.tensor([0, 5, 1], device="cuda"))
    assert (k[:2] == 1).all() and (v[:2] == 1).all() and (k[2] == 0).all()
    reported(lambda: ops.kv4_read(a["kc"], a["vc"], far))
    lens = torch.tensor([20, 20], dtype=torch.int32, device="cuda")
    bad = torch.tensor([[0, 3], [-1, 1]], dtype=torch.int32, device="cuda")
    reported(lambda: ops.kv4_decode(a["q"], a["kc"], a["vc"], bad, lens, 1.0, weights=a["w"]))
    reported(lambda: ops.kv4_decode(a["q"], a["kc"], a["vc"], a["table"], lens + 13, 1.0))
    reported(lambda: ops.kv4_keep(a["w"], a["pos"], bad, lens, lens, 8))
    reported(lambda: ops.kv4_keep(a["w"], a["pos"], a["table"], lens + 13, lens, 8))
    a["keep"][0, 0, 3], a["keep"][1, 1, 2] = 30, 5           # place 30 is in block 3; place 5 is itself filled
    reported(lambda: ops.kv4_move(a["kc"], a["vc"], bad, a["keep"]))
