"""The 4-bit paged cache on the ways through its kernels that small calls do not take, and what it refuses on either device."""
import threading

import pytest
import torch

import kv4_oracle as O
from omni_infer_b200 import ops
from omni_infer_b200.ops import _native as nat
from omni_infer_b200.ops import kv4
from test_kv4_ops import BOTH, Filled, _args, _check_decode, _gen, _rows


# ----------------------------------------------------------------------------- the layout
def _bytes(x, block, values):
    """Rows [block, hkv, d] as the bytes of a piece for each head, word by word as the layout is described: planes of up to two groups of 64
    columns, eight columns a word; keys: of a token, for each 16 columns c and group of the plane, the two words of these columns; values:
    two tokens a row of eight chunks, chunk r in the place r ^ 2 (pair % 4), or r ^ 4 (pair / 2 % 2) with one group a plane, with the words of
    the columns 8 r .. 8 r + 7 of the groups of the even token, then of the odd one.  Behind the codes a step and a lowest value for each
    token and group."""
    n, hkv, d = x.shape
    codes, step, lo = kv4.kv4_quantise_ref(x)
    out = torch.zeros(hkv, block * d * 9 // 16, dtype=torch.uint8)
    groups, per = d // 64, min(d // 64, 2)
    for h in range(hkv):
        for t in range(n):
            for g in range(groups):
                base = g // per * block * 32 * per
                for word in range(8):
                    if values:
                        pair = t // 2
                        chunk = word ^ (2 * (pair % 4)) if per == 2 else word ^ (4 * (pair // 2 % 2))
                        at = base + pair * 64 * per + chunk * 8 * per + (t % 2) * 4 * per + (g % per) * 4
                    else:
                        at = base + t * 32 * per + (word // 2) * 8 * per + (g % per) * 8 + (word % 2) * 4
                    eight = codes[t, h, g * 64 + word * 8:g * 64 + word * 8 + 8].tolist()
                    for i in range(4):
                        out[h, at + i] = eight[2 * i] | eight[2 * i + 1] << 4
                at = block * d // 2 + (t * groups + g) * 4
                out[h, at:at + 4] = torch.stack([step[t, h, g], lo[t, h, g]]).view(torch.uint8)
    return out


@BOTH
@pytest.mark.parametrize("d,block,hkv", [(64, 16, 3), (64, 48, 1), (128, 32, 2), (128, 80, 1), (256, 16, 2), (256, 64, 1)])
def test_the_bytes_of_a_cache(dev, d, block, hkv):
    """The same on either device, so that blocks can go between them; and read back from bytes that no op has written."""
    g = _gen(d + block)
    k, v = _rows(g, block, hkv, d), _rows(g, block, hkv, d, levels=False)
    v[1] = 0.0
    slots = torch.arange(block, 2 * block)
    kc, vc = ops.kv4_cache(3, block, hkv, d, dev)
    ops.kv4_write(k.to(dev), v.to(dev), slots.to(dev), kc, vc)
    want = [torch.zeros(kc.shape, dtype=torch.uint8) for _ in range(2)]
    for w, x, values in zip(want, (k, v), (False, True)):
        w[1] = _bytes(x, block, values).view(hkv, block, -1)
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
    got = ops.kv4_read(want[0].to(dev), want[1].to(dev), slots.to(dev))
    for x, stored in zip(got, (k, v)):
        assert torch.equal(x.cpu(), O.stored(stored)[0].float().bfloat16())


@BOTH
@pytest.mark.parametrize("d,hkv", [(64, 1), (64, 3), (128, 2), (256, 3)])
@pytest.mark.parametrize("shift", [0, 1, 5, 8])
def test_rows_that_do_not_start_on_16_bytes(dev, d, hkv, shift):
    g, T, block = _gen(d + shift), 37, 16
    wide = torch.randn(T, hkv + 2, d + 8, generator=g).bfloat16().to(dev)
    k, v = wide[:, :hkv, shift:shift + d], wide[:, 2:, 8 - shift:8 - shift + d]
    slots = torch.randperm(3 * block, generator=g)[:T]
    kc, vc = ops.kv4_cache(3, block, hkv, d, dev)
    ops.kv4_write(k, v, slots.to(dev), kc, vc)
    for got, x in zip(ops.kv4_read(kc, vc, slots.to(dev)), (k, v)):
        assert torch.equal(got.cpu(), O.stored(x)[0].float().bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("d,rows,rep", [(64, 1, 3), (64, 5, 4), (256, 1, 6), (256, 3, 4)])
@pytest.mark.parametrize("shift", [1, 8])
def test_queries_that_do_not_start_on_16_bytes(d, rows, rep, shift):
    f = Filled(d, [130, 0, 19], 2, d, 16, "cuda")
    q = torch.randn(3 * rows, 2 * rep + 1, d + 8, generator=_gen(rows)).bfloat16().cuda()[:, 1:, shift:shift + d]
    w = torch.zeros(f.k_cache.shape[:3], device="cuda")
    out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, d ** -0.5, weights=w, decay=0.0)
    _check_decode(f, q, rows, d ** -0.5, out, w, torch.zeros(f.k_cache.shape[:3]))


# ----------------------------------------------------------------------------- how work is cut
def _scheme(f, hq, rows):
    """What the decode kernel does with these requests: the rule of its launch and of its shares, in words."""
    rep, d = hq // f.hkv, f.d
    tile = 16 if d <= 128 and rows * rep > 8 else 8
    tokens = 32 if d == 256 else 64
    chunks = -(-rows * rep // tile)
    blocks, least = kv4._blocks(len(f.lens) * f.hkv * chunks, -(-f.table.shape[1] * f.block // tokens), 3 if tile * d <= 1024 else 2)
    if least == 0:
        return "whole"
    busy = sum(n > 0 for n in f.lens) * f.hkv * chunks
    return "parts" if busy * 2 <= blocks else "through"


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 1 << 28])
@pytest.mark.parametrize("B,n,hkv,rep,rows,d,block", [
    (46, 1100, 6, 2, 1, 128, 64),                             # more than 32 requests, 276 items, several to a block and parts of them
    (90, 900, 3, 1, 3, 64, 16),
    (40, 1000, 5, 12, 1, 128, 32),                            # tiles of 16 rows
    (40, 900, 4, 16, 2, 64, 128),                             # two tiles of 16 rows a head
    (46, 500, 4, 4, 1, 256, 16),                              # 256 columns: tiles of 32 tokens, parts, a join of 256 threads
    (70, 1500, 4, 1, 1, 128, 128),
])
def test_tiles_of_all_requests_shared_out(monkeypatch, B, n, hkv, rep, rows, d, block, room):
    """Requests of very uneven lengths, with some of no tokens among them, whose tiles are numbered through: blocks start and end inside items
    and take several of them."""
    monkeypatch.setattr(kv4, "KEPT_SCORES", room)
    lens = [0 if i % 13 == 5 or i == B - 1 else max(1, n - 211 * i % n) for i in range(B)]
    f = Filled(B + d, lens, hkv, d, block, "cuda")
    assert _scheme(f, hkv * rep, rows) == "through"
    q = torch.randn(B * rows, hkv * rep, d, generator=_gen(B)).bfloat16().cuda()
    old = torch.rand(f.k_cache.shape[:3], generator=_gen(1))
    w = old.cuda()
    out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, d ** -0.5, weights=w, decay=0.5)
    _check_decode(f, q, rows, d ** -0.5, out, w, old, 0.5)
    assert torch.equal(out, ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, d ** -0.5, max_seq_len=n))


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 1 << 28])
@pytest.mark.parametrize("rows,rep", [(1, 1), (2, 7)])
def test_256_columns_split_into_parts(monkeypatch, rows, rep, room):
    monkeypatch.setattr(kv4, "KEPT_SCORES", room)
    f = Filled(8, [3000, 0, 401, 31], 2, 256, 48, "cuda")
    assert _scheme(f, 2 * rep, rows) == "parts"
    q = torch.randn(4 * rows, 2 * rep, 256, generator=_gen(rep)).bfloat16().cuda()
    w = torch.ones(f.k_cache.shape[:3], device="cuda")
    out = ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 1 / 16, weights=w)
    _check_decode(f, q, rows, 1 / 16, out, w, torch.ones(f.k_cache.shape[:3]), 1.0)


@BOTH
@pytest.mark.parametrize("d", [64, 128, 256])
def test_equal_weights_keep_the_first_places(dev, d):
    """A fresh cache: all weights are 0, and the places from the budget on go."""
    lens, budget, hkv, block = [900, 300, 40], 128, 2, 16
    f = torch.arange(3 * 60, dtype=torch.int32).view(3, 60).to(dev)
    w = torch.zeros(180, hkv, block, device=dev)
    pos = torch.zeros(180, hkv, block, dtype=torch.int32, device=dev)
    for b in range(3):
        pos[f[b].long()] = torch.arange(60 * block, dtype=torch.int32, device=dev).view(60, 1, block)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    keep, kept = ops.kv4_keep(w, pos, f, n, n, budget, keep_first=4, keep_last=d // 16)
    for b, m in enumerate(lens):
        last = d // 16 if m > budget else 0
        want = list(range(min(m, budget) - last)) + list(range(m - last, m)) + [-1] * max(0, budget - m)
        assert kept[b] == min(m, budget) and all(keep[b, h].tolist() == want for h in range(hkv))


# ----------------------------------------------------------------------------- calls at once, and their count
@pytest.mark.gpu
def test_threads_with_calls_of_different_rows(monkeypatch):
    """Calls from several host threads at once, each with another number of rows and so with another need of shared memory."""
    monkeypatch.setattr(kv4, "KEPT_SCORES", 0)
    f = Filled(14, [300, 80], 1, 64, 16, "cuda")
    each = [1, 256, 9, 130, 2, 64, 255, 33]
    qs = [torch.randn(2 * r, 1, 64, generator=_gen(r)).bfloat16().cuda() for r in each]
    torch.cuda.synchronize()
    got, ready = [None] * len(each), threading.Barrier(len(each))

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            ready.wait()
            for _ in range(5):
                w = torch.zeros(f.k_cache.shape[:3], device="cuda")
                got[i] = (ops.kv4_decode(qs[i], f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 0.125, weights=w), w)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(each))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for r, q, out in zip(each, qs, got):
        assert out is not None, f"the call with {r} rows failed"
        w = torch.zeros(f.k_cache.shape[:3], device="cuda")
        assert torch.equal(out[0], ops.kv4_decode(q, f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 0.125, weights=w)) and torch.equal(out[1], w)


@pytest.mark.gpu
@pytest.mark.parametrize("room", [0, 1 << 28])
@pytest.mark.parametrize("n,weighted,launches", [(100, False, 1), (100, True, 2), (2000, False, 2), (2000, True, 3)])
def test_launches_are_counted(monkeypatch, n, weighted, launches, room):
    monkeypatch.setattr(kv4, "KEPT_SCORES", room)
    f = Filled(1, [n], 1, 64, 16, "cuda")
    w = torch.zeros(f.k_cache.shape[:3], device="cuda") if weighted else None
    before = nat.launch_count()
    ops.kv4_decode(torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda"), f.k_cache, f.v_cache, f.table_dev, f.lens_dev, 1.0, weights=w)
    assert nat.launch_count() - before == launches


# ----------------------------------------------------------------------------- refusals, the same on both devices
def _many(a, n):
    return torch.zeros(n, 2, dtype=torch.int32, device=a["lens"].device), torch.zeros(n, dtype=torch.int32, device=a["lens"].device)


REFUSED = {
    "weights of too many rows": lambda a: ops.kv4_decode(torch.zeros(2 * 129, 4, 64, dtype=torch.bfloat16, device=a["q"].device), a["kc"], a["vc"], a["table"], a["lens"],
                                                         1.0, weights=a["w"]),
    "too many requests to decode": lambda a: ops.kv4_decode(torch.zeros(1 << 16, 2, 64, dtype=torch.bfloat16, device=a["q"].device), a["kc"], a["vc"], *_many(a, 1 << 16), 1.0),
    "too many requests to keep": lambda a: ops.kv4_keep(a["w"], a["pos"], *_many(a, 1 << 16), _many(a, 1 << 16)[1], 4),
    "too many requests to move": lambda a: ops.kv4_move(a["kc"], a["vc"], _many(a, 1 << 16)[0], torch.full((1 << 16, 2, 1), -1, dtype=torch.int32, device=a["q"].device)),
}


@BOTH
@pytest.mark.parametrize("what", list(REFUSED))
def test_refusals_on_both_devices(dev, what):
    with pytest.raises(AssertionError):
        REFUSED[what](_args(dev))


def test_blocks_and_slots_outside_the_cache_on_the_cpu():
    """What a GPU skips and reports later is an error at once on the CPU, ahead of any change."""
    a = _args()
    lens, bad = torch.tensor([20, 20], dtype=torch.int32), torch.tensor([[0, 3], [-1, 1]], dtype=torch.int32)
    before = [a[x].clone() for x in ("kc", "vc", "w", "pos")]
    own, far = a["keep"].clone(), a["keep"].clone()
    own[0, 0, 3] = 5                                         # place 5 is itself filled
    far[0, 1, 2] = 40                                        # behind the table
    for call in (lambda: ops.kv4_write(a["k"] + 1, a["k"] + 1, torch.tensor([0, 48, 1, 5]), a["kc"], a["vc"], weights=a["w"]),
                 lambda: ops.kv4_read(a["kc"], a["vc"], torch.tensor([0, 48])),
                 lambda: ops.kv4_decode(a["q"], a["kc"], a["vc"], bad, lens, 1.0, weights=a["w"]),
                 lambda: ops.kv4_decode(a["q"], a["kc"], a["vc"], bad[1:].expand(2, -1), lens, 1.0, weights=a["w"]),
                 lambda: ops.kv4_decode(a["q"], a["kc"], a["vc"], a["table"], lens + 13, 1.0),
                 lambda: ops.kv4_keep(a["w"], a["pos"], bad[1:].expand(2, -1), lens, lens, 8),
                 lambda: ops.kv4_keep(a["w"], a["pos"], a["table"], lens + 13, lens, 8),
                 lambda: ops.kv4_keep(a["w"], a["pos"], a["table"], lens + 13, lens, 40),
                 lambda: ops.kv4_move(a["kc"], a["vc"], bad[1:].expand(2, -1), torch.full((2, 2, 8), 20, dtype=torch.int32)),
                 lambda: ops.kv4_move(a["kc"], a["vc"], a["table"], own, weights=a["w"]),
                 lambda: ops.kv4_move(a["kc"], a["vc"], a["table"], far)):
        with pytest.raises(IndexError):
            call()
    assert all(torch.equal(a[x], b) for x, b in zip(("kc", "vc", "w", "pos"), before))
