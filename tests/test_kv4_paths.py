"""The 4-bit paged cache on the ways through its kernels that small calls do not take, and what it refuses on either device."""
import threading

import pytest
import torch

from omni_infer_b200 import ops
from omni_infer_b200.ops import _native as nat
from omni_infer_b200.ops import kv4
from test_kv4_ops import BOTH, Filled, _args, _gen


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
