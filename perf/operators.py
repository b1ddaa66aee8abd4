"""The 4-bit paged key/value cache and what works on it: writing rows and reading them back, decode attention with the weights
that it gives to the cached tokens, and eviction by those weights.

A cache is a uint8 tensor [blocks, key/value heads, block size, 9 d / 16].  The piece of one block and head holds its codes
(d / 2 bytes a token) and behind them its scales (for each token and each group of 64 columns one bf16 step and one bf16 lowest
value); value = code * step + lowest.  Codes are laid out for the kernels: see ``code_places``."""
import random

import torch

own = False

GROUP = 64


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # one short conversation, nothing else on the card: latency only (the 32/4 heads of 128 of the framework's GQA model)
        dict(name="decode one short", kind="decode", batch=1, length=200, ragged=False, rows=1, hq=32, hkv=4, d=128, block=128, mode="plain"),
        # a few requests of uneven length that check three speculated tokens each, seven query heads to a key head, small pages
        dict(name="decode speculated ragged", kind="decode", batch=9, length=1531, ragged=True, rows=3, hq=14, hkv=2, d=64, block=16, mode="plain"),
        # an ordinary full decode batch with uneven lengths
        dict(name="decode batch ragged", kind="decode", batch=64, length=8190, ragged=True, rows=1, hq=32, hkv=4, d=128, block=128, mode="plain"),
        # two requests with very long contexts: the whole card on a few rows
        dict(name="decode long", kind="decode", batch=2, length=131067, ragged=False, rows=1, hq=64, hkv=8, d=128, block=128, mode="plain"),
        # a decode step that adds its attention weights to those of the earlier steps
        dict(name="decode adding weights", kind="decode", batch=32, length=4099, ragged=True, rows=1, hq=32, hkv=4, d=128, block=128, mode="add"),
        # the last rows of two long prompts score the whole prompt before it is cut down
        dict(name="decode window weights", kind="decode", batch=2, length=30011, ragged=False, rows=16, hq=32, hkv=4, d=128, block=128, mode="set"),
        # the rows of one decode step of a batch: written, and read back
        dict(name="write read step", kind="rows", new=64, context=64, hkv=4, d=128, block=128),
        # a portion of a prompt: its rows written, the whole context read back for the attention of the portion
        dict(name="write read portion", kind="rows", new=4099, context=40003, hkv=8, d=128, block=128),
        # a decode batch whose caches have run one block over their budget
        dict(name="keep step", kind="keep", batch=32, length=2176, ragged=False, hkv=4, block=128, budget=2048),
        # long prompts cut down to a budget
        dict(name="keep prompt", kind="keep", batch=4, length=60001, ragged=True, hkv=8, block=128, budget=4096),
        # rows of that step brought to their places, and the cache read back as a next portion of a prompt does
        dict(name="move step", kind="move", batch=8, length=640, ragged=False, hkv=2, d=64, block=16, budget=509),
        dict(name="move prompt", kind="move", batch=8, length=16384, ragged=True, hkv=4, d=128, block=128, budget=2048),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng: random.Random):
    kind = rng.choice(["decode", "decode", "decode", "rows", "keep", "move"])
    d, hkv, block = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 48, 64, 128, 256])
    if kind == "rows":
        context = _spread(rng, 1, 40000)
        return dict(kind=kind, new=_spread(rng, 1, min(context, 8192)), context=context, hkv=hkv, d=d if context * hkv < 100000 else 64, block=block)
    batch = _spread(rng, 1, 64)
    length = _spread(rng, 1, max(2, min(131072, 1500000 * 128 // (d * hkv * batch))))
    ragged = rng.random() < 0.6
    if kind == "decode":
        mode = rng.choice(["plain", "plain", "add", "set"])
        rep = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
        rows = rng.choice([1, 1, 2, 3, 4, 8, 16]) if batch * length * hkv < 300000 else 1
        return dict(kind=kind, batch=batch, length=length, ragged=ragged, rows=min(rows, 128 // rep), hq=hkv * rep, hkv=hkv, d=d, block=block, mode=mode)
    length = max(4, length)
    case = dict(kind=kind, batch=batch, length=length, ragged=ragged, hkv=hkv, block=block, budget=max(2, int(length * rng.uniform(0.05, 1.1))))
    if kind == "move":
        case["d"] = d
        case["budget"] = min(case["budget"], max(2, 400000 // (batch * hkv)))
    return case


def lengths(case):
    """Cached tokens of each request: the case's own, or uneven ones with a padding row at the end of a larger batch."""
    n, b = case["length"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    return [0 if i == b - 1 and b >= 8 else max(1, n - (i * 977) % max(1, n * 3 // 4)) for i in range(b)]


# ----------------------------------------------------------------------------- the layout of a cache
def code_places(block, d, values, device):
    """Byte and shift of the code of every (token, column) in the piece of one block and head, flat.

    The codes lie in planes of 128 columns (64 for d = 64), eight columns to a 4-byte word, column j of a word in bits 4 j to
    4 j + 3.  Keys: a token's words one after the other, the words of columns 16 c to 16 c + 15 of all groups of the plane
    together.  Values: two tokens share their words, eight chunks each of eight columns of every group, first the even token's,
    then the odd one's, the chunks' order changed by the pair's number."""
    t = torch.arange(block, device=device)[:, None]
    col = torch.arange(d, device=device)[None, :]
    per = min(d // GROUP, 2)                                  # groups of a plane
    g, plane, j = col // GROUP, col // (GROUP * per), col % 8
    if not values:
        word = (col % 64 // 16) * 2 * per + g % per * 2 + col % 16 // 8
        byte = (plane * block + t) * 32 * per + word * 4 + j // 2
    else:
        pair, chunk = t // 2, col % 64 // 8
        chunk = chunk ^ (pair % 4 * 2) if per == 2 else chunk ^ (pair // 2 % 2 * 4)
        byte = (plane * block + pair * 2) * 32 * per + chunk * 8 * per + t % 2 * 4 * per + g % per * 4 + j // 2
    shift = (4 * (j % 2)).expand(block, d)
    return byte.reshape(-1), shift.reshape(-1)


def quantise(x):
    """x [..., d] bf16 -> codes [..., d] uint8, (step, lowest) [..., d / 64] bf16."""
    v = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = v.amin(-1), v.amax(-1)
    bits = ((hi - lo) / torch.full_like(hi, 15.0)).view(torch.int32)   # a division: a quotient on the grid of bf16 stays there
    step = ((bits + 0xffff) & -0x10000).view(torch.float32)   # rounded up to bf16
    step = torch.where(torch.isfinite(hi - lo), step, torch.full_like(step, float("nan")))
    code = torch.round((v - lo[..., None]) / step[..., None]).clamp(0, 15)
    code = torch.where(step[..., None] > 0, code, torch.zeros_like(code))
    return code.flatten(-2).to(torch.uint8), step.to(torch.bfloat16), lo.to(torch.bfloat16)


def pack(codes, step, lo, values):
    """codes [n, block, d], step and lo [n, block, d / 64] -> pieces [n, block, 9 d / 16]."""
    n, block, d = codes.shape
    byte, shift = code_places(block, d, values, codes.device)
    source = torch.empty(block * d, dtype=torch.int64, device=codes.device)
    source[byte * 2 + shift // 4] = torch.arange(block * d, device=codes.device)
    flat = codes.reshape(n, -1)
    packed = flat[:, source[0::2]] | flat[:, source[1::2]] << 4
    scales = torch.stack([step, lo], -1).reshape(n, -1).contiguous().view(torch.uint8)
    return torch.cat([packed, scales], 1).reshape(n, block, d * 9 // 16)


def unpack(pieces, values):
    """pieces [n, block, 9 d / 16] -> values in 32 bits [n, block, d]."""
    n, block, row = pieces.shape
    d = row * 16 // 9
    flat = pieces.reshape(n, -1)
    byte, shift = code_places(block, d, values, pieces.device)
    codes = (flat[:, byte] >> shift.to(torch.uint8) & 15).reshape(n, block, d // GROUP, GROUP).float()
    scales = flat[:, block * d // 2:].contiguous().view(torch.bfloat16).reshape(n, block, d // GROUP, 2).float()
    return (codes * scales[..., :1] + scales[..., 1:]).reshape(n, block, d)


# ----------------------------------------------------------------------------- inputs
def _keys_values(gen, shape, d):
    """Keys with columns of their own level and spread, as projections give them; values without."""
    dev = gen.device
    level = torch.randn(d, generator=gen, device=dev) * (torch.rand(d, generator=gen, device=dev) < 0.1) * 4
    k = torch.randn(*shape, d, generator=gen, device=dev).add_(level).to(torch.bfloat16)
    v = torch.randn(*shape, d, generator=gen, device=dev).mul_(0.7).to(torch.bfloat16)
    return k, v


def _pages(case, gen):
    """Block table [batch, blocks of a request] over a shuffled pool, and the pool's size."""
    per = -(-case["length"] // case["block"])
    n = case["batch"] * per + 3
    table = torch.randperm(n, generator=gen, device=gen.device)[:case["batch"] * per].reshape(case["batch"], per)
    return table.to(torch.int32), n


def _filled(case, gen, blocks):
    block, hkv, d = case["block"], case["hkv"], case["d"]
    caches = [torch.empty(blocks, hkv, block, d * 9 // 16, dtype=torch.uint8, device=gen.device) for _ in range(2)]
    step = max(1, (1 << 26) // (hkv * block * d))
    for at in range(0, blocks, step):
        n = min(step, blocks - at)
        for c, x, values in zip(caches, _keys_values(gen, (n * hkv, block), d), (False, True)):
            c[at:at + n] = pack(*quantise(x), values).reshape(n, hkv, block, -1)
    return caches


def _weights(case, gen, blocks, table):
    """Weights as attention leaves them (a few heavy tokens, many light ones) and the tokens' positions: those of requests that
    have been cut down before, so that places are not in the order of positions."""
    shape = (blocks, case["hkv"], case["block"])
    w = torch.exp(3 * torch.randn(shape, generator=gen, device=gen.device) - 4)
    w = torch.where(torch.rand(shape, generator=gen, device=gen.device) < 0.05, torch.zeros_like(w), w)
    n = table.shape[1] * case["block"]
    order = torch.rand(case["batch"], case["hkv"], n, generator=gen, device=gen.device).argsort(-1)
    pos = torch.full(shape, -1, dtype=torch.int32, device=gen.device)
    lens = torch.tensor(lengths(case), device=gen.device)
    half = (lens // 2)[:, None, None]                        # the first half of the places are shuffled among themselves
    at = torch.arange(n, device=gen.device).expand(case["batch"], case["hkv"], n)
    key = torch.where(at < half, order, n + at)
    p = key.argsort(-1).argsort(-1).to(torch.int32) + 7      # 7 tokens have been dropped before
    pos[table.long()] = p.unflatten(2, (-1, case["block"])).permute(0, 2, 1, 3)
    return w, pos


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    dev = gen.device
    s = dict(case=case)
    if case["kind"] == "rows":
        hkv, d, block = case["hkv"], case["d"], case["block"]
        blocks = -(-case["context"] // block) + 2
        s["k_cache"], s["v_cache"] = _filled(case, gen, blocks)
        order = torch.randperm(blocks, generator=gen, device=dev)
        at = torch.arange(case["context"], device=dev)
        s["slots"] = order[at // block] * block + at % block                  # of the whole context
        s["new_slots"] = s["slots"][case["context"] - case["new"]:].clone()
        k, v = _keys_values(gen, (case["new"], hkv), d)
        qkv = torch.cat([torch.zeros(case["new"], 4 * hkv, d, dtype=k.dtype, device=dev), k, v], 1)   # the merged projection's rows
        s["k"], s["v"] = qkv[:, 4 * hkv:5 * hkv], qkv[:, 5 * hkv:]
        return s
    table, blocks = _pages(case, gen)
    s["table"], s["lens"] = table, torch.tensor(lengths(case), dtype=torch.int32, device=dev)
    if case["kind"] in ("decode", "move"):
        s["k_cache"], s["v_cache"] = _filled(case, gen, blocks)
    if case["kind"] == "decode":
        t, hq, d = case["batch"] * case["rows"], case["hq"], case["d"]
        qkv = torch.randn(t, hq + 2 * case["hkv"], d, generator=gen, device=dev).mul_(1.5).to(torch.bfloat16)
        s["q"] = qkv[:, :hq]
        if case["mode"] != "plain":
            s["weights"] = torch.rand(blocks, case["hkv"], case["block"], generator=gen, device=dev)
        return s
    s["weights"], s["positions"] = _weights(case, gen, blocks, table)
    s["seen"] = s["lens"] + 7
    s["first"], s["last"] = min(9, case["budget"] // 3), min(32, case["budget"] // 3)
    if case["kind"] == "move":
        s["keep"], kept = plain_keep(s)
        at = torch.arange(case["budget"], device=dev)
        ok = at[None] < kept[:, None]
        per = table.shape[1] * case["block"]
        at = at.clamp(max=per - 1)
        s["slots"] = (table.long()[:, at // case["block"]] * case["block"] + at % case["block"])[ok]
    return s


# ----------------------------------------------------------------------------- one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _run_own(s, kind)
    return {"decode": plain_decode, "rows": plain_rows, "keep": plain_keep, "move": plain_move}[kind](s)


def _run_own(s, kind):
    from omni_infer_b200 import ops
    case = s["case"]
    if kind == "decode":
        scale, longest = case["d"] ** -0.5, case["length"]
        if case["mode"] == "plain":
            return ops.kv4_decode(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], scale, max_seq_len=longest)
        w = s["weights"] if case["mode"] == "set" else s["weights"].clone()      # added to in place
        out = ops.kv4_decode(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], scale, max_seq_len=longest, weights=w,
                             decay=0.0 if case["mode"] == "set" else 1.0)
        return out, w
    if kind == "rows":
        ops.kv4_write(s["k"], s["v"], s["new_slots"], s["k_cache"], s["v_cache"])
        return ops.kv4_read(s["k_cache"], s["v_cache"], s["slots"])
    if kind == "keep":
        return ops.kv4_keep(s["weights"], s["positions"], s["table"], s["lens"], s["seen"], case["budget"], keep_first=s["first"],
                            keep_last=s["last"], max_seq_len=case["length"])
    ops.kv4_move(s["k_cache"], s["v_cache"], s["table"], s["keep"], weights=s["weights"], positions=s["positions"])
    k, v = ops.kv4_read(s["k_cache"], s["v_cache"], s["slots"])
    return k, v, s["weights"], s["positions"]


def _of_requests(x, table):
    """Pieces or numbers by block [blocks, hkv, block, ...] -> by request [batch, hkv, tokens, ...]."""
    return x[table.long()].transpose(1, 2).flatten(2, 3)


def _places(table, block, n):
    """Block and offset of the places 0 .. n - 1 of every request."""
    at = torch.arange(n, device=table.device).clamp(max=table.shape[1] * block - 1)
    return table.long()[:, at // block], at % block


def plain_decode(s):
    case, table = s["case"], s["table"].long()
    b, rows, hq, hkv, d = case["batch"], case["rows"], case["hq"], case["hkv"], case["d"]
    rep = hq // hkv
    k, v = (unpack(c[table].flatten(0, 2), values).reshape(b, -1, hkv, case["block"], d).transpose(1, 2).flatten(2, 3)
            for c, values in ((s["k_cache"], False), (s["v_cache"], True)))
    n = k.shape[2]
    q = s["q"].float().reshape(b, rows, hkv, rep, d).transpose(1, 2).reshape(b, hkv, rows * rep, d)
    score = (torch.matmul(q, k.transpose(2, 3)) * d ** -0.5).reshape(b, hkv, rows, rep, n)
    sees = s["lens"][:, None] - rows + 1 + torch.arange(rows, device=q.device)               # keys that each row sees
    seen = torch.arange(n, device=q.device) < sees[:, None, :, None, None]
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p.reshape(b, hkv, rows * rep, n), v).reshape(b, hkv, rows, rep, d).transpose(1, 2).reshape(b * rows, hq, d)
    out = out.to(torch.bfloat16)
    if case["mode"] == "plain":
        return out
    step = p.sum((2, 3)).unflatten(2, (-1, case["block"])).transpose(1, 2)                    # [b, blocks, hkv, block]
    old = s["weights"][table]
    there = (torch.arange(n, device=q.device) < s["lens"][:, None]).reshape(b, -1, 1, case["block"])
    new = torch.where(there, step if case["mode"] == "set" else old + step, old)
    w = s["weights"].clone()
    w[table] = new
    return out, w


def plain_rows(s):
    case, new = s["case"], s["new_slots"]
    block, hkv, d = case["block"], case["hkv"], case["d"]
    got = []
    for cache, x, values in ((s["k_cache"], s["k"], False), (s["v_cache"], s["v"], True)):
        codes, step, lo = quantise(x)
        # codes: two to a byte, each half of the byte by itself; the other half is kept
        byte, shift = (a.reshape(block, d)[new % block] for a in code_places(block, d, values, new.device))
        flat = cache.reshape(cache.shape[0], hkv, -1)
        at, head = (new // block)[:, None, None], torch.arange(hkv, device=new.device)[None, :, None]
        for half in (0, 4):
            here = shift[0] == half
            where = (at, head, byte[:, here][:, None, :])
            flat[where] = flat[where] & (0xf0 if half == 0 else 0x0f) | codes[:, :, here] << half
        scales = torch.stack([step, lo], -1).flatten(2).view(torch.uint8)                     # [n, hkv, d / 16]
        places = block * d // 2 + (new % block)[:, None] * (d // 16) + torch.arange(d // 16, device=new.device)
        flat[(at, head, places[:, None, :])] = scales
        got.append(_read(cache, s["slots"], values))
    return tuple(got)


def _read(cache, slots, values):
    """Rows of a cache -> [rows, hkv, d] bf16."""
    blocks, hkv, block, row = cache.shape
    d = row * 16 // 9
    byte, shift = (a.reshape(block, d)[slots % block][:, None, :] for a in code_places(block, d, values, cache.device))
    flat = cache.reshape(blocks, hkv, -1)
    at, head = (slots // block)[:, None, None], torch.arange(hkv, device=cache.device)[None, :, None]
    codes = (flat[at, head, byte] >> shift.to(torch.uint8) & 15).float().unflatten(2, (-1, GROUP))
    places = block * d // 2 + (slots % block)[:, None] * (d // 16) + torch.arange(d // 16, device=cache.device)
    scales = flat[at, head, places[:, None, :]].view(torch.bfloat16).float().unflatten(2, (-1, 2))
    return (codes * scales[..., :1] + scales[..., 1:]).flatten(2).to(torch.bfloat16)


def plain_keep(s):
    case, budget = s["case"], s["case"]["budget"]
    w, pos = _of_requests(s["weights"], s["table"]), _of_requests(s["positions"], s["table"])
    n = w.shape[2]
    at = torch.arange(n, device=w.device)
    lens = s["lens"].long()[:, None, None]
    safe = (pos < s["first"]) | (pos >= s["seen"][:, None, None] - s["last"])
    key = torch.where(safe, torch.full_like(w, float("inf")), w)
    key = torch.where(at < lens, key, torch.full_like(w, float("-inf")))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices                     # ties: the lowest place first
    kept = torch.zeros_like(key, dtype=torch.bool).scatter_(-1, order[..., :budget], True) & (at < lens)
    far = kept & (at >= budget)                                                               # these have to move
    far_places = torch.sort((~far).to(torch.uint8), dim=-1, stable=True).indices
    near = torch.zeros(*kept.shape[:2], max(budget, n), dtype=torch.bool, device=w.device)
    near[..., :n] = kept
    near, place = near[..., :budget], torch.arange(budget, device=w.device)
    hole = ~near & (place < lens)
    source = far_places.gather(-1, (hole.long().cumsum(-1) - 1).clamp(0, n - 1))
    keep = torch.where(hole, source, place.expand_as(source))
    keep = torch.where(place < lens, keep, torch.full_like(keep, -1))
    return keep.to(torch.int32), s["lens"].clamp(max=budget)


def plain_move(s):
    case, keep = s["case"], s["keep"].long()
    block, hkv, n = case["block"], case["hkv"], case["budget"]
    moves = (keep >= 0) & (keep != torch.arange(n, device=keep.device))
    b, head, to = moves.nonzero(as_tuple=True)
    frm = keep[b, head, to]
    table = s["table"].long()
    fb, fo, tb, to = table[b, frm // block], frm % block, table[b, to // block], to % block
    d = case["d"]
    for cache, values in ((s["k_cache"], False), (s["v_cache"], True)):
        flat = cache.reshape(cache.shape[0], hkv, -1)
        byte, shift = (a.reshape(block, d) for a in code_places(block, d, values, keep.device))
        codes = flat[fb[:, None], head[:, None], byte[fo]] >> shift[fo].to(torch.uint8) & 15
        for half in (0, 4):
            here = shift[0] == half
            where = (tb[:, None], head[:, None], byte[to][:, here])
            flat[where] = flat[where] & (0xf0 if half == 0 else 0x0f) | codes[:, here] << half
        scales = block * d // 2 + torch.arange(d // 16, device=keep.device)
        flat[tb[:, None], head[:, None], scales + to[:, None] * (d // 16)] = flat[fb[:, None], head[:, None], scales + fo[:, None] * (d // 16)]
    for x in (s["weights"], s["positions"]):
        x[tb, head, to] = x[fb, head, fo]
    return _read(s["k_cache"], s["slots"], False), _read(s["v_cache"], s["slots"], True), s["weights"], s["positions"]


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    hkv = case["hkv"]
    row = case.get("d", 0) * 9 // 16                          # bytes of a token's keys, or values, of one head
    if case["kind"] == "rows":
        wide = case["d"] * 2
        return dict(bytes=2 * hkv * (case["new"] * (wide + row) + case["context"] * (wide + row)) + 8 * (case["new"] + case["context"]),
                    flops=2 * hkv * case["d"] * (8 * case["new"] + 2 * case["context"]))
    total = sum(lengths(case))
    if case["kind"] == "decode":
        t = case["batch"] * case["rows"]
        weights = {"plain": 0, "set": 4, "add": 8}[case["mode"]]
        return dict(bytes=total * hkv * (2 * row + weights) + t * case["hq"] * case["d"] * 4 + 4 * (total // case["block"] + case["batch"]),
                    flops=4 * total * case["rows"] * case["hq"] * case["d"])
    kept = sum(min(n, case["budget"]) for n in lengths(case))
    if case["kind"] == "keep":
        return dict(bytes=total * hkv * 8 + case["batch"] * hkv * case["budget"] * 4, flops=total * hkv * 4)
    moved = sum(max(0.0, case["budget"] * (1 - case["budget"] / n)) for n in lengths(case) if n)
    return dict(bytes=hkv * (moved * 2 * (2 * row + 8) + 4 * case["batch"] * case["budget"] + kept * 2 * (row + case["d"] * 2)), flops=kept * hkv * case["d"] * 4)


# ----------------------------------------------------------------------------- the definition in 64 bits
def _exact_rows(cache, values):
    """All rows of a cache [blocks, hkv, block, 9 d / 16] in 64 bits [blocks, hkv, block, d], by the shape of the layout."""
    blocks, hkv, block, row = cache.shape
    d = row * 16 // 9
    per, flat = min(d // 64, 2), cache.reshape(blocks, hkv, -1)
    codes = flat[..., :block * d // 2]
    codes = torch.stack([codes & 15, codes >> 4], -1)                                         # columns j, j + 1 of a word's byte
    if not values:
        codes = codes.reshape(blocks, hkv, -1, block, 4, per, 2, 8).permute(0, 1, 3, 2, 5, 4, 6, 7)
    else:
        codes = codes.reshape(blocks, hkv, -1, block // 2, 8, 2, per, 8).clone()
        for pair in range(block // 2):
            order = [r ^ (pair % 4 * 2) if per == 2 else r ^ (pair // 2 % 2 * 4) for r in range(8)]
            codes[:, :, :, pair] = codes[:, :, :, pair, order].clone()
        codes = codes.permute(0, 1, 3, 5, 2, 6, 4, 7)
    scales = flat[..., block * d // 2:].contiguous().view(torch.bfloat16).reshape(blocks, hkv, block, d // 64, 1, 2).double()
    return (codes.reshape(blocks, hkv, block, d // 64, 64).double() * scales[..., 0] + scales[..., 1]).reshape(blocks, hkv, block, d)


def _exact_stored(x):
    """What rows x [n, hkv, d] are worth once they have been stored, in 64 bits."""
    v = x.double().reshape(*x.shape[:-1], -1, 64)
    lo, hi = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
    step = (hi - lo) / 15
    unit = torch.exp2(torch.floor(torch.log2(step.clamp(min=1e-30))) - 7)                    # spacing of bf16 at the step
    step = torch.ceil(step / unit) * unit
    code = torch.where(step > 0, torch.round((v - lo) / step.clamp(min=1e-300)).clamp(0, 15), torch.zeros_like(v))
    return (code * step + lo).reshape(x.shape)


def exact(case, seed):
    if case["kind"] == "keep":
        return None
    s = prepare(case, seed)
    if case["kind"] == "rows":
        got = []
        for cache, x, values in ((s["k_cache"], s["k"], False), (s["v_cache"], s["v"], True)):
            rows = _exact_rows(cache, values).transpose(1, 2).flatten(0, 1)[s["slots"]]
            rows[case["context"] - case["new"]:] = _exact_stored(x)
            got.append(rows)
        return tuple(got)
    lens, block, hkv = lengths(case), case["block"], case["hkv"]
    if case["kind"] == "move":
        got = [[], []]
        w = s["weights"].double()
        for i, n in enumerate(lens):
            n = min(n, case["budget"])
            frm = s["keep"][i, :, :n].long()                                                  # [hkv, n]
            for out, cache, values in ((got[0], s["k_cache"], False), (got[1], s["v_cache"], True)):
                rows = _exact_rows(cache[s["table"][i].long()], values).transpose(0, 1).flatten(1, 2)     # [hkv, tokens, d]
                out.append(rows.gather(1, frm[..., None].expand(-1, -1, case["d"])).transpose(0, 1))
            mine = s["weights"][s["table"][i].long()].double().transpose(0, 1).flatten(1, 2)
            mine[:, :n] = mine.clone().gather(1, frm)
            w[s["table"][i].long()] = mine.unflatten(1, (-1, block)).transpose(0, 1)
        return torch.cat(got[0]), torch.cat(got[1]), w, None
    rows, hq, d = case["rows"], case["hq"], case["d"]
    rep, out = hq // hkv, torch.zeros(case["batch"], rows, hkv, hq // hkv, d, dtype=torch.float64, device=s["q"].device)
    w = s["weights"].double() if case["mode"] != "plain" else None
    for i, n in enumerate(lens):
        pages = s["table"][i, :-(-n // block)].long()
        for h in range(hkv if n else 0):
            k = _exact_rows(s["k_cache"][pages, h:h + 1], False).flatten(0, 2)[:n]
            v = _exact_rows(s["v_cache"][pages, h:h + 1], True).flatten(0, 2)[:n]
            sums = torch.zeros(n, dtype=torch.float64, device=k.device)
            for r in range(rows):
                m = n - rows + 1 + r
                if m <= 0:
                    continue
                q = s["q"][i * rows + r, h * rep:(h + 1) * rep].double()
                p = torch.softmax(q @ k[:m].T * d ** -0.5, -1)
                out[i, r, h] = p @ v[:m]
                sums[:m] += p.sum(0)
            if w is not None:
                at = torch.arange(n, device=k.device)
                old = w[pages[at // block], h, at % block]
                w[pages[at // block], h, at % block] = sums if case["mode"] == "set" else old + sums
    out = out.reshape(case["batch"] * rows, hq, d)
    return out if w is None else (out, w)
