"""The 4-bit paged key/value cache: rows written and read back, decode attention over it, and eviction by attention weight
(``csrc/kernels/kv4_cache.cu``, ``csrc/kernels/kv4_decode.cu``), with fp32 PyTorch references.

A cache (one for keys, one for values) is uint8 [blocks, Hkv, block_size, 9 d / 16]; ``kv4_cache`` makes a pair.  64 columns of a
token's row share a bf16 step and a bf16 lowest value and stand for ``code * step + lowest``, so a row takes 4.5 bits an element.
Inside the piece of a block and head the bytes lie as the kernels want them (``csrc/include/kv4.cuh``); ``kv4_read`` gives the
values.  Whole blocks can be copied between caches like those of any paged cache.

A request's tokens lie in the *places* 0, 1, ... of its block table.  Eviction (``kv4_keep``, ``kv4_move``) keeps ``budget`` tokens of
every head, its own choice for each, in the places below the budget; ``positions`` says which token of the sequence a place holds,
``weights`` how much attention it has had.  Keys carry their rotation with them, so attention does not ask for the order.

Calls write to no memory but their outputs and what the allocator gives them for the call: they may run on several streams, and
captured, as their arguments allow.  Block ids and slots outside the cache are reported by ``ops._native.check_status``: rows there
are neither written nor read, and the attention of a request with such a block is not to be used.  The same goes for requests longer than
their block table and for sources of a move below the budget.  On the CPU they are an IndexError, and nothing is changed."""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _native as nat

GROUP = 64
DIMS = (64, 128, 256)


def kv4_cache(num_blocks, block_size, hkv, d, device=None):
    """(keys, values) of ``num_blocks`` blocks, all zero."""
    assert d in DIMS and block_size % 16 == 0, f"head size {DIMS} and blocks of a multiple of 16 tokens: {d}, {block_size}"
    return tuple(torch.zeros(num_blocks, hkv, block_size, d * 9 // 16, dtype=torch.uint8, device=device) for _ in range(2))


# ----------------------------------------------------------------------------- layout and references
def _code_places(block, d, values, device=None):
    """(byte, shift) of the code of every [token, column] in the piece of one block and head."""
    t = torch.arange(block, device=device)[:, None]
    col = torch.arange(d, device=device)[None, :]
    per = min(d // GROUP, 2)
    g, i, j = col // GROUP, col % GROUP // 8, col % 8
    if values:
        pair = t // 2
        chunk = i ^ (pair % 4 * 2) if per == 2 else i ^ (pair // 2 % 2 * 4)
        byte = (g // per * block + pair * 2) * 32 * per + chunk * 8 * per + t % 2 * 4 * per + g % per * 4 + j // 2
    else:
        byte = (g // per * block + t) * 32 * per + (i // 2 * 2 * per + g % per * 2 + i % 2) * 4 + j // 2
    return byte, (j % 2 * 4).expand(block, d)


def kv4_quantise_ref(x):
    """x [..., d] -> codes uint8 [..., d], (step, lowest) bf16 [..., d / 64]."""
    v = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = v.amin(-1), v.amax(-1)
    step = (((hi - lo) / torch.full_like(hi, 15.0)).contiguous().view(torch.int32) + 0xffff & -0x10000).view(torch.float32)
    step = torch.where(torch.isfinite(hi - lo), step, torch.full_like(step, float("nan")))
    code = torch.round((v - lo[..., None]) / step[..., None]).clamp(0, 15)
    code = torch.where(step[..., None] > 0, code, torch.zeros_like(code))
    return code.to(torch.uint8).flatten(-2), step.bfloat16(), lo.bfloat16()


def _inside(what, index, n):
    """On the CPU a call stops at what a GPU skips and reports."""
    if index.numel() and (int(index.min()) < 0 or int(index.max()) >= n):
        raise IndexError(f"{what} outside 0 .. {n - 1}: {int(index.min())} .. {int(index.max())}")


def _fits(block_table, b, n, block):
    if n > block_table.shape[1] * block:
        raise IndexError(f"request {b} of {n} tokens, and a block table for {block_table.shape[1] * block}")


def _request_places(block_table, b, n, block, blocks):
    """(block, place in it) of the first n places of request b"""
    _fits(block_table, b, n, block)
    t = torch.arange(n, device=block_table.device)
    blk = block_table[b].long()[t // block]
    _inside(f"blocks of request {b}", blk, blocks)
    return blk, t % block


def _pieces(cache):
    blocks, hkv, block, row = cache.shape
    return cache.view(blocks, hkv, block * row), block, row * 16 // 9


def _write_ref(x, slots, cache, values):
    flat, block, d = _pieces(cache)
    byte, shift = _code_places(block, d, values)
    head = torch.arange(cache.shape[1])[:, None]
    codes, step, lo = kv4_quantise_ref(x)
    scales = torch.stack([step, lo], -1).flatten(2).contiguous().view(torch.uint8)
    for i, slot in enumerate(slots.tolist()):
        if slot < 0:
            continue
        at, t = flat[slot // block], slot % block
        for half in (0, 4):
            here = shift[t] == half
            b = byte[t][here]
            at[head, b] = at[head, b] & (0xf0 if half == 0 else 0x0f) | codes[i][:, here] << half
        p = block * d // 2 + t * (d // 16)
        at[:, p:p + d // 16] = scales[i]


def _values_ref(cache, blk, t, values, head=None):
    """fp32 values of the rows (blk, t): [..., Hkv, d], or [..., d] of the heads ``head``."""
    flat, block, d = _pieces(cache)
    byte, shift = _code_places(block, d, values, cache.device)
    byte, shift = byte[t], shift[t].to(torch.uint8)
    sc = block * d // 2 + t[..., None] * (d // 16) + torch.arange(d // 16, device=cache.device)
    if head is None:
        head = torch.arange(cache.shape[1], device=cache.device)
        blk, byte, shift, sc = blk[..., None], byte[..., None, :], shift[..., None, :], sc[..., None, :]
    blk, head = blk[..., None], head[..., None]
    codes = (flat[blk, head, byte] >> shift & 15).float().unflatten(-1, (-1, GROUP))
    scales = flat[blk, head, sc].contiguous().view(torch.bfloat16).float().unflatten(-1, (-1, 2))
    # 15 steps may be beyond fp32 where 15 steps and the lowest value are not
    return (codes.double() * scales[..., :1] + scales[..., 1:]).float().flatten(-2)


def kv4_decode_ref(q, k_cache, v_cache, block_table, seq_lens, scale, weights=None, decay=1.0):
    T, hq, d = q.shape
    hkv, block = k_cache.shape[1], k_cache.shape[2]
    B = seq_lens.shape[0]
    rows, rep = T // B if B else 0, hq // hkv
    out = torch.zeros(T, hq, d, dtype=torch.float32, device=q.device)
    lens = [max(n, 0) for n in seq_lens.tolist()]
    places = [_request_places(block_table, b, n, block, k_cache.shape[0]) for b, n in enumerate(lens)]
    for b, (n, (blk, place)) in enumerate(zip(lens, places)):
        if n == 0:
            continue
        t = torch.arange(n, device=q.device)
        k, v = (_values_ref(c, blk, place, x).transpose(0, 1).repeat_interleave(rep, 0) for c, x in ((k_cache, False), (v_cache, True)))
        s = torch.einsum("rhd,hnd->rhn", q[b * rows:(b + 1) * rows].float(), k) * scale
        sees = n - rows + 1 + torch.arange(rows, device=q.device)
        s = s.masked_fill(t >= sees[:, None, None], float("-inf"))
        p = torch.where(t < sees[:, None, None], torch.softmax(s, -1), torch.zeros_like(s))      # a NaN is of what its row sees
        for i in range(rows):
            m = max(0, int(sees[i]))
            out[b * rows + i] = torch.einsum("hn,hnd->hd", p[i, :, :m], v[:, :m])
        if weights is not None:
            step = p.sum(0).view(hkv, rep, n).sum(1).transpose(0, 1)                  # [n, Hkv]
            weights[blk, :, place] = step if decay == 0 else weights[blk, :, place] * decay + step
    return out.to(q.dtype)


def kv4_keep_ref(weights, positions, block_table, seq_lens, seen, budget, keep_first=0, keep_last=0):
    hkv, block = weights.shape[1], weights.shape[2]
    B = seq_lens.shape[0]
    keep = torch.full((B, hkv, budget), -1, dtype=torch.int32)
    lens = seq_lens.clamp(0, budget).to(torch.int32)
    for b, n in enumerate(seq_lens.tolist()):
        _fits(block_table, b, n, block)
        if n > budget:                                        # else no block is looked at
            blk, at = _request_places(block_table, b, n, block, weights.shape[0])
        for h in range(hkv):
            place = list(range(min(n, budget)))
            if n > budget:
                w, pos = weights[blk, h, at].tolist(), positions[blk, h, at].tolist()
                rank = []
                for j in range(n):
                    safe = pos[j] < keep_first or pos[j] >= int(seen[b]) - keep_last
                    rank.append((2, 0.0) if safe else (1, 0.0) if w[j] != w[j] else (0, w[j]))
                stay = set(sorted(range(n), key=lambda j: rank[j], reverse=True)[:budget])     # a stable sort: the lowest of equals
                far = iter(sorted(j for j in stay if j >= budget))
                place = [j if j in stay else next(far) for j in range(budget)]
            keep[b, h, :len(place)] = torch.tensor(place, dtype=torch.int32)
    return keep, lens


def _move_ref(k_cache, v_cache, block_table, keep, weights, positions):
    block = k_cache.shape[2]
    budget = keep.shape[2]
    b, h, j = ((keep >= 0) & (keep != torch.arange(budget))).nonzero(as_tuple=True)
    s = keep[b, h, j].long()
    _inside("places from the budget on that tokens come from", s - budget, block_table.shape[1] * block - budget)
    _inside("blocks of the tokens and of their places", block_table[torch.cat([b, b]), torch.cat([s, j]) // block], k_cache.shape[0])
    fb, ft, tb, tt = block_table[b, s // block].long(), s % block, block_table[b, j // block].long(), j % block
    for cache, values in ((k_cache, False), (v_cache, True)):
        flat, _, d = _pieces(cache)
        byte, shift = _code_places(block, d, values)
        codes = flat[fb[:, None], h[:, None], byte[ft]] >> shift[ft].to(torch.uint8) & 15
        for half in (0, 4):
            here = shift[0] == half
            at = (tb[:, None], h[:, None], byte[tt][:, here])
            flat[at] = flat[at] & (0xf0 if half == 0 else 0x0f) | codes[:, here] << half
        sc = block * d // 2 + torch.arange(d // 16)
        flat[tb[:, None], h[:, None], sc + tt[:, None] * (d // 16)] = flat[fb[:, None], h[:, None], sc + ft[:, None] * (d // 16)]
    for x in (weights, positions):
        if x is not None:
            x[tb, h, tt] = x[fb, h, ft]


# ----------------------------------------------------------------------------- calls
# The argument blocks of the C calls: pointers and 64-bit numbers, then 32-bit ones
_ARGS = {
    "omni_kv4_write": struct.Struct("8Q4q6i"),
    "omni_kv4_read": struct.Struct("5Q2q4i"),
    "omni_kv4_keep": struct.Struct("8Q1q10i"),
    "omni_kv4_move": struct.Struct("6Q1q8i"),
    "omni_kv4_decode": struct.Struct("12Q2q13i2fi"),
}
_bound = {}


def _call(name, device, *args):
    """Launch on the current stream of the tensors' own device."""
    call = _bound.get(name)
    if call is None:
        lib = nat.lib()
        getattr(lib._cdll, name).argtypes = (ctypes.c_char_p, ctypes.c_void_p, ctypes.c_void_p)
        call = _bound[name] = (getattr(lib, name), _ARGS[name].pack)
    fn, pack = call
    index = device.index
    status = nat._status.get(index)
    status, stream = (nat.status_buffer(index) if status is None else status).data_ptr(), torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        rc = fn(pack(*args), status, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(pack(*args), status, stream)
    if rc:
        nat.check_rc(rc, name)


def _p(t):
    return 0 if t is None else t.data_ptr()


def _check_caches(k_cache, v_cache):
    """(blocks, Hkv, block, d, device) of a pair of caches."""
    shape, device = k_cache.shape, k_cache.device
    assert k_cache.dtype is torch.uint8 and v_cache.dtype is torch.uint8 and len(shape) == 4 and shape == v_cache.shape, "a pair of uint8 caches of one shape"
    assert k_cache.is_contiguous() and v_cache.is_contiguous() and device == v_cache.device, "contiguous caches on one device"
    blocks, hkv, block, row = shape
    d = row * 16 // 9
    assert d in DIMS and row * 16 == d * 9 and block > 0 and block % 16 == 0 and hkv > 0, \
        f"rows of 9 d / 16 bytes with d in {DIMS} and blocks of a multiple of 16 tokens: {row}, {block}"
    return blocks, hkv, block, d, device


def _check_rows(name, x, hkv, d, device):
    """(shape, stride) of rows; each is asked for once, since asking costs as much as a check."""
    shape, stride = x.shape, x.stride()
    assert x.dtype is torch.bfloat16 and x.device == device and len(shape) == 3 and stride[2] == 1 and shape[2] == d and (hkv is None or shape[1] == hkv), \
        f"{name}: bf16 [rows, {'heads' if hkv is None else hkv}, {d}] on {device}, columns without gaps"
    return shape, stride


def _check_numbers(name, x, n, device, dtype=torch.int32):
    """How many there are of one number for each of n requests or tokens (any number of them: n None)."""
    shape = x.shape
    assert x.dtype is dtype and x.device == device and len(shape) == 1 and x.is_contiguous() and (n is None or shape[0] == n), \
        f"{name}: contiguous {dtype} [{'n' if n is None else n}] on {device}"
    return shape[0]


def _check_per_place(name, x, shape, device, dtype=torch.float32):
    """``weights`` and ``positions``: a number for every place of the caches."""
    assert x.dtype is dtype and x.device == device and x.is_contiguous() and x.shape == shape, f"{name}: contiguous {dtype} {list(shape)} on {device}"


def _check_table(table, device, B, block):
    """(blocks of a request, row pitch)"""
    shape, stride = table.shape, table.stride()
    assert table.dtype is torch.int32 and table.device == device and len(shape) == 2 and shape[0] >= B and stride[1] == 1, \
        f"block_table: int32 on {device}, a row without gaps for each of the {B} requests"
    assert B < 1 << 16, f"block_table: at most 65,535 requests: {B}"
    assert shape[1] * block < 1 << 30, f"block_table: fewer than 2^30 places for a request: {shape[1]} blocks of {block}"
    return shape[1], stride[0]


def kv4_write(k, v, slots, k_cache, v_cache, weights=None, positions=None, token_positions=None):
    """Rows k, v [T, Hkv, d] (bf16; any row and head pitch) into the slots ``slots`` [T] int64 (block * block size + place in the
    block; negative: not stored).  The slots of a call differ.  ``weights`` / ``positions`` [blocks, Hkv, block], where given, are
    set to 0 and to ``token_positions`` [T] int64 in those slots."""
    blocks, hkv, block, d, device = _check_caches(k_cache, v_cache)
    (T, *_), (k_row, k_head, _) = _check_rows("k", k, hkv, d, device)
    (v_rows, *_), (v_row, v_head, _) = _check_rows("v", v, hkv, d, device)
    assert v_rows == T, "a row of v for every row of k"
    _check_numbers("slots", slots, T, device, torch.int64)
    assert (positions is None) == (token_positions is None), "positions and token_positions come together"
    if weights is not None:
        _check_per_place("weights", weights, (blocks, hkv, block), device)
    if positions is not None:
        _check_per_place("positions", positions, (blocks, hkv, block), device, torch.int32)
        _check_numbers("token_positions", token_positions, T, device, torch.int64)
    if not k.is_cuda:
        _inside("slots", slots.clamp_min(0), blocks * block)
        _write_ref(k, slots, k_cache, False)
        _write_ref(v, slots, v_cache, True)
        ok = slots >= 0
        blk, t = slots[ok] // block, slots[ok] % block
        if weights is not None:
            weights[blk, :, t] = 0.0
        if positions is not None:
            positions[blk, :, t] = token_positions[ok].to(torch.int32)[:, None]
        return
    if T == 0:
        return
    _call("omni_kv4_write", device, k.data_ptr(), v.data_ptr(), slots.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _p(weights), _p(positions), _p(token_positions),
          k_row, v_row, T, blocks, k_head, v_head, block, hkv, d, 0)


def kv4_read(k_cache, v_cache, slots):
    """(k, v) [T, Hkv, d] bf16 of the slots ``slots`` [T] int64; zeros for negative ones.  A slot may be named more than once."""
    blocks, hkv, block, d, device = _check_caches(k_cache, v_cache)
    T = _check_numbers("slots", slots, None, device, torch.int64)
    if not k_cache.is_cuda:
        s = slots.clamp_min(0)
        _inside("slots", s, blocks * block)
        ok = (slots >= 0)[:, None, None]
        return tuple(torch.where(ok, _values_ref(c, s // block, s % block, x), torch.zeros(())).bfloat16() for c, x in ((k_cache, False), (v_cache, True)))
    k = torch.empty((T, hkv, d), dtype=torch.bfloat16, device=device)
    v = torch.empty((T, hkv, d), dtype=torch.bfloat16, device=device)
    if T:
        _call("omni_kv4_read", device, k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), T, blocks, block, hkv, d, 0)
    return k, v


# Bytes up to which the scores of a call are kept for its weights (a number for each row that a tile of them has, key/value head and place of
# the block table); beyond they are made from the keys once more.  Kept, 32 requests of 4099 tokens and 8 rows a key/value head take
# 44 us and not 56, 64 of 16,384 197 and not 259, two of 131,072 with 128 rows 558 and not 578: it is the memory that sets the bound.
KEPT_SCORES = 256 << 20


def _blocks(items, tiles, resident):
    """(blocks, fewest tiles of one) for ``items`` passes over up to ``tiles`` tiles each, with ``resident`` blocks on each of the 148
    SMs; 0 tiles: a block takes a pass, whole."""
    if tiles <= 12:
        return 0, 0
    return min(148 * resident, -(-items * tiles // 4)), 4


def kv4_decode(q, k_cache, v_cache, block_table, seq_lens, scale, max_seq_len=None, weights=None, decay=1.0):
    """Attention of the last tokens of every request over its cached ones: q [B n, Hq, d] bf16 (any row and head pitch), the ``n``
    rows of a request one after the other; row i sees the first ``seq_lens[b] - n + 1 + i`` of the request's places (none: zeros).
    ``block_table`` [B, blocks of a request] int32 (B at most 65,535), ``seq_lens`` [B] int32, with the rows' own tokens.  Returns [B n, Hq, d].
    On a GPU the largest number of a query row is brought to 2^13 .. 2^14: keys beyond 2^98 may leave the range of the fp32 sums, and numbers below
    2^-26 of the row's largest lose bits.

    ``weights`` [blocks, Hkv, block] fp32: of every place below seq_lens[b] becomes decay * weights + the softmax weights that the
    rows and the query heads of its key/value head give it (decay 0: whatever was there is dropped).  Requests that share a block
    would write the same numbers: give ``weights`` only where blocks belong to one request.  At most 256 rows times query
    heads of a key/value head then.  Up to 256 MiB go to scores meanwhile: 32 bytes (8 rows) to 1 KiB (256) for each place of the table
    and key/value head, so a table no wider than needed saves memory; ``ops.kv4.KEPT_SCORES`` is how many bytes they may take, and with fewer they
    are made twice.  A captured graph keeps them.  ``max_seq_len`` (a bound of
    ``seq_lens``) shapes the launch; without it the width of the block table does."""
    blocks, hkv, block, d, device = _check_caches(k_cache, v_cache)
    (T, hq, _), (q_row, q_head, _) = _check_rows("q", q, None, d, device)
    B = _check_numbers("seq_lens", seq_lens, None, device)
    assert hq > 0 and hq % hkv == 0, f"{hq} query heads do not divide over {hkv} key/value heads"
    assert T == 0 if B == 0 else T > 0 and T % B == 0, f"{T} rows are not the same number for each of {B} requests"
    width, table_ld = _check_table(block_table, device, B, block)
    if weights is not None:
        _check_per_place("weights", weights, (blocks, hkv, block), device)
        assert T == 0 or T // B * (hq // hkv) <= 256, f"weights of at most 256 query rows a key/value head at once: {T // B * (hq // hkv)}"
    if not q.is_cuda:
        return kv4_decode_ref(q, k_cache, v_cache, block_table, seq_lens, scale, weights, decay)
    out = torch.empty((T, hq, d), dtype=torch.bfloat16, device=device)
    if T:
        total = T // B * (hq // hkv)
        longest = width * block if max_seq_len is None else max(0, min(max_seq_len, width * block))
        tile = 16 if d <= 128 and total > 8 else 8
        items = B * hkv * -(-total // tile)
        blocks_at_once, min_tiles = _blocks(items, -(-longest // (32 if d == 256 else 64)), 3 if tile * d <= 1024 else 2)
        lse = torch.empty(T * hq, dtype=torch.float32, device=device) if weights is not None else None
        places = -(-width * block // 64) * 64
        scores = None
        if weights is not None and items * tile * places * 4 <= KEPT_SCORES:
            scores = torch.empty(items * tile * places, dtype=torch.float32, device=device)
        o_part = lse_part = shared = 0
        if min_tiles:                                        # partial results, their sums, where the parts of an item are
            n = blocks_at_once * 2 * tile
            scratch = torch.empty(n * (d + 1) + 2 * items, dtype=torch.float32, device=device)
            o_part = scratch.data_ptr()
            lse_part, shared = o_part + 4 * n * d, o_part + 4 * n * (d + 1)
        _call("omni_kv4_decode", device, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), out.data_ptr(),
              o_part, lse_part, _p(lse), _p(weights), shared, _p(scores), q_row, blocks, q_head, block, hkv, d, table_ld, width, B, T // B, hq, longest, tile,
              blocks_at_once, min_tiles, scale, decay, 0)
        nat.add_launches((min_tiles > 0) + (weights is not None))          # the kernels that join parts and make weights
    return out


def kv4_keep(weights, positions, block_table, seq_lens, seen, budget, keep_first=0, keep_last=0, max_seq_len=None):
    """Which tokens stay when every head of a request may keep ``budget`` of its first ``seq_lens[b]`` places: those of positions
    below ``keep_first`` and from ``seen[b] - keep_last`` on (``seen`` [B] int32: tokens that the request has had), then the
    heaviest by ``weights``, among equals the lowest place.  A NaN counts as heavier than any number.

    Returns (keep [B, Hkv, budget] int32, lens [B] int32 = the smaller of seq_lens and budget).  keep[b, h, j] is the place whose token
    is to be in place j: j itself where that stays, else one of the kept places from the budget on, in ascending order over the
    places that become free; -1 from lens[b] on.  Nothing is moved: see ``kv4_move``.  ``max_seq_len``
    as in ``kv4_decode``."""
    assert weights.dim() == 3, "weights: [blocks, Hkv, block]"
    device, shape = weights.device, weights.shape
    blocks, hkv, block = shape
    _check_per_place("weights", weights, shape, device)
    _check_per_place("positions", positions, shape, device, torch.int32)
    B = _check_numbers("seq_lens", seq_lens, None, device)
    _check_numbers("seen", seen, B, device)
    width, table_ld = _check_table(block_table, device, B, block)
    assert budget >= 1 and keep_first >= 0 and keep_last >= 0 and keep_first + keep_last <= budget, \
        f"a budget of {budget} tokens holds at least the {keep_first} first and {keep_last} last ones"
    if not weights.is_cuda:
        return kv4_keep_ref(weights, positions, block_table, seq_lens, seen, budget, keep_first, keep_last)
    keep = torch.empty((B, hkv, budget), dtype=torch.int32, device=device)
    lens = torch.empty(B, dtype=torch.int32, device=device)
    if B:
        scratch = torch.empty((B, hkv, budget), dtype=torch.int32, device=device) if width * block > 4096 else None
        longest = width * block if max_seq_len is None else max(0, min(max_seq_len, width * block))
        _call("omni_kv4_keep", device, weights.data_ptr(), positions.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), seen.data_ptr(),
              keep.data_ptr(), lens.data_ptr(), _p(scratch), blocks,
              block, hkv, table_ld, width, B, budget, keep_first, keep_last, longest, 0)
    return keep, lens


def kv4_move(k_cache, v_cache, block_table, keep, weights=None, positions=None):
    """Brings the tokens that ``keep`` [B, Hkv, budget] names (see ``kv4_keep``) to their places, in place, with their weights and
    positions where given.  What other places hold is left.  Requests that share a block would lose tokens of one another: copy
    such blocks first."""
    blocks, hkv, block, d, device = _check_caches(k_cache, v_cache)
    assert keep.dim() == 3 and keep.shape[1] == hkv and keep.is_contiguous() and keep.dtype is torch.int32 and keep.device == device, \
        f"keep: contiguous int32 [B, {hkv}, budget] on {device}"
    B, _, budget = keep.shape
    width, table_ld = _check_table(block_table, device, B, block)
    if weights is not None:
        _check_per_place("weights", weights, (blocks, hkv, block), device)
    if positions is not None:
        _check_per_place("positions", positions, (blocks, hkv, block), device, torch.int32)
    if not k_cache.is_cuda:
        _move_ref(k_cache, v_cache, block_table, keep, weights, positions)
    elif B and budget:
        _call("omni_kv4_move", device, k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), keep.data_ptr(), _p(weights), _p(positions), blocks, block, hkv, d,
              table_ld, width, B, budget, 0)
