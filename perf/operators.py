"""The 4-bit key/value cache operators: what is measured, and their plain forms.

Four operators over one paged cache (see llm_fa_b200/kv4.py for the calls):

  append   new keys and values are quantised to 4 bits and written behind what a sequence holds
  attend   a few new queries of each sequence attend to its cache; with tracking, the attention
           weight that each cached token received is stored beside it
  select   which tokens of an over-full cache go, by accumulated weight, and which of the rest
           fill their slots
  move     the selected tokens are moved

Definitions. A token's head of 128 channels is cut into 128/group groups. With lo = min(0, x),
hi = max(0, x) over a group: scale = bf16((hi - lo) / 15), zero = round(-lo / scale) in 0..15,
code = clamp(round(x / scale) + zero, 0, 15), halves to even; the cache holds scale * (code -
zero). Attention is softmax(q k^T * scale) v over the slots that a query may see: all of the
sequence's, less, for the i-th of its n new queries, the last n - 1 - i. A query that sees no slot
gives zeros. Eviction keeps `keep` slots: of the others, those of least weight go, lowest slot
first among equals, the `recent` latest positions last of all; freed slots below `keep` take, in
ascending order, the surviving tokens at or above it.

A page holds, for each key/value head, page_size/16 blocks of 16 tokens, a block being
  16 x 64 bytes of key codes, 16 x 128/group (scale, zero) pairs of bf16, then the same of values.
A key's code words (32 bits: 8 channels, low bits first) are stored as the transpose of 4 x 4, a
value's half-words (4 channels) as that of 8 x 4.
"""
import math

import numpy as np
import torch

own = False

D = 128
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one conversation, short: what a chat costs per layer and token; latency is all
        dict(name="attend_1x1000", op="attend", batch=1, heads_q=32, heads_kv=8, tokens=1,
             longest=1000, spread=0.0, page=64, group=64, dtype="bf16", track=False, lse=False),
        # a full serving batch of ragged lengths
        dict(name="attend_32x8192_ragged", op="attend", batch=32, heads_q=64, heads_kv=8, tokens=1,
             longest=8192, spread=0.6, page=64, group=64, dtype="bf16", track=False, lse=False),
        # one very long context: the cache has to be read by the whole GPU
        dict(name="attend_1x131071", op="attend", batch=1, heads_q=32, heads_kv=8, tokens=1,
             longest=131071, spread=0.0, page=128, group=32, dtype="bf16", track=False, lse=False),
        # five drafted tokens verified at once, some drafts shorter; merged elsewhere by its lse
        dict(name="attend_8x16384_drafts", op="attend", batch=8, heads_q=32, heads_kv=8, tokens=5,
             longest=16384, spread=0.3, page=16, group=128, dtype="fp16", track=False, lse=True),
        # a step whose weights feed the eviction; as many key heads as query heads
        dict(name="attend_16x4097_tracked", op="attend", batch=16, heads_q=32, heads_kv=32,
             tokens=1, longest=4097, spread=0.2, page=64, group=64, dtype="bf16", track=True,
             lse=False),
        # the token of a decoding step, for a batch
        dict(name="append_64x1", op="append", batch=64, heads_kv=8, tokens=1, longest=2000,
             spread=0.9, page=64, group=64, dtype="bf16"),
        # a long prompt
        dict(name="append_1x8192", op="append", batch=1, heads_kv=32, tokens=8192, longest=0,
             spread=0.0, page=64, group=32, dtype="bf16"),
        # prompts of several lengths behind prefixes, odd everywhere
        dict(name="append_7x1023_ragged", op="append", batch=7, heads_kv=5, tokens=1023,
             longest=333, spread=0.9, page=16, group=128, dtype="fp16"),
        # half of a batch's cache goes
        dict(name="select_8x8192", op="select", batch=8, heads_kv=8, longest=8192, spread=0.2,
             keep=4096, recent=256, page=64, group=64),
        # half of one very long cache goes
        dict(name="select_1x131072", op="select", batch=1, heads_kv=8, longest=131072, spread=0.0,
             keep=65536, recent=1024, page=128, group=64),
        # the moves of the batch above
        dict(name="move_8x8192", op="move", batch=8, heads_kv=8, longest=8192, spread=0.2,
             keep=4096, recent=256, page=64, group=64),
        # a cache held at its budget: one token in, one token out
        dict(name="move_64x2049_step", op="move", batch=64, heads_kv=8, longest=2049, spread=0.0,
             keep=2048, recent=64, page=64, group=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "select", "move"])
    case = dict(op=op, batch=_log(rng, 1, 64), heads_kv=rng.choice([1, 2, 4, 5, 8, 16, 32]),
                spread=rng.choice([0.0, 0.3, 0.9]), page=rng.choice([16, 32, 64, 128, 256]),
                group=rng.choice([32, 64, 128]))
    budget = 1 << 20  # token-heads: what the largest listed cases hold
    room = max(1, budget // (case["batch"] * case["heads_kv"]))
    if op == "attend":
        case.update(heads_q=case["heads_kv"] * rng.choice([1, 2, 3, 4, 7, 8, 16]),
                    tokens=rng.choice([1, 1, 1, 2, 4, 7]))
        pairs = 14_000_000 // (case["batch"] * case["heads_q"] * case["tokens"])
        case.update(longest=_log(rng, 1, max(1, min(room, pairs, 131072))),
                    dtype=rng.choice(["bf16", "fp16"]), track=rng.choice([False, False, True]),
                    lse=rng.choice([False, True]))
    elif op == "append":
        room = max(1, room // 4)
        tokens = rng.choice([1, _log(rng, 1, min(room, 8192))])
        case.update(tokens=tokens, longest=rng.choice([0, _log(rng, 1, min(room, 4000))]),
                    dtype=rng.choice(["bf16", "fp16"]))
    else:
        longest = _log(rng, 2, max(2, min(room, 131072)))
        keep = max(1, min(longest, int(longest * rng.choice([0.25, 0.5, 0.9, 1.0])) + rng.randint(-1, 0)))
        case.update(longest=longest, keep=keep, recent=rng.randint(0, keep))
    return case


def _lengths(case):
    """Tokens that each sequence holds (attend, select, move: with the new ones; append: before
    them): from `longest` down to (1 - spread) of it, scattered over the batch."""
    return [max(min(1, case["longest"]),
                case["longest"] - int(case["longest"] * case["spread"] * ((b * 0.6180339887) % 1.0)))
            for b in range(case["batch"])]


def _counts(case):
    """New tokens of each sequence; None where all have `tokens` of them."""
    if case["tokens"] == 1 or case["spread"] == 0.0:
        return None
    if case["op"] == "append":
        return [max(1, case["tokens"] - int(case["tokens"] * case["spread"] * ((b * 0.7548776662) % 1.0)))
                for b in range(case["batch"])]
    return [max(1, case["tokens"] - b % 3) for b in range(case["batch"])]


def _block_bytes(group):
    return 16 * 2 * (D // 2 + (D // group) * 4)


def work(case):
    B, H = case["batch"], case["heads_kv"]
    token = _block_bytes(case["group"]) // 16  # bytes of one token's key and value of one head
    lens = _lengths(case)
    if case["op"] == "attend":
        counts = _counts(case) or [case["tokens"]] * B
        rows = sum(counts) * case["heads_q"]
        held = sum(lens) * H
        nbytes = held * token + 2 * rows * D * 2 + sum(-(-n // case["page"]) for n in lens) * 4
        nbytes += rows * 4 if case["lse"] else 0
        nbytes += held * 4 if case["track"] else 0
        pairs = sum(n * c - c * (c - 1) // 2 for n, c in zip(lens, counts)) * case["heads_q"]
        return {"bytes": nbytes, "flops": 4 * D * pairs}
    if case["op"] == "append":
        new = sum(_counts(case) or [case["tokens"]] * B) * H
        # keys and values in, codes out, position and weight; then back, as the outputs show them
        back = B * case["tokens"] * H * 2 * D * 2
        return {"bytes": new * (2 * D * 2 + token + 8 + token) + back, "flops": new * 2 * D * 6}
    keep = case["keep"]
    over = [n for n in lens if n > keep]
    if case["op"] == "select":
        return {"bytes": H * (sum(n * 8 for n in over) + B * keep * 4), "flops": H * sum(over) * 4}
    moved = sum(keep * (n - keep) / n for n in over) * H  # as many as go below `keep`, about
    return {"bytes": int(moved * 2 * (token + 8) + B * H * keep * 4), "flops": int(moved)}


# ---------------------------------------------------------------- the cache's format, plainly
def _quantise(x, group):
    """fp32 [..., 128] -> codes uint8 [..., 128], scale and zero fp32 [..., 128/group] (both bf16
    values). Every step here is exact or the definition's own rounding, so 32 bits are enough:
    a quotient of bf16 or fp16 by a bf16 scale is never close to a half without being one."""
    y = x.unflatten(-1, (-1, group))
    lo, hi = y.amin(-1).clamp(max=0.0), y.amax(-1).clamp(min=0.0)
    # divided by a tensor: torch turns a division by a number into a product with its reciprocal,
    # which can miss the middle between two bf16 values by a bit
    scale = ((hi - lo) / torch.full_like(hi, 15.0)).to(torch.bfloat16).float()
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    zero = torch.round(-lo / safe).clamp(0, 15)
    codes = (torch.round(y / safe[..., None]) + zero[..., None]).clamp(0, 15)
    return codes.flatten(-2).to(torch.uint8), scale, zero


def _values(codes, scale, zero, group):
    y = codes.float().unflatten(-1, (-1, group))
    return (scale[..., None] * (y - zero[..., None])).flatten(-2)


def _rows(codes, value):
    """codes [..., 128] -> the 64 stored bytes of a row."""
    nat = codes[..., 0::2] | (codes[..., 1::2] << 4)
    if value:  # 32 half-words, natural order k * 8 + g, stored g * 4 + k
        return nat.unflatten(-1, (4, 8, 2)).transpose(-3, -2).flatten(-3)
    return nat.unflatten(-1, (4, 4, 4)).transpose(-3, -2).flatten(-3)


def _codes(rows, value):
    if value:
        nat = rows.unflatten(-1, (8, 4, 2)).transpose(-3, -2).flatten(-3)
    else:
        nat = rows.unflatten(-1, (4, 4, 4)).transpose(-3, -2).flatten(-3)
    return torch.stack((nat & 15, nat >> 4), -1).flatten(-2)


def _pairs(scale, zero):
    """(scale, zero) as stored: bytes [..., 128/group * 4]."""
    return torch.stack((scale, zero), -1).to(torch.bfloat16).contiguous().view(torch.uint8).flatten(-2)


def _parts(pages, group):
    """Views of the pool's parts by token: [pages, heads, page_size/16, 16, bytes]."""
    blocks = pages.unflatten(-1, (-1, _block_bytes(group)))
    m = (D // group) * 4
    out, at = [], 0
    for width in (64, m, 64, m):
        out.append(blocks[..., at:at + 16 * width].unflatten(-1, (16, width)))
        at += 16 * width
    return out


def _slots(table, page):
    """Page and slot in it for every slot of a sequence: [batch, capacity] each. Unused entries
    of the table stand for page 0 here; nothing that is read through them is used."""
    i = torch.arange(table.shape[1] * page, device=table.device)
    return table.clamp(min=0).long()[:, i // page], (i % page).expand(table.shape[0], -1)


def _read(pages, group, p, s, value):
    """Values of slots s of pages p (any shape [*]) -> fp32 [*, heads, 128]."""
    parts = _parts(pages, group)
    rows, pair = parts[2 * value], parts[2 * value + 1]
    r = rows[p, :, s // 16, s % 16]
    m = pair[p, :, s // 16, s % 16].contiguous().view(torch.bfloat16).unflatten(-1, (-1, 2)).float()
    return _values(_codes(r, value), m[..., 0], m[..., 1], group)


# ---------------------------------------------------------------- inputs
def _randn(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


def _keys(gen, B, T, H, dtype):
    """Keys as a projection and a rotation leave them: a few channels much larger than the rest."""
    loud = 1.0 + 7.0 * (torch.rand(H, D, generator=gen, device=DEV) < 0.04).float()
    return (torch.randn(B, T, H, D, generator=gen, device=DEV) * loud).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
    B, H, page, group = case["batch"], case["heads_kv"], case["page"], case["group"]
    lens = _lengths(case)
    tokens = case.get("tokens", 0)
    counts = _counts(case) if tokens else None
    most = max(lens) + (tokens if case["op"] == "append" else 0)
    width = -(-most // page)
    pool = B * width + 3  # a pool has pages that belong to nobody
    order = torch.randperm(pool, generator=gen, device=DEV)[:B * width].reshape(B, width)
    held = torch.tensor([-(-(n + (tokens if case["op"] == "append" else 0)) // page) for n in lens],
                        device=DEV)
    used = torch.arange(width, device=DEV) < held[:, None]
    table = torch.where(used, order, -1).to(torch.int32)
    st = dict(case=case, table=table, lengths=torch.tensor(lens, dtype=torch.int32, device=DEV),
              counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV))
    pages = torch.zeros(pool, H, page // 16 * _block_bytes(group), dtype=torch.uint8, device=DEV)
    positions = torch.zeros(pool, H, page, dtype=torch.int32, device=DEV)
    weights = torch.zeros(pool, H, page, device=DEV)
    if case["op"] != "select":  # select reads weights and positions alone
        parts = _parts(pages, group)
        cap = width * page
        step = max(1, (1 << 25) // (cap * H * D))  # sequences at a time: bounded scratch
        p, s = _slots(table, page)
        for b in range(0, B, step):
            rows = torch.nonzero(used[b:b + step].repeat_interleave(page, 1))
            pb, sb = p[b:b + step][rows[:, 0], rows[:, 1]], s[b:b + step][rows[:, 0], rows[:, 1]]
            for value in (0, 1):
                n = min(step, B - b)
                x = (_randn(gen, n, cap, H, D) if value else _keys(gen, n, cap, H, torch.bfloat16))
                c, sc, z = _quantise(x[rows[:, 0], rows[:, 1]].float(), group)
                parts[2 * value][pb, :, sb // 16, sb % 16] = _rows(c, value)
                parts[2 * value + 1][pb, :, sb // 16, sb % 16] = _pairs(sc, z)
                del x, c
    if case["op"] in ("select", "move"):
        # weights as many steps of attention leave them: heavy-tailed, with tokens that never got
        # any; positions as earlier moves leave them: out of order
        p, s = _slots(table, page)
        cap = width * page
        w = torch.exp(2.5 * torch.randn(B, cap, H, generator=gen, device=DEV))
        w = torch.where(torch.rand(B, cap, H, generator=gen, device=DEV) < 0.03, 0.0, w)
        pos = torch.argsort(torch.rand(B, H, cap, generator=gen, device=DEV) * 0.5
                            + torch.arange(cap, device=DEV) / cap, -1).transpose(1, 2)
        seen = st["lengths"] + cap // 2
        pos = torch.where(pos < st["lengths"][:, None, None], pos, 0) + cap // 2
        keepers = used.repeat_interleave(page, 1)
        positions[p[keepers], :, s[keepers]] = pos[keepers].to(torch.int32)
        weights[p[keepers], :, s[keepers]] = w[keepers]
        st["seen"] = seen
    st.update(pages=pages, positions=positions, weights=weights)
    dtype = TYPES[case["dtype"]] if "dtype" in case else None
    if case["op"] == "attend":
        st["q"] = _randn(gen, B, tokens, case["heads_q"], D, dtype=dtype)
    if case["op"] == "append":
        st["k"], st["v"] = _keys(gen, B, tokens, H, dtype), _randn(gen, B, tokens, H, D, dtype=dtype)
    if case["op"] == "move":
        st["src"], _ = _select(st)
    if own:
        from llm_fa_b200 import KV4Cache
        st["cache"] = KV4Cache(pages, positions, weights, page_size=page, group=group)
    return st


# ---------------------------------------------------------------- plain forms
def _attend(st):
    case, q, H = st["case"], st["q"], st["case"]["heads_kv"]
    B, T, Hq, _ = q.shape
    G = Hq // H
    p, s = _slots(st["table"], case["page"])
    cap = p.shape[1]
    n = st["lengths"].long()
    c = st["counts"].long() if st["counts"] is not None else torch.full_like(n, T)
    out = torch.zeros(B, T, Hq, D, dtype=q.dtype, device=q.device)
    lse = torch.full((B, Hq, T), -math.inf, device=q.device)
    k = _read(st["pages"], case["group"], p, s, 0).transpose(1, 2)  # [B, H, cap, 128]
    qs = q.float().unflatten(2, (H, G)).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, D)
    x = (qs @ k.transpose(-1, -2)).unflatten(2, (T, G)) * (1.0 / math.sqrt(D))
    del k
    i = torch.arange(T, device=q.device)
    last = torch.where(i < c[:, None], n[:, None] - c[:, None] + 1 + i, 0)  # slots a query sees
    sees = torch.arange(cap, device=q.device) < last[..., None]  # [B, T, cap]
    x = torch.where(sees[:, None, :, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    w = e / torch.where(total == 0, 1.0, total)
    del e, x
    v = _read(st["pages"], case["group"], p, s, 1).transpose(1, 2)
    held = torch.arange(cap, device=q.device) < n[:, None]
    v = torch.where(held[:, None, :, None], v, 0.0)
    o = (w.flatten(2, 3) @ v).unflatten(2, (T, G)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    out[:] = o.to(q.dtype)
    lse[:] = (torch.log(total) + top).squeeze(-1).permute(0, 1, 3, 2).reshape(B, Hq, T)
    got = [out]
    if case["lse"]:
        got.append(lse)
    if case["track"]:
        sums = w.sum((2, 3)).transpose(1, 2)  # [B, cap, H]
        st["weights"][p[held], :, s[held]] = sums[held]
        got.append(st["weights"])
    return got


def _append(st):
    case = st["case"]
    B, T, H, _ = st["k"].shape
    group, page = case["group"], case["page"]
    n = st["lengths"].long()
    c = st["counts"].long() if st["counts"] is not None else torch.full_like(n, T)
    i = torch.arange(T, device=n.device)
    b, i = torch.nonzero(i < c[:, None], as_tuple=True)
    slot = n[b] + i
    p, s = st["table"].long()[b, slot // page], slot % page
    parts = _parts(st["pages"], group)
    got = []
    for value, x in ((0, st["k"]), (1, st["v"])):
        codes, scale, zero = _quantise(x[b, i].float(), group)
        parts[2 * value][p, :, s // 16, s % 16] = _rows(codes, value)
        parts[2 * value + 1][p, :, s // 16, s % 16] = _pairs(scale, zero)
        y = torch.zeros_like(x)
        y[b, i] = _values(codes, scale, zero, group).to(x.dtype)
        got.append(y)
    st["positions"][p, :, s] = slot[:, None].to(torch.int32)
    st["weights"][p, :, s] = 0.0
    return got + [st["positions"], st["weights"]]


def _select(st):
    case = st["case"]
    keep, H = case["keep"], case["heads_kv"]
    p, s = _slots(st["table"], case["page"])
    B, cap = p.shape
    n = st["lengths"].long()
    w = st["weights"][p, :, s].transpose(1, 2)  # [B, H, cap]
    pos = st["positions"][p, :, s].transpose(1, 2)
    i = torch.arange(cap, device=n.device)
    held = (i < n[:, None])[:, None].expand(B, H, cap)
    safe = held & (pos >= (st["seen"].long() - case["recent"])[:, None, None])
    # ascending (rank, weight), lowest slot first among equals: two stable sorts
    rank = torch.where(~held, 2, torch.where(safe, 1, 0))
    a = torch.argsort(torch.where(safe, 0.0, w), dim=-1, stable=True)
    a = torch.gather(a, -1, torch.argsort(torch.gather(rank, -1, a), dim=-1, stable=True))
    place = torch.empty_like(a).scatter_(-1, a, i.expand(B, H, cap))
    goes = held & (place < (n - keep).clamp(min=0)[:, None, None])
    holes, movers = goes & (i < keep), held & ~goes & (i >= keep)
    # the k-th mover stands in the k-th hole
    src = torch.full((B, H, keep), -1, dtype=torch.int32, device=n.device)
    m = min(keep, cap)
    src[..., :m] = torch.where(held & ~goes, i, -1)[..., :m].to(torch.int32)
    bh, slot = torch.nonzero(movers.flatten(0, 1), as_tuple=True)
    bh2, hole = torch.nonzero(holes.flatten(0, 1), as_tuple=True)
    src.view(B * H, keep)[bh2, hole] = slot.to(torch.int32)
    return src, n.clamp(max=keep).to(torch.int32)


def _move(st):
    case, src = st["case"], st["src"]
    page = case["page"]
    i = torch.arange(src.shape[-1], device=src.device)
    b, h, d = torch.nonzero((src >= 0) & (src != i), as_tuple=True)
    f = src[b, h, d].long()
    t = st["table"].long()
    pf, sf, pd, sd = t[b, f // page], f % page, t[b, d // page], d % page
    for part in _parts(st["pages"], case["group"]):
        part[pd, h, sd // 16, sd % 16] = part[pf, h, sf // 16, sf % 16]
    st["positions"][pd, h, sd] = st["positions"][pf, h, sf]
    st["weights"][pd, h, sd] = st["weights"][pf, h, sf]
    # moves copy what is stored, so the pool has to be equal byte for byte
    return [st["pages"], st["positions"], st["weights"]]


def run(st):
    case = st["case"]
    if not own:
        return {"attend": _attend, "append": _append, "select": _select, "move": _move}[case["op"]](st)
    import llm_fa_b200 as fa
    cache, table, lengths = st["cache"], st["table"], st["lengths"]
    if case["op"] == "attend":
        got = fa.kv4_attention(st["q"], cache, table, lengths, counts=st["counts"],
                               decay=0.0 if case["track"] else None, return_lse=case["lse"])
        got = list(got) if case["lse"] else [got]
        return got + ([cache.weights] if case["track"] else [])
    if case["op"] == "append":
        fa.kv4_append(cache, st["k"], st["v"], table, lengths, counts=st["counts"])
        k, v = fa.kv4_expand(cache, table, lengths, case["tokens"], counts=st["counts"],
                             dtype=st["k"].dtype)
        return [k, v, cache.positions, cache.weights]
    if case["op"] == "select":
        return fa.kv4_evict_select(cache, table, lengths, case["keep"], recent=case["recent"],
                                   seen=st["seen"])
    fa.kv4_evict_move(cache, table, st["src"])
    return [cache.pages, cache.positions, cache.weights]


# ---------------------------------------------------------------- in 64 bits, from the definition
def _where(value):
    """Byte and shift of every channel's code in a stored row."""
    ch = np.arange(D)
    if value:
        half = ch // 4  # natural half-word k * 8 + g
        byte = 2 * ((half % 8) * 4 + half // 8) + (ch % 4) // 2
    else:
        word = ch // 8  # natural word j * 4 + c
        byte = 4 * ((word % 4) * 4 + word // 4) + (ch % 8) // 2
    return byte, 4 * (ch % 2)


def _decode64(pool, group, token, value):
    """fp64 [tokens, heads, 128] of (page, slot) pairs, straight from the stored bytes. `pool` is
    uint8 [pages, heads, bytes], `token` int64 [tokens, 2]."""
    m = (D // group) * 4
    base = (token[:, 1] // 16) * _block_bytes(group) + value * 16 * (64 + m)
    lane = token[:, 1] % 16
    byte, shift = _where(value)
    row = pool[token[:, 0]]  # [tokens, heads, bytes]
    at = (base + lane * 64)[:, None] + torch.as_tensor(byte, device=pool.device)
    code = torch.gather(row, 2, at[:, None].expand(-1, row.shape[1], -1)).to(torch.int32)
    code = ((code >> torch.as_tensor(shift, device=pool.device)) & 15).double()
    at = (base + 16 * 64 + lane * m)[:, None] + torch.arange(m, device=pool.device)
    raw = torch.gather(row, 2, at[:, None].expand(-1, row.shape[1], -1)).to(torch.int32)
    word = raw[..., 0::2] | (raw[..., 1::2] << 8)
    half = (word << 16).view(torch.float32).double()  # a bf16 is the upper half of an fp32
    grp = torch.arange(D, device=pool.device) // group
    return half[..., 0::2][..., grp] * (code - half[..., 1::2][..., grp])


def _bf16_of(x):
    """fp64 numpy -> the nearest bf16 value, halves to even, as fp64."""
    m, e = np.frexp(x)
    return np.ldexp(np.round(m * 256.0), e - 8)


def exact(case, seed):
    st = prepare(case, seed)
    B, H, page, group = case["batch"], case["heads_kv"], case["page"], case["group"]
    table, lens = st["table"].cpu().numpy().astype(np.int64), st["lengths"].tolist()
    if case["op"] == "attend":
        q = st["q"].double()
        T, Hq = q.shape[1], q.shape[2]
        counts = st["counts"].tolist() if st["counts"] is not None else [T] * B
        out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=DEV)
        lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=DEV)
        weights = st["weights"].double()
        for b in range(B):
            n, c = lens[b], counts[b]
            tok = np.arange(n)
            at = torch.as_tensor(np.stack((table[b, tok // page], tok % page), 1), device=DEV)
            k, v = ([torch.cat([_decode64(st["pages"], group, a, side) for a in at.split(4096)])
                     for side in (0, 1)])
            got = torch.zeros(n, H, dtype=torch.float64, device=DEV)
            for i in range(c):
                m = max(0, n - (c - 1 - i))
                if m == 0:
                    continue
                for h in range(H):
                    rows = slice(h * (Hq // H), (h + 1) * (Hq // H))
                    x = q[b, i, rows] @ k[:m, h].T / math.sqrt(D)
                    lse[b, rows, i] = torch.logsumexp(x, -1)
                    w = torch.softmax(x, -1)
                    out[b, i, rows] = w @ v[:m, h]
                    got[:m, h] += w.sum(0)
            weights[at[:, 0], :, at[:, 1]] = got
        return [out] + ([lse] if case["lse"] else []) + ([weights] if case["track"] else [])
    if case["op"] == "append":
        T = case["tokens"]
        counts = st["counts"].tolist() if st["counts"] is not None else [T] * B
        positions, weights = st["positions"].cpu().numpy(), st["weights"].double().cpu().numpy()
        got = []
        for x in (st["k"], st["v"]):
            x = x.double().cpu().numpy().reshape(B, T, H, D // group, group)
            lo, hi = np.minimum(x.min(-1), 0.0), np.maximum(x.max(-1), 0.0)
            scale = _bf16_of((hi - lo) / 15.0)
            by = np.where(scale == 0.0, 1.0, scale)[..., None]
            zero = np.clip(np.rint(-lo[..., None] / by), 0, 15)
            y = scale[..., None] * (np.clip(np.rint(x / by) + zero, 0, 15) - zero)
            for b in range(B):
                y[b, counts[b]:] = 0.0
            got.append(y.reshape(B, T, H, D))
        for b in range(B):
            slot = lens[b] + np.arange(counts[b])
            positions[table[b, slot // page], :, slot % page] = slot[:, None]
            weights[table[b, slot // page], :, slot % page] = 0.0
        return got + [positions, weights]
    keep = case["keep"]
    if case["op"] == "select":
        src = np.full((B, H, keep), -1, np.int32)
        weights, positions = st["weights"].cpu().numpy(), st["positions"].cpu().numpy()
        seen = st["seen"].tolist()
        for b in range(B):
            tok = np.arange(lens[b])
            w = weights[table[b, tok // page], :, tok % page]
            pos = positions[table[b, tok // page], :, tok % page]
            for h in range(H):
                safe = pos[:, h] >= seen[b] - case["recent"]
                by = np.lexsort((tok, np.where(safe, 0.0, w[:, h]), safe))
                stays = np.ones(lens[b], bool)
                stays[by[:max(0, lens[b] - keep)]] = False
                new = min(keep, lens[b])
                row = np.where(stays[:new], tok[:new], -1)
                row[row < 0] = tok[keep:][stays[keep:]]
                src[b, h, :new] = row
        return [src, np.minimum(np.array(lens), keep).astype(np.int32)]
    pages, positions = st["pages"].cpu().numpy(), st["positions"].cpu().numpy()
    weights, src = st["weights"].double().cpu().numpy(), st["src"].cpu().numpy()
    m = (D // group) * 4
    spans = [(0, 64), (16 * 64, m), (16 * (64 + m), 64), (16 * (128 + m), m)]
    for b in range(B):
        for h in range(H):
            to = np.nonzero((src[b, h] >= 0) & (src[b, h] != np.arange(keep)))[0]
            fr = src[b, h][to]
            pt, ss, pf, sf = table[b, to // page], to % page, table[b, fr // page], fr % page
            for off, width in spans:
                j = np.arange(width)
                at_t = ((ss // 16) * _block_bytes(group) + off + (ss % 16) * width)[:, None] + j
                at_f = ((sf // 16) * _block_bytes(group) + off + (sf % 16) * width)[:, None] + j
                pages[pt[:, None], h, at_t] = pages[pf[:, None], h, at_f]
            positions[pt, h, ss] = positions[pf, h, sf]
            weights[pt, h, ss] = weights[pf, h, sf]
    return [pages, positions, weights]
