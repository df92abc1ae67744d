"""Measured cases of generation with caches in 8 bits and with several beams: the quantising write into a paged cache, attention over
such a cache, the selection of beams, and the reordering of a cache after it.

``run`` computes them in plain form (elementary torch operations in 32 bits, the selection in 64) or, with ``own``, through the
framework's entry points.  What a case says fixes sizes and lengths, the seed their order and all values.  A cache in 8 bits holds whole
numbers from -127 to 127 and a scale in 32 bits for each block of tokens and head; where a write returns it, it is returned as the
numbers that it stands for.  Scales of blocks that no sequence has reached are NaN where attention reads them, as memory that nobody
cleared may be.
"""
import math
import random

import torch

own = False

DEV = "cuda"
F32, BF16, I8 = torch.float32, torch.bfloat16, torch.int8
DTYPES = {"fp32": F32, "bf16": BF16}
INF = float("inf")
TINY = 2.0 ** -100                       # a block whose scale would be below this is all zeros


# ------------------------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of a batch on GPT-2 small: each sequence's token joins the 8-bit cache of one layer, in blocks that are begun
        {"name": "append8-decode", "op": "append", "seqs": 16, "kv_heads": 12, "head_dim": 64, "page": 16, "block": 16, "new_lo": 1,
         "new_hi": 1, "len_lo": 1, "len_hi": 256, "dtype": "bf16"},
        # the prompts of a batch join it, some behind what an earlier chunk left
        {"name": "append8-prompts", "op": "append", "seqs": 16, "kv_heads": 12, "head_dim": 64, "page": 16, "block": 16, "new_lo": 500,
         "new_hi": 777, "len_lo": 500, "len_hi": 1024, "dtype": "bf16"},
        # one user, one token, one layer of GPT-2 small: latency
        {"name": "decode8-one", "op": "attend", "seqs": 1, "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "block": 16,
         "new_lo": 1, "new_hi": 1, "len_lo": 701, "len_hi": 701, "drop_every": 0, "dtype": "bf16"},
        # a batch of users at all stages of GPT-2 medium's context
        {"name": "decode8-batch", "op": "attend", "seqs": 64, "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 16, "block": 16,
         "new_lo": 1, "new_hi": 1, "len_lo": 1, "len_hi": 1024, "drop_every": 0, "dtype": "bf16"},
        # long documents, heads that share keys; every ninth page has been dropped
        {"name": "decode8-long-shared", "op": "attend", "seqs": 16, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "block": 32,
         "new_lo": 1, "new_hi": 1, "len_lo": 2000, "len_hi": 32768, "drop_every": 9, "dtype": "bf16"},
        # GPT-2 small: prompts that come in chunks, sequences that are generating among them
        {"name": "chunk8-batch", "op": "attend", "seqs": 16, "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "block": 16,
         "new_lo": 1, "new_hi": 511, "len_lo": 1, "len_hi": 1024, "drop_every": 0, "dtype": "bf16"},
        # large chunks of long documents, heads that share keys
        {"name": "chunk8-long-shared", "op": "attend", "seqs": 2, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "block": 64,
         "new_lo": 1500, "new_hi": 2048, "len_lo": 6001, "len_hi": 8192, "drop_every": 0, "dtype": "bf16"},
        # a character model's lines, queries in fp32
        {"name": "chunk8-fp32", "op": "attend", "seqs": 32, "heads": 4, "kv_heads": 4, "head_dim": 32, "page": 16, "block": 8,
         "new_lo": 8, "new_hi": 64, "len_lo": 8, "len_hi": 256, "drop_every": 0, "dtype": "fp32"},
        # characters: a few prompts with a few beams each
        {"name": "beams-characters", "op": "beams", "groups": 16, "beams": 4, "width": 4, "vocab": 65, "finished": True, "mask": True,
         "dtype": "bf16"},
        # sub-words: the logits of 64 prompts with 16 beams each
        {"name": "beams-batch", "op": "beams", "groups": 64, "beams": 16, "width": 16, "vocab": 50304, "finished": True, "mask": False,
         "dtype": "fp32"},
        # one prompt's beams on GPT-2 small: tables, and the last pages of all layers
        {"name": "reorder-one", "op": "reorder", "groups": 1, "beams": 4, "layers": 12, "kv_heads": 12, "head_dim": 64, "page": 16,
         "len_lo": 701, "len_hi": 701, "dtype": "bf16"},
        # a batch of them on GPT-2 medium
        {"name": "reorder-batch", "op": "reorder", "groups": 8, "beams": 8, "layers": 24, "kv_heads": 16, "head_dim": 64, "page": 16,
         "len_lo": 300, "len_hi": 1001, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "attend", "beams", "beams", "reorder"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "beams":
        vocab = rng.randint(40, 250) if rng.random() < 0.3 else _log(rng, 2000, 50304)
        beams = rng.choice([1, 2, 3, 4, 4, 5, 8, 16])
        return {"op": op, "groups": _log(rng, 1, 1024 // beams), "beams": beams, "width": rng.choice([beams, beams, 2 * beams, 4]),
                "vocab": vocab, "finished": rng.random() < 0.5, "mask": rng.random() < 0.3, "dtype": dtype}
    kv_heads, page = rng.choice([1, 2, 4, 6, 8, 12, 16]), rng.choice([8, 16, 16, 32, 48, 64, 128])
    head_dim = rng.choice([32, 64, 64, 128])
    if op == "reorder":
        layers, beams, length = _log(rng, 1, 24), rng.choice([2, 3, 4, 4, 5, 8, 16]), _log(rng, 1, 1024)
        bytes_of_page = 8 * layers * kv_heads * page * head_dim
        groups = max(1, min(_log(rng, 1, 64), (1 << 29) // (bytes_of_page * (length // page + 2 * beams))))
        return {"op": op, "groups": groups, "beams": beams, "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
                "len_lo": rng.choice([1, length]), "len_hi": length, "dtype": dtype}
    block = rng.choice([b for b in (8, 16, 24, 32, 64, 128) if page % b == 0])
    c = {"op": op, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "block": block, "dtype": dtype}
    if op == "append":
        new_hi = rng.choice([1, _log(rng, 2, 777)])
        length = _log(rng, new_hi, 1024)
        seqs = min(_log(rng, 1, 128), max(1, (1 << 24) // (kv_heads * head_dim * length)))
        return {**c, "seqs": seqs, "new_lo": rng.choice([1, new_hi]), "new_hi": new_hi, "len_lo": rng.choice([1, length]), "len_hi": length}
    group = rng.choice([1, 1, 1, 2, 4, 5, 8]) if kv_heads <= 8 else 1
    c = {**c, "heads": kv_heads * group, "drop_every": rng.choice([0, 0, 0, rng.randint(3, 20)])}
    if rng.random() < 0.6:                                # one token each, a few where the model's guesses are checked
        new_lo, new_hi = rng.choice([(1, 1), (1, 1), (0, 1), (1, 4)])
        length = _log(rng, 16, 32768)
        most = 1 << (28 if dtype == "bf16" else 27)       # tokens of the cache, times the heads' columns
    else:
        new_hi = _log(rng, 2, 2048)
        new_lo = rng.choice([1, new_hi, max(1, new_hi // 2)])
        length = _log(rng, new_hi, 8192)
        most = 1 << 24
        if dtype == "fp32":
            new_hi, new_lo, length = min(new_hi, 512), min(new_lo, 512), min(length, 2048)
    seqs = min(_log(rng, 1, 128), max(1, most // (kv_heads * 128 * length)))
    if new_hi > 4:                                        # as many pairs of tokens as the largest listed case at most
        seqs = max(1, min(seqs, (1 << 30) // (c["heads"] * new_hi * length)))
    return {**c, "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi, "len_lo": rng.choice([1, length, max(1, length // 2)]),
            "len_hi": length}


def _lengths(case):
    """(new tokens, length with them) of each sequence: evenly spread, short prompts beside long caches."""
    n, out = case["seqs"], []
    for b in range(n):
        new = case["new_lo"] + (case["new_hi"] - case["new_lo"]) * b // max(1, n - 1) if n > 1 else case["new_hi"]
        at = (b * 7 + n // 2) % n
        length = case["len_lo"] + (case["len_hi"] - case["len_lo"]) * at // max(1, n - 1) if n > 1 else case["len_hi"]
        out.append((new, max(new, length)))
    return out


def _beams(case):
    """(tokens, parent of each beam) of each group: the best beams of a step go on in two or three, others end."""
    rng, n, out = random.Random(5), case["beams"], []
    for b in range(case["groups"]):
        length = case["len_lo"] + (case["len_hi"] - case["len_lo"]) * b // max(1, case["groups"] - 1) if case["groups"] > 1 else case["len_hi"]
        out.append((length, [min(rng.randrange(n), rng.randrange(n)) for _ in range(n)]))
    return out


# ------------------------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rnd(*shape, scale=1.0, dtype=dt):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype).mul_(scale)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32).to(DEV)

    if case["op"] == "beams":
        B, n, V = case["groups"], case["beams"], case["vocab"]
        s = {"case": case, "logits": rnd(B * n, V, scale=3.0), "finished": None, "allowed": None}
        s["scores"] = (-12.0 - 3.0 * torch.rand(B, n, generator=g, device=DEV)).sort(1, descending=True).values
        if n > 2:
            s["scores"][::3, -1] = -INF                                     # groups that have fewer beams
        if case["finished"]:
            s["finished"] = torch.rand(B, n, generator=g, device=DEV) < 0.2
        if case["mask"]:                                                    # tokens that a grammar allows, one bit each
            both = torch.randint(-2 ** 31, 2 ** 31, (2, B * n, (V + 31) // 32), generator=g, device=DEV)
            s["allowed"] = (both[0] & both[1]).to(torch.int32)              # a quarter of the tokens
            s["allowed"][::7] = 0
        return s

    G, D, P = case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "reorder":
        pairs, n = _beams(case), case["beams"]
        order = torch.randperm(len(pairs), generator=h).tolist()
        pairs = [pairs[i] for i in order]
        width = max(-(-l // P) for l, _ in pairs) + 1
        total = sum(l // P for l, _ in pairs) + 2 * n * len(pairs)
        free = torch.randperm(total, generator=h)
        table = torch.full((len(pairs), n, width), -1, dtype=torch.int32)
        start = 0
        for b, (length, _) in enumerate(pairs):
            full = length // P
            for i in range(n):                                              # pages of a group's past, in each beam's order
                table[b, i, :full] = free[start:start + full].roll(i)
            table[b, :, full] = free[start + full:start + full + n]
            start += full + n
        spare = free[start:start + n * len(pairs)]
        return {"case": case, "pages": table.view(-1, width).to(DEV), "spare": spare.to(torch.int32).to(DEV),
                "parents": ints([p for _, p in pairs]), "lengths": ints([l for l, _ in pairs]),
                "cache_k": rnd(case["layers"], total, G, P, D), "cache_v": rnd(case["layers"], total, G, P, D)}

    pairs = _lengths(case)
    order = torch.randperm(len(pairs), generator=h).tolist()
    new, length = [pairs[i][0] for i in order], [pairs[i][1] for i in order]
    H, drop = case.get("heads", G), case.get("drop_every", 0)
    counts = [-(-l // P) for l in length]
    width, total = max(counts), sum(counts) + 7                             # some pages belong to nobody here
    free = torch.randperm(total, generator=h)
    table = torch.full((len(pairs), width), -1, dtype=torch.int32)
    start = 0
    for b, c in enumerate(counts):
        table[b, :c] = free[start:start + c]
        if drop:
            table[b, :c][(torch.arange(c) * 5 + order[b]) % drop == 1] = -1
        start += c
    N = sum(new)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    s = {"case": case, "pages": table.to(DEV), "offsets": ints(offsets), "lengths": ints(length), "max_new": max(new),
         "max_len": max(length)}
    for name in ("k", "v"):
        s["cache_" + name] = rnd(total, G, P, D, scale=40.0, dtype=BF16).round_().clamp_(-127, 127).to(I8)
        s[name + "_scales"] = 0.02 + 0.02 * torch.rand(total, G, P // case["block"], generator=g, device=DEV)
    qkv = rnd(N, (H + 2 * G) * D)                                           # one projection makes all three
    s["q"] = qkv[:, :H * D].view(N, H, D)
    s["k"] = qkv[:, H * D:(H + G) * D].view(N, G, D)
    s["v"] = qkv[:, (H + G) * D:].view(N, G, D)
    if case["op"] == "attend":
        reached = (torch.arange(0, width * P, case["block"]) < torch.tensor(length)[:, None]).view(len(pairs), width, -1)
        used = torch.zeros(total, P // case["block"], dtype=torch.bool)
        used[table[table >= 0].long()] = reached[table >= 0]
        for name in ("k_scales", "v_scales"):
            s[name].masked_fill_(~used.to(DEV)[:, None], float("nan"))
    return s


# ------------------------------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------------------------------
def _values(cache, scales):
    """The numbers that an 8-bit cache stands for."""
    pages, G, P, D = cache.shape
    blocks = scales.shape[2]
    return (cache.view(pages, G, blocks, P // blocks, D) * scales[..., None, None]).view(pages, G, P, D)


def _tokens(s):
    """Of each new token its sequence, number in it, and position."""
    N = s["q"].shape[0]
    row = torch.arange(N, device=DEV)
    seq = torch.searchsorted(s["offsets"][1:].long(), row, right=True)
    at = row - s["offsets"][seq]
    new = s["offsets"][1:] - s["offsets"][:-1]
    return seq, at, s["lengths"][seq] - new[seq] + at


def _quantise(x, cache, scales, page, slot, first):
    """New tokens' rows x into cache and scales.  A block's scale is the 127th part of the largest magnitude in it; what it held before a
    larger one came is rounded anew.  first: of each sequence the first new token."""
    (pages, G, P, _), blocks = cache.shape, scales.shape[2]
    block = P // blocks
    at = page * blocks + slot // block
    top = torch.zeros(pages * blocks, G, device=DEV).index_reduce_(0, at, x.float().abs().amax(-1), "amax")
    before = scales.transpose(1, 2).reshape(pages * blocks, G)
    begun, slot0, page0 = at[first], slot[first], page[first]               # only a first token's block can hold earlier ones
    held = torch.where((slot0 % block > 0)[:, None], before[begun], 0.0)
    after = torch.zeros_like(top)
    after[begun] = held
    after = torch.maximum(after, top / 127.0)
    after = torch.where(after >= TINY, after, 0.0)
    touched = torch.zeros(pages * blocks, 1, dtype=torch.bool, device=DEV)
    touched[at] = True
    scales.copy_(torch.where(touched, after, before).view(pages, blocks, G).transpose(1, 2))
    ratio = torch.where(after[begun] > 0, held / after[begun], 0.0)
    slots = (slot0 // block * block)[:, None] + torch.arange(block, device=DEV)
    old = cache[page0[:, None], :, slots]                                   # [sequences, block, heads, head size]
    again = torch.round(old.float() * ratio[:, None, :, None]).to(I8)
    cache[page0[:, None], :, slots] = torch.where((slots < slot0[:, None])[..., None, None], again, old)
    step = after[at][..., None]
    inverse = torch.where(step > 0, 1.0 / step, 0.0)
    cache[page, :, slot] = torch.round(x.float() * inverse).clamp(-127.0, 127.0).to(I8)


def _append(s):
    P = s["cache_k"].shape[2]
    seq, _, pos = _tokens(s)
    page, slot, first = s["pages"][seq, pos // P].long(), (pos % P).long(), s["offsets"][:-1].long()
    _quantise(s["k"], s["cache_k"], s["k_scales"], page, slot, first)
    _quantise(s["v"], s["cache_v"], s["v_scales"], page, slot, first)
    return _appended(s)


def _appended(s):
    return _values(s["cache_k"], s["k_scales"]), _values(s["cache_v"], s["v_scales"]), s["k_scales"], s["v_scales"]


def _attend(s):
    q, P, block = s["q"], s["cache_k"].shape[2], s["case"]["block"]
    (N, H, D), G = q.shape, s["cache_k"].shape[1]
    B, L, n = s["lengths"].shape[0], s["max_len"], s["max_new"]
    pos = torch.arange(L, device=DEV)
    page, slot = s["pages"][:, pos // P].long(), pos % P
    there = (pos < s["lengths"][:, None]) & (page >= 0)                                           # [B, L]

    def rows_of(cache, scales):
        x = cache[page.clamp_min(0), :, slot] * scales[page.clamp_min(0), :, slot // block][..., None]
        return torch.where(there[:, :, None, None], x, 0.0).permute(0, 2, 1, 3)                   # [B, G, L, D]

    k, v = rows_of(s["cache_k"], s["k_scales"]), rows_of(s["cache_v"], s["v_scales"])
    i = torch.arange(n, device=DEV)
    new = s["offsets"][1:] - s["offsets"][:-1]
    rows = q[(s["offsets"][:-1, None] + i).clamp_max(N - 1)].float()                              # [B, n, H, D]
    rows = rows.view(B, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * n, D) * D ** -0.5
    seen = there[:, None, :] & (pos <= (s["lengths"] - new)[:, None, None] + i[:, None])         # [B, n, L]
    x = (rows @ k.transpose(2, 3)).view(B, G, H // G, n, L)
    x = torch.where(seen[:, None, None], x, -INF)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -INF, 0.0, m)
    x = torch.exp(x - m)
    l = x.sum(-1, keepdim=True)
    o = (x.view(B, G, -1, L) @ v).view(B, G, H // G, n, D) / torch.where(l > 0, l, 1.0)
    lse = torch.where(l > 0, m + torch.log(l), -INF)[..., 0]
    seq, at, _ = _tokens(s)
    return o.permute(0, 3, 1, 2, 4)[seq, at].reshape(N, H, D).to(q.dtype), lse.permute(0, 3, 1, 2)[seq, at].reshape(N, H)


def _select(s):
    """In 64 bits, so that candidates of different beams do not change places by the rounding of their sums."""
    scores, width = s["scores"].double(), s["case"]["width"]
    (B, n), V = scores.shape, s["logits"].shape[1]
    x = s["logits"].double()
    if s["allowed"] is not None:
        t = torch.arange(V, device=DEV)
        x = torch.where((s["allowed"][:, t // 32] >> (t % 32)) & 1 > 0, x, -INF)
    m = x.amax(1, keepdim=True)
    m = torch.where(m == -INF, 0.0, m)
    lse = m + torch.log(torch.exp(x - m).sum(1, keepdim=True))
    start = scores.view(-1, 1)
    over = torch.zeros_like(start, dtype=torch.bool) if s["finished"] is None else s["finished"].view(-1, 1)
    x = torch.where((lse > -INF) & ~over, start + (x - lse), -INF)
    x = torch.cat([x, torch.where(over, start, -INF)], 1).view(B, n * (V + 1))      # the last one: a finished beam stays as it is
    best, at = x.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :width], at[:, :width]
    token = at % (V + 1)
    some = best > -INF
    slot = torch.arange(width, device=DEV).expand(B, width) % n
    return (torch.where(some, at // (V + 1), slot).to(torch.int32), torch.where(some & (token < V), token, -1).to(torch.int32),
            best.to(F32))


def _reorder(s):
    P, parents, pages, spare = s["cache_k"].shape[3], s["parents"].long(), s["pages"], s["spare"]
    B, n = parents.shape
    own_row = torch.arange(B * n, device=DEV)
    row = (own_row // n * n).view(B, n).add(parents).view(-1)
    length = s["lengths"].repeat_interleave(n)
    full, rest = (length // P).long(), length % P
    col = torch.arange(pages.shape[1], device=DEV)
    moved = (rest > 0) & (row != own_row)
    tail = pages[own_row, full]
    new = torch.where(col < full[:, None], pages[row], pages)
    new = torch.where((col == full[:, None]) & moved[:, None], spare[:, None], new)
    source, to = pages[row, full].long(), spare.long()
    copied = (moved[:, None] & (torch.arange(P, device=DEV) < rest[:, None]))[None, :, None, :, None]
    source = torch.where(moved, source, to)
    s["cache_k"][:, to] = torch.where(copied, s["cache_k"][:, source], s["cache_k"][:, to])
    s["cache_v"][:, to] = torch.where(copied, s["cache_v"][:, source], s["cache_v"][:, to])
    return new, torch.where(moved, tail, spare), s["cache_k"], s["cache_v"]


# ------------------------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if not own:
        return {"append": _append, "attend": _attend, "beams": _select, "reorder": _reorder}[op](s)
    from cme213_final_project_b200 import ops
    if op == "append":
        ops.cache_append(s["k"], s["v"], s["cache_k"], s["cache_v"], s["pages"], s["offsets"], s["lengths"], k_scales=s["k_scales"],
                         v_scales=s["v_scales"])
        return _appended(s)
    if op == "attend":
        return ops.paged_attention(s["q"], s["cache_k"], s["cache_v"], s["pages"], s["offsets"], s["lengths"], k_scales=s["k_scales"],
                                   v_scales=s["v_scales"])
    if op == "beams":
        return ops.beam_step(s["logits"], s["scores"], s["case"]["width"], finished=s["finished"], allowed=s["allowed"])
    new, spare = ops.cache_reorder(s["cache_k"], s["cache_v"], s["pages"], s["spare"], s["parents"], s["lengths"])
    return new, spare, s["cache_k"], s["cache_v"]


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "beams":
        rows = case["groups"] * case["beams"]
        n = rows * case["vocab"]
        return {"bytes": n * e + n / 8 * bool(case["mask"]) + rows * 5 + 12 * case["groups"] * case["width"], "flops": 4 * n}
    G, D, P = case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "reorder":
        n, moved = case["beams"], 0
        pairs = _beams(case)
        for length, parents in pairs:
            from_others = {p for i, p in enumerate(parents) if p != i}
            moved += (length % P) * (len(from_others) + sum(p != i for i, p in enumerate(parents)))
        tables = 8 * n * sum(length // P + 4 for length, _ in pairs)
        return {"bytes": 2 * case["layers"] * G * D * e * moved + tables, "flops": 0}
    pairs = _lengths(case)
    new, length = sum(n for n, _ in pairs), sum(l for _, l in pairs)
    tables = 4 * (length / P + 2 * len(pairs))
    if case["op"] == "append":
        held = sum((l - n) % case["block"] for n, l in pairs)               # tokens of blocks that were begun: read, and written where they grow
        scales = 8 * G * sum((l - 1) // case["block"] - (l - n) // case["block"] + 1 for n, l in pairs)
        return {"bytes": 2 * new * G * D * (e + 1) + 2 * held * G * D + scales + tables, "flops": 4 * new * G * D}
    H, kept = case["heads"], 1 - 1 / case["drop_every"] if case["drop_every"] else 1
    visible = sum(n * (l - n) + n * (n + 1) / 2 for n, l in pairs)
    held = 2 * length * G * (D + 4 / case["block"]) * kept
    return {"bytes": held + new * H * (2 * D * e + 4) + tables, "flops": 4 * D * H * visible * kept}


# ------------------------------------------------------------------------------------------------------------------
# The definitions, in 64 bits, sequence by sequence and group by group
# ------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "reorder":
        return None                                       # copies: held to be equal as they are
    if case["op"] == "append":
        # The numbers stored are roundings that are defined in 32 bits; the scales have values.
        P, block = case["page"], case["block"]
        starts, lengths = s["offsets"].tolist(), s["lengths"].tolist()
        scales = {"k": s["k_scales"].double(), "v": s["v_scales"].double()}
        for b, length in enumerate(lengths):
            lo, n = starts[b], starts[b + 1] - starts[b]
            at = length - n
            while at < length:                            # one block of the sequence at a time
                end = min(length, (at // block + 1) * block)
                page, where = int(s["pages"][b, at // P]), at % P // block
                for name in scales:
                    rows = s[name][lo + at - (length - n):lo + end - (length - n)].double()
                    top = rows.abs().amax(dim=(0, 2)) / 127
                    scales[name][page, :, where] = torch.maximum(top, scales[name][page, :, where]) if at % block else top
                at = end
        return None, None, scales["k"], scales["v"]
    if case["op"] == "attend":
        (N, H, D), P, G, block = s["q"].shape, case["page"], case["kv_heads"], case["block"]
        out, lse = torch.zeros(N, H, D, device=DEV, dtype=torch.float64), torch.full((N, H), -INF, device=DEV, dtype=torch.float64)
        starts, lengths = s["offsets"].tolist(), s["lengths"].tolist()
        for b, length in enumerate(lengths):
            lo, hi = starts[b], starts[b + 1]
            if hi == lo:
                continue
            where = torch.tensor([t for t, p in enumerate(s["pages"][b].repeat_interleave(P).tolist()[:length]) if p >= 0],
                                 device=DEV, dtype=torch.long)
            page = s["pages"][b].long()[where // P]
            reach = length - (hi - lo) + torch.arange(hi - lo, device=DEV)
            hidden = where[None, :] > reach[:, None]
            for h in range(H):
                if where.numel() == 0:
                    break
                at = (page, h * G // H, where % P)
                of = (page, h * G // H, where % P // block)
                k = s["cache_k"][at].double() * s["k_scales"][of].double()[:, None]
                v = s["cache_v"][at].double() * s["v_scales"][of].double()[:, None]
                x = (s["q"][lo:hi, h].double() @ k.T) / math.sqrt(D)
                x[hidden] = -INF
                lse[lo:hi, h] = torch.logsumexp(x, 1)
                out[lo:hi, h] = torch.softmax(x, 1).nan_to_num(0.0) @ v
        return out, lse
    B, n, V, width = case["groups"], case["beams"], case["vocab"], case["width"]
    best = torch.full((B, width), -INF, device=DEV, dtype=torch.float64)
    for b in range(B):
        found = []
        for i in range(n):
            r, start = b * n + i, s["scores"][b, i].double()
            if s["finished"] is not None and bool(s["finished"][b, i]):
                found.append(start.view(1))
                continue
            x = s["logits"][r].double()
            if s["allowed"] is not None:
                bits = (s["allowed"][r][:, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
                x = x[bits.flatten()[:V] > 0]
            if x.numel():
                found.append(start + torch.log_softmax(x, 0))
        v = torch.cat(found).sort(descending=True).values[:width] if found else best[b, :0]
        best[b, :v.numel()] = v
    return None, None, best
