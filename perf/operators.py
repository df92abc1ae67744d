"""Measured cases of the generation operators: the write into a paged cache of keys and values, attention of new tokens over that
cache, and the way from logits to the next token.

``run`` computes them in plain form (elementary torch operations in 32 bits) or, with ``own``, through the framework's entry points.
Sequences of a case differ in length; what a case says fixes the lengths, the seed their order and all values.  The slots of the
cache that no sequence has reached hold NaN where attention reads it, as memory that nobody cleared may.
"""
import math

import torch

own = False

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
DTYPES = {"fp32": F32, "bf16": BF16}
INF = float("inf")


# ------------------------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of a batch on GPT-2 small: each sequence's token joins the cache of one layer
        {"name": "append-decode", "op": "append", "seqs": 16, "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "new_lo": 1,
         "new_hi": 1, "len_lo": 1, "len_hi": 1024, "drop_every": 0, "dtype": "bf16"},
        # the prompts of a batch join it
        {"name": "append-prompts", "op": "append", "seqs": 16, "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16,
         "new_lo": 500, "new_hi": 1024, "len_lo": 500, "len_hi": 1024, "drop_every": 0, "dtype": "bf16"},
        # one user, one token, one layer of GPT-2 small: latency
        {"name": "decode-one", "op": "attend", "seqs": 1, "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "new_lo": 1,
         "new_hi": 1, "len_lo": 701, "len_hi": 701, "drop_every": 0, "dtype": "bf16"},
        # a batch of users at all stages of GPT-2 medium's context
        {"name": "decode-batch", "op": "attend", "seqs": 64, "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 16, "new_lo": 1,
         "new_hi": 1, "len_lo": 1, "len_hi": 1024, "drop_every": 0, "dtype": "bf16"},
        # long documents, heads that share keys; every ninth page has been dropped
        {"name": "decode-long-shared", "op": "attend", "seqs": 16, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "new_lo": 1, "new_hi": 1, "len_lo": 2000, "len_hi": 32768, "drop_every": 9, "dtype": "bf16"},
        # the width-512 model's heads in fp32 storage
        {"name": "decode-fp32", "op": "attend", "seqs": 32, "heads": 4, "kv_heads": 4, "head_dim": 128, "page": 16, "new_lo": 1,
         "new_hi": 1, "len_lo": 1, "len_hi": 2048, "drop_every": 0, "dtype": "fp32"},
        # GPT-2 small: prompts that come in chunks, sequences that are generating among them
        {"name": "chunk-batch", "op": "attend", "seqs": 16, "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "new_lo": 1,
         "new_hi": 511, "len_lo": 1, "len_hi": 1024, "drop_every": 0, "dtype": "bf16"},
        # large chunks of long documents, heads that share keys
        {"name": "chunk-long-shared", "op": "attend", "seqs": 2, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "new_lo": 1500, "new_hi": 2048, "len_lo": 6001, "len_hi": 8192, "drop_every": 0, "dtype": "bf16"},
        # a character model's lines in fp32 storage
        {"name": "chunk-fp32", "op": "attend", "seqs": 32, "heads": 4, "kv_heads": 4, "head_dim": 32, "page": 16, "new_lo": 8,
         "new_hi": 64, "len_lo": 8, "len_hi": 256, "drop_every": 0, "dtype": "fp32"},
        # characters: the row is shorter than a block
        {"name": "pick-characters", "op": "pick", "rows": 64, "vocab": 65, "history": 256, "biases": 0, "mask": True,
         "noise": True, "processed": False, "empty_row": False, "dtype": "bf16"},
        # sub-words: a batch of users with all that the operator has, and the processed logits
        {"name": "pick-batch", "op": "pick", "rows": 64, "vocab": 50304, "history": 1024, "biases": 64, "mask": True,
         "noise": False, "processed": True, "empty_row": True, "dtype": "bf16"},
        # many samples at once
        {"name": "pick-samples", "op": "pick", "rows": 1024, "vocab": 50304, "history": 1024, "biases": 0, "mask": False,
         "noise": True, "processed": True, "empty_row": False, "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "attend", "pick", "pick"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "pick":
        vocab = rng.randint(40, 250) if rng.random() < 0.3 else _log(rng, 2000, 50304)
        return {"op": op, "rows": _log(rng, 1, 1024), "vocab": vocab, "history": _log(rng, 1, 4096),
                "biases": rng.choice([0, rng.randint(1, 40)]), "mask": rng.random() < 0.5, "noise": rng.random() < 0.5,
                "processed": rng.random() < 0.7, "empty_row": rng.random() < 0.3, "dtype": dtype}
    kv_heads, page = rng.choice([1, 2, 4, 6, 8, 12, 16]), rng.choice([8, 16, 16, 32, 48, 64, 128])
    group = rng.choice([1, 1, 1, 2, 4, 5, 8]) if kv_heads <= 8 else 1
    c = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": rng.choice([32, 64, 64, 128]), "page": page,
         "drop_every": rng.choice([0, 0, 0, rng.randint(3, 20)]), "dtype": dtype}
    if op == "attend" and rng.random() < 0.6:             # one token each, a few where the model's guesses are checked
        new_lo, new_hi = rng.choice([(1, 1), (1, 1), (0, 1), (1, 4)])
        length = _log(rng, 16, 32768)
        most = 1 << (28 if dtype == "bf16" else 27)       # tokens of the cache, times the heads' columns
    else:
        new_hi = _log(rng, 2, 2048)
        new_lo = rng.choice([1, new_hi, max(1, new_hi // 2)])
        length = _log(rng, new_hi, 8192)
        most = 1 << 24
        if dtype == "fp32" and op == "attend":
            new_hi, new_lo, length = min(new_hi, 512), min(new_lo, 512), min(length, 2048)
    seqs = min(_log(rng, 1, 128), max(1, most // (kv_heads * 128 * length)))
    if op == "attend" and new_hi > 4:                      # as many pairs of tokens as the largest listed case at most
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

    if case["op"] == "pick":
        R, V, L = case["rows"], case["vocab"], case["history"]
        s = {"case": case, "logits": rnd(R, V, scale=3.0), "noise": None, "bias_ids": None, "bias_values": None, "allowed": None}
        # frequencies of sub-words fall off like 1 / (rank + 20)
        u = torch.rand(R, L, generator=g, device=DEV)
        name = torch.randperm(V, generator=g, device=DEV)
        s["history"] = name[(20 * ((1 + V / 20) ** u - 1)).long().clamp_(0, V - 1)].to(torch.int32)
        s["lengths"] = torch.randint(0, L + 1, (R,), generator=g, device=DEV, dtype=torch.int32)
        s["prompts"] = (s["lengths"] * torch.rand(R, generator=g, device=DEV)).to(torch.int32)
        s["repetition"] = 1.0 + 0.5 * torch.rand(R, generator=g, device=DEV)
        s["presence"] = torch.rand(R, generator=g, device=DEV) - 0.2
        s["frequency"] = 0.3 * torch.rand(R, generator=g, device=DEV)
        s["temperature"] = 0.5 + torch.rand(R, generator=g, device=DEV)
        s["temperature"][::5] = 0.0                                         # greedy rows among the sampled ones
        if case["biases"]:
            k = case["biases"]
            s["bias_ids"] = torch.rand(R, V, generator=g, device=DEV).topk(k, dim=1).indices.to(torch.int32)
            s["bias_values"] = rnd(R, k, scale=4.0, dtype=F32)
            s["bias_ids"][:, k // 2 + 1:][torch.rand(R, k - k // 2 - 1, generator=g, device=DEV) < 0.3] = -1      # fewer of them
        if case["mask"]:                                                    # tokens that a grammar allows, one bit each
            words = (V + 31) // 32
            both = torch.randint(-2 ** 31, 2 ** 31, (2, R, words), generator=g, device=DEV)
            s["allowed"] = (both[0] & both[1]).to(torch.int32)              # a quarter of the tokens
            if case["empty_row"] and R > 1:
                s["allowed"][R // 2] = 0
        if case["noise"]:
            s["noise"] = -(-torch.rand(R, V, generator=g, device=DEV).clamp_(1e-9, 1 - 1e-7).log()).log()
        return s

    pairs = _lengths(case)
    order = torch.randperm(len(pairs), generator=h).tolist()
    new, length = [pairs[i][0] for i in order], [pairs[i][1] for i in order]
    H, G, D, P = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    counts = [-(-l // P) for l in length]
    width, total = max(counts), sum(counts) + 7                             # some pages belong to nobody here
    free = torch.randperm(total, generator=h)
    table = torch.full((len(pairs), width), -1, dtype=torch.int32)
    start = 0
    for b, c in enumerate(counts):
        table[b, :c] = free[start:start + c]
        if case["drop_every"]:
            table[b, :c][(torch.arange(c) * 5 + order[b]) % case["drop_every"] == 1] = -1
        start += c
    N = sum(new)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    s = {"case": case, "pages": table.to(DEV), "offsets": ints(offsets), "lengths": ints(length), "max_new": max(new),
         "max_len": max(length), "cache_k": rnd(total, G, P, D), "cache_v": rnd(total, G, P, D)}
    qkv = rnd(N, (H + 2 * G) * D)                                           # one projection makes all three
    s["q"] = qkv[:, :H * D].view(N, H, D)
    s["k"] = qkv[:, H * D:(H + G) * D].view(N, G, D)
    s["v"] = qkv[:, (H + G) * D:].view(N, G, D)
    if case["op"] == "attend":
        reached = (torch.arange(width * P) < torch.tensor(length)[:, None]).view(len(pairs), width, P)
        used = torch.zeros(total, P, dtype=torch.bool)
        used[table[table >= 0].long()] = reached[table >= 0]
        for name in ("cache_k", "cache_v"):
            s[name].masked_fill_(~used.to(DEV)[:, None, :, None], float("nan"))
    return s


# ------------------------------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------------------------------
def _tokens(s):
    """Of each new token its sequence, number in it, and position."""
    N = s["q"].shape[0]
    row = torch.arange(N, device=DEV)
    seq = torch.searchsorted(s["offsets"][1:].long(), row, right=True)
    at = row - s["offsets"][seq]
    new = s["offsets"][1:] - s["offsets"][:-1]
    return seq, at, s["lengths"][seq] - new[seq] + at


def _append(s):
    P = s["cache_k"].shape[2]
    seq, _, pos = _tokens(s)
    page = s["pages"][seq, pos // P].long()
    slot = (pos % P).long()
    keep = (page >= 0)[:, None, None]
    to = page.clamp_min(0)
    # a dropped page's token goes nowhere: page 0 belongs to somebody else then, and the token to a row behind the cache
    for cache, x in ((s["cache_k"], s["k"]), (s["cache_v"], s["v"])):
        if s["case"]["drop_every"]:
            flat = torch.cat([cache.transpose(1, 2).flatten(0, 1), torch.zeros_like(cache[:1, :, 0])])
            flat[torch.where(keep[:, 0, 0], to * P + slot, cache.shape[0] * P)] = x
            cache.copy_(flat[:-1].view(cache.shape[0], P, *cache.shape[1::2]).transpose(1, 2))
        else:
            cache[to, :, slot] = x
    return s["cache_k"], s["cache_v"]


def _attend(s):
    q, P = s["q"], s["cache_k"].shape[2]
    (N, H, D), G = q.shape, s["cache_k"].shape[1]
    B, L, n = s["lengths"].shape[0], s["max_len"], s["max_new"]
    pos = torch.arange(L, device=DEV)
    page, slot = s["pages"][:, pos // P].long(), pos % P
    there = (pos < s["lengths"][:, None]) & (page >= 0)                                           # [B, L]
    k, v = (torch.where(there[:, :, None, None], c[page.clamp_min(0), :, slot].float(), 0.0).permute(0, 2, 1, 3)
            for c in (s["cache_k"], s["cache_v"]))                                                # [B, G, L, D]
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


def _pick(s):
    x = s["logits"].float()
    R, V = x.shape
    at = torch.arange(s["history"].shape[1], device=DEV)
    there = at < s["lengths"][:, None]
    one = torch.ones((), device=DEV)
    ids = torch.where(there, s["history"], V).long()
    seen = torch.zeros(R, V + 1, device=DEV).scatter_(1, ids, one.expand(ids.shape))[:, :V] > 0
    ids = torch.where(there & (at >= s["prompts"][:, None]), s["history"], V).long()
    count = torch.zeros(R, V + 1, device=DEV).scatter_add_(1, ids, one.expand(ids.shape))[:, :V]
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count
    x = torch.where(count > 0, x - s["presence"][:, None], x)
    if s["bias_ids"] is not None:
        ids = torch.where(s["bias_ids"] >= 0, s["bias_ids"], V).long()
        x = x + torch.zeros(R, V + 1, device=DEV).scatter_(1, ids, s["bias_values"])[:, :V]
    t = s["temperature"][:, None]
    x = torch.where(t > 0, x / torch.where(t > 0, t, 1.0), x)
    if s["allowed"] is not None:
        v = torch.arange(V, device=DEV)
        x = torch.where((s["allowed"][:, v // 32] >> (v % 32)) & 1 > 0, x, -INF)
    y = x if s["noise"] is None else torch.where(t > 0, x + s["noise"], x)
    token = y.argmax(1)
    m = x.amax(1)
    some = m > -INF
    logprob = x.gather(1, token[:, None])[:, 0] - m - torch.log(torch.exp(x - m[:, None]).sum(1))
    logprob = torch.where(some, logprob, -INF)
    return torch.where(some, token, -1).to(torch.int32), logprob, x.to(s["logits"].dtype) if s["case"]["processed"] else None


# ------------------------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if not own:
        return {"append": _append, "attend": _attend, "pick": _pick}[op](s)
    from cme213_final_project_b200 import ops
    if op == "append":
        ops.cache_append(s["k"], s["v"], s["cache_k"], s["cache_v"], s["pages"], s["offsets"], s["lengths"])
        return s["cache_k"], s["cache_v"]
    if op == "attend":
        return ops.paged_attention(s["q"], s["cache_k"], s["cache_v"], s["pages"], s["offsets"], s["lengths"])
    return ops.next_token(s["logits"], history=s["history"], lengths=s["lengths"], prompts=s["prompts"], repetition=s["repetition"],
                          presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                          temperature=s["temperature"], allowed=s["allowed"], noise=s["noise"], processed=s["case"]["processed"])


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "pick":
        n = case["rows"] * case["vocab"]
        moved = n * e * (2 if case["processed"] else 1) + 4 * n * bool(case["noise"]) + n / 8 * bool(case["mask"])
        return {"bytes": moved + case["rows"] * (2 * case["history"] + 8 * case["biases"] + 32), "flops": 6 * n}
    pairs, H, G, D, P = _lengths(case), case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    new, length = sum(n for n, _ in pairs), sum(l for _, l in pairs)
    kept = 1 - 1 / case["drop_every"] if case["drop_every"] else 1
    tables = 4 * (length / P + 2 * len(pairs))
    if case["op"] == "append":
        return {"bytes": 4 * new * G * D * e * kept + tables, "flops": 0}
    visible = sum(n * (l - n) + n * (n + 1) / 2 for n, l in pairs)
    return {"bytes": 2 * length * G * D * e * kept + new * H * (2 * D * e + 4) + tables, "flops": 4 * D * H * visible * kept}


# ------------------------------------------------------------------------------------------------------------------
# The definitions, in 64 bits, sequence by sequence and row by row
# ------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return None                                       # a copy: held to be equal as it is
    if case["op"] == "attend":
        (N, H, D), P, G = s["q"].shape, case["page"], case["kv_heads"]
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
                k = s["cache_k"][page, h * G // H, where % P].double()
                v = s["cache_v"][page, h * G // H, where % P].double()
                x = (s["q"][lo:hi, h].double() @ k.T) / math.sqrt(D)
                x[hidden] = -INF
                lse[lo:hi, h] = torch.logsumexp(x, 1)
                out[lo:hi, h] = torch.softmax(x, 1).nan_to_num(0.0) @ v
        return out, lse
    rows, V = s["logits"].shape
    lengths, prompts = s["lengths"].tolist(), s["prompts"].tolist()
    x = s["logits"].double()
    for r in range(rows):
        told = s["history"][r, :lengths[r]].long()
        seen = torch.bincount(told, minlength=V) > 0
        made = torch.bincount(told[prompts[r]:], minlength=V).double()
        rep = s["repetition"][r].double()
        x[r] = torch.where(seen, torch.where(x[r] > 0, x[r] / rep, x[r] * rep), x[r])
        x[r] -= s["frequency"][r].double() * made + s["presence"][r].double() * (made > 0)
        if s["bias_ids"] is not None:
            ids = s["bias_ids"][r].long()
            x[r].index_add_(0, ids[ids >= 0], s["bias_values"][r].double()[ids >= 0])
        t = s["temperature"][r].double()
        x[r] /= torch.where(t > 0, t, torch.ones_like(t))
        if s["allowed"] is not None:
            bits = (s["allowed"][r][:, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
            x[r].masked_fill_(bits.flatten()[:V] == 0, -INF)
    y = x
    if s["noise"] is not None:
        y = torch.where(s["temperature"][:, None] > 0, x + s["noise"].double(), x)
    best = y.max(1).indices
    logprob = torch.log_softmax(x, 1).gather(1, best[:, None])[:, 0]
    logprob = torch.where(torch.isinf(x).all(1), -INF, logprob)
    return None, logprob, x if case["processed"] else None
