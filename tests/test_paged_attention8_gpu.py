"""A paged cache of 8-bit integers: what is written to it, number by number, and attention over it against a plain 64-bit implementation.

Written numbers are defined by their roundings in 32 bits and are held to be equal.  Tolerances of attention, element by element; p is the
softmax, A = p |v|, S = scale * max sum |q k|:
* integers and bf16 queries are exact in fp16 (times a power of two) and 32 bits, so a score is off by its sum's roundings, below 3e-6 S (as for
  fp32 queries), three factors, 2^-22, and the exponential, 1e-6: p by 2 * (3e-6 S + 2e-6).  bf16: probabilities are rounded to fp16 (2^-11)
  and the result to bf16 (2^-8): |error| <= 2^-11 A + 2^-8 |out| + 2 (3e-6 S + 2e-6) A.
* fp32: queries and probabilities in two fp16 parts lose 2^-22 each, 5e-7 S and 2.4e-7 A; the sums over 32 keys and over all of them 4e-6 A.
* A probability times 2^15 sv / (the largest sv of its 32 keys) that is below fp16's normal numbers is off by half of the smallest one, 2^-25, however
  small it is (one below 2^-40 vanishes).  Times that largest sv, 2^-15 and |integer| <= 128, over l >= 1 (the largest
  probability is 1): 2^-33 of the largest sv for each key, whatever A is.  Proof that a bound without it cannot hold: where all keys with
  p > 2^-40 have sv = 0, A is as small as 2^-40 of the others' |v|, and the result 0.  On tcgen05 (bf16, more than 16 rows) the unit is the largest sv
  of a CTA's first keys, with 2^7: 2^-25 of the sequence's largest sv for each key.
* log-sum-exp: the error of a score, 2^-21 for its sum, 2^-23 |lse|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops

BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8
SINGLES = [(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (1, 129), (1, 700)]
CHUNKS = [(1, 1), (5, 5), (17, 130), (64, 64), (130, 300), (0, 77), (33, 33), (200, 457)]


def make(pairs, heads, kv_heads, D, page, block, dtype, seed=0, drop=0, token_major=False, spread=1.0, q_scale=1.0):
    """(arguments, scales as keywords) for (new tokens, length) pairs.  Integers that no sequence reaches are anything, scales of such blocks NaN.
    ``spread``: of the logarithm of the scales; some are zero."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-max(l, 0) // page) for _, l in pairs]
    total, width, nb = sum(counts) + 3, max(counts + [1]) + 1, page // block
    free = torch.randperm(total, generator=g)
    table = torch.full((len(pairs), width), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = free[at:at + c]
        at += c
    used = torch.zeros(total, nb, dtype=torch.bool)
    for b, (_, l) in enumerate(pairs):
        for t in range(0, l, block):
            used[table[b, t // page], t % page // block] = True
    if drop:
        for b, c in enumerate(counts):
            table[b, :c][(torch.arange(c) + b) % drop == 0] = -1
    shape = (total, page, kv_heads, D) if token_major else (total, kv_heads, page, D)
    caches, scales = [], []
    for i in range(2):
        c = torch.randint(-128, 128, shape, generator=g).to(I8).cuda()
        caches.append(c.transpose(1, 2) if token_major else c)
        s = 0.02 * torch.exp(spread * torch.randn(total, kv_heads, nb, generator=g))
        s[torch.rand(s.shape, generator=g) < 0.05] = 0.0
        s[~used[:, None].expand(s.shape)] = math.nan
        scales.append(s.cuda())
    N = sum(n for n, _ in pairs)
    qkv = (q_scale * torch.randn(N, (heads + 2 * kv_heads) * D, generator=g)).to(dtype).cuda()
    q = qkv[:, :heads * D].view(N, heads, D)
    offsets = torch.tensor([sum(n for n, _ in pairs[:b]) for b in range(len(pairs) + 1)], dtype=torch.int32).cuda()
    lengths = torch.tensor([l for _, l in pairs], dtype=torch.int32).cuda()
    return (q, caches[0], caches[1], table.cuda(), offsets, lengths), dict(k_scales=scales[0], v_scales=scales[1])


def values(cache, scales):
    """The numbers that a cache stands for, in 64 bits, on the host."""
    return cache.cpu().double() * scales.cpu().double().repeat_interleave(cache.shape[2] // scales.shape[2], 2)[..., None]


def reference(args, scales, scale=None, max_len=None):
    """(out, lse, A, S, least) in 64 bits; least: 2^-33 of the largest scale of values among 32 keys, for each key, or 2^-25 of the largest."""
    q, ck, cv, pages, offsets, lengths = args
    N, H, D = q.shape
    KV, page = ck.shape[1], ck.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out, big = torch.zeros(N, H, D, dtype=torch.float64), torch.zeros(N, H, D, dtype=torch.float64)
    lse, S = torch.full((N, H), -math.inf, dtype=torch.float64), torch.zeros(N, H, dtype=torch.float64)
    least = torch.zeros(N, H, dtype=torch.float64)
    sv = scales["v_scales"].cpu().double().nan_to_num(0.0)
    q_dtype = q.dtype
    q, pages = q.double().cpu(), pages.cpu()
    ck, cv = values(ck, scales["k_scales"]), values(cv, scales["v_scales"])
    offs = offsets.tolist()
    for b, length in enumerate(lengths.tolist()):
        lo, hi = offs[b], offs[b + 1]
        end = min(length, pages.shape[1] * page if max_len is None else max_len)
        keys = [t for t in range(end) if 0 <= pages[b, t // page] < ck.shape[0]]
        if not keys or hi == lo:
            continue
        t = torch.tensor(keys)
        pg, slot = pages[b].long()[t // page], t % page
        seen = t[None, :] <= (length - (hi - lo) + torch.arange(hi - lo))[:, None]
        for h in range(H):
            k, v = (c[pg, h * KV // H, slot] for c in (ck, cv))
            k, v = (torch.where(seen.any(0)[:, None], c, 0.0) for c in (k, v))
            x = (q[lo:hi, h] @ k.T) * scale
            x[~seen] = -math.inf
            some = seen.any(1)
            l = torch.logsumexp(x, 1)
            p = torch.exp(x - torch.where(some, l, 0.0)[:, None])
            out[lo:hi, h], big[lo:hi, h], lse[lo:hi, h] = p @ v, p @ v.abs(), l
            S[lo:hi, h] = ((q[lo:hi, h].abs() @ k.abs().T) * scale * seen).amax(1)
            groups = torch.zeros(-(-end // 32), dtype=torch.float64).index_reduce_(0, t // 32, sv[pg, h * KV // H, slot // (page // sv.shape[2])], "amax")
            few = q_dtype == F32 or (hi - lo) * H // KV <= 16 and N * H // KV <= 16 * len(offs)
            least[lo:hi, h] = 2.0 ** -33 * 32 * groups.sum() if few else 2.0 ** -25 * len(keys) * groups.max()
    return out, lse, big, S, least


def check(args, scales, got, **kw):
    q = args[0]
    out, lse = (x.cpu() for x in got)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == F32 and lse.shape == q.shape[:2]
    want, wlse, big, S, least = reference(args, scales, **kw)
    p = 2 * (3e-6 * S + 2e-6)[:, :, None]
    tol = (2 ** -11 * 1.01 + p) * big + 2 ** -8 * want.abs() if q.dtype == BF16 else (p + 2 * 5e-7 * S[:, :, None] + 5e-6) * big
    tol = tol + least[:, :, None]
    none = torch.isinf(wlse)
    assert torch.equal(torch.isinf(lse), none) and bool((lse[none] < 0).all())
    assert bool((out[none] == 0).all())
    assert bool(((out.double() - want).abs() <= tol).all()), ((out.double() - want).abs() - tol).max()
    assert bool(((lse.double() - wlse).abs()[~none] <= (1e-5 + 4e-6 * S + 1e-6 * wlse.abs())[~none]).all())
    assert ops.attention_check_status() == 0


LAYOUTS = [(2, 2, 16, 16), (6, 2, 8, 8), (8, 1, 48, 24), (4, 4, 128, 64)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,page,block", LAYOUTS)
def test_single_tokens(dtype, D, heads, kv_heads, page, block):
    args, scales = make(SINGLES, heads, kv_heads, D, page, block, dtype)
    check(args, scales, ops.paged_attention(*args, **scales))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,page,block", LAYOUTS)
def test_chunks(dtype, D, heads, kv_heads, page, block):
    args, scales = make(CHUNKS, heads, kv_heads, D, page, block, dtype)
    check(args, scales, ops.paged_attention(*args, **scales))


@pytest.mark.parametrize("dtype,backend", [(BF16, "single"), (BF16, "rows"), (BF16, "tc"), (F32, "single"), (F32, "rows")])
@pytest.mark.parametrize("splits", [1, 2, 3, 8, 13, -1, -2, -7])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("pairs", [SINGLES, CHUNKS])
def test_parts_of_the_keys(dtype, backend, splits, D, pairs):
    args, scales = make(pairs, 4, 2, D, 16, 8, dtype, seed=1)
    check(args, scales, ops.paged_attention(*args, **scales, backend=backend, splits=splits))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pairs", [SINGLES, CHUNKS])
@pytest.mark.parametrize("drop", [1, 2, 3])
@pytest.mark.parametrize("page", [8, 64])
def test_pages_that_are_not_there(dtype, pairs, drop, page):
    args, scales = make(pairs, 4, 2, 64, page, 8, dtype, seed=3, drop=drop)          # drop = 1: no page at all
    check(args, scales, ops.paged_attention(*args, **scales))
    for other in (-1, args[1].shape[0], 2 ** 31 - 1, -2 ** 31):
        table = torch.where(args[3] < 0, other, args[3])
        check(args[:3] + (table,) + args[4:], scales, ops.paged_attention(*args[:3], table, *args[4:], **scales))


@pytest.mark.parametrize("dtype,backend", [(BF16, "single"), (BF16, "rows"), (F32, "single"), (F32, "rows"), (BF16, "tc")])
def test_rows_without_keys(dtype, backend):
    args, scales = make([(1, 1), (3, 3), (20, 20), (2, 0), (1, 0)], 4, 2, 64, 16, 16, dtype)
    args = args[:5] + (torch.tensor([1, 2, 5, 0, 0], dtype=torch.int32).cuda(),)
    check(args, scales, ops.paged_attention(*args, **scales, backend=backend))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pairs", [SINGLES, CHUNKS])
@pytest.mark.parametrize("q_scale", [1e-30, 1e-4, 1.0])
def test_scales_far_apart(dtype, pairs, q_scale):
    """Scales of neighbouring blocks differ by e^10 and more, queries are tiny or not."""
    args, scales = make(pairs, 4, 2, 64, 16, 8, dtype, seed=5, spread=4.0, q_scale=q_scale)
    check(args, scales, ops.paged_attention(*args, **scales, scale=1e-2), scale=1e-2)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pairs", [SINGLES, CHUNKS])
@pytest.mark.parametrize("max_len", [0, 1, 100, 10 ** 6])
def test_a_length_at_the_most(dtype, pairs, max_len):
    args, scales = make([(n, l) for n, l in pairs if l - n < max_len or max_len == 0], 4, 2, 64, 16, 16, dtype, seed=6)
    if len(args[5]) and max_len:
        check(args, scales, ops.paged_attention(*args, **scales, max_len=max_len), max_len=min(max_len, args[3].shape[1] * 16))
    else:
        out, lse = ops.paged_attention(*args, **scales, max_len=0)
        assert not bool(out.any()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("dtype,backend", [(BF16, "auto"), (BF16, "single"), (BF16, "rows"), (BF16, "tc"), (F32, "auto"), (F32, "single"), (F32, "rows")])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("which", ["k_scales", "v_scales"])
@pytest.mark.parametrize("splits", [0, 2])
def test_what_is_no_number_behind_a_row(dtype, backend, D, which, splits):
    """A block of new tokens is NaN: rows that see some of it are, those before it, which share its tiles, are as they were."""
    pairs = [(2, 9), (16, 24), (64, 64), (130, 300), (40, 201), (3, 17)]
    args, scales = make(pairs, 4, 2, D, 16, 8, dtype, seed=11)
    clean = ops.paged_attention(*args, **scales, backend=backend, splits=splits)
    table, bad, rows = args[3].cpu(), dict(scales), []
    bad[which] = bad[which].clone()
    for b, (n, length) in enumerate(pairs):
        at = (length - 1 - (n // 3 if n > 16 else 0)) // 8 * 8
        bad[which][int(table[b, at // 16]), :, at % 16 // 8] = math.nan
        rows += [length - n + i >= at for i in range(n)]
    sees = torch.tensor(rows).cuda()
    assert bool(sees.any()) and not bool(sees.all())
    out, lse = ops.paged_attention(*args, **bad, backend=backend, splits=splits)
    assert bool(out[sees].isnan().all()) and bool(out[~sees].isfinite().all())
    check(args, scales, (torch.where(sees[:, None, None], clean[0], out), torch.where(sees[:, None], clean[1], lse)))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_other_strides_and_scales_of_them(dtype):
    args, scales = make(SINGLES + CHUNKS, 4, 2, 64, 32, 16, dtype, seed=7, token_major=True)
    wide = {n: torch.full((s.shape[0], 5, s.shape[1], s.shape[2] + 3), math.nan, device="cuda")[:, 2, :, 1:-2].copy_(s) for n, s in scales.items()}
    check(args, scales, ops.paged_attention(*args, **wide))


def test_equal_calls_give_equal_bits_also_as_a_graph():
    args, scales = make(SINGLES + CHUNKS, 4, 2, 64, 16, 16, BF16, seed=8)
    a, b = ops.paged_attention(*args, **scales), ops.paged_attention(*args, **scales)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = ops.paged_attention(*args, **scales)
    for _ in range(2):
        graph.replay()
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


# ----------------------------------------------------------------------------------------------------------------------
# What is written
# ----------------------------------------------------------------------------------------------------------------------
def written(x, cache, scales, pages, offsets, lengths):
    """New rows into cache and scales, token block by token block, in 32 bits on the host."""
    cache, scales, pages, x = cache.cpu().clone(), scales.cpu().clone(), pages.cpu(), x.cpu().float()
    page, block = cache.shape[2], cache.shape[2] // scales.shape[2]
    one = torch.ones((), dtype=F32)
    for b, length in enumerate(lengths.tolist()):
        lo, n = int(offsets[b]), int(offsets[b + 1] - offsets[b])
        at, end = max(0, length - n), min(length, pages.shape[1] * page)
        while at < end:
            to = min(end, (at // block + 1) * block)
            pg, slot = int(pages[b, at // page]), at % page
            if 0 <= pg < cache.shape[0]:
                rows = x[lo + at - (length - n):lo + to - (length - n)]
                for h in range(cache.shape[1]):
                    top = rows[:, h].abs().amax() * (one / 127.0)
                    held = slot % block
                    old = scales[pg, h, slot // block] if held else torch.zeros(())
                    new = old if old > top else top
                    new = torch.zeros(()) if new < 2.0 ** -100 else new
                    if held and new != old:
                        q = cache[pg, h, slot - held:slot].float()
                        cache[pg, h, slot - held:slot] = torch.round(q * (old / new)).to(I8)
                    inverse = one / new if new > 0 else torch.zeros(())
                    cache[pg, h, slot:slot + to - at] = torch.round(rows[:, h] * inverse).to(I8)
                    scales[pg, h, slot // block] = new
            at = to
    return cache, scales


def empty(pages, kv_heads, page, D, block, token_major=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    shape = (pages, page, kv_heads, D) if token_major else (pages, kv_heads, page, D)
    cache = torch.randint(-128, 128, shape, generator=g).to(I8).cuda()
    scales = torch.full((pages, kv_heads, page // block), math.nan).cuda()
    return (cache.transpose(1, 2) if token_major else cache), scales


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,kv_heads,page,block,token_major", [(64, 12, 16, 16, False), (128, 3, 8, 8, True), (32, 1, 48, 24, False),
                                                               (128, 5, 128, 128, False), (64, 2, 64, 32, True)])
@pytest.mark.parametrize("seqs", [1, 9, 200])
def test_append_call_after_call(dtype, D, kv_heads, page, block, token_major, seqs):
    """Sequences grow in calls of their own numbers of tokens, whose sizes grow and fall; some pages are not there."""
    g = torch.Generator().manual_seed(seqs)
    columns = 2 if seqs > 50 else 4
    pages = torch.randperm(seqs * columns, generator=g).view(seqs, columns).to(torch.int32)
    pages[0, 1] = -1
    pages = pages.cuda()
    (ck, ks), (cv, vs) = (empty(seqs * columns, kv_heads, page, D, block, token_major, s) for s in (0, 1))
    lengths = torch.zeros(seqs, dtype=torch.int64)
    for call in range(3):
        new = torch.randint(0, 1 + (3 if call == 1 else page * columns // 2), (seqs,), generator=g)
        new = torch.minimum(new, page * columns - lengths)
        lengths += new
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(torch.int32).cuda()
        N = int(new.sum())
        rows = torch.randn(N, 2 * kv_heads * D, generator=g) * torch.exp(2 * torch.randn(N, 1, generator=g))
        rows = rows.to(dtype).cuda()
        rows[N // 2:N // 2 + 3] = 0
        k, v = rows[:, :kv_heads * D].view(N, kv_heads, D), rows[:, kv_heads * D:].view(N, kv_heads, D)
        device_lengths = lengths.to(torch.int32).cuda()
        want = written(k, ck, ks, pages, offsets, device_lengths) + written(v, cv, vs, pages, offsets, device_lengths)
        ops.cache_append(k, v, ck, cv, pages, offsets, device_lengths, k_scales=ks, v_scales=vs)
        for got, w in zip((ck, ks, cv, vs), want):
            got = got.cpu()
            assert torch.equal(got.nan_to_num(7.0) if got.is_floating_point() else got, w.nan_to_num(7.0) if w.is_floating_point() else w)


def test_append_of_single_tokens_is_near_the_numbers():
    """A token at a time: a number is off by half of its scale, and half of every smaller one that its block had before."""
    g = torch.Generator().manual_seed(3)
    (ck, ks), (cv, vs) = empty(4, 2, 16, 64, 16), empty(4, 2, 16, 64, 16)
    pages = torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda()
    x = (torch.randn(40, 2, 64, generator=g) * torch.linspace(1, 3, 40)[:, None, None]).cuda()
    off = torch.tensor([0, 1], dtype=torch.int32).cuda()
    allowed = torch.zeros(4, 2, 1)
    for t in range(40):
        before = ks.cpu().clone()
        ops.cache_append(x[t:t + 1], 2 * x[t:t + 1], ck, cv, pages, off, torch.tensor([t + 1], dtype=torch.int32).cuda(), k_scales=ks, v_scales=vs)
        pg = int(pages[0, t // 16])
        grown = ks.cpu()[pg] != before[pg]
        allowed[pg] = torch.where(grown, (allowed[pg] if t % 16 else 0.0) + 0.5 * ks.cpu()[pg], allowed[pg])
    got, got2 = values(ck, ks), values(cv, vs)
    for t in range(40):
        pg = int(pages[0, t // 16])
        bound = allowed[pg] * (1 + 1e-5)
        assert bool(((got[pg, :, t % 16] - x[t].cpu()).abs() <= bound).all())
        assert bool(((got2[pg, :, t % 16] - 2 * x[t].cpu()).abs() <= 2 * bound).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_append_of_what_is_not_finite_or_tiny(dtype):
    (ck, ks), (cv, vs) = empty(2, 2, 16, 64, 8), empty(2, 2, 16, 64, 8)
    pages = torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    x = torch.ones(24, 2, 64).to(dtype)
    x[3, 0, 5] = math.nan
    x[9, 1, 0] = math.inf
    x[16:] = 1e-32
    x = x.cuda()
    ops.cache_append(x, x, ck, cv, pages, torch.tensor([0, 24], dtype=torch.int32).cuda(), torch.tensor([24], dtype=torch.int32).cuda(), k_scales=ks,
                     v_scales=vs)
    got = values(ck, ks)
    assert bool(got[1, 0, :8].isnan().all()) and bool((got[1, 1, :8] - 1).abs().max() < 1e-6)
    assert bool(got[1, 1, 8:].isnan().all()) and bool((got[1, 0, 8:] - 1).abs().max() < 1e-6)
    assert bool((got[0, :, :8] == 0).all()) and bool((ks[0, :, 0] == 0).all())
    # a block begun anew forgets it
    y = torch.full((8, 2, 64), 2.0, dtype=dtype).cuda()
    ops.cache_append(y, y, ck, cv, pages, torch.tensor([0, 8], dtype=torch.int32).cuda(), torch.tensor([8], dtype=torch.int32).cuda(), k_scales=ks, v_scales=vs)
    assert bool((values(ck, ks)[1, :, :8] - 2).abs().max() < 1e-6)


def test_append_drops_what_has_no_place():
    (ck, ks), (cv, vs) = empty(4, 2, 8, 32, 8), empty(4, 2, 8, 32, 8)
    was = ck.clone()
    k = torch.ones(6, 2, 32, device="cuda")
    pages = torch.tensor([[1], [3]], dtype=torch.int32).cuda()
    offsets = torch.tensor([0, 3, 6], dtype=torch.int32).cuda()
    ops.cache_append(k, 2 * k, ck, cv, pages, offsets, torch.tensor([1, 10], dtype=torch.int32).cuda(), k_scales=ks, v_scales=vs)
    # one token of the first sequence has a position, one of the second lies inside its table, in a block whose scale nobody made
    assert bool((ck[1, :, 0] == 127).all()) and torch.equal(ck[1, :, 1:], was[1, :, 1:]) and torch.equal(ck[[0, 2]], was[[0, 2]])
    assert bool(ks[[0, 2]].isnan().all()) and bool((values(cv, vs)[1, :, 0] - 2).abs().max() < 1e-6)


def test_append_then_attention():
    """Prompts in two calls, then tokens one by one, as a run does, against attention over what the cache stands for."""
    g = torch.Generator().manual_seed(11)
    (ck, ks), (cv, vs) = empty(24, 2, 16, 64, 16), empty(24, 2, 16, 64, 16)
    scales = dict(k_scales=ks, v_scales=vs)
    pages = torch.randperm(24, generator=g).view(2, 12).to(torch.int32).cuda()
    length = [0, 0]
    for new in ([40, 3], [17, 90], [1, 1], [1, 1], [0, 1]):
        length = [a + b for a, b in zip(length, new)]
        N = sum(new)
        qkv = torch.randn(N, 8 * 64, generator=g).to(BF16).cuda()
        q, k, v = qkv[:, :256].view(N, 4, 64), qkv[:, 256:384].view(N, 2, 64), qkv[:, 384:].view(N, 2, 64)
        rest = (pages, torch.tensor([0, new[0], N], dtype=torch.int32).cuda(), torch.tensor(length, dtype=torch.int32).cuda())
        ops.cache_append(k, v, ck, cv, *rest, **scales)
        check((q, ck, cv, *rest), scales, ops.paged_attention(q, ck, cv, *rest, **scales))


def test_refusals():
    (q, ck, cv, pages, offsets, lengths), scales = make([(2, 20)], 4, 2, 64, 16, 8, BF16)
    full = dict(q=q, cache_k=ck, cache_v=cv, pages=pages, offsets=offsets, lengths=lengths, **scales)
    call = lambda **kw: ops.paged_attention(**{**full, **kw})
    s = scales["k_scales"]
    bad = [dict(k_scales=None), dict(v_scales=None), dict(k_scales=None, v_scales=None), dict(k_scales=s.double()), dict(k_scales=s.cpu()),
           dict(k_scales=s[:, :1]), dict(k_scales=s[:-1]), dict(k_scales=s[:, :, :1]), dict(k_scales=s[0]), dict(cache_k=ck.float(), cache_v=cv.float()),
           dict(cache_k=ck.to(torch.uint8), cache_v=cv.to(torch.uint8)), dict(q=q.half()), dict(q=q[:, :3]),
           dict(k_scales=s.repeat(1, 1, 2), v_scales=s.repeat(1, 1, 2)), dict(k_scales=s.repeat(1, 1, 5)[..., :3], v_scales=s.repeat(1, 1, 5)[..., :3]),
           dict(k_scales=s[..., :0], v_scales=s[..., :0]), dict(cache_k=ck[..., 8:40], cache_v=cv[..., 8:40], q=q[..., :32]), dict(scale=0.0)]
    for kw in bad:
        with pytest.raises(ops.NativeError):
            call(**kw)
    with pytest.raises(ops.NativeError):
        call(q=q.float(), backend="tc")
    k = torch.zeros(2, 2, 64, dtype=BF16, device="cuda")
    rest = (pages, offsets, lengths)
    for kk, vv, kw in ((k, k.float(), scales), (k, k, {}), (k, k, dict(k_scales=s)), (k[:, :1], k[:, :1], scales), (k.half(), k.half(), scales)):
        with pytest.raises(ops.NativeError):
            ops.cache_append(kk, vv, ck, cv, *rest, **kw)
    with pytest.raises(ops.NativeError):
        ops.cache_append(k, k, k.new_zeros(ck.shape), k.new_zeros(cv.shape), *rest, **scales)
    call()                                                                 # and as it should be


# ----------------------------------------------------------------------------------------------------------------------
# Many sequences, streams and graphs
# ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,page,block", [(64, 16, 16), (64, 8, 8), (32, 16, 8), (128, 32, 32), (128, 8, 8)])
@pytest.mark.parametrize("heads,kv_heads,new", [(4, 4, 1), (16, 1, 1), (5, 1, 3), (24, 2, 2)])
def test_many_sequences(dtype, D, page, block, heads, kv_heads, new):
    """Items of many lengths in one stream of tiles: pages in boxes and in copies, up to 8 and up to 16 rows a tile, some sequences without new tokens."""
    pairs = [(new * (b % 7 != 3), max(new, (b * 37) % 300 + 1)) for b in range(90)]
    args, scales = make(pairs, heads, kv_heads, D, page, block, dtype, seed=9, drop=5)
    check(args, scales, ops.paged_attention(*args, **scales, backend="single", splits=-1))
    check(args, scales, ops.paged_attention(*args, **scales))


def test_calls_on_two_streams_and_a_captured_append():
    args, scales = make(SINGLES + CHUNKS, 4, 2, 64, 16, 16, BF16, seed=10)
    want = ops.paged_attention(*args, **scales)
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for s in side:
            with torch.cuda.stream(s):
                got.append(ops.paged_attention(*args, **scales))
    torch.cuda.synchronize()
    assert all(torch.equal(g[0], want[0]) and torch.equal(g[1], want[1]) for g in got)
    (ck, ks), (cv, vs) = empty(4, 2, 16, 64, 16), empty(4, 2, 16, 64, 16)
    (dk, ls), (dv, ws) = empty(4, 2, 16, 64, 16), empty(4, 2, 16, 64, 16)
    pages, off = torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda()
    x, length = torch.randn(30, 1, 2, 64).cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    row = x[0].clone()
    ops.cache_append(row, row, dk, dv, pages, off, length, k_scales=ls, v_scales=ws)      # (length 0: nothing has a place)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        length.add_(1)
        ops.cache_append(row, row, ck, cv, pages, off, length, k_scales=ks, v_scales=vs)
    length.zero_()
    for t in range(30):
        row.copy_(x[t])
        graph.replay()
        ops.cache_append(x[t], x[t], dk, dv, pages, off, torch.tensor([t + 1], dtype=torch.int32).cuda(), k_scales=ls, v_scales=ws)
    assert torch.equal(values(ck, ks)[[2, 0]].nan_to_num(7.0)[:, :, :14], values(dk, ls)[[2, 0]].nan_to_num(7.0)[:, :, :14])
    assert torch.equal(values(cv, vs)[2], values(dv, ws)[2])
