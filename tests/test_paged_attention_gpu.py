"""Paged cache and attention over it against a plain 64-bit implementation, sequence by sequence.

Tolerances, element by element.  With p the softmax and A = p |v|:
* bf16 (8 bits, unit roundoff 2^-8): probabilities and the result are rounded by up to 2^-8 of themselves each, so |error| <= 2^-8 A +
  2^-8 |out|, both below 2^-8 A; products of bf16 numbers are exact in 32 bits and their sums cost 2^-24 an addition, below
  1 % of that: 2^-7 A * 1.02.
* fp32: a score is made from tf32 halves.  What the products leave out is below 2^-21 of them, and up to 16 additions a score cut up to
  2^-23 each: 3e-6 of S = scale * max sum |q k|, and exponent and exponential 1e-6 more, so p is off by 2 * (3e-6 S + 1e-6) at most, and
  the second product by 4e-6 of A.
* log-sum-exp: the error of a score (D 2^-24 S for bf16), 2^-21 for its sum, 2^-23 |lse|: 1e-5 + 1e-6 (S + |lse|), fp32 3e-6 S.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops

BF16, F32 = torch.bfloat16, torch.float32
BACKENDS = ["single", "rows", "tc"]
SINGLES = [(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (1, 129), (1, 700)]
CHUNKS = [(1, 1), (5, 5), (17, 130), (64, 64), (130, 300), (0, 77), (33, 33), (200, 457)]


def make(pairs, heads, kv_heads, D, page, dtype, seed=0, drop=0, token_major=False, spare=3):
    """Cache, tables and queries for (new tokens, length) pairs; what no sequence reaches is NaN."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-max(l, 0) // page) for _, l in pairs]
    total, width = sum(counts) + spare, max(counts + [1]) + 1
    free = torch.randperm(total, generator=g)
    table = torch.full((len(pairs), width), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = free[at:at + c]
        at += c
    used = torch.zeros(total, page, dtype=torch.bool)
    for b, (_, l) in enumerate(pairs):
        for t in range(l):
            used[table[b, t // page], t % page] = True
    if drop:
        for b, c in enumerate(counts):
            table[b, :c][(torch.arange(c) + b) % drop == 0] = -1
    shape = (total, page, kv_heads, D) if token_major else (total, kv_heads, page, D)
    caches = []
    for _ in range(2):
        c = torch.randn(*shape, generator=g).to(dtype).cuda()
        c = c.transpose(1, 2) if token_major else c
        c.masked_fill_(~used.cuda()[:, None, :, None], float("nan"))
        caches.append(c)
    N = sum(n for n, _ in pairs)
    qkv = torch.randn(N, (heads + 2 * kv_heads) * D, generator=g).to(dtype).cuda()
    q = qkv[:, :heads * D].view(N, heads, D)
    offsets = torch.tensor([sum(n for n, _ in pairs[:b]) for b in range(len(pairs) + 1)], dtype=torch.int32).cuda()
    lengths = torch.tensor([l for _, l in pairs], dtype=torch.int32).cuda()
    return q, caches[0], caches[1], table.cuda(), offsets, lengths


def reference(q, ck, cv, pages, offsets, lengths, scale=None):
    """(out, lse, A, S) in 64 bits."""
    N, H, D = q.shape
    KV, page = ck.shape[1], ck.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(N, H, D, dtype=torch.float64)
    big = torch.zeros(N, H, D, dtype=torch.float64)
    lse = torch.full((N, H), -math.inf, dtype=torch.float64)
    S = torch.zeros(N, H, dtype=torch.float64)
    q, ck, cv, pages = q.double().cpu(), ck.cpu(), cv.cpu(), pages.cpu()
    offs, lens = offsets.tolist(), lengths.tolist()
    for b, length in enumerate(lens):
        lo, hi = offs[b], offs[b + 1]
        length = min(length, pages.shape[1] * page)
        keys = [t for t in range(length) if 0 <= pages[b, t // page] < ck.shape[0]]
        if not keys or hi == lo:
            continue
        t = torch.tensor(keys)
        pg, slot = pages[b].long()[t // page], t % page
        seen = t[None, :] <= (length - (hi - lo) + torch.arange(hi - lo))[:, None]
        for h in range(H):
            k, v = (c[pg, h * KV // H, slot].double() for c in (ck, cv))
            x = (q[lo:hi, h] @ k.T) * scale
            x[~seen] = -math.inf
            some = seen.any(1)
            l = torch.logsumexp(x, 1)
            p = torch.exp(x - torch.where(some, l, 0.0)[:, None])
            out[lo:hi, h], big[lo:hi, h], lse[lo:hi, h] = p @ v, p @ v.abs(), l
            S[lo:hi, h] = ((q[lo:hi, h].abs() @ k.abs().T) * scale * seen).amax(1)
    return out, lse, big, S


def check(args, got, scale=None):
    q = args[0]
    out, lse = (x.cpu() for x in got)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == F32 and lse.shape == q.shape[:2]
    want, wlse, big, S = reference(*args, scale=scale)
    if q.dtype == BF16:
        tol, ltol = 2 ** -7 * 1.02 * big, 1e-5 + 1e-6 * (S + wlse.abs())
    else:
        tol, ltol = (2 * (3e-6 * S + 1e-6)[:, :, None] + 4e-6) * big, 1e-5 + 3e-6 * S + 1e-6 * wlse.abs()
    none = torch.isinf(wlse)
    assert torch.equal(torch.isinf(lse), none) and bool((lse[none] < 0).all())
    assert bool((out[none] == 0).all())
    assert bool(((out.double() - want).abs() <= tol).all()), ((out.double() - want).abs() - tol).max()
    assert bool(((lse.double() - wlse).abs()[~none] <= ltol[~none]).all())
    assert ops.attention_check_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,page", [(2, 2, 16), (6, 2, 8), (8, 1, 48), (4, 4, 128)])
def test_single_tokens(dtype, D, heads, kv_heads, page):
    args = make(SINGLES, heads, kv_heads, D, page, dtype)
    check(args, ops.paged_attention(*args))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,page", [(2, 2, 16), (6, 2, 8), (8, 1, 48), (4, 4, 128)])
def test_chunks(dtype, D, heads, kv_heads, page):
    args = make(CHUNKS, heads, kv_heads, D, page, dtype)
    check(args, ops.paged_attention(*args))


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("splits", [1, 2, 3, 8, 13, -1, -2, -7])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pairs", [SINGLES, CHUNKS])
def test_parts_of_the_keys(backend, splits, D, pairs):
    args = make(pairs, 4, 2, D, 16, BF16, seed=1)
    check(args, ops.paged_attention(*args, backend=backend, splits=splits))


@pytest.mark.parametrize("backend", ["single", "rows"])
@pytest.mark.parametrize("splits", [1, 4, -3])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_parts_of_the_keys_fp32(backend, splits, D):
    args = make(SINGLES + CHUNKS, 4, 2, D, 16, F32, seed=2)
    check(args, ops.paged_attention(*args, backend=backend, splits=splits))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pairs", [SINGLES, CHUNKS])
@pytest.mark.parametrize("drop", [1, 2, 3])
@pytest.mark.parametrize("page", [8, 64])
def test_pages_that_are_not_there(dtype, pairs, drop, page):
    args = make(pairs, 4, 2, 64, page, dtype, seed=3, drop=drop)          # drop = 1: no page at all
    check(args, ops.paged_attention(*args))
    for other in (-1, args[1].shape[0], 2 ** 31 - 1, -2 ** 31):           # any number outside the cache says so
        table = torch.where(args[3] < 0, other, args[3])
        check(args[:3] + (table,) + args[4:], ops.paged_attention(*args[:3], table, *args[4:]))


@pytest.mark.parametrize("backend", BACKENDS)
def test_rows_without_keys(backend):
    # more new tokens than the sequence is long: the first ones have no position and see nothing
    args = make([(1, 1), (3, 3), (20, 20), (2, 0), (1, 0)], 4, 2, 64, 16, BF16)
    lengths = torch.tensor([1, 2, 5, 0, 0], dtype=torch.int32).cuda()
    args = args[:5] + (lengths,)
    check(args, ops.paged_attention(*args, backend=backend))


@pytest.mark.parametrize("backend", BACKENDS)
def test_nothing_to_do(backend):
    args = make([(0, 5), (0, 0)], 4, 2, 64, 16, BF16)
    out, lse = ops.paged_attention(*args, backend=backend)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    q, ck, cv, pages, offsets, lengths = make([(2, 2)], 4, 2, 64, 16, BF16)
    out, lse = ops.paged_attention(q, ck[:0], cv[:0], pages, offsets, lengths, backend=backend)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    out, lse = ops.paged_attention(q, ck, cv, pages[:, :0], offsets, lengths, backend=backend)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("backend", BACKENDS)
def test_layouts(backend):
    """Cache with the slots outside of the heads, a table that is part of a wider one, a scale of one's own."""
    q, ck, cv, pages, offsets, lengths = make(SINGLES + CHUNKS, 6, 2, 64, 16, BF16, seed=4, token_major=True)
    wide = torch.full((pages.shape[0], pages.shape[1] + 5), 10 ** 6, dtype=torch.int32).cuda()
    wide[:, :pages.shape[1]] = pages
    args = (q, ck, cv, wide[:, :pages.shape[1]], offsets, lengths)
    check(args, ops.paged_attention(*args, scale=0.3, backend=backend), scale=0.3)


def test_lengths_are_cut_to_what_is_there():
    q, ck, cv, pages, offsets, lengths = make([(1, 40), (2, 33)], 2, 2, 64, 16, BF16)
    full = torch.arange(6, dtype=torch.int32).view(2, 3).cuda()
    ck, cv = torch.randn(8, 2, 16, 64).to(BF16).cuda(), torch.randn(8, 2, 16, 64).to(BF16).cuda()
    long = torch.full_like(lengths, 10 ** 9)
    args = (q, ck, cv, full, offsets, long)
    check(args, ops.paged_attention(*args))                                # 48 each
    cut = torch.tensor([20, 20], dtype=torch.int32).cuda()
    a, b = ops.paged_attention(*args, max_len=20), ops.paged_attention(q, ck, cv, full, offsets, cut)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("backend", BACKENDS)
def test_infinities_and_nan_of_one_sequence_stay_in_it(backend):
    args = list(make([(1, 70), (4, 90), (130, 200)], 2, 2, 64, 16, BF16, seed=5))
    clean = ops.paged_attention(*args, backend=backend)
    args[1], args[2] = args[1].clone(), args[2].clone()
    first = args[3][0, 0].long()
    args[1][first, 0, 3] = float("inf")
    args[2][first, 0, 5] = float("nan")
    out, lse = ops.paged_attention(*args, backend=backend)
    assert bool(torch.isnan(out[0, 0]).any())
    assert torch.equal(out[1:], clean[0][1:]) and torch.equal(lse[1:], clean[1][1:])
    assert torch.equal(out[0, 1], clean[0][0, 1])


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F32)])
def test_large_scores(D, dtype):
    q, *rest = make([(1, 300), (40, 300)], 2, 2, D, 16, dtype, seed=6)
    args = (q * 40, *rest)                                                 # one key takes all the weight
    check(args, ops.paged_attention(*args))


@pytest.mark.parametrize("backend", BACKENDS)
def test_cache_beyond_32_bits(backend):
    """Pages whose elements lie further than 2^32 into the cache."""
    page, KV, D = 64, 8, 128
    n = (1 << 32) // (page * KV * D) + 8
    ck, cv = (torch.empty(n, KV, page, D, dtype=BF16, device="cuda") for _ in range(2))
    pages = torch.tensor([[n - 1, 3, n - 5]], dtype=torch.int32).cuda()
    for c in (ck, cv):
        c[pages[0].long()] = torch.randn(3, KV, page, D, device="cuda").to(BF16)
    q = torch.randn(5, 16, D).to(BF16).cuda()
    k, v = (torch.randn(5, KV, D).to(BF16).cuda() for _ in range(2))
    offsets, lengths = torch.tensor([0, 5], dtype=torch.int32).cuda(), torch.tensor([170], dtype=torch.int32).cuda()
    ops.cache_append(k, v, ck, cv, pages, offsets, lengths)
    assert torch.equal(ck[n - 5, :, 37:42], k.transpose(0, 1)) and torch.equal(cv[n - 5, :, 37:42], v.transpose(0, 1))
    small = [c[pages[0].long()] for c in (ck, cv)]
    table = torch.arange(3, dtype=torch.int32).view(1, 3).cuda()
    got = ops.paged_attention(q, ck, cv, pages, offsets, lengths, backend=backend)
    check((q, *small, table, offsets, lengths), got)


@pytest.mark.parametrize("D,dtype", [(128, F32), (64, F32), (128, BF16), (64, BF16)])
@pytest.mark.parametrize("splits", [0, 1, 2, 8, -1])
def test_many_long_sequences(D, dtype, splits):
    """Enough keys that their tiles come out of memory in any order; two of the sequences against 64 bits."""
    seqs, page, KV = 16, 16, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    lengths = [2048 + 131 * b for b in range(seqs)]
    width = -(-lengths[-1] // page)
    table = torch.randperm(seqs * width, generator=g, device="cuda").to(torch.int32).view(seqs, width)
    ck, cv = (torch.randn(seqs * width, KV, page, D, generator=g, device="cuda", dtype=dtype) for _ in range(2))
    q = torch.randn(seqs, KV, D, generator=g, device="cuda", dtype=dtype)
    offsets = torch.arange(seqs + 1, dtype=torch.int32).cuda()
    lens = torch.tensor(lengths, dtype=torch.int32).cuda()
    for _ in range(3):
        out, lse = ops.paged_attention(q, ck, cv, table, offsets, lens, backend="single", splits=splits)
    for b in (1, 14):
        check((q[b:b + 1], ck, cv, table[b:b + 1], offsets[:2], lens[b:b + 1]), (out[b:b + 1], lse[b:b + 1]))


def test_another_stream_and_a_graph():
    args = make(SINGLES, 4, 2, 64, 16, BF16, seed=7)
    want = ops.paged_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.paged_attention(*args, splits=-4)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = ops.paged_attention(*args)
        graph.replay()
    torch.cuda.synchronize()
    check(args, got)
    assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, BF16), (128, F32)])
def test_the_same_bits_every_time(D, dtype):
    for pairs in (SINGLES, CHUNKS, [(700, 900)] * 3):
        args = make(pairs, 4, 2, D, 16, dtype, seed=8)
        for splits in (0, 1, -5):
            first = ops.paged_attention(*args, splits=splits)
            for _ in range(40):
                out, lse = ops.paged_attention(*args, splits=splits)
                assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


@pytest.mark.parametrize("heads,kv_heads,page", [(4, 4, 16), (6, 2, 8), (8, 1, 48), (3, 1, 128)])
@pytest.mark.parametrize("drop", [0, 3])
def test_heads_of_32_on_the_tensor_core_kernel(heads, kv_heads, page, drop):
    args = make(CHUNKS, heads, kv_heads, 32, page, BF16, seed=heads, drop=drop, token_major=kv_heads == 2)
    for splits in (0, 1, 3):
        check(args, ops.paged_attention(*args, backend="tc", splits=splits))
    many = make([(700, 900)] * 12, heads, kv_heads, 32, page, BF16, seed=heads)          # three CTAs an SM
    first = ops.paged_attention(*many, backend="tc", splits=1)
    check(many, first)
    for _ in range(20):
        assert all(torch.equal(x, y) for x, y in zip(first, ops.paged_attention(*many, backend="tc", splits=1)))


@pytest.mark.parametrize("D,dtype", [(32, BF16), (64, F32), (128, F32)])
@pytest.mark.parametrize("heads,kv_heads", [(15, 3), (3, 1), (14, 2), (130, 1), (65, 1)])
def test_tiles_in_the_order_of_their_keys(heads, kv_heads, D, dtype):
    """More tiles of rows than run at a time, whose ends lie inside a token's heads, or which are a part of one."""
    pairs = [(n * 16 * kv_heads // heads + 1, l) for n, l in ((130, 700), (0, 50), (70, 500), (170, 640), (1, 3), (100, 110), (160, 900), (7, 0))] * 4
    pairs = [(min(n, l) if l else n, l) for n, l in pairs]
    args = make(pairs, heads, kv_heads, D, 16, dtype, seed=heads)
    for splits in (1, 2):
        check(args, ops.paged_attention(*args, backend="rows", splits=splits))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_whose_maximum_rises_with_every_tile(D, dtype):
    """32 rows of every 128, a warp's, see scores that grow by 6.4 (9.2 in log2 units) from one 64 keys to the next, so that their sums are
    scaled down for every tile; the others' scores stay flat, and their warps could run ahead."""
    args = make([(500, 1500), (130, 700), (60, 900)], 4, 1, D, 16, dtype, seed=11)
    q, ck, cv, pages, offsets, lengths = args
    q.mul_(2 ** -7)
    q[..., 0] = 0
    rows = torch.arange(q.shape[0] * 4, device="cuda").view(-1, 4)
    for b in range(3):
        lo, hi = offsets[b].item(), offsets[b + 1].item()
        steep = (rows[lo:hi] - lo * 4) // 32 % 4 == 1
        q[lo:hi, :, 0][steep] = D ** 0.5 / 10
        for t in range(lengths[b].item()):
            ck[pages[b, t // 16].item(), :, t % 16, 0] = t
    for backend in (["tc"] if dtype == BF16 else []) + ["rows", "single", "auto"]:
        for splits in (0, 1):
            check(args, ops.paged_attention(*args, backend=backend, splits=splits))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,kv_heads,page,token_major", [(64, 12, 16, False), (128, 3, 8, True), (32, 1, 48, False), (128, 40, 16, False)])
@pytest.mark.parametrize("seqs", [1, 9, 70])
def test_append(dtype, D, kv_heads, page, token_major, seqs):
    pairs = [(b * 5 % 7, 3 + b * 11 % 60 + 6) for b in range(seqs)]
    q, ck, cv, pages, offsets, lengths = make(pairs, kv_heads, kv_heads, D, page, dtype, token_major=token_major)
    pages[0, :1] = -1                                                      # a page that is not there
    N = q.shape[0]
    new = torch.randn(N, 2 * kv_heads * D).to(dtype).cuda()
    k, v = new[:, :kv_heads * D].view(N, kv_heads, D), new[:, kv_heads * D:].view(N, kv_heads, D)
    want = [c.clone() for c in (ck, cv)]
    for b, (n, length) in enumerate(pairs):
        for i in range(n):
            pos, row = length - n + i, int(offsets[b]) + i
            pg = int(pages[b, pos // page])
            if pg >= 0:
                want[0][pg, :, pos % page], want[1][pg, :, pos % page] = k[row], v[row]
    ops.cache_append(k, v, ck, cv, pages, offsets, lengths)
    for c, w in zip((ck, cv), want):
        assert torch.equal(c.nan_to_num(7.0), w.nan_to_num(7.0))


def test_append_drops_what_has_no_place():
    ck, cv = torch.zeros(4, 2, 8, 32, device="cuda"), torch.zeros(4, 2, 8, 32, device="cuda")
    k = torch.ones(6, 2, 32, device="cuda")
    pages = torch.tensor([[1], [3]], dtype=torch.int32).cuda()
    offsets = torch.tensor([0, 3, 6], dtype=torch.int32).cuda()
    ops.cache_append(k, 2 * k, ck, cv, pages, offsets, torch.tensor([1, 10], dtype=torch.int32).cuda())
    assert float(ck[1].sum()) == 2 * 32 and float(ck[3].sum()) == 2 * 32 and float(ck.sum()) == 4 * 32 and float(cv.sum()) == 8 * 32


def test_refusals():
    q, ck, cv, pages, offsets, lengths = make([(2, 20)], 4, 2, 64, 16, BF16)
    call = lambda **kw: ops.paged_attention(**{**dict(q=q, cache_k=ck, cache_v=cv, pages=pages, offsets=offsets, lengths=lengths), **kw})
    bad = [dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[:, :, :32]), dict(q=q.cpu()), dict(q=q[0]), dict(cache_v=cv[:, :1]),
           dict(cache_k=ck.float(), cache_v=cv.float()), dict(pages=pages.long()), dict(offsets=offsets[:1]), dict(lengths=lengths.float()),
           dict(q=q.half(), cache_k=ck.half(), cache_v=cv.half()), dict(scale=-1.0), dict(scale=float("nan")), dict(max_len=-1),
           dict(cache_k=ck[:, :, :12], cache_v=cv[:, :, :12]), dict(cache_k=ck.transpose(2, 3), cache_v=cv.transpose(2, 3)),
           dict(q=torch.zeros(2, 4, 72, dtype=BF16, device="cuda")[:, :, 4:68]),
           dict(q=torch.zeros(2, 4, 68, dtype=BF16, device="cuda")[:, :, :64])]
    for kw in bad:
        with pytest.raises(ops.NativeError):
            call(**kw)
    f = [x.float() for x in (q, ck, cv)]
    with pytest.raises(ops.NativeError):
        call(q=f[0], cache_k=f[1], cache_v=f[2], backend="tc")
    with pytest.raises(KeyError):
        call(backend="other")
    with pytest.raises(TypeError):
        call(q=3)
    k = torch.zeros(2, 2, 64, dtype=BF16, device="cuda")
    for kk, vv in ((k, k.float()), (k[:, :1], k[:, :1]), (k, k[:1]), (k.float(), k.float())):
        with pytest.raises(ops.NativeError):
            ops.cache_append(kk, vv, ck, cv, pages, offsets, lengths)
    call()                                                                 # and as it should be
