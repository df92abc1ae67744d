"""The reordering of a paged cache for beams: tables, spare pages and copied slots are held to be equal to their definition."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops

BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8


def make(lengths, beams, layers, heads, slots, D, dtype, block=0, columns=None, seed=0, layout="plain"):
    g = torch.Generator().manual_seed(seed)
    B = len(lengths)
    full = [max(0, l) // slots for l in lengths]
    width = columns or max(full) + 2
    total = sum(full) + 2 * B * beams + 5
    free = torch.randperm(total, generator=g).to(torch.int32)
    table, at = torch.full((B, beams, width), -1, dtype=torch.int32), 0
    for b, f in enumerate(full):
        f = min(f, width)
        for i in range(beams):
            table[b, i, :f] = free[at:at + f].roll(i)
        at += f
        if f < width:
            table[b, :, f] = free[at:at + beams]
            at += beams
    spare = free[at:at + B * beams]
    parents = torch.randint(0, beams, (B, beams), generator=g).to(torch.int32)

    def cache():
        shape = (layers, total, slots, heads, D) if layout == "tokens" else (layers, total, heads, slots, D)
        x = torch.randint(-127, 128, shape, generator=g).to(dtype).cuda()
        return x.transpose(2, 3) if layout == "tokens" else x

    scales = {}
    if block:
        scales = {n: torch.rand(layers, total, heads, slots // block, generator=g).cuda() for n in ("k_scales", "v_scales")}
    return [cache(), cache(), table.view(-1, width).cuda(), spare.cuda(), parents.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()], scales


def reference(args, scales):
    k, v, pages, spare, parents, lengths = (x.cpu() for x in args)
    B, n = parents.shape
    slots, count = k.shape[3], k.shape[1]
    tensors = [x.clone() for x in (k, v)] + [s.cpu().clone() for s in scales.values()]
    was = [x.clone() for x in tensors]
    new, new_spare = pages.clone(), spare.clone()
    for b in range(B):
        length = max(0, int(lengths[b]))
        full = min(length // slots, pages.shape[1])
        rest = length % slots if full < pages.shape[1] else 0
        for i in range(n):
            p = int(parents[b, i])
            p = p if 0 <= p < n else i
            r, f = b * n + i, b * n + p
            new[r, :full] = pages[f, :full]
            if rest and p != i:
                src, to = int(pages[f, full]), int(spare[r])
                if not 0 <= src < count:
                    new[r, full] = src
                elif not 0 <= to < count:
                    new[r, full] = -1
                else:
                    new[r, full], new_spare[r] = to, pages[r, full]
                    for t, w in zip(tensors, was):
                        m = rest if t.dim() == 5 else -(-rest // (slots // t.shape[3]))
                        t[:, to, :, :m] = w[:, src, :, :m]
    return new, new_spare, tensors


def check(args, scales):
    want = reference(args, scales)
    got = ops.cache_reorder(*args, **scales)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    for t, w in zip((args[0], args[1], *scales.values()), want[2]):
        assert torch.equal(t.cpu(), w)
    return got


@pytest.mark.parametrize("dtype,block", [(BF16, 0), (F32, 0), (I8, 8), (I8, 16)])
@pytest.mark.parametrize("lengths,beams,layers,heads,slots,D", [([0], 4, 2, 2, 16, 64), ([1], 1, 1, 1, 16, 32), ([16, 17, 31, 32, 5], 4, 3, 5, 16, 64),
                                                               ([700], 16, 2, 3, 48, 128), ([9] * 70, 3, 1, 2, 16, 32), ([100, 33], 32, 24, 4, 64, 64)])
def test_sizes(dtype, block, lengths, beams, layers, heads, slots, D):
    args, scales = make(lengths, beams, layers, heads, slots, D, dtype, block)
    check(args, scales)


def test_step_after_step():
    """What a step gives is what the next one takes; lengths grow through the ends of pages."""
    args, scales = make([13], 5, 2, 2, 16, 32, I8, 8, columns=6)
    free = [p for p in range(args[0].shape[1]) if p not in set(args[2].cpu().flatten().tolist()) | set(args[3].tolist())]
    big = torch.zeros(2, 64, 2, 16, 32, dtype=I8, device="cuda")
    caches = [big.clone(), big.clone()]
    sc = {n: torch.rand(2, 64, 2, 2).cuda() for n in scales}
    pages = torch.arange(30, dtype=torch.int32).view(5, 6).cuda()
    spare = torch.arange(30, 35, dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(0)
    assert free is not None
    past = [[] for _ in range(5)]                                          # what each beam's tokens should be
    for length in range(1, 60):
        for i in range(5):                                                 # each beam writes its new token's slot
            past[i] = past[i] + [int(torch.randint(-127, 128, (1,), generator=g))]
            page = int(pages[i, (length - 1) // 16])
            for c in caches:
                c[:, page, :, (length - 1) % 16] = past[i][-1]
        parents = torch.randint(0, 5, (1, 5), generator=g).to(torch.int32)
        pages, spare = check([*caches, pages, spare, parents.cuda(), torch.tensor([length], dtype=torch.int32).cuda()], sc)
        past = [past[p] for p in parents[0].tolist()]
        for i in range(5):
            for t in range(0, length, 3):
                assert int(caches[0][0, int(pages[i, t // 16]), 0, t % 16, 0]) == past[i][t]
        tails = pages[:, length // 16:].flatten().tolist() + spare.tolist()
        assert len(set(tails)) == len(tails)                               # pages that are still written belong to one beam each


def test_odd_calls():
    args, scales = make([21, 37, 40], 4, 2, 3, 16, 64, BF16, seed=4)
    args[4][0] = torch.tensor([-1, 4, 2 ** 31 - 1, 0], dtype=torch.int32)  # no such beams: they keep their own
    args[4][1] = torch.tensor([1, 0, 3, 2], dtype=torch.int32)
    args[2][7, 2] = -1                                                     # a last page that is not there
    args[2][6, 2] = 10 ** 6
    args[3][4] = -1                                                        # no spare page
    check(args, scales)
    args, scales = make([21, 37, -5], 4, 2, 3, 16, 64, BF16, columns=2, seed=5)      # as long as the table, longer, and less than nothing
    check(args, scales)
    args, scales = make([21, 37], 4, 2, 3, 16, 64, F32, seed=6, layout="tokens")
    wide = torch.zeros(8, 9, dtype=torch.int32, device="cuda")
    wide[:, 1:1 + args[2].shape[1]] = args[2]
    args[2] = wide[:, 1:1 + args[2].shape[1]]
    check(args, scales)
    args, scales = make([5], 4, 2, 3, 16, 64, F32)
    got = ops.cache_reorder(args[0], args[1], args[2][:0], args[3][:0], args[4][:0], args[5][:0])
    assert got[0].shape == (0, args[2].shape[1]) and got[1].shape == (0,)


def test_captured():
    args, scales = make([21, 37], 4, 2, 3, 16, 64, BF16, seed=8)
    first = ops.cache_reorder(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.cache_reorder(*args)
    args[4].copy_(args[4].flip(1))
    want = reference(args, scales)
    graph.replay()
    assert torch.equal(held[0].cpu(), want[0]) and torch.equal(held[1].cpu(), want[1]) and torch.equal(args[0].cpu(), want[2][0])
    assert first[0].shape == held[0].shape


def test_refusals():
    (k, v, pages, spare, parents, lengths), _ = make([21, 37], 4, 2, 3, 16, 64, BF16)
    call = lambda **kw: ops.cache_reorder(**{**dict(cache_k=k, cache_v=v, pages=pages, spare=spare, parents=parents, lengths=lengths), **kw})
    s = torch.zeros(2, k.shape[1], 3, 2, device="cuda")
    bad = [dict(cache_k=k[0]), dict(cache_v=v[:1]), dict(cache_v=v[:, :-1]), dict(cache_v=v[:, :, :2]), dict(cache_v=v[..., :32]), dict(cache_k=k.cpu()),
           dict(cache_k=k.half(), cache_v=v.half()), dict(cache_k=k.to(I8), cache_v=v.to(I8)), dict(k_scales=s, v_scales=s), dict(pages=pages.long()),
           dict(pages=pages[:-1]), dict(spare=spare[:-1]), dict(lengths=lengths[:1]), dict(parents=parents.t()), dict(spare=spare.float()),
           dict(cache_k=k.to(I8), cache_v=v.to(I8), k_scales=s), dict(cache_k=k.to(I8), cache_v=v.to(I8), k_scales=s[..., :0], v_scales=s),
           dict(cache_k=k.to(I8), cache_v=v.to(I8), k_scales=s[:, :, :2], v_scales=s), dict(cache_k=k.to(I8), cache_v=v.to(I8), k_scales=s.half(), v_scales=s),
           dict(cache_k=k[..., 4:60], cache_v=v[..., 4:60]), dict(cache_k=k.to(I8), cache_v=v, k_scales=s, v_scales=s)]
    for kw in bad:
        with pytest.raises(ops.NativeError):
            call(**kw)
    call()


def test_keys_and_values_of_two_types_are_refused():
    (k, v, *rest), _ = make([21, 37], 4, 2, 3, 16, 64, BF16)
    with pytest.raises(ops.NativeError, match="one type"):
        ops.cache_reorder(k, v[..., :32].float(), *rest)       # (rows of as many bytes)
    ops.cache_reorder(k, v, *rest)
