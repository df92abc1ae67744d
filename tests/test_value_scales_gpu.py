"""Attention over a cache of 8-bit integers whose blocks' scales lie very far apart, each row against 64 bits by what it sees itself.

p is the softmax, A = sum p |v|, S = scale * max sum |q k|, w = max p sv over the keys that a row sees, n their number.  bf16 queries:
* a score is off by its sum's roundings, below 3e-6 S, its factors, 2^-22 S, and the logarithm of sv that is added to it (up to 128, rounded twice: 2^-16), p by twice
  that and the exponential's 2^-20;
* a probability times its sv is rounded to fp16, 2^-11, and where it is below 2^-14 of what is 2^7 at its largest to 2^-25; times an integer up to 2^7,
  over that 2^7: 2^-25 w for each key.  (The reference maximum may lag behind by 2^8, which makes the numbers larger.)
* the result is rounded to bf16, 2^-8; below bf16's normal numbers by 2^-134.
* log-sum-exp: 3e-6 S and, as log2 sv is added to the exponents and taken from the sum, the roundings of numbers up to 128, 2^-15 with the sum's logarithm.
* a scale of values below 2^-100 of the largest one of the call counts as zero: 2^-93 of that for each key.
|error| <= (2^-11 + 6e-6 S + 2^-14) A + 2^-25 n w + 2^-8 |out| + 2^-93 n (largest sv) [only where scales reach so far] + 2^-134.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops

BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8
HEADS, PAGE, BLOCK = 2, 16, 8
FORMS = [("tc", 0), ("tc", 3), ("rows", 0), ("single", 0), ("single", 2)]


def case(n, length, D, sk, sv, q_scale=1.0, seed=0):
    """One sequence; ``sk``, ``sv``: scales of its blocks, one for all heads."""
    g = torch.Generator().manual_seed(seed)
    pages = -(-length // PAGE)
    ck, cv = (torch.randint(-127, 128, (pages, HEADS, PAGE, D), generator=g).to(I8) for _ in range(2))
    q = (q_scale * torch.randn(n, HEADS, D, generator=g)).to(BF16)
    scales = [torch.tensor((list(s) + [1.0])[:2 * pages], dtype=F32).view(pages, 1, 2).expand(-1, HEADS, -1).contiguous() for s in (sk, sv)]
    assert len(sk) == len(sv) == -(-length // BLOCK)
    table = torch.arange(pages, dtype=torch.int32).view(1, -1)
    args = (q, ck, cv, table, torch.tensor([0, n], dtype=torch.int32), torch.tensor([length], dtype=torch.int32))
    return [a.cuda() for a in args], dict(k_scales=scales[0].cuda(), v_scales=scales[1].cuda())


def check(args, scales, got, scale, beyond=False):
    q, ck, cv, _, offsets, lengths = (a.cpu() for a in args)
    n, length, D = q.shape[0], int(lengths[0]), q.shape[2]
    ks, vs = (s.cpu().double().repeat_interleave(BLOCK, 2) for s in (scales["k_scales"], scales["v_scales"]))
    flat = lambda c: c.transpose(0, 1).reshape(HEADS, -1, *c.shape[3:])[:, :length]
    k, v, sv = flat(ck.double() * ks[..., None]), flat(cv.double() * vs[..., None]), flat(vs)
    sv = torch.where(sv < 2.0 ** -100, 0.0, sv)
    v = torch.where(sv[..., None] > 0, v, 0.0)
    seen = torch.arange(length)[None, :] <= (length - n + torch.arange(n))[:, None]
    x = torch.einsum("nhd,hld->hnl", q.double(), k) * scale
    S = (torch.einsum("nhd,hld->hnl", q.double().abs(), k.abs()) * scale * seen).amax(2)[..., None]
    x[:, ~seen] = -math.inf
    lse = torch.logsumexp(x, 2)
    p = torch.exp(x - lse[..., None])
    want, A = p @ v, p @ v.abs()
    w = (p * sv[:, None, :]).amax(2)[..., None]
    count = seen.sum(1)[None, :, None]
    tol = (2 ** -11 + 6e-6 * S + 2 ** -14) * A + 2.0 ** -25 * count * w + 2 ** -8 * want.abs() + 2.0 ** -134
    if beyond:
        tol = tol + 2.0 ** -93 * count * sv.amax()
    out, got_lse = got[0].cpu().double().transpose(0, 1), got[1].cpu().double().transpose(0, 1)
    error = (out - want).abs()
    assert bool((error <= tol).all()), ((error / tol).max(), (error > tol).sum())
    assert bool(((got_lse - lse).abs() <= 2 ** -15 + 4e-6 * S[..., 0] + 1e-6 * lse.abs()).all())
    assert float((tol <= 0.03 * A).double().mean()) > 0.9 or beyond      # (the bound binds)
    assert ops.attention_check_status() == 0


@pytest.mark.parametrize("backend,splits", [("tc", 0), ("tc", 3)])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("small", [-20, -40, -60])
def test_rows_that_see_small_blocks_only(backend, splits, D, small):
    """Blocks of a tile that early rows do not see are larger by 2^20 to 2^60."""
    blocks = 30
    sv = [2.0 ** small if b < 3 else 2.0 ** (small / 2) if b < 12 else 1.5 for b in range(blocks)]
    args, scales = case(233, 233, D, [0.01] * blocks, sv)
    check(args, scales, ops.paged_attention(*args, **scales, backend=backend, splits=splits), D ** -0.5)


@pytest.mark.parametrize("backend,splits", FORMS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("low,high", [(-99, 10), (-99, 12), (-95, 20), (-30, 60), (40, 80), (60, -30)])
def test_scales_that_grow_along_a_sequence(backend, splits, D, low, high):
    """The last keys' scales are up to 2^115 times the first ones'."""
    blocks = 30
    sv = [2.0 ** (low + (high - low) * (b // 5) / 5) for b in range(blocks)]
    args, scales = case(100, 240, D, [0.01] * blocks, sv, seed=1)
    check(args, scales, ops.paged_attention(*args, **scales, backend=backend, splits=splits), D ** -0.5, beyond=high - low > 90)


@pytest.mark.parametrize("backend,splits", FORMS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [0.0, 2.0 ** -110, 2.0 ** -99])
def test_blocks_of_no_values(backend, splits, D, value):
    """All values of a row, or all but few, count as zeros; their probabilities count all the same."""
    blocks = 30
    for sv in ([value] * blocks, [value] * 20 + [3.0] * 10, [value] * 3 + [2.0 ** 40] + [value] * 26, [2.0 ** 40] + [value] * 29):
        args, scales = case(200, 240, D, [0.01] * blocks, sv, seed=2)
        check(args, scales, ops.paged_attention(*args, **scales, backend=backend, splits=splits), D ** -0.5, beyond=True)


@pytest.mark.parametrize("backend,splits", FORMS)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("power", [-90, -60, 60, 90])
def test_large_queries_and_small_keys(backend, splits, D, power):
    """Queries times 2^-power, keys times 2^power: the scores are what they were."""
    args, scales = case(100, 240, D, [0.01 * 2.0 ** power] * 30, [0.02] * 30, q_scale=2.0 ** -power, seed=3)
    check(args, scales, ops.paged_attention(*args, **scales, backend=backend, splits=splits), D ** -0.5)


@pytest.mark.parametrize("backend,splits", [f for f in FORMS if f[0] != "tc"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("small", [-20, -40, -60])
def test_rows_that_see_small_blocks_only_by_warps(backend, splits, D, small):
    test_rows_that_see_small_blocks_only(backend, splits, D, small)


@pytest.mark.parametrize("dtype,backend,splits", [(BF16, *f) for f in FORMS] + [(F32, *f) for f in FORMS if f[0] != "tc"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("n,length", [(8, 20), (100, 140)])
@pytest.mark.parametrize("behind", [0.0, 2.0 ** -60, 2.0 ** 60, math.inf, math.nan])
def test_bits_hang_on_what_a_row_sees(dtype, backend, splits, D, n, length, behind):
    """The scales of blocks that a row does not see, of keys or of values, may be anything."""
    blocks = -(-length // BLOCK)
    args, scales = case(n, length, D, [0.01] * blocks, [0.02] * blocks, seed=4)
    args[0] = args[0].to(dtype)
    clean = ops.paged_attention(*args, **scales, backend=backend, splits=splits)
    at = length - n // 2
    first = -(-at // BLOCK)                                  # of the changed blocks
    rows = first * BLOCK - (length - n)                      # those before it
    assert 0 < rows < n
    for which in scales:
        other = {name: s.clone() for name, s in scales.items()}
        for b in range(first, blocks):
            other[which][b // 2, :, b % 2] = behind
        got = ops.paged_attention(*args, **other, backend=backend, splits=splits)
        for x, y in zip(clean, got):
            assert torch.equal(x[:rows], y[:rows])
        if behind == math.nan or behind == math.inf and which == "v_scales":
            assert bool(got[0][rows:].isnan().any())
    assert ops.attention_check_status() == 0
