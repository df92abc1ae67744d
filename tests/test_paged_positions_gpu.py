"""New tokens keep their positions where a sequence's end lies beyond what the table (or ``max_len``) holds: ``cache_append`` drops the ones
without a place, and attention shows each token the keys up to its own position that are there.

Tolerances as for paged attention in general, with A = softmax |v| and S = scale * max sum |q k|.  bf16: probabilities and result are
rounded by up to 2^-8 of themselves each, 2^-7 A * 1.02 with the sums.  fp32: 2 * (3e-6 S + 1e-6) of a probability and 4e-6 of the second
product.  A key more or less changes a row of some 60 random keys by about 1 / 60 of |v|, several times the tolerance in most columns, and
its log-sum-exp by about 1 / 60, a thousand times its own."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops

BF16, F32 = torch.bfloat16, torch.float32


def expected(q, ck, cv, pages, offsets, lengths, most):
    """(out, lse, A, S) in 64 bits: the token at position p sees keys t <= p, t < most."""
    N, H, D = q.shape
    KV, P = ck.shape[1], ck.shape[2]
    out, big = (torch.zeros(N, H, D, dtype=torch.float64, device="cuda") for _ in range(2))
    lse, S = (torch.zeros(N, H, dtype=torch.float64, device="cuda") for _ in range(2))
    for b, length in enumerate(lengths.tolist()):
        lo, hi = offsets[b].item(), offsets[b + 1].item()
        t = torch.arange(min(length, most), device="cuda")
        page = pages[b].long()[t // P]
        own = length - (hi - lo) + torch.arange(hi - lo, device="cuda")
        hidden = t[None, :] > own[:, None]
        for h in range(H):
            k, v = (c[page, h * KV // H, t % P].double() for c in (ck, cv))
            x = (q[lo:hi, h].double() @ k.T) * D ** -0.5
            S[lo:hi, h] = ((q[lo:hi, h].double().abs() @ k.abs().T) * D ** -0.5).amax(1)
            x[hidden] = -torch.inf
            p = torch.softmax(x, 1)
            out[lo:hi, h], big[lo:hi, h], lse[lo:hi, h] = p @ v, p @ v.abs(), torch.logsumexp(x, 1)
    return out, lse, big, S


def check(q, got, want):
    out, lse = (x.double() for x in got)
    w, wl, big, S = want
    if q.dtype == BF16:
        tol, ltol = 2 ** -7 * 1.02 * big, 1e-5 + 1e-6 * (S + wl.abs())
    else:
        tol, ltol = (2 * (3e-6 * S + 1e-6)[:, :, None] + 4e-6) * big, 1e-5 + 3e-6 * S + 1e-6 * wl.abs()
    assert bool(((lse - wl).abs() <= ltol).all())
    assert bool(((out - w).abs() <= tol).all())
    assert ops.attention_check_status() == 0


def make(new, lengths, heads, kv_heads, D, dtype, slots, seed, P=16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, width = len(new), slots // P
    pages = torch.randperm(B * width, generator=g, device="cuda").to(torch.int32).view(B, width)
    ck, cv = (torch.randn(B * width, kv_heads, P, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    offsets = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32).cuda()
    q = torch.randn(sum(new), heads, D, generator=g, device="cuda").to(dtype)
    k, v = (torch.randn(sum(new), kv_heads, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    return q, k, v, ck, cv, pages, offsets, torch.tensor(lengths, dtype=torch.int32).cuda()


CASES = [("single", 0), ("single", 1), ("single", 4), ("single", -5), ("rows", 1), ("rows", 2), ("tc", 1), ("tc", 2), ("auto", 0)]


@pytest.mark.parametrize("backend,splits", CASES)
@pytest.mark.parametrize("dtype,D", [(BF16, 32), (BF16, 64), (BF16, 128), (F32, 32), (F32, 64), (F32, 128)])
def test_chunks_across_the_end_of_the_table(backend, splits, dtype, D):
    if backend == "tc" and dtype == F32:
        pytest.skip("the tcgen05 kernel takes bf16")
    new, lengths = [10, 2, 40, 3, 64, 5], [70, 65, 100, 64, 127, 40]
    q, k, v, ck, cv, pages, offsets, lens = make(new, lengths, 4, 2, D, dtype, 64, 1)
    ops.cache_append(k, v, ck, cv, pages, offsets, lens)
    got = ops.paged_attention(q, ck, cv, pages, offsets, lens, backend=backend, splits=splits)
    # the first new token of the first sequence is in the cache, at position 60, and sees itself
    assert torch.equal(ck[pages[0, 3].long(), :, 12], k[0]) and torch.equal(cv[pages[0, 3].long(), :, 12], v[0])
    check(q, got, expected(q, ck, cv, pages, offsets, lens, 64))


@pytest.mark.parametrize("backend", ["single", "rows", "tc"])
@pytest.mark.parametrize("D", [64, 128])
def test_max_len_inside_a_chunk(backend, D):
    new, lengths = [30, 4, 150], [300, 201, 250]
    q, k, v, ck, cv, pages, offsets, lens = make(new, lengths, 4, 2, D, BF16, 320, 2)
    lens_cut = 290                                         # 30 tokens over 300: ten of them beyond
    got = ops.paged_attention(q, ck, cv, pages, offsets, lens, max_len=lens_cut, backend=backend)
    check(q, got, expected(q, ck, cv, pages, offsets, lens, lens_cut))


@pytest.mark.parametrize("backend,D,dtype", [("rows", 64, F32), ("rows", 32, BF16), ("tc", 64, BF16), ("tc", 128, BF16)])
def test_more_tiles_than_run_at_a_time(backend, D, dtype):
    """Tiles are taken in the order of the keys that they see."""
    new = [(b * 37) % 180 + 20 for b in range(24)]
    lengths = [256 + (b * 53) % n if b % 3 else n + b for b, n in enumerate(new)]
    q, k, v, ck, cv, pages, offsets, lens = make(new, lengths, 30, 6, D, dtype, 256, 3)
    ops.cache_append(k, v, ck, cv, pages, offsets, lens)
    got = ops.paged_attention(q, ck, cv, pages, offsets, lens, backend=backend, splits=1)
    check(q, got, expected(q, ck, cv, pages, offsets, lens, 256))
