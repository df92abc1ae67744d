"""One step of a search with beams against its definition in 64 bits: parents and tokens are held to be equal, scores to their rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops

BF16, F32 = torch.bfloat16, torch.float32


def bits(mask):
    """[rows, vocab] of truth values as words, the lowest bit first."""
    rows, vocab = mask.shape
    wide = torch.zeros(rows, -(-vocab // 32) * 32, dtype=torch.int64)
    wide[:, :vocab] = mask
    words = (wide.view(rows, -1, 32) << torch.arange(32)).sum(2)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32).cuda()


def reference(logits, scores, width, finished=None, mask=None):
    B, n = scores.shape
    V = logits.shape[1]
    parents, tokens = torch.empty(B, width, dtype=torch.int32), torch.empty(B, width, dtype=torch.int32)
    out = torch.full((B, width), -math.inf, dtype=torch.float64)
    logits, scores = logits.cpu().double(), scores.cpu().double()
    for b in range(B):
        table = torch.full((n, V + 1), -math.inf, dtype=torch.float64)
        for i in range(n):
            if not math.isfinite(scores[b, i]):
                continue
            if finished is not None and finished[b, i]:
                table[i, V] = scores[b, i]
                continue
            x = logits[b * n + i]
            if mask is not None:
                x = torch.where(mask[b * n + i if mask.shape[0] > 1 else 0], x, -math.inf)
            lse = torch.logsumexp(x, 0)
            if bool(torch.isfinite(lse)):
                table[i, :V] = scores[b, i] + (x - lse)
        v, at = table.view(-1).sort(descending=True, stable=True)
        for k in range(width):
            if k < v.numel() and v[k] > -math.inf:
                parents[b, k], t, out[b, k] = int(at[k]) // (V + 1), int(at[k]) % (V + 1), v[k]
                tokens[b, k] = t if t < V else -1
            else:
                parents[b, k], tokens[b, k] = k % n, -1
    return parents, tokens, out


def check(logits, scores, width=None, finished=None, mask=None):
    allowed = None if mask is None else bits(mask)
    got = ops.beam_step(logits, scores, width, finished=None if finished is None else finished.cuda(), allowed=allowed)
    want = reference(logits, scores, width or scores.shape[1], finished, mask)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    g, w = got[2].cpu().double(), want[2]
    assert torch.equal(torch.isinf(g), torch.isinf(w))
    some = ~torch.isinf(w)
    # rounded once, and a log-sum-exp that 32-bit sums are part of (5e-6)
    assert bool(((g - w).abs()[some] <= 2 ** -24 * w.abs()[some] + 5e-6).all())
    return got


def inputs(B, n, V, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = (scale * torch.randn(B * n, V, generator=g)).to(dtype).cuda()
    scores = (-10 - 3 * torch.rand(B, n, generator=g)).cuda()
    return logits, scores, g


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [1, 7, 65, 256, 257, 1000, 5003, 50304])
@pytest.mark.parametrize("B,n,width", [(1, 1, 1), (3, 4, 4), (2, 5, 10), (1, 16, 16), (2, 1, 32), (2, 32, 32), (7, 3, 2)])
def test_sizes(dtype, V, B, n, width):
    if V * n * B > 1 << 20:
        B = 1
    logits, scores, g = inputs(B, n, V, dtype, seed=V + n)
    check(logits, scores, width)
    finished = torch.rand(B, n, generator=g) < 0.3
    scores[0, -1] = -math.inf
    check(logits, scores, width, finished, torch.rand(B * n, V, generator=g) < 0.2)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [65, 3001, 50304])
def test_equal_beams_and_equal_logits(dtype, V):
    """Beams with the same row and score: the lower one first, whatever the rows' places in memory."""
    logits, scores, _ = inputs(2, 4, V, dtype)
    logits[:] = logits[::4].repeat_interleave(4, 0)
    scores[:] = scores[:, :1]
    check(logits, scores)
    check(logits, scores, 16)
    wide = torch.zeros(8, V + 3, dtype=dtype, device="cuda")
    wide[:, 1:V + 1] = logits
    check(wide[:, 1:V + 1], scores, 9)                                 # rows begin at any element
    logits[:] = 0.5                                                    # all tokens equal
    check(logits, scores, 7)
    logits[:, V // 2:] = 0.25
    check(logits, scores, 32)
    logits[:, V // 3] = 1.0
    scores[:, 2] += 0.5
    check(logits, scores, 32)


@pytest.mark.parametrize("V", [65, 3001, 50304])
@pytest.mark.parametrize("seed", range(6))
def test_beams_that_nearly_meet(V, seed):
    """Scores are made so that the best of two beams differ by 1e-9: 32 bits would not tell them apart."""
    logits, scores, g = inputs(1, 3, V, F32, seed=seed)
    x = logits.cpu().double()
    lse = torch.logsumexp(x, 1)
    best = x.amax(1) - lse
    scores = torch.empty(1, 3)
    scores[0, 0] = -10.0
    for b in (1, 2):                                                   # as near as 32 bits allow, then the logit does the rest
        scores[0, b] = float(-10.0 + best[0] - best[b])
        top = int(x[b].argmax())
        want = (-10.0 + best[0]) - scores[0, b].double()
        x[b, top] += float(want - best[b])
        logits[b, top] = float(x[b, top])
    check(logits, scores.cuda(), 3)
    check(logits, scores.cuda(), 1)


def test_rows_that_count_for_nothing():
    logits, scores, _ = inputs(3, 4, 700, F32)
    logits[1, 5] = math.nan
    logits[2, 9] = math.inf
    logits[3] = -math.inf
    logits[5, :690] = -math.inf                                        # ten tokens are left
    scores[2, 0], scores[2, 1], scores[2, 2] = math.nan, math.inf, -math.inf
    for width in (2, 4, 32):
        check(logits, scores, width)
        check(logits[:, :200], scores, width)
    mask = torch.ones(12, 700, dtype=torch.bool)
    mask[1, 5] = mask[2, 9] = False                                    # where the mask takes them out they do no harm
    mask[4:8] = False                                                  # nothing is left of a group
    check(logits, scores, 4, mask=mask)
    check(logits, scores, 4, mask=mask[:1])
    got = check(logits[4:8], scores[1:2], 6, mask=mask[4:8])
    assert got[0].tolist() == [[0, 1, 2, 3, 0, 1]] and bool((got[1] == -1).all())


@pytest.mark.parametrize("order", ["up", "down", "late"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_orders_of_the_logits(order, dtype):
    """Rows that rise, fall, or have all that counts at the end; steps of the exponent's reference among them."""
    V = 20000
    x = torch.linspace(-60, 60, V)
    if order == "down":
        x = x.flip(0)
    if order == "late":
        x = torch.cat([torch.full((V - 40,), -300.0), torch.linspace(0, 9, 40)])
    logits = torch.stack([x, x + 0.001, x.roll(7)]).to(dtype).cuda()
    check(logits, torch.tensor([[-1.0, -1.002, -1.5]]).cuda(), 8)


def test_a_captured_step_and_another_stream():
    logits, scores, _ = inputs(4, 4, 9000, BF16)
    want = ops.beam_step(logits, scores)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.beam_step(logits, scores)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.beam_step(logits, scores)
    logits.copy_(logits.flip(0))
    graph.replay()
    now = ops.beam_step(logits, scores)
    torch.cuda.synchronize()
    for a, b in ((want, other), (held, now)):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals():
    logits, scores, _ = inputs(2, 4, 300, F32)
    call = lambda **kw: ops.beam_step(**{**dict(logits=logits, scores=scores), **kw})
    f = torch.zeros(2, 4, dtype=torch.bool, device="cuda")
    words = torch.zeros(8, 10, dtype=torch.int32, device="cuda")
    bad = [dict(logits=logits.half()), dict(logits=logits[:7]), dict(logits=logits.cpu()), dict(logits=logits.t().contiguous().t()), dict(scores=scores.double()),
           dict(scores=scores[:, :3]), dict(scores=scores.t().contiguous().t()), dict(width=0), dict(width=33), dict(width=-1), dict(finished=f.int()), dict(finished=f[:1]),
           dict(allowed=words[:, :9]), dict(allowed=words[:3]), dict(allowed=words.long()), dict(logits=logits[:, :0]),
           dict(logits=logits[:1].expand(8, 300)), dict(logits=torch.zeros(66, 9, device="cuda"), scores=torch.zeros(2, 33, device="cuda"))]
    for kw in bad:
        with pytest.raises(ops.NativeError):
            call(**kw)
    with pytest.raises(TypeError):
        call(scores=1.0)
    got = call(logits=logits[:0], scores=scores[:0])
    assert [tuple(x.shape) for x in got] == [(0, 4)] * 3
    call(finished=f, allowed=words)
