"""The order of continuations whose values are the same in 64 bits: within a beam that of their logits, between beams the lower one first."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops

BF16, F32 = torch.bfloat16, torch.float32


def expected(logits, scores, width):
    """By value in 64 bits, beam, logit, token."""
    B, n = scores.shape
    V = logits.shape[1]
    x = logits.cpu().double().view(B, n, V)
    value = scores.cpu().double()[..., None] + (x - torch.logsumexp(x, 2, keepdim=True))
    parents, tokens = [], []
    for b in range(B):
        rows = []
        for i in range(n):                                             # a beam's best by logit are its best by value
            best = x[b, i].sort(descending=True, stable=True).indices[:width].tolist()
            rows += [(-float(value[b, i, t]), i, -float(x[b, i, t]), t) for t in best]
        rows = sorted(rows)[:width]
        rows += [(0.0, k % n, 0.0, -1) for k in range(len(rows), width)]
        parents.append([r[1] for r in rows])
        tokens.append([r[3] for r in rows])
    return torch.tensor(parents, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)


def check(logits, scores, width):
    parents, tokens, _ = ops.beam_step(logits, scores, width)
    want = expected(logits, scores, width)
    assert torch.equal(tokens.cpu(), want[1]) and torch.equal(parents.cpu(), want[0])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [3, 65, 256, 257, 3001, 50304])
@pytest.mark.parametrize("width", [1, 5, 32])
def test_logits_too_near_for_the_value(dtype, V, width):
    """Logits of 1e-20 and less: a value of -11 is the same for all of them."""
    g = torch.Generator().manual_seed(V)
    # (distinct in bf16 too: powers of two and their multiples with 7 more bits)
    small = (2.0 ** torch.randint(-120, -70, (V,), generator=g).double()) * (1 + torch.randint(0, 128, (V,), generator=g).double() / 128)
    small = torch.where(torch.rand(V, generator=g) < 0.5, small, -small)
    logits = torch.stack([small, small.flip(0), small.roll(5)]).to(dtype).cuda()
    check(logits[:1], torch.tensor([[-3.0]]).cuda(), width)
    check(logits, torch.tensor([[-3.0, -3.5, -2.0]]).cuda(), width)
    check(logits, torch.tensor([[-3.0], [-1000.0], [0.0]]).cuda(), width)


@pytest.mark.parametrize("V", [65, 3001, 50304])
def test_a_large_score_over_near_logits(V):
    """A score of -1e12 leaves 2^-13 of the values' differences."""
    g = torch.Generator().manual_seed(V)
    logits = torch.randn(2, V, generator=g) * 1e-5
    logits[:, V // 2] = 3e-5
    logits[:, V - 1] = 4e-5
    check(logits.cuda(), torch.tensor([[-1e12], [-2e12]]).cuda(), 8)
    check(logits.cuda(), torch.tensor([[-1e12, -2e12]]).cuda(), 8)
