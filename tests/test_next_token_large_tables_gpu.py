"""Vocabularies and histories whose marks and records fill more shared memory than a cluster has: tokens, processed logits and log-probabilities
against the same steps in torch, one IEEE operation of 32 bits each (tokens and logits equal; the log-probability within 2e-5 of its 64-bit value, as
for smaller vocabularies: terms off by 2^-21 of themselves each, at most 200 additions in a row, and what subtracting numbers below 100 costs)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops


def expected(x, history, lengths, prompts, repetition, presence, frequency, bias_ids, bias_values, temperature, allowed, noise):
    R, V = x.shape
    x = x.float().clone()
    at = torch.arange(history.shape[1], device="cuda")
    told = at < lengths[:, None]
    count = lambda where: torch.zeros(R, V + 1, device="cuda").scatter_add_(1, torch.where(where & (history >= 0) & (history < V), history, V).long(),
                                                                             torch.ones(history.shape, device="cuda"))[:, :V]
    seen, made = count(told) > 0, count(told & (at >= prompts[:, None]))
    rep = repetition[:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(made > 0, (x - frequency[:, None] * made) - presence[:, None], x)
    for r in range(R):
        for t, b in zip(bias_ids[r].tolist(), bias_values[r]):           # (no token twice)
            if 0 <= t < V:
                x[r, t] += b
    t = temperature[:, None]
    x = torch.where(t > 0, x / torch.where(t > 0, t, 1.0), x)
    v = torch.arange(V, device="cuda")
    x = torch.where((allowed[:, v // 32] >> (v % 32)) & 1 > 0, x, -torch.inf)
    y = torch.where((t > 0) & (x > -torch.inf), x + noise, x)
    token = torch.where(y == y.amax(1, keepdim=True), v, V).amin(1)      # the lowest of equals
    logprob = x.double().gather(1, token[:, None])[:, 0] - torch.logsumexp(x.double(), 1)
    return token, logprob, x


# (rows apart by 3 tokens more than a row: no 16-byte boundaries in common with the noise's)
@pytest.mark.parametrize("V,L,apart", [(100000, 16000, 0), (106000, 16384, 0), (128256, 16384, 0), (128256, 13000, 3), (151936, 40000, 0), (151936, 40000, 3), (262147, 30000, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_vocabulary_and_long_history(V, L, apart, dtype):
    R, K = 3, 20
    g = torch.Generator(device="cuda").manual_seed(V + L)
    r = lambda *s: torch.rand(*s, generator=g, device="cuda")
    logits = (torch.randn(R, V + apart, generator=g, device="cuda") * 3).to(dtype)[:, :V]
    history = (r(R, L) * (V + 6)).to(torch.int32) - 3
    history[0, L // 2:] = history[0, :L - L // 2].clone()                # tokens that come twice
    lengths = torch.tensor([L, L - 1, 7], dtype=torch.int32, device="cuda")
    prompts = torch.tensor([L // 3, 0, 3], dtype=torch.int32, device="cuda")
    kw = dict(history=history, lengths=lengths, prompts=prompts, repetition=0.7 + r(R), presence=r(R) - 0.3, frequency=r(R),
              bias_ids=torch.stack([torch.randperm(V + 4, generator=g, device="cuda")[:K] - 2 for _ in range(R)]).to(torch.int32),
              bias_values=torch.randn(R, K, generator=g, device="cuda") * 4, temperature=torch.tensor([0.0, 0.8, 1.3], device="cuda"),
              allowed=torch.randint(-2 ** 31, 2 ** 31, (R, (V + 31) // 32), generator=g, device="cuda").to(torch.int32),
              noise=-torch.log(-torch.log(r(R, V).clamp(1e-9, 1 - 1e-7))))
    token, logprob, out = ops.next_token(logits, processed=True, **kw)
    want, wl, wx = expected(logits, **kw)
    assert torch.equal(token.long(), want) and torch.equal(out, wx.to(dtype))
    assert bool(((logprob.double() - wl).abs() <= 2e-5).all())
    again = ops.next_token(logits, processed=True, **kw)
    assert all(torch.equal(a, b) for a, b in zip(again, (token, logprob, out)))


def test_the_lowest_of_equals_across_slices():
    V = 151936
    x = torch.zeros(4, V, device="cuda")
    for row, at in enumerate(([V - 1, V // 2, 9500], [V - 1, V - 2], [75968, 75967], [9496, 18992, 28488])):
        x[row, at] = 2.0
    history = torch.full((4, 30000), -1, dtype=torch.int32, device="cuda")
    history[2, 0], history[3, 5] = 75967, 9496
    lengths = torch.full((4,), 30000, dtype=torch.int32, device="cuda")
    assert ops.next_token(x, history=history, lengths=lengths)[0].tolist() == [9500, V - 2, 75967, 9496]
    assert ops.next_token(x[:, :V - 1].contiguous(), history=history, lengths=lengths)[0].tolist() == [9500, V - 2, 75967, 9496]
