"""The step from logits to the next token against the same steps in torch on the CPU: one IEEE operation of 32 bits each, so that
processed logits and tokens have to be equal.  The log-probability is held to 64-bit values: x and the maximum are exact, the
logarithm of a sum of up to 50304 terms, each off by 2^-21 (exponent below 2^5 and exponential), by 2e-6 and their additions
(at most 200 in a row, then a tree) 200 * 2^-24: 2e-5 with what subtracting numbers below 100 costs."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops

BF16, F32 = torch.bfloat16, torch.float32


def reference(logits, history=None, lengths=None, prompts=None, repetition=None, presence=None, frequency=None, bias_ids=None,
              bias_values=None, temperature=None, allowed=None, noise=None, processed=False):
    R, V = logits.shape
    x = logits.float().cpu().clone()
    tokens, logprobs = [], []
    of = lambda t, r, d: torch.tensor(d) if t is None else t[r].cpu()
    for r in range(R):
        if history is not None:
            n = max(0, min(int(lengths[r]), history.shape[1]))
            told = history[r, :n].cpu().tolist()
            given = int(prompts[r]) if prompts is not None else 0
            rep = of(repetition, r, 1.0)
            for t in {t for t in told if 0 <= t < V}:
                x[r, t] = x[r, t] / rep if x[r, t] > 0 else x[r, t] * rep
            made = [t for j, t in enumerate(told) if j >= given and 0 <= t < V]
            for t in set(made):
                x[r, t] = x[r, t] - of(frequency, r, 0.0) * float(made.count(t))
                x[r, t] = x[r, t] - of(presence, r, 0.0)
        if bias_ids is not None:
            last = {int(t): j for j, t in enumerate(bias_ids[r].tolist()) if 0 <= t < V}
            for t, j in last.items():
                x[r, t] = x[r, t] + bias_values[r, j].cpu()
        temp = of(temperature, r, 1.0)
        if temp > 0:
            x[r] = x[r] / temp
        if allowed is not None:
            words = allowed[r if allowed.shape[0] > 1 else 0].cpu()
            bits = ((words[:, None] >> torch.arange(32, dtype=torch.int32)) & 1).flatten()[:V]
            x[r][bits == 0] = -math.inf
        y = x[r]
        if noise is not None and temp > 0:
            y = torch.where(x[r] == -math.inf, x[r], x[r] + noise[r].cpu())
        if bool((y == -math.inf).all()):
            tokens.append(-1)
            logprobs.append(-math.inf)
            continue
        nan = torch.isnan(y)
        t = int(nan.nonzero()[0]) if bool(nan.any()) else int((y == y.max()).nonzero()[0])
        tokens.append(t)
        logprobs.append(float(x[r, t].double() - torch.logsumexp(x[r].double(), 0)))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(logprobs, dtype=torch.float64), x.to(logits.dtype)


def check(logits, **kw):
    token, logprob, out = ops.next_token(logits, processed=True, **kw)
    wt, wl, wx = reference(logits, **kw)
    assert token.dtype == torch.int32 and logprob.dtype == F32 and out.dtype == logits.dtype
    assert torch.equal(token.cpu(), wt)
    same = (out.cpu() == wx) | (torch.isnan(out.cpu()) & torch.isnan(wx))
    assert bool(same.all())
    got = logprob.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(wl)) and torch.equal(torch.isinf(got), torch.isinf(wl))
    fine = torch.isfinite(wl)
    assert bool(((got - wl).abs()[fine] <= 2e-5).all())
    t2, l2, none = ops.next_token(logits, **kw)
    assert none is None and torch.equal(t2, token) and torch.equal(l2.nan_to_num(3.0), logprob.nan_to_num(3.0))


def inputs(R, V, dtype, L=50, K=9, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=g)
    return dict(logits=(torch.randn(R, V, generator=g) * 3).to(dtype).cuda(),
                history=torch.randint(-2, V + 3, (R, L), generator=g, dtype=torch.int32).cuda(),
                lengths=torch.randint(0, L + 3, (R,), generator=g, dtype=torch.int32).cuda(),
                prompts=torch.randint(0, L, (R,), generator=g, dtype=torch.int32).cuda(),
                repetition=(0.7 + r(R)).cuda(), presence=(r(R) - 0.3).cuda(), frequency=r(R).cuda(),
                bias_ids=torch.randint(-2, V + 2, (R, K), generator=g, dtype=torch.int32).cuda(),
                bias_values=(torch.randn(R, K, generator=g) * 4).cuda(),
                temperature=(torch.arange(R) % 3 * 0.6).cuda(),
                allowed=torch.randint(-2 ** 31, 2 ** 31, (R, (V + 31) // 32), generator=g).to(torch.int32).cuda(),
                noise=-torch.log(-torch.log(r(R, V).clamp(1e-9, 1 - 1e-7))).cuda())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 2), (5, 31), (7, 65), (4, 1000), (3, 4096), (2, 4097), (9, 8195), (2, 50304), (3, 50257)])
def test_everything_at_once(dtype, R, V):
    check(**inputs(R, V, dtype))


@pytest.mark.parametrize("name", ["history", "bias_ids", "temperature", "allowed", "noise", None])
@pytest.mark.parametrize("V", [65, 5000])
def test_one_at_a_time(name, V):
    kw = inputs(4, V, BF16, seed=1)
    keep = {"history": ["history", "lengths", "prompts", "repetition", "presence", "frequency"], "bias_ids": ["bias_ids", "bias_values"]}
    check(kw["logits"], **{k: kw[k] for k in keep.get(name, [name] if name else [])})


def test_history_without_prompts_or_penalties():
    kw = inputs(4, 300, F32, seed=2)
    check(kw["logits"], history=kw["history"], lengths=kw["lengths"], presence=kw["presence"])
    check(kw["logits"], history=kw["history"], lengths=kw["lengths"])
    check(kw["logits"], history=kw["history"][:, :0], lengths=kw["lengths"])


@pytest.mark.parametrize("V", [40, 5005])
def test_rows_that_the_mask_empties(V):
    kw = inputs(6, V, BF16, seed=3)
    kw["allowed"][1] = 0
    kw["allowed"][4] = 0
    kw["allowed"][4, -1] = 1 << 30                                        # a bit behind the vocabulary allows nothing
    check(**kw)
    token, logprob, _ = ops.next_token(**kw)
    assert int(token[1]) == -1 and float(logprob[1]) == -math.inf and int(token[4]) == -1
    kw["allowed"] = kw["allowed"][1:2]                                     # one mask for all
    check(**kw)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lowest_index_of_equals(dtype):
    x = torch.zeros(3, 9000, dtype=dtype, device="cuda")
    x[1, [8999, 4500, 77]] = 2.0
    x[2, [8999, 8998]] = 1.0
    assert ops.next_token(x)[0].tolist() == [0, 77, 8998]
    # equals in what is done one by one (the ends of a row off the 16-byte boundaries, tokens of the history) and in groups
    x = torch.zeros(9, 4099, dtype=dtype, device="cuda")
    history = torch.tensor([[5], [4000], [0], [4098], [77], [1], [2], [3], [4]], dtype=torch.int32).cuda()
    assert ops.next_token(x, history=history, lengths=torch.ones(9, dtype=torch.int32).cuda())[0].tolist() == [0] * 9
    for row in range(9):
        x[row, row:] = 1.0
        x[row, 4000] = 1.0
    assert ops.next_token(x, history=history, lengths=torch.ones(9, dtype=torch.int32).cuda())[0].tolist() == list(range(9))


@pytest.mark.parametrize("V", [50, 9000])
def test_infinities_and_nan(V):
    kw = inputs(8, V, F32, seed=4)
    x, low = kw["logits"], torch.finfo(F32).min
    x[0, 5], x[1, 6], x[2, 7] = math.inf, -math.inf, math.nan
    x[3], x[4, :] = -math.inf, low
    x[5, 1:], x[6, V - 1] = low, math.nan
    free = {k: v for k, v in kw.items() if k not in ("allowed", "noise")}
    check(**free)
    kw["allowed"][:] = -1
    for row, v in ((0, 5), (2, 7), (6, V - 1)):                             # masked: nothing of them is left
        kw["allowed"][row, v // 32] &= ~(1 << (v % 32)) if v % 32 < 31 else 0x7fffffff
    kw["noise"][2, 7] = math.nan
    check(**kw)
    assert bool(torch.isfinite(ops.next_token(**kw)[1][2]))


def test_long_history():
    kw = inputs(2, 50304, BF16, L=20000, seed=5)
    kw["lengths"][:] = torch.tensor([20000, 19999])
    check(**kw)
    kw = inputs(1, 65, BF16, L=5000, seed=6)
    kw["lengths"][:] = 5000
    check(**kw)


def test_rows_apart_and_streams():
    kw = inputs(5, 1000, BF16, seed=7)
    wide = torch.randn(5, 1008).to(BF16).cuda()
    for view in (wide[:, :1000], wide[:, 3:1003], wide[:, 8:1008]):
        kw["logits"] = view
        check(**kw)
    side = torch.cuda.Stream()
    want = ops.next_token(**kw)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.next_token(**kw)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_samples_follow_the_softmax():
    """200000 samples of eight tokens: a frequency is off by 5 standard deviations, sqrt(p (1 - p) / n), with a chance of 6e-7 each."""
    n = 200000
    p = torch.tensor([0.4, 0.25, 0.15, 0.1, 0.05, 0.03, 0.015, 0.005])
    u = torch.rand(n, 8, generator=torch.Generator().manual_seed(11)).clamp_(1e-9, 1 - 1e-7)
    token, logprob, _ = ops.next_token(p.log().expand(n, 8).contiguous().cuda(), noise=(-torch.log(-torch.log(u))).cuda())
    share = torch.bincount(token.cpu().long(), minlength=8) / n
    assert bool(((share - p).abs() < 5 * torch.sqrt(p * (1 - p) / n)).all())
    assert bool(((logprob.cpu() - p.log()[token.cpu().long()]).abs() < 1e-5).all())


def test_no_rows_and_refusals():
    kw = inputs(3, 100, BF16)
    t, l, x = ops.next_token(kw["logits"][:0], processed=True)
    assert t.shape == (0,) and l.shape == (0,) and x.shape == (0, 100)
    bad = [dict(logits=kw["logits"].half()), dict(logits=kw["logits"].cpu()), dict(logits=kw["logits"][0]), dict(logits=kw["logits"].t()),
           dict(logits=kw["logits"][:1].expand(3, 100)), dict(logits=kw["logits"][:, :0]), dict(lengths=None), dict(history=kw["history"].long()),
           dict(history=kw["history"][:2]), dict(repetition=kw["repetition"].double()), dict(presence=kw["presence"][:2]),
           dict(bias_ids=None), dict(bias_values=kw["bias_values"][:, :3]), dict(allowed=kw["allowed"][:2]), dict(allowed=kw["allowed"][:, :2]),
           dict(noise=kw["noise"].to(BF16)), dict(noise=kw["noise"][:, :50]), dict(temperature=kw["temperature"].cpu())]
    for b in bad:
        with pytest.raises(ops.NativeError):
            ops.next_token(**{**kw, **b})
    with pytest.raises(TypeError):
        ops.next_token(**{**kw, "noise": 1.0})
